"""Calls that torch would follow only in part are refused: no GPU needed."""
import pytest
import torch


@pytest.fixture
def here(monkeypatch):
    """What every operator asks first, on a machine without a GPU."""
    from lssvc_amd import row_ops
    monkeypatch.setattr(row_ops, "_current_device", lambda: 0)
    return lambda: row_ops._elsewhere(torch.device("cuda:0"))


def test_traces_and_transforms_are_refused(here):
    from torch.fx.experimental.proxy_tensor import make_fx
    from lssvc_amd.row_ops import LssvcHipError
    assert here() is False
    x, calls = torch.randn(2, 3), []

    def f(x):
        calls.append(1)
        here()
        return x.sum()
    for run in (lambda: torch.jit.trace(f, x), lambda: make_fx(f)(x), lambda: torch.func.vmap(f)(x), lambda: torch.func.grad(f)(x), lambda: torch.func.jvp(f, (x,), (x,)),
                lambda: torch.func.functionalize(f)(x)):
        n = len(calls)
        with pytest.raises(LssvcHipError, match="traced or transformed"):
            run()
        assert len(calls) > n
    from torch.utils.flop_counter import FlopCounterMode
    with FlopCounterMode(display=False):                              # a mode that records nothing is no hindrance
        assert here() is False
    assert here() is False


def test_derivatives_are_refused_in_both_modes(here):
    from torch.autograd import forward_ad
    from lssvc_amd import row_ops
    x = torch.randn(3, 4)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        ask = lambda *tensors: row_ops._elsewhere(torch.device("cuda:0"), *tensors)
        assert ask(x, None, forward_ad.unpack_dual(d).primal) is False
        for others in ((d,), (x, None, d)):
            with pytest.raises(row_ops.LssvcHipError, match="tangent"):
                ask(*others)
        with torch.no_grad(), pytest.raises(row_ops.LssvcHipError, match="tangent"):       # (which leaves forward mode on)
            ask(d)
    x.requires_grad_()
    with pytest.raises(row_ops.LssvcHipError, match="gradient"):
        row_ops._no_grad(x, "x")
    with torch.no_grad():
        row_ops._no_grad(x, "x")


def test_a_plan_is_recorded_from_its_own_thread_only(here):
    """One thread records a frame plan: its own row operators are refused, another thread's launches and buffers are left alone."""
    import ctypes as C
    import threading
    from lssvc_amd import _lib, hip_ops
    from lssvc_amd.plan_compiler import Recorder
    cpu = torch.device("cpu")
    bad = lambda: _lib.lib.lssvc_fill_zero(C.c_void_p(None), 4, C.c_void_p(None))        # refused on the host, wherever it is called
    got = {}

    def other():
        got["elsewhere"] = here()
        got["status"] = bad()
        t = hip_ops.T.empty(2, 2, 4, cpu)
        got["in arena"] = rec.arena.buf.data_ptr() <= t.buf.data_ptr() < rec.arena.buf.data_ptr() + rec.arena.buf.numel()
        got["recording"] = hip_ops.recording()
    rec = Recorder(cpu, 1 << 16, [], {}, {}, {})
    with rec:
        assert hip_ops.recording()
        with pytest.raises(_lib.LssvcHipError, match="frame plans"):
            here()
        t = hip_ops.T.empty(2, 2, 4, cpu)
        assert rec.arena.buf.data_ptr() <= t.buf.data_ptr() < rec.arena.buf.data_ptr() + rec.arena.buf.numel()
        thread = threading.Thread(target=other)
        thread.start()
        thread.join()
        assert rec.launches == []
        assert bad() != 0 and len(rec.launches) == 1
    assert got == {"elsewhere": False, "status": got["status"], "in arena": False, "recording": False} and got["status"] != 0
    assert not hip_ops.recording() and here() is False


def test_arguments_of_other_types_are_refused_by_name(here):
    from lssvc_amd import row_ops
    E, rows = row_ops.LssvcHipError, row_ops.Fp8Rows.empty
    a, w = rows(8, 64, "cpu"), rows(16, 64, "cpu", 128)
    for call, text in ((lambda: row_ops.matmul_fp8(a, w), "no CPU path"), (lambda: row_ops._act_code([]), "activation"), (lambda: row_ops._act_code(1), "activation"),
                       (lambda: row_ops._whole(4.0, "groups"), "groups"), (lambda: row_ops._whole("4", "images"), "images"), (lambda: row_ops._number(None, "eps"), "eps"),
                       (lambda: row_ops._number("a", "slope"), "slope"), (lambda: row_ops._number("0.1", "slope"), "slope"), (lambda: row_ops._number(torch.tensor(1e-5), "eps"), "tensor"),
                       (lambda: rows(8, 64, "cpu", 1.0), "block_rows"), (lambda: rows(8.0, 64, "cpu"), "rows"), (lambda: rows(8, None, "cpu"), "cols")):
        with pytest.raises(E, match=text):
            call()
    import numpy as np
    assert row_ops._whole(np.int64(4), "groups") == 4 and row_ops._number(1, "eps") == 1.0 and row_ops._number(np.float32(0.5), "slope") == 0.5


INSIDE_TORCH = ("_cuda_getCurrentRawStream", "_cuda_getDevice", "_is_tracing", "_len_torch_dispatch_stack", "_functorch")


def without_private_names(monkeypatch):
    """The module as it is on a torch whose inner names are others."""
    import importlib.util
    from lssvc_amd import row_ops

    class Inner:
        def __getattr__(self, name):
            if name in INSIDE_TORCH:
                raise AttributeError(name)
            return getattr(inner, name)
    inner = torch._C
    monkeypatch.setattr(torch, "_C", Inner())
    spec = importlib.util.spec_from_file_location("lssvc_amd.row_ops_elsewhere", row_ops.__file__)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(torch, "_C", inner)
    return module


def test_the_module_does_not_need_names_inside_torch(monkeypatch):
    module = without_private_names(monkeypatch)
    assert module._current_device is torch.cuda.current_device and module._tracing is torch.jit.is_tracing
    monkeypatch.setattr(torch.cuda, "current_stream", lambda index: type("S", (), {"cuda_stream": 7 + index}))
    assert module._raw_stream(2) == 9
    monkeypatch.setattr(module, "_current_device", lambda: 0)
    assert module._elsewhere(torch.device("cuda:0")) is False and module._elsewhere(torch.device("cuda:1")) is True


def test_dequantize_at_the_ends_of_the_scales():
    """2^-127, which is no normal number, and the byte that stands for NaN."""
    from lssvc_amd.row_ops import Fp8Rows
    q = Fp8Rows.empty(4, 200, "cpu")
    q.values[:] = torch.full((4, 200), 1.5).to(torch.float8_e4m3fn)
    q.scale.view(torch.uint8)[:] = torch.tensor([[0, 1], [254, 255], [127, 126], [253, 2]], dtype=torch.uint8)
    got = q.dequantize(torch.float64)
    want = 1.5 * torch.exp2(torch.tensor([[-127.0, -126], [127, 0], [0, -1], [126, -125]], dtype=torch.float64))
    want[1, 1] = float("nan")
    assert torch.equal(got[:, 0].nan_to_num(7), want[:, 0]) and torch.equal(got[:, 199].nan_to_num(7), want[:, 1].nan_to_num(7))
