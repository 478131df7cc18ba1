"""What the 8-bit product's query of its tile answers and refuses: no GPU needed."""
import ctypes as C


def test_the_tile_query_refuses_what_the_product_refuses():
    from lssvc_amd import _lib
    f = lambda rows=8, cols=64, br=1, e8m0=1: C.byref(_lib.Fp8(4096, 8192, rows, 64, 4, cols, br, e8m0, 0))
    r, c = C.c_int32(), C.c_int32()
    t = lambda a, w, dtype=0, rows=r: _lib.lib.lssvc_matmul_fp8_tile(a, w, dtype, rows and C.byref(rows), C.byref(c))
    assert t(f(), f(32, br=128)) == 0 and (r.value, c.value) == (16, 16)
    assert t(f(), f(32)) != 0 and t(f(), f(32, 63, 128)) != 0 and t(f(), f(32, br=128, e8m0=0)) != 0 and t(f(), f(32, br=128), 3) != 0 and t(f(), f(32, br=128), 0, None) != 0


def test_sizes_beyond_the_operators_range():
    """The workspace's size of what no call takes is 0, not a number that has overflowed; the call says what is wrong."""
    from lssvc_amd import _lib
    size, big = _lib.lib.lssvc_group_norm_workspace_bytes, 2 ** 31 - 1
    for args in ((8, 1, big, 1), (big, 1, big, big), (big, big, big, 1), (2 ** 40, 1, 64, 4), (2 ** 39, 1, 64, 4), (big, big, 2 ** 30, 2 ** 30), (2 ** 62, 2, 8, 8), (8, 1, 2 ** 30 + 1, 1)):
        for dtype in (_lib.F32, _lib.BF16):
            for fp8 in (0, 1):
                assert size(*args, dtype, fp8) == 0, args
    assert size(2 ** 30, 1, 64, 4, 0, 0) > 0 and size(60000, 1, 2 ** 20, 32, 0, 0) > 0
    row = lambda rows, cols, at: C.byref(_lib.Rows(at, rows, cols, cols, 0))
    for rows, images, cols in ((2 ** 39, 1, 64), (big, big, 2 ** 20)):
        assert _lib.lib.lssvc_group_norm(row(rows, cols, 1 << 12), images, 1, None, None, 1e-5, 0, 0.0, row(rows, cols, 1 << 62), None, None, 0, None) != 0
        assert b"too large" in _lib.lib.lssvc_last_error()


def test_scales_with_room_behind_a_row_are_read_in_place():
    import torch
    from lssvc_amd.row_ops import _whole_dwords
    store = torch.zeros(64, dtype=torch.uint8)
    at = lambda rows, kb, ld, off=0, step=1: store.as_strided((rows, kb), (ld, step), off).view(torch.float8_e8m0fnu)
    for rows, kb, ld, off in ((4, 2, 4, 0), (1, 4, 4, 60), (1, 1, 99, 60), (16, 1, 4, 0), (15, 3, 4, 4), (3, 5, 8, 40), (2, 4, 60, 0), (1, 61, 64, 0)):
        assert _whole_dwords(at(rows, kb, ld, off)), (rows, kb, ld, off)
    for rows, kb, ld, off, step in ((4, 2, 2, 0, 1), (4, 2, 6, 0, 1), (1, 2, 4, 61, 1), (1, 2, 4, 62, 1), (4, 2, 4, 2, 1), (2, 2, 4, 58, 1), (4, 2, 0, 0, 1), (4, 3, 16, 0, 2), (4, 5, 4, 0, 1)):
        assert not _whole_dwords(at(rows, kb, ld, off, step)), (rows, kb, ld, off, step)
    short = torch.zeros(10, dtype=torch.uint8).as_strided((2, 2), (8, 1)).view(torch.float8_e8m0fnu)      # its last row ends with the memory
    assert not _whole_dwords(short)


def test_workspace_holds_what_the_passes_hand_on():
    """Sums of 16 bytes per chunk and group; per-channel values only where a pass of their own joins the chunks."""
    from lssvc_amd import _lib
    size = _lib.lib.lssvc_group_norm_workspace_bytes
    assert size(3000, 3000, 8200, 1, _lib.F16, 0) == 16 * 3000 * 9                       # 9 pieces of a group, joined by the last pass
    assert size(20000, 1, 200, 8, _lib.F32, 0) < 16 * 1024 * 8
    many = size(1152 * 1920, 1, 48, 8, _lib.F32, 0)
    assert many >= 12 * 48 and (many - 12 * 48) % (16 * 8) == 0 and many < 1 << 20
