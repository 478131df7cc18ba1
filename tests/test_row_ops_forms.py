"""What the 8-bit product's query of its tile answers and refuses: no GPU needed."""
import ctypes as C


def test_the_tile_query_refuses_what_the_product_refuses():
    from lssvc_amd import _lib
    f = lambda rows=8, cols=64, br=1, e8m0=1: C.byref(_lib.Fp8(4096, 8192, rows, 64, 4, cols, br, e8m0, 0))
    r, c = C.c_int32(), C.c_int32()
    t = lambda a, w, dtype=0, rows=r: _lib.lib.lssvc_matmul_fp8_tile(a, w, dtype, rows and C.byref(rows), C.byref(c))
    assert t(f(), f(32, br=128)) == 0 and (r.value, c.value) == (16, 16)
    assert t(f(), f(32)) != 0 and t(f(), f(32, 63, 128)) != 0 and t(f(), f(32, br=128, e8m0=0)) != 0 and t(f(), f(32, br=128), 3) != 0 and t(f(), f(32, br=128), 0, None) != 0
