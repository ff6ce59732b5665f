"""The entry points of 8-bit rows and of products with weights of 8 and 4 bits against the stand-in for the CUDA runtime: what they refuse
(nothing is launched then), and what they launch."""
import ctypes
from ctypes import c_float, c_int, c_longlong, c_void_p

import pytest

from test_launchers_host import compiled  # noqa: F401  (the fixture)

MB = 1 << 20


def p(mb, extra=0):
    return c_void_p(mb * MB * 16 + extra)


NORM = dict(x=p(1), delta=p(2), delta_dtype=1, gain=p(3), gain_dtype=1, total=p(1), q=p(4), scales=p(5), rows=4, size=64, eps=1e-6)
NORM_TYPES = (c_void_p, c_void_p, c_int, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_int, c_int, c_float)
ROWS = dict(x=p(1), dtype=1, ldx=64, q=p(2), ldq=64, scales=p(3), rows=4, size=64)
ROWS_TYPES = (c_void_p, c_int, c_longlong, c_void_p, c_longlong, c_void_p, c_int, c_int)
E4M3 = dict(x=p(1), ldx=64, xs=p(2), w=p(3), ldw=64, ws=p(4), out=p(5), out_dtype=1, ldo=48, M=4, N=48, K=64)
E4M3_TYPES = (c_void_p, c_longlong, c_void_p, c_void_p, c_longlong, c_void_p, c_void_p, c_int, c_longlong, c_int, c_int, c_int)
INT4 = dict(x=p(1), ldx=64, w=p(2), ldw=64, scales=p(3), zeros=p(4), lds=2, group=32, out=p(5), ldo=48, M=4, N=48, K=64)
INT4_TYPES = (c_void_p, c_longlong, c_void_p, c_longlong, c_void_p, c_void_p, c_longlong, c_int, c_void_p, c_longlong, c_int, c_int, c_int)


def call(lib, entry, types, given, **changed):
    fn = getattr(lib, entry)
    fn.argtypes = [*types, c_void_p]
    before = lib.fake_launches()
    rc = fn(*{**given, **changed}.values(), None)
    return rc, lib.fake_launches() - before


def refused(lib, entry, types, given, cases):
    assert call(lib, entry, types, given) == (0, 1)
    for changed in cases:
        rc, launched = call(lib, entry, types, given, **changed)
        assert rc == -1 and launched == 0, changed
        lib.llme_last_error.restype = ctypes.c_char_p
        assert lib.llme_last_error()


def test_rows_of_8_bits(compiled):  # noqa: F811
    lib = compiled("rows_e4m3")
    refused(lib, "llme_rmsnorm_e4m3", NORM_TYPES, NORM,
            [dict(x=None), dict(gain=None), dict(q=None), dict(scales=None), dict(size=0), dict(eps=0.0), dict(eps=float("nan")), dict(total=None),
             dict(delta_dtype=2), dict(gain_dtype=7), dict(total=p(2)), dict(total=p(1, 16)), dict(q=p(1)), dict(q=p(2, 256)), dict(q=p(3)), dict(scales=p(4)),
             dict(scales=p(1, 64)), dict(delta=p(1))])
    assert call(lib, "llme_rmsnorm_e4m3", NORM_TYPES, NORM, delta=None, total=None) == (0, 1)
    for entry, more in (("llme_rows_e4m3", {}), ("llme_swiglu_e4m3", dict(ldx=128))):
        given = {**ROWS, **more}
        refused(lib, entry, ROWS_TYPES, given, [dict(x=None), dict(q=None), dict(scales=None), dict(size=0), dict(ldx=given["ldx"] - 1), dict(ldq=63),
                                                dict(dtype=3), dict(q=p(1, 128)), dict(scales=p(2)), dict(scales=p(1))])
    for entry, types, given in (("llme_rmsnorm_e4m3", NORM_TYPES, NORM), ("llme_rows_e4m3", ROWS_TYPES, ROWS)):
        assert call(lib, entry, types, given, rows=0) == (0, 0)
    for size in (1, 2, 8, 250, 1000, 4096, 8192, 8194, 17408, 20480, 25600, 30000, 100000):
        for rows in (1, 1000):
            for dtype in (0, 1):
                assert call(lib, "llme_rows_e4m3", ROWS_TYPES, ROWS, rows=rows, size=size, ldx=size, ldq=size, dtype=dtype, q=p(400), scales=p(600)) == (0, 1)


def test_rows_side_by_side(compiled):  # noqa: F811
    """Column ranges of one buffer are apart although one lies between the other's rows; one byte more and they are not."""
    lib = compiled("rows_e4m3")
    given = {**ROWS, "ldx": 96, "ldq": 192, "q": p(1, 128)}        # rows of 192 bytes: 64 bfloat16 values, then 64 bytes
    assert call(lib, "llme_rows_e4m3", ROWS_TYPES, given) == (0, 1)
    assert call(lib, "llme_rows_e4m3", ROWS_TYPES, given, q=p(1, 127))[0] == -1
    assert call(lib, "llme_rows_e4m3", ROWS_TYPES, given, q=p(1, 129))[0] == -1
    assert call(lib, "llme_rows_e4m3", ROWS_TYPES, given, x=p(1, 64), q=p(1)) == (0, 1)
    assert call(lib, "llme_rows_e4m3", ROWS_TYPES, given, x=p(1, 62), q=p(1))[0] == -1


def test_products_of_8_bits(compiled):  # noqa: F811
    lib = compiled("gemm_e4m3")
    cases = [dict(K=56), dict(K=0), dict(ldx=72), dict(ldx=48), dict(ldw=72), dict(ldw=48), dict(ldo=47), dict(out_dtype=2), dict(x=p(1, 8)), dict(w=p(3, 4)), dict(out=p(1)),
             dict(out=p(3, 64)), dict(out=p(2)), dict(out=p(4))]
    refused(lib, "llme_gemm_e4m3", E4M3_TYPES, E4M3, [{k: None} for k in ("x", "xs", "w", "ws", "out")] + cases)
    for changed in (dict(M=0), dict(N=0)):
        assert call(lib, "llme_gemm_e4m3", E4M3_TYPES, E4M3, **changed) == (0, 0)


def test_products_of_4_bits(compiled):  # noqa: F811
    lib = compiled("gemm_int4")
    cases = [dict(K=60), dict(K=0), dict(ldx=68), dict(ldx=56), dict(ldw=48), dict(ldw=72), dict(lds=1), dict(group=16), dict(group=256), dict(group=0), dict(ldo=47), dict(x=p(1, 8)),
             dict(w=p(2, 8)), dict(out=p(1)), dict(out=p(2, 64)), dict(out=p(3)), dict(out=p(4))]
    refused(lib, "llme_gemm_int4", INT4_TYPES, INT4, [{k: None} for k in ("x", "w", "scales", "out")] + cases)
    assert call(lib, "llme_gemm_int4", INT4_TYPES, INT4, zeros=None) == (0, 1)
    for changed in (dict(M=0), dict(N=0)):
        assert call(lib, "llme_gemm_int4", INT4_TYPES, INT4, **changed) == (0, 0)


@pytest.mark.parametrize("key,name", [("gemm_e4m3", "llme_gemm_e4m3_status"), ("gemm_int4", "llme_gemm_int4_status")])
def test_a_wait_that_gave_up_is_told_once(compiled, key, name):  # noqa: F811
    lib = compiled(key)
    status = getattr(lib, name)
    assert status() == 0
    lib.fake_flag(0, 5, 0)                                 # by a kernel that still runs: the device is waited for
    assert status() == 5 and status() == 0
    lib.fake_flag(0, 0, 1)
    assert status() == -1
    lib.fake_flag(0, 0, 0)
    from llmengine_b200.engine.engine import Engine
    assert Engine._STATUS[key] == name


def test_every_size_is_launched_on_every_device(compiled):  # noqa: F811
    """The forms for few, more and many rows ask for their shared memory on the device they are launched on."""
    e4m3, int4 = compiled("gemm_e4m3"), compiled("gemm_int4")
    for device in (0, 1, 65):
        e4m3.fake_device(device), int4.fake_device(device)
        for n in (16, 2048, 4096, 6144, 12288, 24576):
            for m in (1, 16, 17, 77, 300, 4096):
                for k in (128, 4096):
                    for dtype in (0, 1):
                        assert call(e4m3, "llme_gemm_e4m3", E4M3_TYPES, E4M3, M=m, N=n, K=k, ldx=k, ldw=k, ldo=n, out_dtype=dtype, w=p(64), out=p(128)) == (0, 1)
                    for group in (32, 64, 128):
                        assert call(int4, "llme_gemm_int4", INT4_TYPES, INT4, M=m, N=n, K=k, ldx=k, ldw=k // 2, lds=k // group, group=group, ldo=n, w=p(64), scales=p(90),
                                    zeros=p(100) if group == 32 else None, out=p(128)) == (0, 1)
    e4m3.fake_device(0), int4.fake_device(0)


def test_products_of_4_bits_into_32_bits(compiled):  # noqa: F811
    lib = compiled("gemm_int4")
    cases = [dict(K=60), dict(K=0), dict(ldx=68), dict(ldx=56), dict(ldw=48), dict(ldw=72), dict(lds=1), dict(group=16), dict(group=0), dict(ldo=47), dict(x=p(1, 8)),
             dict(w=p(2, 8)), dict(out=p(1)), dict(out=p(2, 64)), dict(out=p(3)), dict(out=p(4))]
    refused(lib, "llme_gemm_int4_f32", INT4_TYPES, INT4, [{k: None} for k in ("x", "w", "scales", "out")] + cases)
    # four bytes a value: an output that ends before the operand behind it in bfloat16 lies over it in 32 bits
    near = dict(out=p(1, -300), M=3)
    assert call(lib, "llme_gemm_int4", INT4_TYPES, INT4, **near)[0] == 0
    assert call(lib, "llme_gemm_int4_f32", INT4_TYPES, INT4, **near)[0] == -1
    for changed in (dict(M=0), dict(N=0)):
        assert call(lib, "llme_gemm_int4_f32", INT4_TYPES, INT4, **changed) == (0, 0)
    for device in (0, 1, 65):
        lib.fake_device(device)
        for m in (1, 16, 17, 77, 300, 4096):
            for group in (32, 64, 128):
                assert call(lib, "llme_gemm_int4_f32", INT4_TYPES, INT4, M=m, N=4096, K=4096, ldx=4096, ldw=2048, lds=4096 // group, group=group, ldo=4096, w=p(64),
                            scales=p(90), zeros=p(100) if group == 32 else None, out=p(128)) == (0, 1)
    lib.fake_device(0)


def test_sizes_at_the_end_of_32_bits(compiled):  # noqa: F811
    """Indices go a block's width past the last value: sizes that leave no room for that below 2^31 are refused, the largest that do are launched."""
    rows, e4m3, int4 = compiled("rows_e4m3"), compiled("gemm_e4m3"), compiled("gemm_int4")
    far = dict(x=p(1), q=p(1 << 12), scales=p(1 << 13))
    most = 0x7FFFFFFF - 8192
    for entry, more in (("llme_rows_e4m3", 1), ("llme_swiglu_e4m3", 2)):
        for size, n in ((most, 1), (2, most)):
            given = {**ROWS, **far, "rows": n, "size": size, "ldx": more * size, "ldq": size}
            assert call(rows, entry, ROWS_TYPES, given) == (0, 1)
            for changed in (dict(rows=n + 1) if n == most else dict(size=size + 1, ldx=more * (size + 1), ldq=size + 1), dict(rows=0x7FFFFFFF), dict(size=0x7FFFFFFF, ldx=1 << 40, ldq=1 << 40)):
                assert call(rows, entry, ROWS_TYPES, given, **changed) == (-1, 0)
    wide = dict(x=p(1), delta=p(1 << 20), total=p(1), q=p(2 << 20), scales=p(3 << 20), gain=p(4 << 20))
    for changed in (dict(size=most), dict(rows=most)):
        assert call(rows, "llme_rmsnorm_e4m3", NORM_TYPES, {**NORM, **wide}, **changed) == (0, 1)
        changed = {k: v + 1 for k, v in changed.items()}
        assert call(rows, "llme_rmsnorm_e4m3", NORM_TYPES, {**NORM, **wide}, **changed) == (-1, 0)
    spread = dict(x=p(1), w=p(1 << 14), out=p(1 << 16))
    large = most // 128 * 128
    for lib, entry, types, given in ((e4m3, "llme_gemm_e4m3", E4M3_TYPES, {**E4M3, **spread, "xs": p(1 << 18), "ws": p(1 << 19)}),
                                     (int4, "llme_gemm_int4", INT4_TYPES, {**INT4, **spread, "scales": p(1 << 18), "zeros": p(1 << 19)}),
                                     (int4, "llme_gemm_int4_f32", INT4_TYPES, {**INT4, **spread, "scales": p(1 << 18), "zeros": p(1 << 19)})):
        for changed in (dict(M=most), dict(N=most, ldo=most)):
            assert call(lib, entry, types, given, **changed) == (0, 1), (entry, changed)
            assert call(lib, entry, types, given, **{k: v + 1 for k, v in changed.items()}) == (-1, 0)
        deep = dict(K=large, ldx=large, ldw=large, **(dict(lds=large // 32) if "int4" in entry else {}))
        for m in (1, 40):
            assert call(lib, entry, types, given, M=m, **deep) == (0, 1)
            assert call(lib, entry, types, given, M=m, **{**deep, "K": large + 128, "ldx": 1 << 40, "ldw": 1 << 40, **(dict(lds=1 << 40) if "int4" in entry else {})}) == (-1, 0)
