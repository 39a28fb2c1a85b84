"""4-bit floating point without a device: sizes, refusals, and the 64-bit forms the GPU tests compare with."""
import numpy as np
import pytest

import _f4 as f4
from bare_metal_b200 import _lib

NULL, SHAPE, ALIGN, LAYOUT = -1, -2, -3, -4


def test_sizes():
    L = _lib.load()
    assert L.bm_f4_value_bytes(3, 33) == 3 * 32 and L.bm_f4_value_bytes(0, 33) == 0
    for fmt, block in ((_lib.BM_F4_E8M0, 32), (_lib.BM_F4_E4M3, 16)):
        for R, K in ((1, 1), (128, 4096), (129, 4100), (5, 1000)):
            g = -(-K // block)
            assert L.bm_f4_scale_bytes(R, K, fmt, _lib.BM_SCALE_ROWS) == R * (-(-g // 16) * 16)
            assert L.bm_f4_scale_bytes(R, K, fmt, _lib.BM_SCALE_TILED) == -(-R // 128) * -(-g // 4) * 512 == f4.tiled(np.zeros((R, g), np.uint8)).size
    assert L.bm_f4_scale_bytes(4, 4, 2, 0) == 0 and L.bm_f4_scale_bytes(4, 4, 0, 2) == 0


def test_refusals():
    L = _lib.load()
    buf = np.zeros(4096 + 64, np.uint8)
    p = (buf.ctypes.data + 15) & ~15
    q = lambda **k: L.bm_quantize_f4(*[{**dict(x=p, t=0, q=p, s=p, r=p, R=4, K=64, ld=64, f=1, l=1, st=None), **k}[n] for n in "x t q s r R K ld f l st".split()])  # noqa: E731
    assert q(x=None) == NULL and q(q=None) == NULL and q(s=None) == NULL and q(r=None) == NULL
    assert q(t=2) == LAYOUT and q(t=5) == LAYOUT and q(f=2) == LAYOUT and q(l=-1) == LAYOUT
    assert q(R=0) == SHAPE and q(K=0) == SHAPE and q(K=-5) == SHAPE and q(ld=63) == SHAPE
    assert q(x=p + 1) == ALIGN and q(q=p + 8) == ALIGN and q(s=p + 4) == ALIGN and q(r=p + 2) == ALIGN
    d = lambda **k: L.bm_dequantize_f4(*[{**dict(q=p, s=p, r=None, o=p, t=2, R=4, K=64, ld=64, f=0, l=0, st=None), **k}[n] for n in "q s r o t R K ld f l st".split()])  # noqa: E731
    assert d(q=None) == NULL and d(s=None) == NULL and d(o=None) == NULL
    assert d(t=3) == LAYOUT and d(f=-1) == LAYOUT and d(l=2) == LAYOUT
    assert d(R=-1) == SHAPE and d(K=0) == SHAPE and d(ld=0) == SHAPE
    assert d(q=p + 1) == ALIGN and d(s=p + 8) == ALIGN and d(o=p + 2) == ALIGN and d(r=p + 1) == ALIGN
    g = lambda **k: L.bm_f4_gemm(*[{**dict(a=p, sa=p, ra=None, w=p, sw=p, rw=None, D=p, t=0, M=4, N=8, K=64, ld=8, f=1, st=None), **k}[n]  # noqa: E731
                                   for n in "a sa ra w sw rw D t M N K ld f st".split()])
    for name in ("a", "sa", "w", "sw", "D"):
        assert g(**{name: None}) == NULL
    assert g(f=7) == LAYOUT and g(t=3) == LAYOUT
    assert g(M=0) == SHAPE and g(N=0) == SHAPE and g(K=-1) == SHAPE and g(ld=7) == SHAPE
    for name in ("a", "sa", "w", "sw"):
        assert g(**{name: p + 8}) == ALIGN
    assert g(D=p + 1) == ALIGN and g(ra=p + 2) == ALIGN and g(t=2, D=p + 2) == ALIGN


def test_sizes_that_do_not_fit_the_arguments():
    """Indexes of 32 bits end before 2^31, and a size beyond an int must not come back as a small one."""
    from bare_metal_b200 import igemm as ig
    L = _lib.load()
    assert L.bm_f4_value_bytes(1, 2 ** 31 - 1) == 2 ** 30 and L.bm_f4_scale_bytes(1, 2 ** 31 - 1, 1, _lib.BM_SCALE_ROWS) == 2 ** 27
    buf = np.zeros(4096 + 64, np.uint8)
    p = (buf.ctypes.data + 15) & ~15
    for R, K in ((4, 2 ** 31 - 65535), (2 ** 31 - 255, 64)):
        assert L.bm_quantize_f4(p, 0, p, p, p, R, K, K, 1, 1, None) == SHAPE
        assert L.bm_dequantize_f4(p, p, None, p, 0, R, K, K, 1, 1, None) == SHAPE
        assert L.bm_f4_gemm(p, p, None, p, p, None, p, 0, R, 8, K, 8, 1, None) == SHAPE
        assert L.bm_f4_gemm(p, p, None, p, p, None, p, 0, 4, R, K, R, 1, None) == SHAPE
    for R, K in ((2 ** 32 + 5, 64), (5, 2 ** 32 + 64), (-2 ** 32 + 5, 64), (0, 64)):
        with pytest.raises(ig.BmError):
            ig._f4_bytes(R, K, _lib.BM_F4_E4M3, _lib.BM_SCALE_ROWS)


def test_expert_layer_sizes_and_refusals():
    L = _lib.load()
    assert L.bm_moe_f4_workspace_bytes(1, 64, 64, 4, 2) > 0
    for bad in ((0, 64, 64, 4, 2), (65, 64, 64, 4, 2), (1, 0, 64, 4, 2), (1, 64, 16385, 4, 2), (1, 64, 64, 257, 2), (1, 64, 64, 4, 5), (1, 64, 64, 32, 17)):
        assert L.bm_moe_f4_workspace_bytes(*bad) == 0
    buf = np.zeros(4096 + 512, np.uint8)
    p = (buf.ctypes.data + 255) & ~255
    names = "x router t w13 s13 r13 w2 s2 r2 y ids wts T H I E top ldx ldy f norm ws wsb st".split()
    good = dict(x=p, router=p, t=1, w13=p, s13=p, r13=None, w2=p, s2=p, r2=None, y=p, ids=None, wts=None, T=2, H=64, I=32, E=4, top=2, ldx=64, ldy=64,
                f=1, norm=1, ws=p, wsb=1 << 30, st=None)
    m = lambda **k: L.bm_moe_f4(*[{**good, **k}[n] for n in names])  # noqa: E731
    for name in ("x", "router", "w13", "s13", "w2", "s2", "y", "ws"):
        assert m(**{name: None}) == NULL
    assert m(f=2) == LAYOUT and m(t=2) == LAYOUT
    assert m(T=0) == SHAPE and m(H=-1) == SHAPE and m(I=0) == SHAPE and m(E=0) == SHAPE and m(top=0) == SHAPE and m(top=5) == SHAPE
    assert m(ldx=63) == SHAPE and m(ldy=63) == SHAPE
    assert m(T=65) == m(H=16385, ldx=20000, ldy=20000) == m(I=16385) == m(E=257) == m(E=32, top=17) == m(wsb=64) == -6
    for name in ("w13", "s13", "w2", "s2"):
        assert m(**{name: p + 8}) == ALIGN
    assert m(ws=p + 128) == ALIGN and m(x=p + 1) == ALIGN and m(y=p + 1) == ALIGN and m(r13=p + 2) == ALIGN and m(ids=p + 1) == ALIGN


@pytest.mark.parametrize("fmt", [f4.E8M0, f4.E4M3_FMT])
def test_the_plain_form_rounds_to_the_nearest(fmt):
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((40, 200)) * np.exp2(rng.uniform(-12, 12, (40, 1)))).astype(np.float16).astype(np.float64)
    code, byte, t = f4.quantize(x, fmt)
    v = f4.values(code, byte, t, fmt)[:, :200]
    s = np.repeat(f4.values(np.full_like(code, 2), byte, t, fmt), 1, 1)[:, :200]              # one times the scale
    assert np.all(np.abs(v) <= 6 * s)
    inside = np.abs(x) <= 6 * s
    step = np.where(np.abs(x) < 2 * s, 0.5, np.where(np.abs(x) < 4 * s, 1.0, 2.0)) * s
    assert np.all(np.abs(v - x)[inside] <= step[inside] / 2)
    if fmt == f4.E8M0:
        assert np.all(s * 4 <= np.abs(np.pad(x, ((0, 0), (0, 24))).reshape(40, -1, 32)).max(-1).repeat(32, 1)[:, :200] + (s < 2.0 ** -100))
    assert np.array_equal(f4.unpack(f4.pack(code)), code)
