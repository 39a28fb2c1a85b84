"""4-bit floating point: quantiser, its inverse and the product against plain 64-bit forms."""
import numpy as np
import pytest
import torch

import _f4 as f4
from bare_metal_b200 import igemm as ig
from _gpu import T, assert_clean_status, dev, options

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def rows(R, K, dtype, seed=0, spread=6):
    """Rows of different size, ties on the grids, zeros of both signs, a row and a block of zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K, generator=g) * torch.exp2((torch.rand(R, 1, generator=g) * 2 - 1) * spread)
    x[:, ::5] = (x[:, ::5] * 4).round() / 4
    x[:, 3::7] = x[:, 3::7].sign() * torch.tensor([0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])[torch.randint(9, x[:, 3::7].shape, generator=g)]
    x[:, K // 2:K // 2 + 32] *= 2.0 ** -9
    if R > 2:
        x[1] = 0
        x[2, :16] = -0.0
    return x.to(dtype)


def check_parts(q, s, r, x, fmt, layout):
    code, byte, t = f4.quantize(x.double().numpy(), fmt)
    got = f4.unpack(q.cpu().numpy())
    assert np.array_equal(s.cpu().numpy().ravel(), (f4.in_rows(byte) if layout == ig.BM_SCALE_ROWS else f4.tiled(byte)).ravel())
    if t is None:
        assert r is None
    else:
        assert np.array_equal(r.cpu().numpy(), t.astype(np.float32))
    assert np.array_equal(np.where(got == 8, 0, got), np.where(code == 8, 0, code))     # zeros of either sign
    return code, byte, t


@pytest.mark.parametrize("layout", [ig.BM_SCALE_ROWS, ig.BM_SCALE_TILED])
@pytest.mark.parametrize("fmt", [ig.BM_F4_E8M0, ig.BM_F4_E4M3])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("R,K", [(1, 1), (1, 32), (3, 17), (130, 100), (5, 4096), (149, 264), (150, 1040), (257, 4100), (2, 16400), (150, 16416), (3, 33000)])
def test_quantise_and_read_back(R, K, dtype, fmt, layout):
    x = rows(R, K, DTYPES[dtype], seed=R + K)
    q, s, r = ig.quantize_f4(x.to(dev()), fmt, layout)
    code, byte, t = check_parts(q, s, r, x, fmt, layout)
    want = torch.from_numpy(f4.values(code, byte, t, fmt)[:, :K])
    for out in (DTYPES[dtype], torch.float32):
        got = ig.dequantize_f4(q, s, r, R, K, out, fmt, layout)
        assert torch.equal(got.cpu(), want.to(out))                                     # exact in fp32, rounded once
    assert_clean_status()


@pytest.mark.parametrize("fmt", [ig.BM_F4_E8M0, ig.BM_F4_E4M3])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_every_16_bit_pattern(dtype, fmt):
    """All numbers of the type, each the largest of one block and a small one in others."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(DTYPES[dtype])
    x = torch.stack([bits[torch.randperm(65536, generator=torch.Generator().manual_seed(s))] for s in range(3)] + [bits])
    x = torch.where(x.isfinite(), x, torch.zeros((), dtype=x.dtype))
    q, s, r = ig.quantize_f4(x.to(dev()), fmt, ig.BM_SCALE_ROWS)
    check_parts(q, s, r, x, fmt, ig.BM_SCALE_ROWS)
    x = x.view(-1, 64)
    q, s, r = ig.quantize_f4(x.to(dev()), fmt, ig.BM_SCALE_TILED)
    check_parts(q, s, r, x, fmt, ig.BM_SCALE_TILED)


@pytest.mark.parametrize("fmt", [ig.BM_F4_E8M0, ig.BM_F4_E4M3])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_infinities_and_nans_mark_their_block(dtype, fmt):
    x = rows(6, 200, DTYPES[dtype], seed=3)
    x[0, 5], x[3, 199], x[4, 64:96] = float("inf"), float("nan"), float("-inf")
    x[5] = float("nan")
    q, s, r = ig.quantize_f4(x.to(dev()), fmt, ig.BM_SCALE_TILED)
    code, byte, t = check_parts(q, s, r, x, fmt, ig.BM_SCALE_TILED)
    got = ig.dequantize_f4(q, s, r, 6, 200, torch.float32, fmt)
    want = torch.from_numpy(f4.values(code, byte, t, fmt)[:, :200]).float()
    assert torch.equal(got.cpu().isnan(), want.isnan()) and torch.equal(got.cpu().nan_to_num(), want.nan_to_num())
    assert got[5].isnan().all()


@pytest.mark.parametrize("offset,pitch", [(0, 512), (8, 264), (1, 301), (3, 264)])
@pytest.mark.parametrize("fmt", [ig.BM_F4_E8M0, ig.BM_F4_E4M3])
def test_strided_rows_and_outputs(fmt, offset, pitch):
    R, K = 140, 250
    x = rows(R, K, torch.float16, seed=9)
    wide = torch.full((R * pitch + 16,), 7.0, dtype=torch.float16, device=dev())
    view = torch.as_strided(wide, (R, K), (pitch, 1), offset)
    view.copy_(x)
    q, s, r = ig.quantize_f4(view, fmt, ig.BM_SCALE_TILED)
    code, byte, t = check_parts(q, s, r, x, fmt, ig.BM_SCALE_TILED)
    before = wide.clone()
    ig.dequantize_f4(q, s, r, R, K, fmt=fmt, out=view)
    assert torch.equal(view.cpu(), torch.from_numpy(f4.values(code, byte, t, fmt)[:, :K]).half())
    keep = torch.ones_like(wide, dtype=torch.bool)
    torch.as_strided(keep, (R, K), (pitch, 1), offset).fill_(False)
    assert torch.equal(wide[keep], before[keep])


def product_inputs(M, N, K, fmt, seed=0, dtype=torch.float16):
    x, w = rows(M, K, dtype, seed), rows(N, K, dtype, seed + 1) / 16
    X, W = ig.quantize_f4(x.to(dev()), fmt), ig.quantize_f4(w.to(dev()), fmt)
    a, b = (f4.values(*f4.quantize(v.double().numpy(), fmt), fmt) for v in (x, w))
    return X, W, a, b


def check_product(D, a, b):
    """Each fp32 addition is off by at most 2^-23 of what has been added so far (truncation), over at most K / 16 of them; the
    two factors and the rounding to the output type half a step each."""
    want, size = a @ b.T, np.abs(a) @ np.abs(b).T
    half = HALF_STEP[D.dtype]
    bound = (a.shape[1] / 16 + 1) * 2.0 ** -23 * size + (half + 2 * 2.0 ** -24) * np.abs(want) * 1.01 + 2.0 ** -25 * (D.dtype == torch.float16)
    got = D.double().cpu().numpy()
    most = {torch.float16: 65504.0}.get(D.dtype, np.inf)
    fits = np.abs(want) < most
    assert np.all(np.abs(got - want)[fits] <= bound[fits]), float(np.max((np.abs(got - want) / bound)[fits]))


SHAPES = [(1, 1, 1), (1, 128, 64), (16, 128, 256), (7, 300, 1000), (64, 520, 2080), (100, 136, 544), (128, 128, 256), (129, 257, 288),
          (300, 500, 1504), (600, 700, 96), (1000, 520, 4096)]


@pytest.mark.parametrize("kernel", [0, 1, 2, 3])
@pytest.mark.parametrize("fmt", [ig.BM_F4_E8M0, ig.BM_F4_E4M3])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(M, N, K, fmt, kernel):
    X, W, a, b = product_inputs(M, N, K, fmt, seed=M + N + K)
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        D = torch.full((M, N), 7.0, dtype=dtype, device=dev())
        with options(f4_kernel=kernel):
            ig.f4_linear(*X, *W, D, M, N, K, fmt)
        assert_clean_status()
        check_product(D, a, b)


@pytest.mark.parametrize("kernel,M", [(1, 40), (2, 200), (3, 300)])
@pytest.mark.parametrize("fmt", [ig.BM_F4_E8M0, ig.BM_F4_E4M3])
def test_product_into_a_part_of_a_wider_matrix(kernel, M, fmt):
    N, K = 333, 640
    X, W, a, b = product_inputs(M, N, K, fmt, seed=kernel)
    for dtype in (torch.float16, torch.float32):
        for pitch, offset in ((N + 3, 0), (N + 51, 8), (384, 0), (344, 1)):
            wide = torch.full((M * pitch + 16,), 7.0, dtype=dtype, device=dev())
            D = torch.as_strided(wide, (M, N), (pitch, 1), offset)
            with options(f4_kernel=kernel):
                ig.f4_linear(*X, *W, D, M, N, K, fmt)
            check_product(D, a, b)
            keep = torch.ones_like(wide, dtype=torch.bool)
            torch.as_strided(keep, (M, N), (pitch, 1), offset).fill_(False)
            assert (wide[keep] == 7.0).all()
    assert_clean_status()


@pytest.mark.parametrize("kernel,M", [(1, 128), (2, 1000), (3, 3000)])
@pytest.mark.parametrize("fmt", [ig.BM_F4_E8M0, ig.BM_F4_E4M3])
def test_product_is_the_same_on_every_call(kernel, M, fmt):
    """Several tiles a CTA, back to back: scales and accumulators of one tile must not reach another's."""
    N, K = 2600, 1200
    X, W, a, b = product_inputs(M, N, K, fmt, seed=5)
    with options(f4_kernel=kernel):
        outs = []
        for _ in range(6):
            D = torch.empty((M, N), dtype=torch.float32, device=dev())
            outs.append(ig.f4_linear(*X, *W, D, M, N, K, fmt))
    assert_clean_status()
    check_product(outs[0], a, b)
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("fmt", [ig.BM_F4_E8M0, ig.BM_F4_E4M3])
@pytest.mark.parametrize("M,N", [(2560, 2048), (2500, 2300), (2304, 2432)])                 # 80 and 90 pair tiles: the last wave of 74 pairs is cut up
def test_product_with_a_partly_filled_last_wave(M, N, fmt):
    K = 800
    X, W, a, b = product_inputs(M, N, K, fmt, seed=6)
    for dtype in (torch.float16, torch.float32):
        D = torch.full((M, N), 7.0, dtype=dtype, device=dev())
        with options(f4_kernel=3):
            ig.f4_linear(*X, *W, D, M, N, K, fmt)
            with options(tail_narrow=0):
                whole = ig.f4_linear(*X, *W, torch.empty_like(D), M, N, K, fmt)
        assert torch.equal(D, whole)
        check_product(D, a, b)
    assert_clean_status()


@pytest.mark.parametrize("kernel,M", [(1, 9), (2, 150), (3, 260)])
@pytest.mark.parametrize("fmt", [ig.BM_F4_E8M0, ig.BM_F4_E4M3])
def test_nan_scales_reach_their_rows_and_columns_only(kernel, M, fmt):
    N, K = 270, 512
    x, w = rows(M, K, torch.bfloat16, 1), rows(N, K, torch.bfloat16, 2)
    x[3, 100], w[5, 7], w[N - 1, K - 1] = float("nan"), float("inf"), float("nan")
    X, W = ig.quantize_f4(x.to(dev()), fmt), ig.quantize_f4(w.to(dev()), fmt)
    D = torch.empty((M, N), dtype=torch.float32, device=dev())
    with options(f4_kernel=kernel):
        ig.f4_linear(*X, *W, D, M, N, K, fmt)
    want = torch.zeros(M, N, dtype=torch.bool)
    want[3], want[:, 5], want[:, N - 1] = True, True, True
    assert torch.equal(D.isnan().cpu(), want)


def test_product_without_row_factors_and_with_own_ones():
    M, N, K = 70, 200, 320
    X, W, a, b = product_inputs(M, N, K, ig.BM_F4_E4M3, seed=2)
    ra, rb = torch.rand(M, device=dev()) + 0.5, torch.rand(N, device=dev()) + 0.5
    a0, b0 = a / X[2].double().cpu().numpy()[:, None], b / W[2].double().cpu().numpy()[:, None]
    for kernel in (1, 2, 3):
        for fa, fb in ((None, None), (ra, None), (None, rb), (ra, rb)):
            D = torch.empty((M, N), dtype=torch.float32, device=dev())
            with options(f4_kernel=kernel):
                ig.f4_linear(X[0], X[1], fa, W[0], W[1], fb, D, M, N, K)
            one = np.ones(1)
            check_product(D, a0 * (one if fa is None else fa.double().cpu().numpy()[:, None]),
                          b0 * (one if fb is None else fb.double().cpu().numpy()[:, None]))


def test_linear_on_another_stream_and_in_a_graph():
    """Quantise and multiply as a decoding step does, captured once and replayed on new activations."""
    M, N, K = 16, 512, 1024
    w = rows(N, K, torch.float16, 1)
    W = ig.quantize_f4(w.to(dev()))
    x = rows(M, K, torch.float16, 2).to(dev())
    D = torch.empty((M, N), dtype=torch.float16, device=dev())

    def step():
        ig.f4_linear(*ig.quantize_f4(x), *W, D, M, N, K)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    b = f4.values(*f4.quantize(w.double().numpy(), 1), 1)
    for seed in (3, 4):
        new = rows(M, K, torch.float16, seed)
        x.copy_(new.to(dev()))
        graph.replay()
        torch.cuda.synchronize()
        check_product(D, f4.values(*f4.quantize(new.double().numpy(), 1), 1), b)
    assert_clean_status()
