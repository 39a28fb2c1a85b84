"""4-bit operators at sizes whose offsets pass 31 and 32 bits, and the pair kernel's banded tile order."""
import pytest
import torch

from bare_metal_b200 import igemm as ig
from _gpu import assert_clean_status, dev, options

pytestmark = pytest.mark.gpu
BOTH = [ig.BM_F4_E8M0, ig.BM_F4_E4M3]


def small_integers(R, K, seed, limit=4, most=6.0):
    """Rows of the 4-bit numbers -4 ... 4 with `most` in every block.  6: quantised without loss in both formats (the scale is 1, or
    256 times the row's 2^-8), so products and sums are integers.  4: without loss in E8M0; E4M3's scale is 4/6 * 2^8 rounded to 176."""
    g = torch.Generator(device=dev()).manual_seed(seed)
    x = torch.empty(R, K, dtype=torch.float16, device=dev())
    for r in range(0, R, 8192):
        part = x[r:r + 8192]
        part.copy_(torch.randint(-limit, limit + 1, part.shape, generator=g, device=dev(), dtype=torch.int8))
    x[:, ::16] = most
    return x


# banded order (16 or more row tiles, twice as many as column tiles): whole bands and a short one, a cut-up last wave, narrow last tiles
@pytest.mark.parametrize("fmt", BOTH)
@pytest.mark.parametrize("M,N,K", [(4100, 520, 320), (4096, 2048, 256), (8292, 520, 544), (6150, 1030, 96)])
def test_bands_of_row_tiles(M, N, K, fmt):
    x, w = (torch.randn(n, K, generator=torch.Generator().manual_seed(n)).half().to(dev()) for n in (M, N))
    X, W = ig.quantize_f4(x, fmt), ig.quantize_f4(w, fmt)
    a, b = (ig.dequantize_f4(*q, n, K, torch.float32, fmt).double() for q, n in ((X, M), (W, N)))
    want, size = a @ b.T, a.abs() @ b.abs().T
    # each fp32 addition off by at most 2^-23 of what has been added so far (truncation), K / 16 of them; factors and the result half a step
    bound = (K / 16 + 1) * 2.0 ** -23 * size + 3 * 2.0 ** -24 * want.abs() * 1.01
    for tail in (1, 0):
        D = torch.full((M, N + 4), 7.0, dtype=torch.float32, device=dev())
        with options(f4_kernel=3, tail_narrow=tail):
            ig.f4_linear(*X, *W, D[:, :N], M, N, K, fmt)
        assert_clean_status()
        assert ((D[:, :N].double() - want).abs() <= bound).all()
        assert (D[:, N:] == 7).all()


@pytest.mark.parametrize("layout", [ig.BM_SCALE_ROWS, ig.BM_SCALE_TILED])
@pytest.mark.parametrize("fmt", BOTH)
@pytest.mark.parametrize("R,K", [(70001, 32768), (2200003, 32)])        # 2^31 numbers and more; more rows than a grid's second dimension reaches
def test_quantise_and_read_back(R, K, fmt, layout):
    x = small_integers(R, K, 1, most=4.0)
    q, s, r = ig.quantize_f4(x, fmt, layout)
    back = ig.dequantize_f4(q, s, r, R, K, torch.float16, fmt, layout)
    assert_clean_status()
    if fmt == ig.BM_F4_E8M0:
        assert torch.equal(back, x)
    else:
        v = torch.arange(-4, 5).double()                                # what 176 / 256 times the nearest of the nine numbers is
        grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6]).double()
        near = grid[(v.abs()[:, None] * 256 / 176 - grid).abs().argmin(1)] * v.sign() * 176 / 256
        near = near.half().to(dev())
        for r0 in range(0, R, 1 << 14):
            assert torch.equal(back[r0:r0 + (1 << 14)], near[x[r0:r0 + (1 << 14)].long() + 4])
    tail = ig.quantize_f4(x[-1:], fmt, ig.BM_SCALE_ROWS)
    assert torch.equal(q[-1:], tail[0])


@pytest.mark.parametrize("kernel,M", [(1, 3), (2, 130), (3, 260)])
@pytest.mark.parametrize("fmt", BOTH)
def test_weights_of_more_than_two_to_the_31_bytes(fmt, kernel, M):
    N, K = 140003, 32768
    if kernel != 1:
        N, K = N // 4 * 4 + 1, K // 2                                   # the same offsets in the scales' rows, half the products
    w = small_integers(N, K, 2, 2)
    w[-1] = 6.0
    W = ig.quantize_f4(w, fmt)
    x = small_integers(M, K, 3, 2)
    X = ig.quantize_f4(x, fmt)
    D = torch.empty(M, N, dtype=torch.float32, device=dev())
    with options(f4_kernel=kernel):
        ig.f4_linear(*X, *W, D, M, N, K, fmt)
    assert_clean_status()
    for cols in (slice(0, 300), slice(N - 300, N)):
        assert torch.equal(D[:, cols], (x.double() @ w[cols].double().T).float())


@pytest.mark.parametrize("kernel", [2, 3])
def test_results_of_more_than_two_to_the_31_numbers(kernel):
    M, N, K = 70001, 32765, 64                                          # rows off 16 bytes: copied, not stored by TMA
    x, w = small_integers(M, K, 4), small_integers(N, K, 5)
    X, W = ig.quantize_f4(x), ig.quantize_f4(w)
    for pitch in (N, 32768):
        D = torch.full((M, pitch), 7.0, dtype=torch.float16, device=dev())
        with options(f4_kernel=kernel):
            ig.f4_linear(*X, *W, D[:, :N], M, N, K)
        assert_clean_status()
        for rows in (slice(0, 300), slice(M - 300, M)):
            assert torch.equal(D[rows, :N], (x[rows].float() @ w.float().T).half())
        assert (D[:, N:] == 7).all()


@pytest.mark.parametrize("fmt", BOTH)
def test_experts_of_more_than_two_to_the_32_bytes(fmt):
    """The last two of 72 experts, against a layer of these two alone."""
    T, H, I, E = 3, 16384, 4096, 72
    g = torch.Generator(device=dev()).manual_seed(6)

    def weights(rows, k):
        groups = -(-k // (32 if fmt == ig.BM_F4_E8M0 else 16))
        q = torch.empty(rows, k // 2, dtype=torch.uint8, device=dev())
        s = torch.empty(rows, -(-groups // 16) * 16, dtype=torch.uint8, device=dev())
        low, high = (118, 122) if fmt == ig.BM_F4_E8M0 else (0x18, 0x38)
        for r in range(0, rows, 1 << 16):
            q[r:r + (1 << 16)].random_(0, 256, generator=g)
            s[r:r + (1 << 16)].random_(low, high, generator=g)
        return q, s, None if fmt == ig.BM_F4_E8M0 else torch.exp2(torch.randint(-9, -5, (rows,), device=dev(), generator=g).float())

    w13, w2 = weights(E * 2 * I, H), weights(E * H, I)
    x = torch.randn(T, H, device=dev(), generator=g).bfloat16()
    router = torch.zeros(E, H, device=dev(), dtype=torch.bfloat16)
    x[:, 0], router[E - 1, 0], router[E - 2, 0] = 1.0, 3.0, 2.0
    y, ids, p = ig.moe_f4(x, router, w13, w2, 2, I, fmt)
    few = lambda w, rows: tuple(None if t is None else t[-2 * rows:].contiguous() for t in w)  # noqa: E731
    y2, ids2, p2 = ig.moe_f4(x, router[-2:].contiguous(), few(w13, 2 * I), few(w2, H), 2, I, fmt)
    assert_clean_status()
    assert (ids == torch.tensor([E - 1, E - 2], device=dev())).all() and torch.equal(ids, ids2 + E - 2) and torch.equal(p, p2)
    assert y.isfinite().all() and y.abs().max() > 0 and torch.equal(y, y2)
