"""Expert layer on 4-bit weights: inputs that show in how many bits it holds its activations and logits."""
import numpy as np
import pytest
import torch

import _f4 as f4
from bare_metal_b200 import igemm as ig
from _gpu import assert_clean_status, dev
from test_gpu_moe_f4 import FMT, HALF, LOST, Layer

pytestmark = pytest.mark.gpu


class FineLayer(Layer):
    def left(self, v, dv=0.0):
        """Eight digits of base 8 under a power of two s: off by at most half a unit, 2^-23 s, with s at most 2 / 1.7 of the block's
        largest, 2^-22.76 of it.  E4M3's smallest scale is 2^-9 where the row's largest is 2^7 or more: 2^-39 of that."""
        a = np.abs(v) + dv
        n = f4.BLOCK[self.fmt]
        top = np.pad(a, ((0, 0), (0, -a.shape[1] % n))).reshape(a.shape[0], -1, n).max(-1).repeat(n, 1)[:, :a.shape[1]]
        return 2.0 ** -22.7 * top + (2.0 ** -39 * a.max(1, keepdims=True) if self.fmt == ig.BM_F4_E4M3 else 0.0)

    def reweigh(self, name, by_row=None, by_column=None):
        w = self.plain[name].float()
        w = w if by_row is None else w * by_row[:, None]
        w = w if by_column is None else w * by_column
        self.plain[name] = w.bfloat16()
        self.w[name] = ig.quantize_f4(self.plain[name].to(dev()), self.fmt, ig.BM_SCALE_ROWS)


def with_large_channels(T, H, I, E, top, dtype, fmt, factor, seed):
    """A few channels of x, and of the hidden activations, are `factor` times larger than their neighbours, and the weights that read
    them as much smaller: the other channels make the results."""
    layer = FineLayer(T, H, I, E, top, dtype, fmt, seed=seed, spread=0.0)
    wide, deep = torch.ones(H), torch.ones(I)
    wide[torch.arange(7, H, 101)] = factor
    deep[torch.arange(3, I, 53)] = factor
    layer.x = (layer.x.float() * wide).to(dtype)
    layer.router = (layer.router.float() / wide).to(dtype)
    layer.router_here = layer.router.to(dev())
    layer.reweigh("w13", by_row=torch.cat((torch.ones(I), deep)).repeat(E), by_column=1 / wide)
    layer.reweigh("w2", by_column=1 / deep)
    return layer


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("T,H,I", [(1, 1024, 512), (12, 520, 300)])
def test_small_activations_beside_much_larger_ones(T, H, I, fmt, dtype):
    layer = with_large_channels(T, H, I, 8, 3, dtype, FMT[fmt], 4096.0, seed=T)
    out = layer.run()
    assert_clean_status()
    layer.check(*out)


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("scale", [2.0 ** -110, 2.0 ** -122, 2.0 ** 115])
def test_tiny_and_huge_bf16_activations_under_weights_that_bring_them_back(scale, fmt):
    """E8M0 blocks whose scale times 2^-22 is no normal fp32 number; E4M3 rows whose factor, or whose weights' factors, are beyond it with the sums.
    (Below 2^-119 E4M3's row factor stays at 2^-126, and every bf16 number is a multiple of 2^-133: exact.)"""
    layer = FineLayer(3, 128, 64, 4, 2, torch.bfloat16, FMT[fmt], seed=21, spread=0.0)
    layer.router = (layer.router.float() * (2.0 ** 100 if scale < 1 else 2.0 ** -100)).bfloat16()
    layer.router_here = layer.router.to(dev())
    layer.x = (layer.x.float() * scale).bfloat16()
    layer.reweigh("w13", by_row=torch.full((4 * 128,), 1.0 / scale))
    out = layer.run()
    assert_clean_status()
    layer.check(*out)
    assert out[0].abs().max() > 0.01


def check_on_device(layer, y, ids, weights):
    """Layer.check's bound in 64 bits on the device, for layers that are too large for it, with the selection and the weights given."""
    T, H, I, E = layer.T, layer.H, layer.I, layer.E
    assert np.array_equal(ids.cpu().numpy(), layer.select()[1])
    w13, w2 = (ig.dequantize_f4(*layer.w[n], r, k, torch.float32, layer.fmt, ig.BM_SCALE_ROWS) for n, r, k in (("w13", E * 2 * I, H), ("w2", E * H, I)))
    u1, u2 = (H / 16 + 32) * 2.0 ** -23, (I / 16 + 32) * 2.0 ** -23
    left = lambda v, dv: torch.from_numpy(layer.left(v.cpu().numpy(), dv.cpu().numpy())).to(dev())  # noqa: E731
    x = layer.x.to(dev()).double()
    dx = left(x, torch.zeros_like(x))
    want, bound = torch.zeros(T, H, dtype=torch.float64, device=dev()), torch.zeros(T, H, dtype=torch.float64, device=dev())
    for e in range(E):
        t, k = (ids == e).nonzero(as_tuple=True)
        if len(t) == 0:
            continue
        a, b = w13[e * 2 * I:(e + 1) * 2 * I].double(), w2[e * H:(e + 1) * H].double()
        gu, du = x[t] @ a.T, (u1 * x[t].abs() + dx[t]) @ a.abs().T
        g, u = gu[:, :I], gu[:, I:]
        s = g / (1 + torch.exp(-g))
        h = s * u
        dh = 1.1 * du[:, :I] * (u.abs() + du[:, I:]) + s.abs() * du[:, I:] + h.abs() * (8 + g.abs()) * 2.0 ** -24
        dh = dh + left(h, dh)
        p = weights[t, k].double()[:, None]
        want.index_add_(0, t, p * (h @ b.T))
        bound.index_add_(0, t, p * ((dh + u2 * h.abs()) @ b.abs().T + 1e-6 * (h @ b.T).abs()))
    bound = bound * 1.01 + HALF[layer.dtype] * (want.abs() + bound) + LOST[layer.dtype]
    assert ((y.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("T,H,I,E,top", [(64, 16384, 64, 16, 16), (64, 64, 16384, 16, 16), (64, 2304, 64, 64, 16), (48, 2048, 80, 200, 16)])
def test_many_short_runs_beside_a_busy_stream(T, H, I, E, top, fmt):
    """Tiles of activations that change hands after every unit of work, while other kernels take their share of the SMs."""
    layer = FineLayer(T, H, I, E, top, torch.bfloat16, FMT[fmt], seed=31)
    x = layer.x.to(dev())
    first = layer.run(x)
    torch.cuda.synchronize()
    check_on_device(layer, *first)
    side, noise = torch.cuda.Stream(), torch.zeros(1 << 24, device=dev())
    for _ in range(12):
        with torch.cuda.stream(side):
            noise.add_(1.0)
        again = layer.run(x)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    assert_clean_status()


def test_large_channels_that_cancel_in_the_logits():
    """Products of 3e6 and -3e6 beside ones around 1: fp32 holds no more than quarters there, and the experts lie closer."""
    T, H, E, top = 10, 256, 32, 6
    g = torch.Generator().manual_seed(41)
    x, router = torch.randn(T, H, generator=g), torch.randn(E, H, generator=g) / 16
    x[:, 0], x[:, 1], x[:, 77], x[:, 79] = 30000.0, -30000.0, -20000.0, 20000.0
    router[:, 0] = router[:, 1] = torch.randint(50, 200, (E,), generator=g).float()
    router[:, 77] = router[:, 79] = torch.randint(50, 200, (E,), generator=g).float()
    for norm in (True, False):
        layer = FineLayer(T, H, 48, E, top, torch.float16, ig.BM_F4_E8M0, norm, seed=42, x=x, router=router)
        y, ids, weights = layer.run()
        assert_clean_status()
        logits, order, p = layer.select()
        assert np.array_equal(ids.cpu().numpy(), order)
        assert np.allclose(weights.double().cpu().numpy(), p, rtol=2e-6 * (1 + np.abs(logits).max(1)[:, None]), atol=1e-30)
        assert not y.isnan().any()                                # (most are 10^7 and more, infinities in fp16)


def test_equal_logits_from_rows_that_are_not_equal():
    """Rows with the same numbers in other orders, all of x one: exact in 64 bits (fp16 numbers are multiples of 2^-24), so equal, lowest index first."""
    T, H, E, top = 3, 1024, 20, 9
    g = torch.Generator().manual_seed(43)
    numbers = (torch.randn(H, generator=g) * torch.exp2(torch.rand(H, generator=g) * 24 - 14)).half()
    router = torch.stack([numbers[torch.randperm(H, generator=g)] for _ in range(E)])
    router[4, 0] = router[11, 0] = 30000.0
    layer = FineLayer(T, H, 32, E, top, torch.float16, ig.BM_F4_E4M3, seed=44, x=torch.ones(T, H), router=router)
    _, ids, weights = layer.run()
    assert_clean_status()
    order = sorted(range(E), key=lambda e: (-router[e].double().sum().item(), e))
    assert ids.tolist() == [order[:top]] * T and sorted(order[:2]) == [4, 11]
    equal = [n for n, e in enumerate(order[:top]) if e not in (4, 11)]
    assert (weights[:, equal] == weights[:, equal[:1]]).all()


@pytest.mark.parametrize("norm", [True, False])
def test_bf16_logits_beyond_the_range_of_fp32(norm):
    """Logits of 2^140 are numbers in 64 bits: the largest takes the whole weight, as with a router 2^-60 times as large."""
    T, H, I, E, top = 5, 200, 48, 12, 4
    g = torch.Generator().manual_seed(45)
    x, router = torch.randn(T, H, generator=g) * 2.0 ** 80, torch.randn(E, H, generator=g) * 2.0 ** 60
    layer = FineLayer(T, H, I, E, top, torch.bfloat16, ig.BM_F4_E8M0, norm, seed=46, x=x, router=router)
    layer.reweigh("w13", by_row=torch.full((E * 2 * I,), 2.0 ** -80))
    y, ids, weights = layer.run()
    assert_clean_status()
    assert np.array_equal(ids.cpu().numpy(), layer.select()[1])
    assert (weights[:, 0] == 1).all() and (weights[:, 1:] == 0).all()
    layer.router_here = (layer.router.float() * 2.0 ** -60).bfloat16().to(dev())
    again = layer.run()
    assert torch.equal(ids, again[1]) and torch.equal(weights, again[2]) and torch.equal(y, again[0])
    assert y.isfinite().all() and y.abs().max() > 0.01


@pytest.mark.parametrize("fmt,in_x", [("e8m0", True), ("e8m0", False), ("e4m3", False)])
def test_gates_far_below_zero(fmt, in_x):
    """silu(-88) is -88 * 6e-39, and 2^119 times that is a number: SiLU by exp(-g) and one division gives nothing beyond 2^126.  (Not E4M3 with
    2^100 in x: a number of 88 is then below 2^-39 of its row's largest, and the gates may be anything up to 2^61.)"""
    gates = [-80.0, -87.0, -87.5, -88.0, -88.5, -12.0, 3.0]
    T, H, I = len(gates), 64, 32
    layer = FineLayer(T, H, I, 1, 1, torch.bfloat16, FMT[fmt], seed=51, x=torch.zeros(T, H), router=torch.zeros(1, H))
    layer.x[:, 0], layer.x[:, 40] = torch.tensor(gates).bfloat16(), 2.0 ** 100 if in_x else 1.0
    w13, w2 = torch.zeros(2 * I, H), torch.zeros(H, I)
    w13[:I, 0], w13[I:, 40], w2[:, 5] = 1.0, 2.0 ** 19 if in_x else 2.0 ** 119, 1.0
    for name, w in (("w13", w13), ("w2", w2)):
        layer.plain[name] = w.bfloat16()
        layer.w[name] = ig.quantize_f4(layer.plain[name].to(dev()), layer.fmt, ig.BM_SCALE_ROWS)
    y, _, _ = layer.run()
    assert_clean_status()
    # the exponential 8 + |g| units; the weights 1 and 2^119 are off by up to a sixteenth in E4M3 (as read back); the output's rounding
    one, much = (ig.dequantize_f4(*layer.w["w13"], 2 * I, H, torch.float32, layer.fmt, ig.BM_SCALE_ROWS)[r, k].item() for r, k in ((0, 0), (I, 40)))
    last = ig.dequantize_f4(*layer.w["w2"], H, I, torch.float32, layer.fmt, ig.BM_SCALE_ROWS)[0, 5].item()
    g = np.array(gates) * one
    want = (g / (1 + np.exp(-g)) * (2.0 ** 100 if in_x else 1.0) * much * last)[:, None]
    bound = np.abs(want) * ((8 + np.abs(g[:, None])) * 2.0 ** -24 + 2.0 ** -8 * 1.01 + 2.0 ** -22)
    assert (np.abs(y.double().cpu().numpy() - want) <= bound).all()
