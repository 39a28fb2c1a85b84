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


@pytest.mark.parametrize("scale", [2.0 ** -110, 2.0 ** -122])
def test_tiny_bf16_activations_under_weights_with_large_scales(scale):
    """E8M0 blocks whose scale times 2^-22 is no normal fp32 number, brought back into range by the weights' scales and factors."""
    layer = FineLayer(3, 128, 64, 4, 2, torch.bfloat16, ig.BM_F4_E8M0, seed=21, spread=0.0)
    layer.router = (layer.router.float() * 2.0 ** 100).bfloat16()
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
