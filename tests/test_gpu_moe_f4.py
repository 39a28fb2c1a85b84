"""Expert layer on 4-bit weights against a plain 64-bit form."""
import numpy as np
import pytest
import torch

import _f4 as f4
from bare_metal_b200 import igemm as ig
from _gpu import assert_clean_status, dev

pytestmark = pytest.mark.gpu

FMT = {"e8m0": ig.BM_F4_E8M0, "e4m3": ig.BM_F4_E4M3}
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# below the types' range: half of fp16's smallest number; bf16's and fp32's smallest normal one (hidden activations of 2^-240 in
# test_the_largest_activations, outputs of 2^-239: neither exists in fp32, zero is the right answer and all of it is the error)
LOST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


class Layer:
    def __init__(self, T, H, I, E, top, dtype, fmt, norm=True, seed=0, x=None, router=None, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.T, self.H, self.I, self.E, self.top, self.dtype, self.fmt, self.norm = T, H, I, E, top, dtype, fmt, norm
        self.x = (torch.randn(T, H, generator=g) * torch.exp2(spread * torch.randn(T, 1, generator=g)) if x is None else x).to(dtype)
        self.router = (torch.randn(E, H, generator=g) * (1.5 / H ** 0.5) if router is None else router).to(dtype)
        self.router_here = self.router.to(dev())
        weight = lambda R, K: (torch.randn(R, K, generator=g) / K ** 0.5 * torch.exp2(torch.randn(R, 1, generator=g))).bfloat16()  # noqa: E731
        self.plain = {"w13": weight(E * 2 * I, H), "w2": weight(E * H, I)}
        self.w = {n: ig.quantize_f4(v.to(dev()), fmt, ig.BM_SCALE_ROWS) for n, v in self.plain.items()}

    def run(self, x=None, **kw):
        return ig.moe_f4((self.x.to(dev()) if x is None else x), self.router_here, self.w["w13"], self.w["w2"], self.top, self.I, self.fmt, self.norm, **kw)

    def select(self):
        logits = self.x.double().numpy() @ self.router.double().numpy().T
        order = np.argsort(-logits, axis=1, kind="stable")[:, :self.top]
        z = np.exp(logits - logits.max(1, keepdims=True))
        p = np.take_along_axis(z, order, 1)
        return logits, order, p / (p if self.norm else z).sum(1, keepdims=True)

    def left(self, v, dv=0.0):
        """What the digits may leave of rows of activations (known up to dv)."""
        a = np.abs(v) + dv
        n = f4.BLOCK[self.fmt]
        top = np.pad(a, ((0, 0), (0, -a.shape[1] % n))).reshape(a.shape[0], -1, n).max(-1).repeat(n, 1)[:, :a.shape[1]]
        return 2.0 ** -16.7 * top + 2.0 ** -34 * a.max(1, keepdims=True)

    def check(self, y, ids, weights):
        """Errors: an fp32 sum over K is off by at most 2^-23 of the sum of sizes for each of K / 16 + 32 additions (truncated);
        SiLU moves by at most 1.1 times what its argument g does; its evaluation is off by 8 + |g| units of 2^-24 (the exponent g
        log2(e) is rounded).  Activations and hidden activations are written with six digits of base 8: off by at most half a
        unit, s / 2 * 8^-5 / 2 = 2^-17 s, and s is at most 2 / 1.7 of the block's largest (a power of two), or 1.0625 / 1.6 of it (E4M3;
        at least 2^-9 of a unit of which the row's largest has 2^8 or more): 2^-16.7 of the block's, 2^-34 of the row's.  (A
        block is at most 32 long.)  Then the sum over the choices, and the rounding to the output type."""
        logits, order, p = self.select()
        ranked = -np.sort(-logits, 1)
        size = np.abs(logits).max(1)                              # of a token's logits: what is added up is its own row's
        if self.top < self.E:
            assert (ranked[:, self.top - 1] - ranked[:, self.top] > 1e-6 * size).all(), "inputs too close to a tie"
        assert np.array_equal(ids.cpu().numpy(), order)
        assert np.allclose(weights.double().cpu().numpy(), p, rtol=2e-6 * (1 + size[:, None]), atol=1e-30)
        x = self.x.double().numpy()
        want, bound = np.zeros((self.T, self.H)), np.zeros((self.T, self.H))
        w13 = f4.values(*f4.quantize(self.plain["w13"].double().numpy(), self.fmt), self.fmt)[:, :self.H]
        w2 = f4.values(*f4.quantize(self.plain["w2"].double().numpy(), self.fmt), self.fmt)[:, :self.I]
        u1, u2 = (self.H / 16 + 32) * 2.0 ** -23, (self.I / 16 + 32) * 2.0 ** -23
        dx = self.left(x)
        for t in range(self.T):
            for k, e in enumerate(order[t]):
                a, b = w13[e * 2 * self.I:(e + 1) * 2 * self.I], w2[e * self.H:(e + 1) * self.H]
                gu, du = a @ x[t], u1 * (np.abs(a) @ np.abs(x[t])) + np.abs(a) @ dx[t]
                g, u = gu[:self.I], gu[self.I:]
                s = g / (1 + np.exp(-g))
                h = s * u
                dh = 1.1 * du[:self.I] * (np.abs(u) + du[self.I:]) + np.abs(s) * du[self.I:] + np.abs(h) * (8 + np.abs(g)) * 2.0 ** -24
                dh = dh + self.left(h[None], dh[None])[0]
                y1, d1 = b @ h, np.abs(b) @ dh + u2 * (np.abs(b) @ np.abs(h))
                want[t] += p[t, k] * y1
                bound[t] += p[t, k] * (d1 + 1e-6 * (1 + size[t]) * np.abs(y1))
        bound = bound * 1.01 + HALF[self.dtype] * (np.abs(want) + bound) + LOST[self.dtype]
        got = y.double().cpu().numpy()
        assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) / bound))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("T,H,I,E,top,norm", [
    (1, 256, 64, 4, 2, True), (1, 1024, 512, 16, 4, False), (1, 1, 1, 1, 1, True), (2, 33, 17, 3, 3, False), (5, 261, 100, 10, 3, True),
    (7, 1044, 250, 5, 2, False), (16, 512, 96, 64, 8, True), (64, 320, 72, 8, 2, True), (33, 96, 40, 256, 16, True), (64, 128, 136, 2, 1, False),
    (40, 2048, 24, 3, 2, True), (3, 64, 2080, 2, 2, True)])
def test_against_the_plain_form(T, H, I, E, top, norm, fmt, dtype):
    layer = Layer(T, H, I, E, top, dtype, FMT[fmt], norm, seed=T + H + I)
    out = layer.run()
    assert_clean_status()
    layer.check(*out)


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("T,H,I", [(64, 64, 48), (9, 16384, 8), (6, 40, 16384), (64, 4100, 24)])
def test_all_tokens_on_one_expert(T, H, I, fmt):
    """More tokens than one pass takes; the longest rows, of which a pass takes few."""
    router = torch.zeros(5, H)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(1))
    x[:, 0] = x[:, 0].abs() + 1
    router[3, 0], router[1, 0] = 2.0, 1.0
    layer = Layer(T, H, I, 5, 2, torch.float16, FMT[fmt], True, seed=2, x=x, router=router)
    out = layer.run()
    assert_clean_status()
    layer.check(*out)
    assert (out[1] == torch.tensor([3, 1], device=dev())).all()


def test_ties_go_to_the_lowest_index_and_batches_do_not_change_a_token():
    H, E = 200, 12
    router = torch.randn(E, H, generator=torch.Generator().manual_seed(3))
    router[5], router[9], router[2] = router[1], router[1], router[11]
    layer = Layer(20, H, 64, E, 7, torch.bfloat16, ig.BM_F4_E4M3, seed=4, router=router)
    y, ids, weights = layer.run()
    logits, order, p = layer.select()
    rounded = np.round(logits, 9)                                 # equal rows give equal logits whatever the order of the sum
    assert np.array_equal(ids.cpu().numpy(), np.argsort(-rounded, axis=1, kind="stable")[:, :7])
    for t in (0, 7, 19):
        one = layer.run(layer.x[t:t + 1].to(dev()))
        assert torch.equal(one[1][0], ids[t]) and torch.equal(one[2][0], weights[t])
        assert torch.allclose(one[0][0].float(), y[t].float(), rtol=2.0 ** -6, atol=2.0 ** -10 * y[t].abs().max().item())    # K may be cut differently


@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** 100])
def test_bf16_activations_far_from_one(scale):
    """Rows beyond fp16's range: x is moved by a power of two, the hidden activations likewise."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(3, 128, generator=g)
    layer = Layer(3, 128, 64, 4, 2, torch.bfloat16, ig.BM_F4_E4M3, seed=6, x=x * scale, router=torch.randn(4, 128, generator=g) / scale / 11)
    if scale > 1:                                                 # silu(g) * u of 2^200 would leave fp32: weights that keep it inside
        layer.plain["w13"] = (layer.plain["w13"].float() * 2.0 ** -60).bfloat16()
        layer.w["w13"] = ig.quantize_f4(layer.plain["w13"].to(dev()), layer.fmt, ig.BM_SCALE_ROWS)
    out = layer.run()
    assert_clean_status()
    if scale < 1:                                                 # products of 2^-200 vanish in fp32: only that nothing else appears
        assert torch.isfinite(out[0]).all() and out[0].abs().max() < 2.0 ** -100
        logits, order, p = layer.select()
        assert np.array_equal(out[1].cpu().numpy(), order)
    else:
        layer.check(*out)


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_nan_and_infinity_stay_in_their_token_and_expert(dtype, fmt):
    layer = Layer(6, 96, 48, 4, 2, dtype, FMT[fmt], seed=7)
    clean = layer.run()
    x = layer.x.clone()
    x[2, 5] = float("nan")
    x[4, 9] = float("inf")
    y, ids, weights = layer.run(x.to(dev()))
    for t in (0, 1, 3, 5):
        assert torch.equal(y[t], clean[0][t])
    assert y[2].isnan().all() and weights[2].isnan().all() and not y[4].isfinite().any()
    assert sorted(ids[2].tolist()) == [0, 1]
    bad = layer.plain["w13"].clone()
    bad[(1 * 2 * 48) + 3, 7] = float("nan")                       # gate row 3 of expert 1
    layer.w["w13"] = ig.quantize_f4(bad.to(dev()), layer.fmt, ig.BM_SCALE_ROWS)
    y, ids, _ = layer.run()
    for t in range(6):
        if 1 in ids[t].tolist():
            assert y[t].isnan().all()
        else:
            assert torch.equal(y[t], clean[0][t])
    assert_clean_status()


def test_strided_rows_row_factors_and_a_dirty_workspace():
    layer = Layer(11, 130, 70, 6, 3, torch.float16, ig.BM_F4_E8M0, seed=8)
    wide = torch.full((11, 301), 9.0, dtype=torch.float16, device=dev())
    wide[:, 3:133] = layer.x.to(dev())
    out = torch.full((11, 207), 9.0, dtype=torch.float16, device=dev())
    from bare_metal_b200 import _lib
    ws = torch.full((_lib.load().bm_moe_f4_workspace_bytes(11, 130, 70, 6, 3) + 512,), 255, dtype=torch.uint8, device=dev())
    layer.check(*layer.run(wide[:, 3:133], out=out[:, 5:135], workspace=ws))
    assert (out[:, :5] == 9).all() and (out[:, 135:] == 9).all()
    # factors of E8M0 rows: the same as scaling the rows
    f = torch.exp2(torch.randint(-3, 4, (6 * 140,), generator=torch.Generator().manual_seed(1)).float())
    layer.plain["w13"] = (layer.plain["w13"].float() * f[:, None]).bfloat16()
    layer.w["w13"] = (*layer.w["w13"][:2], f.to(dev()))
    layer.check(*layer.run(workspace=ws))
    assert_clean_status()


def test_the_same_bits_on_every_call_on_streams_and_in_a_graph():
    layer = Layer(24, 512, 200, 16, 4, torch.bfloat16, ig.BM_F4_E4M3, seed=9)
    x = layer.x.to(dev())
    first = layer.run(x)
    for _ in range(5):
        again = layer.run(x)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for i in range(12):                                           # calls that may overlap, a workspace each
        with torch.cuda.stream(streams[i % 3]):
            outs.append(layer.run(x))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(first, o))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer.run(x)
    other = Layer(24, 512, 200, 16, 4, torch.bfloat16, ig.BM_F4_E4M3, seed=10).x
    x.copy_(other.to(dev()))
    graph.replay()
    torch.cuda.synchronize()
    layer.x = other
    layer.check(*held)
    x.copy_(other.to(dev()))
    graph.replay()
    torch.cuda.synchronize()
    layer.check(*held)
    assert_clean_status()


@pytest.mark.parametrize("fmt", list(FMT))
def test_a_busy_layer_gives_the_same_bits_and_the_right_ones(fmt):
    """Every CTA has many units in a row, experts in two passes, calls follow one another without a pause."""
    T, H, I, E, top = 32, 4096, 1408, 16, 6
    layer = Layer(T, H, I, E, top, torch.bfloat16, FMT[fmt], seed=11)
    x = layer.x.to(dev())
    outs = [layer.run(x) for _ in range(40)]
    torch.cuda.synchronize()
    assert_clean_status()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(outs[0], o))
    y, ids, weights = outs[0]
    assert np.array_equal(ids.cpu().numpy(), layer.select()[1])
    # the bound of Layer.check, on the device and with the weights given
    w13, w2 = (ig.dequantize_f4(*layer.w[n], r, k, torch.float32, layer.fmt, ig.BM_SCALE_ROWS) for n, r, k in
               (("w13", E * 2 * I, H), ("w2", E * H, I)))
    u1, u2 = (H / 16 + 32) * 2.0 ** -23, (I / 16 + 32) * 2.0 ** -23
    left = lambda v, dv: torch.from_numpy(layer.left(v.cpu().numpy(), dv if isinstance(dv, float) else dv.cpu().numpy())).to(dev())  # noqa: E731
    xd = x.double()
    dx = left(xd, 0.0)
    want, bound = torch.zeros(T, H, dtype=torch.float64, device=dev()), torch.zeros(T, H, dtype=torch.float64, device=dev())
    for e in range(E):
        t, k = (ids == e).nonzero(as_tuple=True)
        if len(t) == 0:
            continue
        a, b = w13[e * 2 * I:(e + 1) * 2 * I].double(), w2[e * H:(e + 1) * H].double()
        gu, du = xd[t] @ a.T, (u1 * xd[t].abs() + dx[t]) @ a.abs().T
        g, u = gu[:, :I], gu[:, I:]
        s = g / (1 + torch.exp(-g))
        h = s * u
        dh = 1.1 * du[:, :I] * (u.abs() + du[:, I:]) + s.abs() * du[:, I:] + h.abs() * (8 + g.abs()) * 2.0 ** -24
        dh = dh + left(h, dh)
        p = weights[t, k].double()[:, None]
        want.index_add_(0, t, p * (h @ b.T))
        bound.index_add_(0, t, p * ((dh + u2 * h.abs()) @ b.abs().T + 1e-6 * (h @ b.T).abs()))
    bound = bound * 1.01 + HALF[torch.bfloat16] * (want.abs() + bound)
    assert ((y.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("T,H,I,E,top", [(64, 16384, 64, 16, 16), (64, 64, 16384, 16, 16), (64, 256, 64, 256, 16)])
def test_runs_of_one_unit(T, H, I, E, top):
    """Units so short that the sums wait while the next experts' activations are made ready."""
    layer = Layer(T, H, I, E, top, torch.bfloat16, ig.BM_F4_E8M0, seed=12)
    x = layer.x.to(dev())
    outs = [layer.run(x) for _ in range(10)]
    torch.cuda.synchronize()
    assert_clean_status()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(outs[0], o))
    if E == 256:
        layer.check(*outs[0])


def test_the_largest_activations():
    """E8M0 blocks hold up to 1.7 * 2^127; a larger number's token is NaN, not a wrong number, and the others are not touched."""
    layer = Layer(4, 96, 40, 3, 2, torch.bfloat16, ig.BM_F4_E8M0, seed=13, spread=0.0)
    layer.plain["w13"] = (layer.plain["w13"].float() * 2.0 ** -120).bfloat16()
    layer.w["w13"] = ig.quantize_f4(layer.plain["w13"].to(dev()), layer.fmt, ig.BM_SCALE_ROWS)
    layer.router_here = (layer.router.float() * 2.0 ** -125).bfloat16().to(dev())
    layer.router = layer.router_here.cpu()
    x = layer.x.float()
    x[1] *= 2.0 ** 126 / x[1].abs().max()
    x[1, 7] = 1.69 * 2.0 ** 127
    layer.x = x.bfloat16()
    first = layer.run()
    layer.check(*first)
    layer.x[2, 11] = 1.75 * 2.0 ** 127
    y, ids, weights = layer.run()
    assert y[2].isnan().all()
    for t in (0, 1, 3):
        assert torch.equal(y[t], first[0][t])
    assert_clean_status()


def test_the_output_may_take_the_place_of_the_input():
    layer = Layer(19, 136, 48, 6, 2, torch.float16, ig.BM_F4_E4M3, seed=14)
    x = layer.x.to(dev())
    out = layer.run(x, out=x)
    assert out[0] is x
    layer.check(*out)
    assert_clean_status()
