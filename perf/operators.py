"""The 4-bit floating-point operators of this library, as cases that can be timed and compared.

Kinds
  readback   rows of fp16 / bf16 are quantised to 4-bit values with block scales and read back: what a program
             does that keeps weights or activations in 4 bits and needs them as numbers again
  linear     one linear layer with 4-bit weights: 16-bit activations are quantised, then multiplied
  moe        a whole mixture-of-experts layer for a few tokens: router, selection, gate / up, SiLU, down, weighted sum

Formats of the 4-bit data (values E2M1, two to a byte, the lower position in the low bits)
  e8m0       blocks of 32 along a row, scale 2^(byte - 127)
  e4m3       blocks of 16, the scale an E4M3 byte, and one power of two per row

`own` chooses between the library's calls and the plain form of the same operators in elementary torch operations.
"""
import math

import torch

own = False

_DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BLOCK = {"e8m0": 32, "e4m3": 16}


def listed():
    return [
        # a decoding step's activations: latency and launch cost count
        dict(name="readback_16x4096", kind="readback", rows=16, k=4096, dtype="f16", fmt="e4m3", layout="tiled"),
        # an odd number of rows that are a part of wider ones, and a length that ends inside a block
        dict(name="readback_777x4100", kind="readback", rows=777, k=4100, dtype="f16", fmt="e8m0", layout="rows"),
        # a weight matrix or a full prefill batch
        dict(name="readback_8192x11008", kind="readback", rows=8192, k=11008, dtype="bf16", fmt="e4m3", layout="tiled"),
        # decoding, one sequence: a very wide layer whose weights are read once for one token
        dict(name="linear_1_token", kind="linear", m=1, n=28672, k=8192, dtype="f16", out="f16", fmt="e8m0"),
        # decoding with a batch of 16 sequences
        dict(name="linear_16_tokens", kind="linear", m=16, n=4096, k=4096, dtype="f16", out="f16", fmt="e4m3"),
        # every dimension off the tiles, fp32 results
        dict(name="linear_ragged", kind="linear", m=777, n=2260, k=1000, dtype="bf16", out="f32", fmt="e4m3"),
        # a square layer in prefill
        dict(name="linear_4096", kind="linear", m=4096, n=4096, k=4096, dtype="f16", out="f16", fmt="e4m3"),
        # gate and up projection of a full prefill batch
        dict(name="linear_8192_tokens", kind="linear", m=8192, n=22016, k=4096, dtype="bf16", out="bf16", fmt="e8m0"),
        # one token through a layer of 64 experts
        dict(name="moe_1_token", kind="moe", t=1, h=4096, i=1408, e=64, top=6, dtype="f16", fmt="e4m3", norm=True),
        # small odd sizes, probabilities kept as they are
        dict(name="moe_ragged", kind="moe", t=5, h=1044, i=1000, e=10, top=3, dtype="f16", fmt="e8m0", norm=False),
        # a batch of 16 tokens over many small experts
        dict(name="moe_16_tokens", kind="moe", t=16, h=2048, i=768, e=128, top=8, dtype="bf16", fmt="e4m3", norm=True),
        # the largest batch: nearly every expert has work, several tokens each
        dict(name="moe_64_tokens", kind="moe", t=64, h=4096, i=1408, e=64, top=6, dtype="bf16", fmt="e8m0", norm=True),
    ]


def draw(rng):
    def size(low, high, step=1):
        return max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / step)) * step)

    kind = rng.choice(("readback", "linear", "linear", "moe", "moe"))
    dtype, fmt = rng.choice(("f16", "bf16")), rng.choice(("e8m0", "e4m3"))
    step = rng.choice((1, 4, 32, 128))
    if kind == "readback":
        k = size(32, 16384, step)
        rows = size(1, min(16384, 8192 * 11008 // k))
        return dict(kind=kind, rows=rows, k=k, dtype=dtype, fmt=fmt, layout=rng.choice(("rows", "tiled")))
    if kind == "linear":
        k = size(64, 11008, step)
        n = size(64, min(28672, 28672 * 8192 // k), rng.choice((1, 4, 64)))
        m = size(1, min(8192, max(16, 8192 * 22016 * 4096 // (n * k))))
        return dict(kind=kind, m=m, n=n, k=k, dtype=dtype, out=rng.choice((dtype, dtype, "f32")), fmt=fmt)
    h, e = size(256, 4096, step), size(2, 128)
    i = size(64, max(64, min(11008, 64 * 4096 * 1408 // (e * h))), rng.choice((1, 8, 64)))
    return dict(kind=kind, t=size(1, 64), h=h, i=i, e=e, top=rng.randint(1, min(8, e)), dtype=dtype, fmt=fmt, norm=rng.random() < 0.7)


# ---------------------------------------------------------------------------------------------------------------
# the formats in elementary operations
# ---------------------------------------------------------------------------------------------------------------
def _magnitudes(device):
    return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=device)


def _pow2(exponent):
    """2 ** exponent for whole exponents from -126 to 127."""
    return ((exponent.to(torch.int32) + 127) << 23).view(torch.float32)


def _blocks(x, fmt):
    """fp32 rows -> (4-bit codes, blocks' scales as stored bytes, rows' exponents or None), K padded to whole 32s."""
    rows, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % 32)).view(rows, -1, _BLOCK[fmt])
    size = x.abs()
    good = torch.isfinite(size)
    whole = good.all(-1)
    size = torch.where(good, size, 0.0).amax(-1)
    if fmt == "e8m0":
        lg = torch.frexp(size)[1] - 1
        byte = torch.where(size > 0, (lg - 2 + 127).clamp(0, 254), 0)
        y = x * _pow2(127 - byte)[..., None]
        byte, row = torch.where(whole, byte, 255).to(torch.uint8), None
    else:
        top = size.amax(-1)
        row = torch.where(top > 0, (torch.frexp(top)[1] - 11).clamp(min=-126), 0)
        inv = _pow2(-row)[:, None]
        scale = (size * inv / 6.0).to(torch.float8_e4m3fn)
        s = scale.float()[..., None]
        y = torch.where(s > 0, x * inv[..., None] / torch.where(s > 0, s, 1.0), 0.0)
        byte = torch.where(whole, scale.view(torch.uint8), 127)
    y = torch.where(whole[..., None], y, 0.0)
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
            + torch.where(torch.signbit(y), 8, 0)).to(torch.uint8)
    return code.view(rows, -1), byte, row


def _scale_values(byte, fmt):
    if fmt == "e4m3":
        return byte.view(torch.float8_e4m3fn).float()
    b = byte.int()
    return torch.where(b == 0, 2.0 ** -127, torch.where(b == 255, math.nan, _pow2(b.clamp(1, 254) - 127)))


def _lut(device):
    m = _magnitudes(device)
    return torch.cat((m, -m))


def _values(code, byte, fmt):
    """Codes and scale bytes -> fp32 numbers, without the rows' factors."""
    v = _lut(code.device).index_select(0, code.int().flatten()).view(*byte.shape, _BLOCK[fmt])
    return (v * _scale_values(byte, fmt)[..., None]).flatten(-2)


def _pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _unpacked(q, byte, fmt):
    """Packed rows and their scale bytes -> fp32 numbers, without the rows' factors."""
    lut = _lut(q.device)
    pairs = torch.stack((lut.repeat(16), lut.repeat_interleave(16)), -1)
    v = pairs.index_select(0, q.int().flatten()).view(*byte.shape, _BLOCK[fmt])
    return (v * _scale_values(byte, fmt)[..., None]).flatten(-2)


def _tiled(byte):
    """Scale bytes [rows, groups] -> tiles of 128 rows x 4 groups, 512 bytes each, zero-filled."""
    rows, groups = byte.shape
    byte = torch.nn.functional.pad(byte, (0, -groups % 4, 0, -rows % 128))
    return byte.view(byte.shape[0] // 128, 4, 32, -1, 4).permute(0, 3, 2, 1, 4).contiguous().flatten()


def _untiled(tiles, rows, groups):
    t = tiles.view(-(-rows // 128), -(-groups // 4), 32, 4, 4).permute(0, 3, 2, 1, 4)
    return t.reshape(-(-rows // 128) * 128, -1)[:rows, :groups]


def _in_rows(byte):
    """Scale bytes [rows, groups] in rows of a multiple of 16 bytes, zero-filled."""
    return torch.nn.functional.pad(byte, (0, -byte.shape[-1] % 16))


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _activations(g, rows, k, dtype, wider=0):
    """Token rows of different size with a few channels that are much larger than the others."""
    x = torch.randn(rows, k + wider, device="cuda", generator=g)
    x *= torch.exp2(torch.randn(rows, 1, device="cuda", generator=g))
    x[:, torch.randint(0, k, (max(1, k // 200),), device="cuda", generator=g)] *= 20.0
    return x.to(dtype)[:, :k]


def _weights(g, rows, k, fmt):
    w = torch.randn(rows, k, device="cuda", generator=g) * (0.02 * torch.exp2(torch.randn(rows, 1, device="cuda", generator=g) / 4))
    code, byte, row = _blocks(w.bfloat16().float(), fmt)
    return _pack(code), byte, None if row is None else _pow2(row)


def _expert_weights(g, e, rows, k, fmt):
    parts = [_weights(g, rows, k, fmt) for _ in range(e)]
    q, byte = torch.cat([p[0] for p in parts]), _in_rows(torch.cat([p[1] for p in parts]))
    return q, byte, None if fmt == "e8m0" else torch.cat([p[2] for p in parts])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    st, fmt, dtype = dict(case), case["fmt"], _DTYPE[case["dtype"]]
    if case["kind"] == "readback":
        st["x"] = _activations(g, case["rows"], case["k"], dtype, wider=-case["k"] % 8 + 8 if case["layout"] == "rows" else 0)
    elif case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        st["x"] = _activations(g, m, k, dtype)
        q, byte, row = _weights(g, n, k, fmt)
        st["w"] = (q, _tiled(byte), row)
        st["d"] = torch.empty(m, n, dtype=_DTYPE[case["out"]], device="cuda")
    else:
        t, h, i, e = (case[k] for k in ("t", "h", "i", "e"))
        st["x"] = torch.randn(t, h, device="cuda", generator=g).to(dtype)
        st["router"] = (torch.randn(e, h, device="cuda", generator=g) * (1.5 / math.sqrt(h))).to(dtype)
        st["w13"] = _expert_weights(g, e, 2 * i, h, fmt)
        st["w2"] = _expert_weights(g, e, h, i, fmt)
        st["y"] = torch.empty(t, h, dtype=dtype, device="cuda")
    return st


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(st):
    return {"readback": _readback, "linear": _linear, "moe": _moe}[st["kind"]](st)


def _fmt_tag(ig, fmt):
    return ig.BM_F4_E8M0 if fmt == "e8m0" else ig.BM_F4_E4M3


def _scale_view(s, fmt):
    return s.view(torch.float8_e8m0fnu if fmt == "e8m0" else torch.float8_e4m3fn)


def _readback(st):
    x, fmt = st["x"], st["fmt"]
    if own:
        from bare_metal_b200 import igemm as ig
        layout = ig.BM_SCALE_ROWS if st["layout"] == "rows" else ig.BM_SCALE_TILED
        q, s, r = ig.quantize_f4(x, _fmt_tag(ig, fmt), layout)
        values = ig.dequantize_f4(q, s, r, st["rows"], st["k"], x.dtype, _fmt_tag(ig, fmt), layout)
        out = {"values": values, "scales": _scale_view(s, fmt)}
        return out if r is None else {**out, "rows": r}
    code, byte, row = _blocks(x.float(), fmt)
    v = _values(code, byte, fmt)
    if row is not None:
        v = v * _pow2(row)[:, None]
    out = {"values": v[:, :st["k"]].to(x.dtype),
           "scales": _scale_view(_in_rows(byte) if st["layout"] == "rows" else _tiled(byte), fmt)}
    return out if row is None else {**out, "rows": _pow2(row)}


def _linear(st):
    x, (wq, ws, wr), fmt, m, n, k = st["x"], st["w"], st["fmt"], st["m"], st["n"], st["k"]
    if own:
        from bare_metal_b200 import igemm as ig
        q, s, r = ig.quantize_f4(x, _fmt_tag(ig, fmt), ig.BM_SCALE_TILED)
        return ig.f4_linear(q, s, r, wq, ws, wr, st["d"], m, n, k, _fmt_tag(ig, fmt))
    code, byte, row = _blocks(x.float(), fmt)
    a = _values(code, byte, fmt)
    w = _unpacked(wq, _untiled(ws, n, byte.shape[1]).contiguous(), fmt)
    d = a @ w.t()
    if row is not None:
        d = d * (_pow2(row)[:, None] * wr)
    return d.to(_DTYPE[st["out"]])


def _select(st):
    """Router: the experts of each token, their weights in fp32.  Logits in 64 bits: two that are near decide a token's way."""
    logits = st["x"].double() @ st["router"].double().t()
    ranked, ids = torch.sort(logits, dim=1, descending=True, stable=True)
    part = ranked[:, :st["top"]]
    p = torch.softmax(part, 1) if st["norm"] else torch.softmax(logits, 1).gather(1, ids[:, :st["top"]])
    return ids[:, :st["top"]], p.float()


def _moe(st):
    fmt, e, i, h, t, top = st["fmt"], st["e"], st["i"], st["h"], st["t"], st["top"]
    if own:
        from bare_metal_b200 import igemm as ig
        y, ids, p = ig.moe_f4(st["x"], st["router"], st["w13"], st["w2"], top, i, _fmt_tag(ig, fmt), st["norm"], out=st["y"])
        return {"y": y, "experts": ids, "weights": p}
    ids, p = _select(st)
    x = st["x"].float()

    def experts(weights, rows, which):
        q, byte, row = weights
        groups = q.shape[1] * 2 // _BLOCK[fmt]
        q, byte = q.view(e, rows, -1), byte.view(e, rows, -1)[..., :groups]
        row = None if row is None else row.view(e, rows)
        if which is not None:
            q, byte, row = q[which], byte[which], None if row is None else row[which]
        w = _unpacked(q, byte.contiguous(), fmt)
        return w if row is None else w * row[..., None]

    if t * top <= e:                                  # every chosen expert's weights for its one token
        which = ids.flatten()
        w13 = experts(st["w13"], 2 * i, which)
        xs = torch.nn.functional.pad(x, (0, w13.shape[2] - h))[torch.arange(t, device=x.device).repeat_interleave(top)]
        gu = torch.bmm(w13, xs[..., None])[..., 0]
        a = torch.nn.functional.silu(gu[:, :i]) * gu[:, i:]
        w2 = experts(st["w2"], h, which)
        y = torch.bmm(w2, torch.nn.functional.pad(a, (0, w2.shape[2] - i))[..., None])[..., 0]
        y = (y.view(t, top, h) * p[..., None]).sum(1)
    else:                                             # all experts for all tokens, then the chosen ones
        w13 = experts(st["w13"], 2 * i, None)
        gu = torch.matmul(torch.nn.functional.pad(x, (0, w13.shape[2] - h)), w13.transpose(1, 2))
        a = torch.nn.functional.silu(gu[..., :i]) * gu[..., i:]
        w2 = experts(st["w2"], h, None)
        y = torch.matmul(torch.nn.functional.pad(a, (0, w2.shape[2] - i)), w2.transpose(1, 2))
        share = torch.zeros(t, e, device=x.device).scatter(1, ids, p)
        y = (y * share.t()[..., None]).sum(0)
    return {"y": y.to(st["x"].dtype), "experts": ids.int(), "weights": p}


# ---------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------
_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _nearest(v, grid):
    """Index of the nearest point of an ascending grid, of two equally near ones the even index; beyond the last: the last."""
    grid = torch.tensor(grid, dtype=torch.float64, device=v.device)
    hi = torch.searchsorted(grid, v).clamp(1, len(grid) - 1)
    down, up = v - grid[hi - 1], grid[hi] - v
    return torch.where((down < up) | ((down == up) & (hi % 2 == 1)), hi - 1, hi)


def _exact_rows(x, fmt):
    """(values without the rows' factors, scales, rows' factors) of finite rows, in 64 bits."""
    x = x.double()
    rows, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % 32)).view(rows, -1, _BLOCK[fmt])
    most = x.abs().amax(-1, keepdim=True)
    def pow2(n):
        return torch.ldexp(torch.ones(n.shape, dtype=torch.float64, device=x.device), n)

    if fmt == "e8m0":
        scale = pow2((torch.frexp(most)[1] - 3).clamp(-127, 127))
        scale = torch.where(most > 0, scale, 2.0 ** -127)
        row = None
    else:
        top = most.amax(1, keepdim=True)
        row = torch.where(top > 0, pow2((torch.frexp(top)[1] - 11).clamp(min=-126)), 1.0)
        e4m3 = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1]
        points = torch.tensor(e4m3, dtype=torch.float64, device=x.device)
        scale = points[_nearest(most / (6 * row), e4m3)]
        x = x / row
    safe = torch.where(scale > 0, scale, 1.0)
    v = torch.tensor(_GRID, dtype=torch.float64, device=x.device)[_nearest(x.abs() / safe, _GRID)] * torch.sign(x) * scale
    return v.flatten(1), scale[..., 0], None if row is None else row.flatten()


def _exact_stored(q, byte, row, fmt):
    """Stored rows as numbers, in 64 bits."""
    low, high = (q & 15).long(), (q >> 4).long()
    code = torch.stack((low, high), -1).flatten(1)
    v = torch.tensor(_GRID + [-x for x in _GRID], dtype=torch.float64, device=q.device)[code]
    groups = v.shape[1] // _BLOCK[fmt]
    s = _scale_view(byte[:, :groups].contiguous(), fmt).double().repeat_interleave(_BLOCK[fmt], 1)
    v = v * s
    return v if row is None else v * row.double()[:, None]


def exact(case, seed):
    st = prepare(case, seed)
    fmt, x = case["fmt"], st["x"]
    if case["kind"] == "readback":
        v, s, row = _exact_rows(x, fmt)
        v = v if row is None else v * row[:, None]
        s = torch.nn.functional.pad(s, (0, -s.shape[1] % 16), value=2.0 ** -127 if fmt == "e8m0" else 0.0) if case["layout"] == "rows" else None
        out = {"values": v[:, :case["k"]], "scales": s}
        return out if row is None else {**out, "rows": row}
    if case["kind"] == "linear":
        a, _, row = _exact_rows(x, fmt)
        wq, ws, wr = st["w"]
        groups = wq.shape[1] * 2 // _BLOCK[fmt]
        w = _exact_stored(wq, _untiled(ws, case["n"], groups), wr, fmt)
        d = a @ w.t()
        return d if row is None else d * row[:, None]
    t, h, i, e, top = (case[k] for k in ("t", "h", "i", "e", "top"))
    x = x.double()
    logits = x @ st["router"].double().t()
    order = torch.argsort(-logits, dim=1, stable=True)[:, :top]
    z = torch.exp(logits - logits.amax(1, keepdim=True))
    p = z.gather(1, order)
    p = p / (p if case["norm"] else z).sum(1, keepdim=True)
    y = torch.zeros(t, h, dtype=torch.float64, device=x.device)
    for n in range(e):
        at = (order == n).nonzero()
        if not len(at):
            continue
        w13, w2 = (_exact_stored(q[n * r:(n + 1) * r], byte[n * r:(n + 1) * r], None if row is None else row[n * r:(n + 1) * r], fmt)
                   for (q, byte, row), r in ((st["w13"], 2 * i), (st["w2"], h)))
        gu = x[at[:, 0]] @ w13[:, :h].t()
        a = gu[:, :i] / (1 + torch.exp(-gu[:, :i])) * gu[:, i:]
        y.index_add_(0, at[:, 0], (a @ w2[:, :i].t()) * p[at[:, 0], at[:, 1], None])
    return {"y": y, "experts": None, "weights": p}


# ---------------------------------------------------------------------------------------------------------------
# what one pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def _stored_bytes(rows, k, fmt):
    """Values and scales of quantised rows (and the rows' factors)."""
    return rows * (-(-k // 2) + -(-k // _BLOCK[fmt]) + (4 if fmt == "e4m3" else 0))


def work(case):
    fmt = case["fmt"]
    if case["kind"] == "readback":
        n = case["rows"] * case["k"]
        return {"bytes": 4 * n + _stored_bytes(case["rows"], case["k"], fmt) - -(-case["k"] // 2) * case["rows"], "flops": 0}
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * k + _stored_bytes(n, k, fmt) + m * n * (4 if case["out"] == "f32" else 2), "flops": 2.0 * m * n * k}
    t, h, i, e, top = (case[k] for k in ("t", "h", "i", "e", "top"))
    busy = e * (1 - (1 - top / e) ** t)                          # experts that have work, on average
    return {"bytes": 2 * e * h + 4 * t * h + busy * (_stored_bytes(2 * i, h, fmt) + _stored_bytes(h, i, fmt)),
            "flops": 2.0 * t * (e * h + top * 3 * h * i)}
