"""What the 4-bit operators' Python entry points refuse, on device tensors: an error before any launch."""
import pytest
import torch

from bare_metal_b200 import igemm as ig
from _gpu import assert_clean_status, dev

pytestmark = pytest.mark.gpu


def bad(call, *args, **kw):
    with pytest.raises(ig.BmError):
        call(*args, **kw)


def test_quantize_and_back():
    x = torch.randn(5, 96, device=dev()).half()
    for t in (x.cpu(), x.float(), x[0], x.t(), x[:, ::2], x[:1].expand(5, 96), x[:0], x[:, :0]):
        bad(ig.quantize_f4, t)
    bad(ig.quantize_f4, x, 7)
    bad(ig.quantize_f4, x, ig.BM_F4_E8M0, 9)
    q, s, r = ig.quantize_f4(x)
    for parts in ((q.cpu(), s, r), (q[:4], s, r), (q, s[:-1], r), (q.view(torch.int8), s, r), (q, s, r[:4]), (q, s, r.double()),
                  (torch.empty(5, 96, dtype=torch.uint8, device=dev())[:, ::2], s, r)):
        bad(ig.dequantize_f4, *parts, 5, 96)
    bad(ig.dequantize_f4, q, s, r, 5, 96, torch.int8)
    for out in (torch.empty(5, 95, device=dev()), torch.empty(5, 96), torch.empty(5, 96, dtype=torch.float64, device=dev()),
                torch.empty(96, 5, device=dev()).t(), torch.empty(1, 96, device=dev()).expand(5, 96)):
        bad(ig.dequantize_f4, q, s, r, 5, 96, out=out)
    off = torch.empty(q.numel() + 16, dtype=torch.uint8, device=dev())[1:1 + q.numel()]
    bad(ig.dequantize_f4, off, s, r, 5, 96)                       # not 16-byte aligned
    assert torch.isfinite(ig.dequantize_f4(q, s, r, 5, 96)).all()
    assert_clean_status()


def test_linear():
    x, w = ig.quantize_f4(torch.randn(5, 96, device=dev()).half()), ig.quantize_f4(torch.randn(40, 96, device=dev()).half())
    d = torch.empty(5, 40, dtype=torch.float16, device=dev())
    for out in (d.cpu(), d[:4], d.double(), d.t(), torch.empty(40, 5, dtype=torch.float16, device=dev()).t(), d[:1].expand(5, 40)):
        bad(ig.f4_linear, *x, *w, out, 5, 40, 96)
    bad(ig.f4_linear, *x, *w, d, 5, 40, 160)                      # more columns than the operands hold
    bad(ig.f4_linear, *x, *w, d, 5, 40, 96, 5)
    bad(ig.f4_linear, x[0], x[1][:-1], x[2], *w, d, 5, 40, 96)
    bad(ig.f4_linear, *x, w[0], w[1], w[2][:39], d, 5, 40, 96)
    assert torch.isfinite(ig.f4_linear(*x, *w, d, 5, 40, 96)).all()
    assert_clean_status()


def test_expert_layer():
    T, H, I, E, top = 3, 64, 32, 4, 2
    x, router = torch.randn(T, H, device=dev()).half(), torch.randn(E, H, device=dev()).half()
    w13 = ig.quantize_f4(torch.randn(E * 2 * I, H, device=dev()).half(), scale_layout=ig.BM_SCALE_ROWS)
    w2 = ig.quantize_f4(torch.randn(E * H, I, device=dev()).half(), scale_layout=ig.BM_SCALE_ROWS)
    good = dict(X=x, router=router, w13=w13, w2=w2, top=top, inter=I)
    run = lambda **k: ig.moe_f4(**{**good, **k})  # noqa: E731
    for t in (x.cpu(), x.float(), x[0], x.t(), x[:, :60], torch.randn(65, H, device=dev()).half(), x[:0], x[:1].expand(T, H)):
        bad(run, X=t)
    for t in (router.cpu(), router.bfloat16(), router[:, :60], router[0], router[:0], router.t().contiguous().t()):
        bad(run, router=t)
    for k in (0, 5, -1):
        with pytest.raises((ig.BmError, RuntimeError)):           # (torch refuses a negative shape by itself)
            run(top=k)
    bad(run, inter=33)
    bad(run, inter=0)
    bad(run, fmt=3)
    bad(run, w13=(w13[0][:-1], *w13[1:]))
    bad(run, w2=(w2[0], w2[1][:-1], w2[2]))
    bad(run, w2=(w2[0], w2[1], w2[2][:-1]))
    bad(run, out=torch.empty(T, H, device=dev()))
    bad(run, out=torch.empty(T, H - 1, dtype=torch.float16, device=dev()))
    need = ig._moe_f4_bytes(T, H, I, E, top)
    bad(run, workspace=torch.empty(need - 1, dtype=torch.uint8, device=dev()))
    bad(run, workspace=torch.empty(need + 256, dtype=torch.uint8, device=dev())[16:])
    bad(run, workspace=torch.empty(need, dtype=torch.uint8))
    assert torch.isfinite(run()[0]).all()
    assert_clean_status()
