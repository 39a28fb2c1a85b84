"""Expert layers, linear layers and other kernels on several streams and in graphs that are replayed at the same time."""
import pytest
import torch

from bare_metal_b200 import igemm as ig
from _gpu import assert_clean_status, dev
from test_gpu_moe_f4 import Layer

pytestmark = pytest.mark.gpu


def test_graphs_that_are_replayed_at_the_same_time():
    """Two decoding steps (linear layer, expert layer, linear layer), each with its own workspace, beside each other and a third stream's kernels."""
    steps = []
    for seed, (T, H, I, E, top, fmt) in enumerate([(24, 1024, 512, 32, 4, ig.BM_F4_E4M3), (7, 2048, 256, 64, 6, ig.BM_F4_E8M0)]):
        layer = Layer(T, H, I, E, top, torch.bfloat16, fmt, seed=60 + seed)
        w = ig.quantize_f4((torch.randn(H, H, generator=torch.Generator().manual_seed(seed)) / H ** 0.5).bfloat16().to(dev()), fmt)
        x, a, b = layer.x.to(dev()), torch.empty(T, H, dtype=torch.bfloat16, device=dev()), torch.empty(T, H, dtype=torch.bfloat16, device=dev())
        workspace = torch.empty(ig._moe_f4_bytes(T, H, I, E, top), dtype=torch.uint8, device=dev())

        def step(layer=layer, w=w, x=x, a=a, b=b, workspace=workspace, T=T, H=H, fmt=fmt):
            ig.f4_linear(*ig.quantize_f4(x, fmt), *w, a, T, H, H, fmt)
            y, ids, weights = layer.run(a, workspace=workspace)
            ig.f4_linear(*ig.quantize_f4(y, fmt), *w, b, T, H, H, fmt)
            return y, ids, weights, b

        alone = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = [step() for _ in range(3)]
        steps.append((graph, held, alone, step))
    streams = [torch.cuda.Stream() for _ in range(3)]
    noise = torch.zeros(1 << 22, device=dev())
    torch.cuda.synchronize()
    for i in range(40):
        for (graph, _, _, _), stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            noise.add_(1.0)
    torch.cuda.synchronize()
    assert_clean_status()
    for _, held, alone, step in steps:
        for out in (*held, step()):
            assert all(torch.equal(p, q) for p, q in zip(alone, out))
    assert alone[0].isfinite().all()


def test_calls_on_three_streams():
    """Every expert layer wants all SMs at once; whichever comes first, all end with their own results."""
    layers = [Layer(T, 768, 384, 24, 3, torch.float16, fmt, seed=70 + T) for T, fmt in ((1, ig.BM_F4_E4M3), (16, ig.BM_F4_E8M0), (64, ig.BM_F4_E4M3))]
    inputs = [layer.x.to(dev()) for layer in layers]
    alone = [layer.run(x) for layer, x in zip(layers, inputs)]
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    for _ in range(60):
        outs = []
        for layer, x, stream in zip(layers, inputs, streams):
            with torch.cuda.stream(stream):
                outs.append(layer.run(x))
    torch.cuda.synchronize()
    assert_clean_status()
    for want, got in zip(alone, outs):
        assert all(torch.equal(p, q) for p, q in zip(want, got))
