"""The bf16 product that walks several tiles per workgroup, captured into graphs: its tile counters belong to one launch, whatever
else replays or runs meanwhile."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_streaming_product_in_two_graphs_and_eager():
    from distributed_pytorch_amd import _ext

    C = _ext.C()
    M, N, K = 49152, 1024, 256  # 768 tiles of 256 x 256: three per compute unit
    w = torch.randint(-3, 4, (N, K), device=DEV).bfloat16()
    xs = [torch.randint(-3, 4, (M, K), device=DEV).bfloat16() for _ in range(3)]
    want = [C.gemm(x, w, True, True) for x in xs]
    for x, y in zip(xs, want):
        assert torch.equal(y.float(), (x.float() @ w.float().t()).bfloat16().float())  # whole numbers: exact sums
    inputs = [xs[0].clone(), xs[1].clone()]
    graphs, outs = [], []
    for x in inputs:
        C.gemm(x, w, True, True)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(C.gemm(x, w, True, True))
        graphs.append(g)
    side = torch.cuda.Stream()
    for k in range(6):
        inputs[0].copy_(xs[k % 3])
        inputs[1].copy_(xs[(k + 1) % 3])
        torch.cuda.synchronize()
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        eager = C.gemm(xs[2], w, True, True)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[k % 3]) and torch.equal(outs[1], want[(k + 1) % 3]) and torch.equal(eager, want[2])
