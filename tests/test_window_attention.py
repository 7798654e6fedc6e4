"""Attention with a sliding window and sinks: outputs and gradients against float64 with bounds derived from the roundings,
padded batches, strides, streams, graphs, refusals."""
import math

import pytest
import torch

from distributed_pytorch_amd.ops import causal_attention_qkvpacked, window_attention_qkvpacked

gpu = pytest.mark.gpu
DEV = "cuda"


def reference(qkv, do, H, KV, window, sinks, lens=None, scale=None, dtype=torch.bfloat16):
    """(o, dqkv) in float64 and, element by element, how far a kernel may be from them that rounds the probabilities, the
    score gradients and its results to `dtype` and does everything else in float32."""
    B, T, W = qkv.shape
    D, G = W // (H + 2 * KV), H // KV
    scale = D ** -0.5 if scale is None else scale
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0       # below its normal range a rounding is absolute
    x = qkv.double().view(B, T, H + 2 * KV, D).transpose(1, 2)
    i = torch.arange(T, device=qkv.device)
    ok = (i[None] <= i[:, None]) & ((i[:, None] - i[None] < window) | (i[None] < sinks))
    live = torch.ones(B, T, dtype=torch.bool, device=qkv.device) if lens is None else i[None] < lens[:, None]
    x = torch.where(live[:, None, :, None], x, 0.0)
    q, k, v = x[:, :H], x[:, H:H + KV].repeat_interleave(G, 1), x[:, H + KV:].repeat_interleave(G, 1)
    do = torch.where(live[:, None, :, None], do.double().view(B, T, H, D).transpose(1, 2), 0.0)
    on = live[:, None, :, None].double()

    def mm(a, b):
        return torch.matmul(a, b.contiguous())

    s = mm(q, k.transpose(2, 3)) * scale
    p = torch.softmax(s.masked_fill(~ok, -math.inf), 3) * on
    o = mm(p, v)
    # float32 scores: D products of which each rounding is 2^-24 of the running sum, and the exponent's own rounding
    es = (mm(q.abs(), k.abs().transpose(2, 3)) * scale * D + 64) * 2.0 ** -23
    ep = p * es + half * p + tiny                               # one probability
    ep = torch.where(ok, ep, 0.0) * on
    eo_f = 2 * mm(ep, v.abs())                                  # numerator and row sum carry the same roundings
    eo = eo_f + half * o.abs() + tiny
    dv_h = mm(p.transpose(2, 3), do)
    edv = mm(ep.transpose(2, 3), do.abs())
    dp = mm(do, v.transpose(2, 3))
    delta = (do * o).sum(3, keepdim=True)
    ds = p * (dp - delta)
    e_delta = (do.abs() * eo).sum(3, keepdim=True)
    e_dp = mm(do.abs(), v.abs().transpose(2, 3)) * D * 2.0 ** -24
    eds = torch.where(ok, p * (e_delta + e_dp) + p * es * (dp - delta).abs() + half * ds.abs() + tiny, 0.0) * on
    dq, edq = mm(ds, k) * scale, mm(eds, k.abs()) * scale
    dk_h, edk = mm(ds.transpose(2, 3), q) * scale, mm(eds.transpose(2, 3), q.abs()) * scale

    def group(t):
        return t.view(B, KV, G, T, D).sum(2)

    g = torch.cat([dq, group(dk_h), group(dv_h)], 1)
    eg = torch.cat([edq, group(edk), group(edv)], 1)
    eg = 1.01 * eg + half * g.abs() + tiny + 1e-6
    out = lambda t: t.transpose(1, 2).reshape(B, T, -1)  # noqa: E731
    return out(o), out(1.01 * eo + 1e-6), out(g), out(eg)


def run(qkv, do, H, KV, window, sinks, **kw):
    x = qkv.detach().requires_grad_()
    o = window_attention_qkvpacked(x, H, window, sinks, n_kv_head=KV, impl="native", **kw)
    (g,) = torch.autograd.grad(o, x, do)
    return o.detach(), g


def check(qkv, do, H, KV, window, sinks, lens=None, **kw):
    o, g = run(qkv, do, H, KV, window, sinks, seq_lens=lens, **kw)
    ro, eo, rg, eg = reference(qkv, do, H, KV, window, sinks, lens, kw.get("softmax_scale"), qkv.dtype)
    assert bool(((o.double() - ro).abs() <= eo).all()), float(((o.double() - ro).abs() / eo).max())
    assert bool(((g.double() - rg).abs() <= eg).all()), float(((g.double() - rg).abs() / eg).max())
    return o, g


def make(B, T, H, KV, D, dtype=torch.bfloat16, seed=0, device=DEV):
    gen = torch.Generator().manual_seed(seed)
    qkv = torch.randn(B, T, (H + 2 * KV) * D, generator=gen)
    do = torch.randn(B, T, H * D, generator=gen)
    return qkv.to(dtype).to(device), do.to(dtype).to(device)


# ------------------------------------------------------------------------------------------------ CPU
def test_composed_gradient_against_differences():
    qkv = torch.randn(2, 7, 4 * 3, dtype=torch.float64, requires_grad=True)
    lens = torch.tensor([7, 4])
    assert torch.autograd.gradcheck(lambda x: window_attention_qkvpacked(x, 2, 3, 1, n_kv_head=1, seq_lens=lens), qkv)


def test_composed_against_a_loop():
    B, T, H, KV, D, window, sinks = 2, 11, 4, 2, 8, 4, 2
    qkv = torch.randn(B, T, (H + 2 * KV) * D)
    lens = torch.tensor([11, 5], dtype=torch.int32)
    qkv[1, 5:] = float("nan")
    o = window_attention_qkvpacked(qkv, H, window, sinks, n_kv_head=KV, seq_lens=lens).view(B, T, H, D)
    x = qkv.view(B, T, H + 2 * KV, D)
    for b in range(B):
        for h in range(H):
            for i in range(T):
                if i >= lens[b]:
                    assert torch.equal(o[b, i, h], torch.zeros(D))
                    continue
                js = [j for j in range(i + 1) if i - j < window or j < sinks]
                s = torch.stack([x[b, i, h] @ x[b, j, H + h // 2] for j in js]) / math.sqrt(D)
                want = torch.softmax(s, 0) @ torch.stack([x[b, j, H + KV + h // 2] for j in js])
                torch.testing.assert_close(o[b, i, h], want, rtol=1e-5, atol=1e-5)


def test_a_window_of_the_whole_sequence_is_causal_attention():
    qkv = torch.randn(2, 9, 3 * 4 * 8)
    torch.testing.assert_close(window_attention_qkvpacked(qkv, 4, 9), causal_attention_qkvpacked(qkv, 4), rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals(device):
    qkv = torch.randn(2, 5, 6 * 64, device=device).bfloat16()
    for kw in (dict(window=0), dict(window=3, sinks=-1), dict(window=3, n_kv_head=3), dict(window=3, n_kv_head=0), dict(window=3, softmax_scale=0.0),
               dict(window=3, softmax_scale=-1.0), dict(window=3, softmax_scale=float("nan")), dict(window=3, impl="fast"),
               dict(window=3, seq_lens=torch.tensor([1, 2, 3], device=device)), dict(window=3, seq_lens=torch.tensor([1.0, 2.0], device=device))):
        with pytest.raises(ValueError):
            window_attention_qkvpacked(qkv, 2, **kw)
    with pytest.raises(ValueError):
        window_attention_qkvpacked(qkv, 5, 3)
    with pytest.raises(ValueError):
        window_attention_qkvpacked(qkv[0], 2, 3)
    with pytest.raises(RuntimeError):  # head size 32, and a type the kernels lack
        window_attention_qkvpacked(qkv, 4, 3, impl="native")
    with pytest.raises(RuntimeError):
        window_attention_qkvpacked(qkv.float(), 2, 3, impl="native")
    if device == "cuda":
        with pytest.raises(ValueError):
            window_attention_qkvpacked(qkv, 2, 3, seq_lens=torch.tensor([1, 2]))


# ------------------------------------------------------------------------------------------------ GPU
SHAPES = [
    # B, T, H, KV, window, sinks
    (1, 1, 1, 1, 1, 0), (2, 2, 2, 1, 1, 0), (3, 5, 2, 2, 3, 2), (1, 63, 2, 1, 7, 0), (2, 64, 1, 1, 64, 0), (1, 65, 2, 2, 1, 1), (2, 127, 2, 1, 40, 3),
    (1, 128, 2, 2, 128, 0), (1, 129, 3, 1, 5, 130), (2, 200, 4, 2, 33, 4), (1, 257, 2, 2, 65, 63), (1, 513, 2, 1, 100, 64), (1, 640, 2, 2, 128, 127),
    (1, 700, 2, 1, 700, 0), (3, 300, 6, 2, 64, 1), (1, 1000, 4, 1, 64, 200), (1, 2100, 4, 1, 64, 3),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,T,H,KV,window,sinks", SHAPES)
def test_against_float64(B, T, H, KV, window, sinks, D, dtype):
    check(*make(B, T, H, KV, D, dtype, seed=T), H, KV, window, sinks)


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_more_blocks_than_workgroup_slots(D):
    check(*make(8, 1000, 8, 8, D), 8, 8, 150, 5)


@gpu
def test_large_scores_and_other_scales():
    qkv, do = make(2, 300, 2, 1, 64)
    check(qkv * 6, do, 2, 1, 64, 4)                  # nearly one-hot rows: the running maximum keeps moving
    check(qkv, do, 2, 1, 64, 4, softmax_scale=0.02)
    grow = qkv * torch.linspace(0.1, 5, 300, device=DEV).view(1, 300, 1).bfloat16()
    check(grow, do, 2, 1, 200, 0)


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,H,KV,window,sinks", [(6, 130, 2, 1, 20, 2), (6, 300, 4, 2, 64, 100), (6, 65, 1, 1, 65, 0)])
def test_padded_batches(B, T, H, KV, window, sinks, D, dtype):
    lens = torch.tensor([0, 1, T, T // 2, T - 1, 64], device=DEV, dtype=torch.int32)
    qkv, do = make(B, T, H, KV, D, dtype)
    for fill in (float("nan"), float("inf")):
        for b, n in enumerate(lens.tolist()):
            qkv[b, n:] = fill
            do[b, n:] = fill
        o, g = check(qkv, do, H, KV, window, sinks, lens)
        for b, n in enumerate(lens.tolist()):
            assert torch.equal(o[b, n:], torch.zeros_like(o[b, n:])) and torch.equal(g[b, n:], torch.zeros_like(g[b, n:]))
    # lengths outside 0 .. T are taken into it, int64 works too
    wild = torch.where(lens == T, T + 1000, torch.where(lens == 0, -5, lens)).long()
    o2, g2 = run(qkv, do, H, KV, window, sinks, seq_lens=wild)
    assert torch.equal(o, o2) and torch.equal(g, g2)
    o3, g3 = run(qkv, do, H, KV, window, sinks, seq_lens=wild.int())
    assert torch.equal(o, o3) and torch.equal(g, g3)


@gpu
def test_what_no_query_sees_may_be_non_finite():
    qkv, do = make(1, 900, 2, 1, 64)
    clean, gc = run(qkv, do, 2, 1, 64, 4)
    bad = qkv.clone()
    bad[:, 10] = float("nan")        # position 10 is no sink: queries from 74 on do not see it
    o, _ = run(bad, do, 2, 1, 64, 4)
    assert torch.equal(o[:, 10 + 64 + 128:], clean[:, 10 + 64 + 128:]) and bool(torch.isnan(o[:, 10:74]).all())


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_strides_and_offsets(D):
    H, KV = 4, 2
    W = (H + 2 * KV) * D
    qkv, do = make(2, 150, H, KV, D)
    want = run(qkv, do, H, KV, 40, 3)
    wide = torch.zeros(2, 200, W + 64, dtype=qkv.dtype, device=DEV)
    view = wide[:, 20:170, 32:32 + W]
    view.copy_(qkv)
    odd = torch.zeros(2 * 150 * W + 1, dtype=qkv.dtype, device=DEV)[1:].view(2, 150, W)
    odd.copy_(qkv)
    swapped = qkv.transpose(0, 1).contiguous().transpose(0, 1)
    last = qkv.transpose(1, 2).contiguous().transpose(1, 2)
    for x in (view, odd, swapped, last):
        got = run(x, do, H, KV, 40, 3)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd_do = torch.zeros(do.numel() + 1, dtype=do.dtype, device=DEV)[1:].view_as(do)
    odd_do.copy_(do)
    for d in (odd_do, do.transpose(1, 2).contiguous().transpose(1, 2)):
        got = run(qkv, d, H, KV, 40, 3)
        assert torch.equal(got[1], want[1])


@gpu
def test_rows_further_apart_than_32_bits_reach():
    H = KV = 1
    T, stride = 2400, 1 << 20
    qkv, do = make(1, T, H, KV, 64)
    big = torch.empty(T * stride, dtype=torch.bfloat16, device=DEV)  # 5 GB
    view = big.as_strided((1, T, 3 * 64), (T * stride, stride, 1))
    view.copy_(qkv)
    want, got = run(qkv, do, H, KV, 100, 2), run(view, do, H, KV, 100, 2)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
def test_empty_batch_and_no_gradient():
    for B, T in ((0, 5), (3, 0)):
        x = torch.zeros(B, T, 6 * 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
        o = window_attention_qkvpacked(x, 2, 4)
        assert o.shape == (B, T, 128)
        o.sum().backward()
        assert x.grad.shape == x.shape
    qkv, do = make(2, 130, 2, 2, 64)
    with torch.no_grad():
        quiet = window_attention_qkvpacked(qkv, 2, 33, 3)
    assert torch.equal(quiet, run(qkv, do, 2, 2, 33, 3)[0])


@gpu
def test_composed_on_the_gpu_and_autocast():
    qkv, do = make(2, 90, 2, 1, 32)  # a head size without kernels
    x = qkv.detach().requires_grad_()
    o = window_attention_qkvpacked(x, 2, 20, 2, n_kv_head=1)
    (g,) = torch.autograd.grad(o, x, do)
    ro, eo, rg, eg = reference(qkv, do, 2, 1, 20, 2)
    assert bool(((o.double() - ro).abs() <= eo).all()) and bool(((g.double() - rg).abs() <= eg).all())
    full = torch.randn(1, 70, 6 * 64, device=DEV)
    with torch.autocast("cuda", torch.bfloat16):
        assert torch.equal(window_attention_qkvpacked(full, 2, 9), window_attention_qkvpacked(full.bfloat16(), 2, 9))


@gpu
def test_same_bits_every_time_and_on_other_streams():
    a, b = make(2, 1500, 4, 1, 64, seed=1), make(2, 1500, 4, 1, 64, seed=2)
    want = [run(*a, 4, 1, 90, 5), run(*b, 4, 1, 90, 5)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        with torch.cuda.stream(s1):
            x = run(*a, 4, 1, 90, 5)
        with torch.cuda.stream(s2):
            y = run(*b, 4, 1, 90, 5)
        torch.cuda.synchronize()
        for got, ref in ((x, want[0]), (y, want[1])):
            assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


@gpu
def test_captured_and_replayed():
    qkv, do = make(2, 600, 4, 2, 64)
    lens = torch.tensor([600, 333], dtype=torch.int32, device=DEV)
    x = qkv.clone().requires_grad_()

    def step():
        o = window_attention_qkvpacked(x, 4, 70, 3, n_kv_head=2, seq_lens=lens)
        return o, torch.autograd.grad(o, x, do)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, g = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(qkv * (1 + 0.1 * k))
            lens.copy_(torch.tensor([600 - 10 * k, 333 + k], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        wo, wg = step()
        assert torch.equal(o, wo) and torch.equal(g, wg)


@gpu
def test_gradient_against_differences():
    qkv, do = make(1, 200, 2, 1, 64)
    _, g = run(qkv, do, 2, 1, 50, 3)
    _, _, _, eg = reference(qkv, do, 2, 1, 50, 3)
    way = torch.randn(qkv.shape, device=DEV, dtype=torch.float64)
    h = 1e-5
    at = [float((reference(qkv.double() + s * way, do, 2, 1, 50, 3)[0] * do.double()).sum()) for s in (h, -h)]
    diff = (at[0] - at[1]) / (2 * h)
    # central differences are exact to h^2 times a third derivative of the order of the values (1e-4 here)
    assert abs(diff - float((g.double() * way).sum())) <= float((eg * way.abs()).sum()) + 1e-3


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_scales_beyond_float32_are_refused(device):
    qkv = torch.randn(1, 5, 3 * 64, device=device).bfloat16()
    for scale in (1e-50, 1e-31, 1e31, float("inf")):
        with pytest.raises(ValueError):
            window_attention_qkvpacked(qkv, 1, 3, softmax_scale=scale)


@gpu
def test_a_second_derivative_is_refused():
    qkv = torch.randn(1, 5, 3 * 64, device=DEV).bfloat16().requires_grad_()
    (g,) = torch.autograd.grad(window_attention_qkvpacked(qkv, 1, 3).float().sum(), qkv, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().square().sum().backward()


@gpu
def test_many_short_sequences():
    # one position attends to itself alone; a launch counts its threads in 32 bits, so 2^24 blocks of queries are not the kernels' any more
    qkv = torch.randn(1 << 21, 1, 9 * 64, device=DEV, dtype=torch.bfloat16)[:, :, : 3 * 64]
    o = window_attention_qkvpacked(qkv, 1, 1)
    assert torch.equal(o, qkv[..., 128:])
    from distributed_pytorch_amd import _ext

    assert not _ext.C().window_attention_supported(1 << 24, 1, 1, 1, 64, 192, "bfloat16")
    assert _ext.C().window_attention_supported((1 << 24) - 1, 1, 1, 1, 64, 192, "bfloat16")


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sinks", [1, 150])
def test_padded_batches_whose_key_blocks_are_cut(sinks, D, dtype):
    # a block with sinks meets 13 query tiles of three heads here, more than one piece of the dK / dV work holds: partial sums, with lengths that end the
    # sequence inside, ahead of and at the end of what a piece walks
    T = 777
    lens = torch.tensor([0, 1, 64, 333, T - 1, T], device=DEV, dtype=torch.int32)
    qkv, do = make(6, T, 12, 4, D, dtype, seed=sinks)
    for b, n in enumerate(lens.tolist()):
        qkv[b, n:] = float("nan")
        do[b, n:] = float("nan")
    o, g = check(qkv, do, 12, 4, 128, sinks, lens)
    for b, n in enumerate(lens.tolist()):
        assert torch.equal(o[b, n:], torch.zeros_like(o[b, n:])) and torch.equal(g[b, n:], torch.zeros_like(g[b, n:]))
    again = run(qkv, do, 12, 4, 128, sinks, seq_lens=lens)
    assert torch.equal(o, again[0]) and torch.equal(g, again[1])
