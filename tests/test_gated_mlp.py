"""The gated feed-forward block: outputs and gradients against float64 with bounds derived from the roundings, every kernel path,
views, streams, graphs, refusals."""
import math

import pytest
import torch
import torch.nn.functional as F

from distributed_pytorch_amd.ops import gated_mlp

gpu = pytest.mark.gpu
DEV = "cuda"


def make(M, K, H, N, dtype=torch.bfloat16, bias=True, device=DEV, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(dtype).to(device)  # noqa: E731
    t = dict(x=r(M, K), w_fc=r(2 * H, K, std=1.3 * K ** -0.5), w_proj=r(N, H, std=H ** -0.5))
    if bias:
        t.update(b_fc=r(2 * H, std=0.3), b_proj=r(N, std=0.3))
    return t, r(M, N)


def run(t, dy, act):
    leaf = {k: v.detach().requires_grad_() for k, v in t.items()}
    y = gated_mlp(leaf["x"], leaf["w_fc"], leaf.get("b_fc"), leaf["w_proj"], leaf.get("b_proj"), act=act)
    grads = torch.autograd.grad(y, list(leaf.values()), dy)
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(leaf, grads)}}


def reference(t, dy, act):
    """{name: (float64 value, how far a kernel may be)} for one that stores h, g | u, dg | du and its results in the inputs' type and
    computes everything between in float32."""
    half = torch.finfo(dy.dtype).eps / 2 if dy.dtype != torch.float32 else 2.0 ** -24
    tiny = 2.0 ** -25 if dy.dtype == torch.float16 else 0.0
    d = {k: v.double() for k, v in t.items()}
    x, wf, wp, dy = d["x"], d["w_fc"], d["w_proj"], dy.double()
    M, K, H, N = x.shape[0], x.shape[1], wp.shape[1], wp.shape[0]
    acc = 2.0 ** -24  # one addition in float32; a sum of n products is off by at most n of them times the sum of magnitudes

    def store(v, e):  # rounded to the storage type
        return 1.05 * e + half * v.abs() + tiny

    gu = x @ wf.t() + d.get("b_fc", 0.0)
    e_gu = (K + 1) * acc * (x.abs() @ wf.abs().t() + (d["b_fc"].abs() if "b_fc" in d else 0.0))
    g, u, e_g, e_u = gu[:, :H], gu[:, H:], e_gu[:, :H], e_gu[:, H:]
    g = g.detach().requires_grad_()
    a = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu}[act](g)
    (s,) = torch.autograd.grad(a.sum(), g)
    a, g = a.detach(), g.detach()
    fn = 2e-6  # the exponential, reciprocal and rational forms, relative to max(1, |g|)
    big = g.abs().clamp(min=1)
    h = a * u
    e_h = store(h, u.abs() * (1.13 * e_g + fn * big) + a.abs() * e_u)
    y = h @ wp.t() + d.get("b_proj", 0.0)
    out = {"y": (y, store(y, e_h @ wp.abs().t() + (H + 1) * acc * (h.abs() @ wp.abs().t() + (d["b_proj"].abs() if "b_proj" in d else 0.0))))}
    dh = dy @ wp
    e_dh = N * acc * (dy.abs() @ wp.abs())
    if dy.dtype == torch.float64 and half == 2.0 ** -24:
        e_dh = e_dh + half * dh.abs()                      # float32 products pass through memory
    ge, ue = e_g + half * g.abs() + tiny, e_u + half * u.abs() + tiny   # as stored
    curve = {"silu": 0.5, "gelu": 0.8, "relu": 0.0}[act]
    e_s = curve * ge + fn
    if act == "relu":
        e_s = e_s + (g.abs() <= ge).double()                # the sign itself is in doubt
    dg, du = dh * u * s, dh * a
    e_dg = e_dh * (u * s).abs() + dh.abs() * (ue * (s.abs() + e_s) + u.abs() * e_s)
    e_du = e_dh * a.abs() + dh.abs() * (1.13 * ge + fn * big)
    dgu = torch.cat([dg, du], 1)
    e = store(dgu, torch.cat([e_dg, e_du], 1))
    dx = dgu @ wf
    out["dx"] = dx, store(dx, e @ wf.abs() + 2 * H * acc * (dgu.abs() @ wf.abs()))
    dwf = dgu.t() @ x
    out["dw_fc"] = dwf, store(dwf, e.t() @ x.abs() + M * acc * (dgu.abs().t() @ x.abs()))
    dwp = dy.t() @ h
    out["dw_proj"] = dwp, store(dwp, dy.abs().t() @ e_h + M * acc * (dy.abs().t() @ h.abs()))
    if "b_fc" in d:
        out["db_fc"] = dgu.sum(0), store(dgu.sum(0), e.sum(0) + M * acc * dgu.abs().sum(0))
        out["db_proj"] = dy.sum(0), store(dy.sum(0), M * acc * dy.abs().sum(0))
    return out


def check(t, dy, act):
    got, want = run(t, dy, act), reference(t, dy, act)
    assert set(got) == set(want)
    for k, (v, e) in want.items():
        assert got[k].shape == v.shape and got[k].dtype == dy.dtype, k
        worst = float(((got[k].double() - v).abs() / (e + 1e-12)).max()) if v.numel() else 0.0
        assert worst <= 1.0, (k, worst)
    return got


# ------------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_cpu_matches_the_formula(act):
    t, dy = make(5, 7, 6, 4, torch.float32, device="cpu")
    check(t, dy, act)


def test_cpu_gradient_against_differences():
    t, _ = make(3, 4, 3, 2, torch.float64, device="cpu")
    for v in t.values():
        v.requires_grad_()
    assert torch.autograd.gradcheck(lambda x, wf, wp, bf, bp: gated_mlp(x, wf, bf, wp, bp, act="silu"), tuple(t.values()))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals(device):
    t, _ = make(4, 8, 6, 5, device=device)
    args = (t["x"], t["w_fc"], t["b_fc"], t["w_proj"], t["b_proj"])

    def call(i, v, **kw):
        a = list(args)
        a[i] = v
        return gated_mlp(*a, **kw)

    gated_mlp(*args)
    for i, v in ((0, t["x"][:, :7]), (0, t["x"].float()), (0, t["x"][0, 0]), (1, t["w_fc"][:11]), (1, t["w_fc"][:10]), (1, t["w_fc"][0]), (1, t["w_fc"].float()),
                 (2, t["b_fc"][:11]), (2, t["b_fc"].float()), (3, t["w_proj"][:, :5]), (3, t["w_proj"][:0]), (4, t["b_proj"][:4]), (4, t["b_proj"].half())):
        with pytest.raises(ValueError):
            call(i, v)
    for act in ("tanh", None, 1):
        with pytest.raises(ValueError):
            gated_mlp(*args, act=act)
    if device == "cuda":
        with pytest.raises(ValueError):
            call(1, t["w_fc"].cpu())
        with pytest.raises(RuntimeError):
            gated_mlp(*(a.double() for a in args))


# ------------------------------------------------------------------------------------------------ GPU
SMALL = [(1, 1, 1, 1), (1, 64, 16, 8), (3, 5, 7, 9), (17, 33, 40, 20), (5, 1, 3, 2), (64, 128, 64, 64), (129, 72, 130, 66), (200, 96, 100, 17), (130, 200, 257, 63)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("M,K,H,N", SMALL)
def test_small_and_odd(M, K, H, N, act, dtype):
    check(*make(M, K, H, N, dtype, seed=M), act)


# the kernel of 256 x 256 tiles: one tile a workgroup and several, one to many k-steps, whole and ragged tiles in either dimension
@gpu
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("M,K,H,N", [(2048, 64, 2048, 64), (4096, 128, 2048, 128), (2100, 192, 2056, 192), (4100, 256, 2048, 64), (4096, 320, 2064, 256),
                                     (12288, 192, 2048, 128), (12300, 256, 2056, 64)])
def test_large_tiles(M, K, H, N, act, bias):
    check(*make(M, K, H, N, bias=bias, seed=K), act)


@gpu
@pytest.mark.parametrize("M,K,H,N", [(1, 768, 2048, 768), (7, 768, 2048, 768), (16, 520, 1386, 520), (33, 1024, 2816, 1024), (16, 64, 50, 40), (2, 1000, 1001, 999)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_few_tokens(M, K, H, N, dtype):
    t, dy = make(M, K, H, N, dtype)
    got = check(t, dy, "silu")
    with torch.no_grad():
        quiet = gated_mlp(t["x"], t["w_fc"], t["b_fc"], t["w_proj"], t["b_proj"])
    want, e = reference(t, dy, "silu")["y"]
    assert bool(((quiet.double() - want).abs() <= e).all()) and got["y"].shape == quiet.shape


@gpu
def test_without_gradients_the_same_values():
    for M, K, H, N in ((4096, 128, 2048, 128), (12288, 192, 2048, 128), (100, 72, 130, 66)):
        t, dy = make(M, K, H, N)
        with torch.no_grad():
            quiet = gated_mlp(t["x"], t["w_fc"], t["b_fc"], t["w_proj"], t["b_proj"])
        assert torch.equal(quiet, run(t, dy, "silu")["y"])


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_extreme_gates(act):
    t, dy = make(64, 64, 64, 32, torch.float32)
    t["b_fc"][:64] = torch.linspace(-300, 300, 64, device=DEV)
    got = check(t, dy, act)
    assert all(bool(torch.isfinite(v).all()) for v in got.values())
    t, dy = make(4096, 64, 2048, 64)
    t["b_fc"][:2048] = torch.linspace(-300, 300, 2048, device=DEV).bfloat16()
    got = check(t, dy, act)
    assert all(bool(torch.isfinite(v).all()) for v in got.values())


@gpu
def test_rows_do_not_mix():
    t, dy = make(300, 64, 100, 40)
    want = run(t, dy, "silu")
    t["x"][7] = float("nan")
    got = run(t, dy, "silu")
    keep = torch.arange(300, device=DEV) != 7
    assert torch.equal(got["y"][keep], want["y"][keep]) and torch.equal(got["dx"][keep], want["dx"][keep]) and bool(torch.isnan(got["y"][7]).all())


@gpu
def test_shapes_views_and_missing_gradients():
    t, dy = make(60, 72, 130, 66)
    want = run(t, dy, "silu")
    y = gated_mlp(t["x"].view(3, 4, 5, 72), t["w_fc"], t["b_fc"], t["w_proj"], t["b_proj"])
    assert y.shape == (3, 4, 5, 66) and torch.equal(y.view(60, 66), want["y"])
    assert gated_mlp(t["x"][0], t["w_fc"], t["b_fc"], t["w_proj"], t["b_proj"]).shape == (66,)
    odd = {}
    for k, v in t.items():  # one element off a 16-byte boundary
        flat = torch.zeros(v.numel() + 1, dtype=v.dtype, device=DEV)[1:]
        odd[k] = flat.view(v.shape).copy_(v)
    turned = {k: v.t().contiguous().t() if v.dim() == 2 else v for k, v in t.items()}
    for u in (odd, turned):
        got = run(u, dy.t().contiguous().t(), "silu")
        assert all(torch.equal(got[k], want[k]) for k in want)
    for names in (("x",), ("w_fc",), ("w_proj",), ("b_fc",), ("b_proj",), ("x", "b_fc"), ("w_fc", "w_proj")):
        leaf = {k: v.detach().requires_grad_(k in names) for k, v in t.items()}
        y = gated_mlp(leaf["x"], leaf["w_fc"], leaf["b_fc"], leaf["w_proj"], leaf["b_proj"])
        for n, g in zip(names, torch.autograd.grad(y, [leaf[n] for n in names], dy)):
            assert torch.equal(g, want["d" + n]), n


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_rows(dtype):
    t, dy = make(0, 72, 130, 66, dtype)
    got = run(t, dy, "silu")
    assert got["y"].shape == (0, 66) and got["dx"].shape == (0, 72)
    for k in ("dw_fc", "dw_proj", "db_fc", "db_proj"):
        assert torch.equal(got[k], torch.zeros_like(got[k])), k


@gpu
def test_same_bits_every_time_and_on_other_streams():
    a, b = make(12288, 192, 2048, 128, seed=1), make(12288, 192, 2048, 128, seed=2)
    want = [run(*a, "silu"), run(*b, "silu")]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            x = run(*a, "silu")
        with torch.cuda.stream(s2):
            y = run(*b, "silu")
        torch.cuda.synchronize()
        for got, ref in ((x, want[0]), (y, want[1])):
            assert all(torch.equal(got[k], ref[k]) for k in ref)


@gpu
@pytest.mark.parametrize("M,K,H,N", [(12288, 192, 2048, 128), (100, 72, 130, 66), (1, 768, 2048, 768)])
def test_captured_and_replayed(M, K, H, N):
    t, dy = make(M, K, H, N)
    leaf = {k: v.clone().requires_grad_() for k, v in t.items()}

    def step():
        y = gated_mlp(leaf["x"], leaf["w_fc"], leaf["b_fc"], leaf["w_proj"], leaf["b_proj"])
        return [y, *torch.autograd.grad(y, list(leaf.values()), dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            leaf["x"].copy_(t["x"] * (1 + 0.1 * k))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)


@gpu
def test_gradient_against_differences():
    t, dy = make(40, 48, 64, 24, torch.float32)
    got, want = run(t, dy, "gelu"), reference(t, dy, "gelu")
    for k in ("x", "w_fc", "b_proj"):
        way = torch.randn(t[k].shape, device=DEV, dtype=torch.float64)
        h, at = 1e-6, []
        for s in (h, -h):
            d = {n: v.double() for n, v in t.items()}
            d[k] = d[k] + s * way
            gu = d["x"] @ d["w_fc"].t() + d["b_fc"]
            at.append(float(((F.gelu(gu[:, :64]) * gu[:, 64:]) @ d["w_proj"].t() + d["b_proj"]).mul(dy.double()).sum()))
        diff = (at[0] - at[1]) / (2 * h)
        # the differences carry 1e-16 of a sum of a few thousand over 1e-6
        assert abs(diff - float((got["d" + k].double() * way).sum())) <= float((want["d" + k][1] * way.abs()).sum()) + 1e-4


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_second_derivative_is_refused(dtype):
    x = torch.randn(5, 16, device=DEV, dtype=dtype, requires_grad=True)
    y = gated_mlp(x, torch.randn(24, 16, device=DEV, dtype=dtype), None, torch.randn(8, 12, device=DEV, dtype=dtype), None)
    (g,) = torch.autograd.grad(y.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().square().sum().backward()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,N", [(1, 24), (63, 33), (64, 64), (513, 100), (1003, 2772), (2047, 71), (2048, 40), (2049, 40)])
def test_bias_gradients_of_few_and_many_rows(M, N, dtype):
    from distributed_pytorch_amd import _ext

    g = torch.randn(M, N, device=DEV).to(dtype)
    g[M // 2, N - 1] = float("inf")                      # an infinite sum, not a NaN
    x, w = torch.randn(M, 8, device=DEV).to(dtype), torch.randn(N, 8, device=DEV).to(dtype)
    db = _ext.C().linear_backward(g, x, w, False, True, None, True)[2]
    want = g.double().sum(0)
    # M float32 additions and one rounding to the type
    bound = M * 2.0 ** -24 * g.double().abs().sum(0) + torch.finfo(dtype).eps / 2 * want.abs() + 1e-12
    assert db[N - 1] == float("inf")
    assert bool(((db.double() - want).abs() <= bound)[: N - 1].all())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", [(200, 130, 1400), (129, 33, 1999), (5, 1000, 1283), (1031, 37, 40), (1400, 640, 520), (300, 300, 4096)])
def test_products_whose_contraction_is_spread(M, N, K, dtype):
    from distributed_pytorch_amd import _ext

    C = _ext.C()
    x, w, b = torch.randn(M, K, device=DEV).to(dtype), torch.randn(N, K, device=DEV).to(dtype), torch.randn(N, device=DEV).to(dtype)
    g = torch.randn(M, N, device=DEV).to(dtype)
    y = C.linear_forward(x, w, b, 0, False, True)[0]
    dx, dw, db = C.linear_backward(g, x, w, True, True, None, True)
    X, W, G = x.double(), w.double(), g.double()
    half = torch.finfo(dtype).eps / 2
    for got, want, size, n in ((y, X @ W.t() + b.double(), X.abs() @ W.abs().t() + b.double().abs(), K), (dx, G @ W, G.abs() @ W.abs(), N),
                               (dw, G.t() @ X, G.abs().t() @ X.abs(), M), (db, G.sum(0), G.abs().sum(0), M)):
        # n float32 products and additions, each off by 2^-24 of the sum of sizes at most; then one rounding to the type
        bound = 2 * (n + 2) * 2.0 ** -24 * size + half * want.abs() + 1e-12
        assert bool(((got.double() - want).abs() <= bound).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,K,H,N", [(1003, 520, 1386, 520), (64, 1472, 640, 200), (2300, 256, 256, 128)])
def test_spread_products_captured_and_replayed(M, K, H, N, dtype):
    t, dy = make(M, K, H, N, dtype)
    leaf = {k: v.clone().requires_grad_() for k, v in t.items()}

    def step():
        y = gated_mlp(leaf["x"], leaf["w_fc"], leaf["b_fc"], leaf["w_proj"], leaf["b_proj"])
        with torch.no_grad():
            quiet = gated_mlp(leaf["x"], leaf["w_fc"], leaf["b_fc"], leaf["w_proj"], leaf["b_proj"])
        return [y.detach(), quiet, *torch.autograd.grad(y, list(leaf.values()), dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        graphs.append((torch.cuda.CUDAGraph(), None))
        with torch.cuda.graph(graphs[-1][0]):
            out = step()
        graphs[-1] = (graphs[-1][0], out)
    for k in range(4):
        with torch.no_grad():
            leaf["x"].copy_(t["x"] * (1 + 0.1 * k))
        want = step()
        assert torch.equal(want[0], want[1])
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for got, w in zip(out, want):
                assert torch.equal(got, w)


# one size for each kernel: few rows, 128 x 128 and 256 x 256 tiles, fp32 products with the gate behind them
@gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("M,H,dtype", [(3, 40, torch.bfloat16), (150, 40, torch.float16), (4096, 2304, torch.bfloat16), (70, 40, torch.float32)])
def test_a_gate_that_is_not_a_number_shows(M, H, dtype, act):
    from distributed_pytorch_amd import _ext

    C = _ext.C()
    code = {"silu": C.ACT_SILU, "gelu": C.ACT_GELU, "relu": C.ACT_RELU}[act]
    t, dy = make(M, 64, H, 64, dtype)
    plain_h, plain_gu = C.gated_forward(t["x"], t["w_fc"], t["b_fc"], code, True)
    plain_d = C.gated_backward(dy, t["w_proj"], plain_gu, code, True)
    lost = H // 3
    t["b_fc"][lost] = float("nan")       # the gate's half only: u stays finite
    h, gu = C.gated_forward(t["x"], t["w_fc"], t["b_fc"], code, True)
    quiet, _ = C.gated_forward(t["x"], t["w_fc"], t["b_fc"], code, False)
    d, db = C.gated_backward(dy, t["w_proj"], gu, code, True)
    assert torch.isnan(h[:, lost]).all() and torch.isnan(quiet[:, lost]).all() and torch.isnan(gu[:, lost]).all()
    for got in (d, db):
        assert torch.isnan(got[..., lost]).all() and torch.isnan(got[..., H + lost]).all()
    rest = [i for i in range(2 * H) if i % H != lost]
    for got, want in ((h, plain_h), (quiet, plain_h)):
        assert torch.equal(got[:, rest[: H - 1]], want[:, rest[: H - 1]])
    assert torch.equal(d[:, rest], plain_d[0][:, rest]) and torch.equal(db[rest], plain_d[1][rest])


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_bias_gradients_are_summed_ahead_of_the_rounding(act):
    # Products of a contraction of 64 and g | u as stored are exact to float32 here; what is left is the additions and one rounding.  Summed after
    # the rounding to bf16, 4096 terms of size d would leave 64 d 2^-10, which shows in the columns whose sum nearly cancels.
    from distributed_pytorch_amd import _ext

    C = _ext.C()
    M, H, N = 4096, 2304, 64
    g = torch.Generator().manual_seed(5)
    dy = torch.randn(M, N, generator=g).bfloat16().to(DEV)
    w = (torch.randn(N, H, generator=g) / 8).bfloat16().to(DEV)
    gu = torch.randn(M, 2 * H, generator=g).bfloat16().to(DEV)
    _, db = C.gated_backward(dy, w, gu, {"silu": C.ACT_SILU, "gelu": C.ACT_GELU, "relu": C.ACT_RELU}[act], True)
    gate, u = gu.double().chunk(2, 1)
    gate = gate.requires_grad_()
    a = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu}[act](gate)
    (slope,) = torch.autograd.grad(a.sum(), gate)
    dh = dy.double() @ w.double()
    d = torch.cat([dh * u * slope, dh * a.detach()], 1)
    want = d.sum(0)
    # bf16's own rounding of the sum; of every term the activation's 2e-6 and of the sums 2^-24 an addition, of unlike sign: their root sum of squares, 6 of those
    near = 2.0 ** -8 * want.abs() + 6 * (2e-6 + 64 * 2.0 ** -24) * d.square().sum(0).sqrt() + 6 * 2.0 ** -24 * 64 * d.square().sum(0).sqrt()
    assert bool(((db.double() - want).abs() <= near).all())


# sizes whose products are spread, few rows, 256 x 256 tiles, degenerate extents
@gpu
@pytest.mark.parametrize("M,K,H,N,dtype", [(300, 96, 2048, 96, torch.float16), (464, 104, 1056, 40, torch.float32), (1003, 520, 1386, 520, torch.bfloat16),
                                           (60, 72, 1040, 66, torch.float16), (4096, 256, 2304, 256, torch.bfloat16), (200, 1, 24, 7, torch.float32),
                                           (200, 1, 24, 16, torch.bfloat16), (33, 5, 8, 1, torch.float16)])
def test_frozen_tensors_leave_the_other_gradients_as_they_are(M, K, H, N, dtype):
    t, dy = make(M, K, H, N, dtype)
    want = run(t, dy, "silu")
    every = list(t)
    for frozen in (["w_fc"], ["w_proj"], ["w_fc", "w_proj"], ["x"], ["x", "w_fc"], ["b_fc"], ["b_proj"], ["x", "w_fc", "w_proj"], ["b_fc", "b_proj", "w_fc"]):
        names = [n for n in every if n not in frozen]
        leaf = {k: v.detach().requires_grad_(k in names) for k, v in t.items()}
        y = gated_mlp(leaf["x"], leaf["w_fc"], leaf["b_fc"], leaf["w_proj"], leaf["b_proj"])
        for n, g in zip(names, torch.autograd.grad(y, [leaf[n] for n in names], dy)):
            assert torch.equal(g, want["d" + n]), (n, frozen)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K,H,N", [(50, 72, 130, 67), (300, 64, 256, 129), (2100, 40, 96, 33), (150, 1, 24, 7)])
def test_an_upstream_gradient_that_starts_anywhere(M, K, H, N, dtype):
    t, dy = make(M, K, H, N, dtype)
    want = run(t, dy, "silu")
    off = torch.cat([dy.new_zeros(1), dy.reshape(-1)])[1:].view(M, N)
    got = run(t, off, "silu")
    assert off.is_contiguous() and off.data_ptr() % 16 and set(got) == set(want)
    for k in want:  # (other loads, the same sums)
        assert torch.equal(got[k], want[k]), k
