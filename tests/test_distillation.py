"""Distillation from a teacher's top logits: loss, by-products and gradients against float64, refusals, streams, graphs."""
import math

import pytest
import torch
import torch.nn.functional as F
from torch.utils._python_dispatch import TorchDispatchMode

from distributed_pytorch_amd.ops import TopKDistillation, projection_topk_distillation, topk_distillation

gpu = pytest.mark.gpu
DEV = "cuda"
NEG = float("-inf")


def make(N, C, K, dtype=torch.float32, device="cpu", width=None, seed=0, pad_rows=True):
    """Logits [N, width], K distinct entries a row in no order, targets with some rows ignored."""
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(N, width or C, generator=g) * 3 - 20).to(dtype)  # an offset, as real vocabularies have
    ids = torch.stack([torch.randperm(C, generator=g)[:K] for _ in range(N)])
    teacher = torch.randn(N, K, generator=g) * 2
    targets = torch.randint(0, C, (N,), generator=g)
    if pad_rows and N > 2:
        targets[1] = -100
        ids[2, K // 2:] = -1
    return logits.to(device), ids.to(device), teacher.to(device), targets.to(device)


def reference(logits, ids, teacher, targets, tau=1.0, a=0.0, C=None, ignore_index=-100):
    """Row losses and mean-loss gradient in float64, entry by entry from the definition."""
    C = C or logits.shape[1]
    N = logits.shape[0]
    z = logits.detach().double().cpu()
    out, grad = torch.zeros(N, dtype=torch.float64), torch.zeros_like(z)
    live = [targets is None or 0 <= int(targets[r]) < C for r in range(N)]
    n = max(1, N if targets is None else int((targets != ignore_index).sum()))
    for r in range(N):
        if not live[r]:
            grad[r] = 0
            continue
        x = z[r, :C]
        q, q1 = torch.softmax(x / tau, 0), torch.softmax(x, 0)
        there = [(int(i), float(t)) for i, t in zip(ids[r].cpu(), teacher[r].double().cpu()) if 0 <= int(i) < C and float(t) != NEG]
        if there and a < 1:
            p = torch.softmax(torch.tensor([t for _, t in there], dtype=torch.float64) / tau, 0)
            log_q = torch.log_softmax(x / tau, 0)
            out[r] += (1 - a) * tau ** 2 * sum(float(pk * (pk.log() - log_q[i])) for (i, _), pk in zip(there, p) if pk > 0)
            grad[r, :C] += (1 - a) * tau * q
            for (i, _), pk in zip(there, p):
                grad[r, i] -= (1 - a) * tau * pk
        if a > 0:
            y = int(targets[r])
            out[r] -= a * float(torch.log_softmax(x, 0)[y])
            grad[r, :C] += a * q1
            grad[r, y] -= a
    return out, grad, n


def check(logits, ids, teacher, targets, tau, a, C=None, seed_grad=None):
    C = C or logits.shape[1]
    x = logits.detach().clone().requires_grad_()
    r = topk_distillation(x, ids, teacher, targets, tau, a, n_classes=C)
    rows, grad, n = reference(logits, ids, teacher, targets, tau, a, C)
    # float32 arithmetic: an exponent off by 2^-23 of its size (below 64 here), sums of positive terms, a few roundings
    near = 64 * 2.0 ** -23
    size = max(1.0, tau ** 2) * (1 + float(rows.abs().max()) / max(1.0, tau ** 2))
    assert abs(float(r.loss.detach()) - float(rows.sum() / n)) <= near * size
    up = 1.0
    if seed_grad is not None:
        up = seed_grad
    (r.loss * up).backward()
    half = torch.finfo(logits.dtype).eps / 2
    atol = near * max(tau, 1.0) * up / n + (2.0 ** -25 if logits.dtype == torch.float16 else 0.0)
    rtol = half * (1.01 if up == 1.0 else 2.02)  # another upstream gradient: rounded once more
    torch.testing.assert_close(x.grad.double().cpu(), grad * up / n, rtol=rtol, atol=atol)
    assert torch.equal(x.grad[:, C:], torch.zeros_like(x.grad[:, C:]))
    m = r.metrics.cpu()
    live = torch.ones(len(rows), dtype=torch.bool) if targets is None else (targets.cpu() != -100)
    best = logits[:, :C].float().argmax(1).cpu()
    # equal maxima: the lowest index
    best = torch.tensor([int((logits[i, :C] == logits[i, b]).nonzero()[0]) if live[i] else -1 for i, b in enumerate(best.tolist())])
    if targets is not None:
        assert torch.equal(r.correct.cpu(), (best == targets.cpu()) & live)
    assert m[1] == r.correct.sum().cpu() and m[2] == live.sum()
    return x.grad


# ------------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize("tau,a", [(1.0, 0.0), (2.0, 0.5), (0.5, 1.0), (4.0, 0.1)])
def test_composed_matches_the_definition(tau, a):
    logits, ids, teacher, targets = make(6, 40, 7)
    check(logits, ids, teacher, targets, tau, a, C=37)


def test_composed_gradient_against_differences():
    logits, ids, teacher, targets = make(5, 23, 6, dtype=torch.float64)
    f = lambda z: topk_distillation(z, ids, teacher.double(), targets, 3.0, 0.3, n_classes=20).loss  # noqa: E731
    ids.clamp_(max=19)
    targets.clamp_(max=19)
    assert torch.autograd.gradcheck(f, logits.requires_grad_())


def test_rows_that_count_for_nothing():
    logits, ids, teacher, targets = make(4, 11, 3)
    logits[1] = float("nan")          # ignored row
    ids[2] = -1                       # no entries: the soft term is 0
    teacher[3] = NEG
    x = logits.requires_grad_()
    r = topk_distillation(x, ids, teacher, targets, 2.0, 0.0, reduction="none")
    assert r.loss.tolist()[1:] == [0.0, 0.0, 0.0] and r.loss[0] > 0
    r.loss.sum().backward()
    assert torch.equal(x.grad[1:], torch.zeros(3, 11)) and bool(x.grad[0].abs().sum() > 0)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals(device):
    logits, ids, teacher, targets = make(4, 11, 3, device=device)
    bad = [
        (dict(temperature=0.0), ValueError), (dict(temperature=-1.0), ValueError), (dict(temperature=float("nan")), ValueError),
        (dict(temperature=float("inf")), ValueError), (dict(hard_weight=1.5, targets=targets), ValueError), (dict(hard_weight=0.5), ValueError),
        (dict(reduction="avg"), ValueError), (dict(n_classes=12), ValueError), (dict(n_classes=0), ValueError),
        (dict(targets=targets[:3]), ValueError), (dict(targets=targets.int()), ValueError),
        (dict(targets=targets.clamp(min=0) + 11, check_targets=True), IndexError),
    ]
    for kw, err in bad:
        with pytest.raises(err):
            topk_distillation(logits, ids, teacher, **kw)
    with pytest.raises(ValueError):
        topk_distillation(logits, ids[:3], teacher[:3])
    with pytest.raises(ValueError):
        topk_distillation(logits, ids, teacher[:, :2])
    with pytest.raises(ValueError):
        topk_distillation(logits, ids[:, :0], teacher[:, :0])
    with pytest.raises(ValueError):
        topk_distillation(logits, ids.float(), teacher)
    with pytest.raises(ValueError):
        topk_distillation(logits, ids, teacher.long())
    with pytest.raises(ValueError):
        topk_distillation(logits.reshape(2, 2, 11), ids, teacher)
    with pytest.raises(IndexError):
        topk_distillation(logits, ids + 11, teacher, check_targets=True)
    w = torch.randn(11, 8, device=device)
    with pytest.raises(ValueError):
        projection_topk_distillation(torch.randn(4, 8, device=device), w, ids, teacher, reduction="none")


def test_module_and_projection_on_the_cpu():
    logits, ids, teacher, targets = make(6, 30, 4)
    crit = TopKDistillation(2.0, 0.25)
    loss = crit(logits.view(2, 3, 30), ids.view(2, 3, 4), teacher.view(2, 3, 4), targets.view(2, 3))
    rows, _, n = reference(logits, ids, teacher, targets, 2.0, 0.25)
    assert abs(float(loss) - float(rows.sum() / n)) < 1e-4 and crit.last_metrics[2] == n and crit.last_correct.shape == (6,)
    w = torch.randn(30, 5, requires_grad=True)
    x = torch.randn(2, 3, 5, requires_grad=True)
    r = projection_topk_distillation(x, w, ids.view(2, 3, 4), teacher.view(2, 3, 4), targets.view(2, 3), 2.0, 0.25)
    s = topk_distillation(F.linear(x, w).view(6, 30), ids, teacher, targets, 2.0, 0.25)
    assert torch.equal(r.loss, s.loss)


# ------------------------------------------------------------------------------------------------ GPU
# widths on both sides of every kernel's limit, odd ones (rows that start anywhere), one class
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("C,K", [(1, 1), (7, 3), (64, 5), (1000, 64), (1003, 64), (2041, 9), (2049, 100), (4099, 33), (7170, 64), (14343, 65),
                                 (50257, 64), (57345, 7), (65543, 128), (131083, 1024)])
def test_against_float64(C, K, dtype):
    logits, ids, teacher, targets = make(5, C, K, dtype, DEV, seed=C)
    check(logits, ids, teacher, targets, 2.0, 0.25)
    check(logits, ids, teacher, None, 1.0, 0.0)


@gpu
@pytest.mark.parametrize("tau,a", [(1.0, 0.0), (1.0, 0.5), (1.0, 1.0), (3.0, 0.0), (3.0, 1.0), (0.25, 0.5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weights_and_temperatures(tau, a, dtype):
    logits, ids, teacher, targets = make(7, 5000, 17, dtype, DEV)
    check(logits, ids, teacher, targets, tau, a)
    check(logits, ids, teacher, targets, tau, a, seed_grad=0.375)


@gpu
@pytest.mark.parametrize("C,width", [(50257, 50304), (1000, 1024), (1001, 1021)])
def test_padding_columns_may_hold_anything(C, width):
    logits, ids, teacher, targets = make(6, C, 12, torch.bfloat16, DEV, width=width)
    logits[0, C:] = float("nan")
    logits[3, C:] = float("inf")
    logits[4, C:] = 100.0
    check(logits, ids, teacher, targets, 2.0, 0.5, C=C)


@gpu
def test_rows_without_entries_and_ignored_rows():
    logits, ids, teacher, targets = make(8, 999, 10, torch.float32, DEV)
    logits[1] = float("nan")           # targets[1] is ignore_index
    ids[0] = -1
    teacher[3] = NEG
    ids[4, ::2] = 999                  # beyond the classes: absent
    teacher[4, ::2] = float("nan")     # the value of an absent entry does not matter
    teacher[5, 1:] = NEG
    targets[6] = 5000                  # out of range: like an ignored row, but counted
    check(logits, ids, teacher, targets, 2.0, 0.5)
    check(logits, ids, teacher, targets, 2.0, 0.0)
    targets.fill_(-100)                # nothing counts: loss 0, no gradient
    logits.fill_(float("nan"))
    x = logits.requires_grad_()
    r = topk_distillation(x, ids, teacher, targets, 2.0, 0.5)
    r.loss.backward()
    assert float(r.loss) == 0.0 and torch.equal(x.grad, torch.zeros_like(x.grad)) and r.metrics.tolist() == [0, 0, 0, 0]


@gpu
def test_non_finite_values_stay_in_their_row():
    logits, ids, teacher, targets = make(4, 700, 5, torch.float32, DEV, pad_rows=False)
    logits[1, 3] = float("nan")
    teacher[2, 0] = float("nan")
    logits[3, 5:300] = NEG             # masked classes of a row that is fine otherwise
    ids[3] = torch.tensor([0, 1, 2, 300, 301], device=DEV)
    targets[3] = 400
    x = logits.clone().requires_grad_()
    r = topk_distillation(x, ids, teacher, targets, 2.0, 0.5, reduction="none")
    r.loss[[0, 3]].sum().backward()
    rows, grad, _ = reference(logits[[0, 3]], ids[[0, 3]], teacher[[0, 3]], targets[[0, 3]], 2.0, 0.5)
    assert torch.isnan(r.loss[1]) and torch.isnan(r.loss[2])
    torch.testing.assert_close(r.loss[[0, 3]].double().cpu(), rows, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(x.grad[[0, 3]].double().cpu(), grad, rtol=1e-6, atol=2e-5)


@gpu
@pytest.mark.parametrize("C", [9, 3000, 60001])
def test_entries_of_one_class_add_up(C):
    logits, ids, teacher, targets = make(4, C, 9, torch.float32, DEV, pad_rows=False)
    ids[0] = 8 if C > 9 else 3                     # all of them
    ids[1, ::2] = ids[1, 0].item()
    ids[2] = torch.tensor([0, 1, 2, 3, 0, 1, 2, 3, 4], device=DEV)  # neighbours in one vector
    a = check(logits, ids, teacher, targets, 2.0, 0.5)
    for _ in range(3):
        assert torch.equal(a, check(logits, ids, teacher, targets, 2.0, 0.5))
    many = torch.randint(0, min(C, 40), (4, 1024), device=DEV)
    t = torch.randn(4, 1024, device=DEV)
    b = check(logits, many, t, targets, 1.5, 0.0)
    assert torch.equal(b, check(logits, many, t, targets, 1.5, 0.0))


@gpu
def test_equal_maxima_count_for_the_lowest_class():
    logits = torch.zeros(3, 5001, device=DEV, dtype=torch.bfloat16)
    logits[1, 17] = logits[1, 4000] = 3.0
    ids = torch.tensor([[0, 1], [4000, 17], [7, 0]], device=DEV)
    teacher = torch.zeros(3, 2, device=DEV)
    targets = torch.tensor([0, 17, 1], device=DEV)
    assert topk_distillation(logits, ids, teacher, targets).correct.tolist() == [True, True, False]
    assert topk_distillation(logits, ids, teacher).correct.tolist() == [True, False, False]


@gpu
@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("t_dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
def test_types_and_strides_of_the_teacher(ids_dtype, t_dtype):
    logits, ids, teacher, targets = make(6, 3001, 20, torch.bfloat16, DEV)
    ids = ids.to(ids_dtype).t().contiguous().t()
    check(logits, ids, teacher.to(t_dtype).t().contiguous().t(), targets, 2.0, 0.5)


@gpu
def test_logits_of_any_stride_and_offset():
    base, ids, teacher, targets = make(6, 3001, 20, torch.bfloat16, DEV)
    flat = torch.empty(6 * 3001 + 3, dtype=base.dtype, device=DEV)
    flat[3:] = base.reshape(-1)
    want = check(base, ids, teacher, targets, 2.0, 0.5)
    for view in (flat[3:].view(6, 3001), base.t().contiguous().t(), torch.cat([base, base], 1)[:, :3001]):
        x = view.detach().requires_grad_()
        topk_distillation(x, ids, teacher, targets, 2.0, 0.5).loss.backward()
        assert torch.equal(x.grad, want)


@gpu
def test_reductions_and_a_second_backward():
    logits, ids, teacher, targets = make(9, 5003, 20, torch.float32, DEV)
    rows, grad, n = reference(logits, ids, teacher, targets, 2.0, 0.5)
    x = logits.clone().requires_grad_()
    up = torch.rand(9, device=DEV) + 0.5
    r = topk_distillation(x, ids, teacher, targets, 2.0, 0.5, reduction="none")
    torch.testing.assert_close(r.loss.double().cpu(), rows, rtol=1e-5, atol=1e-5)
    (g,) = torch.autograd.grad(r.loss, x, up)
    torch.testing.assert_close(g.double().cpu(), grad * up.double().cpu().unsqueeze(1), rtol=1e-6, atol=2e-5)
    for reduction, k in (("sum", 1), ("mean", n)):
        r = topk_distillation(x, ids, teacher, targets, 2.0, 0.5, reduction=reduction)
        first = torch.autograd.grad(r.loss * 3, x, retain_graph=True)[0]
        second = torch.autograd.grad(r.loss, x, retain_graph=True)[0]
        third = torch.autograd.grad(r.loss, x)[0]
        torch.testing.assert_close(first.double().cpu(), grad * 3 / k, rtol=1e-6, atol=5e-5 / k)
        torch.testing.assert_close(second.double().cpu(), grad / k, rtol=1e-6, atol=2e-5 / k)
        assert torch.equal(second, third)
    with torch.no_grad():
        quiet = topk_distillation(logits, ids, teacher, targets, 2.0, 0.5)
    assert torch.equal(quiet.loss, r.loss.detach())


@gpu
def test_empty_batch_and_one_row():
    for N in (0, 1):
        x = torch.randn(N, 70, device=DEV, requires_grad=True)
        r = topk_distillation(x, torch.zeros(N, 2, dtype=torch.long, device=DEV), torch.zeros(N, 2, device=DEV))
        r.loss.backward()
        assert x.grad.shape == (N, 70) and torch.isfinite(r.loss)


@gpu
@pytest.mark.parametrize("N,C,width,K_in", [(64, 1000, 1024, 96), (257, 5003, 5008, 64), (3, 131, 136, 40), (40, 70, 72, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_projection_against_float64(N, C, width, K_in, dtype):
    _, ids, teacher, targets = make(N, C, 11, dtype, DEV)
    x = torch.randn(N, K_in, device=DEV).to(dtype)
    w = (torch.randn(width, K_in, device=DEV) / math.sqrt(K_in)).to(dtype)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    r = projection_topk_distillation(xs, ws, ids, teacher, targets, 2.0, 0.5, n_classes=C)
    (r.loss * 0.5).backward()
    half = torch.finfo(dtype).eps / 2
    logits = (x.double() @ w.double().t())
    rows, grad, n = reference(logits, ids, teacher, targets, 2.0, 0.5, C)
    grad = grad.to(DEV) * 0.5 / n
    # logits off by half a step of their own size move a row's loss by at most tau (1 - a) + a times twice that
    zmax = float(logits.abs().max())
    slack = half * zmax * 2 * 1.5 + 1e-4 * (1 if dtype == torch.float32 else 0) + 1e-5
    assert abs(float(r.loss.detach()) - float(rows.sum() / n)) <= slack
    # dlogits: the probabilities move by a factor exp(2 half zmax), and the result is rounded; then one product and two roundings
    factor = math.expm1(2 * half * zmax) + 3 * half + 2e-5
    z = logits[:, :C]
    q = grad.abs() + 0.5 / n * F.pad(torch.softmax(z / 2, 1) + 0.5 * torch.softmax(z, 1), (0, width - C))  # every positive part of dlogits
    for got, want, bound in ((xs.grad, grad @ w.double(), q @ w.double().abs()), (ws.grad, grad.t() @ x.double(), q.t() @ x.double().abs())):
        err = (got.double() - want).abs()
        assert bool((err <= factor * bound + half * want.abs() + 1e-9).all())
    assert torch.equal(ws.grad[C:], torch.zeros_like(ws.grad[C:]))


@gpu
def test_gradient_against_differences():
    logits, ids, teacher, targets = make(3, 900, 8, torch.float32, DEV, pad_rows=False)
    x = logits.clone().requires_grad_()
    topk_distillation(x, ids, teacher, targets, 3.0, 0.3).loss.backward()
    # central differences of the float64 loss: exact to h^2
    h = 1e-4
    for r, j in ((0, int(ids[0, 0])), (1, int(targets[1])), (2, int(ids[2, 5])), (0, 3)):
        at = []
        for s in (h, -h):
            z = logits.double()
            z[r, j] += s
            rows, _, n = reference(z, ids, teacher, targets, 3.0, 0.3)
            at.append(float(rows.sum() / n))
        assert abs((at[0] - at[1]) / (2 * h) - float(x.grad[r, j])) < 2e-6


@gpu
def test_other_stream_and_two_calls_at_once():
    a = make(64, 20011, 30, torch.bfloat16, DEV, seed=1)
    b = make(64, 20011, 30, torch.bfloat16, DEV, seed=2)

    def grad(t):
        x = t[0].detach().requires_grad_()
        (g,) = torch.autograd.grad(topk_distillation(x, t[1], t[2], t[3], 2.0, 0.5).loss, x)
        return g

    want = [grad(a), grad(b)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            ga = grad(a)
        with torch.cuda.stream(s2):
            gb = grad(b)
        torch.cuda.synchronize()
        assert torch.equal(ga, want[0]) and torch.equal(gb, want[1])


@gpu
def test_captured_and_replayed():
    logits, ids, teacher, targets = make(32, 5003, 30, torch.bfloat16, DEV)
    x = logits.clone().requires_grad_()

    def step():
        r = topk_distillation(x, ids, teacher, targets, 2.0, 0.5)
        (g,) = torch.autograd.grad(r.loss, x)
        return r.loss, g

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, g = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(logits * (1 + 0.1 * k))
        graph.replay()
        torch.cuda.synchronize()
        want_loss, want_g = step()
        assert torch.equal(loss, want_loss) and torch.equal(g, want_g)


@gpu
def test_widest_rows_and_wider_ones():
    C = 1 << 20
    logits, ids, teacher, targets = make(2, C, 5, torch.float32, DEV)
    check(logits, ids, teacher, targets, 2.0, 0.5)
    with pytest.raises(RuntimeError, match="width"):
        topk_distillation(torch.zeros(1, C + 8, device=DEV), ids[:1], teacher[:1])


@gpu
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_more_rows_than_one_launch_takes(reduction):
    N, C, K = (1 << 21) + 5, 8, 2
    g = torch.Generator(device=DEV).manual_seed(3)
    logits = torch.randn(N, C, generator=g, device=DEV) * 3
    ids = torch.randint(0, C, (N, K), generator=g, device=DEV)
    teacher = torch.randn(N, K, generator=g, device=DEV)
    targets = torch.randint(0, C, (N,), generator=g, device=DEV)
    x, z = logits.clone().requires_grad_(), logits.double().requires_grad_()
    got = topk_distillation(x, ids, teacher, targets, 2.0, 0.5, reduction=reduction)
    want = topk_distillation(z.cpu(), ids.cpu(), teacher.double().cpu(), targets.cpu(), 2.0, 0.5, reduction=reduction)
    got.loss.sum().backward()
    want.loss.sum().backward()
    # exponents below 64 in float32, a few roundings; a sum of N positive rows in blocks: below 2^12 roundings on the way
    near = 64 * 2.0 ** -23 * 4
    torch.testing.assert_close(got.loss.detach().double().cpu(), want.loss.detach(), rtol=2.0 ** -12 if reduction == "sum" else 2.0 ** -20, atol=near)
    torch.testing.assert_close(x.grad.double(), z.grad, rtol=2.0 ** -22, atol=near)
    assert torch.equal(got.correct.cpu(), want.correct)


@gpu
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_half_precision_gradients_survive_the_division_by_the_rows(reduction):
    # a loss scale has to come in ahead of the rounding: 1 / (1500 * 600) is about the smallest fp16 step
    N, C, up = 1500, 600, 2.0 ** (16 if reduction == "mean" else 4)
    logits, ids, teacher, targets = make(N, C, 9, torch.float16, DEV)
    x = (logits + 20).requires_grad_()
    rows, grad, n = reference(x, ids, teacher, targets, 2.0, 0.5)
    grad = grad * up / (n if reduction == "mean" else 1)
    r = topk_distillation(x, ids, teacher, targets, 2.0, 0.5, reduction=reduction)
    (r.loss * up).backward()
    half = 2.0 ** -11
    # one rounding; a subnormal's is half of 2^-24; float32 arithmetic as in check()
    near = 64 * 2.0 ** -23 * 2 * up / (n if reduction == "mean" else 1)
    torch.testing.assert_close(x.grad.double().cpu(), grad, rtol=half * 1.01, atol=near + 2.0 ** -25)


@gpu
def test_half_precision_projection_under_a_loss_scale():
    N, C, width, K_in, up = 1500, 600, 608, 64, 2.0 ** 16
    _, ids, teacher, targets = make(N, C, 9, torch.float16, DEV)
    x = torch.randn(N, K_in, device=DEV).half()
    w = (torch.randn(width, K_in, device=DEV) / math.sqrt(K_in)).half()
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    r = projection_topk_distillation(xs, ws, ids, teacher, targets, 2.0, 0.5, n_classes=C)
    first = torch.autograd.grad(r.loss * up, (xs, ws), retain_graph=True)
    (r.loss * up).backward()
    assert torch.equal(first[0], xs.grad) and torch.equal(first[1], ws.grad)
    half, tiny = 2.0 ** -11, 2.0 ** -25
    logits = x.double() @ w.double().t()
    _, grad, n = reference(logits, ids, teacher, targets, 2.0, 0.5, C)
    grad = grad.to(DEV) * up / n
    zmax = float(logits.abs().max())
    # as test_projection_against_float64, and every element of dlogits off by half of the smallest step besides
    factor = math.expm1(2 * half * zmax) + 3 * half + 2e-5
    z = logits[:, :C]
    q = grad.abs() + up / n * F.pad(torch.softmax(z / 2, 1) + 0.5 * torch.softmax(z, 1), (0, width - C))
    on = torch.ones_like(grad)
    for got, want, bound, steps in ((xs.grad, grad @ w.double(), q @ w.double().abs(), on @ w.double().abs()),
                                    (ws.grad, grad.t() @ x.double(), q.t() @ x.double().abs(), on.t() @ x.double().abs())):
        err = (got.double() - want).abs()
        assert bool((err <= factor * bound + half * want.abs() + tiny * (steps + 1)).all())
        assert float(err.norm() / want.norm()) < 0.01


@gpu
def test_one_upstream_value_for_many_rows():
    from distributed_pytorch_amd import _ext

    logits, ids, teacher, targets = make(7, 100, 5, torch.float32, DEV)
    cfg = (100, -100, 2.0, 0.5)
    out = _ext.C().distill_forward(logits, ids, teacher, targets, *cfg, True, "none")
    args = (logits, ids, teacher, targets, out[5], out[4])
    one = _ext.C().distill_backward(*args, torch.full((), 3.0, device=DEV), *cfg)
    assert torch.equal(one, _ext.C().distill_backward(*args, torch.full((1,), 3.0, device=DEV), *cfg))
    assert torch.equal(one, _ext.C().distill_backward(*args, torch.full((7,), 3.0, device=DEV), *cfg))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_a_second_derivative_is_refused(dtype):
    logits, ids, teacher, targets = make(4, 11, 3, dtype, DEV)
    x, w = logits.requires_grad_(), torch.randn(16, 11, device=DEV).to(dtype)
    for r in (topk_distillation(x, ids, teacher, targets, 2.0, 0.5), projection_topk_distillation(x, w, ids, teacher, targets, 2.0, 0.5)):
        (g,) = torch.autograd.grad(r.loss, x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.float().square().sum().backward()


@gpu
@pytest.mark.parametrize("N", [1, 2, 63, 64, 65, 512, 513])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rows_are_counted_alike_by_few_and_many(N, dtype):
    logits, ids, teacher, targets = make(N, 40, 6, dtype, DEV)
    logits = logits + 20
    targets[N // 2:] = -100 if N > 2 else targets[N // 2:]
    near = 64 * 2.0 ** -23 * 2
    for reduction in ("mean", "sum"):
        x = logits.clone().requires_grad_()
        r = topk_distillation(x, ids, teacher, targets, 2.0, 0.5, reduction=reduction)
        rows, grad, n = reference(logits, ids, teacher, targets, 2.0, 0.5)
        n = n if reduction == "mean" else 1
        (g,) = torch.autograd.grad(r.loss, x, retain_graph=True)
        (again,) = torch.autograd.grad(r.loss, x)
        assert torch.equal(g, again)
        torch.testing.assert_close(g.double().cpu(), grad / n, rtol=torch.finfo(dtype).eps / 2 * 1.01, atol=near / n + (2.0 ** -25 if dtype == torch.float16 else 0))
    x = logits.clone().requires_grad_()
    r = topk_distillation(x, ids, teacher, None, 2.0, 0.0)
    rows, grad, n = reference(logits, ids, teacher, None, 2.0, 0.0)
    assert n == N
    (g,) = torch.autograd.grad(r.loss, x)
    torch.testing.assert_close(g.double().cpu(), grad / n, rtol=torch.finfo(dtype).eps / 2 * 1.01, atol=near / n + (2.0 ** -25 if dtype == torch.float16 else 0))


def projected(N, V, K_in, dtype, seed=0, K=11, C=None):
    """Inputs of a vocabulary projection near its initialisation."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, K_in, generator=g).to(dtype).to(DEV)
    w = (torch.randn(V, K_in, generator=g) * 0.02).to(dtype).to(DEV)
    _, ids, teacher, targets = make(N, C or V, K, dtype, DEV, seed=seed, pad_rows=False)
    return x, w, ids, teacher, targets


# The loss is float32, so logits rounded to 16 bits (half a step of theirs is 2^-9 or 2^-12) are not good enough for it.  What float32 leaves, with
# logits below 4 in size and sums of 768 products below 8: of a logit 96 roundings at most (a matrix instruction adds 8 products or more at once), half a step of
# 2^-24 each, mostly of unlike sign, and some 30 more in exponents, sums of positive terms and logarithms: 2^-17 of a loss near 7 covers them, at any number of rows.
@gpu
@pytest.mark.parametrize("N", [1, 2, 4, 16, 64, 700])
@pytest.mark.parametrize("V,K_in", [(1000, 768), (1003, 768), (5000, 250)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_projected_loss_is_as_exact_as_its_type(N, V, K_in, dtype):
    for seed in range(3):
        x, w, ids, teacher, targets = projected(N, V, K_in, dtype, seed)
        z = x.double() @ w.double().t()
        for tau, a in ((2.0, 0.5), (1.0, 0.0), (1.0, 1.0)):
            rows, _, n = reference(z, ids, teacher, targets, tau, a)
            for reduction, k in (("mean", n), ("sum", 1)):
                r = projection_topk_distillation(x, w, ids, teacher, targets, tau, a, reduction)
                assert abs(float(r.loss) - float(rows.sum()) / k) <= 2.0 ** -17 * max(1.0, tau ** 2) * n / k
                assert abs(float(r.metrics[3]) - float(rows.sum()) / n) <= 2.0 ** -17 * max(1.0, tau ** 2)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_projected_predictions_are_those_of_the_unrounded_logits(dtype):
    x, w, ids, teacher, _ = projected(2048, 1000, 256, dtype)
    z = x.double() @ w.double().t()
    top = z.topk(2, 1)
    clear = top.values[:, 0] - top.values[:, 1] > 1e-4
    r = projection_topk_distillation(x, w, ids, teacher, top.indices[:, 0].contiguous(), 2.0, 0.5)
    assert clear.float().mean() > 0.95 and bool(r.correct[clear].all())


# both kernels of the float32 product: 128 x 128 tiles, 256 x 256 tiles one to a workgroup and several to a workgroup, with ragged edges
@gpu
@pytest.mark.parametrize("N,V,K_in", [(1, 17, 8), (130, 1003, 77), (2049, 4103, 64), (2048, 4096, 128), (4100, 12301, 192), (4096, 12544, 256)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_projected_logits_and_parts_of_the_rows(N, V, K_in, dtype):
    from distributed_pytorch_amd import _ext

    x, w, ids, teacher, targets = projected(N, V, K_in, dtype, K=5)
    targets[::7] = -100
    args = (x, w, ids, teacher, targets, V, -100, 2.0, 0.5, True)
    loss, correct, metrics, scale, stats, logits, _ = _ext.C().projection_distill_forward(*args, "logits")
    assert logits.dtype == torch.float32 and logits.shape == (N, (V + 3) // 4 * 4)
    z = x.float() @ w.float().t()  # (float64 does not fit the largest comfortably; the bound takes both sides' roundings)
    bound = 2 * K_in * 2.0 ** -24 * (x.float().abs() @ w.float().abs().t()) + 1e-30
    assert bool(((logits[:, :V] - z).abs() <= bound).all())
    quiet = _ext.C().projection_distill_forward(*args, "none", workspace_bytes=1)  # 256 rows at a time
    assert torch.equal(quiet[1], correct) and abs(float(quiet[0] - loss)) <= 2.0 ** -17
    if dtype == torch.bfloat16:
        d1 = _ext.C().projection_distill_forward(*args, "gradient")[6]
        # the same arithmetic as the gradient of the float32 logits on their own, but rounded to bf16
        whole = logits[:, :V].contiguous()
        d2 = _ext.C().distill_forward(whole, ids, teacher, targets, V, -100, 2.0, 0.5, True, "new")[6]
        if V % 4 == 0:
            assert torch.equal(d1, d2.bfloat16())
        else:  # rows that start elsewhere add up their exponentials in another order
            torch.testing.assert_close(d1.float(), d2, rtol=2.0 ** -8 * 1.01, atol=4e-6 / N)
        part = _ext.C().projection_distill_forward(*args, "gradient", workspace_bytes=1)
        # (256 rows may run on the other kernel, whose products add up in another order)
        torch.testing.assert_close(part[6].float(), d1.float(), rtol=2.0 ** -7, atol=2.0 ** -15 / N)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,V,K_in", [(65, 1003, 96), (2100, 4100, 64), (4096, 12301, 192)])
def test_projected_pass_captured_and_replayed(N, V, K_in, dtype):
    x, w, ids, teacher, targets = projected(N, V, K_in, dtype, K=5)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()

    def step():
        r = projection_topk_distillation(xs, ws, ids, teacher, targets, 2.0, 0.5)
        return (r.loss, r.correct, *torch.autograd.grad(r.loss * 1024, (xs, ws)))

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
            xs.copy_(x * (1 + 0.25 * k))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_projection_without_gradients_and_without_rows(dtype):
    x, w, ids, teacher, targets = projected(50, 300, 64, dtype)
    w.requires_grad_()
    r = projection_topk_distillation(x, w, ids, teacher, targets, 2.0, 0.5)
    with torch.no_grad():
        s = projection_topk_distillation(x, w, ids, teacher, targets, 2.0, 0.5)
    assert torch.equal(r.loss.detach(), s.loss) and torch.equal(r.metrics, s.metrics) and not s.loss.requires_grad
    x0 = x[:0].requires_grad_()
    r = projection_topk_distillation(x0, w, ids[:0], teacher[:0], targets[:0], 2.0, 0.5)
    r.loss.backward()
    assert float(r.loss) == 0.0 and x0.grad.shape == (0, 64) and torch.equal(w.grad, torch.zeros_like(w))


class _Calls(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func))
        return func(*args, **(kwargs or {}))

    def products(self):
        return [n for n in self.names if any(w in n for w in ("mm", "matmul", "linear", "dot", "mv"))]


@gpu
@pytest.mark.parametrize("N,V,K_in", [(50, 304, 64), (3, 16, 8), (33, 7, 96), (70, 1003, 77)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_projection_takes_no_library_product(N, V, K_in, dtype):
    x, w, ids, teacher, targets = projected(N, V, K_in, dtype, K=5)
    x.requires_grad_()
    w.requires_grad_()
    with _Calls() as seen:
        r = projection_topk_distillation(x, w, ids, teacher, targets, 2.0, 0.5)
        r.loss.backward()
    assert seen.names and seen.products() == []
    with _Calls() as seen:  # (the mode sees the products of a forward and of a backward)
        F.linear(x, w).sum().backward()
    assert len(seen.products()) >= 3


@gpu
@pytest.mark.parametrize("N,V,K_in", [(5, 7, 3), (33, 16, 96), (257, 5003, 64), (1000, 72, 333), (64, 20000, 520)])
def test_half_precision_projection_against_float64(N, V, K_in):
    x, w, ids, teacher, targets = projected(N, V, K_in, torch.float16, K=5)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    r = projection_topk_distillation(xs, ws, ids, teacher, targets, 2.0, 0.5)
    up = 2.0 ** 12
    (r.loss * up).backward()
    z = x.double() @ w.double().t()
    rows, grad, n = reference(z, ids, teacher, targets, 2.0, 0.5)
    grad = grad.to(DEV) * up / n
    assert abs(float(r.loss.detach()) - float(rows.sum()) / n) <= 2.0 ** -17 * 4
    # dlogits: probabilities of float32 logits (2^-17 of their size), rounded to half a step of theirs or of the smallest; then one product
    # of V or N terms in float32 and its rounding
    half, tiny = 2.0 ** -11, 2.0 ** -25
    q = grad.abs() + up / n * (torch.softmax(z / 2, 1) + 0.5 * torch.softmax(z, 1))
    for got, want, bound, steps, terms in ((xs.grad, grad @ w.double(), q @ w.double().abs(), w.double().abs().sum(0), V),
                                           (ws.grad, grad.t() @ x.double(), q.t() @ x.double().abs(), x.double().abs().sum(0), N)):
        err = (got.double() - want).abs()
        near = half + 2.0 ** -15 + terms * 2.0 ** -24
        assert bool((err <= near * bound + half * want.abs() + tiny * (steps + 1)).all())


# Every kernel by width, rows that start on and off the 16-byte grid (a row's vectors at its ends are its neighbours' as well, which other workgroups
# write over meanwhile), rows held in registers and rows read again from the memory that their gradient takes over.
@gpu
@pytest.mark.parametrize("width,C", [(70, 64), (1003, 1003), (1021, 900), (7171, 7171), (14343, 14340), (28672, 28000), (28673, 28673), (50257, 50257),
                                     (57345, 57345), (65543, 65543), (131083, 131000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_over_the_logits_is_that_beside_them(width, C, dtype):
    from distributed_pytorch_amd import _ext

    logits, ids, teacher, targets = make(37, C, min(C, 30), dtype, DEV, width=width)
    for tau, a in ((2.0, 0.5), (1.0, 0.0), (1.5, 0.5)):
        args = (ids, teacher, targets, C, -100, tau, a, True)
        want = _ext.C().distill_forward(logits, *args, "new")
        over = logits.clone()
        got = _ext.C().distill_forward(over, *args, "inplace")
        assert got[6].data_ptr() == over.data_ptr()
        for k in (0, 1, 2, 3, 6):
            assert torch.equal(got[k], want[k]), k


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("t_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tau", [0.25, 0.5, 1.0, 2.0])
def test_entries_of_the_lowest_and_largest_values_are_entries(tau, t_dtype, device):
    logits, ids, teacher, _ = make(5, 60, 6, torch.float32, device, pad_rows=False)
    low, high = torch.finfo(t_dtype).min, torch.finfo(t_dtype).max
    teacher = teacher.to(t_dtype)
    teacher[0] = low                                      # all alike: one sixth each
    teacher[1, :5] = low                                  # one entry takes it all
    teacher[2] = high
    teacher[3, ::2], teacher[3, 1::2] = high, low
    teacher[4, 2] = NEG
    x = logits.clone().requires_grad_()
    r = topk_distillation(x, ids, teacher, None, tau, reduction="none")
    (g,) = torch.autograd.grad(r.loss.sum(), x)
    z = logits.double().cpu()
    t = teacher.double().cpu()
    p = torch.softmax((t - t.amax(1, keepdim=True)) / tau, 1)
    log_q = torch.log_softmax(z / tau, 1).gather(1, ids.cpu())
    want = tau ** 2 * (torch.special.xlogy(p, p) - torch.where(p > 0, p * log_q, 0.0)).sum(1)
    grad = tau * torch.softmax(z / tau, 1).scatter_add(1, ids.cpu(), -p)
    near = 64 * 2.0 ** -23 * max(1.0, 1 / tau)  # as in check(), of exponents up to 4 times as large
    torch.testing.assert_close(r.loss.detach().double().cpu(), want, rtol=near, atol=near * max(1.0, tau ** 2))
    torch.testing.assert_close(g.double().cpu(), grad, rtol=near, atol=near * max(tau, 1.0))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_temperatures_beyond_float32_are_refused(device):
    logits, ids, teacher, targets = make(4, 11, 3, device=device)
    for tau in (1e-50, 1e-30, 1e30, 1e50):
        with pytest.raises(ValueError, match="temperature"):
            topk_distillation(logits, ids, teacher, targets, tau, 0.5)
        with pytest.raises(ValueError, match="temperature"):
            projection_topk_distillation(logits, torch.randn(11, 11, device=device), ids, teacher, targets, tau, 0.5)
    for tau in (1e-4, 1e4, 1e12):  # inside: finite, the soft term tau^2 log(C / K) of two flat distributions at last
        r = topk_distillation(logits, ids, teacher, None, tau)
        assert torch.isfinite(r.loss)
    assert abs(float(r.loss) / 1e24 - math.log(11 / 3) * 3 / 4 - math.log(11 / 1) / 4) < 1e-5  # (one row keeps one entry)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_no_gradient_reaches_the_teacher(device):
    logits, ids, teacher, targets = make(4, 11, 3, device=device)
    x, t = logits.requires_grad_(), teacher.requires_grad_()
    r = topk_distillation(x, ids, t, targets, 2.0, 0.5)
    gx, gt = torch.autograd.grad(r.loss, (x, t), allow_unused=True)
    assert gx is not None and gt is None
    assert not topk_distillation(x.detach(), ids, t, targets, 2.0, 0.5).loss.requires_grad


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_an_unknown_product_is_refused(device):
    _, ids, teacher, targets = make(4, 11, 3, device=device)
    with pytest.raises(ValueError, match="impl"):
        projection_topk_distillation(torch.randn(4, 8, device=device), torch.randn(11, 8, device=device), ids, teacher, impl="stock")


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_projection_of_views_and_single_gradients(dtype):
    x, w, ids, teacher, targets = projected(120, 1003, 96, dtype)
    up = 256.0

    def run(a, b, names="xw", **kw):
        a, b = a.detach().requires_grad_("x" in names), b.detach().requires_grad_("w" in names)
        r = projection_topk_distillation(a, b, ids, teacher, targets, 2.0, 0.5, **kw)
        return r.loss.detach(), dict(zip(names, torch.autograd.grad(r.loss * up, [a if n == "x" else b for n in names])))

    loss, want = run(x, w)
    for names in ("x", "w"):
        one, got = run(x, w, names)
        assert torch.equal(one, loss) and torch.equal(got[names], want[names])
    off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)  # noqa: E731  one element off a 16-byte boundary
    turned = lambda t: t.t().contiguous().t()  # noqa: E731
    for view in (off, turned):
        same, got = run(view(x), view(w))
        assert torch.equal(same, loss) and torch.equal(got["x"], want["x"]) and torch.equal(got["w"], want["w"])
    # the vendor's products: logits rounded to the type, half a step of about 2 at most; gradients of those
    other, got = run(x, w, impl="library")
    half = torch.finfo(dtype).eps / 2
    assert abs(float(other) - float(loss)) <= 4 * half * 2 + 2e-5
    for n in "xw":
        assert float((got[n].float() - want[n].float()).norm()) <= (8 * half + 2e-5) * float(want[n].float().norm())


@gpu
def test_projections_on_two_streams():
    a, b = projected(2100, 4100, 64, torch.bfloat16, 1), projected(2100, 4100, 64, torch.bfloat16, 2)

    def grads(t):
        x, w = t[0].detach().requires_grad_(), t[1].detach().requires_grad_()
        r = projection_topk_distillation(x, w, *t[2:], 2.0, 0.5)
        return (r.loss.detach(), *torch.autograd.grad(r.loss, (x, w)))

    want = [grads(a), grads(b)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            ga = grads(a)
        with torch.cuda.stream(s2):
            gb = grads(b)
        torch.cuda.synchronize()
        for got, w in ((ga, want[0]), (gb, want[1])):
            assert all(torch.equal(p, q) for p, q in zip(got, w))


# rows of float32 logits that are read twice, with the sums taken along with the maximum: one vector a thread, several, and a ragged last one
@gpu
@pytest.mark.parametrize("N,V,C", [(7, 28676, 28676), (5, 30011, 29000), (40, 50304, 50257), (3, 131083, 131083)])
@pytest.mark.parametrize("tau,a", [(1.0, 0.0), (2.0, 0.5), (4.0, 0.25), (3.0, 0.5), (2.0, 1.0)])
def test_wide_projected_rows(N, V, C, tau, a):
    from distributed_pytorch_amd import _ext

    x, w, ids, teacher, targets = projected(N, V, 64, torch.bfloat16, K=9, C=C)
    x = x * 12                                       # logits of about 2, with a long tail
    x[1] = 0                                         # all alike
    targets[2] = -100
    r = _ext.C().projection_distill_forward(x, w, ids, teacher, targets, C, -100, tau, a, True, "gradient")
    z = x.double() @ w.double().t()
    rows, grad, n = reference(z, ids, teacher, targets, tau, a, C)
    near = 64 * 2.0 ** -23                           # as in check()
    size = max(1.0, tau ** 2) * (1 + float(rows.abs().max()) / max(1.0, tau ** 2))
    assert abs(float(r[0]) - float(rows.sum()) / n) <= near * size
    torch.testing.assert_close(r[6].double().cpu(), grad / n, rtol=2.0 ** -9 * 2.02, atol=near * max(tau, 1.0) / n)
    best = z[:, :C].argmax(1).cpu()
    top = z[:, :C].topk(2, 1).values.cpu()
    sure = (top[:, 0] - top[:, 1] > 1e-4) & (targets.cpu() != -100)
    assert torch.equal(r[1].cpu()[sure], (best == targets.cpu())[sure])


# classes hidden by a large negative logit: whole threads see nothing else at first, on rows that are held, read twice, and read again in the backward
@gpu
@pytest.mark.parametrize("hide", [-1e9, -1e30, "lowest", NEG])
@pytest.mark.parametrize("C,dtype", [(900, torch.float32), (20011, torch.bfloat16), (70001, torch.float32), (140003, torch.bfloat16), (140003, torch.float16)])
def test_hidden_classes(C, dtype, hide):
    if dtype == torch.float16 and hide in (-1e9, -1e30):
        hide = "lowest"
    value = torch.finfo(dtype).min if hide == "lowest" else hide
    logits, ids, teacher, targets = make(4, C, 6, dtype, DEV, pad_rows=False)
    logits = logits + 20
    g = torch.Generator().manual_seed(C)
    open_ = [torch.arange(C - 50, C), torch.arange(0, 50), torch.randperm(C, generator=g)[:50], torch.arange(C)]
    for r, keep in enumerate(open_):
        row = torch.full((C,), value, dtype=dtype, device=DEV)
        row[keep.to(DEV)] = logits[r, keep.to(DEV)]
        logits[r] = row
        ids[r] = keep[torch.randperm(len(keep), generator=g)[:6]].to(DEV)
        targets[r] = int(keep[7])
    for tau, a in ((1.0, 0.0), (2.0, 0.5), (4.0, 0.25), (3.0, 0.5)):
        check(logits, ids, teacher, targets, tau, a)
        x = logits.clone().requires_grad_()
        r = topk_distillation(x, ids, teacher, targets, tau, a, reduction="none")
        rows, grad, _ = reference(logits, ids, teacher, targets, tau, a)
        near = 64 * 2.0 ** -23 * max(1.0, tau ** 2)
        torch.testing.assert_close(r.loss.detach().double().cpu(), rows, rtol=near, atol=near)
        (d,) = torch.autograd.grad(r.loss.sum(), x)
        torch.testing.assert_close(d.double().cpu(), grad, rtol=torch.finfo(dtype).eps / 2 * 1.01, atol=near + (2.0 ** -25 if dtype == torch.float16 else 0.0))
