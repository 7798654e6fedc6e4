"""Measured cases of three operators of a transformer's training step: causal attention with a sliding window and
sinks, the gated feed-forward block, and distillation from a teacher's top logits.

``run`` computes a case with elementary torch operations in float32 where ``own`` is false and through the package's
public entry points where it is true; ``exact`` computes the same in float64 from the definitions.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# --------------------------------------------------------------------------------------------------- cases
def _attention(name, B, T, H, KV, D, window, sinks, dtype="bf16", lens=False, train=True):
    return dict(name=name, op="attention", B=B, T=T, H=H, KV=KV, D=D, window=window, sinks=sinks, dtype=dtype, lens=lens, train=train)


def _gated(name, M, K, H, act="silu", bias=False, dtype="bf16", train=True):
    return dict(name=name, op="gated", M=M, K=K, H=H, act=act, bias=bias, dtype=dtype, train=train)


def _distill(name, N, V, classes, K, tau, hard, dtype="bf16", width=0, padded=False):
    return dict(name=name, op="distill", N=N, V=V, classes=classes, K=K, tau=tau, hard=hard, dtype=dtype, width=width, padded=padded)


def listed():
    return [
        # a training step of the 12-head model on 1024-token sequences, local attention in every layer
        _attention("attention train", 64, 1024, 12, 12, 64, 256, 4),
        # one long document, shared k/v heads, head size 128
        _attention("attention long", 1, 16384, 8, 2, 128, 1024, 4),
        # a padded fine-tuning batch in fp16: lengths from 0 to T, no multiple of any tile
        _attention("attention ragged", 16, 777, 12, 4, 64, 128, 1, dtype="fp16", lens=True),
        # a short prompt scored without gradients: latency
        _attention("attention prompt", 1, 61, 12, 12, 64, 32, 2, train=False),
        # a training step's feed-forward block at the small width, 64 sequences of 1024 tokens
        _gated("gated train", 65536, 768, 2048),
        # the wider model with biases and the GELU gate
        _gated("gated train bias", 16384, 1024, 2816, act="gelu", bias=True),
        # a small odd batch in fp16, no extent a multiple of a tile
        _gated("gated ragged", 1003, 520, 1386, dtype="fp16", bias=True),
        # one token through the block: weight bytes and latency
        _gated("gated token", 1, 768, 2048, train=False),
        # vocabulary projection + loss of a student step: 24 sequences of 1024 tokens
        _distill("distill projection", 24576, 50304, 50257, 64, 2.0, 0.5, width=768),
        # the loss on logits that the program already has, padded vocabulary, ignored rows
        _distill("distill logits", 8192, 50304, 50257, 32, 1.0, 0.0, padded=True),
        # float32 logits of an odd vocabulary, more teacher entries, teacher rows of different lengths
        _distill("distill fp32 odd", 2049, 50257, 50257, 100, 3.0, 0.1, dtype="fp32", padded=True),
        # a small classifier: latency
        _distill("distill small", 32, 1000, 1000, 5, 4.0, 0.7),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "gated", "distill"])
    if op == "attention":
        H = rng.choice([1, 2, 4, 6, 8, 12, 16])
        KV = rng.choice([d for d in range(1, H + 1) if H % d == 0])
        T = _log_int(rng, 1, 8192)
        B = _log_int(rng, 1, max(1, min(64, 400_000_000 // (H * T * T))))
        c = _attention("", B, T, H, KV, rng.choice([64, 128]), _log_int(rng, 1, max(1, T)), rng.choice([0, 1, 4, 37, 150]),
                       dtype=rng.choice(["bf16", "bf16", "fp16"]), lens=rng.random() < 0.4, train=rng.random() < 0.7)
    elif op == "gated":
        K = rng.choice([64 * rng.randint(2, 16), 8 * rng.randint(10, 130), rng.randint(65, 1000)])
        H = rng.choice([256 * rng.randint(1, 11), 8 * rng.randint(20, 350), rng.randint(100, 2700)])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c = _gated("", _log_int(rng, 1, 4096 if dtype == "fp32" else 32768), K, H, act=rng.choice(["silu", "gelu", "relu"]), bias=rng.random() < 0.5,
                   dtype=dtype, train=rng.random() < 0.7)
    else:
        V = _log_int(rng, 70, 60000)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        width = rng.choice([0, 0, 0, 256, 768]) if dtype == "bf16" and V % 8 == 0 else 0
        c = _distill("", _log_int(rng, 1, 4096), V, V - rng.choice([0, 0, V // 50]), _log_int(rng, 1, 60), rng.choice([1.0, 1.5, 2.0, 4.0]),
                     rng.choice([0.0, 0.1, 0.5, 1.0]), dtype=dtype, width=width, padded=rng.random() < 0.5)
    c.pop("name")
    return c


# --------------------------------------------------------------------------------------------------- inputs
def _lens_of(case):
    """The lengths of a padded batch, shortest (0 where the batch has more than one sequence) to longest."""
    B, T = case["B"], case["T"]
    return [T] if B == 1 else [round(T * i / (B - 1)) for i in range(B)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    s = {"case": case}
    if case["op"] == "attention":
        B, T, H, KV, D = (case[k] for k in ("B", "T", "H", "KV", "D"))
        s["qkv"] = normal(B, T, (H + 2 * KV) * D)
        s["do"] = normal(B, T, H * D) if case["train"] else None
        s["lens"] = None
        if case["lens"]:
            order = torch.randperm(B, generator=gen, device="cuda")
            s["lens"] = torch.tensor(_lens_of(case), dtype=torch.int32, device="cuda")[order].contiguous()
    elif case["op"] == "gated":
        M, K, H = case["M"], case["K"], case["H"]
        s["x"] = normal(M, K)                               # behind a norm: unit variance
        s["w_fc"] = normal(2 * H, K, std=K ** -0.5)
        s["w_proj"] = normal(K, H, std=H ** -0.5)
        s["b_fc"] = normal(2 * H, std=0.1) if case["bias"] else None
        s["b_proj"] = normal(K, std=0.1) if case["bias"] else None
        s["dy"] = normal(M, K, std=0.1) if case["train"] else None
    else:
        N, V, C, K = case["N"], case["V"], case["classes"], case["K"]
        if case["width"]:
            s["x"] = normal(N, case["width"])
            s["w"] = normal(V, case["width"], std=0.02)     # a student near its initialisation
        else:
            s["logits"] = normal(N, V, std=2.0)
        # a teacher's stored answer for every token: K different classes and their logits, largest first
        first = torch.randint(0, C, (N, 1), generator=gen, device="cuda")
        gap = torch.randint(1, max(2, C // K), (N, K), generator=gen, device="cuda")
        s["ids"] = (first + gap.cumsum(1)) % C
        s["teacher"] = (torch.randn(N, K, generator=gen, device="cuda") * 2 + 6).sort(1, descending=True).values
        s["targets"] = torch.randint(0, C, (N,), generator=gen, device="cuda")
        if case["padded"]:
            count = torch.randint(0, K + 1, (N, 1), generator=gen, device="cuda")
            s["ids"] = torch.where(torch.arange(K, device="cuda") < count, s["ids"], -1)
            s["targets"] = torch.where(torch.rand(N, generator=gen, device="cuda") < 0.2, -100, s["targets"])
    return s


# --------------------------------------------------------------------------------------------------- plain forms
def _visible(case, lens):
    T = case["T"]
    i = torch.arange(T, device="cuda").view(1, 1, T, 1)
    j = torch.arange(T, device="cuda").view(1, 1, 1, T)
    ok = (j <= i) & ((i - j < case["window"]) | (j < case["sinks"]))
    if lens is not None:
        n = lens.view(-1, 1, 1, 1)
        ok = ok & (i < n) & (j < n)
    return ok


def _plain_attention(s):
    c = s["case"]
    B, T, H, KV, D = (c[k] for k in ("B", "T", "H", "KV", "D"))
    dt, G = s["qkv"].dtype, H // KV
    x = s["qkv"].float().view(B, T, H + 2 * KV, D).transpose(1, 2)
    q = x[:, :H].contiguous()
    k = x[:, H:H + KV].repeat_interleave(G, 1).contiguous()
    v = x[:, H + KV:].repeat_interleave(G, 1).contiguous()
    scale = D ** -0.5
    p = (q @ k.transpose(2, 3).contiguous()).mul_(scale).masked_fill_(~_visible(c, s["lens"]), -math.inf)
    p.sub_(p.amax(3, keepdim=True).clamp_min(-1e30)).exp_()
    p.div_(p.sum(3, keepdim=True).clamp_min(1e-30))
    o = p @ v
    out = {"o": o.transpose(1, 2).reshape(B, T, H * D).to(dt)}
    if s["do"] is None:
        return out
    do = s["do"].float().view(B, T, H, D).transpose(1, 2).contiguous()
    dv = p.transpose(2, 3).contiguous() @ do
    ds = do @ v.transpose(2, 3).contiguous()
    ds.sub_((do * o).sum(3, keepdim=True)).mul_(p).mul_(scale)
    dq = ds @ k
    dk = ds.transpose(2, 3).contiguous() @ q
    dk, dv = (t.view(B, KV, G, T, D).sum(2) for t in (dk, dv))
    out["dqkv"] = torch.cat([dq, dk, dv], 1).transpose(1, 2).reshape(B, T, (H + 2 * KV) * D).to(dt)
    return out


def _act_and_slope(g, act):
    if act == "silu":
        t = 1 / (1 + torch.exp(-g))
        return g * t, t * (1 + g * (1 - t))
    if act == "gelu":
        t = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * t, t + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    on = (g > 0).to(g.dtype)
    return g * on, on


def _plain_gated(s):
    c, dt = s["case"], s["x"].dtype
    H = c["H"]
    x, w_fc, w_proj = s["x"].float(), s["w_fc"].float(), s["w_proj"].float()
    gu = x @ w_fc.t()
    if c["bias"]:
        gu = gu + s["b_fc"].float()
    g, u = gu[:, :H], gu[:, H:]
    a, slope = _act_and_slope(g, c["act"])
    h = a * u
    y = h @ w_proj.t()
    if c["bias"]:
        y = y + s["b_proj"].float()
    out = {"y": y.to(dt)}
    if s["dy"] is None:
        return out
    dy = s["dy"].float()
    dh = dy @ w_proj
    dgu = torch.cat([dh * u * slope, dh * a], 1)
    out.update(dx=(dgu @ w_fc).to(dt), dw_fc=(dgu.t() @ x).to(dt), dw_proj=(dy.t() @ h).to(dt))
    if c["bias"]:
        out.update(db_fc=dgu.sum(0).to(dt), db_proj=dy.sum(0).to(dt))
    return out


def _plain_distill(s):
    c = s["case"]
    V, C, tau, hard = c["V"], c["classes"], c["tau"], c["hard"]
    z = (s["x"].float() @ s["w"].float().t() if c["width"] else s["logits"].float())[:, :C]
    counted = (s["targets"] != -100).float()
    rows = counted.sum().clamp_min(1)
    there = s["ids"] >= 0
    ids = s["ids"].clamp_min(0)
    some = there.any(1).float()
    t = (s["teacher"] / tau).masked_fill(~there, -math.inf)
    t = t - t.amax(1, keepdim=True).clamp_min(-1e30)
    log_p = t - t.exp().sum(1, keepdim=True).clamp_min(1e-30).log()
    p = log_p.exp()
    top = z.amax(1, keepdim=True)
    e = torch.exp((z - top) / tau)
    e1 = torch.exp(z - top)
    l, l1 = e.sum(1, keepdim=True), e1.sum(1, keepdim=True)
    log_q = (z.gather(1, ids) - top) / tau - l.log()
    soft = torch.where(there, p * (log_p - log_q), 0.0).sum(1) * tau * tau
    y = s["targets"].clamp_min(0).unsqueeze(1)
    nll = l1.log().squeeze(1) - (z.gather(1, y) - top).squeeze(1)
    loss = (((1 - hard) * soft + hard * nll) * counted).sum() / rows
    d = e.div_(l).mul_(some.unsqueeze(1)).scatter_add_(1, ids, torch.where(there, -p, 0.0)).mul_((1 - hard) * tau)
    d.add_(e1.div_(l1).scatter_add_(1, y, torch.full_like(y, -1.0, dtype=torch.float32)), alpha=hard)
    d.mul_((counted / rows).unsqueeze(1))
    d = torch.cat([d, d.new_zeros(d.shape[0], V - C)], 1) if V > C else d
    if c["width"]:
        return {"loss": loss, "dx": (d @ s["w"].float()).to(s["x"].dtype), "dw": (d.t() @ s["x"].float()).to(s["w"].dtype)}
    best = torch.where(z == top, torch.arange(C, device="cuda"), C).amin(1)
    return {"loss": loss, "correct": best == s["targets"], "dlogits": d.to(s["logits"].dtype)}


# --------------------------------------------------------------------------------------------------- the framework's calls
def _own_attention(s):
    from distributed_pytorch_amd.ops import window_attention_qkvpacked

    c = s["case"]
    args = dict(sinks=c["sinks"], n_kv_head=c["KV"], seq_lens=s["lens"])
    if s["do"] is None:
        with torch.no_grad():
            return {"o": window_attention_qkvpacked(s["qkv"], c["H"], c["window"], **args)}
    qkv = s["qkv"].detach().requires_grad_()
    o = window_attention_qkvpacked(qkv, c["H"], c["window"], **args)
    (dqkv,) = torch.autograd.grad(o, qkv, s["do"])
    return {"o": o, "dqkv": dqkv}


def _own_gated(s):
    from distributed_pytorch_amd.ops import gated_mlp

    act = s["case"]["act"]
    if s["dy"] is None:
        with torch.no_grad():
            return {"y": gated_mlp(s["x"], s["w_fc"], s["b_fc"], s["w_proj"], s["b_proj"], act=act)}
    names = ["x", "w_fc", "w_proj"] + (["b_fc", "b_proj"] if s["b_fc"] is not None else [])
    leaf = {n: s[n].detach().requires_grad_() for n in names}
    y = gated_mlp(leaf["x"], leaf["w_fc"], leaf.get("b_fc"), leaf["w_proj"], leaf.get("b_proj"), act=act)
    grads = torch.autograd.grad(y, [leaf[n] for n in names], s["dy"])
    return {"y": y, **{"d" + n: g for n, g in zip(names, grads)}}


def _own_distill(s):
    from distributed_pytorch_amd.ops import projection_topk_distillation, topk_distillation

    c = s["case"]
    args = dict(targets=s["targets"], temperature=c["tau"], hard_weight=c["hard"], n_classes=c["classes"])
    if c["width"]:
        x, w = s["x"].detach().requires_grad_(), s["w"].detach().requires_grad_()
        r = projection_topk_distillation(x, w, s["ids"], s["teacher"], **args)
        dx, dw = torch.autograd.grad(r.loss, [x, w])
        return {"loss": r.loss, "dx": dx, "dw": dw}
    logits = s["logits"].detach().requires_grad_()
    r = topk_distillation(logits, s["ids"], s["teacher"], **args)
    (dlogits,) = torch.autograd.grad(r.loss, logits)
    return {"loss": r.loss, "correct": r.correct, "dlogits": dlogits}


def run(state):
    op = state["case"]["op"]
    if op == "attention":
        return _own_attention(state) if own else _plain_attention(state)
    if op == "gated":
        return _own_gated(state) if own else _plain_gated(state)
    return _own_distill(state) if own else _plain_distill(state)


# --------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attention":
        H, KV, D, W, S = (case[k] for k in ("H", "KV", "D", "window", "sinks"))
        lens = _lens_of(case) if case["lens"] else [case["T"]] * case["B"]
        pairs = 0
        for n in lens:
            i = np.arange(n, dtype=np.int64)
            pairs += int((np.minimum(i + 1, W) + np.minimum(S, np.maximum(0, i + 1 - W))).sum())
        tokens, width = sum(lens), H + 2 * KV
        flops = 4.0 * D * H * pairs
        moved = tokens * D * size * (width + H)
        if case["train"]:  # gradients of q|k|v from do; five products, the scores among them
            flops += 10.0 * D * H * pairs
            moved += tokens * D * size * (width + H)
        return {"bytes": moved + 2 * size * (case["B"] * case["T"] - tokens) * H * D, "flops": flops}
    if case["op"] == "gated":
        M, K, H = case["M"], case["K"], case["H"]
        flops, moved = 6.0 * M * K * H, size * (2 * M * K + 3 * K * H)
        if case["train"]:
            flops, moved = 3 * flops, moved + size * (2 * M * K + 3 * K * H)
        return {"bytes": moved, "flops": flops}
    N, V, K = case["N"], case["V"], case["K"]
    side = N * (K * 12 + 8)
    if case["width"]:
        return {"bytes": size * 2 * (N + V) * case["width"] + side, "flops": 6.0 * N * V * case["width"]}
    return {"bytes": 2 * size * N * V + side, "flops": 12.0 * N * V}


# --------------------------------------------------------------------------------------------------- float64
def _exact_attention(case, s):
    B, T, H, KV, D, W, S = (case[k] for k in ("B", "T", "H", "KV", "D", "window", "sinks"))
    G = H // KV
    lens = [T] * B if s["lens"] is None else s["lens"].tolist()
    o = torch.zeros(B, T, H, D, dtype=torch.float64, device="cuda")
    d = torch.zeros(B, T, H + 2 * KV, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        n = lens[b]
        x = s["qkv"][b, :n].double().view(n, H + 2 * KV, D).transpose(0, 1)
        do = s["do"][b, :n].double().view(n, H, D).transpose(0, 1) if case["train"] else None
        for lo in range(0, n, 1024):
            hi = min(n, lo + 1024)
            first = max(0, lo - W + 1)
            keys = torch.cat([torch.arange(0, min(S, first)), torch.arange(first, hi)]).cuda()
            qi = torch.arange(lo, hi, device="cuda").unsqueeze(1)
            hide = (keys > qi) | ((keys <= qi - W) & (keys >= S))
            q = x[:H, lo:hi].reshape(KV, G * (hi - lo), D)
            k, v = x[H:H + KV, keys], x[H + KV:, keys]
            z = (torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(D)).view(KV, G, hi - lo, -1)
            p = torch.softmax(z.masked_fill(hide, -math.inf), 3).view(KV, G * (hi - lo), -1)
            r = torch.bmm(p, v.contiguous())
            o[b, lo:hi, :] = r.view(H, hi - lo, D).transpose(0, 1)
            if do is None:
                continue
            g = do[:, lo:hi].reshape(KV, G * (hi - lo), D)
            dz = p * (torch.bmm(g, v.transpose(1, 2).contiguous()) - (g * r).sum(2, keepdim=True)) / math.sqrt(D)
            d[b, lo:hi, :H] = torch.bmm(dz, k.contiguous()).view(H, hi - lo, D).transpose(0, 1)
            d[b, :, H:H + KV].index_add_(0, keys, torch.bmm(dz.transpose(1, 2).contiguous(), q).transpose(0, 1).contiguous())
            d[b, :, H + KV:].index_add_(0, keys, torch.bmm(p.transpose(1, 2).contiguous(), g).transpose(0, 1).contiguous())
    out = {"o": o.view(B, T, H * D)}
    if case["train"]:
        out["dqkv"] = d.view(B, T, -1)
    return out


def _exact_gated(case, s):
    names = [n for n in ("x", "w_fc", "w_proj", "b_fc", "b_proj") if s[n] is not None]
    t = {n: s[n].double().requires_grad_(case["train"]) for n in names}
    f = torch.nn.functional
    gate, up = (f.linear(t["x"], w, b) for w, b in zip(t["w_fc"].chunk(2), t["b_fc"].chunk(2) if case["bias"] else (None, None)))
    y = f.linear({"silu": f.silu, "gelu": f.gelu, "relu": f.relu}[case["act"]](gate) * up, t["w_proj"], t.get("b_proj"))
    out = {"y": y.detach()}
    if case["train"]:
        out.update(zip(["d" + n for n in names], torch.autograd.grad(y, [t[n] for n in names], s["dy"].double())))
    return out


def _exact_distill(case, s):
    N, V, C, K, tau, hard = (case[k] for k in ("N", "V", "classes", "K", "tau", "hard"))
    f = torch.nn.functional
    rows = max(1, int((s["targets"] != -100).sum()))
    total, grads, dw = 0.0, [], 0.0
    w = s["w"].double() if case["width"] else None
    for lo in range(0, N, 2048):
        part = slice(lo, lo + 2048)
        x = s["x"][part].double() if case["width"] else None
        z = (x @ w.t() if case["width"] else s["logits"][part].double()).requires_grad_()
        ids, y = s["ids"][part], s["targets"][part]
        absent = ids < 0
        log_p = torch.log_softmax((s["teacher"][part].double() / tau).masked_fill(absent, -1e300), 1)
        log_q = torch.log_softmax(z[:, :C] / tau, 1).gather(1, ids.clamp_min(0))
        soft = (log_p.exp() * (log_p - log_q)).masked_fill(absent, 0.0).sum(1) * tau ** 2
        nll = f.cross_entropy(z[:, :C], y, reduction="none", ignore_index=-100)
        loss = ((1 - hard) * soft * (y != -100) + hard * nll).sum() / rows
        (dz,) = torch.autograd.grad(loss, z)
        total += float(loss)
        grads.append(dz @ w if case["width"] else dz)
        if case["width"]:
            dw = dw + dz.t() @ x
    out = {"loss": torch.tensor(total, dtype=torch.float64, device="cuda")}
    if case["width"]:
        return {**out, "dx": torch.cat(grads), "dw": dw}
    return {**out, "correct": None, "dlogits": torch.cat(grads)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "gated": _exact_gated, "distill": _exact_distill}[case["op"]](case, s)
