"""Windowed attention, shared key / value heads, the gated feed-forward block and the distillation loss together, as a student GPT-2
uses them: loss and gradients against stock operators, a step under graph replay, optimizer steps."""
import pytest
import torch
import torch.nn.functional as F

from distributed_pytorch_amd.models import GPT2, GPT2Config

gpu = pytest.mark.gpu


def config(**kw):
    base = dict(block_size=160, vocab_size=301, n_layer=2, n_head=4, n_embd=256, n_kv_head=2, attention_window=48, attention_sinks=3, mlp="gated")
    base.update(kw)
    return GPT2Config(**base)


def batch(B, T, vocab, K=9, device="cpu", seed=0):
    g = torch.Generator().manual_seed(seed)
    idx = torch.randint(0, vocab, (B, T), generator=g)
    targets = torch.randint(0, vocab, (B, T), generator=g)
    targets[0, :3] = -100
    ids = torch.rand(B, T, vocab, generator=g).topk(K, -1).indices
    values = torch.randn(B, T, K, generator=g) * 2
    return [t.to(device) for t in (idx, targets, ids, values)]


def stock_loss(model, cfg, idx, targets, ids, values, tau, a):
    """The same model out of elementary operators, in the parameters' type."""
    p = dict(model.named_parameters())
    B, T = idx.shape
    H, KV, D = cfg.n_head, cfg.n_kv_head, cfg.n_embd // cfg.n_head
    x = p["wte.weight"][idx] + p["wpe.weight"][torch.arange(T, device=idx.device)]
    i = torch.arange(T, device=idx.device)
    hide = (i[None] > i[:, None]) | ((i[:, None] - i[None] >= cfg.attention_window) & (i[None] >= cfg.attention_sinks))
    for n in range(cfg.n_layer):
        w = lambda s: p[f"h.{n}.{s}"]  # noqa: E731, B023
        y = F.layer_norm(x, (cfg.n_embd,), w("ln_1.weight"), w("ln_1.bias"))
        qkv = F.linear(y, w("attn.c_attn.weight"), w("attn.c_attn.bias")).view(B, T, H + 2 * KV, D).transpose(1, 2)
        q, k, v = qkv[:, :H], qkv[:, H:H + KV].repeat_interleave(H // KV, 1), qkv[:, H + KV:].repeat_interleave(H // KV, 1)
        s = torch.softmax((q @ k.transpose(2, 3).contiguous() * D ** -0.5).masked_fill(hide, float("-inf")), -1)
        y = (s @ v).transpose(1, 2).reshape(B, T, -1)
        x = x + F.linear(y, w("attn.c_proj.weight"), w("attn.c_proj.bias"))
        y = F.layer_norm(x, (cfg.n_embd,), w("ln_2.weight"), w("ln_2.bias"))
        g, u = F.linear(y, w("mlp.c_fc.weight"), w("mlp.c_fc.bias")).chunk(2, -1)
        x = x + F.linear(F.silu(g) * u, w("mlp.c_proj.weight"), w("mlp.c_proj.bias"))
    x = F.layer_norm(x, (cfg.n_embd,), p["ln_f.weight"], p["ln_f.bias"])
    z = F.linear(x, p["wte.weight"])[..., : cfg.vocab_size].flatten(0, 1)
    t = targets.flatten()
    log_p = torch.log_softmax(values.flatten(0, 1).to(z.dtype) / tau, 1)
    log_q = torch.log_softmax(z / tau, 1).gather(1, ids.flatten(0, 1))
    soft = (log_p.exp() * (log_p - log_q)).sum(1) * tau ** 2
    row = (1 - a) * soft + a * F.cross_entropy(z, t.clamp(min=0), reduction="none")
    live = t != -100
    return torch.where(live, row, 0.0).sum() / live.sum()


def grads(loss, model):
    return dict(zip([n for n, _ in model.named_parameters()], torch.autograd.grad(loss, list(model.parameters()))))


def test_configuration():
    assert config().hidden_width == 768 and GPT2Config.small(mlp="gated").hidden_width == 2048 and GPT2Config.medium(mlp="gated").hidden_width == 2816
    assert GPT2Config.small().hidden_width == 4 * 768 and not GPT2Config.small().local_attention
    assert GPT2(config()).h[0].attn.c_attn.weight.shape == (8 * 64, 256)
    for kw in (dict(n_kv_head=3), dict(attention_window=-1), dict(attention_window=0, attention_sinks=2), dict(mlp="swish")):
        with pytest.raises(ValueError):
            GPT2(config(**kw))


def test_flops_count_the_visible_keys():
    m = GPT2(config())
    T, W, S = 100, 48, 3
    pairs = sum(min(i + 1, W) + min(S, max(0, i + 1 - W)) for i in range(T))
    base = m.flops_per_token(T) - 12.0 * 2 * 256 * pairs / T
    assert abs(base - 6.0 * sum(p.numel() for n, p in m.named_parameters() if not n.startswith("wpe"))) < 1e-3


def test_student_matches_stock_operators_on_the_cpu():
    torch.manual_seed(0)
    cfg = config(n_embd=64)
    m = GPT2(cfg)
    data = batch(2, 70, cfg.vocab_size)
    idx, targets, ids, values = data
    loss = m(idx, targets, teacher=(ids, values), temperature=2.0, hard_weight=0.25)
    want = stock_loss(m, cfg, *data, 2.0, 0.25)
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-4
    got, ref = grads(loss, m), grads(want, m)
    for n in ref:
        torch.testing.assert_close(got[n], ref[n], rtol=1e-3, atol=2e-6, msg=n)
    # unfused path, no targets, and the plain loss of the same architecture
    m2 = GPT2(config(n_embd=64, fused_lm_head_loss=False))
    m2.load_state_dict(m.state_dict())
    assert abs(float(m2(idx, targets, teacher=(ids, values), temperature=2.0, hard_weight=0.25).detach()) - float(want.detach())) < 1e-4
    assert m(idx, teacher=(ids, values)).dim() == 0 and m(idx, targets).dim() == 0 and m(idx).shape == (2, 1, cfg.vocab_size)


@gpu
@pytest.mark.parametrize("T,kw", [(160, {}), (77, {}), (160, dict(n_kv_head=4, n_embd=512, mlp_hidden=1024)), (160, dict(attention_window=0, attention_sinks=0))])
def test_student_on_the_gpu_against_float64(T, kw):
    torch.manual_seed(0)
    cfg = config(**kw)
    m = GPT2(cfg).to("cuda", torch.bfloat16)
    exact = GPT2(cfg).to("cuda", torch.float64)
    exact.load_state_dict({k: v.double() for k, v in m.state_dict().items()})
    plain = GPT2(cfg).to("cuda", torch.float32)
    plain.load_state_dict({k: v.float() for k, v in m.state_dict().items()})
    data = batch(3, T, cfg.vocab_size, device="cuda")
    idx, targets, ids, values = data
    ref_cfg = cfg if cfg.attention_window else config(**{**kw, "attention_window": T})
    want = stock_loss(exact, ref_cfg, *data, 2.0, 0.25)
    ref = grads(want, exact)

    def worst(loss, model):
        g = grads(loss, model)
        return abs(float(loss.detach()) - float(want.detach())), {n: float((g[n].double() - ref[n]).norm() / ref[n].norm()) for n in ref}

    loss = m(idx, targets, teacher=(ids, values), temperature=2.0, hard_weight=0.25)
    off, rel = worst(loss, m)
    # bf16 activations: every tensor between two operators is rounded by up to 2^-8 of each value; a gradient passes some twenty of them,
    # whose errors add up in quadrature to at most 20^0.5 2^-8, doubled for the cancellations inside the sums
    assert off < 20 ** 0.5 * 2.0 ** -8 * float(want.detach())
    assert max(rel.values()) < 2 * 20 ** 0.5 * 2.0 ** -8, rel
    # the loss of the float32 model goes through the composed / float32 paths
    off, rel = worst(plain(idx, targets, teacher=(ids, values), temperature=2.0, hard_weight=0.25), plain)
    assert off < 1e-4 and max(rel.values()) < 1e-3, rel


@gpu
def test_student_step_captured_and_replayed():
    torch.manual_seed(0)
    cfg = config()
    m = GPT2(cfg).to("cuda", torch.bfloat16)
    idx, targets, ids, values = batch(4, 160, cfg.vocab_size, device="cuda")

    def step():
        loss = m(idx, targets, teacher=(ids, values), temperature=2.0, hard_weight=0.5)
        return [loss, *torch.autograd.grad(loss, list(m.parameters()))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        idx.copy_(torch.randint(0, cfg.vocab_size, idx.shape, device="cuda"))
        values.mul_(1.1)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)


@gpu
def test_optimizer_steps_change_every_parameter():
    from distributed_pytorch_amd.ops import FusedAdamW

    torch.manual_seed(0)
    cfg = config()
    m = GPT2(cfg).to("cuda", torch.bfloat16)
    before = {n: p.detach().clone() for n, p in m.named_parameters()}
    opt = FusedAdamW(m.parameters(), lr=1e-2, master_weights=True)
    idx, targets, ids, values = batch(4, 160, cfg.vocab_size, device="cuda")
    for _ in range(3):
        loss = m(idx, targets, teacher=(ids, values), temperature=2.0, hard_weight=0.5)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
    assert bool(torch.isfinite(loss.detach())) and all(not torch.equal(p, before[n]) for n, p in m.named_parameters())


@pytest.fixture()
def one_rank():
    from distributed_pytorch_amd.parallel import process_group as pg
    from distributed_pytorch_amd.parallel.store import Store

    store = Store("127.0.0.1", 0, is_host=True, bind_addr="127.0.0.1")
    pg.init_process_group(0, 1, "rccl", store=store)
    yield pg
    pg.destroy_process_group()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_student_under_the_reducer_matches_plain_training(one_rank, dtype):
    """Weight gradients go straight into their bucket slices (the tied embedding's second one, and those of a second backward before
    the step, have to be added): exactly the weights of training without the wrapper."""
    from distributed_pytorch_amd.ops import FusedAdamW
    from distributed_pytorch_amd.parallel.ddp import DistributedDataParallel

    cfg = config()
    torch.manual_seed(0)
    plain, twin = GPT2(cfg).to("cuda", dtype), GPT2(cfg).to("cuda", dtype)
    twin.load_state_dict(plain.state_dict())
    ddp = DistributedDataParallel(twin, device_ids=[0], bucket_cap_mb=0.25, first_bucket_mb=0.05)
    optimizers = [FusedAdamW(m.parameters(), 1e-3, master_weights=dtype != torch.float32) for m in (plain, ddp)]
    losses = ([], [])
    for step in range(4):
        for k, (model, opt) in enumerate(zip((plain, ddp), optimizers)):
            opt.zero_grad(set_to_none=True)
            for part in range(2 if step == 3 else 1):
                idx, targets, ids, values = batch(3, 160, cfg.vocab_size, device="cuda", seed=2 * step + part)
                if part == 0 and step == 3 and model is ddp:
                    with ddp.no_sync():
                        loss = model(idx, targets, teacher=(ids, values), temperature=2.0, hard_weight=0.5)
                        (loss * 0.5).backward()
                else:
                    loss = model(idx, targets, teacher=(ids, values), temperature=2.0, hard_weight=0.5)
                    (loss * 0.5 if step == 3 else loss).backward()
                losses[k].append(float(loss.detach()))
            opt.step()
    assert losses[0] == losses[1], losses
    for (n, a), b in zip(plain.named_parameters(), ddp.module.parameters()):
        assert torch.equal(a, b), n


@gpu
@pytest.mark.parametrize("rows", [5, 300])
def test_a_gated_block_used_twice_under_the_reducer(one_rank, rows):
    from distributed_pytorch_amd.ops import gated_mlp
    from distributed_pytorch_amd.parallel.ddp import DistributedDataParallel

    class Twice(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w_fc, self.b_fc = torch.nn.Parameter(torch.randn(2 * 136, 72) / 8), torch.nn.Parameter(torch.randn(2 * 136))
            self.w_proj, self.b_proj = torch.nn.Parameter(torch.randn(72, 136) / 11), torch.nn.Parameter(torch.randn(72))

        def forward(self, x):
            for _ in range(2):
                x = gated_mlp(x, self.w_fc, self.b_fc, self.w_proj, self.b_proj)
            return x

    torch.manual_seed(0)
    plain, twin = Twice().to("cuda", torch.bfloat16), Twice().to("cuda", torch.bfloat16)
    twin.load_state_dict(plain.state_dict())
    ddp = DistributedDataParallel(twin, device_ids=[0])
    x = torch.randn(rows, 72, device="cuda").bfloat16()
    for m in (plain, ddp):
        m(x).float().square().mean().backward()
    for a, b in zip(plain.parameters(), ddp.module.parameters()):
        assert torch.equal(a.grad, b.grad)
