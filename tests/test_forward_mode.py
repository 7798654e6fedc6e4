"""Forward-mode tangents through the operators of a student model: followed by the stock compositions, refused by the kernels, never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from distributed_pytorch_amd.ops import gated_mlp, projection_topk_distillation, topk_distillation, window_attention_qkvpacked

gpu = pytest.mark.gpu


def calls(device, dtype):
    """(name, function of one tensor, that tensor)"""
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)  # noqa: E731
    x, w_fc, w_proj = r(5, 8), r(12, 8), r(8, 6)
    ids, teacher = torch.randint(0, 12, (5, 3), generator=g).to(device), torch.randn(5, 3, generator=g).to(device)
    yield "attention", lambda t: window_attention_qkvpacked(t, 1, 3), r(1, 5, 3 * 64)
    yield "gated x", lambda t: gated_mlp(t, w_fc, None, w_proj, None), x
    yield "gated w_fc", lambda t: gated_mlp(x, t, None, w_proj, None), w_fc
    yield "gated w_proj", lambda t: gated_mlp(x, w_fc, None, t, None), w_proj
    yield "gated b_proj", lambda t: gated_mlp(x, w_fc, None, w_proj, t), r(8)
    yield "distillation", lambda t: topk_distillation(t, ids, teacher).loss, r(5, 12)
    yield "projection x", lambda t: projection_topk_distillation(t, w_fc, ids, teacher).loss, x
    yield "projection w", lambda t: projection_topk_distillation(x, t, ids, teacher).loss, w_fc


def test_followed_on_the_cpu():
    for name, f, t in calls("cpu", torch.float64):
        way = torch.randn_like(t)
        with fwAD.dual_level():
            tangent = fwAD.unpack_dual(f(fwAD.make_dual(t, way))).tangent
        h = 1e-6
        assert tangent is not None, name
        diff = (f(t + h * way) - f(t - h * way)) / (2 * h)
        torch.testing.assert_close(tangent.to(diff.dtype), diff, rtol=1e-6, atol=1e-7)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_refused_by_the_kernels(dtype):
    for name, f, t in calls("cuda", dtype):
        want = f(t)
        for grad in (True, False):
            with torch.set_grad_enabled(grad), fwAD.dual_level():
                with pytest.raises(RuntimeError):
                    f(fwAD.make_dual(t, torch.randn_like(t)))
                assert torch.equal(f(t), want), name  # no tangent here: as ever
        assert torch.equal(f(t), want)
