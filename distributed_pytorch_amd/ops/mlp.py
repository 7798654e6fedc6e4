"""Two-layer MLP ``proj(act(fc(x)))`` as one autograd node.

A transformer MLP (``c_fc`` -> GELU -> ``c_proj``) is not in the reference's two-layer toy model
(reference min_DDP.py:41-49, which has no nonlinearity at all); it is the largest block of the
GPT-2 benchmark configuration.  Treating the pair of layers as one node lets the backward fuse
across the layer boundary: the input-gradient GEMM of ``proj`` applies the activation derivative
of ``fc`` in its epilogue and accumulates ``fc``'s bias gradient on the way out, so the
[tokens, 4*C] gradient is written once and never re-read by an elementwise pass.

    forward   pre, h = x W_fc^T + b_fc, act(.)   MFMA GEMM, both outputs from one epilogue (GELU; GEMM + elementwise
                                                   pass for other activations)
              y   = h W_proj^T (+ b_proj)  MFMA GEMM
    backward  g, db_fc = (dy W_proj) * act'(pre), colsum(.)   MFMA GEMM, fused epilogue
              dW_proj  = dy^T h                                split-K MFMA GEMM
              dx       = g W_fc                                MFMA GEMM
              dW_fc    = g^T x                                 split-K MFMA GEMM

``impl="library"`` sends the three plain products to the vendor GEMM (A/B measurements only).

``gated_mlp`` is the block whose hidden layer is a product of two projections, ``(act(x W_g^T) * (x W_u^T)) W_proj^T``, with both
in one packed weight.  Forward and backward are one node as well:

    forward   h, g | u = act(g) * u, x W_fc^T + b_fc            one MFMA GEMM over interleaved rows, the product in its epilogue
              y        = h W_proj^T (+ b_proj)                  MFMA GEMM
    backward  dg | du  = dh u act'(g) | dh act(g), dh = dy W_proj    one MFMA GEMM, both gradients (and db_fc) in its epilogue
              dW_proj, dx, dW_fc                                plain MFMA GEMMs
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from .. import _ext
from . import gemm
from .grad_sink import weight_grad_buffer
from .linear import ACT_GELU, ACT_RELU, ACT_SILU, _act_code, _torch_act, linear_bias_act
from .tangents import is_differentiated


class _FusedMLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, w_fc, b_fc, w_proj, b_proj, act: int, impl: str):
        if act == ACT_GELU:
            # one GEMM writes the activation and the pre-activation from its epilogue
            h, pre = _ext.C().linear_forward(x2, w_fc, b_fc, act, True)
        else:
            pre = gemm.nt(x2, w_fc, b_fc, impl)
            h = _torch_act(pre, act)
        y = gemm.nt(h, w_proj, b_proj, impl)
        ctx.act = act
        ctx.impl = impl
        ctx.has_b_proj = b_proj is not None
        ctx.save_for_backward(x2, w_fc, w_proj, pre if act == ACT_GELU else h, h)
        return y

    @staticmethod
    def backward(ctx, dy):
        C = _ext.C()
        x2, w_fc, w_proj, aux, h = ctx.saved_tensors
        dy = dy.contiguous()
        g, db_fc = C.dgrad_act_backward(dy, w_proj, aux, ctx.act, True)
        dw_proj = gemm.weight_grad(dy, h, w_proj, ctx.impl)
        db_proj = C.colsum(dy) if ctx.has_b_proj else None
        dx = gemm.nn(g, w_fc, ctx.impl) if ctx.needs_input_grad[0] else None
        dw_fc = gemm.weight_grad(g, x2, w_fc, ctx.impl)
        return dx, dw_fc, db_fc, dw_proj, db_proj, None, None


def fused_mlp_supported(x: torch.Tensor, w_fc: torch.Tensor, b_fc, w_proj: torch.Tensor, act) -> bool:
    if not (x.is_cuda and x.dtype == torch.bfloat16 and w_fc.dtype == torch.bfloat16 and w_proj.dtype == torch.bfloat16):
        return False
    if b_fc is None or _act_code(act) not in (ACT_GELU, ACT_RELU) or not _ext.have_C():
        return False
    tokens = x.numel() // x.shape[-1]
    hidden, out = w_fc.shape[0], w_proj.shape[0]
    # the fused epilogue lives in the 256x256-tile kernel: whole tiles only
    return bool(_ext.C().dgrad_act_backward_supported(tokens, hidden, out)) and w_proj.is_contiguous() and w_fc.is_contiguous()


def fused_mlp(x: torch.Tensor, w_fc: torch.Tensor, b_fc: Optional[torch.Tensor], w_proj: torch.Tensor,
              b_proj: Optional[torch.Tensor], act="gelu", impl: str = "native") -> torch.Tensor:
    """``act(x @ w_fc.T + b_fc) @ w_proj.T (+ b_proj)`` for x of shape ``[..., K]``.

    Falls back to the two separate linear ops when the shapes do not fill whole 256x256 tiles or the
    tensors are not bf16 on the GPU.
    """
    code = _act_code(act)
    if not fused_mlp_supported(x, w_fc, b_fc, w_proj, code):
        if x.is_cuda:
            return linear_bias_act(linear_bias_act(x, w_fc, b_fc, code), w_proj, b_proj, None)
        return F.linear(_torch_act(F.linear(x, w_fc, b_fc), code), w_proj, b_proj)
    lead = x.shape[:-1]
    x2 = x.reshape(-1, x.shape[-1])
    x2 = x2 if x2.is_contiguous() else x2.contiguous()
    y = _FusedMLP.apply(x2, w_fc, b_fc, w_proj, b_proj, code, impl)
    return y.reshape(*lead, w_proj.shape[0])


_GATES = {"relu": ACT_RELU, "gelu": ACT_GELU, "silu": ACT_SILU}


class _GatedMLP(torch.autograd.Function):
    """The activation and its slope are taken from g | u as they are stored, in 32 bits; the forward's h from the values before that
    rounding.  h is kept for dW_proj rather than computed again: it costs M H elements next to the 2 M H of g | u."""

    @staticmethod
    def forward(ctx, x2, w_fc, b_fc, w_proj, b_proj, act: int):
        C = _ext.C()
        h, gu = C.gated_forward(x2, w_fc, b_fc, act, True)
        y, _ = C.linear_forward(h, w_proj, b_proj, 0, False, True)
        ctx.save_for_backward(x2, w_fc, w_proj, gu, h)
        ctx.act = act
        ctx.biases = (b_fc is not None, b_proj is not None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        C = _ext.C()
        x2, w_fc, w_proj, gu, h = ctx.saved_tensors
        dy = dy.contiguous()
        need = ctx.needs_input_grad
        has_fc, has_proj = ctx.biases
        dx = dw_fc = db_fc = dw_proj = db_proj = None
        # (a frozen weight changes nothing but its own gradient: the others come from the same kernels)
        if need[3] or (has_proj and need[4]):
            _, dw_proj, db_proj = C.linear_backward(dy, h, w_proj, False, has_proj and need[4], _sink(w_proj) if need[3] else None, True, need[3])
        if need[0] or need[1] or need[2]:
            dgu, db_fc = C.gated_backward(dy, w_proj, gu, ctx.act, has_fc and need[2])
            if need[0] or need[1]:
                dx, dw_fc, _ = C.linear_backward(dgu, x2, w_fc, need[0], False, _sink(w_fc) if need[1] else None, True, need[1])
        return dx, dw_fc, db_fc, dw_proj, db_proj, None


def _sink(weight: torch.Tensor) -> Optional[torch.Tensor]:
    """The parameter's gradient-bucket slice, where the data-parallel wrapper offers one that fits."""
    out = weight_grad_buffer(weight)
    return out if out is not None and out.shape == weight.shape and out.dtype == weight.dtype else None


def _aligned(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Contiguous, on a 16-byte boundary (a view into a larger tensor may start anywhere)."""
    if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def gated_mlp(x: torch.Tensor, w_fc: torch.Tensor, b_fc: Optional[torch.Tensor], w_proj: torch.Tensor, b_proj: Optional[torch.Tensor],
              act: str = "silu") -> torch.Tensor:
    """``(act(x @ w_g.T + b_g) * (x @ w_u.T + b_u)) @ w_proj.T + b_proj`` for x of shape ``[..., K]``, where ``w_fc`` [2*H, K] holds the
    rows of ``w_g`` before those of ``w_u`` (``b_fc`` [2*H] likewise) and ``w_proj`` is [N, H].  act: silu | gelu | relu.

    bf16, fp16 and fp32 of any extents run on the native kernels on the GPU; all tensors share one dtype and device.
    """
    code = _GATES.get(act)
    if code is None:
        raise ValueError(f"unknown gate activation {act!r} (silu | gelu | relu)")
    grad = is_differentiated(x, w_fc, b_fc, w_proj, b_proj)
    if x.is_cuda and not grad:
        y = _ext.C().gated_mlp_forward(x, w_fc, b_fc, w_proj, b_proj, code)
        if y is not None:
            return y
    if w_fc.dim() != 2 or w_proj.dim() != 2 or w_fc.shape[0] % 2 or w_fc.shape[0] == 0 or w_proj.shape[1] * 2 != w_fc.shape[0]:
        raise ValueError(f"w_fc must be [2 * H, K] and w_proj [N, H], got {tuple(w_fc.shape)} and {tuple(w_proj.shape)}")
    if x.dim() < 1 or x.shape[-1] != w_fc.shape[1] or w_fc.shape[1] == 0 or w_proj.shape[0] == 0:
        raise ValueError(f"x {tuple(x.shape)} does not fit w_fc {tuple(w_fc.shape)} and w_proj {tuple(w_proj.shape)}")
    for name, b, n in (("b_fc", b_fc, w_fc.shape[0]), ("b_proj", b_proj, w_proj.shape[0])):
        if b is not None and b.shape != (n,):
            raise ValueError(f"{name} must be [{n}], got {tuple(b.shape)}")
    for name, t in (("w_fc", w_fc), ("b_fc", b_fc), ("w_proj", w_proj), ("b_proj", b_proj)):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise ValueError(f"{name} is {t.dtype} on {t.device}, x is {x.dtype} on {x.device}")
    H = w_proj.shape[1]
    if not x.is_cuda or x.numel() == 0:  # (no rows: nothing to launch)
        gu = F.linear(x, w_fc, b_fc)
        gate = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu}[act]
        return F.linear(gate(gu[..., :H]) * gu[..., H:], w_proj, b_proj)
    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise RuntimeError(f"gated_mlp: no native kernel for {x.dtype}")
    x2 = _aligned(x.reshape(-1, x.shape[-1]))
    tensors = [_aligned(t) for t in (w_fc, b_fc, w_proj, b_proj)]
    if grad:
        y = _GatedMLP.apply(x2, *tensors, code)
    else:
        y = _ext.C().gated_mlp_forward(x2, *tensors, code)
    return y.reshape(*x.shape[:-1], w_proj.shape[0])
