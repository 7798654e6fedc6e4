"""Causal self-attention with a sliding window and sinks on a packed q|k|v projection.

Query i of a sequence sees key j when ``j <= i`` and either ``i - j < window`` or ``j < sinks``: the last ``window`` positions
(its own among them) and the first ``sinks`` ones, which stay visible to everybody.  Beside ``causal_attention_qkvpacked`` it
also takes key / value heads that several query heads share, padded batches, fp16 and head size 128.

The packed layout is [B, T, (n_head + 2 * n_kv_head) * D]: the query heads, the key heads, the value heads; query head h reads
key / value head ``h // (n_head // n_kv_head)``.  On gfx950 the forward and backward are hand-written kernels that visit only
the tiles the window and the sinks reach (bf16 / fp16, head size 64 or 128, any length); rows may be strided.  Other types,
head sizes and CPU tensors run a composition of stock operators with an explicit mask.

The reference contains no attention (its model is two linear layers, reference min_DDP.py:41-49).
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _ext
from .tangents import is_differentiated

_NAMES = {torch.bfloat16: "bfloat16", torch.float16: "float16"}


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, cfg, lens):
        o, lse2 = _ext.C().window_attention_forward(qkv, *cfg, lens, True)
        ctx.save_for_backward(qkv, o, lse2, lens)
        ctx.cfg = cfg
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o):
        qkv, o, lse2, lens = ctx.saved_tensors
        if not (d_o.is_contiguous() and d_o.data_ptr() % 16 == 0):
            d_o = d_o.clone(memory_format=torch.contiguous_format)
        return _ext.C().window_attention_backward(d_o, qkv, o, lse2, *ctx.cfg, lens), None, None


def _native_layout(qkv: torch.Tensor) -> bool:
    """Contiguous rows that start on 16-byte boundaries, at any distance from one another."""
    if qkv.stride(2) != 1 or qkv.data_ptr() % 16:
        return False
    B, T, W = qkv.shape
    return (T <= 1 or (qkv.stride(1) >= W and qkv.stride(1) % 8 == 0)) and (B <= 1 or (qkv.stride(0) >= 0 and qkv.stride(0) % 8 == 0))


def native_window_attention_supported(qkv: torch.Tensor, n_head: int, n_kv_head: int, layout: Optional[bool] = None) -> bool:
    """True when the kernels take ``qkv`` (after a copy, where its rows are not contiguous and aligned).  layout: ``_native_layout(qkv)``, where
    it is known."""
    name = _NAMES.get(qkv.dtype)
    if name is None or not qkv.is_cuda or not _ext.have_C():
        return False
    B, T, W = qkv.shape
    stride = qkv.stride(1) if T > 1 and (_native_layout(qkv) if layout is None else layout) else W
    return bool(_ext.C().window_attention_supported(B, T, n_head, n_kv_head, W // (n_head + 2 * n_kv_head), stride, name))


def _composed(qkv, n_head, n_kv_head, window, sinks, scale, lens):
    B, T, W = qkv.shape
    D, G = W // (n_head + 2 * n_kv_head), n_head // n_kv_head
    work = qkv.dtype if qkv.dtype in (torch.float32, torch.float64) else torch.float32
    x = qkv.to(work).reshape(B, T, n_head + 2 * n_kv_head, D).transpose(1, 2)
    i = torch.arange(T, device=qkv.device)
    ok = (i[None, :] <= i[:, None]) & ((i[:, None] - i[None, :] < window) | (i[None, :] < sinks))
    live = torch.ones(B, T, dtype=torch.bool, device=qkv.device) if lens is None else i[None, :] < lens[:, None]
    x = torch.where(live[:, None, :, None], x, x.new_zeros(()))  # rows behind a sequence may hold anything
    q = x[:, :n_head]
    k = x[:, n_head:n_head + n_kv_head].repeat_interleave(G, 1)
    v = x[:, n_head + n_kv_head:].repeat_interleave(G, 1)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    p = torch.softmax(s.masked_fill(~ok, float("-inf")), 3)  # (a row always sees itself)
    o = torch.matmul(p, v) * live[:, None, :, None]
    return o.transpose(1, 2).reshape(B, T, n_head * D).to(qkv.dtype)


def window_attention_qkvpacked(qkv: torch.Tensor, n_head: int, window: int, sinks: int = 0, n_kv_head: Optional[int] = None,
                               seq_lens: Optional[torch.Tensor] = None, softmax_scale: Optional[float] = None,
                               impl: str = "auto") -> torch.Tensor:
    """qkv: [B, T, (n_head + 2 * n_kv_head) * D] -> [B, T, n_head * D]; see the module's description.

    ``n_kv_head`` defaults to ``n_head``.  ``seq_lens`` ([B], int32 or int64, on the device of ``qkv``) gives the lengths of a
    padded batch, taken into 0 .. T: positions behind a sequence are never looked at, their outputs and gradients are zero.
    ``softmax_scale`` (1e-30 .. 1e30) defaults to D ** -0.5.  impl: "auto", "native" (raise where the kernels do not apply), "composed".
    A NaN or infinity at a position of a sequence reaches the queries that see it, and may reach others within 128 positions
    of those.  Scaled scores are taken to stay below 2 ** 24 in size, beyond which float32 tells no neighbouring ones apart.
    """
    if impl not in ("auto", "native", "composed"):
        raise ValueError(f"impl must be auto | native | composed, got {impl}")
    if qkv.dim() != 3:
        raise ValueError(f"qkv must be [B, T, heads * head_dim], got {tuple(qkv.shape)}")
    n_kv = n_head if n_kv_head is None else int(n_kv_head)
    if n_head < 1 or n_kv < 1 or n_head % n_kv:
        raise ValueError(f"n_head ({n_head}) must be a positive multiple of n_kv_head ({n_kv})")
    W, heads = qkv.shape[2], n_head + 2 * n_kv
    if W == 0 or W % heads:
        raise ValueError(f"the last dimension ({W}) must be (n_head + 2 * n_kv_head) * head_dim with {heads} heads")
    if window < 1 or sinks < 0:
        raise ValueError(f"window must be at least 1 and sinks at least 0, got {window} and {sinks}")
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(W // heads)
    if not 1e-30 <= scale <= 1e30:  # (in float32 neither zero nor infinite, times log2(e) either)
        raise ValueError(f"softmax_scale must lie in 1e-30 .. 1e30, got {scale}")
    lens = seq_lens
    if lens is not None:
        if lens.shape != (qkv.shape[0],) or lens.dtype not in (torch.int32, torch.int64) or lens.device != qkv.device:
            raise ValueError(f"seq_lens must be int32 or int64 [{qkv.shape[0]}] on {qkv.device}, got {lens.dtype} {tuple(lens.shape)} on {lens.device}")
    if impl != "composed":
        if torch.is_autocast_enabled() and qkv.is_cuda and qkv.dtype not in _NAMES:
            qkv = qkv.to(torch.get_autocast_dtype("cuda"))
        layout = _native_layout(qkv)
        if native_window_attention_supported(qkv, n_head, n_kv, layout):
            if not layout:
                qkv = qkv.clone(memory_format=torch.contiguous_format)
            if lens is not None:
                lens = (lens if lens.dtype == torch.int32 else lens.clamp(0, qkv.shape[1]).to(torch.int32)).contiguous()
            cfg = (n_head, n_kv, int(window), int(sinks), scale)
            if not is_differentiated(qkv):
                return _ext.C().window_attention_forward(qkv, *cfg, lens, False)[0]
            return _WindowAttention.apply(qkv, cfg, lens)
        if impl == "native":
            raise RuntimeError(f"native window attention does not cover qkv {tuple(qkv.shape)} {qkv.dtype} on {qkv.device} with {n_head} / {n_kv} heads "
                               "(needs bf16 or fp16 and head size 64 or 128)")
    if qkv.shape[0] == 0 or qkv.shape[1] == 0:
        return qkv[..., : n_head * (W // heads)].clone()
    return _composed(qkv, n_head, n_kv, window, sinks, scale, lens)
