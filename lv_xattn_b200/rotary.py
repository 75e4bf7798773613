"""Head norms and the rotary embedding of a text layer's queries and keys, in one pass over them.

The reference's text layers run the norm, the rotation and the transposition into [B, H, S, D] as separate torch modules
(test_llama3.py:294-312 for the self-attention, :394-419 for the norms); here they are one kernel, which reads the
projections' output where it is and writes the layout that the attention kernels read.
"""
from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib, ops

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


_HERE = contextlib.nullcontext()


def on_device(t):
    """Makes t's device current for the duration of a call (kernels launch on the current device)."""
    return _HERE if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def watch_status(t):
    """Start of a call, with t's device current: raises if a kernel of an earlier call gave up on a bounded wait (see
    peer_memory.StatusWatch)."""
    from .peer_memory import status_watch
    status_watch.watch(t.device.index)


def refuse_forward_mode(who, *tensors):
    """The kernels make no tangents, and a tensor that carries one does not require a gradient: it would be lost without a word."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{who}: forward-mode derivatives are not supported")


def refuse_gradient(who, name, t):
    """For arguments that no gradient flows into."""
    if torch.is_grad_enabled() and torch.is_tensor(t) and t.requires_grad:
        raise ValueError(f"{who}: no gradient flows into {name}: detach")


def _check(q, k, q_weight, k_weight, cos, sin, eps):
    like = q if q is not None else k
    if like is None:
        raise ValueError("head_norm_rope: q or k must be given")
    dtype, device = like.dtype, like.device
    for t in (q, k):
        if t is not None and (t.dim() != 4 or t.shape[3] != 128):
            raise ValueError(f"head_norm_rope: q and k must be [batch, tokens, heads, 128], got {tuple(t.shape)}")
    if dtype not in _TYPES:
        raise ValueError(f"head_norm_rope: dtype {dtype} unsupported; expected bfloat16, float16 or float32")
    B, S = like.shape[:2]
    if q is not None and k is not None and (k.dtype != dtype or k.shape[:2] != (B, S)):
        raise ValueError("head_norm_rope: q and k must agree on dtype, batch and tokens")
    if (q is None and q_weight is not None) or (k is None and k_weight is not None):
        raise ValueError("head_norm_rope: a weight without the tensor that it scales")
    weight = q_weight if q_weight is not None else k_weight
    if weight is not None:
        kind = weight.dtype
        for w in (q_weight, k_weight):
            if w is not None and (w.shape != (128,) or (kind != dtype and kind != torch.float32) or w.dtype != kind):
                raise ValueError("head_norm_rope: weights must be [128], both fp32 or both in the dtype of q and k")
    if (cos is None) != (sin is None):
        raise ValueError("head_norm_rope: cos and sin go together")
    if cos is not None:
        if cos.requires_grad or sin.requires_grad:
            refuse_gradient("head_norm_rope", "cos and sin", cos if cos.requires_grad else sin)
        shape, kind = cos.shape, cos.dtype
        if sin.shape != shape or not (shape == (B, S, 128) or shape == (S, 128) or shape == (1, S, 128)):
            raise ValueError(f"head_norm_rope: cos and sin must be [{S}, 128] or [1 or {B}, {S}, 128], got {tuple(cos.shape)} and {tuple(sin.shape)}")
        if sin.dtype != kind or (kind != dtype and kind != torch.float32):
            raise ValueError("head_norm_rope: cos and sin must be fp32 or in the dtype of q and k")
    elif weight is None:
        raise ValueError("head_norm_rope: neither a weight nor cos and sin: nothing to do")
    if not eps >= 0:
        raise ValueError("head_norm_rope: eps must be non-negative")
    for t in (q, k, cos, sin, q_weight, k_weight):
        if t is not None and (t.device != device or not t.is_cuda):
            if not t.is_cuda:
                raise _lib.LvxError("lv_xattn_b200 runs on CUDA tensors only; there is no CPU path")
            raise ValueError("head_norm_rope: all tensors must be on one device")


def _rows(t):
    """A table or a weight as the kernel reads it: contiguous, 16-byte aligned rows (a copy where it is not so)."""
    if t is None:
        return None
    if t.dim() == 2:
        t = t[None]
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.contiguous().clone()


class HeadNormRopeFunc(torch.autograd.Function):
    """(q, k, q_weight, k_weight, cos, sin, eps) -> (q_out, k_out). Keeps its inputs for the backward, nothing else."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, eps):
        out = ops.head_norm_rope(q, k, q_weight, k_weight, cos, sin, eps)
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_weight, k_weight, cos, sin = ctx.saved_tensors
        want = list(ctx.needs_input_grad[:4])
        # an output that nothing used has no gradient, and neither have what it was made of
        if gq is None:
            q = q_weight = None
            want[0] = want[2] = False
        if gk is None:
            k = k_weight = None
            want[1] = want[3] = False
        if not any(want):
            return (None,) * 7
        with on_device(q if q is not None else k):
            grads = ops.head_norm_rope_bwd(q, k, q_weight, k_weight, cos, sin, ctx.eps, gq, gk, want)
        return (*grads, None, None, None)


def head_norm_rope(q, k, q_weight=None, k_weight=None, cos=None, sin=None, eps=1e-6):
    """Per-head RMSNorm and rotary embedding of queries and keys in one pass: (q_out, k_out), dense [B, H, S, 128].

    q [B, S, Hq, 128] and k [B, S, Hkv, 128] are the projections' outputs seen by head (any strides; either may be None),
    bf16, fp16 or fp32. q_weight and k_weight [128] scale the normalised heads (None: that tensor is not normalised). cos and
    sin [S, 128] or [1 or B, S, 128] are the rotary tables as Hugging Face models hand them to their layers, both halves of
    the 128 columns filled (None: no rotation). Computed in fp32 and rounded once. Gradients flow into q, k and the weights;
    the weights' are summed in a fixed order; none flow into cos and sin, which may not ask for one. No second and no forward-mode derivatives."""
    refuse_forward_mode("head_norm_rope", q, k, q_weight, k_weight, cos, sin)
    _check(q, k, q_weight, k_weight, cos, sin, eps)
    q_weight, k_weight, cos, sin = (_rows(t) for t in (q_weight, k_weight, cos, sin))
    like = q if q is not None else k
    args = (q, k, q_weight, k_weight, cos, sin, float(eps))
    with on_device(like):
        watch_status(like)
        if torch.is_grad_enabled() and ((q is not None and q.requires_grad) or (k is not None and k.requires_grad)
                                        or (q_weight is not None and q_weight.requires_grad)
                                        or (k_weight is not None and k_weight.requires_grad)):
            return HeadNormRopeFunc.apply(*args)
        return ops.head_norm_rope(*args)
