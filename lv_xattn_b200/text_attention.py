"""Attention of the text tokens on one GPU: causal, with a sliding window and sinks.

The reference's text layers gather K/V over the group and call torch's scaled_dot_product_attention with a dense causal mask
(test_llama3.py:313-340). Here only the keys that a query sees are read and multiplied, forward, backward and for the
single tokens of a generation. The layouts are those of `attention`: q [B, Hq, Sq, 128], k and v [B, Hkv, Skv, 128].
"""
from __future__ import annotations

import math
import operator

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .rotary import on_device, refuse_forward_mode, refuse_gradient, watch_status

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_MOST = 1 << 28          # lengths and positions are below this


def _check_q(who, q):
    shape, dtype = q.shape, q.dtype
    if len(shape) != 4 or shape[3] != 128:
        raise ValueError(f"{who}: q must be [batch, heads, tokens, 128], got {tuple(shape)}")
    if dtype not in _TYPES:
        raise ValueError(f"{who}: dtype {dtype} unsupported; expected bfloat16, float16 or float32")
    if 0 in shape:
        raise ValueError(f"{who}: q is empty, {tuple(shape)}")
    if shape[2] >= _MOST:
        raise ValueError(f"{who}: lengths must be below {_MOST}")
    return shape, dtype


def _check_kv(who, name, k, v, q_heads, dtype):
    """The shape of keys and values, which `name` calls them."""
    shape = k.shape
    if len(shape) != 4 or shape[3] != 128 or shape != v.shape:
        raise ValueError(f"{who}: {name} must be two tensors [batch, KV heads, keys, 128] of one shape, got {tuple(shape)} and {tuple(v.shape)}")
    if k.dtype != dtype or v.dtype != dtype:
        raise ValueError(f"{who}: q and {name} must share one dtype")
    if shape[1] == 0 or q_heads % shape[1]:
        raise ValueError(f"{who}: {q_heads} query heads are not a multiple of the {shape[1]} heads of {name}")
    if shape[2] >= _MOST:
        raise ValueError(f"{who}: lengths must be below {_MOST}")
    return shape


def _check_devices(who, q, *kv):
    device = q.device
    for t in kv:
        if t.device != device:
            raise ValueError(f"{who}: all tensors must be on one device")
    if not q.is_cuda:
        raise _lib.LvxError("lv_xattn_b200 runs on CUDA tensors only; there is no CPU path")
    return device


def _scale(who, sm_scale):
    if sm_scale is None:
        return 128 ** -0.5
    if type(sm_scale) is not float:
        refuse_gradient(who, "sm_scale", sm_scale)
    if not (sm_scale > 0 and math.isfinite(sm_scale)):
        raise ValueError(f"{who}: sm_scale must be positive and finite")
    return float(sm_scale)


def whole_number(who, name, n):
    """n, an integer of any kind, as an int."""
    try:
        return operator.index(n)
    except TypeError:
        raise ValueError(f"{who}: {name} must be an integer, got {n!r}") from None


class WindowAttentionFunc(torch.autograd.Function):
    """(q, k, v, sm_scale, window, sinks, query_start, kv_valid_len on the device) -> (o, lse)."""

    @staticmethod
    def forward(ctx, q, k, v, sm_scale, window, sinks, query_start, kv_valid_len):
        o, lse, low = ops.window_forward(q, k, v, sm_scale, window, sinks, query_start, kv_valid_len, True,
                                         ops.window_low_rows(q, k, query_start, kv_valid_len))
        ctx.save_for_backward(q, k, v, o, low, lse, kv_valid_len)
        ctx.args = sm_scale, window, sinks, query_start
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, do, _):
        if do is None:
            return (None,) * 8
        q, k, v, o, low, lse, kv_valid_len = ctx.saved_tensors
        with on_device(q):
            grads = ops.window_backward(do, q, k, v, o, low, lse, *ctx.args, kv_valid_len)
        return (*(g if want else None for g, want in zip(grads, ctx.needs_input_grad)), None, None, None, None, None)


def window_attention(q, k, v, sm_scale=None, window=None, sinks=0, kv_valid_len=None, query_start=None, return_lse=False):
    """Causal attention with a sliding window and sinks: o like q, dense; with `return_lse` also the log-sum-exp of every
    row's scores, fp32 [B*Hq, Sq] (no gradient flows through it).

    q [B, Hq, Sq, 128], k and v [B, Hkv, Skv, 128] in bf16, fp16 or fp32, Hq a multiple of Hkv, any strides. Query i of
    batch entry b sits at position p = query_start + i, or, where that is None, p = n_b - Sq + i: the last query on the last
    of the entry's n_b valid keys, as the newest tokens of a generation do. It sees key j iff j < n_b, j <= p, and j > p -
    window or j < sinks. window None: all keys behind it. kv_valid_len: n_b, one integer per entry (a list, or a tensor on
    the host or the device; values are taken into 0..Skv), None: Skv. Keys from n_b on are never looked at, whatever they
    hold: a cache may be longer than what has been written. A query that sees nothing gets zeros, and -inf in the
    log-sum-exp. In the forward a key that a query does not see has no effect on it, whatever it holds; a NaN
    in the query or in a key that it sees is NaN in both results, and one in a value in o. In the backward q, the valid keys and the
    gradient of o have to be finite (NaN reaches more of the gradients).
    sm_scale scales the scores (None: 1 / sqrt(128)). Gradients flow into q, k and v; no second and no forward-mode derivatives."""
    who = "window_attention"
    refuse_forward_mode(who, q, k, v)
    sm_scale = _scale(who, sm_scale)
    sinks = whole_number(who, "sinks", sinks)
    if window is not None:
        window = whole_number(who, "window", window)
    if query_start is not None:
        query_start = whole_number(who, "query_start", query_start)
    if window is not None and window < 1:
        raise ValueError(f"{who}: window must be at least 1 (a query's own position), got {window}")
    if sinks < 0:
        raise ValueError(f"{who}: sinks must not be negative, got {sinks}")
    if query_start is not None and not 0 <= query_start < _MOST:
        raise ValueError(f"{who}: query_start must lie in 0..{_MOST - 1}, got {query_start}")
    q_shape, dtype = _check_q(who, q)
    k_shape = _check_kv(who, "k and v", k, v, q_shape[1], dtype)
    if k_shape[0] != q_shape[0]:
        raise ValueError(f"{who}: q has {q_shape[0]} batch entries, k and v {k_shape[0]}")
    device = _check_devices(who, q, k, v)
    with on_device(q):
        watch_status(q)
        lengths = ops.device_lengths(kv_valid_len, q_shape[0], k_shape[2], device)
        args = (q, k, v, sm_scale, 0 if window is None or window >= _MOST else window, min(sinks, _MOST),
                -1 if query_start is None else query_start, lengths)
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
            o, lse = WindowAttentionFunc.apply(*args)
        else:
            o, lse = ops.window_forward(*args)
    return (o, lse) if return_lse else o


class SharedPrefixAttentionFunc(torch.autograd.Function):
    """(q, k_prefix, v_prefix, k, v, sm_scale, prefix_valid_len, kv_valid_len, both on the device) -> (o, lse)."""

    @staticmethod
    def forward(ctx, q, pk, pv, k, v, sm_scale, prefix_valid_len, kv_valid_len):
        o, lse = ops.shared_forward(q, pk, pv, k, v, sm_scale, prefix_valid_len, kv_valid_len)
        ctx.save_for_backward(q, pk, pv, k, v, o, lse, prefix_valid_len, kv_valid_len)
        ctx.sm_scale = sm_scale
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, do, _):
        if do is None:
            return (None,) * 8
        q, pk, pv, k, v, o, lse, prefix_valid_len, kv_valid_len = ctx.saved_tensors
        with on_device(q):
            grads = ops.shared_backward(do, q, pk, pv, k, v, o, lse, ctx.sm_scale, prefix_valid_len, kv_valid_len)
        return (*(g if want else None for g, want in zip(grads, ctx.needs_input_grad)), None, None, None)


def shared_prefix_attention(q, k_prefix, v_prefix, k=None, v=None, sm_scale=None, prefix_valid_len=None, kv_valid_len=None,
                            return_lse=False):
    """Attention of a batch of requests that share a long prefix (the tokens of a video, of a system prompt), which is read
    once for all of them: o like q, dense; with `return_lse` also the log-sum-exp of every row's scores, fp32 [B*Hq, Sq].

    q [B, Hq, Sq, 128]; k_prefix and v_prefix [P, Hkv, N, 128], B a multiple of P: the first B / P requests share the first
    prefix, the next ones the second, and so on. k and v [B, Hkv, Skv, 128] are each request's own keys behind its prefix, or
    None. Every query sees the whole prefix, and own key j where j < n_b and j <= n_b - Sq + i: as in `window_attention`, the
    last query sits on the last of the n_b valid own keys. One softmax over both. bf16, fp16 or fp32, any strides.
    prefix_valid_len (P integers) and kv_valid_len (B integers), a list or a tensor on the host or the device: how many keys
    are valid; keys behind them are never looked at, whatever they hold. A query that sees nothing gets zeros, and -inf in
    the log-sum-exp. Gradients flow into q and all keys and values; those of a prefix are summed over its requests. No second and no
    forward-mode derivatives."""
    who = "shared_prefix_attention"
    refuse_forward_mode(who, q, k_prefix, v_prefix, k, v)
    sm_scale = _scale(who, sm_scale)
    if (k is None) != (v is None):
        raise ValueError(f"{who}: k and v go together")
    if k is None and kv_valid_len is not None:
        raise ValueError(f"{who}: valid lengths of own keys that are not there")
    q_shape, dtype = _check_q(who, q)
    B, P, _, N = q_shape[0], *_check_kv(who, "the prefix", k_prefix, v_prefix, q_shape[1], dtype)[:3]
    if P == 0 or B % P:
        raise ValueError(f"{who}: {B} requests are not a multiple of {P} prefixes")
    if N == 0:
        raise ValueError(f"{who}: the prefix is empty")
    if k is None:
        own = 0
        device = _check_devices(who, q, k_prefix, v_prefix)
    else:
        b, heads, own, _ = _check_kv(who, "k and v", k, v, q_shape[1], dtype)
        if b != B or heads != k_prefix.shape[1]:
            raise ValueError(f"{who}: own keys {tuple(k.shape)} for {B} requests and {k_prefix.shape[1]} KV heads")
        device = _check_devices(who, q, k_prefix, v_prefix, k, v)
    with on_device(q):
        watch_status(q)
        args = (q, k_prefix, v_prefix, k, v, sm_scale, ops.device_lengths(prefix_valid_len, P, N, device),
                ops.device_lengths(kv_valid_len, B, own, device))
        if torch.is_grad_enabled() and (q.requires_grad or k_prefix.requires_grad or v_prefix.requires_grad
                                        or (k is not None and (k.requires_grad or v.requires_grad))):
            o, lse = SharedPrefixAttentionFunc.apply(*args)
        else:
            o, lse = ops.shared_forward(*args)
    return (o, lse) if return_lse else o
