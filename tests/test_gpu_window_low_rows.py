"""What O's rounding drops, kept in as many rows as a call has early queries: the same values as by position, and no more memory."""
import pytest
import torch

import lv_xattn_b200 as lvx
from lv_xattn_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def normal(device, dtype, B, Hq, Hkv, Sq, Skv):
    gen = torch.Generator(device=device).manual_seed(Sq + Skv)
    return [torch.empty(B, h, n, 128, device=device, dtype=dtype).normal_(generator=gen) for h, n in ((Hq, Sq), (Hkv, Skv), (Hkv, Skv), (Hq, Sq))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths", [False, True])
@pytest.mark.parametrize("start", [None, 0, 200, 255])
@pytest.mark.parametrize("shape", [(3, 8, 2, 9, 9), (3, 8, 2, 1, 40), (2, 4, 4, 100, 160), (3, 8, 2, 100, 60), (2, 8, 2, 300, 300), (1, 4, 1, 30, 5000),
                                   (1, 4, 1, 200, 420)])
def test_same_as_by_position(cuda_device, shape, start, lengths, dtype):
    B, Hq, Hkv, Sq, Skv = shape
    q, k, v, do = normal(cuda_device, dtype, *shape)
    valid = [max(0, Skv - 17 * b) for b in range(B)]
    lens = torch.tensor(valid, device=cuda_device, dtype=torch.int32) if lengths else None
    args = (0.09, 0, 0, -1 if start is None else start, lens)
    n = ops.window_low_rows(q, k, args[3], lens)
    o, lse, low = ops.window_forward(q, k, v, *args, True)
    o1, lse1, few = ops.window_forward(q, k, v, *args, True, n)
    assert torch.equal(o, o1) and torch.equal(lse, lse1)
    if n == 0:
        assert low is None and few is None
        return
    assert few.shape == (B * Hq, n, 128)
    low, few = low.view(B, Hq, _lib.LOW_ROWS, 128), few.view(B, Hq, n, 128)
    for b in range(B):
        first = (valid[b] if lengths else Skv) - Sq if start is None else start
        for i in range(Sq):
            p = first + i
            if 0 <= p < _lib.LOW_ROWS:
                at = p if n == _lib.LOW_ROWS else p - max(0, first)
                assert torch.equal(low[b, :, p], few[b, :, at])
    grads = [ops.window_backward(do, q, k, v, o, t.view(B * Hq, -1, 128), lse, *args) for t in (low, few)]
    for a, b in zip(*(g[1:] for g in grads)):
        assert torch.equal(a, b)
    assert (grads[0][0].float() - grads[1][0].float()).abs().max() <= torch.finfo(dtype).eps * 2 * grads[0][0].float().abs().max()


@pytest.mark.parametrize("Sq,Skv,lengths", [(16, 16, False), (16, 16, True), (1, 1, False), (64, 64, True), (1000, 8192, False)])
def test_what_a_short_text_keeps(cuda_device, Sq, Skv, lengths):
    """Saved for the backward: q, k, v, O, the log-sum-exp, and of what was dropped at most as much as O."""
    B = 32
    q, k, v, _ = (t.requires_grad_() for t in normal(cuda_device, torch.bfloat16, B, 8, 2, Sq, Skv))
    saved = {}

    def pack(t):
        saved[t.data_ptr()] = t.numel() * t.element_size()
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        o = lvx.window_attention(q, k, v, kv_valid_len=[Skv] * B if lengths else None)
    size = lambda t: t.numel() * t.element_size()
    assert sum(saved.values()) <= size(q) + size(k) + size(v) + 2 * size(o) + B * 8 * Sq * 4 + B * 4
    if Skv > Sq:
        assert sum(saved.values()) <= size(q) + size(k) + size(v) + size(o) + B * 8 * Sq * 4
