"""Gradients of the text attention in 16 bits: what the kernels round besides the result, and no more.

A rounding to a type whose step is u = finfo.eps relative to a power of two is off by a uniform error of at most half a step, and
relative to a value whose logarithm is spread evenly its root mean square is u / 2 / sqrt(3) * sqrt(3 / (8 ln 2)) = 0.2123 u. A gradient
is rounded when it is stored and made of products whose dS was rounded: sqrt(2) of that. P's rounding reaches it through O and
delta: an error of each P_ij times dP_ij, summed over a row and given back to the row in proportion to P, so its square is that
of one rounding times the sum of the row's squared P, at most 1. Together at most sqrt(3) times one rounding. O's own rounding adds
the same once more where rows see few keys, unless delta is made from O in two parts.
"""
import math

import pytest
import torch

from lv_xattn_b200 import ops

pytestmark = pytest.mark.gpu


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


def exact(q, k, v, do):
    q, k, v = (t.double().requires_grad_() for t in (q, k, v))
    S, g = q.shape[2], q.shape[1] // k.shape[1]
    s = q @ k.repeat_interleave(g, 1).mT / math.sqrt(128)
    s = s.masked_fill(~torch.ones(S, S, dtype=torch.bool, device=q.device).tril(), float("-inf"))
    return torch.autograd.grad(s.softmax(-1) @ v.repeat_interleave(g, 1), (q, k, v), do.double())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S", [16, 40, 300])
def test_short_texts(cuda_device, S, dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(S)
    B = max(2, 1000 // S)
    q, k, v, do = (torch.empty(B, h, S, 128, device=cuda_device, dtype=dtype).normal_(generator=gen) for h in (8, 2, 2, 8))
    args = (128 ** -0.5, 0, 0, -1, None)
    ref = exact(q, k, v, do)
    o, lse, low = ops.window_forward(q, k, v, *args, True)
    one = torch.finfo(dtype).eps * 0.2123
    parts = [rel(t, r) for t, r in zip(ops.window_backward(do, q, k, v, o, low, lse, *args), ref)]
    rounded = [rel(t, r) for t, r in zip(ops.window_backward(do, q, k, v, o, None, lse, *args), ref)]
    assert max(parts) < math.sqrt(3) * one, (parts, one)
    assert parts[0] < rounded[0] and parts[1] < rounded[1], (parts, rounded)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(2, 8, 2, 300, 300), (3, 8, 2, 100, 160), (2, 32, 8, 9, 9), (1, 4, 4, 500, 500)])
@pytest.mark.parametrize("start", [None, 0, 200])
def test_dropped_part(cuda_device, shape, dtype, start):
    """O and its dropped part are together O to fp32's place, by the kernel that makes O itself and by the one that merges parts of
    it, for the rows at early positions; other places are left as they were."""
    B, Hq, Hkv, Sq, Skv = shape
    gen = torch.Generator(device=cuda_device).manual_seed(Skv)
    q, k, v = (torch.empty(B, h, n, 128, device=cuda_device, dtype=dtype).normal_(generator=gen) for h, n in ((Hq, Sq), (Hkv, Skv), (Hkv, Skv)))
    valid = [Skv - 7 * b for b in range(B)]
    lengths = torch.tensor(valid, device=cuda_device, dtype=torch.int32)
    args = (0.1, 0, 0, -1 if start is None else start, lengths)
    real = q.new_empty
    q.new_empty = lambda shape, **kw: real(shape, **kw).fill_(float("nan"))      # (what the call allocates)
    o, lse, low = ops.window_forward(q, k, v, *args, True)
    del q.new_empty
    o1, lse1 = ops.window_forward(q, k, v, *args)
    assert torch.equal(o, o1) and torch.equal(lse, lse1)
    eps = torch.finfo(dtype).eps
    low = low.view(B, Hq, 256, 128)
    pos = torch.stack([torch.arange(Sq) + (n - Sq if start is None else start) for n in valid])      # [B, Sq]
    kept = torch.zeros(B, 256, dtype=torch.bool)
    for b in range(B):
        kept[b, pos[b][(pos[b] >= 0) & (pos[b] < 256)]] = True
        for i in range(0, Sq, 13):
            p = int(pos[b, i])
            if 0 <= p < 256:
                half = eps / 2 * o[b, :, i].double().abs() * (1 + eps) + eps * torch.finfo(dtype).smallest_normal
                assert (low[b, :, p].double().abs() <= half).all()
                n = min(p + 1, valid[b])
                if n > 1:      # (one key: O is its V, of which nothing is dropped)
                    assert low[b, :, p].count_nonzero() > 0.9 * Hq * 128
                # without the rounding of P for its product nothing but fp32 rounding would be between the two
                kk, vv = (t[b, :, :n].double().repeat_interleave(Hq // Hkv, 0) for t in (k, v))
                P = (torch.einsum("hd,hnd->hn", q[b, :, i].double(), kk) * 0.1).softmax(-1)
                bound = eps / 2 * torch.einsum("hn,hnd->hd", P, vv.abs()) * 1.01
                assert ((o[b, :, i].double() + low[b, :, p].double() - torch.einsum("hn,hnd->hd", P, vv)).abs() <= bound + 1e-5).all()
    assert (low.isnan().any(-1).all(1).cpu() == ~kept).all()
