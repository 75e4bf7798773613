"""Keys that weigh little beside a dominant one, or because there are many of them: fp16's range is enough for their probabilities."""
import math

import pytest
import torch

import lv_xattn_b200 as lvx

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)


def check(got, want, eps):
    """Off by eps in all, and in fp16 by half a step of its subnormal values in each place: a result below 2^-14 is a multiple of 2^-24,
    so that its own rounding alone is off by up to 2^-25, which for gradients of 1e-6 is more than eps of them."""
    tiny = 2.0 ** -25 * want.numel() ** 0.5 if got.dtype == torch.float16 else 0.0
    off = (got.double() - want).norm().item()
    assert off <= eps * want.norm().item() + tiny, (off / want.norm().item(), tiny / want.norm().item())


def dominated(device, dtype, B, heads, Sq, Skv, at, below):
    """q, k, v, dO: key `at`, whose value is zero, outweighs every other one by 2^below."""
    gen = torch.Generator(device=device).manual_seed(77)
    r = lambda *s: torch.empty(s, device=device).normal_(0, 0.5, generator=gen)
    q = torch.zeros(B, heads[0], Sq, 128, device=device, dtype=dtype)
    q[..., 0] = 10
    k, v = r(B, heads[1], Skv, 128).to(dtype), (1 + r(B, heads[1], Skv, 128)).to(dtype)
    k[..., 0] = 0
    k[:, :, at, 0] = below * math.log(2.0) / SCALE / 10
    v[:, :, at] = 0
    return q, k, v, r(B, heads[0], Sq, 128).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("below", [18.3, 25.5])
@pytest.mark.parametrize("at", [0, 3])
@pytest.mark.parametrize("gain", [1, 4096])      # of dO: with 4,096 the gradients are not subnormal
@pytest.mark.parametrize("B,heads,Sq,Skv,window,sinks", [
    (2, (8, 2), 1, 6000, None, 0), (1, (8, 2), 4, 3000, 500, 4), (1, (4, 1), 20, 9000, None, 0), (1, (4, 2), 200, 2000, None, 0),
    (2, (16, 8), 300, 1000, 600, 4)])
def test_beside_a_dominant_key(cuda_device, B, heads, Sq, Skv, window, sinks, gain, at, below, dtype):
    """Single tokens, a few, query tiles, with a window and a dominant sink. P keeps all bits of the smaller probabilities (2^-25.5 of
    the maximum is above what SoftmaxRef gives up), so O errs by the roundings of P and O: half a step each at most."""
    q, k, v, do = dominated(cuda_device, dtype, B, heads, Sq, Skv, at, below)
    do = do * gain
    pos = Skv - Sq + torch.arange(Sq, device=cuda_device)[:, None]
    j = torch.arange(Skv, device=cuda_device)
    seen = (j <= pos) if window is None else (j <= pos) & ((j > pos - window) | (j < sinks))
    g = heads[0] // heads[1]
    kk, vv = (t.double().repeat_interleave(g, 1) for t in (k, v))
    s = (q.double() @ kk.mT * SCALE).masked_fill(~seen, -math.inf)
    p = s.softmax(-1)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o, lse = lvx.window_attention(*leaves, window=window, sinks=sinks, return_lse=True)
    eps = torch.finfo(dtype).eps
    check(o.detach(), p @ vv, eps)
    assert (lse.view(s.shape[:3]).double() - s.logsumexp(-1)).abs().max() <= 1e-4
    (dv,) = torch.autograd.grad(o, leaves[2:], do)
    want = (p.mT @ do.double()).view(B, heads[1], g, Skv, 128).sum(2)
    others = j != at
    check(dv[:, :, others], want[:, :, others], eps)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("below", [18.3, 25.5])
@pytest.mark.parametrize("Sq", [1, 5, 60])
def test_a_dominant_key_of_the_prefix(cuda_device, Sq, below, dtype):
    B, N, own = 6, 5000, 64
    q, pk, pv, do = dominated(cuda_device, dtype, 1, (8, 2), Sq, N, 0, below)
    q, do = (t.expand(B, -1, -1, -1).contiguous() for t in (q, do))
    _, k, v, _ = dominated(cuda_device, dtype, B, (8, 2), 1, own, 0, 0.0)
    pos = own - Sq + torch.arange(Sq, device=cuda_device)[:, None]
    seen = torch.cat([torch.ones(Sq, N, dtype=torch.bool, device=cuda_device), torch.arange(own, device=cuda_device) <= pos], 1)
    kk, vv = (torch.cat([a.expand(B, -1, -1, -1), b], 2).double().repeat_interleave(4, 1) for a, b in ((pk, k), (pv, v)))
    p = (q.double() @ kk.mT * SCALE).masked_fill(~seen, -math.inf).softmax(-1)
    leaves = [t.requires_grad_() for t in (q, pk, pv, k, v)]
    o = lvx.shared_prefix_attention(*leaves)
    eps = torch.finfo(dtype).eps
    check(o.detach(), p @ vv, eps)
    dpv, dv = torch.autograd.grad(o, [leaves[2], leaves[4]], do)
    want = (p.mT @ do.double()).view(B, 2, 4, N + own, 128).sum(2)
    check(dpv[0, :, 1:], want[:, :, 1:N].sum(0), eps)
    check(dv, want[:, :, N:], eps)


def test_many_keys(cuda_device):
    """Training behind 100,000 keys in fp16: their probabilities are around 2^-17. The values' gradients err by the roundings of P and of
    themselves, half a step each at most."""
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    r = lambda *s: torch.empty(s, device=cuda_device, dtype=torch.float16).normal_(generator=gen)
    B, N, Sq = 2, 100000, 20
    q, pk, pv, k, v, do = r(B, 4, Sq, 128), r(1, 2, N, 128), r(1, 2, N, 128), r(B, 2, Sq, 128), r(B, 2, Sq, 128), r(B, 4, Sq, 128)
    leaves = [t.requires_grad_() for t in (q, pk, pv, k, v)]
    dpv, dv = torch.autograd.grad(lvx.shared_prefix_attention(*leaves), [leaves[2], leaves[4]], do)
    seen = torch.cat([torch.ones(Sq, N, dtype=torch.bool, device=cuda_device), torch.ones(Sq, Sq, dtype=torch.bool, device=cuda_device).tril()], 1)
    kk = torch.cat([pk.expand(B, -1, -1, -1), k], 2).double().repeat_interleave(2, 1)
    p = (q.double() @ kk.mT * SCALE).masked_fill(~seen, -math.inf).softmax(-1)
    want = (p.mT @ do.double()).view(B, 2, 2, N + Sq, 128).sum(2)
    eps = torch.finfo(torch.float16).eps
    check(dpv[0], want[:, :, :N].sum(0), eps)
    check(dv, want[:, :, N:], eps)
