"""Few query rows whose keys one CTA walks alone, and what a NaN inside does, in every form that a call can take."""
import math

import pytest
import torch

import lv_xattn_b200 as lvx

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def inputs(device, B, Hq, Hkv, Sq, Skv, dtype, seed):
    gen = torch.Generator(device=device).manual_seed(seed)
    return [torch.empty(B, h, n, 128, device=device, dtype=dtype).normal_(generator=gen) for h, n in ((Hq, Sq), (Hkv, Skv), (Hkv, Skv))]


def seen(Sq, Skv, valid, window, sinks, device):
    pos = torch.tensor(valid, device=device)[:, None, None] - Sq + torch.arange(Sq, device=device)[None, :, None]
    j = torch.arange(Skv, device=device)[None, None]
    m = (j <= pos) & (j < torch.tensor(valid, device=device)[:, None, None])
    return (m if window is None else m & ((j > pos - window) | (j < sinks)))[:, None]


def exact(q, k, v, m):
    g = q.shape[1] // k.shape[1]
    s = (q.double() @ k.double().repeat_interleave(g, 1).mT / math.sqrt(128)).masked_fill(~m, float("-inf"))
    return s.softmax(-1).masked_fill(~m, 0.0).nan_to_num(0.0) @ v.double().repeat_interleave(g, 1), s.logsumexp(-1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", [(32, 8), (4, 4), (12, 2)])
@pytest.mark.parametrize("Sq,Skv,window,sinks", [(1, 1, None, 0), (1, 40, None, 0), (1, 128, 64, 4), (5, 129, None, 0), (3, 200, 1, 0), (8, 256, 100, 130)])
def test_one_walk(cuda_device, Sq, Skv, window, sinks, heads, dtype):
    q, k, v = inputs(cuda_device, 20, *heads, Sq, Skv, dtype, Skv)
    valid = [max(0, Skv - 13 * b) if b % 4 else Skv for b in range(20)]
    m = seen(Sq, Skv, valid, window, sinks, cuda_device)
    for b, n in enumerate(valid):      # never looked at
        k[b, :, n:] = float("nan")
        v[b, :, n:] = float("inf")
    o, lse = lvx.window_attention(q, k, v, window=window, sinks=sinks, kv_valid_len=valid, return_lse=True)
    dead = ~(torch.arange(Skv, device=cuda_device)[None, :] < torch.tensor(valid, device=cuda_device)[:, None])[:, None, :, None]
    ro, rl = exact(q, k.masked_fill(dead, 0), v.masked_fill(dead, 0), m)
    # P is rounded for its product and O when it is stored, each by half a step at most, against the largest |V| that enters
    eps = torch.finfo(dtype).eps if dtype != torch.float32 else 2.0 ** -18      # (three tf32 products: 2^-20 each, and the sums)
    assert ((o.double() - ro).abs() <= eps * 6).all() and o.isfinite().all()
    assert v.masked_fill(dead, 0).abs().max() < 6
    lse = lse.view(20, heads[0], Sq).double()
    empty = (~m.any(-1)).expand(20, heads[0], Sq)
    assert (lse[empty] == float("-inf")).all() and (o.permute(0, 1, 2, 3)[empty] == 0).all()
    assert ((lse - rl)[~empty].abs() < 1e-4).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,heads,Sq,Skv,window", [
    (20, (32, 8), 4, 100, None),        # one CTA a KV head
    (1, (8, 2), 3, 3000, None),         # its keys shared out, and merged
    (2, (8, 2), 700, 700, 150),         # query tiles
    (1, (4, 1), 100, 5000, None),       # query tiles, merged
])
def test_nan_in_a_key(cuda_device, B, heads, Sq, Skv, window, dtype):
    """The rows that see it, and only those, are NaN in both results."""
    q, k, v = inputs(cuda_device, B, *heads, Sq, Skv, dtype, Sq)
    at = Skv - Sq + Sq // 2
    k[0, 0, at, 5] = float("nan")
    o, lse = lvx.window_attention(q, k, v, window=window, return_lse=True)
    g = heads[0] // heads[1]
    hit = torch.zeros(B, heads[0], Sq, dtype=torch.bool, device=cuda_device)
    hit[0, :g] = seen(Sq, Skv, [Skv] * B, window, 0, cuda_device)[0, 0, :, at]
    assert hit.any()
    assert (o.isnan().all(-1) == hit).all() and (o.isnan().any(-1) == hit).all()
    assert (lse.view(B, heads[0], Sq).isnan() == hit).all()


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("B,heads,Sq,Skv,window,sinks", [
    (2, (8, 2), 1, 300, None, 0), (2, (8, 2), 8, 2000, None, 0), (2, (32, 2), 4, 1100, 500, 130), (1, (1, 1), 1, 20000, None, 0), (3, (16, 16), 64, 900, None, 0),
])
def test_shared_out(cuda_device, B, heads, Sq, Skv, window, sinks, dtype):
    """Keys of a KV head shared out over CTAs that merge what they have, some of them without a key; the same result every time."""
    q, k, v = inputs(cuda_device, B, *heads, Sq, Skv, dtype, Skv)
    for valid in ([Skv] * B, [0] + [Skv // 2] * (B - 1), [1] + [Skv - 1] * (B - 1), [129] * B):
        m = seen(Sq, Skv, valid, window, sinks, cuda_device)
        o, lse = lvx.window_attention(q, k, v, window=window, sinks=sinks, kv_valid_len=valid, return_lse=True)
        again, lse_again = lvx.window_attention(q, k, v, window=window, sinks=sinks, kv_valid_len=valid, return_lse=True)
        assert torch.equal(o, again) and torch.equal(lse, lse_again)
        ro, rl = exact(q, k, v, m)
        assert v.abs().max() < 6
        assert ((o.double() - ro).abs() <= torch.finfo(dtype).eps * 6).all()      # as above
        empty = (~m.any(-1)).expand(B, heads[0], Sq)
        lse = lse.view(B, heads[0], Sq).double()
        assert (lse[empty] == float("-inf")).all() and (o[empty] == 0).all()
        assert ((lse - rl)[~empty].abs() < 1e-4).all()
