"""shared_prefix_attention against masked attention over both kinds of keys in 64 bits (bars in _text_oracle.py)."""
import math

import pytest
import torch

import lv_xattn_b200 as lvx
import _text_oracle as oracle

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
SCALE = 1 / math.sqrt(128)


def inputs(device, B, P, Hq, Hkv, Sq, prefix, Skv, dtype, seed):
    """q, pk, pv, k, v, dO (k and v None where Skv is)"""
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=device, generator=g)
    own = [r(B, Hkv, Skv, 128).to(dtype), (0.5 * r(B, Hkv, Skv, 128)).to(dtype)] if Skv is not None else [None, None]
    return [r(B, Hq, Sq, 128).to(dtype), r(P, Hkv, prefix, 128).to(dtype), (0.5 * r(P, Hkv, prefix, 128)).to(dtype), *own,
            r(B, Hq, Sq, 128).to(dtype)]


def reference(q, pk, pv, k, v, do, prefix_valid, valid):
    B, Hq, Sq, _ = q.shape
    P, Hkv, N, _ = pk.shape
    Skv = 0 if k is None else k.shape[2]
    out = {n: [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for _ in range(2)]
           for n, t in dict(o=q, lse=q[..., 0], dq=q, dpk=pk, dpv=pv, dk=k, dv=v).items() if t is not None}
    for b in range(B):
        p = b // (B // P)
        n = min(max(prefix_valid[p], 0), N) if prefix_valid is not None else N
        seen = (torch.arange(N) < n).expand(Sq, -1)
        if Skv:
            m = min(max(valid[b], 0), Skv) if valid is not None else Skv
            seen = torch.cat([seen, oracle.visible(m, Sq, Skv, None, 0, None)], 1)
        seen = seen.to(q.device)
        for h in range(Hq):
            kv = h * Hkv // Hq
            keys, values = (torch.cat([t[p, kv], u[b, kv]]) if Skv else t[p, kv] for t, u in ((pk, k), (pv, v)))
            got = oracle.masked_attention(q[b, h], keys, values, seen, SCALE, None if do is None else do[b, h])
            for name, pair in got.items():
                for i, part in enumerate(pair):
                    if name in ("dk", "dv"):
                        out["dp" + name[1]][i][p, kv] += part[:N]
                        if Skv:
                            out[name][i][b, kv] += part[N:]
                    else:
                        out[name][i][b, h] += part
    return out


def run_and_check(q, pk, pv, k, v, do, prefix_valid=None, valid=None, backward=True):
    from lv_xattn_b200 import _lib
    leaves = [t.detach().requires_grad_(backward) for t in (q, pk, pv, k, v) if t is not None]
    o, lse = lvx.shared_prefix_attention(*leaves, sm_scale=SCALE, prefix_valid_len=prefix_valid, kv_valid_len=valid, return_lse=True)
    grads = torch.autograd.grad(o, leaves, do) if backward else ()
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    ref = reference(q, pk, pv, k, v, do if backward else None, prefix_valid, valid)
    oracle.check(o.detach(), *ref["o"], "o")
    oracle.check(lse.view(q.shape[:3]), *ref["lse"], "lse")
    for n, g in zip(("dq", "dpk", "dpv", "dk", "dv"), grads):
        oracle.check(g, *ref[n], n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,P,heads", [(1, 1, (4, 2)), (3, 1, (4, 2)), (16, 1, (8, 2)), (17, 1, (4, 1)), (33, 1, (8, 2)), (70, 1, (8, 2)),
                                       (6, 2, (6, 2)), (4, 4, (4, 4))])
def test_one_token(cuda_device, B, P, heads, dtype):
    q, pk, pv, k, v, do = inputs(cuda_device, B, P, *heads, 1, 1601, 60, dtype, 1)
    run_and_check(q, pk, pv, k, v, do, prefix_valid=[1601 - 400 * p for p in range(P)], valid=[(7 * b) % 61 for b in range(B)], backward=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,P,heads,Sq,prefix", [(1, 1, (1, 1), 1, 1), (2, 1, (4, 2), 5, 129), (3, 1, (3, 1), 77, 300), (4, 2, (4, 2), 40, 700),
                                                 (2, 1, (5, 5), 130, 257), (2, 2, (8, 2), 33, 128)])
def test_training(cuda_device, B, P, heads, Sq, prefix, dtype):
    q, pk, pv, k, v, do = inputs(cuda_device, B, P, *heads, Sq, prefix, Sq + 9, dtype, 2)
    run_and_check(q, pk, pv, k, v, do)
    run_and_check(q, pk, pv, k, v, do, prefix_valid=[prefix - prefix // 3 * (p + 1) for p in range(P)], valid=[(Sq + 9) // (b + 1) for b in range(B)])
    run_and_check(q, pk, pv, None, None, do, prefix_valid=[prefix - 1] * P)


@pytest.mark.parametrize("dtype", TYPES)
def test_empty_parts(cuda_device, dtype):
    """No valid prefix, no valid own keys, neither."""
    args = inputs(cuda_device, 4, 2, 4, 2, 20, 150, 30, dtype, 3)
    run_and_check(*args, prefix_valid=[0, 150], valid=[30, 0, 11, 0])
    args = inputs(cuda_device, 4, 2, 4, 2, 1, 150, 30, dtype, 4)
    run_and_check(*args, prefix_valid=[0, 150], valid=[30, 0, 11, 0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq", [1, 50])
def test_rows_behind_the_last_key(cuda_device, Sq, dtype):
    q, pk, pv, k, v, do = inputs(cuda_device, 4, 2, 8, 2, Sq, 400, 100, dtype, 5)
    prefix_valid, valid = [300, 129], [100, 77, 51, 60]
    for t, lens in ((pk, prefix_valid), (pv, prefix_valid), (k, valid), (v, valid)):
        for b, n in enumerate(lens):
            t[b, :, n:] = float("nan") if t is pk or t is k else float("inf")
    run_and_check(q, pk, pv, k, v, do, prefix_valid, valid)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(cuda_device, dtype):
    q, pk, pv, k, v, do = inputs(cuda_device, 3, 1, 8, 2, 21, 333, 40, dtype, 6)
    by_token = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, pk, pv, k, v, do)]
    run_and_check(*by_token)
    longer = torch.full((2, 1, 2, 500, 128), float("nan"), device=cuda_device, dtype=dtype)
    longer[0, :, :, :333], longer[1, :, :, :333] = pk, pv
    run_and_check(q, longer[0, :, :, :333], longer[1, :, :, :333], k, v[:, :1].expand(-1, 2, -1, -1), do)
    # one request a prefix: the queries need no packing, unless they are strided
    q, pk, pv, k, v, do = inputs(cuda_device, 2, 2, 8, 2, 21, 333, 40, dtype, 7)
    run_and_check(q, pk, pv, k, v, do)
    run_and_check(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, pk, pv, k, v, do)))


@pytest.mark.parametrize("dtype", TYPES)
def test_long_prefix(cuda_device, dtype):
    """Keys split over the GPU for one, a few and many rows."""
    for B, Sq in ((1, 1), (8, 3), (5, 60)):
        run_and_check(*inputs(cuda_device, B, 1, 4, 1, Sq, 9000, 70, dtype, 8), prefix_valid=[8901])


@pytest.mark.parametrize("dtype", TYPES)
def test_same_as_the_parts(cuda_device, dtype):
    """One request without own keys is a plain attention; one whose prefix is not valid is a causal one."""
    q, pk, pv, k, v, _ = inputs(cuda_device, 2, 2, 8, 2, 30, 500, 64, dtype, 9)
    o, lse = lvx.shared_prefix_attention(q, pk, pv, return_lse=True)
    _, _, _, o2, lse2 = lvx._attn_forward(q, pk, pv, False, SCALE, None)
    tol = 2 * max(oracle.unit(dtype)[0], 2.0 ** -17)
    assert (o.float() - o2.float()).abs().max() <= 2 * tol * pv.float().abs().max() and (lse - lse2).abs().max() <= 2.0 ** -13
    o, lse = lvx.shared_prefix_attention(q, pk, pv, k, v, prefix_valid_len=[0, 0], return_lse=True)
    o2, lse2 = lvx.window_attention(q, k, v, return_lse=True)
    assert (o.float() - o2.float()).abs().max() <= 2 * tol * v.float().abs().max() and (lse - lse2).abs().max() <= 2.0 ** -13


def test_captured_and_on_another_stream(cuda_device):
    """As for the windowed attention: a captured pass, replayed on new inputs and lengths, and one on another stream."""
    q, pk, pv, k, v, do = inputs(cuda_device, 4, 2, 8, 2, 40, 700, 90, torch.bfloat16, 10)
    plens, lens = (torch.tensor(t, device=cuda_device, dtype=torch.int32) for t in ([700, 333], [90, 60, 41, 88]))

    def both():
        leaves = [t.detach().requires_grad_() for t in (q, pk, pv, k, v)]
        o = lvx.shared_prefix_attention(*leaves, prefix_valid_len=plens, kv_valid_len=lens)
        one = lvx.shared_prefix_attention(q[:, :, :1], pk, pv, k, v, prefix_valid_len=plens, kv_valid_len=lens)
        return [o.detach(), one, *torch.autograd.grad(o, leaves, do)]

    def same(a, b):
        for i, (x, y) in enumerate(zip(a, b)):
            assert torch.equal(x, y) if i != 2 else (x.float() - y.float()).abs().max() <= 2.0 ** -8 * y.float().abs().max()

    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = both()
    side.synchronize()
    same(again, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = both()
    for seed in (11, 12):
        for old, new in zip((q, pk, pv, k, v, do), inputs(cuda_device, 4, 2, 8, 2, 40, 700, 90, torch.bfloat16, seed)):
            old.copy_(new)
        plens.copy_(torch.tensor([seed * 20, 700]))
        graph.replay()
        torch.cuda.synchronize()
        same(kept, both())


def test_word_already_set(cuda_device):
    from lv_xattn_b200 import ops, _lib, peer_memory as pm
    from lv_xattn_b200.async_communication import P2PTimeoutError
    for dtype in TYPES[::2]:
        q, pk, pv, k, v, do = inputs(cuda_device, 4, 1, 8, 2, 40, 700, 90, dtype, 13)
        leaves = [t.requires_grad_() for t in (q, pk, pv, k, v)]
        good = lvx.shared_prefix_attention(*leaves)
        lib = _lib.load()
        lib.lvx_p2p_set_timeout(0.001)
        try:
            for backward in (False, True):
                ops.p2p_wait(torch.zeros(8 * 16, dtype=torch.int32, device=cuda_device), 1, 0, 1)
                if backward:
                    torch.autograd.grad(good, leaves, do, retain_graph=True)
                else:
                    lvx.shared_prefix_attention(*leaves)
                torch.cuda.synchronize()
                with pytest.raises(P2PTimeoutError):
                    lvx.shared_prefix_attention(*leaves)
                pm.check_device_status()
        finally:
            lib.lvx_p2p_set_timeout(120.0)
            _lib.device_status()
        assert torch.equal(lvx.shared_prefix_attention(*leaves), good)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,P,heads,N", [(6, 2, (8, 2), 300), (40, 1, (32, 8), 700), (64, 2, (16, 2), 1000), (5, 1, (12, 4), 129)])
def test_single_tokens_where_they_are(cuda_device, B, P, heads, N, dtype):
    """Queries of single tokens in layouts that are read without being packed, few rows and many: as in the dense layout."""
    q, pk, pv, k, v, _ = inputs(cuda_device, B, P, *heads, 1, N, 50, dtype, B)
    dense = lvx.shared_prefix_attention(q, pk, pv, k, v, return_lse=True)
    wide = torch.full((B, heads[0], 3, 128), float("nan"), device=cuda_device, dtype=dtype)
    wide[:, :, 1:2] = q
    by_token = q.transpose(1, 2).contiguous().transpose(1, 2)
    for other in (wide[:, :, 1:2], by_token):
        o, lse = lvx.shared_prefix_attention(other, pk, pv, k, v, return_lse=True)
        assert torch.equal(o, dense[0]) and torch.equal(lse, dense[1])
    run_and_check(q, pk, pv, k, v, torch.randn_like(q), backward=False)
