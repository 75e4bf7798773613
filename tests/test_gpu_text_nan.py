"""NaN that a row sees stays in its results, however the call is cut into parts: also where all scores of a part are NaN, whose
maximum is then that of an empty part."""
import pytest
import torch

import lv_xattn_b200 as lvx

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def normal(device, dtype, seed, *shapes):
    gen = torch.Generator(device=device).manual_seed(seed)
    return [torch.empty(s, device=device, dtype=dtype).normal_(generator=gen) for s in shapes]


def only_nan_at(o, lse, hit):
    """NaN in the rows `hit` [B, Hq, Sq] of both results, and nowhere else."""
    assert (o.isnan().all(-1) == hit).all() and (o.isnan().any(-1) == hit).all()
    assert (lse.view(hit.shape).isnan() == hit).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,heads,Sq,Skv", [
    (20, (32, 8), 4, 100),       # one CTA a KV head
    (1, (8, 2), 3, 3000),        # up to eight CTAs, merged as a cluster
    (1, (8, 2), 1, 40000),       # more of them, merged by a kernel: eight warps a row
    (9, (64, 4), 3, 30000),      # one warp a row
    (2, (8, 2), 700, 700),       # query tiles
    (1, (4, 1), 100, 5000),      # merged
    (1, (4, 1), 20, 20000),      # one query tile, two warpgroups in turn
])
def test_nan_in_a_query(cuda_device, B, heads, Sq, Skv, dtype):
    q, k, v = normal(cuda_device, dtype, Sq, (B, heads[0], Sq, 128), (B, heads[1], Skv, 128), (B, heads[1], Skv, 128))
    hit = torch.zeros(B, heads[0], Sq, dtype=torch.bool, device=cuda_device)
    for b, h, i in ((0, 1, Sq // 2), (B - 1, heads[0] - 1, Sq - 1)):
        q[b, h, i, 77] = float("nan")
        hit[b, h, i] = True
    only_nan_at(*lvx.window_attention(q, k, v, return_lse=True), hit)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,P,heads,Sq,prefix,own", [
    (1, 1, (4, 2), 1, 300, None), (8, 1, (8, 2), 1, 6404, 512), (32, 1, (8, 2), 1, 20000, 300), (4, 2, (8, 2), 33, 700, 40), (2, 2, (4, 1), 90, 3000, 100),
])
def test_nan_in_a_query_behind_a_prefix(cuda_device, B, P, heads, Sq, prefix, own, dtype):
    q, pk, pv = normal(cuda_device, dtype, B, (B, heads[0], Sq, 128), (P, heads[1], prefix, 128), (P, heads[1], prefix, 128))
    keys = normal(cuda_device, dtype, 1, (B, heads[1], own, 128), (B, heads[1], own, 128)) if own else (None, None)
    hit = torch.zeros(B, heads[0], Sq, dtype=torch.bool, device=cuda_device)
    q[B - 1, 2, Sq // 2, 5] = float("nan")
    hit[B - 1, 2, Sq // 2] = True
    only_nan_at(*lvx.shared_prefix_attention(q, pk, pv, *keys, return_lse=True), hit)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq,Skv,window,sinks", [
    (1, 12801, None, 0),         # a CTA a key tile, the newest key alone in the last
    (1, 300, 1, 4), (1, 5000, 1, 4), (1, 40000, 1, 300),      # the sinks, and the newest key
])
def test_nan_in_a_key_alone(cuda_device, Sq, Skv, window, sinks, dtype):
    q, k, v = normal(cuda_device, dtype, Skv, (2, 4, Sq, 128), (2, 1, Skv, 128), (2, 1, Skv, 128))
    k[1, 0, -1, 3] = float("nan")
    hit = torch.zeros(2, 4, Sq, dtype=torch.bool, device=cuda_device)
    hit[1] = True
    only_nan_at(*lvx.window_attention(q, k, v, window=window, sinks=sinks, return_lse=True), hit)


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_in_own_keys_alone(cuda_device, dtype):
    """A request's only own key: the prefix' part is finite."""
    q, pk, pv, k, v = normal(cuda_device, dtype, 4, (3, 4, 1, 128), (1, 2, 2000, 128), (1, 2, 2000, 128), (3, 2, 8, 128), (3, 2, 8, 128))
    k[1, 0, 0, 9] = float("nan")
    hit = torch.zeros(3, 4, 1, dtype=torch.bool, device=cuda_device)
    hit[1, :2] = True
    only_nan_at(*lvx.shared_prefix_attention(q, pk, pv, k, v, kv_valid_len=[1, 1, 1], return_lse=True), hit)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_a_nan_query(cuda_device, dtype):
    """They are NaN too, and not the zeros of a query that sees nothing."""
    q, k, v, pk, pv = normal(cuda_device, dtype, 6, (2, 4, 70, 128), (2, 2, 70, 128), (2, 2, 70, 128), (1, 2, 900, 128), (1, 2, 900, 128))
    q[0, 1, 30, 2] = float("nan")
    for call in (lambda *t: lvx.window_attention(*t), lambda *t: lvx.shared_prefix_attention(t[0], pk, pv, *t[1:])):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        dq, dk, dv = torch.autograd.grad(call(*leaves).sum(), leaves)
        assert dq[0, 1, 30].isnan().all() and dk[0, 0, :31].isnan().all() and dv[0, 0, :31].isnan().all()
        assert not dk[0, 1].isnan().any() and not dv[1].isnan().any() and not dq[1].isnan().any()
