"""window_attention against masked attention in 64 bits (bars in _text_oracle.py)."""
import math

import pytest
import torch

import lv_xattn_b200 as lvx
import _text_oracle as oracle

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
SCALE = 1 / math.sqrt(128)


def inputs(device, B, Hq, Hkv, Sq, Skv, dtype, seed, gain=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=device, generator=g)
    return [t.to(dtype) for t in (gain * r(B, Hq, Sq, 128), r(B, Hkv, Skv, 128), 0.5 * r(B, Hkv, Skv, 128), r(B, Hq, Sq, 128))]


def reference(q, k, v, do, window, sinks, valid, start):
    B, Hq, Sq, _ = q.shape
    Hkv, Skv = k.shape[1:3]
    out = {n: [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for _ in range(2)]
           for n, t in dict(o=q, lse=q[..., 0], dq=q, dk=k, dv=v).items()}
    for b in range(B):
        seen = oracle.visible(min(max(valid[b], 0), Skv) if valid is not None else Skv, Sq, Skv, window, sinks, start).to(q.device)
        for h in range(Hq):
            kv = h * Hkv // Hq
            got = oracle.masked_attention(q[b, h], k[b, kv], v[b, kv], seen, SCALE, None if do is None else do[b, h])
            for n, pair in got.items():
                for total, part in zip(out[n], pair):
                    total[b, kv if n in ("dk", "dv") else h] += part
    return out


def run_and_check(q, k, v, do, window=None, sinks=0, valid=None, start=None, backward=True, lengths=None):
    from lv_xattn_b200 import _lib
    leaves = [t.detach().requires_grad_(backward) for t in (q, k, v)]
    o, lse = lvx.window_attention(*leaves, SCALE, window=window, sinks=sinks, kv_valid_len=valid if lengths is None else lengths,
                                  query_start=start, return_lse=True)
    grads = torch.autograd.grad(o, leaves, do) if backward else ()
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    ref = reference(q, k, v, do if backward else None, window, sinks, valid, start)
    oracle.check(o.detach(), *ref["o"], "o")
    oracle.check(lse.view(q.shape[:3]), *ref["lse"], "lse")
    for n, g in zip(("dq", "dk", "dv"), grads):
        oracle.check(g, *ref[n], n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Skv,window,sinks", [(1, None, 0), (77, 16, 4), (129, None, 0), (700, 1, 0), (700, 128, 4), (700, 300, 130),
                                              (1601, 129, 300), (1601, 5000, 2)])
def test_one_token(cuda_device, Skv, window, sinks, dtype):
    run_and_check(*inputs(cuda_device, 2, 8, 2, 1, Skv, dtype, 1), window, sinks, backward=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,Sq", [((1, 1), 17), ((4, 2), 16), ((3, 1), 11), ((4, 1), 16), ((5, 1), 13), ((12, 4), 5)])
def test_a_few_tokens_behind_a_cache(cuda_device, heads, Sq, dtype):
    q, k, v, do = inputs(cuda_device, 3, *heads, Sq, 900, dtype, 2)
    run_and_check(q, k, v, do, 200, 4, valid=[900, 333, 7])
    run_and_check(q, k, v, do, None, 0, valid=[128, 900, 0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", [(1, 1), (4, 1), (3, 1), (8, 2), (10, 2), (130, 1)])
@pytest.mark.parametrize("S,window,sinks", [(130, None, 0), (333, 64, 4), (257, 130, 140)])
def test_whole_texts(cuda_device, heads, S, window, sinks, dtype):
    if heads[0] > 100 and S > 200:
        pytest.skip("the same tiles, three times the work")
    run_and_check(*inputs(cuda_device, 1, *heads, S, S, dtype, 3), window, sinks, start=0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("start", [0, 5, 300, None])
def test_padded_texts(cuda_device, start, dtype):
    """Fewer keys than queries, none at all, rows whose window ends before the first key or begins behind the last."""
    run_and_check(*inputs(cuda_device, 4, 4, 2, 150, 200, dtype, 4), 40, 3, valid=[200, 131, 20, 0], start=start)
    run_and_check(*inputs(cuda_device, 4, 4, 2, 150, 200, dtype, 5), None, 0, valid=[200, 131, 20, 0], start=start)


@pytest.mark.parametrize("dtype", TYPES)
def test_chunk_of_a_long_text(cuda_device, dtype):
    """Tiles that are too few for the GPU: the keys are split, and the parts merged."""
    run_and_check(*inputs(cuda_device, 1, 8, 2, 40, 5000, dtype, 6), None, 0, backward=False)
    run_and_check(*inputs(cuda_device, 1, 8, 2, 40, 5000, dtype, 7), 1500, 200, valid=[4321])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq", [1, 16, 100])
def test_rows_behind_the_last_key_and_masked_keys(cuda_device, Sq, dtype):
    """Rows of a cache that nothing was written to yet hold NaN and infinities, and so do keys that a query does not see."""
    q, k, v, do = inputs(cuda_device, 2, 4, 2, Sq, 400, dtype, 8)
    valid = [300, 257]
    for b, n in enumerate(valid):
        k[b, :, n:] = float("nan")
        v[b, :, n:] = float("inf")
    run_and_check(q, k, v, do, 64, 4, valid=valid)
    # keys that every query but the first one or none at all has left behind
    for bad in (float("nan"), float("inf"), float("-inf")):
        for b, n in enumerate(valid):
            at = n - Sq - 64 + 1          # the first query's oldest key but one
            k[b, :, at], v[b, :, at - 1] = bad, bad
        run_and_check(q, k, v, do, 63, 4, valid=valid, backward=False)
    # a later token of the same tile: the queries before it do not see it
    if Sq > 2:
        q, k, v, do = inputs(cuda_device, 1, 4, 2, Sq, 400, dtype, 9)
        v[0, :, 400 - Sq + 2, 7] = float("inf")
        o = lvx.window_attention(q, k, v, SCALE, window=64, sinks=4)
        assert torch.isfinite(o[:, :, :2]).all()
        assert torch.isposinf(o[:, :, 2:60, 7]).all() and torch.isfinite(o[:, :, 2:, 8:]).all()
        v[0, :, 400 - Sq + 2, 7] = 0
        oracle.check(o[:, :, :2], *(t[:, :, :2] for t in reference(q, k, v, None, 64, 4, None, None)["o"]), "o")


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(cuda_device, dtype):
    """Views of the projections' layout, of a longer cache, of a fused buffer, and rows off their alignment."""
    for Sq, Skv in ((3, 200), (140, 140)):
        q, k, v, do = inputs(cuda_device, 2, 8, 2, Sq, Skv, dtype, 10)
        by_token = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, do)]
        run_and_check(*by_token, 50, 4)
        cache = torch.full((2, 2, 2, 512, 128), float("nan"), device=cuda_device, dtype=dtype)
        cache[0, :, :, :Skv], cache[1, :, :, :Skv] = k, v
        run_and_check(q, cache[0, :, :, :Skv], cache[1, :, :, :Skv], do, 50, 4)
        fused = torch.cat([k, v], -1)
        run_and_check(q, fused[..., :128], fused[..., 128:], do, 50, 4)
        odd = torch.zeros(k.numel() + 1, device=cuda_device, dtype=dtype)
        odd[1:] = k.flatten()
        run_and_check(q, odd[1:].view_as(k), v[:, :1].expand(-1, 2, -1, -1), do, 50, 4)


def test_large_scores(cuda_device):
    """Running maxima that jump from tile to tile."""
    run_and_check(*inputs(cuda_device, 1, 4, 1, 300, 900, torch.bfloat16, 11, gain=8.0), 400, 4, backward=False)
    run_and_check(*inputs(cuda_device, 1, 4, 1, 2, 900, torch.bfloat16, 12, gain=8.0), 400, 4, backward=False)


def test_lengths_in_every_form(cuda_device):
    q, k, v, do = inputs(cuda_device, 3, 4, 2, 70, 200, torch.bfloat16, 13)
    lens = [500, 77, -5]              # taken into 0..Skv
    for form in (lens, torch.tensor(lens), torch.tensor(lens, dtype=torch.int32), torch.tensor(lens, device=cuda_device),
                 torch.tensor(lens, device=cuda_device, dtype=torch.int32)):
        run_and_check(q, k, v, do, 60, 2, valid=lens, lengths=form)
    for bad in (lens[:2], [1.0, 2.0, 3.0], torch.zeros(3, 1, dtype=torch.int32)):
        with pytest.raises(ValueError):
            lvx.window_attention(q, k, v, kv_valid_len=bad)


def test_no_keys(cuda_device):
    q, k, v, do = inputs(cuda_device, 2, 4, 2, 70, 200, torch.bfloat16, 14)
    for Sq in (2, 70):
        leaves = [t.requires_grad_() for t in (q[:, :, :Sq], k[:, :, :0], v[:, :, :0])]
        o, lse = lvx.window_attention(*leaves, window=5, return_lse=True)
        assert (o == 0).all() and torch.isneginf(lse).all()
        dq, dk, dv = torch.autograd.grad(o, leaves, do[:, :, :Sq])
        assert (dq == 0).all() and dk.shape == leaves[1].shape and dv.shape == leaves[2].shape


@pytest.mark.parametrize("dtype", TYPES)
def test_differences(cuda_device, dtype):
    """Gradients against differences of the forward (in fp32, whose forward has the digits for it)."""
    q, k, v, do = inputs(cuda_device, 1, 4, 2, 90, 120, dtype, 15)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(lvx.window_attention(*leaves, window=33, sinks=2), leaves, do)
    f = [t.detach().float() for t in (q, k, v)]
    loss = lambda ts: (lvx.window_attention(*ts, window=33, sinks=2).double() * do.double()).sum()
    g = torch.Generator(device=cuda_device).manual_seed(16)
    for i in range(3):
        step, h = torch.randn(f[i].shape, device=cuda_device, generator=g), 2.0 ** -6
        ends = [loss([t + s * h * step if j == i else t for j, t in enumerate(f)]) for s in (1, -1)]
        terms = got[i].double() * step.double()
        # rounding of the gradients (three roundings of e of terms that do not cancel in the bar), the third derivative's h^2 / 6
        assert abs((ends[0] - ends[1]) / (2 * h) - terms.sum()) <= (4 * oracle.unit(dtype)[0] + 1e-3) * terms.abs().sum()


def test_captured_and_on_another_stream(cuda_device):
    """A captured forward and backward, replayed on new inputs and lengths with larger calls in between; the same on another
    stream. dQ is summed by reduce-adds in any order: one rounding apart."""
    q, k, v, do = inputs(cuda_device, 2, 8, 2, 150, 300, torch.bfloat16, 17)
    token, lens = inputs(cuda_device, 2, 8, 2, 1, 300, torch.bfloat16, 18)[0], torch.tensor([300, 150], device=cuda_device, dtype=torch.int32)

    def both():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = lvx.window_attention(*leaves, window=64, sinks=4, kv_valid_len=lens, query_start=0)
        one = lvx.window_attention(token, k, v, window=64, sinks=4, kv_valid_len=lens)
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
    big = inputs(cuda_device, 1, 8, 2, 700, 700, torch.bfloat16, 19)
    for seed in (20, 21):
        for old, new in zip((q, k, v, do), inputs(cuda_device, 2, 8, 2, 150, 300, torch.bfloat16, seed)):
            old.copy_(new)
        lens.copy_(torch.tensor([seed * 10, seed], device=cuda_device))
        lvx.window_attention(*big[:3], window=200)
        graph.replay()
        torch.cuda.synchronize()
        same(kept, both())


def test_word_already_set(cuda_device):
    """A wait that ran out earlier has left its code in the status word: nothing is computed, and the next call says so."""
    from lv_xattn_b200 import ops, _lib, peer_memory as pm
    from lv_xattn_b200.async_communication import P2PTimeoutError
    for dtype, Sq in ((torch.bfloat16, 2), (torch.bfloat16, 150), (torch.float32, 150)):
        q, k, v, do = inputs(cuda_device, 2, 8, 2, Sq, 4000, dtype, 22)
        leaves = [t.requires_grad_() for t in (q, k, v)]
        good = lvx.window_attention(*leaves, window=64)
        torch.autograd.grad(good, leaves, do, retain_graph=True)
        lib = _lib.load()
        lib.lvx_p2p_set_timeout(0.001)
        try:
            for backward in (False, True):
                ops.p2p_wait(torch.zeros(8 * 16, dtype=torch.int32, device=cuda_device), 1, 0, 1)
                if backward:
                    torch.autograd.grad(good, leaves, do, retain_graph=True)
                else:
                    lvx.window_attention(*leaves, window=64)
                torch.cuda.synchronize()
                with pytest.raises(P2PTimeoutError):
                    lvx.window_attention(*leaves, window=64)
                pm.check_device_status()
        finally:
            lib.lvx_p2p_set_timeout(120.0)
            _lib.device_status()
        assert torch.equal(lvx.window_attention(*leaves, window=64), good)


@pytest.mark.parametrize("Sq", [1, 70])
def test_offsets_past_32_bits(cuda_device, Sq):
    """A cache of 2.2 million keys: 2^31 values lie before its last head. What is compared is that head, at its end."""
    Skv, Hkv, window, sinks = 2_200_000, 8, 300, 4
    q, small_k, small_v, do = inputs(cuda_device, 1, 2 * Hkv, Hkv, Sq, 1024, torch.bfloat16, 23)
    k, v = (torch.zeros(1, Hkv, Skv, 128, device=cuda_device, dtype=torch.bfloat16) for _ in range(2))
    for big, small in ((k, small_k), (v, small_v)):
        big[:, :, :512], big[:, :, -512:] = small[:, :, :512], small[:, :, 512:]
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = lvx.window_attention(*leaves, SCALE, window=window, sinks=sinks)
    grads = torch.autograd.grad(o, leaves, do)
    seen = oracle.visible(1024, Sq, 1024, window, sinks, None).to(cuda_device)      # the keys between have no part in it
    h, kv = 2 * Hkv - 1, Hkv - 1
    parts = [oracle.masked_attention(q[0, i], small_k[0, kv], small_v[0, kv], seen, SCALE, do[0, i]) for i in (h - 1, h)]
    oracle.check(o[0, h].detach(), *parts[1]["o"], "o")
    oracle.check(grads[0][0, h], *parts[1]["dq"], "dq")
    for name, got in zip(("dk", "dv"), grads[1:]):
        ref, bar = (parts[0][name][i] + parts[1][name][i] for i in range(2))
        oracle.check(torch.cat([got[0, kv, :512], got[0, kv, -512:]]), ref, bar, name)
        assert not got[0, kv, 512:-512].any()
