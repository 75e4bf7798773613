"""The text-side operators together, as a decoder uses them: norm and rotation, windowed attention in training, generation
token by token behind a cache, questions about one video, and the self-attention hook that runs on them."""
import copy
import math

import pytest
import torch

import lv_xattn_b200 as lvx
import _text_oracle as oracle

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)


def tables(positions):
    angle = positions.double()[:, None] * 500000.0 ** (-torch.arange(64, device=positions.device).double() / 64)
    return [f(angle).repeat(1, 2) for f in (torch.cos, torch.sin)]


def test_gradients_through_both(cuda_device):
    """fp32, from the projections' output to the attention's, against autograd over the formulas in 64 bits. Each operator loses
    at most 2^-18 of the sizes of the terms of its sums; three of them in a row, whose terms are a few times their sums: 2^-15."""
    B, S, Hq, Hkv, window, sinks = 2, 70, 4, 2, 20, 3
    g = torch.Generator(device=cuda_device).manual_seed(1)
    r = lambda *s: torch.randn(*s, device=cuda_device, generator=g)
    x = [r(B, S, Hq, 128), r(B, S, Hkv, 128), r(B, S, Hkv, 128), 1 + 0.2 * r(128), 1 + 0.2 * r(128)]
    do = r(B, Hq, S, 128)
    cos, sin = tables(torch.arange(S, device=cuda_device) + 1000)
    leaves = [t.requires_grad_() for t in x]
    q, k = lvx.head_norm_rope(leaves[0], leaves[1], *leaves[3:], cos.float(), sin.float())
    o = lvx.window_attention(q, k, leaves[2].transpose(1, 2), window=window, sinks=sinks, query_start=0)
    got = torch.autograd.grad(o, leaves, do)

    leaves64 = [t.detach().double().requires_grad_() for t in x]

    def prepared(t, w):
        y = w * t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6)
        c, s = cos.float().double()[:, None], sin.float().double()[:, None]
        return (y * c + torch.cat([-y[..., 64:], y[..., :64]], -1) * s).transpose(1, 2)

    q, k = prepared(leaves64[0], leaves64[3]), prepared(leaves64[1], leaves64[4]).repeat_interleave(Hq // Hkv, 1)
    v = leaves64[2].transpose(1, 2).repeat_interleave(Hq // Hkv, 1)
    seen = oracle.visible(S, S, S, window, sinks, 0).to(cuda_device)
    o64 = (q @ k.transpose(-1, -2) * SCALE).masked_fill(~seen, -math.inf).softmax(-1) @ v
    want = torch.autograd.grad(o64, leaves64, do.double())
    for a, b in zip((o.detach(), *got), (o64.detach(), *want)):
        assert (a.double() - b).norm() <= 2.0 ** -15 * b.norm()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_generation_behind_a_cache(cuda_device, dtype):
    """A prompt, then tokens one by one, each written behind the last in a cache whose rest was never written."""
    B, Hq, Hkv, prompt, total, window, sinks = 2, 8, 2, 90, 96, 48, 4
    g = torch.Generator(device=cuda_device).manual_seed(2)
    r = lambda *s: torch.randn(*s, device=cuda_device, generator=g).to(dtype)
    xq, xk, v = r(B, total, Hq, 128), r(B, total, Hkv, 128), r(B, Hkv, total, 128)
    w = (1 + 0.1 * r(128).float()).to(dtype)
    cos, sin = (t.float() for t in tables(torch.arange(total, device=cuda_device)))
    cache = torch.full((2, B, Hkv, 256, 128), float("nan"), device=cuda_device, dtype=dtype)
    lens = torch.zeros(B, device=cuda_device, dtype=torch.int32)
    outs, done = [], 0
    for n in [prompt] + [1] * (total - prompt):
        rows = slice(done, done + n)
        q, k = lvx.head_norm_rope(xq[:, rows], xk[:, rows], w, w, cos[rows], sin[rows])
        cache[0, :, :, rows], cache[1, :, :, rows] = k, v[:, :, rows]
        lens += n
        outs.append(lvx.window_attention(q, cache[0], cache[1], window=window, sinks=sinks, kv_valid_len=lens))
        done += n
    q, k = lvx.head_norm_rope(xq, xk, w, w, cos, sin)
    assert torch.equal(k, cache[0, :, :, :total])
    seen = oracle.visible(total, total, total, window, sinks, 0).to(cuda_device)
    o = torch.cat(outs, 2)
    for b in range(B):
        for h in range(Hq):
            ref = oracle.masked_attention(q[b, h], k[b, h * Hkv // Hq], v[b, h * Hkv // Hq], seen, SCALE)
            oracle.check(o[b, h], *ref["o"], "o")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_questions_about_one_video(cuda_device, dtype):
    """Keys of a video from the fused projection, questions of different lengths about it, then a token each: the same as one
    causal attention per question over the video's keys and its own."""
    from lv_xattn_b200 import ops
    B, Hq, Hkv, N, S, hidden = 3, 8, 2, 700, 33, 256
    g = torch.Generator(device=cuda_device).manual_seed(3)
    r = lambda *s: torch.randn(*s, device=cuda_device, generator=g).to(dtype)
    pk, pv, _ = ops.kv_project(r(1, N, hidden), 0.05 * r(Hkv * 128, hidden), 0.05 * r(Hkv * 128, hidden), torch.ones(128, device=cuda_device), 1e-5, Hkv)
    lens = [33, 20, 5]
    k, v = (torch.full((B, Hkv, 64, 128), float("nan"), device=cuda_device, dtype=dtype) for _ in range(2))
    xq, xk = r(B, S + 1, Hq, 128), r(B, S + 1, Hkv, 128)
    values = r(B, Hkv, S + 1, 128)
    cos, sin = (t.float() for t in tables(torch.arange(S + 1, device=cuda_device)))
    q_all, k_all = lvx.head_norm_rope(xq, xk, cos=cos, sin=sin)
    for b, n in enumerate(lens):
        k[b, :, :n], v[b, :, :n] = k_all[b, :, :n], values[b, :, :n]
    # the questions, right-aligned: query i of request b is its token n_b - S + i
    q = torch.zeros(B, Hq, S, 128, device=cuda_device, dtype=dtype)
    for b, n in enumerate(lens):
        q[b, :, S - n:] = q_all[b, :, :n]
    first = lvx.shared_prefix_attention(q, pk, pv, k, v, kv_valid_len=lens)
    for b, n in enumerate(lens):
        k[b, :, n], v[b, :, n] = k_all[b, :, n], values[b, :, n]
    token = torch.stack([q_all[b, :, n:n + 1] for b, n in enumerate(lens)])
    second = lvx.shared_prefix_attention(token, pk, pv, k, v, kv_valid_len=[n + 1 for n in lens])
    for b, n in enumerate(lens):
        for h in range(Hq):
            kv = h * Hkv // Hq
            keys, vals = torch.cat([pk[0, kv], k[b, kv, :n + 1]]), torch.cat([pv[0, kv], v[b, kv, :n + 1]])
            seen = torch.cat([torch.ones(n + 1, N, dtype=torch.bool), oracle.visible(n + 1, n + 1, n + 1, None, 0, 0)], 1).to(cuda_device)
            ref, bar = oracle.masked_attention(torch.cat([q[b, h, S - n:], token[b, h]]), keys, vals, seen, SCALE)["o"]
            oracle.check(torch.cat([first[b, h, S - n:], second[b, h]]), ref, bar, "o")


def test_windowed_self_attention_hook(cuda_device):
    """The hook with a window and sinks in bf16 against the stock module in fp32 with the mask spelled out (bars of the hook
    without a window, which has the same roundings: weights, projections, attention, output)."""
    from lv_xattn_b200 import hf_patch
    mllama = pytest.importorskip("transformers.models.mllama.modeling_mllama")
    cfg = mllama.MllamaTextConfig(hidden_size=512, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=2,
                                  intermediate_size=512, vocab_size=64)
    cfg._attn_implementation = "eager"
    torch.manual_seed(1)
    ref_mod = mllama.MllamaTextSelfAttention(cfg, layer_idx=1).to(cuda_device)
    rope = mllama.MllamaRotaryEmbedding(cfg).to(cuda_device)
    S, window, sinks = 160, 37, 5
    x = torch.randn(2, S, 512, device=cuda_device)
    cos, sin = rope(x, torch.arange(S, device=cuda_device)[None].expand(2, -1))
    seen = oracle.visible(S, S, S, window, sinks, 0).to(cuda_device)
    mask = torch.zeros(S, S, device=cuda_device).masked_fill_(~seen, float("-inf"))[None, None].expand(2, 1, -1, -1)
    xr = x.clone().requires_grad_(True)
    ref, _ = ref_mod(xr, attention_mask=mask, position_embeddings=(cos, sin))
    g = torch.randn_like(ref)
    ref.backward(g)
    xb = x.to(torch.bfloat16).requires_grad_(True)
    saved = mllama.MllamaTextSelfAttention.forward
    mod = copy.deepcopy(ref_mod).to(torch.bfloat16)
    hf_patch.install_hooks("lv_xattn", window=window, sinks=sinks)
    try:
        assert mllama.MllamaTextSelfAttention.forward is not saved
        out, _ = mod(xb, attention_mask=None, position_embeddings=(cos.to(torch.bfloat16), sin.to(torch.bfloat16)))
        out.backward(g.to(torch.bfloat16))
    finally:
        hf_patch.uninstall_hooks()
    assert mllama.MllamaTextSelfAttention.forward is saved

    def rel(a, b):
        return ((a.float() - b).norm() / b.norm()).item()

    assert rel(out, ref) <= 2e-2, rel(out, ref)
    assert rel(xb.grad, xr.grad) <= 3e-2, rel(xb.grad, xr.grad)
    for (n, p), (_, pr) in zip(mod.named_parameters(), ref_mod.named_parameters()):
        assert p.grad is not None and rel(p.grad, pr.grad) <= 3e-2, (n, rel(p.grad, pr.grad))


def test_two_threads_on_two_streams(cuda_device):
    """Calls that two threads launch at the same time, each on its own stream, give what they give one after the other (dQ up to
    the order of its additions: one rounding)."""
    import threading
    g = torch.Generator(device=cuda_device).manual_seed(4)
    r = lambda *s: torch.randn(*s, device=cuda_device, generator=g).bfloat16()
    inputs = []
    for S, N in ((150, 900), (77, 2500)):
        inputs.append([r(2, S, 8, 128), r(2, S, 2, 128), r(128), r(128), r(2, 2, S, 128), r(1, 2, N, 128), r(1, 2, N, 128), r(2, 8, S, 128)])
    cs = [t.float() for t in tables(torch.arange(200, device=cuda_device))]

    def work(xq, xk, wq, wk, v, pk, pv, do):
        S = xq.shape[1]
        leaves = [t.detach().requires_grad_() for t in (xq, xk, wq, wk, v, pk, pv)]
        q, k = lvx.head_norm_rope(*leaves[:4], cs[0][:S], cs[1][:S])
        o = lvx.window_attention(q, k, leaves[4], window=40, sinks=4) + lvx.shared_prefix_attention(q, *leaves[5:], k, leaves[4])
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    alone = [work(*x) for x in inputs]
    torch.cuda.synchronize()
    got = [[], []]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(12):
                got[i].append(work(*inputs[i]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(got[i]) == 12
        for outs in got[i]:
            assert torch.equal(outs[0], alone[i][0])
            # what dQ's order reaches: the queries' and their weight's gradients; two roundings of 2^-8 of the largest at most
            for j, (a, b) in enumerate(zip(outs[1:], alone[i][1:])):
                if j in (0, 2):
                    assert (a.float() - b.float()).abs().max() <= 2.0 ** -6 * b.float().abs().max(), j
                else:
                    assert torch.equal(a, b), j


def test_no_second_derivatives(cuda_device):
    x = torch.randn(1, 8, 2, 128, device=cuda_device, requires_grad=True)
    cs = [t.float() for t in tables(torch.arange(8, device=cuda_device))]
    for out in (lvx.head_norm_rope(x, None, cos=cs[0], sin=cs[1])[0], lvx.window_attention(x, x, x, window=3),
                lvx.shared_prefix_attention(x, x, x)):
        (g,) = torch.autograd.grad((out * out).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


def test_broadcast_gradients_and_unused_outputs(cuda_device):
    """An upstream gradient of one repeated value (what .sum() gives), and a result whose log-sum-exp alone is used."""
    g = torch.Generator(device=cuda_device).manual_seed(5)
    x = torch.randn(1, 4, 70, 128, device=cuda_device, generator=g).bfloat16().requires_grad_()
    for f in (lambda t: lvx.window_attention(t, t, t, window=9), lambda t: lvx.shared_prefix_attention(t, t, t, t, t),
              lambda t: lvx.head_norm_rope(t, None, torch.ones(128, device=cuda_device))[0]):
        (a,) = torch.autograd.grad(f(x).sum(), x)
        out = f(x)
        (b,) = torch.autograd.grad(out, x, torch.ones_like(out))
        assert (a.float() - b.float()).abs().max() <= 2.0 ** -6 * b.float().abs().max()
    _, lse = lvx.window_attention(x, x, x, window=9, return_lse=True)
    assert not lse.requires_grad
