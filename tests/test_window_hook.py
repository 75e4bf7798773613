"""The self-attention hook with a window: what it refuses when it is made, and a window as long as the text."""
import copy

import pytest
import torch

from lv_xattn_b200 import hf_patch


@pytest.mark.parametrize("args", [dict(window=2.5), dict(window="8"), dict(window=8, sinks=0.5), dict(window=8, sinks=None)])
def test_whole_numbers(args):
    """Refused before a class is changed, and not in the first forward."""
    mllama = pytest.importorskip("transformers.models.mllama.modeling_mllama")
    before = mllama.MllamaTextCrossAttention.forward, mllama.MllamaTextSelfAttention.forward
    with pytest.raises(ValueError, match="integer"):
        hf_patch.install_hooks("lv_xattn", **args)
    assert before == (mllama.MllamaTextCrossAttention.forward, mllama.MllamaTextSelfAttention.forward)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [96, 97, 1 << 40])
def test_a_window_as_long_as_the_text(cuda_device, window):
    """The plain causal mask: the stock module's output and gradients, in fp32. A product of the layer loses at most 2^-18 of its terms'
    sizes; there are four of them one behind the other, whose terms are up to four times their sums: 2^-14. (torch's own products may
    run in tf32, which loses 2^-11, so that is off.)"""
    mllama = pytest.importorskip("transformers.models.mllama.modeling_mllama")
    cfg = mllama.MllamaTextConfig(hidden_size=512, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=2,
                                  intermediate_size=512, vocab_size=64)
    cfg._attn_implementation = "eager"
    torch.manual_seed(2)
    stock = mllama.MllamaTextSelfAttention(cfg, layer_idx=1).to(cuda_device)
    rope = mllama.MllamaRotaryEmbedding(cfg).to(cuda_device)
    S = 96
    x = torch.randn(2, S, 512, device=cuda_device)
    tables = rope(x, torch.arange(S, device=cuda_device)[None].expand(2, -1))
    mask = torch.full((S, S), float("-inf"), device=cuda_device).triu(1)[None, None].expand(2, 1, -1, -1)
    hooked, g = copy.deepcopy(stock), torch.randn(2, S, 512, device=cuda_device)
    tf32, torch.backends.cuda.matmul.allow_tf32 = torch.backends.cuda.matmul.allow_tf32, False
    try:
        xs = [x.clone().requires_grad_() for _ in range(2)]
        want = stock(xs[0], attention_mask=mask, position_embeddings=tables)[0]
        want.backward(g)
        got = hf_patch.patch_self_attention_forward("lv_xattn", window=window)(hooked, xs[1], position_embeddings=tables)[0]
        got.backward(g)
    finally:
        torch.backends.cuda.matmul.allow_tf32 = tf32

    def close(a, b):
        assert (a - b).norm() <= 2.0 ** -14 * b.norm()

    close(got, want)
    close(xs[1].grad, xs[0].grad)
    for (_, a), (_, b) in zip(hooked.named_parameters(), stock.named_parameters()):
        close(a.grad, b.grad)
