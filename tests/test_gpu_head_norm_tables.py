"""Rotary tables of a single token whose strides, which nothing uses, are not those of aligned rows."""
import pytest
import torch

import lv_xattn_b200 as lvx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("table", [torch.float32, None])
@pytest.mark.parametrize("form", ["row", "row of one", "row per entry", "row of one, two dimensions"])
def test_one_token(cuda_device, form, table, dtype):
    table = table or dtype
    B = 3
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    q, k = (torch.empty(B, 1, h, 128, device=cuda_device, dtype=dtype).normal_(generator=gen).requires_grad_() for h in (4, 2))
    wide = [torch.empty(B, 133, device=cuda_device, dtype=table).normal_(generator=gen) for _ in range(2)]
    made = {"row": lambda t: t[:1, :128][None], "row of one": lambda t: t[:1].as_strided((1, 1, 128), (133, 130, 1)),
                "row per entry": lambda t: t.reshape(-1)[:B * 128].as_strided((B, 1, 128), (128, 131, 1)),
                "row of one, two dimensions": lambda t: t[1:, :128][:1].clone().as_strided((1, 128), (130, 1))}[form]
    cos, sin = (made(t) for t in wide)
    assert cos.is_contiguous()
    plain = [t.reshape(-1).clone().view(cos.shape) for t in (cos, sin)]
    grads = [torch.empty(B, h, 1, 128, device=cuda_device, dtype=dtype).normal_(generator=gen) for h in (4, 2)]
    outs = [lvx.head_norm_rope(q, k, cos=c, sin=s) for c, s in ((cos, sin), plain)]
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    for a, b in zip(*(torch.autograd.grad(o, (q, k), grads) for o in outs)):
        assert torch.equal(a, b)
