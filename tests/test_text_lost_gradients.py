"""Arguments of the text operators that no gradient flows into may not ask for one."""
import pytest
import torch

import lv_xattn_b200 as lvx
from lv_xattn_b200._lib import LvxError

T = torch.zeros(2, 4, 3, 128)


@pytest.mark.parametrize("which", ["cos", "sin"])
def test_tables(which):
    args = dict(q=T, k=None, cos=torch.zeros(4, 128), sin=torch.zeros(4, 128))
    args[which] = args[which].clone().requires_grad_()
    with pytest.raises(ValueError, match=which):
        lvx.head_norm_rope(**args)
    with torch.no_grad(), pytest.raises(LvxError):      # (only the CPU path is missing)
        lvx.head_norm_rope(**args)


def test_scale():
    scale = torch.tensor(0.1, requires_grad=True)
    for call in (lambda s: lvx.window_attention(T, T, T, s), lambda s: lvx.shared_prefix_attention(T, T, T, sm_scale=s)):
        with pytest.raises(ValueError, match="sm_scale"):
            call(scale)
        with torch.no_grad(), pytest.raises(LvxError):
            call(scale)
        with pytest.raises(LvxError):
            call(scale.detach())
