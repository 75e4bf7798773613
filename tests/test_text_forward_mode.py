"""The text operators refuse tensors that carry a forward-mode tangent, which their results would not."""
import pytest
import torch
from torch.autograd import forward_ad

import lv_xattn_b200 as lvx
from lv_xattn_b200._lib import LvxError

T = torch.zeros(2, 4, 3, 128)
TABLE = torch.zeros(4, 128)
CALLS = {
    "head_norm_rope": (lvx.head_norm_rope, dict(q=T, k=T, q_weight=torch.ones(128), k_weight=torch.ones(128), cos=TABLE, sin=TABLE)),
    "window_attention": (lvx.window_attention, dict(q=T, k=T, v=T)),
    "shared_prefix_attention": (lvx.shared_prefix_attention, dict(q=T, k_prefix=T, v_prefix=T, k=T, v=T)),
}


@pytest.mark.parametrize("name", CALLS)
def test_tangents_are_refused(name):
    call, args = CALLS[name]
    for which, t in args.items():
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(t.clone(), torch.ones_like(t))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(**{**args, which: dual})
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call(**{**args, which: dual})


@pytest.mark.parametrize("name", CALLS)
def test_tensors_without_one_are_not(name):
    """The call ends at the missing CPU path."""
    call, args = CALLS[name]
    with forward_ad.dual_level(), pytest.raises(LvxError):
        call(**args)
    with pytest.raises(LvxError):
        call(**args)


@pytest.mark.parametrize("name", CALLS)
def test_function_transforms(name):
    call, args = CALLS[name]
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: call(**{**args, next(iter(args)): t}), (T,), (torch.ones_like(T),))
