"""What head_norm_rope refuses, on tensors that never reach a GPU."""
import pytest
import torch

import lv_xattn_b200 as lvx
from lv_xattn_b200._lib import LvxError

Q, K, W = torch.zeros(2, 5, 4, 128), torch.zeros(2, 5, 2, 128), torch.ones(128)
T = torch.ones(5, 128)


@pytest.mark.parametrize("args", [
    dict(q=None, k=None, q_weight=None, k_weight=None),
    dict(q=Q[..., :64]),
    dict(q=Q[0]),
    dict(q=Q.long()),
    dict(k=K[:1]),
    dict(k=K[:, :4]),
    dict(k=K.bfloat16()),
    dict(q=None),                                    # its weight is left over
    dict(q_weight=W[:64]),
    dict(q_weight=W.half()),
    dict(q_weight=None, k_weight=None, cos=None, sin=None),
    dict(cos=None),
    dict(cos=T[:4], sin=T[:4]),
    dict(sin=T[None]),
    dict(cos=T.bfloat16(), sin=T.bfloat16()),
    dict(cos=torch.ones(3, 5, 128), sin=torch.ones(3, 5, 128)),
    dict(eps=-1.0),
    dict(eps=float("nan")),
])
def test_refusals(args):
    with pytest.raises(ValueError):
        lvx.head_norm_rope(**{**dict(q=Q, k=K, q_weight=W, k_weight=W, cos=T, sin=T), **args})


def test_no_cpu_path():
    with pytest.raises(LvxError):
        lvx.head_norm_rope(Q, K, W, W, T, T)
