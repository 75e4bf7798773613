"""What shared_prefix_attention refuses, on tensors that never reach a GPU."""
import ctypes

import pytest
import torch

import lv_xattn_b200 as lvx
from lv_xattn_b200._lib import LvxError

Q, P, K = torch.zeros(4, 6, 3, 128), torch.zeros(2, 2, 9, 128), torch.zeros(4, 2, 5, 128)


@pytest.mark.parametrize("args", [
    dict(q=Q[:3]),
    dict(q=Q[:, :5]),
    dict(q=Q[..., :64]),
    dict(q=Q[:, :, :0]),
    dict(q=Q.long()),
    dict(k_prefix=P[:, :, :0], v_prefix=P[:, :, :0]),
    dict(k_prefix=P[:0], v_prefix=P[:0]),
    dict(v_prefix=P[:, :, :8]),
    dict(k_prefix=P.half(), v_prefix=P.half()),
    dict(k=None),
    dict(k=K[:2], v=K[:2]),
    dict(k=K[:, :1], v=K[:, :1]),
    dict(v=K[:, :, :4]),
    dict(k=None, v=None, kv_valid_len=[1, 1, 1, 1]),
    dict(sm_scale=-1.0),
])
def test_tensors(args):
    with pytest.raises(ValueError):
        lvx.shared_prefix_attention(**{**dict(q=Q, k_prefix=P, v_prefix=P, k=K, v=K), **args})


def test_no_cpu_path():
    with pytest.raises(LvxError):
        lvx.shared_prefix_attention(Q, P, P, K, K)


def test_abi_refusals():
    from lv_xattn_b200 import _lib
    lib = _lib.load()
    f, b = ctypes.c_size_t(0), ctypes.c_size_t(0)

    def workspace(prefixes, length, shape=(4, 4, 2, 16, 16, 128, 0, 0)):
        return lib.lvx_shared_workspace(ctypes.byref(_lib.LvxShape(*shape)), prefixes, length, ctypes.byref(f), ctypes.byref(b))

    assert workspace(2, 100) == 0 and f.value > 0 and b.value > 0
    assert workspace(2, 100, (4, 4, 2, 16, 0, 128, 2, 0)) == 0
    assert workspace(3, 100) == -2 and workspace(0, 100) == -2 and workspace(2, 0) == -2 and workspace(2, 1 << 28) == -2
    assert workspace(1, 100, (4096, 4, 1, 1 << 18, 16, 128, 0, 0)) == -2         # 2^32 packed rows
    assert workspace(1, 100, (1, 32, 1, 1 << 20, 16, 128, 0, 0)) == -8           # more query tiles than a grid has rows
