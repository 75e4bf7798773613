"""What window_attention refuses, on tensors that never reach a GPU, and the list of key tiles that the kernels walk."""
import itertools

import pytest
import torch

import lv_xattn_b200 as lvx
from lv_xattn_b200._lib import LvxError

Q, K = torch.zeros(2, 4, 3, 128), torch.zeros(2, 2, 9, 128)


@pytest.mark.parametrize("args", [
    dict(q=Q[0]),
    dict(q=Q[..., :64]),
    dict(q=Q[:, :3]),
    dict(q=Q[:, :, :0]),
    dict(q=Q.double()),
    dict(k=K.half()),
    dict(v=K[:, :, :8]),
    dict(k=K[:, :0], v=K[:, :0]),
    dict(k=K[..., :64], v=K[..., :64]),
    dict(k=K[:1], v=K[:1]),
    dict(sm_scale=0.0),
    dict(sm_scale=float("inf")),
    dict(sm_scale=float("nan")),
    dict(window=0),
    dict(sinks=-1),
    dict(query_start=-1),
    dict(query_start=1 << 28),
])
def test_tensors(args):
    with pytest.raises(ValueError):
        lvx.window_attention(**{**dict(q=Q, k=K, v=K), **args})


def test_no_cpu_path():
    with pytest.raises(LvxError):
        lvx.window_attention(Q, K, K)


def test_abi_refusals():
    import ctypes
    from lv_xattn_b200 import _lib
    lib = _lib.load()
    f, b = ctypes.c_size_t(0), ctypes.c_size_t(0)

    def workspace(shape=(1, 4, 2, 16, 16, 128, 0, 0), window=(8, 0, -1)):
        return lib.lvx_window_workspace(ctypes.byref(_lib.LvxShape(*shape)), ctypes.byref(_lib.LvxWindow(*window)),
                                        ctypes.byref(f), ctypes.byref(b))

    assert workspace() == 0 and f.value == 0 and b.value > 0      # few rows, up to eight CTAs a KV head: no partials
    assert workspace((1, 4, 2, 1, 100000, 128, 0, 0), (0, 0, -1)) == 0 and f.value > 0
    assert workspace(window=(-1, 0, -1)) == -2 and workspace(window=(8, -1, 0)) == -2 and workspace(window=(8, 0, -2)) == -2
    assert workspace((1, 4, 2, 1 << 28, 16, 128, 0, 0)) == -2 and workspace((1, 4, 2, 16, 1 << 28, 128, 0, 0)) == -2
    assert workspace((1, 4, 2, 16, 16, 128, 0, 2)) == -2 and workspace((1, 4, 2, 16, 16, 64, 0, 0)) == -2
    assert workspace((1, 1, 1, (1 << 24) + 1, 16, 128, 0, 0)) == -8
    assert workspace((1, 32, 8, 4096, 4096, 128, 0, 0)) == 0 and f.value == 0      # fills the GPU: no partials


def tiles(window, sinks, valid, p0, p1, size):
    """key_tiles of csrc/window.cuh, restated."""
    hi, lo = min(p1, valid - 1), max(0, p0 - window + 1)
    sink_end = min(sinks, hi + 1)
    ns = -(-sink_end // size) if sink_end > 0 else 0
    w0, nw = lo // size, 0
    if hi >= lo:
        nw = hi // size + 1 - w0
        ns = min(ns, w0)
    elif w0 < ns:
        w0 = ns
    return [*range(ns), *range(w0, w0 + nw)]


def test_every_seen_key_is_walked_once():
    for window, sinks, valid, p0, n in itertools.product((1, 3, 8, 100), (0, 1, 5, 9), (0, 1, 7, 24), (-3, 0, 2, 13, 40), (1, 4, 11)):
        walked = tiles(window, sinks, valid, p0, p0 + n - 1, 4)
        assert len(set(walked)) == len(walked)
        seen = {j // 4 for p in range(p0, p0 + n) for j in range(min(valid, p + 1)) if j > p - window or j < sinks}
        assert seen <= set(walked) and all(4 * t < valid for t in walked)


def test_hook_refusals():
    from lv_xattn_b200 import hf_patch
    mllama = pytest.importorskip("transformers.models.mllama.modeling_mllama")
    before = mllama.MllamaTextCrossAttention.forward, mllama.MllamaTextSelfAttention.forward
    for args in (dict(sinks=4), dict(window=0), dict(window=8, sinks=-1)):
        with pytest.raises(ValueError):
            hf_patch.patch_self_attention_forward("lv_xattn", **args)
        with pytest.raises(ValueError):
            hf_patch.install_hooks("lv_xattn", **args)
    assert before == (mllama.MllamaTextCrossAttention.forward, mllama.MllamaTextSelfAttention.forward)


@pytest.mark.parametrize("args", [dict(window=2.5), dict(window="4"), dict(sinks=0.5), dict(sinks=None), dict(query_start=1.0)])
def test_whole_numbers(args):
    with pytest.raises(ValueError, match="integer"):
        lvx.window_attention(Q, K, K, **args)


def test_whole_numbers_of_any_kind():
    """Integers of other kinds are taken: the call ends at the missing CPU path, not at its arguments."""
    with pytest.raises(LvxError):
        lvx.window_attention(Q, K, K, window=torch.tensor(4), sinks=torch.tensor(2), query_start=torch.tensor(6))
