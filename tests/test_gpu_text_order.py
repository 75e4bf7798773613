"""The order in which a call's kernels stand in the stream, where one of them may start without waiting for the one before it."""
import pytest
import torch

import lv_xattn_b200 as lvx

pytestmark = pytest.mark.gpu
NAMES = ("pack_rows", "window_fwd", "fwd_rows", "shared_combine")


def kernels(call, n):
    """Names of the last n kernels of a few calls, by start (a profile may lack its first ones)."""
    from torch.profiler import ProfilerActivity, profile
    call()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA]) as p:
        for _ in range(5):
            call()
        torch.cuda.synchronize()
    events = sorted((e for e in p.events() if e.device_type == torch.autograd.DeviceType.CUDA), key=lambda e: e.time_range.start)
    return [name for e in events for name in NAMES if name in e.name][-n:]


def test_packed_rows_are_read_by_the_next_kernel(cuda_device):
    """Four tokens of eight requests: the prefix has 128 packed rows a KV head and a kernel for many rows, the own keys 16 and the
    one for few. The packing's reader follows it, and waits; the own keys' kernel, which needs nothing of it, may come beside."""
    r = lambda *s: torch.randn(*s, device=cuda_device).bfloat16()
    q, pk, pv, k, v = r(8, 8, 4, 128), r(1, 2, 700, 128), r(1, 2, 700, 128), r(8, 2, 90, 128), r(8, 2, 90, 128)
    got = kernels(lambda: lvx.shared_prefix_attention(q, pk, pv, k, v), 4)
    if not got:
        pytest.skip("no kernel activity recorded")
    assert got == ["pack_rows", "window_fwd", "fwd_rows", "shared_combine"]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_same_every_time(cuda_device, dtype):
    """Back to back on one stream, where a call's kernels meet those of the next: O and lse, and the gradients but for dQ's order,
    bit for bit."""
    gen = torch.Generator(device=cuda_device).manual_seed(8)
    r = lambda *s: torch.empty(s, device=cuda_device, dtype=dtype).normal_(generator=gen)
    for B, P, Sq, N, own in ((8, 1, 4, 700, 90), (6, 2, 40, 1500, 64), (32, 1, 1, 5000, 300), (3, 1, 77, 900, 77)):
        t = [x.requires_grad_() for x in (r(B, 8, Sq, 128), r(P, 2, N, 128), r(P, 2, N, 128), r(B, 2, own, 128), r(B, 2, own, 128))]
        do = r(B, 8, Sq, 128)

        def step():
            o, lse = lvx.shared_prefix_attention(*t, return_lse=True)
            return [o.detach(), lse, *torch.autograd.grad(o, t, do)]

        torch.cuda.synchronize()
        runs = [step() for _ in range(20)]
        for run in runs[1:]:
            for i, (a, b) in enumerate(zip(run, runs[0])):
                if i == 2:      # dQ: two roundings of the largest at most
                    assert (a.float() - b.float()).abs().max() <= torch.finfo(dtype).eps * 2 * b.float().abs().max()
                else:
                    assert torch.equal(a, b), (B, i)
