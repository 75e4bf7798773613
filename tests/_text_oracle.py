"""Attention over masked keys in 64 bits, with the bars that follow from what the kernels round.

For 16-bit types e is half a step of the type (eps / 2). The kernels round P for the product with V (e of each term), O when
it is stored (e of it), and in the backward P and dS (e each) and the results (e). delta = rowsum(dO O) is taken from the
rounded O. fp16 has subnormal values: a P or dS below 2^-14 errs by up to 2^-25 whatever its size. Sums, exponentials and
scores are fp32: 2^-14 of a sum's terms is far more than they lose at these sizes. fp32 inputs are rounded nowhere on the way; three
tf32 products leave 2^-21 of each term and a few additions, taken as 2^-18 of the terms' sizes."""
import math

import torch


def unit(dtype):
    """(e, absolute part, what fp32 sums may lose)."""
    if dtype == torch.float32:
        return 0.0, 0.0, 2.0 ** -18
    return torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0, 2.0 ** -14


def masked_attention(q, k, v, seen, scale, do=None):
    """q [n, 128], k and v [m, 128], seen [n, m] bool: dict of o, lse (and dq, dk, dv) with their bars, in 64 bits. Keys that no
    row sees are taken as zeros, whatever they hold."""
    e, tiny, lost = unit(q.dtype)
    q, k, v = q.double(), k.double(), v.double()
    k, v = (torch.where(seen.any(0)[:, None], t, 0.0) for t in (k, v))
    s = (q @ k.T * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[:, None]).masked_fill(~seen, 0.0)
    o = p @ v
    o_bar = (e + lost) * (p @ v.abs()) + e * o.abs() + tiny * (seen.double() @ v.abs())
    out = dict(o=(o, o_bar), lse=(lse, torch.full_like(lse, 2.0 ** -14)))
    if do is None:
        return out
    do = do.double()
    delta, d_delta = (do * o).sum(-1, keepdim=True), (do.abs() * o_bar).sum(-1, keepdim=True)
    dp = do @ v.T
    ds = p * (dp - delta)
    size = p * (do.abs() @ v.abs().T + (do.abs() * o.abs()).sum(-1, keepdim=True))
    ds_bar = 2 * e * ds.abs() + lost * size + p * d_delta + tiny * seen * (1 + (dp - delta).abs())
    p_bar = (e + lost) * p + tiny * seen
    for name, x, bar in (("dq", ds @ k * scale, ds_bar @ k.abs() * scale), ("dk", ds.T @ q * scale, ds_bar.T @ q.abs() * scale),
                         ("dv", p.T @ do, p_bar.T @ do.abs())):
        out[name] = (x, bar + e * x.abs())
    return out


def visible(n, sq, skv, window, sinks, start):
    """[sq, skv]: the keys that a batch entry's queries see, from the definition."""
    p = (n - sq if start is None else start) + torch.arange(sq)[:, None]
    j = torch.arange(skv)
    seen = (j < n) & (j <= p)
    return seen if window is None else seen & ((j > p - window) | (j < sinks))


def check(got, ref, bar, name):
    """Every value within its bar (and half a step of fp32 or a subnormal of its type), -inf where the reference has it."""
    got, fin = got.double(), torch.isfinite(ref)
    assert got.shape == ref.shape, name
    assert torch.equal(got[~fin], ref[~fin]), f"{name}: not the same infinite values"
    assert torch.isfinite(got[fin]).all(), f"{name}: non-finite values"
    bar = bar + 2.0 ** -23 * ref.abs() + 2.0 ** -24
    off = ((got - ref).abs() / bar)[fin]
    assert off.numel() == 0 or off.max() <= 1, f"{name}: {off.max().item():.2f} of the bar"
