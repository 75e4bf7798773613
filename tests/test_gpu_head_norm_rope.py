"""Head norms and rotation in one pass, against the formulas in 64 bits.

Bars: the kernel computes in fp32 and rounds once, so a value is off by at most half a step of its type (eps / 2 of the
value) and what fp32 loses on the way: the mean of 128 squares, a handful of products and one cancellation, together below
2^-19 of the largest value of its row. A weight's gradient is a sum over rows: below 2^-18 of the sum of the terms' sizes."""
import pytest
import torch

import lv_xattn_b200 as lvx

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def formula(x, w, cos, sin, eps):
    y = x
    if w is not None:
        y = w * x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    if cos is not None:
        c, s = (t.expand(x.shape[0], -1, -1)[:, :, None] for t in (cos, sin))
        y = torch.cat([y[..., :64] * c[..., :64] - y[..., 64:] * s[..., :64], y[..., 64:] * c[..., 64:] + y[..., :64] * s[..., 64:]], -1)
    return y.transpose(1, 2)


def check(got, ref, slack, name):
    eps = torch.finfo(got.dtype).eps
    bar = eps / 2 * ref.abs() + slack + torch.finfo(got.dtype).tiny
    off = (got.double() - ref).abs()
    assert got.shape == ref.shape and (off <= bar).all(), f"{name}: {(off / bar).max().item():.2f} of the bar"


def inputs(device, B, S, H, dtype, wtype, table, seed, gain=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=device, generator=g)
    x = [(gain * r(B, S, h, 128)).to(dtype) for h in H]
    w = [(1 + 0.3 * r(128)).to(wtype) for _ in H]
    angle = r(*table, 64).double() * 1000 if table else None
    cs = [f(angle).repeat(*[1] * len(table), 2).float() for f in (torch.cos, torch.sin)] if table else [None, None]
    return x, w, cs, [r(B, h, S, 128).to(dtype) for h in H]


def run_and_check(x, w, cs, grads, eps=1e-5):
    leaves = [t.detach().requires_grad_() for t in x] + [t.detach().requires_grad_() for t in w if t is not None]
    named = dict(zip(["wq" if w[0] is not None else "wk", "wk"], leaves[2:])) if any(t is not None for t in w) else {}
    out = lvx.head_norm_rope(leaves[0], leaves[1], named.get("wq"), named.get("wk"), *cs, eps=eps)
    got = torch.autograd.grad(out, leaves, grads)
    leaves64 = [t.detach().double().requires_grad_() for t in leaves]
    named64 = dict(zip(named, leaves64[2:]))
    cs64 = [None if t is None else t.double().view(-1, *t.shape[-2:]) for t in cs]
    ref = [formula(x64, named64.get(n), *cs64, eps) for x64, n in zip(leaves64, ("wq", "wk"))]
    want = torch.autograd.grad(ref, leaves64, [g.double() for g in grads])
    for name, a, b in zip(("q", "k"), out, ref):
        assert a.is_contiguous() and a.dtype == x[0].dtype
        check(a, b.detach(), 2.0 ** -19 * b.detach().abs().amax(-1, keepdim=True), name)
    for name, a, b, x64, w64 in zip(("dq", "dk"), got, want, leaves64, (named64.get("wq"), named64.get("wk"))):
        r = torch.rsqrt(x64.detach().pow(2).mean(-1, keepdim=True) + eps) if w64 is not None else 1.0
        size = grads[("dq", "dk").index(name)].double().transpose(1, 2).abs().amax(-1, keepdim=True) * 2 * r
        if w64 is not None:     # w dy and xh mean(w dy xh) cancel; both are at most that times |w| and |xh|'s largest
            size = size * w64.detach().abs().max() * (1 + (x64.detach() * r).abs().amax(-1, keepdim=True))
        check(a, b, 2.0 ** -19 * size, name)
    for (name, _), a, b in zip(named.items(), got[2:], want[2:]):
        i = ("wq", "wk").index(name)
        x64, g64 = leaves64[i].detach(), grads[i].double().transpose(1, 2)
        xh = x64 * torch.rsqrt(x64.pow(2).mean(-1, keepdim=True) + eps)
        size = ((g64.abs() + g64.roll(64, -1).abs()) * xh.abs()).sum((0, 1, 2))
        check(a, b, 2.0 ** -18 * size, f"d{name}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,S,H", [(1, 1, (1, 1)), (2, 1, (32, 8)), (3, 7, (5, 3)), (1, 333, (4, 4)), (2, 130, (12, 2))])
def test_shapes(cuda_device, B, S, H, dtype):
    run_and_check(*inputs(cuda_device, B, S, H, dtype, dtype, (B, S), 1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("norm", ["both", "q", "k", "none"])
@pytest.mark.parametrize("table", [(61,), (1, 61), None])
def test_parts(cuda_device, norm, table, dtype):
    if norm == "none" and table is None:
        pytest.skip("nothing to do")
    x, w, cs, grads = inputs(cuda_device, 2, 61, (6, 2), dtype, torch.float32, table, 2)
    w = [w[0] if norm in ("both", "q") else None, w[1] if norm in ("both", "k") else None]
    if dtype != torch.float32 and table == (61,):
        cs = [t.to(dtype) for t in cs]
    run_and_check(x, w, cs, grads)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(cuda_device, dtype):
    """Heads of a fused projection, tokens of a longer buffer, a row that starts off its alignment, transposed gradients."""
    x, w, cs, grads = inputs(cuda_device, 2, 19, (4, 2), dtype, dtype, (2, 19), 3)
    fused = torch.cat(x, 2)
    longer = torch.zeros(2, 40, 6, 128, device=cuda_device, dtype=dtype)
    longer[:, 3:22] = fused
    odd = torch.zeros(2 * 19 * 6 * 128 + 1, device=cuda_device, dtype=dtype)
    odd[1:] = fused.flatten()
    for buf in (fused, longer[:, 3:22], odd[1:].view_as(fused)):
        run_and_check([buf[:, :, :4], buf[:, :, 4:]], w, cs, [g.transpose(1, 2).contiguous().transpose(1, 2) for g in grads])


def test_extremes(cuda_device):
    """A row of zeros, values whose squares are near fp32's largest, and a NaN that stays in its row."""
    x, w, cs, grads = inputs(cuda_device, 1, 8, (2, 1), torch.bfloat16, torch.bfloat16, (8,), 4, gain=1e18)
    x[0][0, 2] = 0
    run_and_check(x, w, cs, grads)
    x[0][0, 3, 1, 5] = float("nan")
    q, k = lvx.head_norm_rope(x[0], x[1], w[0], w[1], *cs)
    bad = torch.isnan(q)
    assert bad[0, 1, 3].all() and bad.sum() == 128 and not torch.isnan(k).any()


def test_one_of_the_two(cuda_device):
    x, w, cs, grads = inputs(cuda_device, 2, 9, (4, 2), torch.bfloat16, torch.bfloat16, (9,), 5)
    both = lvx.head_norm_rope(*x, *w, *cs)
    q, none = lvx.head_norm_rope(x[0], None, w[0], None, *cs)
    assert none is None and torch.equal(q, both[0])
    none, k = lvx.head_norm_rope(None, x[1], None, w[1], *cs)
    assert none is None and torch.equal(k, both[1])
    # an output that nothing used: its input and weight get no gradient
    leaves = [t.requires_grad_() for t in (*x, *w)]
    q, k = lvx.head_norm_rope(*leaves, *cs)
    got = torch.autograd.grad(q, leaves, grads[0], allow_unused=True)
    assert got[1] is None and got[3] is None
    both = torch.autograd.grad(lvx.head_norm_rope(*leaves, *cs), leaves, grads)
    assert torch.equal(got[0], both[0]) and torch.equal(got[2], both[2])
    empty = lvx.head_norm_rope(x[0][:, :0], x[1][:, :0], *w, cs[0][:0], cs[1][:0])
    assert empty[0].shape == (2, 4, 0, 128)
    dw = torch.autograd.grad(empty, leaves[2:], [torch.zeros_like(t) for t in empty])
    assert all((t == 0).all() for t in dw)


def test_differences(cuda_device):
    """Gradients against differences of the forward, in fp32."""
    x, w, cs, grads = inputs(cuda_device, 1, 5, (2, 1), torch.float32, torch.float32, (5,), 6)
    leaves = [t.requires_grad_() for t in (*x, *w)]
    loss = lambda ts: sum((o.double() * g.double()).sum() for o, g in zip(lvx.head_norm_rope(*ts, *cs), grads))
    got = torch.autograd.grad(lvx.head_norm_rope(*leaves, *cs), leaves, grads)
    g = torch.Generator(device=cuda_device).manual_seed(7)
    with torch.no_grad():
        for i in range(4):
            step = torch.randn(leaves[i].shape, device=cuda_device, generator=g)
            h = 2.0 ** -7
            ends = [[t + s * h * step if j == i else t for j, t in enumerate(leaves)] for s in (1, -1)]
            slope = (loss(ends[0]) - loss(ends[1])) / (2 * h)
            want = (got[i].double() * step.double()).sum()
            # the third derivative's h^2 / 6 (values, weights and steps are of size 1, about 1,500 terms) and fp32's rounding / h
            assert abs(slope - want) <= 2e-3 * (got[i].double() * step.double()).abs().sum()


def test_same_result_every_time_and_in_a_graph(cuda_device):
    x, w, cs, grads = inputs(cuda_device, 2, 500, (8, 2), torch.bfloat16, torch.bfloat16, (2, 500), 8)

    def both():
        leaves = [t.detach().requires_grad_() for t in (*x, *w)]
        out = lvx.head_norm_rope(*leaves, *cs)
        return [t.detach() for t in (*out, *torch.autograd.grad(out, leaves, grads))]

    first = both()
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        again = both()
        torch.cuda.current_stream().synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = both()
    for t in x:
        t.mul_(-0.5)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(kept, both()))
