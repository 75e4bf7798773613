"""The text-side operators of the framework, as cases that can be timed and compared.

Three operators, each through its public entry point where `own` is true and in its plain form where it is not:
  "norm_rope"  head_norm_rope: RMSNorm of every query and key head and the rotary embedding in one pass, from the
               projections' layout [B, S, H, 128] to the attention kernels' [B, H, S, 128].
  "window"     window_attention: causal attention with a sliding window and a few first keys that stay visible (sinks).
               Query i of batch entry b sits at position p = i of a whole text, or p = n_b - Sq + i where a few new tokens
               come behind a cache of n_b valid keys, and sees key j where j < n_b, j <= p and (j > p - window or j < sinks).
  "shared"     shared_prefix_attention: requests that share a long prefix (a video's tokens), read once for all of them,
               with keys of their own behind it: a query sees the whole prefix, and its own keys up to its position.
Queries and keys are N(0, 1), as behind a norm, values N(0, 0.5^2), upstream gradients N(0, 1).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SCALE = 1.0 / math.sqrt(128.0)
IMAGE = 6404            # visual tokens of one image: 4 tiles of 1,601
EPS = 1e-5


def _norm_rope(name, dtype, B, S, Hq, Hkv, norm, rope, backward):
    c = dict(op="norm_rope", dtype=dtype, B=B, S=S, Hq=Hq, Hkv=Hkv, norm=norm, rope=rope, backward=backward)
    return dict(c, name=name) if name else c


def _window(name, dtype, B, Hq, Hkv, Sq, Skv, window, sinks, backward, padded=False):
    c = dict(op="window", dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, Sq=Sq, Skv=Skv, window=window, sinks=sinks, backward=backward,
             padded=padded)
    return dict(c, name=name) if name else c


def _shared(name, dtype, B, P, Hq, Hkv, Sq, prefix, Skv, backward, padded=False):
    c = dict(op="shared", dtype=dtype, B=B, P=P, Hq=Hq, Hkv=Hkv, Sq=Sq, prefix=prefix, Skv=Skv, backward=backward, padded=padded)
    return dict(c, name=name) if name else c


def listed():
    return [
        # generation: the queries and keys of four requests' new tokens
        _norm_rope("norm_rope_token", "bf16", 4, 1, 32, 8, True, True, False),
        # a training step's 2 x 4,096 text tokens, norms and rotation, with the gradients
        _norm_rope("norm_rope_train", "bf16", 2, 4096, 32, 8, True, True, True),
        # rotation alone (the Llama text layers have no head norms), an odd number of tokens, 16 heads without grouping, fp16
        _norm_rope("rope_train_fp16", "fp16", 1, 1333, 16, 16, False, True, True),
        # generation with a sliding window: eight requests at different places of a cache of 8,192 tokens
        _window("window_token", "bf16", 8, 32, 8, 1, 8192, 4096, 4, False, padded=True),
        # prefill of a long text of odd length with a window
        _window("window_prefill", "bf16", 1, 32, 8, 7777, 7777, 1024, 4, False),
        # training on 4,096 tokens with a window and sinks
        _window("window_train", "bf16", 1, 32, 8, 4096, 4096, 1024, 4, True),
        # training without a window: plain causal attention of two padded texts, 16 heads without grouping, fp16
        _window("causal_train_fp16", "fp16", 2, 16, 16, 2048, 2048, None, 0, True, padded=True),
        # the fp32 configuration, used for checking a model against its full-precision self
        _window("window_train_fp32", "fp32", 1, 32, 8, 512, 512, 128, 4, True),
        # generation: eight questions about one image, one new token each
        _shared("shared_token_image", "bf16", 8, 1, 32, 8, 1, IMAGE, 512, False, padded=True),
        # generation: 32 questions about one video of 16 frames, one new token each
        _shared("shared_token_video", "bf16", 32, 1, 32, 8, 1, 16 * IMAGE, 2048, False, padded=True),
        # prefill of four questions of odd length about four images
        _shared("shared_prefill", "bf16", 4, 1, 32, 8, 333, 4 * IMAGE, 333, False),
        # training on eight short texts, four about each of two videos
        _shared("shared_train", "bf16", 8, 2, 32, 8, 77, 4 * IMAGE, 77, True),
    ]


def _log_int(rng, lo, hi):
    """An integer from lo to hi, spread over its logarithm; most of what comes out is neither even nor a power of two."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: single tokens to texts of 8,192 tokens, prefixes of 1,000 to 102,464 visual tokens."""
    what = rng.choices(["norm_rope", "window", "shared"], [3, 5, 4])[0]
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (16, 16), (8, 2), (12, 4), (4, 4)])
    backward = rng.random() < 0.5
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if what == "norm_rope":
        B = rng.choice([1, 2, 3, 4])
        norm, rope = rng.choice([(True, True), (True, True), (True, False), (False, True)])
        return _norm_rope(None, dtype, B, _log_int(rng, 1, 8192 // B), Hq, Hkv, norm, rope, backward)
    # an fp32 case has at most the products of 512 x 8,192, another one those of window_prefill's 7,777 x 1,024
    most = (1 << 22 if dtype == "fp32" else 7777 * 1024) * 32
    if what == "window":
        B = rng.choice([1, 1, 2, 3, 8])
        window = rng.choice([None, _log_int(rng, 64, 4096), _log_int(rng, 64, 4096)])
        sinks = rng.choice([0, 4, 4, 130]) if window else 0
        if backward or rng.random() < 0.5:         # a whole text
            most_s = 4096 if backward else 7777
            Sq = Skv = _log_int(rng, 16, max(16, min(most_s, int(math.sqrt(most / (B * Hq))))))
        else:                                      # one token or a few behind a cache
            Sq = rng.choice([1, 1, 1, 2, 5, 17])
            Skv = _log_int(rng, 100, 32768)
        return _window(None, dtype, B, Hq, Hkv, Sq, max(Sq, Skv), window, sinks, backward, padded=B > 1)
    P = rng.choice([1, 1, 1, 2])
    B = P * rng.choice([1, 2, 5, 8, 16])
    Sq = _log_int(rng, 16, 512) if backward else rng.choice([1, 1, 1, 3, _log_int(rng, 16, 512)])
    prefix = _log_int(rng, 1000, max(1000, min(16 * IMAGE, most // (B * Hq * Sq))))
    return _shared(None, dtype, B, P, Hq, Hkv, Sq, prefix, Sq + _log_int(rng, 1, 1024), backward, padded=True)


def _valid(case):
    """Valid keys of each batch entry: all, then ever fewer, down to about half (behind a cache never fewer than the queries)."""
    B, length = case["B"], case["Skv"]
    least = 0 if _start(case) == 0 else case["Sq"]
    return [max(length - b * (length // (2 * B)), least) if case["padded"] else length for b in range(B)]


def _start(case):
    """Position of the first query: 0 in a whole text, None (behind the valid keys) for the newest tokens."""
    return 0 if case["op"] == "window" and case["Sq"] == case["Skv"] else None


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    B, Hq, Hkv, train = case["B"], case["Hq"], case["Hkv"], case["backward"]

    def normal(std, *shape):
        return torch.empty(*shape, device=device, dtype=dtype).normal_(0, std, generator=g)

    def leaf(std, *shape):
        return normal(std, *shape).requires_grad_(train)

    s = dict(case=case)
    if case["op"] == "norm_rope":
        S = case["S"]
        s["q"], s["k"] = leaf(1.0, B, S, Hq, 128), leaf(1.0, B, S, Hkv, 128)
        if case["norm"]:
            s["wq"], s["wk"] = ((1 + 0.1 * normal(1.0, 128)).requires_grad_(train) for _ in range(2))
        if case["rope"]:
            # tokens of a chunk that starts somewhere in the text, its own place for each batch entry
            start = torch.randint(0, 100000, (B, 1), device=device, generator=g)
            pos = (start + torch.arange(S, device=device)).double()
            angle = pos[..., None] * 500000.0 ** (-torch.arange(64, device=device).double() / 64)
            s["cos"], s["sin"] = (f(angle).repeat(1, 1, 2).float() for f in (torch.cos, torch.sin))
        if train:
            s["gq"], s["gk"] = normal(1.0, B, Hq, S, 128), normal(1.0, B, Hkv, S, 128)
        return s
    Sq, Skv = case["Sq"], case["Skv"]
    s["q"] = leaf(1.0, B, Hq, Sq, 128)
    s["k"], s["v"] = leaf(1.0, B, Hkv, Skv, 128), leaf(0.5, B, Hkv, Skv, 128)
    if case["op"] == "shared":
        s["pk"], s["pv"] = leaf(1.0, case["P"], Hkv, case["prefix"], 128), leaf(0.5, case["P"], Hkv, case["prefix"], 128)
    s["valid"] = torch.tensor(_valid(case), device=device, dtype=torch.int32) if case["padded"] else None
    if train:
        s["grad"] = normal(1.0, B, Hq, Sq, 128)
    return s


# ---- plain forms ------------------------------------------------------------------------------------------
def _rotate(x, cos, sin):
    """[..., 128] with its halves as the two coordinates of 64 planes; cos and sin broadcast against it."""
    return x * cos + torch.cat([-x[..., 64:], x[..., :64]], -1) * sin


def _rotate_back(g, cos, sin):
    gs = g * sin
    return g * cos + torch.cat([gs[..., 64:], -gs[..., :64]], -1)


def _norm_rope_plain(x, w, cos, sin, g):
    """Output [B, H, S, 128] of x [B, S, H, 128]; with an upstream gradient g also dx, and dw where there is a weight."""
    dtype, x = x.dtype, x.detach().float()
    rstd = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS) if w is not None else None
    y = x * rstd * w.detach().float() if w is not None else x
    if cos is not None:
        cos, sin = cos[:, :, None], sin[:, :, None]
        y = _rotate(y, cos, sin)
    out = [y.transpose(1, 2).contiguous().to(dtype)]
    if g is not None:
        dy = g.float().transpose(1, 2)
        if cos is not None:
            dy = _rotate_back(dy, cos, sin)
        if w is not None:
            xhat, wdy = x * rstd, dy * w.detach().float()
            out.append((rstd * (wdy - xhat * (wdy * xhat).mean(-1, keepdim=True))).to(dtype))
            out.append((dy * xhat).sum((0, 1, 2)).to(dtype))
        else:
            out.append(dy.contiguous().to(dtype))
    return out


def _visible(Sq, Skv, valid, start, window, sinks, B, device):
    """[B, Sq, Skv]: which keys a query sees."""
    n = valid.long() if valid is not None else torch.full((B,), Skv, device=device)
    first = n - Sq if start is None else torch.full_like(n, start)
    p = first[:, None, None] + torch.arange(Sq, device=device)[:, None]
    j = torch.arange(Skv, device=device)
    seen = (j <= p) & (j < n[:, None, None])
    if window is not None:
        seen &= (j > p - window) | (j < sinks)
    return seen


def _by_group(x, Hkv):
    """[B, Hq, Sq, ...] -> [B, Hkv, g * Sq, ...]"""
    return x.reshape(x.shape[0], Hkv, -1, *x.shape[3:])


def _softmax(scores):
    """Probabilities and log-sum-exp of the last axis; rows without any key get 0 and -inf."""
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.clamp_min(torch.finfo(scores.dtype).min))
    total = p.sum(-1, keepdim=True)
    return p / total.clamp_min(torch.finfo(scores.dtype).tiny), (top + torch.log(total)).squeeze(-1)


def _window_plain(s):
    case, dtype = s["case"], s["q"].dtype
    B, Hq, Hkv, Sq, Skv = (case[n] for n in ("B", "Hq", "Hkv", "Sq", "Skv"))
    q, k, v = (s[n].detach().float() for n in "qkv")
    q = _by_group(q, Hkv)
    seen = _visible(Sq, Skv, s["valid"], _start(case), case["window"], case["sinks"], B, q.device)
    scores = (q @ k.transpose(-1, -2) * SCALE).view(B, Hq, Sq, Skv).masked_fill_(~seen[:, None], -math.inf)
    p, lse = _softmax(scores)
    p = _by_group(p, Hkv)
    o = p @ v
    if not case["backward"]:
        return [o.reshape(B, Hq, Sq, 128).to(dtype), lse.reshape(B * Hq, Sq)]
    do = _by_group(s["grad"].float(), Hkv)
    ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True)) * SCALE
    grads = (ds @ k).reshape(B, Hq, Sq, 128), ds.transpose(-1, -2) @ q, p.transpose(-1, -2) @ do
    return [t.to(dtype) for t in (o.reshape(B, Hq, Sq, 128), *grads)]


def _shared_plain(s):
    case, dtype = s["case"], s["q"].dtype
    B, P, Hq, Hkv, Sq, Skv, prefix = (case[n] for n in ("B", "P", "Hq", "Hkv", "Sq", "Skv", "prefix"))
    q, k, v, pk, pv = (s[n].detach().float() for n in ("q", "k", "v", "pk", "pv"))

    def to_prefix(x):       # [B, Hkv, g * Sq, n] -> [P, Hkv, (B / P) * g * Sq, n]
        return x.reshape(P, B // P, Hkv, -1, x.shape[-1]).transpose(1, 2).reshape(P, Hkv, -1, x.shape[-1])

    def from_prefix(x):
        return x.reshape(P, Hkv, B // P, -1, x.shape[-1]).transpose(1, 2).reshape(B, Hkv, -1, x.shape[-1])

    q = _by_group(q, Hkv)
    seen = _visible(Sq, Skv, s["valid"], None, None, 0, B, q.device)
    mine = (q @ k.transpose(-1, -2) * SCALE).view(B, Hq, Sq, Skv).masked_fill_(~seen[:, None], -math.inf)
    scores = torch.cat([from_prefix(to_prefix(q) @ pk.transpose(-1, -2) * SCALE), _by_group(mine, Hkv)], -1)
    p, lse = _softmax(scores)
    pp, po = to_prefix(p[..., :prefix]), p[..., prefix:]
    o = from_prefix(pp @ pv) + po @ v
    if not case["backward"]:
        return [o.reshape(B, Hq, Sq, 128).to(dtype), lse.reshape(B * Hq, Sq)]
    do = _by_group(s["grad"].float(), Hkv)
    delta = (do * o).sum(-1, keepdim=True)
    dsp = pp * (to_prefix(do) @ pv.transpose(-1, -2) - to_prefix(delta)) * SCALE
    dso = po * (do @ v.transpose(-1, -2) - delta) * SCALE
    grads = [(from_prefix(dsp @ pk) + dso @ k).reshape(B, Hq, Sq, 128), dsp.transpose(-1, -2) @ to_prefix(q),
             pp.transpose(-1, -2) @ to_prefix(do), dso.transpose(-1, -2) @ q, po.transpose(-1, -2) @ do]
    return [t.to(dtype) for t in (o.reshape(B, Hq, Sq, 128), *grads)]


def run(s):
    """Forward: the outputs (attention with its log-sum-exp). Training: the output and the gradients of every input."""
    case = s["case"]
    train = case["backward"]
    if not own:
        if case["op"] == "window":
            return _window_plain(s)
        if case["op"] == "shared":
            return _shared_plain(s)
        cos, sin = s.get("cos"), s.get("sin")
        return [*_norm_rope_plain(s["q"], s.get("wq"), cos, sin, s.get("gq")),
                *_norm_rope_plain(s["k"], s.get("wk"), cos, sin, s.get("gk"))]
    import lv_xattn_b200 as lvx
    if case["op"] == "norm_rope":
        wq, wk = s.get("wq"), s.get("wk")
        q, k = lvx.head_norm_rope(s["q"], s["k"], wq, wk, s.get("cos"), s.get("sin"), eps=EPS)
        if not train:
            return [q, k]
        leaves = [s["q"], s["k"]] + ([wq, wk] if wq is not None else [])
        dq, dk, *dw = torch.autograd.grad((q, k), leaves, (s["gq"], s["gk"]))
        return [q.detach(), dq, *dw[:1], k.detach(), dk, *dw[1:]]
    if case["op"] == "window":
        out = lvx.window_attention(s["q"], s["k"], s["v"], SCALE, window=case["window"], sinks=case["sinks"],
                                   kv_valid_len=s["valid"], query_start=_start(case), return_lse=not train)
        leaves = [s["q"], s["k"], s["v"]]
    else:
        out = lvx.shared_prefix_attention(s["q"], s["pk"], s["pv"], s["k"], s["v"], SCALE, kv_valid_len=s["valid"],
                                          return_lse=not train)
        leaves = [s["q"], s["pk"], s["pv"], s["k"], s["v"]]
    return [out.detach(), *torch.autograd.grad(out, leaves, s["grad"])] if train else list(out)


# ---- what a pass cannot do without ------------------------------------------------------------------------
def _pairs(case, n):
    """Visible (query, key) pairs of a batch entry with n valid keys, and the keys that any query sees."""
    Sq, window, sinks = case["Sq"], case.get("window"), case.get("sinks", 0)
    first = n - Sq if _start(case) is None else 0
    p = torch.arange(first, first + Sq)
    hi = (p + 1).clamp_max(n)
    lo = torch.zeros_like(p) if window is None else (p - window + 1).clamp_min(0)
    low = int(lo[0])
    return int(((hi - lo).clamp_min(0) + lo.clamp_max(min(sinks, n))).sum()), n - low + min(low, sinks)


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    B, Hq, Hkv, train = case["B"], case["Hq"], case["Hkv"], case["backward"]
    if case["op"] == "norm_rope":
        values = B * case["S"] * (Hq + Hkv) * 128
        tables = 2 * 4 * 128 * B * case["S"] if case["rope"] else 0
        # forward: x in, out; backward: the gradient in too, and dx out
        return {"bytes": es * values * (4 if train else 2) + tables, "flops": values * (20 if train else 8)}
    Sq = case["Sq"]
    pairs, keys = (sum(t) for t in zip(*(_pairs(case, n) for n in _valid(case))))
    all_keys = B * case["Skv"]
    if case["op"] == "shared":
        pairs += B * Sq * case["prefix"]
        keys += case["P"] * case["prefix"]
        all_keys += case["P"] * case["prefix"]
    q_bytes, kv_bytes = es * B * Hq * Sq * 128, 2 * es * Hkv * 128
    if train:     # q, k, v, dO in; o, dQ, dK, dV out (gradients of padded keys are written too)
        return {"bytes": 4 * q_bytes + kv_bytes * (keys + all_keys), "flops": 7 * 2 * 128 * Hq * pairs}
    return {"bytes": 2 * q_bytes + 4 * B * Hq * Sq + kv_bytes * keys, "flops": 2 * 2 * 128 * Hq * pairs}


# ---- the same in 64 bits, from the definitions ------------------------------------------------------------
def _norm_rope64(x, w, cos, sin, g):
    leaves = [x.detach().double().requires_grad_()] + ([w.detach().double().requires_grad_()] if w is not None else [])
    y = leaves[0]
    if w is not None:
        y = leaves[1] * y / torch.sqrt((y * y).sum(-1, keepdim=True) / 128 + EPS)
    if cos is not None:
        c, s = cos.double()[:, :, None], sin.double()[:, :, None]
        a, b = y[..., :64], y[..., 64:]
        y = torch.cat([a * c[..., :64] - b * s[..., :64], b * c[..., 64:] + a * s[..., 64:]], -1)
    y = y.permute(0, 2, 1, 3)
    return [y.detach(), *(torch.autograd.grad(y, leaves, g.double()) if g is not None else [])]


def _attention64(q, keys, values, seen, do):
    """One query head [Sq, 128] over keys and values that lists of tensors hold one after the other, `seen` [Sq, number of
    keys] or None: o, lse, and with an upstream gradient dq and the gradients of every tensor of the lists."""
    k, v = torch.cat(keys), torch.cat(values)
    scores = q @ k.T * SCALE
    if seen is not None:
        scores[~seen] = -math.inf
    lse = torch.logsumexp(scores, -1)
    p = torch.exp(scores - torch.where(lse == -math.inf, 0.0, lse)[:, None])
    o = p @ v
    if do is None:
        return o, lse
    ds = p * (do @ v.T - (do * o).sum(-1, keepdim=True)) * SCALE
    sizes = [t.shape[0] for t in keys]
    return o, lse, ds @ k, (ds.T @ q).split(sizes), (p.T @ do).split(sizes)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm_rope":
        cos, sin = s.get("cos"), s.get("sin")
        return [*_norm_rope64(s["q"], s.get("wq"), cos, sin, s.get("gq")), *_norm_rope64(s["k"], s.get("wk"), cos, sin, s.get("gk"))]
    B, Hq, Hkv, Sq, Skv = (case[n] for n in ("B", "Hq", "Hkv", "Sq", "Skv"))
    names = ("pk", "pv", "k", "v") if case["op"] == "shared" else ("k", "v")
    t = {n: s[n].detach().double() for n in ("q", *names)}
    o, lse = torch.zeros_like(t["q"]), t["q"].new_zeros(B, Hq, Sq)
    grads = {n: torch.zeros_like(x) for n, x in t.items()}
    for b, n in enumerate(_valid(case)):
        seen = torch.zeros(Sq, Skv, dtype=torch.bool, device="cuda")
        for i in range(Sq):       # a query's keys are two ranges: the window behind it, and the sinks
            p = i if _start(case) == 0 else n - Sq + i
            seen[i, :min(p + 1, n)] = True
            if case.get("window") is not None:
                seen[i, min(case["sinks"], n):max(p - case["window"] + 1, min(case["sinks"], n))] = False
        for h in range(Hq):
            at = [(m, b * case["P"] // B if m[0] == "p" else b, h * Hkv // Hq) for m in names]
            keys, values = ([t[m][i, j] for m, i, j in at if m[-1] == kind] for kind in "kv")
            mask = seen if len(keys) == 1 else torch.cat([seen.new_ones(Sq, keys[0].shape[0]), seen], 1)
            got = _attention64(t["q"][b, h], keys, values, mask, s["grad"][b, h].double() if case["backward"] else None)
            o[b, h], lse[b, h] = got[:2]
            if case["backward"]:
                grads["q"][b, h] = got[2]
                for kind, parts in zip("kv", got[3:]):
                    for (m, i, j), part in zip([a for a in at if a[0][-1] == kind], parts):
                        grads[m][i, j] += part
    return [o, *(grads[n] for n in ("q", *names))] if case["backward"] else [o, lse.view(B * Hq, Sq)]
