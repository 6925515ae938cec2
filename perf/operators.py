"""Measured cases of the operators around a video transformer's flat attention: rotary positions over several
axes (with the query / key RMS norm and the change to head-major order in the same pass), and cross attention
to an encoder's states of another length; each forward and backward.

``own`` selects the framework's kernels; otherwise ``run`` computes the same thing with elementary torch
operations in float32, rounded once at the end.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------- cases
def _rotary(name, way, *, grid, batch, heads, kv_heads, dim, axes, pairs, norm, heads_first, dtype):
    """grid "t,h,w" (positions of a video latent) or "n" (a sequence with positions from 0, or one late
    position each when n is 1)."""
    return {"name": name, "op": "rotary", "way": way, "grid": grid, "batch": batch, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "axes": axes, "pairs": pairs, "norm": norm,
            "heads_first": heads_first, "dtype": dtype}


def _cross(name, way, *, batch, queries, keys, heads, kv_heads, dim, mask, heads_first, dtype):
    """mask: none, lengths (padded batch, one entry may be empty), bool (key mask), bias (additive key mask whose
    masked places hold the type's lowest value) or pairs (a mask for each query and key, some rows empty)."""
    return {"name": name, "op": "cross", "way": way, "batch": batch, "queries": queries, "keys": keys,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "mask": mask, "heads_first": heads_first,
            "dtype": dtype}


def listed():
    return [
        # q and k of a whole 1344 x 768, 124-frame latent (24 heads) before flat attention: norm, rotation and
        # the move to head-major rows in one pass
        _rotary("rotary_video", "forward", grid="32,48,84", batch=1, heads=24, kv_heads=24, dim=128,
                axes="44,42,42", pairs="interleaved", norm=True, heads_first=True, dtype="bf16"),
        # the same layer at the small latent while an adapter is trained: dq, dk and the two norm weights'
        # gradients
        _rotary("rotary_video_grad", "backward", grid="16,32,32", batch=2, heads=24, kv_heads=24, dim=128,
                axes="44,42,42", pairs="interleaved", norm=True, heads_first=True, dtype="bf16"),
        # one new token for each of 16 sequences, grouped key heads: a launch, nothing else
        _rotary("rotary_token", "forward", grid="1", batch=16, heads=24, kv_heads=8, dim=128, axes="32,48,48",
                pairs="half", norm=True, heads_first=False, dtype="f16"),
        # an odd latent with narrow heads, a partial rotation and no norm, in float32
        _rotary("rotary_odd", "forward", grid="5,17,29", batch=1, heads=5, kv_heads=5, dim=80, axes="16,24,24",
                pairs="half", norm=False, heads_first=False, dtype="f32"),
        # the whole latent against 512 prompt tokens, head-major as flat attention holds its rows
        _cross("cross_video", "forward", batch=1, queries=129024, keys=512, heads=24, kv_heads=24, dim=128,
               mask="none", heads_first=True, dtype="bf16"),
        # a prompt and its negative in one padded batch, at the small latent
        _cross("cross_prompts", "forward", batch=2, queries=16384, keys=256, heads=24, kv_heads=24, dim=128,
               mask="lengths", heads_first=False, dtype="bf16"),
        # a short clip against a long condition (the states of a reference clip)
        _cross("cross_long", "forward", batch=1, queries=4096, keys=16384, heads=24, kv_heads=24, dim=128,
               mask="none", heads_first=False, dtype="bf16"),
        # one new token for each of 16 sequences over its encoder's states, grouped key heads
        _cross("cross_token", "forward", batch=16, queries=1, keys=2000, heads=24, kv_heads=8, dim=128,
               mask="lengths", heads_first=False, dtype="bf16"),
        # a small odd image against 77 tokens with narrow heads and an additive mask
        _cross("cross_odd", "forward", batch=2, queries=1001, keys=77, heads=10, kv_heads=10, dim=72,
               mask="bias", heads_first=False, dtype="f16"),
        # gradients of the small latent's cross attention
        _cross("cross_video_grad", "backward", batch=1, queries=16384, keys=512, heads=24, kv_heads=24, dim=128,
               mask="none", heads_first=True, dtype="bf16"),
        # gradients with a mask for each region and token, shared key heads, odd sizes and empty rows
        _cross("cross_regions_grad", "backward", batch=3, queries=777, keys=130, heads=12, kv_heads=4, dim=64,
               mask="pairs", heads_first=False, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "cross"])
    way = rng.choice(["forward", "forward", "backward"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    group = rng.choice([1, 1, 2, 3])
    batch = rng.choice([1, 1, 2, 3, 5])
    if op == "rotary":
        dim, axes = rng.choice([(128, "44,42,42"), (128, "32,48,48"), (128, "128"), (64, "20,22,22"), (80, "16,24,24"),
                                (96, "32,32"), (72, "24,24,24")])
        kv = rng.choice([1, 2, 5, 8])
        if way == "forward" and rng.random() < 0.25:
            dtype = "f32"
        values = 129024 * 24 * 128 / (8 if way == "backward" else 2 if dtype == "f32" else 1)
        tokens = _log(rng, 1, min(129024, values / (batch * kv * group * dim)))
        if axes.count(",") == 2:
            h, w = rng.randint(1, 48), rng.randint(1, 84)
            if tokens < h * w:
                h, w = 1, min(tokens, 84)
            grid = "%d,%d,%d" % (min(61, tokens // (h * w)), h, w)
        else:
            grid = str(min(tokens, 32768))
        return _rotary("", way, grid=grid, batch=batch, heads=kv * group, kv_heads=kv, dim=dim, axes=axes,
                       pairs=rng.choice(["interleaved", "half"]), norm=rng.random() < 0.6,
                       heads_first=rng.random() < 0.5, dtype=dtype)
    dim = rng.choice([32, 64, 64, 72, 96, 128, 128, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * group
    # training runs no single tokens (and one key alone has no gradient to compare: its weight is always 1)
    least = 16 if way == "backward" else 1
    keys = _log(rng, least, 16384)
    # the plain form holds float32 scores of every head: at most a few gigabytes
    most = 129024 * 512 * 24 / 2 / (4 if way == "backward" else 1) / (batch * heads * keys)
    queries = _log(rng, least, max(least, min(129024, most)))
    mask = rng.choice(["none", "lengths", "bool", "bias", "pairs"])
    if mask == "pairs":
        queries = max(least, min(queries, int(4e8 / (batch * keys))))
    return _cross("", way, batch=batch, queries=queries, keys=keys, heads=heads, kv_heads=kv, dim=dim, mask=mask,
                  heads_first=rng.random() < 0.5, dtype=dtype)


# ---------------------------------------------------------------------------------------------- inputs
def _ints(text):
    return [int(x) for x in text.replace("x", ",").split(",")]


def _tokens(case):
    return math.prod(_ints(case["grid"]))


def _key_lengths(case):
    """A padded batch's key counts before their seeded shuffle: a ramp up to all keys; from three entries on, the
    first is empty."""
    b, m = case["batch"], case["keys"]
    return [m * i // (b - 1) for i in range(b)] if b > 2 else [m * (i + 1) // b for i in range(b)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)

    b, d, hq, hk = case["batch"], case["dim"], case["heads"], case["kv_heads"]
    s = {"case": case}
    if case["op"] == "rotary":
        n, axes = _tokens(case), _ints(case["axes"])
        s["axes"] = tuple(axes)
        # float32 frequencies of every pair, theta ** (-2 i / width) over each axis' own width
        freqs = [10000.0 ** (-2.0 * i / w) for w in axes for i in range(w // 2)]
        s["freqs"] = torch.tensor(freqs, dtype=torch.float32, device="cuda")
        s["axis_of"] = torch.tensor([a for a, w in enumerate(axes) for _ in range(w // 2)], device="cuda")
        # q and k as the projection leaves them: slices of one [tokens, (q | k) heads, dim] buffer
        qk = normal(b, n, hq + hk, d, scale=1.7)
        s["q"], s["k"] = qk[:, :, :hq], qk[:, :, hq:]
        if "," in case["grid"]:
            t, h, w = _ints(case["grid"])
            start = torch.randint(0, 8, (3,), generator=gen, device="cuda", dtype=torch.int32)
            at = torch.arange(n, device="cuda", dtype=torch.int32)
            pos = torch.stack([at // (h * w), at // w % h, at % w], -1) + start
            pos = pos.expand(b, n, 3)
        else:
            first = torch.randint(0, 4096 if n == 1 else 8, (b, 1, 1), generator=gen, device="cuda",
                                  dtype=torch.int32)
            at = torch.arange(n, device="cuda", dtype=torch.int32)[None, :, None]
            side = 64 if len(axes) > 1 or case["dtype"] == "f32" else 1 << 30
            pos = (first + at).expand(b, n, len(axes)) % side
        s["positions"] = pos.to(torch.int32).contiguous()
        s["q_weight"] = 1 + normal(d, dtype=torch.float32, scale=0.1) if case["norm"] else None
        s["k_weight"] = 1 + normal(d, dtype=torch.float32, scale=0.1) if case["norm"] else None
        if case["way"] == "backward":
            shape = (lambda h: (b, h, n, d)) if case["heads_first"] else (lambda h: (b, n, h, d))
            s["dq"], s["dk"] = normal(*shape(hq)), normal(*shape(hk))
        return s

    n, m = case["queries"], case["keys"]
    shape = (lambda r, h: (b, h, r, d)) if case["heads_first"] else (lambda r, h: (b, r, h, d))
    # logits of a trained layer spread over a few units
    s["q"] = normal(*shape(n, hq), scale=2.0)
    s["k"], s["v"] = normal(*shape(m, hk)), normal(*shape(m, hk))
    s["lengths"] = s["mask"] = None
    if case["mask"] == "lengths":
        order = torch.randperm(b, generator=gen, device="cuda")
        s["lengths"] = torch.tensor(_key_lengths(case), dtype=torch.int32, device="cuda")[order]
    elif case["mask"] in ("bool", "bias"):
        keep = torch.rand((b, 1, 1, m), generator=gen, device="cuda") < 0.8
        keep[..., 0] = True
        if case["mask"] == "bool":
            s["mask"] = keep
        else:
            soft = torch.rand((b, 1, 1, m), generator=gen, device="cuda") - 0.5
            s["mask"] = torch.where(keep, soft, torch.finfo(dt).min).to(dt)
    elif case["mask"] == "pairs":
        s["mask"] = torch.rand((b, 1, n, m), generator=gen, device="cuda") < 0.5
        s["mask"] &= (torch.rand((b, 1, n, 1), generator=gen, device="cuda") < 0.95)
    if case["way"] == "backward":
        with torch.no_grad():
            s["out"], s["lse"] = _attend(s)
        s["dout"] = normal(*shape(n, hq))
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _angles(s):
    angle = s["positions"].float()[..., s["axis_of"]] * s["freqs"]           # [b, n, pairs]
    return angle.cos()[:, :, None], angle.sin()[:, :, None]


def _turn(x, cos, sin, pairs):
    """Rotates the pairs of x [b, n, h, d] (float32); what lies past the rotated width stays."""
    r = 2 * cos.shape[-1]
    if pairs == "interleaved":
        x0, x1 = x[..., 0:r:2], x[..., 1:r:2]
    else:
        x0, x1 = x[..., :r // 2], x[..., r // 2:r]
    y0, y1 = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    y = torch.stack([y0, y1], -1).flatten(-2) if pairs == "interleaved" else torch.cat([y0, y1], -1)
    return torch.cat([y, x[..., r:]], -1)


def _rotate(s, x, weight):
    c = s["case"]
    cos, sin = _angles(s)
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight
    y = _turn(x, cos, sin, c["pairs"]).to(DTYPES[c["dtype"]])
    return y.transpose(1, 2).contiguous() if c["heads_first"] else y


def _rotate_back(s, dy, x, weight):
    c = s["case"]
    cos, sin = _angles(s)
    dy = dy.transpose(1, 2) if c["heads_first"] else dy
    g = _turn(dy.float(), cos, -sin, c["pairs"])
    if weight is None:
        return g.to(DTYPES[c["dtype"]]), None
    x = x.float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    dw = (g * x * r).sum((0, 1, 2))
    g = g * weight
    dx = r * (g - x * (r * r) * (g * x).mean(-1, keepdim=True))
    return dx.to(DTYPES[c["dtype"]]), dw


def _scores(s):
    """float32 scores [b, hk, group, n, m] with what the mask excludes at -inf, the operands head-major, and the
    excluded keys [b, 1, m, 1] (or None)."""
    c = s["case"]
    q, k, v = (x.float() if c["heads_first"] else x.transpose(1, 2).float() for x in (s["q"], s["k"], s["v"]))
    b, hq, n, d = q.shape
    q = q.reshape(b, c["kv_heads"], -1, n, d)
    x = q @ k[:, :, None].transpose(-1, -2) / math.sqrt(d)
    if s["lengths"] is not None:
        x = x.masked_fill(torch.arange(c["keys"], device="cuda") >= s["lengths"][:, None, None, None, None], -math.inf)
    elif s["mask"] is not None and s["mask"].dtype == torch.bool:
        x = x.masked_fill(~s["mask"][:, :, None], -math.inf)
    elif s["mask"] is not None:
        x = x + s["mask"][:, :, None].float()
    return x, q, k, v


def _softmax(x):
    """Rows of probabilities and their log sums; a row with nothing in it is zero, its log sum -inf."""
    top = x.amax(-1, keepdim=True)
    p = (x - top.clamp_min(torch.finfo(torch.float32).min)).exp()
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    return p, (top + total.log()).squeeze(-1)


def _attend(s):
    c = s["case"]
    x, q, k, v = _scores(s)
    p, lse = _softmax(x)
    out = (p @ v[:, :, None]).flatten(1, 2).to(DTYPES[c["dtype"]])
    return (out if c["heads_first"] else out.transpose(1, 2).contiguous()), lse.flatten(1, 2)


def _attend_back(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    x, q, k, v = _scores(s)
    p, _ = _softmax(x)
    do = (s["dout"] if c["heads_first"] else s["dout"].transpose(1, 2)).float().reshape(q.shape)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    dp = do @ v[:, :, None].transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(q.shape[-1])
    dq = (ds @ k[:, :, None]).flatten(1, 2)
    dk = (ds.transpose(-1, -2) @ q).sum(2)
    grads = (dq, dk, dv)
    return [g.to(dt) if c["heads_first"] else g.transpose(1, 2).to(dt).contiguous() for g in grads]


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if own:
        import htrc_b200
        if c["op"] == "rotary":
            kw = dict(axes=s["axes"], pairs=c["pairs"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                      heads_first=c["heads_first"])
            if c["way"] == "forward":
                return htrc_b200.rotary_qk(s["q"], s["k"], s["positions"], **kw)
            return htrc_b200.rotary_qk_backward(s["dq"], s["dk"], s["q"], s["k"], s["positions"], **kw)
        kw = dict(key_lengths=s["lengths"], mask=s["mask"], heads_first=c["heads_first"])
        if c["way"] == "forward":
            return htrc_b200.cross_attention(s["q"], s["k"], s["v"], return_lse=True, **kw)
        return htrc_b200.cross_attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], **kw)
    if c["op"] == "rotary":
        if c["way"] == "forward":
            return _rotate(s, s["q"], s["q_weight"]), _rotate(s, s["k"], s["k_weight"])
        dq, dqw = _rotate_back(s, s["dq"], s["q"], s["q_weight"])
        dk, dkw = _rotate_back(s, s["dk"], s["k"], s["k_weight"])
        return dq, dk, dqw, dkw
    return _attend(s) if c["way"] == "forward" else _attend_back(s)


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    b, d, hq, hk = case["batch"], case["dim"], case["heads"], case["kv_heads"]
    if case["op"] == "rotary":
        n, axes = _tokens(case), _ints(case["axes"])
        values = b * n * (hq + hk) * d
        weights = 2 * d * 4 * (case["norm"] is True)
        if case["way"] == "forward":
            return {"bytes": 2 * values * es + b * n * len(axes) * 4 + weights,
                    "flops": values * (3 + 4 * case["norm"])}
        moved = (3 if case["norm"] else 2) * values * es
        return {"bytes": moved + b * n * len(axes) * 4 + 2 * weights, "flops": values * (3 + 12 * case["norm"])}
    n, m = case["queries"], case["keys"]
    held = sum(_key_lengths(case)) if case["mask"] == "lengths" else b * m
    pairs = held * n * hq
    q, kv, rows = b * n * hq * d * es, 2 * held * hk * d * es, b * n * hq * 4
    mask = {"none": 0, "lengths": 4 * b, "bool": b * m, "bias": 2 * b * m, "pairs": b * n * m}[case["mask"]]
    if case["way"] == "forward":
        return {"bytes": 2 * q + kv + rows + mask, "flops": 4 * pairs * d}
    return {"bytes": 4 * q + 2 * kv + rows + mask, "flops": 10 * pairs * d}


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_rotary(s):
    """Complex numbers: each pair is one, and a rotation the product with exp(i * angle)."""
    c = s["case"]
    freq = torch.cat([10000.0 ** (-torch.arange(0, w, 2, dtype=torch.float64, device="cuda") / w) for w in s["axes"]])
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       s["positions"].double()[..., s["axis_of"]] * freq)[:, :, None]
    r = 2 * freq.numel()

    def rotated(x, by):
        z = x[..., :r].unflatten(-1, (-1, 2)) if c["pairs"] == "interleaved" else \
            x[..., :r].unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * by)
        z = z.flatten(-2) if c["pairs"] == "interleaved" else z.transpose(-1, -2).flatten(-2)
        return torch.cat([z, x[..., r:]], -1)

    def forward(x, w):
        x = x.double()
        if w is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * w.double()
        y = rotated(x, turn)
        return y.transpose(1, 2).contiguous() if c["heads_first"] else y

    def backward(dy, x, w):
        dy, x = (dy.transpose(1, 2) if c["heads_first"] else dy).double(), x.double()
        g = rotated(dy, turn.conj())
        if w is None:
            return g, None
        size = (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt()
        unit = x / size
        h = g * w.double()
        return (h - unit * (h * unit).sum(-1, keepdim=True) / x.shape[-1]) / size, (g * unit).sum((0, 1, 2))

    if c["way"] == "forward":
        return forward(s["q"], s["q_weight"]), forward(s["k"], s["k_weight"])
    (dq, dqw), (dk, dkw) = backward(s["dq"], s["q"], s["q_weight"]), backward(s["dk"], s["k"], s["k_weight"])
    return dq, dk, dqw, dkw


def _exact_cross(s):
    """One batch entry and query head at a time."""
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    hf = c["heads_first"]
    n, m = c["queries"], c["keys"]

    def head(x, b, h):
        return (x[b, h] if hf else x[b, :, h]).double()

    def like(x):
        return torch.zeros(x.shape, dtype=torch.float64, device="cuda")

    out, lse = like(s["q"]), torch.empty((c["batch"], c["heads"], n), dtype=torch.float64, device="cuda")
    dq, dk, dv = (like(s[x]) for x in "qkv")
    for b in range(c["batch"]):
        keep = torch.ones((1, m), dtype=torch.bool, device="cuda")
        bias = 0.0
        if s["lengths"] is not None:
            keep = torch.arange(m, device="cuda")[None] < s["lengths"][b]
        elif s["mask"] is not None and s["mask"].dtype == torch.bool:
            keep = s["mask"][b, 0]
        elif s["mask"] is not None:
            bias = s["mask"][b, 0].double()
        for h in range(c["heads"]):
            q, k, v = head(s["q"], b, h), head(s["k"], b, h // group), head(s["v"], b, h // group)
            x = torch.where(keep, q @ k.T * c["dim"] ** -0.5 + bias, -math.inf)
            z = torch.logsumexp(x, -1)
            lse[b, h] = z
            p = torch.exp(x - torch.where(z == -math.inf, 0.0, z)[:, None])
            if c["way"] == "forward":
                (out[b, h] if hf else out[b, :, h]).copy_(p @ v)
                continue
            do = head(s["dout"], b, h)
            o = p @ v
            ds = p * (do @ v.T - (o * do).sum(-1, keepdim=True)) * c["dim"] ** -0.5
            (dq[b, h] if hf else dq[b, :, h]).copy_(ds @ k)
            (dk[b, h // group] if hf else dk[b, :, h // group]).add_(ds.T @ q)
            (dv[b, h // group] if hf else dv[b, :, h // group]).add_(p.T @ do)
    return (out, lse) if c["way"] == "forward" else [dq, dk, dv]


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_rotary(s) if case["op"] == "rotary" else _exact_cross(s)
