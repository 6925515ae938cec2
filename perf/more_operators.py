"""Measured cases of the operators that feed a video transformer layer's projections: layer norm with a learned affine
and a modulation per batch entry, forward and backward; the matrix product in 8-bit integers with a scale for each
token and each channel; and the two as a layer runs them, the norm written as 8-bit rows that the product reads.

``own`` selects the framework's kernels; otherwise ``run`` computes the same thing with elementary torch operations in
float32, rounded once at the end.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
LEAST = 1e-30          # a row whose largest magnitude is below this is quantised as if it were this


# ---------------------------------------------------------------------------------------------- cases
def _norm(name, way, *, batch, tokens, width, terms, joined, dtype):
    """terms: what follows the normalisation: none, affine (float32 weight and bias), modulated (scale and shift per
    batch entry, in the rows' type) or both.  joined: the rows are slices of a wider buffer."""
    return {"name": name, "op": "norm", "way": way, "batch": batch, "tokens": tokens, "width": width, "terms": terms,
            "joined": joined, "dtype": dtype}


def _linear(name, *, batch, tokens, width, channels, bias, joined, dtype, op="linear8", terms="none"):
    """op: linear8 (rows as they are) or norm_linear8 (a layer norm with ``terms`` before)."""
    return {"name": name, "op": op, "batch": batch, "tokens": tokens, "width": width, "channels": channels,
            "bias": bias, "terms": terms, "joined": joined, "dtype": dtype}


def listed():
    return [
        # the tokens of a whole 1344 x 768, 124-frame latent before a layer's projections, modulated by the timestep
        _norm("norm_video", "forward", batch=1, tokens=129024, width=2048, terms="modulated", joined=False, dtype="bf16"),
        # the small latent while an adapter is trained: gradients of the rows and of the modulation
        _norm("norm_video_grad", "backward", batch=2, tokens=16384, width=2048, terms="modulated", joined=False,
              dtype="bf16"),
        # an encoder's states with a learned affine: few rows, every gradient
        _norm("norm_states_grad", "backward", batch=4, tokens=512, width=768, terms="affine", joined=False, dtype="f16"),
        # one new token for each of 16 sequences: a launch, nothing else
        _norm("norm_token", "forward", batch=16, tokens=1, width=1024, terms="affine", joined=False, dtype="bf16"),
        # an odd width in float32, slices of a wider buffer, every term
        _norm("norm_odd", "forward", batch=3, tokens=777, width=1001, terms="both", joined=True, dtype="f32"),
        # q, k and v of the whole latent: a joint projection of 16 heads of 128
        _linear("linear8_video", batch=1, tokens=129024, width=2048, channels=6144, bias=False, joined=False, dtype="bf16"),
        # two encoders' states projected for cross attention
        _linear("linear8_states", batch=2, tokens=512, width=768, channels=2048, bias=True, joined=False, dtype="f16"),
        # one new token for each of 16 sequences through a wide layer: its weights are what is read
        _linear("linear8_token", batch=16, tokens=1, width=4096, channels=16384, bias=True, joined=False, dtype="bf16"),
        # a single token through a small layer: latency
        _linear("linear8_one", batch=1, tokens=1, width=2048, channels=6144, bias=False, joined=False, dtype="bf16"),
        # odd in every direction, float32, slices of a wider buffer
        _linear("linear8_odd", batch=1, tokens=1001, width=777, channels=515, bias=True, joined=True, dtype="f32"),
        # the small latent's norm, modulation and up-projection
        _linear("norm_linear8_video", op="norm_linear8", batch=2, tokens=16384, width=2048, channels=8192, bias=True,
                terms="modulated", joined=False, dtype="bf16"),
        # the same for one new token of 16 sequences
        _linear("norm_linear8_token", op="norm_linear8", batch=16, tokens=1, width=1024, channels=4096, bias=True,
                terms="both", joined=False, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "linear8", "linear8", "norm_linear8"])
    batch = rng.choice([1, 1, 2, 3, 7, 16])
    terms = rng.choice(["none", "affine", "modulated", "both"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    joined = rng.random() < 0.25
    # a multiple of 64 as models have them, or any number
    step = rng.choice([64, 64, 64, 1])
    if op == "norm":
        way = rng.choice(["forward", "backward"])
        width = max(1, _log(rng, 16, 8192) // step) * step
        values = 129024 * 2048 / (4 if way == "backward" else 1) / (2 if dtype == "f32" else 1)
        tokens = _log(rng, 1, max(1, min(129024, values / width) / batch))
        # training runs no single rows
        if way == "backward":
            tokens = max(tokens, 8)
        return _norm("", way, batch=batch, tokens=tokens, width=width, terms=terms, joined=joined, dtype=dtype)
    width = max(1, _log(rng, 64, 16384) // step) * step
    channels = max(1, _log(rng, 64, 16384) // step) * step
    rows = min(129024, 129024 * 2048 * 6144 / (width * channels), 129024 * 2048 / width, 129024 * 6144 / channels)
    if dtype == "f32":
        rows /= 2
    tokens = _log(rng, 1, max(1, rows / batch))
    if op == "norm_linear8":
        # a norm's last bits move single 8-bit codes: more than float32 answers are compared to
        dtype = "bf16" if dtype == "f32" else dtype
        width = min(width, 8192)
    return _linear("", op=op, batch=batch, tokens=tokens, width=width, channels=channels, bias=rng.random() < 0.5,
                   terms=terms if op == "norm_linear8" else "none", joined=joined, dtype=dtype)


# ---------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    b, n, w = case["batch"], case["tokens"], case["width"]

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)

    # a residual stream: channels of different sizes, some with an offset
    room = w + (24 if case["joined"] else 0)
    x = torch.randn((b, n, room), generator=gen, device="cuda", dtype=dt)
    x = x.mul_(normal(room, scale=0.6).exp().to(dt)).add_(normal(room, scale=0.3).to(dt))
    s = {"case": case, "x": x[..., room - w:] if case["joined"] else x}
    learned, modulated = case["terms"] in ("affine", "both"), case["terms"] in ("modulated", "both")
    s["weight"] = 1 + normal(w, scale=0.1) if learned else None
    s["bias"] = normal(w, scale=0.1) if learned else None
    s["scale"] = normal(b, w, dtype=dt, scale=0.2) if modulated else None
    s["shift"] = normal(b, w, dtype=dt, scale=0.2) if modulated else None
    if case["op"] == "norm":
        if case["way"] == "backward":
            s["dy"] = torch.randn((b, n, w), generator=gen, device="cuda", dtype=dt)
            s["mean"], s["rstd"] = _statistics(s["x"].float())
        return s
    # the layer's weights, quantised once; their rows start at multiples of 16 bytes
    m = case["channels"]
    full = normal(m, w, scale=w ** -0.5)
    codes, s["weight_scales"] = _quantise(full)
    s["weight_codes"] = torch.zeros((m, (w + 15) // 16 * 16), dtype=torch.int8, device="cuda")[:, :w]
    s["weight_codes"].copy_(codes)
    s["out_bias"] = normal(m, dtype=dt, scale=0.1) if case["bias"] else None
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _statistics(x):
    """A row's mean and the reciprocal of its standard deviation."""
    mean = x.mean(-1)
    return mean, torch.rsqrt((x - mean[..., None]).square().mean(-1) + EPS)


def _terms(s, y):
    """weight, bias, scale and shift applied to y [b, n, w] (float32), those that there are."""
    if s["weight"] is not None:
        y = y * s["weight"] + s["bias"]
    if s["scale"] is not None:
        y = y * (1 + s["scale"].float()[:, None]) + s["shift"].float()[:, None]
    return y


def _normalise(s):
    x = s["x"].float()
    mean, rstd = _statistics(x)
    return _terms(s, (x - mean[..., None]) * rstd[..., None])


def _normalise_back(s):
    dy, x, w = s["dy"].float(), s["x"].float(), s["weight"]
    unit = (x - s["mean"][..., None]) * s["rstd"][..., None]
    grads = {}
    g = dy
    if s["scale"] is not None:
        y = unit if w is None else unit * w + s["bias"]
        grads["scale"], grads["shift"] = (dy * y).sum(1).to(x_type(s)), dy.sum(1).to(x_type(s))
        g = dy * (1 + s["scale"].float()[:, None])
    if w is not None:
        grads["weight"], grads["bias"] = (g * unit).sum((0, 1)), g.sum((0, 1))
        g = g * w
    dx = s["rstd"][..., None] * (g - g.mean(-1, keepdim=True) - unit * (g * unit).mean(-1, keepdim=True))
    return dx.to(x_type(s)), *(grads.get(k) for k in ("weight", "bias", "scale", "shift"))


def x_type(s):
    return DTYPES[s["case"]["dtype"]]


def _quantise(x):
    """int8 codes [.., w] and float32 scales [..] of float32 rows."""
    top = x.abs().amax(-1).clamp_min(LEAST)
    # one division (a number over a tensor is a reciprocal and a product): elements of half the largest stand on a border
    by = torch.full_like(top, 127.0) / top
    return (x * by[..., None]).round().to(torch.int8), top / 127.0


def _product(s, codes, scales):
    y = codes.float() @ s["weight_codes"].float().T
    y = y * scales[..., None] * s["weight_scales"]
    if s["out_bias"] is not None:
        y = y + s["out_bias"].float()
    return y.to(x_type(s))


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if own:
        import htrc_b200
        kw = dict(weight=s["weight"], bias=s["bias"], scale=s["scale"], shift=s["shift"])
        if c["op"] == "norm":
            if c["way"] == "forward":
                return htrc_b200.layer_norm(s["x"], **kw, return_stats=True)
            return htrc_b200.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], **kw)
        rows = s["x"] if c["op"] == "linear8" else htrc_b200.layer_norm_int8(s["x"], **kw)
        return htrc_b200.int8_linear(rows, htrc_b200.Int8Rows(s["weight_codes"], s["weight_scales"]), bias=s["out_bias"],
                                     dtype=s["x"].dtype)
    if c["op"] == "norm":
        if c["way"] == "backward":
            return _normalise_back(s)
        mean, rstd = _statistics(s["x"].float())
        return _normalise(s).to(x_type(s)), mean, rstd
    return _product(s, *_quantise(s["x"].float() if c["op"] == "linear8" else _normalise(s)))


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    b, n, w = case["batch"], case["tokens"], case["width"]
    terms = 0
    if case["terms"] in ("affine", "both"):
        terms += 2 * w * 4
    if case["terms"] in ("modulated", "both"):
        terms += 2 * b * w * es
    values = b * n * w
    if case["op"] == "norm":
        if case["way"] == "forward":
            return {"bytes": 2 * values * es + terms + 8 * b * n, "flops": 8 * values}
        return {"bytes": 3 * values * es + 2 * terms + 8 * b * n, "flops": 16 * values}
    m = case["channels"]
    return {"bytes": values * es + b * n * m * es + m * w + 4 * m + (m * es if case["bias"] else 0) + terms,
            "flops": 2 * values * m}


# ---------------------------------------------------------------------------------------------- 64 bits
def _wide(t):
    return None if t is None else t.to(torch.float64)


def _exact_norm(s):
    """One batch entry at a time: (result, mean, reciprocal deviation, normalised rows)."""
    out = []
    for i in range(s["x"].shape[0]):
        x = _wide(s["x"][i])
        mean = x.sum(-1) / x.shape[-1]
        low = x - mean[:, None]
        rstd = 1.0 / torch.sqrt((low * low).sum(-1) / x.shape[-1] + EPS)
        unit = low * rstd[:, None]
        y = unit
        if s["weight"] is not None:
            y = torch.addcmul(_wide(s["bias"]), y, _wide(s["weight"]))
        if s["scale"] is not None:
            y = torch.addcmul(_wide(s["shift"][i]), y, 1.0 + _wide(s["scale"][i]))
        out.append((y, mean, rstd, unit))
    return out


def _exact_back(s):
    dx, ds, dt = [], [], []
    dw = db = None
    for i, (_, _, rstd, unit) in enumerate(_exact_norm(s)):
        dy = _wide(s["dy"][i])
        p, q = torch.einsum("nw,nw->w", dy, unit), dy.sum(0)
        gain = torch.ones_like(q) if s["scale"] is None else 1.0 + _wide(s["scale"][i])
        if s["scale"] is not None:
            ds.append(p if s["weight"] is None else p * _wide(s["weight"]) + q * _wide(s["bias"]))
            dt.append(q)
        if s["weight"] is not None:
            dw = p * gain if dw is None else dw + p * gain
            db = q * gain if db is None else db + q * gain
            gain = gain * _wide(s["weight"])
        g = dy * gain
        w = g.shape[-1]
        dx.append(rstd[:, None] * (g - (g.sum(-1, keepdim=True) + unit * (g * unit).sum(-1, keepdim=True)) / w))
    return torch.stack(dx), dw, db, torch.stack(ds) if ds else None, torch.stack(dt) if dt else None


def _exact_product(s, rows, single):
    """Rows [n, w] in 64 bits.  Codes are the nearest integers to x * (127 / top), whose two roundings to float32
    belong to the definition where the rows are the call's own input (``single``)."""
    out = []
    weight = _wide(s["weight_codes"]) * _wide(s["weight_scales"])[:, None]
    for x in rows.split(16384):
        top = x.abs().amax(-1, keepdim=True).clamp_min(LEAST)
        by = 127.0 / top
        z = _wide((x * _wide(by.float())).float()) if single else x * by
        y = (torch.round(z) * (top / 127.0)) @ weight.T
        out.append(y if s["out_bias"] is None else y + _wide(s["out_bias"]))
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        if case["way"] == "backward":
            return _exact_back(s)
        return tuple(torch.stack(p) for p in list(zip(*_exact_norm(s)))[:3])
    if case["op"] == "linear8":
        return torch.stack([_exact_product(s, _wide(x), True) for x in s["x"]])
    return torch.stack([_exact_product(s, e[0], False) for e in _exact_norm(s)])
