"""The operators right before and right after the head that this library is timed
on: the root-mean-square norm with the residual's addition (forward, backward,
and with its output in e4m3 for the 8-bit head), drawing tokens from logits with
temperature, top-k, top-p and min-p, and the global gradient norm with clipping.

A case is a plain dict. ``prepare`` makes its inputs on the GPU, ``run`` makes
one pass (the plain form in elementary torch operations, or the library's own
calls where ``own`` is set), ``exact`` recomputes the outputs in float64.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
CLIP_EPS = 1e-6
E4M3_MAX = 448.0
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "bf16": 2}


def _norm(name, dtype, n, h, *, residual=True, offset=0.0):
    """Forward alone."""
    return {"name": name, "op": "norm", "dtype": dtype, "n": n, "h": h, "residual": residual, "offset": offset}


def _norm_fp8(name, dtype, n, h, *, residual=True, offset=0.0):
    """Forward with e4m3 codes and a scale for each row and 128 columns."""
    return {"name": name, "op": "norm_fp8", "dtype": dtype, "n": n, "h": h, "residual": residual, "offset": offset}


def _norm_train(name, dtype, n, h, *, residual=True, offset=0.0):
    """Forward and backward; with a residual the sum has a gradient of its own."""
    return {"name": name, "op": "norm_train", "dtype": dtype, "n": n, "h": h, "residual": residual, "offset": offset}


def _sample(name, dtype, n, v, *, t=1.0, k=0, p=1.0, m=0.0, mixed=False, banned=0.0, flat=False):
    """Temperature ``t``, top-k ``k`` (0: none), top-p ``p``, min-p ``m``; ``mixed``: a
    batch of requests, each with its own; ``banned``: the share of tokens that a
    grammar masks; ``flat``: the logits of a model early in training."""
    return {"name": name, "op": "sample", "dtype": dtype, "n": n, "v": v, "t": t, "k": k, "p": p, "m": m,
            "mixed": mixed, "banned": banned, "flat": flat}


def _clip(name, dtype, layers, h, v, *, out="", reached=True):
    """Gradients of a tied embedding [v, h] and of layers of nine tensors (16 h^2
    values in seven matrices, two norms). ``out``: the type that the clipped gradients
    are written in, apart from the gradients; "": in place. ``reached``: whether
    the norm is over the limit."""
    return {"name": name, "op": "clip", "dtype": dtype, "layers": layers, "h": h, "v": v, "out": out,
            "reached": reached}


def listed():
    return [
        # one token of a serving step before the next layer: latency
        _norm("norm_bf16_1x4096", "bf16", 1, 4096),
        # a ragged batch before a head in 8 bits, weights held around zero
        _norm_fp8("norm_fp8_bf16_300x1500", "bf16", 300, 1500, offset=1.0),
        # a prefill's rows before a head in 8 bits
        _norm_fp8("norm_fp8_bf16_8192x4096", "bf16", 8192, 4096),
        # odd sizes in fp32 without a residual: a small model's final norm
        _norm_train("norm_train_f32_1000x1531", "f32", 1000, 1531, residual=False),
        # a training batch
        _norm_train("norm_train_bf16_8192x4096", "bf16", 8192, 4096),
        # one token of a serving step, the usual filters
        _sample("sample_f32_1x131072_k50_p0.9", "f32", 1, 131072, t=0.8, k=50, p=0.9),
        # a serving batch of different requests, a grammar's mask, an odd vocabulary
        _sample("sample_bf16_64x50257_mixed", "bf16", 64, 50257, mixed=True, banned=0.3),
        # nucleus sampling where it keeps tens of thousands of tokens
        _sample("sample_f32_256x131072_p0.95", "f32", 256, 131072, p=0.95, flat=True),
        # rollouts of on-policy distillation: nothing is filtered
        _sample("sample_bf16_512x131072", "bf16", 512, 131072),
        # a small model: launches and host time count
        _clip("clip_f32_4x256x8192", "f32", 4, 256, 8192, out="f32"),
        # the usual step of a run that goes well: in place, and the limit is not reached
        _clip("clip_bf16_12x1531x50257_below", "bf16", 12, 1531, 50257, reached=False),
        # a 131k vocabulary's fp32 gradient and two layers
        _clip("clip_f32_2x4096x131072", "f32", 2, 4096, 131072, out="f32"),
    ]


def _spread(rng, lo, hi):
    """A size spread over its logarithm, odd ones as likely as even ones; one in
    three a multiple of 64."""
    x = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if x >= 128 and rng.random() < 1 / 3:
        x = x // 64 * 64
    return max(lo, min(hi, x))


def draw(rng):
    op = rng.choice(["norm", "norm_fp8", "norm_train", "sample", "sample", "sample", "clip", "clip"])
    dtype = "f32" if rng.random() < 0.35 else "bf16"
    if op in ("norm", "norm_fp8", "norm_train"):
        return {"op": op, "dtype": dtype, "n": _spread(rng, 1, 8192 if dtype == "bf16" else 4096),
                "h": _spread(rng, 64, 4096), "residual": rng.random() < 0.7, "offset": rng.choice([0.0, 0.0, 1.0])}
    if op == "sample":
        return {"op": op, "dtype": dtype, "n": _spread(rng, 1, 512 if dtype == "bf16" else 256),
                "v": _spread(rng, 1000, 131072), "t": rng.choice([1.0, 0.7, 1.5, 0.0]),
                "k": rng.choice([0, 0, 1, 20, 50, 400, 5000]), "p": rng.choice([1.0, 0.9, 0.95, 0.5]),
                "m": rng.choice([0.0, 0.0, 0.05, 0.2]), "mixed": rng.random() < 0.25,
                "banned": rng.choice([0.0, 0.0, 0.5]), "flat": rng.random() < 0.3}
    while True:
        layers, h, v = rng.randint(1, 24), _spread(rng, 32, 4096), _spread(rng, 1000, 131072)
        if 16 * layers * h * h + v * h <= 2 ** 30:
            break
    return {"op": op, "dtype": dtype, "layers": layers, "h": h, "v": v, "out": rng.choice(["", "f32", "bf16"]),
            "reached": rng.random() < 0.7}


# ------------------------------------------------------------------ inputs
def _normal(shape, std, g, dtype):
    out = torch.empty(shape, dtype=DTYPES[dtype], device="cuda")
    return out.normal_(0.0, std, generator=g)


def _logits(case, g):
    """Rows as a head gives them: a bulk, and some tokens above it by up to a dozen
    units, each row with a sharpness of its own."""
    n, v = case["n"], case["v"]
    x = torch.empty((n, v), dtype=torch.float32, device="cuda").normal_(0.0, 2.0, generator=g)
    if not case["flat"]:
        likely = torch.randint(0, v, (n, 30), generator=g, device="cuda")
        sharp = 1.0 + 6.0 * torch.rand((n, 1), generator=g, device="cuda")
        above = 4.0 + torch.empty((n, 30), device="cuda").exponential_(1.0, generator=g) * sharp.sqrt()
        # (places may repeat: the largest, whatever the order in which they are written)
        x.scatter_reduce_(1, likely, above.clamp_max(20.0), "amax", include_self=False)
    if case["banned"]:
        mask = torch.rand(v, generator=g, device="cuda") < case["banned"]
        x.masked_fill_(mask, -math.inf)
        x[:, 5] = 0.0   # one is always allowed
    return x.to(DTYPES[case["dtype"]])


def _shapes(case):
    h = case["h"]
    layer = [(h, h)] * 4 + [(4 * h, h)] * 2 + [(h, 4 * h)] + [(h,)] * 2
    return [(case["v"], h)] + layer * case["layers"]


def _views(flat, shapes):
    out, at = [], 0
    for s in shapes:
        n = math.prod(s)
        out.append(flat[at:at + n].view(s))
        at += n
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 6151 + 3)
    op = case["op"]
    if op in ("norm", "norm_fp8", "norm_train"):
        n, h, dt = case["n"], case["h"], case["dtype"]
        st = {"case": case, "x": _normal((n, h), 1.0, g, dt),
              "weight": _normal((h,), 0.2, g, dt).add_(1.0 - case["offset"]), "residual": None}
        if case["residual"]:   # a stream that many layers have added to
            st["residual"] = _normal((n, h), 4.0, g, dt)
        if op == "norm_train":
            st["grad"] = _normal((n, h), 1.0 / n, g, dt)
            for k in ("x", "weight", "residual"):
                if st[k] is not None:
                    st[k].requires_grad_(True)
            if case["residual"]:
                st["grad_total"] = _normal((n, h), 1.0 / n, g, dt)
        return st
    if op == "sample":
        n = case["n"]
        st = {"case": case, "logits": _logits(case, g), "u": torch.rand(n, generator=g, device="cuda")}
        st["t"], st["k"], st["p"], st["m"] = case["t"], case["k"], case["p"], case["m"]
        if case["mixed"]:
            def pick(values, dtype):
                at = torch.randint(0, len(values), (n,), generator=g, device="cuda")
                return torch.tensor(values, dtype=dtype, device="cuda")[at]
            st["t"] = pick([1.0, 0.7, 1.3, 0.0], torch.float32)
            st["k"] = pick([0, 1, 20, 50, 500], torch.int32)
            st["p"] = pick([1.0, 0.9, 0.95], torch.float32)
            st["m"] = pick([0.0, 0.0, 0.05], torch.float32)
        return st
    shapes = _shapes(case)
    total = sum(math.prod(s) for s in shapes)
    # buckets as a data-parallel trainer keeps them, a tensor's gradient a view
    st = {"case": case, "flat": _normal((total,), 1.0 / math.sqrt(total), g, case["dtype"])}
    st["grads"] = _views(st["flat"], shapes)
    st["max_norm"] = 0.25 if case["reached"] else 4.0   # the norm is about 1
    if case["out"]:
        st["out_flat"] = torch.empty((total,), dtype=DTYPES[case["out"]], device="cuda")
        st["out"] = _views(st["out_flat"], shapes)
    return st


# ------------------------------------------------------------------ plain forms
def _plain_total(st):
    x = st["x"].detach()
    if st["residual"] is None:
        return x
    return (x.float() + st["residual"].detach().float()).to(x.dtype)


def _plain_quantize(v):
    """e4m3 codes and one float32 scale for each row and 128 columns of v (float32)."""
    r, c = v.shape
    b = torch.nn.functional.pad(v, (0, -c % 128)).view(r, -1, 128)
    top = b.abs().amax(dim=2)
    # (a quotient: torch turns a division by a plain number into a product)
    scales = (top / torch.full_like(top, E4M3_MAX)).clamp_min(2.0 ** -126)
    return (b / scales[:, :, None]).to(torch.float8_e4m3fn).view(r, -1)[:, :c], scales


def _plain_norm(st):
    case = st["case"]
    total = _plain_total(st)
    # 64 bits where a value is rounded to e4m3: next to a border of two codes
    # fp32's own error would decide
    dt = torch.float64 if case["op"] == "norm_fp8" else torch.float32
    y, w = total.to(dt), st["weight"].detach().to(dt) + case["offset"]
    s = (y.square().mean(1, keepdim=True) + EPS).rsqrt()
    v = y * s * w
    if case["op"] == "norm_fp8":
        codes, scales = _plain_quantize(v.float())
        res = {"codes": codes, "scales": scales}
    else:
        res = {"out": v.to(total.dtype)}
    if st["residual"] is not None:
        res["total"] = total
    if case["op"] == "norm_train":
        g = st["grad"].float()
        gw = g * w
        dot = (gw * y).mean(1, keepdim=True)
        dy = s * gw - y * (s * s * s * dot)
        if st["residual"] is not None:
            dy = dy + st["grad_total"].float()
        res["grad_x"] = dy.to(total.dtype)
        if st["residual"] is not None:
            res["grad_residual"] = res["grad_x"]
        res["grad_weight"] = (g * y * s).sum(0).to(st["weight"].dtype)
    return res


def _plain_sample(st):
    """In 64 bits: the distribution function has as many borders as tokens."""
    x = st["logits"].double()
    n, v = x.shape

    def rows(a):
        return a.double()[:, None] if torch.is_tensor(a) else torch.full((n, 1), float(a), dtype=x.dtype, device=x.device)
    # (parameters are held in 32 bits)
    t, p, m = (rows(a).float().double() for a in (st["t"], st["p"], st["m"]))
    k = rows(st["k"])
    k = torch.where(k > 0, k, torch.full_like(k, v))
    top = x.amax(1, keepdim=True)
    z = (x - top) / torch.where(t > 0, t, torch.ones_like(t))
    w = z.exp()
    order = x.sort(dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    ws = torch.where(torch.arange(v, device=x.device) < k, ws, torch.zeros_like(ws))
    before = ws.cumsum(1) - ws
    ws = torch.where((before < p * ws.sum(1, keepdim=True)) & (ws >= m), ws, torch.zeros_like(ws))
    kept = torch.zeros_like(w).scatter_(1, order, ws)
    cdf = kept.cumsum(1)
    mass = cdf[:, -1:]
    token = (cdf <= st["u"].double()[:, None] * mass).sum(1)
    greedy = (t == 0)[:, 0]
    token = torch.where(greedy, order[:, 0], token)
    logp = z.gather(1, token[:, None])[:, 0] - mass[:, 0].log()
    return {"tokens": token, "logprobs": torch.where(greedy, torch.zeros_like(logp), logp).float()}


def _plain_clip(st):
    # (long sums: in 64 bits)
    sums = torch.stack([(g.double() * g.double()).sum() for g in st["grads"]])
    norm = sums.sum().sqrt()
    scale = (st["max_norm"] / (norm + CLIP_EPS)).clamp_max(1.0).float()
    if not st["case"]["out"]:
        for g in st["grads"]:
            g.copy_(g.float() * scale)
        return {"norm": norm.float(), "grads": st["flat"]}
    for g, o in zip(st["grads"], st["out"]):
        o.copy_(g.float() * scale)
    return {"norm": norm.float(), "grads": st["out_flat"]}


# ------------------------------------------------------------------ the library's calls
_lib = None


def _library():
    global _lib
    if _lib is None:
        path = os.path.abspath("orda-cutile-rs_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import orda_hip
        import orda_hip.autograd
        _lib = orda_hip
    return _lib


def _run_own(st):
    H = _library()
    case = st["case"]
    op = case["op"]
    if op == "sample":
        tokens, logprobs = H.sample_tokens(st["logits"], st["u"], temperature=st["t"], top_k=st["k"], top_p=st["p"],
                                           min_p=st["m"])
        return {"tokens": tokens, "logprobs": logprobs}
    if op == "clip":
        out = st["out"] if case["out"] else None
        norm = H.clip_gradients(st["grads"], st["max_norm"], eps=CLIP_EPS, out=out)
        return {"norm": norm, "grads": st["out_flat"] if case["out"] else st["flat"]}
    x, w, r = st["x"], st["weight"], st["residual"]
    kw = dict(residual=r, eps=EPS, weight_offset=case["offset"])
    if op == "norm_fp8":
        got = H.rms_norm_fp8(x, w, **kw)
        res = {"codes": got[0], "scales": got[1]}
        if r is not None:
            res["total"] = got[2]
        return res
    if op == "norm":
        got = H.rms_norm(x, w, **kw)
        return {"out": got} if r is None else {"out": got[0], "total": got[1]}
    got = H.autograd.rms_norm_autograd(x, w, **kw)
    if r is None:
        gx, gw = torch.autograd.grad([got], [x, w], [st["grad"]])
        return {"out": got.detach(), "grad_x": gx, "grad_weight": gw}
    gx, gr, gw = torch.autograd.grad(list(got), [x, r, w], [st["grad"], st["grad_total"]])
    return {"out": got[0].detach(), "total": got[1].detach(), "grad_x": gx, "grad_residual": gr, "grad_weight": gw}


def run(st):
    if own:
        return _run_own(st)
    op = st["case"]["op"]
    if op == "sample":
        return _plain_sample(st)
    return _plain_clip(st) if op == "clip" else _plain_norm(st)


# ------------------------------------------------------------------ float64
def _e4m3(q):
    """Values nearest to q among those of e4m3 (ties to even), |q| <= 448."""
    _, e = torch.frexp(q)
    step = torch.exp2((e - 4).clamp_min(-9).double())   # 3 stored bits; subnormals 2^-9 apart
    return torch.round(q / step) * step


def _exact_norm(st):
    case = st["case"]
    x = st["x"].detach()
    t = x.double()
    if st["residual"] is not None:   # the sum is held in the inputs' type
        t = (t + st["residual"].detach().double()).to(x.dtype).double()
    t.requires_grad_(True)
    w = st["weight"].detach().double().requires_grad_(True)
    out = t / torch.sqrt(t.pow(2).sum(1, keepdim=True) / case["h"] + EPS) * (w + case["offset"])
    res = {}
    if case["op"] == "norm_fp8":   # values, scales and quotients are float32
        v = out.detach().float().double()
        r, c = v.shape
        pad = -c % 128
        b = torch.cat([v, v.new_zeros(r, pad)], 1).view(r, -1, 128)
        top = b.abs().amax(2)
        s = (top / torch.full_like(top, E4M3_MAX)).float().double().clamp_min(2.0 ** -126)
        res["codes"] = _e4m3((b / s[:, :, None]).float().double()).reshape(r, -1)[:, :c]
        res["scales"] = s
    else:
        res["out"] = out.detach()
    if st["residual"] is not None:
        res["total"] = t.detach()
    if case["op"] == "norm_train":
        gt, gw = torch.autograd.grad([out], [t, w], [st["grad"].double()])
        if st["residual"] is not None:
            gt = gt + st["grad_total"].double()
        res["grad_x"] = gt
        if st["residual"] is not None:
            res["grad_residual"] = gt
        res["grad_weight"] = gw
    return res


def _exact_row(a, u, t, k, p, m):
    """Token and log-probability of one row, from its distinct values."""
    a = a.double()
    if t == 0:
        best = torch.nonzero(a == a.max())[0, 0]
        return best, torch.zeros((), dtype=torch.float64, device=a.device)
    values, place, count = torch.unique(a, return_inverse=True, return_counts=True)
    values, count = values.flip(0), count.flip(0).double()   # largest first
    place = len(values) - 1 - place
    if k <= 0:
        k = len(a)
    before = count.cumsum(0) - count
    count_k = (k - before).clamp(min=0).minimum(count)
    each = torch.exp((values - values[0]) / t)
    mass = count_k * each
    above = mass.cumsum(0) - mass
    want = p * mass.sum()
    # ties of a value are kept one by one while the mass before them is under p's
    kept = torch.where(each > 0, torch.ceil((want - above) / each), torch.zeros_like(each))
    kept = kept.clamp(min=0).minimum(count_k)
    kept = torch.where(each >= m, kept, torch.zeros_like(kept))
    # how many of its value stand before a token
    order = torch.argsort(place, stable=True)
    start = (torch.bincount(place).cumsum(0) - torch.bincount(place))
    rank = torch.empty_like(order)
    rank[order] = torch.arange(len(a), device=a.device) - start[place[order]]
    w = torch.where(rank < kept[place], each[place], torch.zeros((), dtype=a.dtype, device=a.device))
    c = w.cumsum(0)
    token = torch.searchsorted(c, (u * c[-1]).reshape(1), right=True)[0]
    return token, torch.log(w[token] / c[-1])


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "sample":
        def at(a, i):
            a = a[i] if torch.is_tensor(a) else torch.tensor(a, dtype=torch.float32)
            return a.double().to("cuda")
        rows = [_exact_row(st["logits"][i], at(st["u"], i), *(at(st[q], i) for q in "tkpm")) for i in range(case["n"])]
        return {"tokens": torch.stack([r[0] for r in rows]), "logprobs": torch.stack([r[1] for r in rows])}
    if op == "clip":
        parts = st["flat"].split(2 ** 27)
        norm = math.sqrt(math.fsum(float(p.double().square().sum()) for p in parts))
        c = torch.tensor(min(1.0, st["max_norm"] / (norm + CLIP_EPS)), dtype=torch.float32).double().item()
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": st["flat"].double() * c}
    return _exact_norm(st)


# ------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    if op == "sample":
        n, v = case["n"], case["v"]
        return {"bytes": n * v * SIZES[case["dtype"]] + 16 * n, "flops": 2 * n * v}
    if op == "clip":
        total = sum(math.prod(s) for s in _shapes(case))
        read = total * SIZES[case["dtype"]]
        # in place below the limit nothing is written
        written = total * SIZES[case["out"]] if case["out"] else read if case["reached"] else 0
        return {"bytes": read + written, "flops": 2 * total + (total if written else 0)}
    n, h, es = case["n"], case["h"], SIZES[case["dtype"]]
    arrays = 4 if case["residual"] else 2   # x, out, and the residual and the sum
    if op == "norm_fp8":
        return {"bytes": ((arrays - 1) * es + 1) * n * h + 4 * n * -(-h // 128) + h * es, "flops": 6 * n * h}
    if op == "norm_train":   # the gradient in, the sum again, the gradient out, and the sum's own
        arrays += 4 if case["residual"] else 3
        return {"bytes": arrays * n * h * es + 2 * h * es, "flops": 16 * n * h}
    return {"bytes": arrays * n * h * es + h * es, "flops": 5 * n * h}
