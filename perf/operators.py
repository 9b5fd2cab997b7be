"""The vocabulary-side operators this library is timed on besides its loss: the
linear cross entropy that keeps no logits (scores and training), the embedding
and its gradient by sorted tokens, and the product in 8-bit floating point with
a scale for each block of 128.

A case is a plain dict. ``prepare`` makes its inputs on the GPU, ``run`` makes
one pass (the plain form in float32 torch operations, or the library's own
calls where ``own`` is set), ``exact`` recomputes the outputs in float64.
"""
import math
import os
import sys

import torch

own = False

IGNORE = -100
E4M3_MAX = 448.0
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "bf16": 2}


def _score(name, dtype, n, h, v, *, ignored=0.0, alpha=0.0):
    """Each row's loss and log-sum-exp, no gradients."""
    return {"name": name, "op": "score", "dtype": dtype, "n": n, "h": h, "v": v, "ignored": ignored,
            "alpha": alpha}


def _train(name, dtype, n, h, v, *, ignored=0.0, alpha=0.0, z=0.0):
    """Forward and backward; ``z`` weights a z-loss z * lse**2 (a gradient into
    lse), ``ignored`` the share of rows without a label."""
    return {"name": name, "op": "train", "dtype": dtype, "n": n, "h": h, "v": v, "ignored": ignored,
            "alpha": alpha, "z": z}


def _lookup(name, dtype, t, h, v, *, scale=1.0):
    return {"name": name, "op": "lookup", "dtype": dtype, "t": t, "h": h, "v": v, "scale": scale}


def _embed(name, dtype, t, h, v, *, scale=1.0, padded=0.0):
    """Lookup and gradient; ``padded`` is the share of padding tokens."""
    return {"name": name, "op": "embed", "dtype": dtype, "t": t, "h": h, "v": v, "scale": scale,
            "padded": padded}


def _fp8(name, m, k, n, *, out="bf16", quant_w=False):
    """bf16 rows quantised in the call, times a weight held as codes and scales
    (``quant_w``: held as bf16 and quantised in the call too)."""
    return {"name": name, "op": "fp8", "m": m, "k": k, "n": n, "out": out, "quant_w": quant_w}


def listed():
    return [
        # the log-probability of one token of a serving step: the weight's bytes
        _score("score_bf16_1x4096x131072", "bf16", 1, 4096, 131072),
        # perplexity of an evaluation batch at a 32k vocabulary
        _score("score_bf16_2048x4096x32000", "bf16", 2048, 4096, 32000),
        # a unit-test or CI training step, where launches and latency count
        _train("train_f32_256x512x8192", "f32", 256, 512, 8192),
        # odd sizes: a vocabulary of 50257, a padded batch, label smoothing
        _train("train_bf16_1000x1536x50257", "bf16", 1000, 1536, 50257, ignored=0.1, alpha=0.1),
        # a full fine-tuning batch at a 131k vocabulary: prompt tokens carry no
        # label, and a z-loss on lse
        _train("train_bf16_8192x4096x131072", "bf16", 8192, 4096, 131072, ignored=0.4, z=1e-4),
        # one token of a serving step
        _lookup("lookup_bf16_1x4096x131072", "bf16", 1, 4096, 131072, scale=64.0),
        # odd sizes in fp32, with padding tokens
        _embed("embed_f32_1000x1531x50257", "f32", 1000, 1531, 50257, padded=0.2),
        # a training batch, and a long-context or accumulated one
        _embed("embed_bf16_8192x4096x131072", "bf16", 8192, 4096, 131072, scale=64.0),
        _embed("embed_bf16_65536x4096x131072", "bf16", 65536, 4096, 131072),
        # a teacher's logits of one token, of a ragged batch (weights quantised
        # on the fly), and of the benchmark's batch
        _fp8("fp8_1x4096x131072", 1, 4096, 131072),
        _fp8("fp8_300x1500x50257_f32", 300, 1500, 50257, out="f32", quant_w=True),
        _fp8("fp8_8192x4096x131072", 8192, 4096, 131072),
    ]


def _spread(rng, lo, hi):
    """A size spread over its logarithm, odd ones as likely as even ones; one in
    three a multiple of 64."""
    x = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if x >= 128 and rng.random() < 1 / 3:
        x = x // 64 * 64
    return max(lo, min(hi, x))


def draw(rng):
    op = rng.choice(["score", "train", "train", "lookup", "embed", "embed", "fp8", "fp8"])
    dtype = "f32" if rng.random() < 0.25 else "bf16"
    if op in ("score", "train"):
        # fp32 products cost several times a bf16 one: smaller batches
        n = _spread(rng, 1, 2048 if dtype == "f32" else 8192)
        c = {"op": op, "dtype": dtype, "n": n, "h": _spread(rng, 256, 4096),
             "v": _spread(rng, 1000, 131072), "ignored": rng.choice([0.0, 0.1, 0.5]),
             "alpha": rng.choice([0.0, 0.1])}
        if op == "train":
            c["z"] = rng.choice([0.0, 1e-4])
        return c
    if op in ("lookup", "embed"):
        c = {"op": op, "dtype": dtype, "t": _spread(rng, 1, 65536 if dtype == "bf16" else 32768),
             "h": _spread(rng, 64, 4096 if dtype == "bf16" else 2048),
             "v": _spread(rng, 1000, 131072), "scale": rng.choice([1.0, 64.0, 0.3])}
        if op == "embed":
            c["padded"] = rng.choice([0.0, 0.2])
        return c
    return {"op": "fp8", "m": _spread(rng, 1, 8192), "k": _spread(rng, 128, 4096),
            "n": _spread(rng, 1000, 131072), "out": rng.choice(["bf16", "bf16", "f32"]),
            "quant_w": rng.random() < 0.25}


# ------------------------------------------------------------------ inputs
def _tokens(t, v, g):
    """Token ids as text has them: frequency falls with the rank, ranks spread
    over the ids."""
    u = torch.rand(t, generator=g, device="cuda", dtype=torch.float64)
    rank = torch.exp(u * math.log(v + 1)).long().sub_(1).clamp_(0, v - 1)
    step = 48271
    while math.gcd(step, v) != 1:
        step += 1
    return (rank * step + 17) % v


def _normal(shape, std, g, dtype):
    out = torch.empty(shape, dtype=DTYPES[dtype], device="cuda")
    return out.normal_(0.0, std, generator=g)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 1)
    op = case["op"]
    if op in ("score", "train"):
        n, h, v = case["n"], case["h"], case["v"]
        st = {"case": case,
              # unit hidden rows (the final norm's output) and logits of a few units
              "hidden": _normal((n, h), 1.0, g, case["dtype"]),
              "weight": _normal((v, h), 2.0 / math.sqrt(h), g, case["dtype"]),
              "labels": _tokens(n, v, g)}
        k = int(n * case["ignored"])
        if k:
            st["labels"][torch.randperm(n, generator=g, device="cuda")[:k]] = IGNORE
        if op == "train":
            valid = max(1, n - k)
            # a mean over the labelled rows, each with a weight of its own
            st["row_weight"] = (0.5 + torch.rand(n, generator=g, device="cuda")) / valid
            st["z"] = case["z"] / valid
            st["hidden"].requires_grad_(True)
            st["weight"].requires_grad_(True)
        return st
    if op in ("lookup", "embed"):
        t, h, v = case["t"], case["h"], case["v"]
        st = {"case": case, "ids": _tokens(t, v, g), "weight": _normal((v, h), 0.02, g, case["dtype"])}
        if op == "embed":
            st["pad"] = v - 1
            k = int(t * case["padded"])
            if k:
                st["ids"][t - k:] = st["pad"]
            st["grad"] = _normal((t, h), 1.0 / t, g, case["dtype"])
            st["weight"].requires_grad_(True)
        return st
    m, k, n = case["m"], case["k"], case["n"]
    st = {"case": case, "x": _normal((m, k), 1.0, g, "bf16")}
    w = _normal((n, k), 2.0 / math.sqrt(k), g, "bf16")
    if case["quant_w"]:
        st["w"] = w
    else:   # a checkpoint's codes and scales
        st["w_codes"], st["w_scales"] = _quantize(w, 128)
    return st


# ------------------------------------------------------------------ plain forms
def _blocks(m, block_rows):
    """[R, C] as [rb, block_rows, cb, 128], padded with zeros."""
    r, c = m.shape
    pr, pc = -r % block_rows, -c % 128
    if pr or pc:
        m = torch.nn.functional.pad(m, (0, pc, 0, pr))
    return m.view((r + pr) // block_rows, block_rows, (c + pc) // 128, 128)


def _quantize(m, block_rows):
    """e4m3 codes and one float32 scale for each block_rows x 128 block."""
    r, c = m.shape
    b = _blocks(m.float(), block_rows)
    top = b.abs().amax(dim=(1, 3))
    # (a quotient: torch turns a division by a plain number into a product)
    scales = (top / torch.full_like(top, E4M3_MAX)).clamp_min(2.0 ** -126)
    q = (b / scales[:, None, :, None]).to(torch.float8_e4m3fn)
    q = q.view(torch.uint8).view(b.shape[0] * block_rows, -1)[:r, :c].contiguous()
    return q.view(torch.float8_e4m3fn), scales


def _dequantize(codes, scales, block_rows, dtype):
    r, c = codes.shape
    out = codes.to(dtype)
    s = scales.to(dtype).repeat_interleave(block_rows, 0)[:r]
    for b in range(s.shape[1]):
        out[:, b * 128:(b + 1) * 128] *= s[:, b:b + 1]
    return out


def _row_losses(x, labels, alpha):
    """Row losses and log-sum-exps of logits x; 0 where there is no label."""
    valid = labels != IGNORE
    y = labels.clamp_min(0)
    top = x.amax(1)
    lse = top + (x - top[:, None]).exp().sum(1).log()
    nll = lse - (1.0 - alpha) * x.gather(1, y[:, None])[:, 0]
    if alpha:
        nll = nll - alpha * x.mean(1)
    zero = torch.zeros((), dtype=x.dtype, device=x.device)
    return torch.where(valid, nll, zero), torch.where(valid, lse, zero)


def _row_grads(x, labels, lse, g_nll, g_lse, alpha):
    """Gradient of the logits, in place of x."""
    valid = labels != IGNORE
    y = labels.clamp_min(0)
    n, v = x.shape
    d = x.sub_(lse[:, None]).exp_().mul_((g_nll + g_lse)[:, None])
    if alpha:
        d.sub_((g_nll * (alpha / v))[:, None])
    d[torch.arange(n, device=x.device), y] -= (1.0 - alpha) * g_nll
    return d.masked_fill_(~valid[:, None], 0.0)


def _plain_ce(st, dtype):
    case = st["case"]
    h, w = st["hidden"].detach().to(dtype), st["weight"].detach().to(dtype)
    x = h @ w.t()
    nll, lse = _row_losses(x, st["labels"], case["alpha"])
    if case["op"] == "score":
        return nll, lse, None, None
    g_lse = 2.0 * st["z"] * lse
    d = _row_grads(x, st["labels"], lse, st["row_weight"].to(dtype), g_lse, case["alpha"])
    return nll, lse, d @ w, d.t() @ h


def _plain_embed(st, dtype):
    case, ids = st["case"], st["ids"]
    w = st["weight"].detach()
    out = w[ids].to(dtype) * case["scale"]
    if case["op"] == "lookup":
        return out, None
    g = st["grad"].to(dtype) * case["scale"]
    g = torch.where((ids != st["pad"])[:, None], g, torch.zeros((), dtype=dtype, device=g.device))
    return out, torch.zeros(w.shape, dtype=dtype, device=w.device).index_add_(0, ids, g)


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
    if op == "score":
        nll, lse = H.linear_cross_entropy(st["hidden"], st["weight"], st["labels"],
                                          ignore_index=IGNORE, label_smoothing=case["alpha"])
        return {"nll": nll, "lse": lse}
    if op == "train":
        nll, lse = H.autograd.linear_cross_entropy_autograd(
            st["hidden"], st["weight"], st["labels"], ignore_index=IGNORE,
            label_smoothing=case["alpha"])
        outs, grads = [nll], [st["row_weight"]]
        if st["z"]:
            outs.append(lse)
            grads.append(2.0 * st["z"] * lse.detach())
        gh, gw = torch.autograd.grad(outs, [st["hidden"], st["weight"]], grads)
        return {"nll": nll.detach(), "lse": lse.detach(), "grad_hidden": gh, "grad_weight": gw}
    if op == "lookup":
        return {"out": H.embedding(st["ids"], st["weight"], scale=case["scale"])}
    if op == "embed":
        out = H.autograd.embedding_autograd(st["ids"], st["weight"], scale=case["scale"],
                                            padding_idx=st["pad"])
        (gw,) = torch.autograd.grad([out], [st["weight"]], [st["grad"]])
        return {"out": out.detach(), "grad_weight": gw}
    codes, scales = H.quantize_fp8_blocks(st["x"])
    if case["quant_w"]:
        w_codes, w_scales = H.quantize_fp8_blocks(st["w"], block_rows=128)
    else:
        w_codes, w_scales = st["w_codes"], st["w_scales"]
    return {"logits": H.fp8_block_matmul(codes, scales, w_codes, w_scales,
                                         out_dtype=DTYPES[case["out"]])}


def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    op = case["op"]
    if op in ("score", "train"):
        nll, lse, gh, gw = _plain_ce(st, torch.float32)
        if op == "score":
            return {"nll": nll, "lse": lse}
        dt = DTYPES[case["dtype"]]
        return {"nll": nll, "lse": lse, "grad_hidden": gh.to(dt), "grad_weight": gw.to(dt)}
    if op in ("lookup", "embed"):
        dt = DTYPES[case["dtype"]]
        out, gw = _plain_embed(st, torch.float32)
        return {"out": out.to(dt)} if op == "lookup" else {"out": out.to(dt), "grad_weight": gw.to(dt)}
    x = _dequantize(*_quantize(st["x"], 1), 1, torch.float32)
    wq = _quantize(st["w"], 128) if case["quant_w"] else (st["w_codes"], st["w_scales"])
    return {"logits": (x @ _dequantize(*wq, 128, torch.float32).t()).to(DTYPES[case["out"]])}


# ------------------------------------------------------------------ float64
def _e4m3(q):
    """Values nearest to q among those of e4m3 (ties to even), |q| <= 448."""
    _, e = torch.frexp(q)
    step = torch.exp2((e - 4).clamp_min(-9).double())   # 3 stored bits; subnormals 2^-9 apart
    return torch.round(q / step) * step


def _exact_fp8(m, block_rows):
    """What the codes of m stand for, in float64: a scale is a float32, and so
    is the quotient that is rounded to e4m3."""
    r, c = m.shape
    b = _blocks(m.double(), block_rows)
    top = b.abs().amax(dim=(1, 3))
    s = (top / torch.full_like(top, E4M3_MAX)).float().double().clamp_min(2.0 ** -126)
    q = (b / s[:, None, :, None]).float().double()
    out = _e4m3(q) * s[:, None, :, None]
    return out.reshape(out.shape[0] * block_rows, -1)[:r, :c]


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in ("score", "train"):
        h, w, labels = st["hidden"].detach().double(), st["weight"].detach().double(), st["labels"]
        n, v, a = case["n"], case["v"], case["alpha"]
        nll, lse = torch.zeros(n, dtype=h.dtype, device=h.device), torch.zeros(n, dtype=h.dtype, device=h.device)
        gh, gw = torch.zeros_like(h), torch.zeros_like(w)
        rows = torch.nonzero(labels != IGNORE)[:, 0]
        for part in rows.split(1024):   # labelled rows only
            hp, y = h[part], labels[part]
            x = hp @ w.t()
            xy = x[torch.arange(len(part), device=x.device), y]
            lse[part] = torch.logsumexp(x, 1)
            nll[part] = lse[part] - (1 - a) * xy - a * x.mean(1)
            if op == "train":
                gn = st["row_weight"][part].double()
                p = torch.softmax(x, 1) * (gn + 2.0 * st["z"] * lse[part])[:, None]
                p -= (gn * a / v)[:, None]
                p[torch.arange(len(part), device=x.device), y] -= gn * (1 - a)
                gh[part] = p @ w
                gw += p.t() @ hp
        if op == "score":
            return {"nll": nll, "lse": lse}
        return {"nll": nll, "lse": lse, "grad_hidden": gh, "grad_weight": gw}
    if op in ("lookup", "embed"):
        w, ids = st["weight"].detach(), st["ids"]
        out = w[ids].double() * case["scale"]
        if op == "lookup":
            return {"out": out}
        gw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
        keep = ids != st["pad"]
        gw.index_add_(0, ids[keep], st["grad"][keep].double() * case["scale"])
        return {"out": out, "grad_weight": gw}
    x = _exact_fp8(st["x"], 1)
    if case["quant_w"]:
        w = _exact_fp8(st["w"], 128)
    else:
        w = _dequantize(st["w_codes"], st["w_scales"], 128, torch.float64)
    return {"logits": x @ w.t()}


# ------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    if op in ("score", "train"):
        es = SIZES[case["dtype"]]
        n, h, v = case["n"], case["h"], case["v"]
        valid = n - int(n * case["ignored"])
        read = (valid * h + v * h) * es + 8 * n
        if op == "score":
            return {"bytes": read + 8 * n, "flops": 2 * valid * h * v}
        # three products (a form that keeps no logits does a fourth)
        return {"bytes": read + (n * h + v * h) * es + 12 * n, "flops": 6 * valid * h * v}
    if op in ("lookup", "embed"):
        es = SIZES[case["dtype"]]
        t, h, v = case["t"], case["h"], case["v"]
        look = 8 * t + 2 * t * h * es
        if op == "lookup":
            return {"bytes": look, "flops": t * h}
        k = t - int(t * case["padded"])
        return {"bytes": look + k * h * es + v * h * es, "flops": t * h + k * h}
    m, k, n = case["m"], case["k"], case["n"]
    out = SIZES[case["out"]]
    return {"bytes": 2 * m * k + n * k * (2 if case["quant_w"] else 1) + m * n * out,
            "flops": 2 * m * n * k}
