"""Drawn tokens against the definition in float64: the tokens equal, the
log-probabilities right to their rounding to fp32.

Two sums of the same masses in 64 bits differ by about 1e-13; a token differs where a
border of the distribution lies within that of the number drawn, which the inputs
here, drawn once, do not meet."""
import math

import numpy as np
import pytest
import torch

import orda_hip as H

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
LOWEST = {"f32": torch.finfo(torch.float32).min, "bf16": torch.finfo(torch.bfloat16).min}


def f32(x):
    return float(np.float32(x))


def reference(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """(token, log-probability) of a row x (float64 numpy)."""
    t, p, m, v = f32(t), f32(p), f32(m), len(x)
    bad = not (0 <= t < math.inf) or math.isnan(p) or math.isnan(m) or not 0 <= u <= 1
    if bad or np.isnan(x).any() or not (x > -math.inf).any():
        return -1, math.nan
    if t == 0:
        return int(np.argmax(x)), 0.0
    if x.max() == math.inf:
        x = np.where(x == math.inf, 0.0, -math.inf)
    with np.errstate(over="ignore"):
        z = (x - x.max()) / t
    w = np.where(z > -690, np.exp(z), 0.0)
    order = np.argsort(-x, kind="stable")
    ws = w[order]
    rank = np.arange(v)
    keep = rank < (k if 0 < k < v else v)
    masses = np.where(keep, ws, 0.0)
    if p < 1:
        before = np.cumsum(masses) - masses
        keep &= (before < p * masses.sum()) | (rank == 0)
    keep &= (ws >= m) | (rank == 0)
    kept = np.zeros(v)
    kept[order[keep]] = ws[keep]
    cdf = np.cumsum(kept)
    token = int(np.searchsorted(cdf, u * cdf[-1], side="right"))
    if token == v or kept[token] == 0:
        token = int(np.nonzero(kept)[0][-1])
    return token, z[token] - math.log(cdf[-1])


def compare(logits, u, t=1.0, k=0, p=1.0, m=0.0, call=None):
    """call: what sample_tokens is given for the parameters (default: the numbers)."""
    kw = dict(temperature=t, top_k=k, top_p=p, min_p=m) if call is None else call
    tokens, logprobs = H.sample_tokens(logits, u, **kw)
    assert tokens.dtype == torch.int64 and logprobs.dtype == torch.float32 and tokens.shape == u.shape
    x, us = logits.double().cpu().numpy(), u.double().cpu().numpy()

    def of(a, i):
        return a[i] if isinstance(a, (list, np.ndarray)) else a
    for i in range(len(us)):
        token, logp = reference(x[i], us[i], of(t, i), of(k, i), of(p, i), of(m, i))
        got, lp = int(tokens[i]), float(logprobs[i])
        assert got == token, f"row {i}: token {got}, not {token}"
        if math.isnan(logp):
            assert math.isnan(lp), f"row {i}: {lp}"
        else:
            # (a distribution of one token: log 1 from sums that are off by 1e-13)
            assert abs(lp - logp) <= 2.0 ** -24 * abs(logp) + 1e-11, f"row {i}: {lp}, not {logp}"


def rows(kind, n, v, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 5 * n + v)
    x = torch.randn(n, v, generator=g) * 2
    if kind == "peaked":      # as a trained head gives them
        x.scatter_(1, torch.randint(0, v, (n, 12), generator=g), 6 + 8 * torch.rand(n, 12, generator=g))
    elif kind == "equal":
        x[:] = 1.5
    elif kind == "ties":      # a few distinct values
        x = x.round()
    elif kind == "wide":      # masses down to nothing
        x *= 200
    elif kind == "masked":    # half of the vocabulary banned, one row but for its last token, one down to two
        x[:, torch.rand(v, generator=g) < 0.5] = -math.inf
        x[0, :-1] = -math.inf
        x[0, -1] = -3.0
        x[1 % n] = -math.inf
        x[1 % n, [0, v // 2]] = torch.tensor([1.0, 1.5])
    elif kind == "lowest":    # banned by the type's lowest value
        x[:, torch.rand(v, generator=g) < 0.5] = LOWEST[dtype]
    elif kind == "near zero":
        x *= 1e-30
    u = torch.rand(n, generator=g)
    u[0] = 0.0
    u[-1] = 1 - 2.0 ** -24
    return x.to(DT[dtype]).cuda(), u.cuda()


KINDS = ["normal", "peaked", "equal", "ties", "wide", "masked", "lowest", "near zero"]
FILTERS = [dict(), dict(t=0.7), dict(t=0.0), dict(k=1), dict(k=2), dict(k=50), dict(p=0.9), dict(p=0.5, t=1.5), dict(m=0.1),
           dict(k=50, p=0.9, t=0.8), dict(k=20, p=0.95, m=0.05), dict(p=0.95, m=0.2), dict(k=700), dict(k=700, p=0.8),
           dict(p=1e-6), dict(m=1.0), dict(p=0.0), dict(t=1e-3, p=0.9), dict(t=100.0, p=0.99), dict(k=3000, p=0.99, m=0.001),
           dict(t=1e-30), dict(t=1e30, k=10)]


@pytest.mark.parametrize("filters", FILTERS, ids=lambda f: "_".join(f"{k}{v}" for k, v in f.items()) or "none")
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("v, dtype", [(1000, "f32"), (5003, "bf16"), (50257, "f32"), (32000, "bf16")])
def test_tokens(v, dtype, kind, filters):
    logits, u = rows(kind, 6, v, dtype)
    compare(logits, u, **filters)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("v", [1, 2, 3, 63, 64, 65, 127, 1023, 1024, 1025, 2047, 4096, 4097, 70001])
def test_vocabularies(v, dtype):
    """At and beside the 64s and 1024s that are summed up first."""
    for kind in ("normal", "ties"):
        logits, u = rows(kind, 9, v, dtype)
        for f in (dict(), dict(k=5), dict(k=v // 2), dict(p=0.6), dict(m=0.3, p=0.9), dict(k=v - 1, p=0.7), dict(k=v), dict(k=v + 1)):
            compare(logits, u, **f)


def test_every_token_of_a_small_vocabulary():
    """u over the whole range: each token is drawn where its part of it lies."""
    x = torch.tensor([[0.5, -1.0, 2.0, -math.inf, 2.0, 0.0]])
    u = torch.linspace(0, 1, 1000)[:-1]
    logits = x.repeat(len(u), 1)
    for f in (dict(), dict(k=3), dict(k=1), dict(p=0.75), dict(p=0.4), dict(m=0.2), dict(t=0.25)):
        compare(logits.cuda(), u.cuda(), **f)
        got = set(H.sample_tokens(logits.cuda(), u.cuda(), temperature=f.get("t", 1.0), top_k=f.get("k"), top_p=f.get("p"),
                                  min_p=f.get("m"))[0].tolist())
        assert 3 not in got
    assert H.sample_tokens(logits[:3].cuda(), torch.tensor([0.0, 1.0, 0.999]).cuda())[0].tolist() == [0, 5, 5]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_equal_logits_than_the_list_holds(dtype):
    """Cuts within 20000 equal logits, of which the lowest tokens are kept."""
    v = 30011
    g = torch.Generator().manual_seed(3)
    x = torch.full((8, v), -2.0)
    x[:, torch.randperm(v, generator=g)[:20000]] = 1.0
    x[:, torch.randperm(v, generator=g)[:9]] = 2.0
    u = torch.rand(8, generator=g)
    for f in (dict(k=9000), dict(p=0.3), dict(p=0.3, k=15000), dict(m=0.3), dict(k=20500, p=0.999), dict(t=0.5, p=0.7, m=0.01)):
        compare(x.to(DT[dtype]).cuda(), u.cuda(), **f)


def test_values_crowded_together():
    """Thousands of logits within one bin of the selection's first pass, and of its second."""
    g = torch.Generator().manual_seed(8)
    v = 40000
    x = torch.randn(6, v, generator=g)
    x[:, ::3] = 3 + 1e-5 * torch.rand(6, (v + 2) // 3, generator=g)
    x[:, 1::9] = 3 + 1e-6
    u = torch.rand(6, generator=g)
    for f in (dict(k=7000), dict(p=0.4), dict(k=9000, p=0.5), dict(p=0.8), dict(m=0.9), dict(t=5.0, p=0.3, k=20000)):
        compare(x.cuda(), u.cuda(), **f)


def test_a_parameter_for_each_row():
    n, v = 40, 20011
    logits, u = rows("peaked", n, v, "bf16")
    r = np.random.default_rng(1)
    t, p, m = r.choice([0.0, 0.5, 1.0, 1.3], n), r.choice([0.3, 0.9, 1.0, 2.0, 0.0], n), r.choice([0.0, 0.1, -1.0, 1.5], n)
    k = r.choice([0, 1, 7, 400, 5000, v, 2 ** 31 - 1, -5], n)

    def gpu(a, dtype=torch.float32):
        return torch.tensor(a, dtype=dtype, device="cuda")
    for kd in (torch.int32, torch.int64):
        compare(logits, u, t, k, p, m, dict(temperature=gpu(t), top_k=gpu(k, kd), top_p=gpu(p), min_p=gpu(m)))
    compare(logits, u, t, 50, 0.9, m, dict(temperature=gpu(t), top_k=50, top_p=0.9, min_p=gpu(m)))
    huge = gpu([2 ** 40 + 3] * n, torch.int64)   # more than an int32
    compare(logits, u, 1.0, 0, 0.9, 0.0, dict(top_k=huge, top_p=0.9))


def test_rows_without_an_answer():
    nan, inf = math.nan, math.inf
    x, u = rows("normal", 12, 3001, "f32")
    x[1, 2999], x[2, 0] = nan, -nan
    x[3] = -inf
    x[4, [5, 2000]] = inf
    x[5] = inf
    x[6, 17] = inf
    x[7, [3, 4]] = torch.tensor([nan, inf], device="cuda")
    for f in (dict(), dict(k=5), dict(p=0.5), dict(m=0.5), dict(t=0.0), dict(k=1000, p=0.9), dict(t=0.5, m=0.1, p=0.7)):
        compare(x, u, **f)
    u[8], u[9], u[10], u[11] = -0.1, 1.5, nan, 1.0
    compare(x, u)
    compare(x, u, k=5, p=0.9)
    for name, bad in (("temperature", [nan, -1.0, inf]), ("top_p", [nan]), ("min_p", [nan])):
        a = torch.full((12,), 0.5, device="cuda")
        a[:len(bad)] = torch.tensor(bad)
        key = {"temperature": "t", "top_p": "p", "min_p": "m"}[name]
        compare(x, u, **{key: a.cpu().numpy()}, call={name: a})


def test_infinities_past_the_list():
    x, u = rows("normal", 4, 20000, "f32")
    x[:, 1::2] = math.inf
    for f in (dict(), dict(k=6000), dict(p=0.7), dict(k=9000, p=0.5), dict(m=0.5), dict(t=0.0), dict(k=15000)):
        compare(x, u, **f)


def test_strides_and_shapes():
    logits, u = rows("peaked", 12, 1003, "bf16")
    want = H.sample_tokens(logits, u, top_k=40, top_p=0.9)
    wide = torch.zeros(12, 1100, dtype=torch.bfloat16, device="cuda")
    wide[:, 7:1010] = logits
    for view in (wide[:, 7:1010], logits.t().contiguous().t()):
        for a, b in zip(H.sample_tokens(view, u, top_k=40, top_p=0.9), want):
            assert torch.equal(a, b)
    spread = torch.stack([u, u], 1)
    assert torch.equal(H.sample_tokens(logits, spread[:, 1], top_k=40, top_p=0.9)[0], want[0])
    t, lp = H.sample_tokens(logits.view(3, 4, 1003), u.view(3, 4), top_k=40, top_p=0.9)
    assert t.shape == (3, 4) and torch.equal(t.reshape(-1), want[0]) and torch.equal(lp.reshape(-1), want[1])
    t, _ = H.sample_tokens(logits[2], u[2], top_k=40, top_p=0.9)
    assert t.shape == () and t == want[0][2]
    t, lp = H.sample_tokens(logits[:0], u[:0])
    assert t.shape == (0,) and lp.shape == (0,)
    one = H.sample_tokens(logits[:1].expand(12, 1003), u, top_k=40)   # one row, many numbers
    assert torch.equal(one[0], H.sample_tokens(logits[:1].repeat(12, 1), u, top_k=40)[0])


def test_offsets_past_32_bits():
    n, v = 4200, 2 ** 20
    x = torch.zeros((n, v), dtype=torch.bfloat16, device="cuda")
    x[:, 12345] = 30.0
    last, u = rows("peaked", 3, v, "bf16")
    x[-3:] = last
    us = torch.full((n,), 0.5, device="cuda")
    us[-3:] = u
    for f in (dict(), dict(k=40), dict(p=0.9)):
        tokens, _ = H.sample_tokens(x, us, top_k=f.get("k"), top_p=f.get("p"))
        assert (tokens[:-3] == 12345).all()
        want, _ = H.sample_tokens(last, u, top_k=f.get("k"), top_p=f.get("p"))
        assert torch.equal(tokens[-3:], want)
    compare(last, u)
    compare(last, u, p=0.9)
    flat, u = rows("normal", 2, v, "f32")
    compare(flat, u, p=0.9)
    compare(flat, u, k=200000, p=0.9)
    compare(flat, u, k=10000)


def test_the_same_tokens_on_other_streams_and_in_graphs():
    logits, u = rows("peaked", 50, 33333, "f32")
    flat, _ = rows("normal", 50, 33333, "f32", seed=9)

    def step():
        return (*H.sample_tokens(logits, u, temperature=0.9, top_k=50, top_p=0.9), *H.sample_tokens(flat, u, top_p=0.8),
                *H.sample_tokens(flat, u))
    want = step()
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)] * 2:
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    for o in got:
        assert all(torch.equal(a, b) for a, b in zip(o, want))
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    for seed in (1, 2, 3):
        logits.copy_(rows("peaked", 50, 33333, "f32", seed=seed)[0])
        flat.copy_(rows("normal", 50, 33333, "f32", seed=seed + 20)[0])
        u.copy_(torch.rand(50, generator=torch.Generator().manual_seed(seed)))
        want = step()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_refusals():
    x, u = rows("normal", 4, 100, "f32")
    ones = torch.ones(4, device="cuda")
    for a, kw in (((x.half(), u), {}), ((x, u.double()), {}), ((x, u[:3]), {}), ((x.cpu(), u), {}), ((x, u.cpu()), {}),
                  ((x[:, :0], u), {}), ((x, u), dict(temperature=-1.0)), ((x, u), dict(top_p=1.5)), ((x, u), dict(min_p=-0.5)),
                  ((x, u), dict(temperature=ones[:3])), ((x, u), dict(top_k=ones)), ((x, u), dict(top_p=ones.double())),
                  ((x, u), dict(min_p=ones.cpu())), ((x, u), dict(temperature=float("nan")))):
        with pytest.raises(H.OrdaError):
            H.sample_tokens(*a, **kw)


@pytest.mark.parametrize("kw", [dict(top_k=2.5), dict(top_k="2"), dict(temperature=1e39), dict(temperature="1"),
                                dict(top_p="0.9"), dict(min_p=[0.1]), dict(top_k=float("inf"))], ids=str)
def test_parameters_that_are_no_numbers(kw):
    with pytest.raises(H.OrdaError, match="numbers"):
        H.sample_tokens(torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda"), **kw)


@pytest.mark.parametrize("t", [1e30, 1e33, 1e34, 1e36, 3e38])
@pytest.mark.parametrize("v", [10, 3000])
def test_logits_and_temperatures_at_the_types_end(v, t):
    """Masses that are all alike, or nothing, and tokens that are banned beside them."""
    g = torch.Generator().manual_seed(v)
    x = -3.3e38 + 1e37 * torch.randn(6, v, generator=g).clamp(-0.9, 2)
    x[:, torch.rand(v, generator=g) < 0.3] = -math.inf
    x[:, 3] = -3.35e38
    x[3:] = -x[3:].abs().clamp_max(3.4e38) * torch.where(torch.isinf(x[3:]), 1.0, -1.0)   # large, some banned
    u = torch.rand(6, generator=g)
    u[0] = 0
    for kw in (dict(), dict(p=0.9), dict(k=7), dict(m=0.5), dict(k=2000, p=0.5)):
        compare(x.cuda(), u.cuda(), t=t, **kw)
