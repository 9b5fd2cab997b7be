"""The norm of many gradients and their clipping against float64.

Squares of fp32 values are exact in 64 bits, so the norm is right to its rounding to
fp32 (U); the factor has two roundings of 64 bits and one of fp32, a value one more
and that to its type."""
import math

import pytest
import torch

import orda_hip as H

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -24


def normal(shape, dtype="f32", seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * len(shape) + sum(shape))
    return (torch.randn(shape, generator=g, device="cuda") * std).to(DT[dtype])


def norm_of(grads):
    return math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))


def check_norm(got, want):
    assert got.dtype == torch.float32 and got.dim() == 0
    assert abs(float(got) - want) <= 1.01 * U * want


def check_scaled(got, grad, norm, max_norm, eps=1e-6):
    f = min(1.0, max_norm / (norm + eps))
    ref = grad.double() * f
    bound = (ROUND[got.dtype] + 3 * U) * ref.abs() + 2.0 ** -140   # (values under fp32's normal range)
    bad = ~((got.double() - ref).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} off"


# one value, odd sizes, a piece and its neighbours, several pieces, more gradients than one launch holds
LISTS = [[(1,)], [(7,), (1, 1), (3, 5, 7)], [(4095,), (4096,), (4097,)], [(300, 257), (1000003,), (8,)], [(64,)] * 56,
         [(129,)] * 57, [(33, 5), (2000,), (1,)] * 70, [(5, 7)] * 400 + [(3000, 1000)], [(12345, 678), (13, 77)]]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "both"])
@pytest.mark.parametrize("shapes", LISTS, ids=lambda s: f"{len(s)}x{s[0]}")
def test_clipped(shapes, dtype):
    grads = [normal(s, dtype if dtype != "both" else ("f32", "bf16")[i % 2], seed=i) for i, s in enumerate(shapes)]
    old = [g.clone() for g in grads]
    norm = norm_of(old)
    check_norm(H.gradient_norm(grads), norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, old))
    # to other tensors, of either type
    for to in ("f32", "bf16"):
        for limit in (0.3 * norm, 2 * norm):
            out = [torch.full_like(g, float("nan"), dtype=DT[to]) for g in grads]
            got = H.clip_gradients(grads, limit, out=out)
            check_norm(got, norm)
            for o, g in zip(out, old):
                check_scaled(o, g, norm, limit)
    assert all(torch.equal(a, b) for a, b in zip(grads, old))
    # in place
    check_norm(H.clip_gradients(grads, 2 * norm), norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, old))
    version = grads[0]._version
    check_norm(H.clip_gradients(grads, 0.3 * norm), norm)
    assert grads[0]._version > version
    for g, o in zip(grads, old):
        check_scaled(g, o, norm, 0.3 * norm)
    assert (H.clip_gradients(grads, 0.0) > 0) and all((g == 0).all() for g in grads)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_any_start_pitch_and_order(dtype):
    base = normal((50 * 400 + 64,), dtype)
    for at in (0, 1, 3, 7, 17):
        b = base.clone()
        views = [b[at:at + 4000], b[at + 4000:at + 4003], b[at + 4003:at + 9999].view(4, -1).t()]
        norm = norm_of(views)
        check_norm(H.gradient_norm(views), norm)
        out = [torch.empty_strided(v.shape, v.stride(), dtype=v.dtype, device="cuda") for v in views]
        H.clip_gradients(views, 0.5 * norm, out=out)
        for v, o in zip(views, out):
            check_scaled(o, v, norm, 0.5 * norm)
        H.clip_gradients(views, 0.5 * norm)
        for v, o in zip(views, out):
            assert torch.equal(v, o)
        keep = torch.ones_like(b, dtype=torch.bool)
        keep[at:at + 9999] = False
        assert torch.equal(b[keep], base[keep])
    # columns of one frame, beside one another, and a matrix whose rows are adjacent
    frame = base[:50 * 400].view(50, 400).clone()
    old = frame.clone()
    parts = [frame[:, :100], frame[:, 100:257], frame.t()[300:333]]
    norm = norm_of(parts)
    check_norm(H.clip_gradients(parts, 0.25 * norm), norm)
    for p, q in zip(parts, (old[:, :100], old[:, 100:257], old.t()[300:333])):
        check_scaled(p, q, norm, 0.25 * norm)
    assert torch.equal(frame[:, 257:300], old[:, 257:300]) and torch.equal(frame[:, 333:], old[:, 333:])
    # channels last, a broadcast of one
    x = normal((4, 6, 5, 3), dtype).to(memory_format=torch.channels_last)
    old = x.clone()
    norm = norm_of([x])
    H.clip_gradients([x], 0.5 * norm)
    check_scaled(x, old, norm, 0.5 * norm)


@pytest.mark.parametrize("dtype, to", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
def test_more_than_the_cache_holds(dtype, to):
    """Over 256 MB, in two launches, from any start."""
    base = normal((75_000_003 * 4 // (4 if dtype == "f32" else 2),), dtype)
    grads = [base[5:-4_000_000]] + [base[i:i + 57001] for i in range(base.numel() - 4_000_000, base.numel() - 57001, 57003)]
    assert len(grads) > 57
    norm = norm_of(grads)
    check_norm(H.gradient_norm(grads), norm)
    out = [torch.empty_like(g, dtype=DT[to]) for g in grads]
    check_norm(H.clip_gradients(grads, 0.5 * norm, out=out), norm)
    for o, g in zip(out, grads):
        check_scaled(o, g, norm, 0.5 * norm)
    H.clip_gradients(grads, 0.5 * norm)
    if to == dtype:
        assert all(torch.equal(a, b) for a, b in zip(out, grads))


def test_long_rows_of_a_frame():
    """Rows of several pieces, apart from one another."""
    frame = normal((3, 300000))
    old = frame.clone()
    part = frame[:, 5:200006]
    norm = norm_of([part])
    check_norm(H.clip_gradients([part], 0.5 * norm), norm)
    check_scaled(part, old[:, 5:200006], norm, 0.5 * norm)
    assert torch.equal(frame[:, :5], old[:, :5]) and torch.equal(frame[:, 200006:], old[:, 200006:])


def test_extremes():
    """Squares beyond fp32's range, zeros, nothing, infinities and NaN."""
    big, small = normal((1000,)) * 1e30, normal((1000,)) * 1e-30
    for g in (big, small):
        norm = norm_of([g])
        check_norm(H.gradient_norm([g]), norm)
        out = [torch.empty_like(g)]
        H.clip_gradients([g], 0.5 * norm, eps=0.0, out=out)
        check_scaled(out[0], g, norm, 0.5 * norm, 0.0)
    zero = torch.zeros(100, device="cuda")
    assert float(H.clip_gradients([zero], 1.0)) == 0 and (zero == 0).all()
    assert float(H.gradient_norm([zero[:0], zero.view(10, 10)[:, :0]])) == 0
    assert float(H.clip_gradients([zero[:0]], 1.0)) == 0
    check_norm(H.gradient_norm([None, big, None, zero]), norm_of([big]))
    for bad, rest in ((float("inf"), 0.0), (float("nan"), float("nan"))):
        a, b = normal((5000,)), normal((5000,), "bf16")
        a[4321] = bad
        got = H.clip_gradients([a, b], 1.0)
        assert math.isinf(got) if bad == float("inf") else math.isnan(got)
        assert math.isnan(a[4321])
        a[4321] = rest
        for t in (a, b):
            assert (t == 0).all() if rest == 0 else torch.isnan(t).all()
    a = normal((5000,))
    old = a.clone()
    check_norm(H.clip_gradients([a], float("inf")), norm_of([old]))   # a limit that is none
    assert torch.equal(a, old)


def test_more_values_than_32_bits_count():
    g = torch.zeros(2 ** 32 + 70, dtype=torch.bfloat16, device="cuda")
    g[-3:] = torch.tensor([3.0, 4.0, 12.0], device="cuda")
    assert float(H.gradient_norm([g])) == 13
    assert float(H.clip_gradients([g], 6.5, eps=0.0)) == 13
    assert g[-3:].tolist() == [1.5, 2.0, 6.0] and float(H.gradient_norm([g])) == 6.5


def test_the_same_bits_on_other_streams_and_in_graphs():
    shapes = [(300, 257), (1000003,), (8,)] + [(77,)] * 100
    grads = [normal(s, ("f32", "bf16")[i % 2], seed=i) for i, s in enumerate(shapes)]
    out = [torch.empty_like(g) for g in grads]
    want = H.clip_gradients(grads, 1.0, out=out)
    want_out = [o.clone() for o in out]
    torch.cuda.synchronize()
    runs = []
    for s in [torch.cuda.Stream() for _ in range(3)] * 2:
        with torch.cuda.stream(s):
            o = [torch.empty_like(g) for g in grads]
            runs.append((H.clip_gradients(grads, 1.0, out=o), o))
    torch.cuda.synchronize()
    for n, o in runs:
        assert torch.equal(n, want) and all(torch.equal(a, b) for a, b in zip(o, want_out))
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    places = [[torch.empty_like(g) for g in grads] for _ in graphs]
    for graph, place in zip(graphs, places):
        with torch.cuda.graph(graph):
            outs.append(H.clip_gradients(grads, 1.0, out=place))
    for seed in (1, 2, 3):
        for i, g in enumerate(grads):
            g.copy_(normal(tuple(g.shape), "f32", seed=100 * seed + i))
        want = H.clip_gradients(grads, 1.0, out=out)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for n, place in zip(outs, places):
            assert torch.equal(n, want) and all(torch.equal(a, b) for a, b in zip(place, out))
    # in place, in a graph: each replay clips what is there
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = H.clip_gradients(grads, 1.0)
    for seed in (5, 6):
        for i, g in enumerate(grads):
            g.copy_(normal(tuple(g.shape), "f32", seed=100 * seed + i))
        want = H.clip_gradients(grads, 1.0, out=out)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(grads, out))


def test_refusals():
    g = normal((64, 32))
    for grads, kw in (([g, g], {}), ([g, g[3]], {}), ([g.half()], {}), ([g.cpu()], {}), ([g], dict(max_norm=-1.0)),
                      ([g[:, ::2]], {}), ([g[:1].expand(64, 32)], {}), ([g, g.cpu()], {}),
                      ([g], dict(out=[g])), ([g], dict(out=[g.t()])), ([g], dict(out=[g[:32].clone()])), ([g], dict(out=[g.half()])),
                      ([g, None], dict(out=[g.clone(), g.clone()])), ([g], dict(eps=-1.0)),
                      ([g], dict(out=[g.clone().requires_grad_(True)]))):
        with pytest.raises(H.OrdaError):
            H.clip_gradients(grads, kw.pop("max_norm", 1.0), **kw)
    old = g.clone()
    assert torch.equal(g, old)


@pytest.mark.parametrize("limit, kw", [("1", {}), (None, {}), (1.0, dict(eps="0")), (10 ** 400, {})], ids=lambda v: str(v)[:8])
def test_limits_that_are_no_numbers(limit, kw):
    g = normal((8,))
    old = g.clone()
    with pytest.raises(H.OrdaError, match="numbers"):
        H.clip_gradients([g], limit, **kw)
    assert torch.equal(g, old)
