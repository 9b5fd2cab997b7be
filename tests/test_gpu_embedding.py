"""The embedding and its gradient against float64. The lookup rounds the product
in fp32 and then to the weight's type; a gradient row of c tokens is off by at
most c + 1 roundings of fp32 (2^-24 each of the sum of magnitudes) and one of its
own type."""
import pytest
import torch

import orda_hip as H
from orda_hip.autograd import embedding_autograd

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -24


def tokens(t, v, kind, seed=0):
    g = torch.Generator().manual_seed(seed * 31 + t + v)
    if kind == "one":
        ids = torch.full((t,), v // 2)
    elif kind == "few":
        ids = torch.randint(0, min(v, 3), (t,), generator=g)
    elif kind == "text":
        ids = (torch.rand(t, generator=g).mul(torch.tensor(float(v)).log()).exp().long() - 1).clamp(0, v - 1)
    else:
        ids = torch.randint(0, v, (t,), generator=g)
    return ids.cuda()


def grad_of(t, h, dtype, seed=0):
    return torch.randn(t, h, generator=torch.Generator().manual_seed(seed + 5 * t + h)).to(DT[dtype]).cuda()


def check_grad(got, grad, ids, v, scale=1.0, pad=None, old=None):
    g = grad.double().cpu().reshape(-1, grad.size(-1)) * torch.tensor(scale, dtype=torch.float32).double()
    i = ids.reshape(-1).long().cpu()
    keep = (i >= 0) & (i < v)
    if pad is not None:
        keep &= i != pad
    g, i = g[keep], i[keep]
    ref = torch.zeros(v, g.size(1), dtype=torch.float64)
    mag, count = ref.clone(), torch.zeros(v, dtype=torch.float64)
    ref.index_add_(0, i, g)
    mag.index_add_(0, i, g.abs())
    count.index_add_(0, i, torch.ones(len(i), dtype=torch.float64))
    if old is not None:
        o = old.double().cpu()
        ref, mag = ref + o, mag + o.abs()
    bound = (count[:, None] + 2) * U * mag
    bound = bound + ROUND[got.dtype] * (ref.abs() + bound)
    e = (got.double().cpu() - ref).abs()
    bad = ~(e <= bound)
    assert not bad.any(), f"{int(bad.sum())} off, the first at {bad.nonzero()[0].tolist()}"
    untouched = count == 0
    if old is None:
        assert (got[untouched.to(got.device)] == 0).all()
    else:
        assert torch.equal(got[untouched.to(got.device)], old[untouched.to(got.device)])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("index", [torch.int64, torch.int32])
@pytest.mark.parametrize("t, h, v", [(1, 1, 1), (1, 8, 3), (5, 7, 100), (64, 64, 300), (1000, 1531, 257), (3, 4096, 1000),
                                     (777, 2056, 50)])
def test_lookup(t, h, v, dtype, index):
    w = grad_of(v, h, dtype)
    ids = tokens(t, v, "uniform").to(index)
    assert torch.equal(H.embedding(ids, w), w[ids.long()])
    for scale in (64.0, 0.3):
        got = H.embedding(ids, w, scale=scale)
        s = torch.tensor(scale, dtype=torch.float32).double()
        ref = w[ids.long()].double() * s
        assert got.dtype == w.dtype
        assert ((got.double() - ref).abs() <= (ROUND[w.dtype] + 2 * U) * ref.abs()).all()


def test_lookup_shapes_strides_and_ids_out_of_range():
    w = grad_of(100, 96, "bf16")
    ids = tokens(24, 100, "uniform").view(2, 3, 4)
    assert H.embedding(ids, w).shape == (2, 3, 4, 96)
    wide = torch.zeros(100, 131, dtype=torch.bfloat16, device="cuda")
    wide[:, 5:101] = w
    assert torch.equal(H.embedding(ids, wide[:, 5:101]), w[ids])
    assert torch.equal(H.embedding(ids.transpose(0, 2), w), w[ids.transpose(0, 2)])
    assert H.embedding(ids[:0], w).shape == (0, 3, 4, 96)
    assert H.embedding(torch.tensor(7, device="cuda"), w).shape == (96,)
    bad = torch.tensor([0, 100, -1, 99, 2 ** 40], device="cuda")
    out = H.embedding(bad, w)
    assert torch.equal(out[[0, 3]], w[[0, 99]]) and torch.isnan(out[[1, 2, 4]]).all()
    none = H.embedding(bad, torch.zeros(0, 96, device="cuda"))   # no rows at all
    assert none.shape == (5, 96) and torch.isnan(none).all()
    w[3] = float("inf")
    assert torch.equal(H.embedding(torch.tensor([3], device="cuda"), w, scale=2.0)[0], w[3])


# below, at and past the chunk of sorted tokens, the tokens whose ranks are
# counted, a workgroup of the passes; one to three digits of the ids
SIZES = [(1, 8, 1), (1, 7, 3), (31, 64, 100), (32, 64, 100), (33, 64, 100), (64, 520, 9), (65, 1531, 700),
         (500, 100, 511), (2048, 72, 512), (2049, 72, 300), (4096, 16, 1000), (4097, 16, 40000), (9000, 40, 300000),
         (20000, 8, 70)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["uniform", "one", "few", "text"])
@pytest.mark.parametrize("t, h, v", SIZES)
def test_gradient(t, h, v, kind, dtype):
    ids, g = tokens(t, v, kind), grad_of(t, h, dtype)
    check_grad(H.embedding_backward(g, ids, v), g, ids, v)


@pytest.mark.parametrize("kind", ["uniform", "one", "text"])
@pytest.mark.parametrize("t", [1023, 1025, 2049, 8192, 15360, 15361, 40000])   # counted ranks up to 15360, then passes
def test_gradient_of_many_tokens(t, kind):
    v, h = 3000, 40
    ids, g = tokens(t, v, kind), grad_of(t, h, "bf16")
    check_grad(H.embedding_backward(g, ids, v), g, ids, v)


@pytest.mark.parametrize("kind", ["uniform", "one", "few", "text"])
@pytest.mark.parametrize("t, v", [(16385, 511), (16385, 512), (16500, 262143), (16384, 262144), (15000, 300000), (20000, 2 ** 27)])
def test_digits_of_the_sort(t, v, kind):
    """Sorts in passes of 9 bits where the ids (and v, which stands for no id) end at and after a digit: one to four
    passes. (Of 2^27 rows only those that are named are compared, the others looked at.)"""
    ids, g = tokens(t, v, kind), grad_of(t, 2, "bf16")
    if kind == "uniform":
        ids[::100] = v - 1
    if v < 2 ** 20:
        check_grad(H.embedding_backward(g, ids, v), g, ids, v)
        return
    out = torch.zeros(v, 2, dtype=torch.bfloat16, device="cuda")
    H.embedding_backward(g, ids, v, out=out, accumulate=True)
    named, place = torch.unique(ids, return_inverse=True)
    check_grad(out[named], g, place, len(named))
    out[named] = 0
    assert (out == 0).all()


@pytest.mark.parametrize("kind", ["uniform", "one", "few", "text"])
@pytest.mark.parametrize("t, v", [(131072, 600), (131073, 600), (135169, 400), (530001, 300000), (4194305, 5000)])
def test_gradient_of_more_workgroups_than_count_for_themselves(t, v, kind):
    """Past 32 workgroups of 4096 pairs their counts are summed by a launch of its own: 128 runs of them, one or many
    rows each, digits in one to three passes."""
    ids, g = tokens(t, v, kind), grad_of(t, 3, "bf16")
    check_grad(H.embedding_backward(g, ids, v), g, ids, v)


@pytest.mark.parametrize("kind", ["uniform", "one", "text"])
@pytest.mark.parametrize("t", [0, 5, 4000, 20000])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_without_tokens_are_zero_and_nothing_else_is(t, kind, dtype):
    """Whole and strided outputs at every start within a line, over memory that held something else."""
    v, h = 701, 33
    ids, g = tokens(t, v, kind), grad_of(t, h, dtype)
    want = H.embedding_backward(g, ids, v)
    check_grad(want, g, ids, v)
    for at in (0, 1, 5, 31, 63):
        flat = torch.full((at + v * h + 70,), 7.0, dtype=DT[dtype], device="cuda")
        H.embedding_backward(g, ids, v, out=flat[at:at + v * h].view(v, h))
        assert torch.equal(flat[at:at + v * h].view(v, h), want)
        assert (flat[:at] == 7).all() and (flat[at + v * h:] == 7).all()
        frame = torch.full((v, h + 70), 7.0, dtype=DT[dtype], device="cuda")
        H.embedding_backward(g, ids, v, out=frame[:, at:at + h])
        assert torch.equal(frame[:, at:at + h], want)
        assert (frame[:, :at] == 7).all() and (frame[:, at + h:] == 7).all()


@pytest.mark.parametrize("dtype, out", [("bf16", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("t, h, v", [(40, 64, 30), (300, 77, 1000), (5000, 64, 1000)])
def test_accumulated(t, h, v, dtype, out):
    ids, g = tokens(t, v, "text").to(torch.int32), grad_of(t, h, dtype)
    old = grad_of(v, h, out, seed=9)
    got = H.embedding_backward(g, ids, v, scale=0.5, out=old.clone(), accumulate=True)
    check_grad(got, g, ids, v, scale=0.5, old=old)
    got = H.embedding_backward(g, ids, v, scale=0.5, out=old.clone())
    check_grad(got, g, ids, v, scale=0.5)


@pytest.mark.parametrize("t", [100, 3000])
def test_padding_and_ids_out_of_range(t):
    v, h = 200, 64
    ids, g = tokens(t, v, "text"), grad_of(t, h, "bf16")
    ids[::7] = v - 1
    ids[1::11] = -5
    ids[2::13] = v
    ids[3::17] = 2 ** 33 + 4
    g[ids == v - 1] = float("nan")
    for pad in (v - 1, -1):
        check_grad(H.embedding_backward(g, ids, v, padding_idx=pad), g.nan_to_num(0), ids, v, pad=v - 1)
    only = torch.full((t,), v - 1, device="cuda")
    assert (H.embedding_backward(g, only, v, padding_idx=v - 1) == 0).all()


def test_no_tokens_no_rows_no_columns():
    g = torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda")
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert (H.embedding_backward(g, none, 50) == 0).all()
    old = grad_of(50, 64, "f32")
    assert torch.equal(H.embedding_backward(g, none, 50, out=old.clone(), accumulate=True), old)
    ids = torch.zeros(5, dtype=torch.int64, device="cuda")
    assert H.embedding_backward(grad_of(5, 8, "f32"), ids, 0).shape == (0, 8)
    assert H.embedding_backward(torch.zeros(5, 0, device="cuda"), ids, 9).shape == (9, 0)


def test_strided_gradients_and_outputs():
    ids, g = tokens(300, 50, "text"), grad_of(300, 64, "bf16")
    want = H.embedding_backward(g, ids, 50)
    wide = torch.zeros(300, 99, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:67] = g
    assert torch.equal(H.embedding_backward(wide[:, 3:67], ids, 50), want)
    assert torch.equal(H.embedding_backward(g.t().contiguous().t(), ids, 50), want)
    assert torch.equal(H.embedding_backward(g.view(3, 100, 64), ids.view(3, 100), 50), want)
    frame = torch.full((50, 99), 7.0, dtype=torch.bfloat16, device="cuda")
    H.embedding_backward(g, ids, 50, out=frame[:, 3:67])
    assert torch.equal(frame[:, 3:67], want) and (frame[:, :3] == 7).all() and (frame[:, 67:] == 7).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_autograd(dtype):
    w = grad_of(400, 72, dtype).requires_grad_(True)
    ids = tokens(500, 400, "text").view(5, 100)
    out = embedding_autograd(ids, w, scale=8.0, padding_idx=-1)
    g = grad_of(500, 72, dtype, seed=3).view(5, 100, 72)
    out.backward(g)
    check_grad(w.grad, g, ids, 400, scale=8.0, pad=399)
    w.grad = None
    embedding_autograd(ids, w).sum().backward()      # a broadcast gradient
    check_grad(w.grad, torch.ones_like(g), ids, 400)
    with torch.no_grad():
        assert torch.equal(embedding_autograd(ids, w), w[ids])


def test_more_tokens_than_one_launch_holds():
    """2^26 tokens' rows are 2^32 threads of the lookup, which HIP takes in no one launch."""
    w = grad_of(1000, 8, "bf16")
    ids = torch.randint(-1, 1000, (2 ** 26 + 70,), dtype=torch.int32, device="cuda",
                        generator=torch.Generator(device="cuda").manual_seed(1))
    out = H.embedding(ids, w)
    for i, o in zip(ids.split(2 ** 24), out.split(2 ** 24)):
        want = w[i.clamp_min(0).long()]
        want[i < 0] = float("nan")
        assert torch.equal(o.isnan(), want.isnan()) and torch.equal(o.nan_to_num(), want.nan_to_num())


def test_no_second_derivative():
    """A gradient of the gradient is reported, not silently zero."""
    w = grad_of(40, 16, "f32").requires_grad_(True)
    ids = tokens(30, 40, "text")
    g = grad_of(30, 16, "f32").requires_grad_(True)
    (gw,) = torch.autograd.grad(embedding_autograd(ids, w), w, g, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gw.sum().backward()


def test_the_same_bits_and_another_stream():
    ids, g = tokens(6000, 3000, "text"), grad_of(6000, 200, "f32")
    want = H.embedding_backward(g, ids, 3000)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams * 2:
        with torch.cuda.stream(s):
            got.append(H.embedding_backward(g, ids, 3000))
    torch.cuda.synchronize()
    for x in got:
        assert torch.equal(x, want)


@pytest.mark.parametrize("t", [500, 5000])
def test_captured_and_replayed(t):
    v, h = 900, 136
    w, ids, g = grad_of(v, h, "bf16"), tokens(t, v, "text"), grad_of(t, h, "bf16")

    def step():
        return H.embedding(ids, w, scale=2.0), H.embedding_backward(g, ids, v, scale=2.0)
    step()
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.cuda.graph(other):
        out2 = step()
    for seed in (1, 2, 3):
        ids.copy_(tokens(t, v, "text", seed=seed))
        g.copy_(grad_of(t, h, "bf16", seed=seed))
        want = step()
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        for a, b in zip(want + want, out + out2):
            assert torch.equal(a, b)


def test_refusals():
    w, ids, g = grad_of(50, 64, "bf16"), tokens(20, 50, "uniform"), grad_of(20, 64, "bf16")
    for a in ((ids.float(), w), (ids, w.half()), (ids, w[0]), (ids.cpu(), w), (ids, w.cpu())):
        with pytest.raises(H.OrdaError):
            H.embedding(*a)
    for kw in (dict(grad=g[:5]), dict(grad=g[0]), dict(ids=ids.view(4, 5)), dict(num_rows=-1), dict(padding_idx=50),
               dict(padding_idx=-51), dict(accumulate=True), dict(out=w[:, :63]), dict(out=w.half()),
               dict(out=torch.zeros(64, 50, device="cuda").t()), dict(grad=g.half()),
               dict(ids=tokens(50, 50, "uniform"), grad=w, out=w)):
        a = dict(grad=g, ids=ids, num_rows=50)
        a.update(kw)
        with pytest.raises(H.OrdaError):
            H.embedding_backward(**a)
    memory = torch.zeros(50 * 64, dtype=torch.bfloat16, device="cuda")
    shared = memory[:80].view(torch.int64)   # 20 ids in out's first row
    with pytest.raises(H.OrdaError, match="share memory"):
        H.embedding_backward(g, shared, 50, out=memory.view(50, 64))
    with pytest.raises(H.OrdaError):
        embedding_autograd(ids, w, padding_idx=50)
