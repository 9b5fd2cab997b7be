"""e4m3 with block scales: the quantiser bit for bit against torch's division and
conversion on the CPU, the product against float64 of the same codes.

A product's element is a sum of K terms in fp32 (2·K roundings of 2^-24 of the sum
of magnitudes: the matrix units may round each step towards zero), each block's
sum scaled and added (two roundings a block, one for the product of the scales),
and one rounding to the output's type."""
import pytest
import torch

import orda_hip as H

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -24


def normal(r, c, dtype="bf16", seed=0, std=1.0):
    return (torch.randn(r, c, generator=torch.Generator().manual_seed(seed + 3 * r + 7 * c)) * std).to(DT[dtype]).cuda()


def blocks(m, block_rows):
    r, c = m.shape
    m = torch.nn.functional.pad(m, (0, -c % 128, 0, -r % block_rows))
    return m.view(m.size(0) // block_rows, block_rows, m.size(1) // 128, 128)


def quantized(m, block_rows):
    """On the CPU, where a quotient is rounded once."""
    r, c = m.shape
    b = blocks(m.float().cpu(), block_rows)
    top = b.abs().amax(dim=(1, 3))
    s = (top / torch.full_like(top, 448.0)).clamp_min(2.0 ** -126)
    q = (b / s[:, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return q.reshape(b.size(0) * block_rows, -1)[:r, :c], s


def same_codes(codes, want):
    got = codes.cpu().view(torch.uint8)
    assert torch.equal(got, want), f"{int((got != want).sum())} of {want.numel()} codes differ"


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("r, c", [(1, 1), (1, 128), (3, 129), (16, 512), (17, 1500), (130, 520), (300, 77), (513, 1024)])
def test_quantiser(r, c, dtype, block_rows):
    m = normal(r, c, dtype)
    codes, scales = H.quantize_fp8_blocks(m, block_rows=block_rows)
    want, s = quantized(m, block_rows)
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == m.shape
    assert torch.equal(scales.cpu(), s)
    same_codes(codes, want)


def test_quantiser_extremes():
    """Zero blocks, blocks below the smallest scale, the largest values, and
    blocks with an infinity or a NaN."""
    m = normal(8, 1024, "f32")
    m[0, :128] = 0
    m[1, :128] *= 1e-42
    m[2, :128] *= 3e38 / m[2, :128].abs().max()
    m[3, :128] *= 1e-36
    m[4, 5] = 1e-30        # codes below the smallest subnormal round to 0
    codes, scales = H.quantize_fp8_blocks(m)
    want, s = quantized(m, 1)
    assert torch.equal(scales.cpu(), s)
    same_codes(codes, want)
    m[5, 130], m[6, 260] = float("nan"), -float("inf")
    codes, scales = H.quantize_fp8_blocks(m)
    bad = torch.zeros(8, 8, dtype=torch.bool)
    bad[5, 1] = bad[6, 2] = True
    assert torch.equal(torch.isnan(scales).cpu(), bad)
    assert torch.equal(torch.isnan(codes.float()).cpu(), bad.repeat_interleave(128, 1))
    blk, sb = H.quantize_fp8_blocks(m, block_rows=128)
    assert torch.isnan(sb[0, 1:3]).all() and torch.isfinite(sb[0, [0, 3, 4, 5, 6, 7]]).all()


def test_quantiser_strides():
    m = normal(40, 300)
    wide = torch.zeros(40, 333, dtype=torch.bfloat16, device="cuda")
    wide[:, 5:305] = m
    for view in (wide[:, 5:305], m.t().contiguous().t()):
        for b in (1, 128):
            for x, y in zip(H.quantize_fp8_blocks(m, block_rows=b), H.quantize_fp8_blocks(view, block_rows=b)):
                assert torch.equal(x.float(), y.float())
    assert H.quantize_fp8_blocks(m[:0])[0].shape == (0, 300)
    assert H.quantize_fp8_blocks(m[:, :0])[1].shape == (40, 0)


def check_product(got, a, sa, b, sb):
    def values(c, s, rows):
        s = s.double().cpu().repeat_interleave(rows, 0)[:c.size(0)].repeat_interleave(128, 1)[:, :c.size(1)]
        return c.float().double().cpu() * s
    x, w = values(a, sa, 1), values(b, sb, 128)
    ref, mag = x @ w.t(), x.abs() @ w.abs().t()
    k = a.size(1)
    bound = 2 * (k + k // 128 + 4) * U * mag
    bound = bound + ROUND[got.dtype] * (ref.abs() + bound) + 1e-37
    e = (got.double().cpu() - ref).abs()
    bad = ~(e <= bound)
    assert not bad.any(), f"{int(bad.sum())} off, the first at {bad.nonzero()[0].tolist()}, largest {e.max():.3g}"


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m, k, n", [(1, 1, 1), (1, 128, 256), (1, 4096, 1000), (3, 100, 5), (16, 256, 384), (17, 130, 129),
                                     (64, 144, 300), (100, 1500, 777), (257, 512, 513), (300, 1024, 130), (520, 384, 1100)])
def test_product(m, k, n, out):
    x, w = normal(m, k), normal(n, k, seed=1, std=0.1)
    x[0] *= 1e4
    a, sa = H.quantize_fp8_blocks(x)
    b, sb = H.quantize_fp8_blocks(w, block_rows=128)
    got = H.fp8_block_matmul(a, sa, b, sb, out_dtype=DT[out])
    assert got.dtype == DT[out] and got.shape == (m, n)
    check_product(got, a, sa, b, sb)


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m", [1, 15, 17, 33, 63, 64, 65])
@pytest.mark.parametrize("k, n", [(100, 40), (256, 1000), (384, 700), (640, 66001), (900, 66001), (1160, 33)])
def test_product_of_few_rows(m, k, n, out):
    """Up to 64 rows, at few and many columns, whole and partial blocks of K, an
    even and an odd number of them."""
    x, w = normal(m, k), normal(n, k, seed=1, std=0.1)
    a, sa = H.quantize_fp8_blocks(x)
    b, sb = H.quantize_fp8_blocks(w, block_rows=128)
    check_product(H.fp8_block_matmul(a, sa, b, sb, out_dtype=DT[out]), a, sa, b, sb)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantiser_near_midpoints(dtype):
    """Quotients at and next to the midpoints of two codes, normal and subnormal,
    where the rounded quotient decides."""
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (codes[1:] + codes[:-1]) / 2
    rows = []
    for top in (448.0, 447.0, 1.0, 3.7, 1e-3, 12345.0, 2.0 ** -100, 2.0 ** 90):
        s = (torch.tensor(top, dtype=torch.float32) / torch.tensor(448.0)).double()
        v = (mid * s).to(DT[dtype])
        near = [v]
        for d in (1, -1, 2, -2, 3, -3):   # neighbours in the input's type
            near.append((v.view(torch.int16 if dtype == "bf16" else torch.int32) + d).view(DT[dtype]))
        flat = torch.cat(near)
        flat = flat[flat.abs().double() <= top]
        for part in flat.split(127):
            row = torch.zeros(128, dtype=DT[dtype])
            row[0] = top
            row[1:1 + len(part)] = part * (1 - 2 * (torch.arange(len(part)) % 2)).to(DT[dtype])
            rows.append(row)
    m = torch.stack(rows).cuda()
    for block_rows in (1,):
        got, scales = H.quantize_fp8_blocks(m, block_rows=block_rows)
        want, s = quantized(m, block_rows)
        assert torch.equal(scales.cpu(), s)
        same_codes(got, want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pitch", [128, 130, 132, 129])
def test_block_quantiser_near_midpoints(dtype, pitch):
    """Blocks of 128 rows whose quotients lie at and next to the midpoints of two codes, normal and subnormal, read at
    every width the rows' alignment allows."""
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (codes[1:] + codes[:-1]) / 2
    made = []
    for top in (448.0, 447.0, 1.0, 3.7, 1e-3, 12345.0, 2.0 ** -100, 2.0 ** 90):
        s = (torch.tensor(top, dtype=torch.float32) / torch.tensor(448.0)).double()
        v = (mid * s).to(DT[dtype])
        bits = v.view(torch.int16 if dtype == "bf16" else torch.int32)
        flat = torch.cat([v] + [(bits + d).view(DT[dtype]) for d in (1, -1, 2, -2, 3, -3)])
        flat = flat[flat.abs().double() <= top]
        block = flat[torch.arange(128 * 128) % len(flat)].view(128, 128).clone()
        block[1::2] = -block[1::2]
        block[77, 5] = top
        made.append(block)
    frame = torch.zeros(128 * len(made), pitch, dtype=DT[dtype], device="cuda")
    m = frame[:, pitch - 128:]
    m.copy_(torch.cat(made))
    got, scales = H.quantize_fp8_blocks(m, block_rows=128)
    want, s = quantized(m, 128)
    assert torch.equal(scales.cpu(), s)
    same_codes(got, want)


def test_quantiser_of_more_rows_than_one_launch_holds():
    """2^28 rows are 2^32 threads, which HIP takes in no one launch. A block of one value has its code at the top."""
    r = 2 ** 28 + 33
    m = torch.empty(r, 1, dtype=torch.bfloat16, device="cuda").uniform_(0.5, 2.0)
    m[::3].neg_()
    codes, scales = H.quantize_fp8_blocks(m)
    assert torch.equal(scales[:, 0], m[:, 0].abs().float().div_(torch.full((1,), 448.0, device="cuda")))
    assert torch.equal(codes.view(torch.uint8)[:, 0], torch.where(m[:, 0] < 0, 0xfe, 0x7e).to(torch.uint8))


def test_product_of_more_columns_than_one_launch_holds():
    """One row by 2^30: 2^32 threads. The first and last columns hold values, the others zeros."""
    n, k = 2 ** 30, 16
    a, sa = H.quantize_fp8_blocks(normal(1, k))
    b = torch.zeros(n, k, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    sb = torch.ones(n // 128, 1, device="cuda")
    part, sp = H.quantize_fp8_blocks(normal(1024, k, seed=1), block_rows=128)
    b.view(torch.uint8)[:1024] = part.view(torch.uint8)
    b.view(torch.uint8)[-1024:] = part.view(torch.uint8)
    sb[:8], sb[-8:] = sp, sp
    got = H.fp8_block_matmul(a, sa, b, sb)
    want = H.fp8_block_matmul(a, sa, part, sp)
    assert torch.equal(got[:, :1024], want) and torch.equal(got[:, -1024:], want)
    assert (got[:, 1024:-1024] == 0).all()
    check_product(want, a, sa, part, sp)


@pytest.mark.parametrize("k", [128, 1000, 1500])
def test_product_layouts(k):
    """Contiguous codes (pitches that are no multiple of 16 are copied), column
    slices, scales by rows and by blocks, expanded scales."""
    m, n = 70, 300
    a, sa = H.quantize_fp8_blocks(normal(m, k))
    b, sb = H.quantize_fp8_blocks(normal(n, k, seed=1), block_rows=128)
    want = H.fp8_block_matmul(a, sa, b, sb)
    assert torch.equal(H.fp8_block_matmul(a.contiguous(), sa.contiguous(), b.contiguous(), sb.t().contiguous().t()), want)
    for at, pitch in ((0, 2048), (16, 2048), (7, 2047)):
        wide = torch.full((n, pitch), 448.0, device="cuda").to(torch.float8_e4m3fn)
        wide.view(torch.uint8)[:, at:at + k] = b.view(torch.uint8) if b.is_contiguous() else b.contiguous().view(torch.uint8)
        assert torch.equal(H.fp8_block_matmul(a, sa, wide[:, at:at + k], sb), want)
    one = torch.ones(1, 1, device="cuda")
    got = H.fp8_block_matmul(a, one.expand(sa.shape), b, one.expand(sb.shape), out_dtype=torch.float32)
    check_product(got, a, torch.ones_like(sa), b, torch.ones_like(sb))


def test_codes_at_a_wide_pitch():
    """Columns of a table up to 2^24 + 32 bytes wide: 300 rows lie 5 GB apart."""
    a, sa = H.quantize_fp8_blocks(normal(70, 144))
    b, sb = H.quantize_fp8_blocks(normal(300, 144, seed=1), block_rows=128)
    want = H.fp8_block_matmul(a, sa, b, sb)
    for pitch in (2 ** 20 + 16, 2 ** 20 + 32, 2 ** 24 + 32):
        table = torch.empty((300, pitch), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        for at in (0, 16):
            wide = table[:, at:at + 144]
            wide.view(torch.uint8).copy_(b.view(torch.uint8))
            assert torch.equal(H.fp8_block_matmul(a, sa, wide, sb), want)
            assert torch.equal(H.fp8_block_matmul(a[:3], sa[:3], wide, sb), want[:3])
    far = torch.empty((70, 2 ** 22 + 4), device="cuda")[:, 1:3]
    far.copy_(sa)
    assert torch.equal(H.fp8_block_matmul(a, far, b, sb), want)


def test_product_carries_nan():
    x, w = normal(40, 300), normal(200, 300, seed=1)
    x[3, 200] = float("nan")
    a, sa = H.quantize_fp8_blocks(x)
    b, sb = H.quantize_fp8_blocks(w, block_rows=128)
    got = H.fp8_block_matmul(a, sa, b, sb)
    assert torch.isnan(got[3]).all() and torch.isfinite(got[[0, 1, 2, 4, 39]]).all()


def test_no_rows():
    a, sa = H.quantize_fp8_blocks(normal(4, 256))
    b, sb = H.quantize_fp8_blocks(normal(300, 256), block_rows=128)
    assert H.fp8_block_matmul(a[:0], sa[:0], b, sb).shape == (0, 300)
    assert H.fp8_block_matmul(a, sa, b[:0], sb[:0]).shape == (4, 0)


def test_streams_and_graphs():
    x, w = normal(130, 520), normal(700, 520, seed=1)
    b, sb = H.quantize_fp8_blocks(w, block_rows=128)

    def step():
        a, sa = H.quantize_fp8_blocks(x)
        return H.fp8_block_matmul(a, sa, b, sb), H.fp8_block_matmul(a.contiguous(), sa, b, sb, out_dtype=torch.float32)
    want = step()
    torch.cuda.synchronize()
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            got = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, got))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = step()
    with torch.cuda.graph(g2):
        o2 = step()
    for seed in (4, 5, 6):
        x.copy_(normal(130, 520, seed=seed))
        want = step()
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        for p, q, r in zip(want, o1, o2):
            assert torch.equal(p, q) and torch.equal(p, r)


def test_refusals():
    x = normal(20, 256)
    a, sa = H.quantize_fp8_blocks(x)
    b, sb = H.quantize_fp8_blocks(normal(300, 256), block_rows=128)
    for args in ((x, sa, b, sb), (a, sa[:5], b, sb), (a, sa, b, sa), (a, sa.double(), b, sb), (a, sa, b[:, :128], sb[:, :1]),
                 (a, sa, b.view(torch.uint8), sb), (a.cpu(), sa, b, sb), (a[0], sa, b, sb)):
        with pytest.raises(H.OrdaError):
            H.fp8_block_matmul(*args)
    with pytest.raises(H.OrdaError):
        H.fp8_block_matmul(a, sa, b, sb, out_dtype=torch.float16)
    for kw in (dict(m=x.half()), dict(m=x, block_rows=64), dict(m=x[0])):
        with pytest.raises(H.OrdaError):
            H.quantize_fp8_blocks(**kw)
