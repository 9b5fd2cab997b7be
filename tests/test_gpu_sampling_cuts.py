"""Cuts of top-k and top-p among thousands of tokens that are equal or next to it, where the
list of candidates does not hold them and bins are summed in fixed point. The oracle adds up
in numpy's long double: its sums of 2e4 masses are off by 1e-15 of themselves."""
import math

import numpy as np
import pytest
import torch

import orda_hip as H

pytestmark = pytest.mark.gpu


def kept(x, t=1.0, k=0, p=1.0, m=0.0):
    """The masses of a row's tokens (float64 numpy), 0 of those that are not kept."""
    t, p, m = (float(np.float32(a)) for a in (t, p, m))
    if x.max() == math.inf:
        x = np.where(x == math.inf, 0.0, -math.inf)
    w = np.exp((x - x.max()).astype(np.longdouble) / t)
    order = np.argsort(-x, kind="stable")
    ws, rank = w[order], np.arange(len(x))
    keep = (rank < (k if 0 < k < len(x) else len(x))) & (x[order] > -math.inf)
    masses = np.where(keep, ws, 0)
    if p < 1:
        keep &= (np.cumsum(masses) - masses < p * masses.sum()) | (rank == 0)
    keep &= (ws >= m) | (rank == 0)
    out = np.zeros_like(w)
    out[order[keep]] = ws[keep]
    return out


def check(x, seed=0, draws=24, **f):
    """x: a row. Numbers that are drawn lie in the middle of a kept token's share."""
    w = kept(x.double().numpy(), **f)
    at = np.nonzero(w)[0]
    cdf = np.cumsum(w[at])
    pick = np.unique(np.r_[0, len(at) - 1, np.random.default_rng(seed).integers(0, len(at), draws)])
    u = torch.tensor([float((cdf[i] - w[at[i]] / 2) / cdf[-1]) for i in pick], dtype=torch.float32)
    tokens, logprobs = H.sample_tokens(x.cuda().expand(len(u), -1).contiguous(), u.cuda(), temperature=f.get("t", 1.0),
                                       top_k=f.get("k"), top_p=f.get("p"), min_p=f.get("m"))
    assert tokens.tolist() == at[pick].tolist()
    want = [float(np.log(w[at[i]] / cdf[-1])) for i in pick]
    for a, b in zip(logprobs.tolist(), want):
        assert abs(a - b) <= 2.0 ** -24 * abs(b) + 1e-11


@pytest.mark.parametrize("beside", [10001, 100])
@pytest.mark.parametrize("k", [0, 20002])
def test_a_border_within_the_roundings_of_fixed_point(beside, k):
    """One 0, 10000 tokens at a, whose mass is 0.45 steps of 2^-43 over a whole number of them, `beside` at the
    next value b and the others at the one after. Half of all masses is 2e-10 under the sum up to the last a,
    which in fixed point is 5e-10 too small: the bin of b is found, where nothing is kept."""
    v = 20002
    a = np.float32(-3500.55 * 2.0 ** -43)
    b = np.nextafter(a, np.float32(-1))
    x = np.full(v, np.nextafter(b, np.float32(-1)), np.float32)
    at = np.random.default_rng(1).permutation(v)
    x[at[0]], x[at[1:10001]], x[at[10001:10001 + beside]] = 0, a, b
    if k:   # top-k first: all but one more
        x = np.insert(x, 7777, np.float32(-30))
    w = kept(x.astype(np.float64), k=k, p=0.5)
    assert (w > 0).sum() == 10001
    check(torch.from_numpy(x), k=k, p=0.5)


@pytest.mark.parametrize("v, n, largest", [(32000, 10000, 0), (32000, 10000, 20), (5000, 2600, 3)])
@pytest.mark.parametrize("banned", [-math.inf, math.inf], ids=["banned", "infinite"])
def test_top_k_of_more_than_there_are_among_equal_ones(v, n, largest, banned):
    """n equal logits and a few over them, the others banned (or n of +infinity, which alone count): top-p's share
    is of the tokens that there are, not of k."""
    at = np.random.default_rng(v + n).permutation(v)
    if banned < 0:
        x = np.full(v, -math.inf)
        x[at[:n]], x[at[:largest]] = 1.5, 2.0
    else:
        x = np.random.default_rng(n).standard_normal(v)
        x[at[:n]] = math.inf
    for k, p in ((n + n // 2, 0.5), (n + 1, 0.9), (n, 0.5), (n - 100, 0.5), (n + n // 2, 1.0), (n + n // 2, 0.001)):
        for dtype in (torch.float32, torch.bfloat16):
            check(torch.from_numpy(x).to(dtype), k=k, p=p)
            check(torch.from_numpy(x).to(dtype), k=k, p=p, m=0.9, t=0.7)


@pytest.mark.parametrize("listed", [0, 100])
@pytest.mark.parametrize("k", [0, 1])
def test_a_border_past_a_bin_that_fixed_point_ends_in(listed, k):
    """The same with masses that round up: half of all is 3e-10 over the sum up to the last of 10000 tokens at a (or
    of 100 at b, which a list holds), which in fixed point is 5e-10 too large. The token after those is kept too."""
    n = 10001 + listed
    a = np.float32(-3500.45 * 2.0 ** -43)
    b = np.nextafter(a, np.float32(-1))
    x = np.full(2 * n, np.nextafter(b, np.float32(-1)) if listed else b, np.float32)
    at = np.random.default_rng(2).permutation(2 * n)
    x[at[0]], x[at[1:10001]], x[at[10001:n]] = 0, a, b
    x = np.insert(x, 999, np.float32(math.log(1e-9)))
    if k:   # top-k first: all but one more
        k, x = len(x), np.insert(x, 7777, np.float32(-30))
    assert (kept(x.astype(np.float64), k=k, p=0.5) > 0).sum() == n + 1
    check(torch.from_numpy(x), k=k, p=0.5)
    m = float(np.float32(1 - 2.0 ** -24))   # (under all of them)
    assert (kept(x.astype(np.float64), k=k, p=0.5, m=m) > 0).sum() == n + 1
    check(torch.from_numpy(x), k=k, p=0.5, m=m)
