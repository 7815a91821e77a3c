"""Token sampling against a plain implementation in 64 bits.

The index has to be equal: the kernel's weights are doubles rounded to 2^-43 and
summed exactly, so only a draw within about 1e-11 of a border could differ.  prob
is rounded once to fp32 (2^-24); its total is off by 2^-44 per weight, below 2^-24
of a total that is at least 1 for 2^20 weights.
"""
import math

import numpy as np
import pytest
import torch

from reef_b200 import _lib
from reef_b200 import kernels as K

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_lib):
    yield
    K.check_device_error()


def plain(x, u, t=1.0, k=0, p=1.0, m=0.0):
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    if not (x > -np.inf).any():
        return -1, 0.0
    if not t > 0:
        return int(np.argmax(x)), 1.0
    top = x.max()
    if math.isinf(top):
        w = (x == top).astype(np.float64)
    else:
        w = np.exp(np.where(x > -np.inf, (x - top) / np.float64(t), -np.inf))
    order = np.argsort(-x, kind="stable")
    if 0 < k < x.size:
        order = order[:k]
    if p < 1:
        run = np.cumsum(w[order])
        before = run - w[order]
        stay = before < np.float64(p) * run[-1]
        stay[0] = True
        order = order[stay]
    if m > 0:
        order = order[w[order] >= min(np.float64(m), 1.0)]
    kept = np.sort(order)
    run = np.cumsum(w[kept])
    at = min(int(np.searchsorted(run, np.float64(u) * run[-1], side="right")), kept.size - 1)
    while w[kept[at]] == 0:  # u = 1: the last that weighs anything
        at -= 1
    return int(kept[at]), w[kept[at]] / run[-1]


def check(x, u, t=None, k=None, p=None, m=None):
    x, u = np.asarray(x, np.float32), np.asarray(u, np.float32)
    par = {"temperature": t, "top_k": k, "top_p": p, "min_p": m}
    dev = {n: None if v is None else torch.from_numpy(
        np.asarray(v, np.int32 if n == "top_k" else np.float32)).cuda() for n, v in par.items()}
    index, prob = K.sample_f32(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda(), **dev)
    index, prob = index.cpu().numpy(), prob.cpu().numpy()
    for r in range(x.shape[0]):
        f = lambda v, d: d if v is None else np.asarray(v, np.float32)[r]
        uu = u[r] if 0 <= u[r] <= 1 else (1.0 if u[r] > 1 else 0.0)
        i, q = plain(x[r], uu, f(t, 1.0), 0 if k is None else int(k[r]), f(p, 1.0), f(m, 0.0))
        assert index[r] == i, (r, index[r], i, u[r])
        assert abs(prob[r] - q) <= 2.0**-23 * q, (r, prob[r], q)


def logits(rows, n, seed, std=3.0, coarse=False):
    x = np.random.RandomState(seed).randn(rows, n).astype(np.float32) * std
    return np.round(x * 4) / 4 if coarse else x


SIZES = [1, 2, 3, 31, 33, 255, 1000, 4097, 32000, 50257, 65537]


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("coarse", [False, True])
def test_every_filter(n, coarse):
    rows = 24
    r = np.random.RandomState(n)
    x, u = logits(rows, n, n, coarse=coarse), r.rand(rows).astype(np.float32)
    t = r.uniform(0.3, 2.0, rows)
    check(x, u)
    check(x, u, t)
    check(x, u, t, k=r.randint(1, n + 2, rows))
    check(x, u, t, p=r.uniform(0.01, 0.999, rows))
    check(x, u, t, m=r.uniform(0.001, 0.5, rows))
    check(x, u, t, k=r.randint(1, min(n, 300) + 1, rows), p=r.uniform(0.3, 1.1, rows),
          m=r.uniform(-0.1, 0.2, rows))


@pytest.mark.parametrize("rows,n", [(1, 128000), (5, 262144), (160, 20000), (2, 500001), (1, 1 << 20)])
def test_large_rows(rows, n):
    """From several CTAs a row to rows that do not fit on chip."""
    r = np.random.RandomState(rows)
    x, u = logits(rows, n, rows), r.rand(rows).astype(np.float32)
    check(x, u, np.full(rows, 0.9))
    check(x, u, np.full(rows, 1.3), k=r.randint(1, 2000, rows), p=np.full(rows, 0.95))
    check(x, u, np.full(rows, 3.0), p=np.full(rows, 0.8), m=np.full(rows, 1e-4))


def test_flat_rows_and_ties():
    """All logits equal: the order is the index; the draw is a share of the vocabulary."""
    n, rows = 5003, 64
    x = np.full((rows, n), -1.25, np.float32)
    u = (np.arange(rows) / rows).astype(np.float32)
    check(x, u)
    check(x, u, k=np.full(rows, 17))
    check(x, u, p=np.full(rows, 0.25))
    x[:, 100:200] = 2.0
    check(x, u, k=np.full(rows, 50), p=np.full(rows, 0.5))
    check(x, u, k=np.full(rows, 150), p=np.full(rows, 0.999))
    check(x, u, m=np.full(rows, 1.0))


@pytest.mark.parametrize("n", [900, 20000, 128000])
@pytest.mark.parametrize("equal", [40, 300, 700, 899])
def test_borders_among_equal_values(n, equal):
    """Top-p's border inside a block of equal logits, from a few to more than a step
    of the histogram is sorted for, with heavier ones above and lighter ones below."""
    rows = 6
    r = np.random.RandomState(n + equal)
    x = r.randn(rows, n).astype(np.float32) - 30.0
    for i in range(rows):
        at = r.permutation(n)[:equal]
        x[i, at] = 2.0
        x[i, at[:10]] = 2.0 + np.arange(10, dtype=np.float32) / 4
    u = r.rand(rows).astype(np.float32)
    check(x, u, p=np.full(rows, 0.7))
    check(x, u, p=r.uniform(0.2, 0.999, rows), m=np.full(rows, 0.05))
    check(x, u, k=np.full(rows, equal // 2 + 5), p=r.uniform(0.2, 0.999, rows))


@pytest.mark.parametrize("n", [1000, 20000])
def test_steps_with_more_elements_than_are_sorted(n):
    """A list that one CTA takes over (at most 1024) with more than 512 equal logits in
    top-p's step: the count of them is read by every warp before the selection that
    follows clears it, whatever the warps' pace, in many rows at once and again and again."""
    rows = 600
    r = np.random.RandomState(n)
    x = np.full((rows, n), -80.0, np.float32)
    equal = 513 + np.arange(rows) % 488
    for i in range(rows):
        at = r.permutation(n)[: equal[i]]
        x[i, at] = 1.5
        x[i, at[: i % 7]] = 1.5 + np.arange(i % 7, dtype=np.float32) / 8
    u, p = r.rand(rows).astype(np.float32), r.uniform(0.3, 0.95, rows).astype(np.float32)
    check(x, u, p=p)
    dev = [torch.from_numpy(a).cuda() for a in (x, u, p)]
    want = K.sample_f32(dev[0], dev[1], top_p=dev[2])
    for _ in range(20):
        got = K.sample_f32(dev[0], dev[1], top_p=dev[2])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def tail_value(bits, t):
    """A float near -bits ln 2 t whose weight against 0, in units of 2^-43, is a quarter
    or less off a whole number: a weight off by less than a quarter rounds to it."""
    x = np.float32(-bits * math.log(2.0) * t)
    while True:
        w = math.exp(float(x) / float(t)) * 2.0**43
        if abs(w - round(w)) <= 0.25:
            return x, round(w)
        x = np.nextafter(x, np.float32(-math.inf))


@pytest.mark.parametrize("n", [5000, 128000, 1 << 20])
@pytest.mark.parametrize("t", [0.7, 1.3])
@pytest.mark.parametrize("bits", [(20.3,), (21.4,), (22.6,), (23.5,), (25.2,), (26.7,), (28.1,),
                                  (20.1, 20.9, 21.8, 22.4, 24.3, 26.9, 29.5)])
def test_equal_logits_that_weigh_little(n, t, bits):
    """One logit ahead of a tail of equal ones that weigh 2^-20 to 2^-30 of it.  Equal
    weights share their rounding, so it adds up over the tail: with every weight the
    whole number of 2^-43 next to it, sums and draws are exact (u times the total is
    rounded to 53 bits, 2 units here).  Against weights that are not rounded a border, or
    u times the total, moves by 0.625 units for each of n at most."""
    t, rows = np.float32(t), 32
    r = np.random.RandomState(n % 1000 + int(10 * bits[0]))
    values = [tail_value(b, t) for b in bits]
    pick = r.randint(0, len(values), n)
    at = n // 3
    x = np.array([v for v, _ in values], np.float32)[pick]
    w = np.array([q for _, q in values], np.int64)[pick]
    x[at], w[at] = 0.0, 1 << 43
    run = np.cumsum(w)
    total = int(run[-1])
    exact = np.exp(x.astype(np.float64) / np.float64(t))
    run64 = np.cumsum(exact.astype(np.longdouble))
    # most draws into the tail, before and behind the first
    tail = (total - (1 << 43)) / total
    u = np.concatenate([r.rand(rows // 2) * tail / 3, 1 - r.rand(rows // 2) * tail * 2 / 3])
    u = np.minimum(u.astype(np.float32), np.nextafter(np.float32(1), np.float32(0)))
    xs = torch.from_numpy(x).cuda().expand(rows, n).contiguous()
    us, ts = torch.from_numpy(u).cuda(), torch.full((rows,), float(t), device="cuda")
    index, prob = K.sample_f32(xs, us, temperature=ts)
    index, prob = index.cpu().numpy(), prob.cpu().numpy()
    slack = np.longdouble(n * 0.625 * 2.0**-43)
    checked = 0
    for i in range(rows):
        goal = int(np.float64(u[i]) * np.float64(total))
        lo, hi = (int(np.searchsorted(run, goal + e, side="right")) for e in (-2, 2))
        if lo == hi:
            checked += 1
            assert index[i] == lo, (i, index[i], lo)
        j, goal = index[i], np.longdouble(u[i]) * run64[-1]
        assert (run64[j - 1] if j else 0.0) <= goal + 2 * slack and run64[j] >= goal - 2 * slack
        assert abs(prob[i] - exact[j] / (total * 2.0**-43)) <= 2.0**-23 * prob[i]
    assert checked >= rows // 2
    # top-p with its border in the tail: the largest values first, then by index
    order = np.argsort(-x, kind="stable")
    before = np.cumsum(w[order]) - w[order]
    for p in (np.float32(0.9), np.float32(1.0 - tail / 2)):
        want = float(p) * total
        kept = order[before < want]
        if abs(before[kept.size - 1] - want) < 4 or abs(before[min(kept.size, n - 1)] - want) < 4:
            continue
        kept = np.sort(kept)
        run = np.cumsum(w[kept])
        index, _ = K.sample_f32(xs, us, temperature=ts, top_p=torch.full((rows,), float(p), device="cuda"))
        for i, got in enumerate(index.cpu().numpy()):
            goal = int(np.float64(u[i]) * np.float64(run[-1]))
            lo, hi = (int(np.searchsorted(run, goal + e, side="right")) for e in (-2, 2))
            if lo == hi:
                assert got == kept[lo], (p, i, got, kept[lo])


@pytest.mark.parametrize("p", [0.99, 0.999999])
def test_nearly_everything_kept(p):
    """Flat rows of which top-p leaves out little: what is kept does not fit a list."""
    rows, n = 4, 128000
    r = np.random.RandomState(5)
    x = (r.randn(rows, n) * 0.2).astype(np.float32)
    check(x, r.rand(rows).astype(np.float32), p=np.full(rows, p))


def test_masks_and_values_that_are_no_numbers():
    n = 3001
    low, inf, nan = np.finfo(np.float32).min, np.inf, np.nan
    x = logits(10, n, 3)
    x[0, :] = -inf                      # nothing left
    x[1, :] = nan
    x[2, :] = -inf
    x[2, 2000] = -5.0                   # one left
    x[3, ::2] = -inf
    x[4, ::3] = nan
    x[5, 5:] = low                      # masked with the lowest value
    x[6, :] = low                       # and everywhere: equal weights
    x[7, 700] = inf                     # only +inf weighs
    x[7, 900] = inf
    x[8, :] = -inf
    x[8, 17] = nan
    x[8, 18] = low
    x[9, 0] = -0.0
    x[9, 1:] = np.where(np.arange(n - 1) % 2, 0.0, -0.0)  # zeros of both signs are equal
    for u in (0.0, 0.3, 0.999, np.nextafter(np.float32(1), np.float32(0))):
        us = np.full(10, u, np.float32)
        check(x, us)
        check(x, us, np.full(10, 0.7), k=np.full(10, 40))
        check(x, us, np.full(10, 0.7), p=np.full(10, 0.6))
        check(x, us, np.full(10, 0.7), k=np.full(10, 2000), p=np.full(10, 0.9), m=np.full(10, 0.01))
        check(x, us, np.zeros(10))
        check(x, us, np.full(10, inf))
        check(x, us, np.full(10, inf), k=np.full(10, 3))


def test_parameters_at_their_ends():
    rows, n = 12, 777
    x, u = logits(rows, n, 1), np.linspace(0, 0.99, rows).astype(np.float32)
    inf, nan = np.inf, np.nan
    check(x, u, [0.0, -1.0, nan, 1e-30, 1e30, inf, 1.0, 1e-3, 5.0, 1e-45, 0.5, 2.0])
    check(x, u, k=[0, -5, 1, 2, n - 1, n, n + 1, 2**31 - 1, -2**31, 3, 700, 40])
    check(x, u, p=[0.0, -1.0, 1.0, 1.5, 1e-30, 0.99999994, 0.5, inf, 1e-7, 0.1, 0.9, -inf])
    check(x, u, m=[0.0, -1.0, 1.0, 1.5, 1e-30, 0.99999994, 0.5, inf, 1e-7, 0.1, 0.9, -inf])
    bad = torch.tensor([nan], device="cuda")
    one = torch.from_numpy(x[:1]).cuda()
    half = torch.tensor([0.5], device="cuda")
    want = K.sample_f32(one, half)
    for got in (K.sample_f32(one, half, top_p=bad), K.sample_f32(one, half, min_p=bad)):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check(x, [-1.0, 1.0, 1.5, inf, -inf, 0, 1, 0.25, 1, 1, 1, 1], p=np.full(rows, 0.5))
    zero = K.sample_f32(one, torch.zeros(1, device="cuda"))
    assert torch.equal(K.sample_f32(one, bad)[0], zero[0])


def test_draws_follow_the_distribution():
    """Evenly spaced u give every token its share, to one draw of 4096."""
    n, rows = 50, 4096
    row = logits(1, n, 5, std=1.0)
    x = np.repeat(row, rows, 0)
    u = ((np.arange(rows) + 0.5) / rows).astype(np.float32)
    index, _ = K.sample_f32(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda())
    got = np.bincount(index.cpu().numpy(), minlength=n)
    w = np.exp(row[0].astype(np.float64))
    assert np.all(np.abs(got - rows * w / w.sum()) <= 1.0 + 1e-3)


def test_rows_at_any_alignment_same_bits_streams_and_graphs():
    x = torch.from_numpy(logits(7, 10007, 9)).cuda()  # odd rows: no two aligned alike
    u = torch.rand(7, device="cuda")
    p = torch.full((7,), 0.9, device="cuda")
    want = K.sample_f32(x, u, top_p=p)
    flat = torch.empty(7 * 10007 + 1, device="cuda")
    flat[1:] = x.flatten()
    moved = flat[1:].view(7, 10007)
    for _ in range(3):
        got = K.sample_f32(moved, u, top_p=p)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.sample_f32(x, u, top_p=p)
    side.synchronize()
    assert torch.equal(got[0], want[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = K.sample_f32(x, u, top_p=p)
    x.neg_()
    g.replay()
    want = K.sample_f32(x, u, top_p=p)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_index_only():
    x, u = torch.randn((3, 100), device="cuda"), torch.rand(3, device="cuda")
    index = torch.empty(3, dtype=torch.int32, device="cuda")
    _lib.call("reef_b200_sample_f32", 3, 100, x.data_ptr(), None, None, None, None, u.data_ptr(),
              index.data_ptr(), None, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(index, K.sample_f32(x, u)[0])
