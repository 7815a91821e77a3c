"""Attention of drafted tokens over the int8 KV cache against a plain
implementation in 64 bits on the dequantised inputs.

Tolerance, per output element, relative to W = sum p |v| / sum p (what the
element's terms add up to without cancelling).  P, with the key's V scale and
lifted to 2^11 at the largest or more, goes into the product as two f16 terms, each
rounding off by half a step, 2^-12 of what is left (2^-24 together), or by half
of the smallest number, 2^-25, where that is more: whatever W is, an element
may be off by 2^-36 of the row's largest p * v_scale for each unit of the keys'
codes, 2^-36 max(p v_scale) sum |code| in all (it is what is left where the keys
that count have a code of 0 there).  exp2 is
off by 2 ulp (2^-22), log2 of a V scale by 2^-22 and a score s (log2 units,
that log2 in it) by four fp32 roundings, 2^-22 max|s| of p, in the numerator and in
the denominator.  A tensor-core add may lose 2^-23, and at most seven tiles of
them (112, two terms for 16 keys each) follow one another before a rounded add, one
per 512 keys and some where warps, parts and CTAs are joined.
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


def rows8(gen, shape, std):
    x = torch.randn(shape + (128,), generator=gen, device="cuda") * std
    sc = x.abs().amax(-1) / 127.0
    return torch.round(x / sc[..., None]).clamp(-127, 127).to(torch.int8), sc


def trees(seed, b, t):
    r = np.random.RandomState(seed)
    p = np.floor(r.random_sample((b, t)) * np.arange(t)).astype(np.int32)
    p[:, 0] = -1
    if t > 3:
        p[0, 2] = -1  # a second root
    return p


def make(b, t, hq, hkv, max_len, seed, std=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q8, qs = rows8(g, (b, t, hq), std)
    k8, ks = rows8(g, (b, hkv, max_len), std)
    v8, vs = rows8(g, (b, hkv, max_len), 1.0)
    return dict(q8=q8, q_scale=qs, k_cache=k8, k_scale=ks, v_cache=v8, v_scale=vs)


def check(x, lens, parents, draft_lens, out, sm):
    """Every live row of `out` against 64 bits; rows behind stay -7."""
    q8, ks, vs = x["q8"], x["k_scale"], x["v_scale"]
    b, t, hq, _ = q8.shape
    hkv = ks.shape[1]
    for i in range(b):
        n, d = int(lens[i]), t if draft_lens is None else int(draft_lens[i])
        assert torch.all(out[i, max(d, 0):] == -7.0)
        if d <= 0:
            continue
        sees = torch.zeros((d, n + d), dtype=torch.bool)
        sees[:, :n] = True
        for r in range(d):
            j = r
            while j >= 0:
                sees[r, n + j] = True
                up = j - 1 if parents is None else int(parents[i][j])
                j = up if up < j else -1
        sees = sees.cuda()
        for h in range(hq):
            kh = h // (hq // hkv)
            q = q8[i, :d, h].double() * x["q_scale"][i, :d, h, None].double()
            k = x["k_cache"][i, kh, : n + d].double() * ks[i, kh, : n + d, None].double()
            v = x["v_cache"][i, kh, : n + d].double() * vs[i, kh, : n + d, None].double()
            s = torch.where(sees, q @ k.T * sm, -math.inf)
            p = torch.softmax(s, -1)
            v = torch.nan_to_num(v) if not torch.isfinite(v).all() else v
            want, weight = p @ v, p @ v.abs()
            smax = float(s[sees].abs().max()) * math.log2(math.e)
            smax += float(torch.log2(vs[i, kh, : n + d]).abs().max())
            rel = 2.0**-24 + 2 * (2 + smax) * 2.0**-22 + ((n + d) / 512 + 192) * 2.0**-23
            codes = x["v_cache"][i, kh, : n + d].double().abs().sum(0)
            small = 2.0**-36 * (p * vs[i, kh, : n + d].double()).amax(1, keepdim=True) * codes
            off = (out[i, :d, h].double() - want).abs()
            assert bool((off <= rel * weight + small).all()), (i, h, float((off / weight).max()), rel)


def run(x, lens, parents=None, draft_lens=None, sm=None, **kw):
    b, t, hq, _ = x["q8"].shape
    dev = lambda a: None if a is None else torch.tensor(np.asarray(a, np.int32), device="cuda")
    out = torch.full((b, t, hq, 128), -7.0, device="cuda")
    got = K.tree_attn_i8(**x, lens=dev(lens), parents=dev(parents), draft_lens=dev(draft_lens),
                         sm_scale=sm, out=out, **kw)
    assert got is out
    torch.cuda.synchronize()
    return out


CASES = [
    # batch, drafts, heads_q, heads_kv, max_len, lens, draft_lens, tree
    (1, 1, 1, 1, 4, [0], None, False),               # one token, nothing committed
    (1, 1, 4, 4, 132, [131], None, False),           # the last row of the cache
    (2, 4, 8, 2, 300, [0, 296], None, True),         # empty and full
    (3, 7, 4, 1, 520, [127, 128, 250], None, True),  # drafts across a tile's border
    (3, 5, 6, 2, 260, [121, 5, 255], [5, 0, 1], True),   # three heads a group; no drafts
    (1, 64, 2, 1, 1024, [901], None, True),          # the widest tree
    (1, 64, 8, 8, 192, [128], None, False),          # a chain of 64
    (5, 8, 8, 1, 2048, [2040, 1, 1000, 129, 0], [8, 3, 8, 1, 8], True),
    (2, 3, 16, 1, 4096, [4000, 77], None, True),     # 48 rows, several row tiles
    (1, 2, 40, 2, 640, [600], None, False),          # 40 rows of one KV head
    (2, 48, 32, 4, 1500, [1400, 129], [48, 11], True),   # 384 rows: several tiles of 128
    (1, 17, 8, 1, 1024, [1000], None, True),         # 136 rows: a tile of eight
    (150, 3, 8, 1, 400, [(97 * i) % 398 for i in range(150)], None, False),  # 24 rows, many segments
    (300, 2, 2, 1, 256, [(37 * i) % 254 for i in range(300)], None, False),  # more than CTAs
    (40, 16, 8, 2, 512, [(61 * i) % 497 for i in range(40)], [i % 17 for i in range(40)], True),
]


@pytest.mark.parametrize("b,t,hq,hkv,max_len,lens,draft_lens,tree", CASES)
def test_against_64_bits(b, t, hq, hkv, max_len, lens, draft_lens, tree):
    x = make(b, t, hq, hkv, max_len, seed=b + t + hq + max_len)
    parents = trees(7 * b + t, b, t) if tree else None
    sm = 1.0 / math.sqrt(128)
    check(x, lens, parents, draft_lens, run(x, lens, parents, draft_lens, sm), sm)


@pytest.mark.parametrize("t,hq", [(1, 8), (2, 8), (16, 8)])
def test_long_rows_lose_nothing(t, hq):
    """Over 16k keys in one CTA's hands the error stays that of a few dozen adds: in
    the 2-norm below 64 adds that truncate by 2^-24 on average, and 2^-20 for the
    scores."""
    b, hkv, max_len = 150, 1, 16384
    x = make(b, t, hq, hkv, max_len, seed=4 + t)
    lens = [max_len - t] * b
    out = run(x, lens, sm=128**-0.5)
    far = norm = 0.0
    for i in range(0, b, 37):
        k = x["k_cache"][i, 0].double() * x["k_scale"][i, 0, :, None].double()
        v = x["v_cache"][i, 0].double() * x["v_scale"][i, 0, :, None].double()
        for r in range(t):
            q = x["q8"][i, r].double() * x["q_scale"][i, r, :, None].double()
            s = q @ k.T * 128**-0.5
            s[:, max_len - t + r + 1:] = -math.inf
            want = torch.softmax(s, -1) @ v
            far += float((out[i, r].double() - want).square().sum())
            norm += float(want.square().sum())
    assert math.sqrt(far / norm) < 64 * 2.0**-24 + 2.0**-20


@pytest.mark.parametrize("t", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("grows", [False, True])
def test_every_count_of_tiles(t, grows):
    """One to sixteen tiles of 128 keys in one CTA's hands (a sequence each), the scores
    growing from tile to tile or not: sums that are moved and rescaled."""
    b, sm = 150, 128**-0.5
    x = make(b, t, 8, 1, 2048, seed=60 + t)
    if grows:
        x["k_scale"] *= 1.0 + 0.5 * (torch.arange(2048, device="cuda") // 128)
    for tiles in range(1, 17):
        out = run(x, [tiles * 128 - t] * b, sm=sm)
        for i in (0, 77, 149):
            check({k: v[i:i + 1] for k, v in x.items()}, [tiles * 128 - t], None, None,
                  out[i:i + 1], sm)


@pytest.mark.parametrize("std,sm", [(0.01, 1.0), (6.0, 0.3), (1.5, 0.0)])
def test_flat_and_peaked_scores(std, sm):
    x = make(2, 6, 8, 2, 400, seed=11, std=std)
    check(x, [390, 17], None, None, run(x, [390, 17], None, None, sm), sm)


@pytest.mark.parametrize("hq", [4, 16])
def test_scales_far_apart(hq):
    """V scales of 2^-60 to 2^60 in one sequence: P times the scale keeps its range."""
    x = make(1, 4, hq, 1, 256, seed=3)
    e = torch.arange(256, device="cuda").float() % 121 - 60
    x["v_scale"] = torch.exp2(e)[None, None].contiguous()
    check(x, [250], None, None, run(x, [250], None, None, 0.01), 0.01)


@pytest.mark.parametrize("hq", [2, 16])
def test_v_scales_of_zero(hq):
    """Keys whose V scale is 0 take their share of the softmax and add nothing; where
    all are, the output is 0."""
    x = make(2, 4, hq, 1, 256, seed=13)
    x["v_scale"][0, 0, ::2] = 0.0
    x["v_scale"][1] = 0.0
    out = run(x, [250, 100], sm=0.05)
    assert not out[1].any()
    v = x["v_cache"][0, 0, :254].double() * x["v_scale"][0, 0, :254, None].double()
    k = x["k_cache"][0, 0, :254].double() * x["k_scale"][0, 0, :254, None].double()
    q = x["q8"][0, 3].double() * x["q_scale"][0, 3, :, None].double()
    p = torch.softmax(q @ k.T * 0.05, -1)
    assert bool(((out[0, 3].double() - p @ v).abs() <= 1e-5 * (p @ v.abs())).all())


def zeros_lifted(x):
    """The same product with V scales of 0 as codes of 0 (what `check` takes log2 of)."""
    none = x["v_scale"] == 0
    return x | dict(v_cache=torch.where(none[..., None], 0, x["v_cache"]),
                    v_scale=torch.where(none, 2.0**-64, x["v_scale"]))


@pytest.mark.parametrize("t,hq", [(1, 8), (2, 8), (4, 8), (8, 8), (16, 8)])
def test_a_long_stretch_of_v_scales_of_zero(t, hq):
    """24576 keys whose V scale is 0 before 8192 with values: their part of the softmax
    sum stays finite wherever the keys are cut, also where their scores pass the first
    ones' by just less than what raises the running maximum."""
    b, max_len, zeros = 150, 32768, 24576
    x = make(b, t, hq, 1, 4, seed=70 + t)
    g = torch.Generator(device="cuda").manual_seed(71)
    v8, vs = rows8(g, (1, 1, max_len), 1.0)
    vs[:, :, :zeros] = 0.0
    x |= dict(q8=torch.ones_like(x["q8"]), q_scale=torch.ones_like(x["q_scale"]),
              k_cache=torch.ones((b, 1, max_len, 128), dtype=torch.int8, device="cuda"),
              k_scale=torch.full((b, 1, max_len), 2.6, device="cuda"),
              v_cache=v8.expand(b, -1, -1, -1).contiguous(),
              v_scale=vs.expand(b, -1, -1).contiguous())
    x["k_scale"][:, :, :128] = 0.0
    out = run(x, [max_len - t] * b, sm=1.0 / 128)
    for i in range(0, b, 13):
        check(zeros_lifted({k: v[i:i + 1] for k, v in x.items()}), [max_len - t], None, None,
              out[i:i + 1], 1.0 / 128)


@pytest.mark.parametrize("t,hq", [(4, 2), (4, 4), (8, 4), (8, 8), (8, 16)])
def test_v_scales_of_zero_beside_large_ones(t, hq):
    """Keys with V scales of 0 keep their share beside scales of 2^48."""
    x = make(2, t, hq, 1, 1024, seed=14)
    x["v_scale"][0, 0, ::2] = 0.0
    x["v_scale"][0, 0, 1::2] = 2.0**48
    x["v_scale"][1] = 2.0**48
    x["v_scale"][1, 0, :700] = 0.0
    out = run(x, [1000, 900], sm=0.02)
    check(zeros_lifted(x), [1000, 900], None, None, out, 0.02)


@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf, 3.4e38])
@pytest.mark.parametrize("hq", [2, 8])  # 8 and 32 query rows: both kernels
def test_rows_nobody_sees_add_nothing(junk, hq):
    """Scales behind the drafts, and of a sibling's row, that are not numbers."""
    x = make(2, 4, hq, 1, 260, seed=5)
    parents = [[-1, 0, 0, 1], [-1, 0, 1, 2]]  # nodes 1 and 2 of sequence 0 are siblings
    lens = [126, 200]
    want = run(x, lens, parents, None, 0.1)
    for c in ("k_scale", "v_scale"):
        x[c][0, :, 130:] = junk
        x[c][1, :, 204:] = junk
    got = run(x, lens, parents, None, 0.1)
    assert torch.equal(got, want)
    for c in ("k_scale", "v_scale"):
        x[c][0, :, 128] = junk  # node 2: seen by itself alone
    got = run(x, lens, parents, None, 0.1)
    assert torch.equal(got[0, [0, 1, 3]], want[0, [0, 1, 3]]) and torch.equal(got[1], want[1])


def test_parents_that_are_no_earlier_node_count_as_roots():
    x = make(1, 5, 2, 1, 128, seed=9)
    assert torch.equal(run(x, [100], [[-1, 1, 7, -5, 2]]), run(x, [100], [[-1, -1, -1, -1, 2]]))


def test_a_chain_is_the_default_and_a_single_token_is_decode():
    x = make(3, 6, 8, 2, 512, seed=21)
    lens = [500, 3, 128]
    chain = run(x, lens)
    assert torch.equal(chain, run(x, lens, [[-1, 0, 1, 2, 3, 4]] * 3))
    # the existing single-token head on the row that token 5 stands in
    ws = torch.empty(_lib.lib().reef_b200_decode_attn_workspace_bytes(3, 8, 512),
                     dtype=torch.uint8, device="cuda")
    n = torch.tensor([v + 6 for v in lens], dtype=torch.int32, device="cuda")
    q8, qs = x["q8"][:, 5].contiguous(), x["q_scale"][:, 5].contiguous()
    out = torch.empty((3, 8, 128), device="cuda")
    _lib.call("reef_b200_decode_attn_i8", 3, 8, 2, 128, 512, n.data_ptr(), 0, 128**-0.5,
              q8.data_ptr(), qs.data_ptr(), x["k_cache"].data_ptr(), x["k_scale"].data_ptr(),
              x["v_cache"].data_ptr(), x["v_scale"].data_ptr(), ws.data_ptr(), ws.numel(),
              out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert float((chain[:, 5] - out).abs().max()) < 1e-2  # that head's own tolerance


def test_same_call_same_bits():
    x = make(9, 8, 16, 2, 1500, seed=2)
    lens, par = [(331 * i) % 1490 for i in range(9)], trees(4, 9, 8)
    first = run(x, lens, par)
    for _ in range(3):
        assert torch.equal(run(x, lens, par), first)


def test_positions_outside_the_cache_are_reported_and_left_out():
    x = make(3, 4, 2, 1, 64, seed=1)
    out = run(x, [60, 61, -1])
    assert torch.all(out[1:] == -7.0)
    check({k: v[:1] for k, v in x.items()}, [60], None, None, out[:1], 128**-0.5)
    with pytest.raises(_lib.ReefError, match="0x201"):
        K.check_device_error()


@pytest.mark.parametrize("t,hq", [(4, 2), (4, 4), (8, 4), (8, 8), (16, 8)])
def test_shares_pass_over_sequences_that_are_empty_or_do_not_fit(t, hq):
    """8 to 128 query rows over a cache long enough that CTAs take equal shares of all
    sequences' keys: some at the beginning, in the middle and at the end have no drafts or
    a place outside the cache; draft_lens above the drafts count as all of them."""
    max_len = 2048
    rows = [(max_len - t + 1, t), (-1, t), (5, 0), (700, t), (max_len + 1, 1), (1999, -1),
            (2000, t + 3), (0, 1), (3, -2**31), (129, 2), (max_len, 0), (1500, t), (17, 0),
            (2**31 - 1, t), (max_len - 1, 2), (127, t - 1), (max_len - t, t), (1, 0), (-5, 1)]
    lens, drafts = [a for a, _ in rows], [d for _, d in rows]
    x = make(len(rows), t, hq, 1, max_len, seed=90 + t + hq)
    parents = trees(91, len(rows), t)
    out = run(x, lens, parents, drafts)
    live = 0
    for i, (n, d) in enumerate(rows):
        d = min(d, t)
        if d <= 0 or n < 0 or n + d > max_len:
            assert torch.all(out[i] == -7.0), i
            continue
        live += 1
        check({k: v[i:i + 1] for k, v in x.items()}, [n], parents[i:i + 1], [d], out[i:i + 1],
              128**-0.5)
    assert live == 7
    with pytest.raises(_lib.ReefError, match="0x201"):
        K.check_device_error()
    none = run(x, [5] * len(rows), parents, [0] * len(rows))  # nobody has any
    assert torch.all(none == -7.0)


def test_on_another_stream_and_in_a_graph():
    x = make(2, 8, 8, 1, 700, seed=31)
    lens = torch.tensor([690, 333], dtype=torch.int32, device="cuda")
    want = K.tree_attn_i8(**x, lens=lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.tree_attn_i8(**x, lens=lens)
    side.synchronize()
    assert torch.equal(got, want)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(K.tree_attn_i8(**x, lens=lens))
        graphs.append(g)
    lens.fill_(12)
    x["q8"].neg_()
    for g in graphs + graphs:
        g.replay()
    torch.cuda.synchronize()
    want = K.tree_attn_i8(**x, lens=lens)
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_a_row_of_scales_past_two_to_the_31_bytes():
    """Offsets of K rows pass 32 bits: the last of 140 sequences x 4 heads x 32768 rows."""
    b, hkv, max_len = 140, 4, 32768
    x = make(b, 2, 4, hkv, 4, seed=8)
    k = torch.zeros((b, hkv, max_len, 128), dtype=torch.int8, device="cuda")
    assert k.numel() > 1 << 31
    sc = torch.zeros((b, hkv, max_len), device="cuda")
    g = torch.Generator(device="cuda").manual_seed(6)
    full = dict(q8=x["q8"], q_scale=x["q_scale"], k_cache=k, k_scale=sc, v_cache=k.clone(),
                v_scale=sc.clone())
    for c, std in (("k", 1.5), ("v", 1.0)):
        full[c + "_cache"][-1, :, -500:], full[c + "_scale"][-1, :, -500:] = rows8(g, (hkv, 500), std)
    lens = [0] * (b - 1) + [max_len - 2]
    draft_lens = [0] * (b - 1) + [2]
    out = run(full, lens, None, draft_lens)
    last = {n: v[-1:] for n, v in full.items()}
    check(last, lens[-1:], None, None, out[-1:], 128**-0.5)
