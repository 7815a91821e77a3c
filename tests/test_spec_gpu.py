"""The walk that accepts drafted tokens, the compaction of the int8 KV cache to
it (both exact, against plain loops), the residual RMSNorm with int8 output
(the bits of the two operators it joins), and a run of them together."""
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


def dev(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype)).cuda()


# ---- tree_accept -----------------------------------------------------------------


def walk(parents, tokens, chosen, d):
    t = len(tokens)
    path, cur = [], 0 if d > 0 else -1
    while cur >= 0:
        path.append(cur)
        cur = next((c for c in range(cur + 1, d)
                    if (c - 1 if parents is None else parents[c]) == cur and
                    tokens[c] == chosen[cur]), -1)
    return path + [-1] * (t - len(path)), len(path), chosen[path[-1]] if path else -1


@pytest.mark.parametrize("b,t", [(1, 1), (3, 2), (130, 8), (9, 31), (9, 32), (9, 33), (70, 64)])
@pytest.mark.parametrize("kinds", [2, 30])
@pytest.mark.parametrize("shape", ["tree", "chain", "ragged"])
def test_accept_walks_the_tree(b, t, kinds, shape):
    r = np.random.RandomState(b + t + kinds)
    parents = np.floor(r.random_sample((b, t)) * np.arange(t)).astype(np.int32)
    parents[:, 0] = -1
    if t > 5:
        parents[0, 3], parents[0, 4], parents[0, 5] = 3, 60, -9  # no earlier nodes: never reached
    if shape == "chain":
        parents = None
    lens = r.randint(-1, t + 3, b) if shape == "ragged" else None
    tokens, chosen = r.randint(0, kinds, (b, t)), r.randint(0, kinds, (b, t))
    for i in range(1, t):
        hit = np.nonzero(r.rand(b) < 0.6)[0]
        up = np.full(len(hit), i - 1) if parents is None else np.clip(parents[hit, i], 0, i - 1)
        chosen[hit, up] = tokens[hit, i]
    path, accepted, following = K.tree_accept(
        dev(tokens), dev(chosen), parents=None if parents is None else dev(parents),
        draft_lens=None if lens is None else dev(lens))
    for i in range(b):
        d = t if lens is None else min(max(int(lens[i]), 0), t)
        want = walk(None if parents is None else parents[i], tokens[i], chosen[i], d)
        assert (path[i].tolist(), int(accepted[i]), int(following[i])) == want


def test_accept_full_chain_and_ids_of_32_bits():
    tokens = torch.full((2, 64), -1, dtype=torch.int32, device="cuda")  # the id 2^32 - 1
    path, accepted, following = K.tree_accept(tokens, tokens.clone())
    assert accepted.tolist() == [64, 64] and path.tolist() == [list(range(64))] * 2
    assert following.tolist() == [-1, -1]


# ---- kv_compact_i8 ---------------------------------------------------------------


def cache(shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = {}
    for n in ("k", "v"):
        c[n + "_cache"] = torch.randint(-128, 128, shape + (128,), generator=g, device="cuda",
                                        dtype=torch.int8)
        c[n + "_scale"] = torch.rand(shape, generator=g, device="cuda")
    return c


def compacted(c, lens, path, accepted):
    want = {n: v.clone() for n, v in c.items()}
    for b, n in enumerate(lens):
        for i in range(accepted[b]):
            for name in want:
                src = c[name].movedim(-4 if name.endswith("cache") else -3, 0)[b]
                dst = want[name].movedim(-4 if name.endswith("cache") else -3, 0)[b]
                if name.endswith("cache"):
                    dst[..., n + i, :] = src[..., n + path[b][i], :]
                else:
                    dst[..., n + i] = src[..., n + path[b][i]]
    return want


@pytest.mark.parametrize("layers,b,hkv,max_len,t", [(None, 1, 1, 4, 1), (None, 3, 2, 70, 7),
                                                     (3, 4, 3, 200, 64), (2, 9, 8, 130, 16)])
def test_compact_moves_the_accepted_rows(layers, b, hkv, max_len, t):
    r = np.random.RandomState(b + t)
    c = cache(((layers,) if layers else ()) + (b, hkv, max_len), b)
    lens = r.randint(0, max_len - t + 1, b)
    lens[0] = max_len - t  # up to the last row
    accepted = r.randint(0, t + 1, b)
    accepted[-1] = t
    path = np.full((b, t), -1)
    for i in range(b):
        if i % 3 == 0:    # in order, as a walk gives it
            path[i, : accepted[i]] = np.sort(r.permutation(t)[: accepted[i]])
        elif i % 3 == 1:  # any order
            path[i, : accepted[i]] = r.permutation(t)[: accepted[i]]
        else:             # the same row more than once
            path[i, : accepted[i]] = r.randint(0, t, accepted[i])
    want = compacted(c, lens, path, accepted)
    new = K.kv_compact_i8(**c, lens=dev(lens), path=dev(path), accepted=dev(accepted))
    assert new.tolist() == (lens + accepted).tolist()
    for n in want:
        assert torch.equal(c[n], want[n]), n


def test_compact_keeps_bits_that_are_no_numbers():
    c = cache((1, 1, 8), 1)
    c["k_scale"].view(torch.int32)[0, 0, 5] = 0x7fc12345  # a NaN with a payload
    K.kv_compact_i8(**c, lens=dev([2]), path=dev([[0, 3, -1, -1]]), accepted=dev([2]))
    assert int(c["k_scale"].view(torch.int32)[0, 0, 3]) == 0x7fc12345


@pytest.mark.parametrize("lens,path,accepted", [
    ([-1], [[0, 1, 2]], [2]), ([7], [[0, 1, 2]], [3]), ([9], [[0, 1, 2]], [0]),
    ([2], [[0, 3, 1]], [2]), ([2], [[0, -1, 1]], [3]), ([2], [[0, 1, 2]], [4]),
    ([2], [[0, 1, 2]], [-1]), ([6], [[0, 2, 1]], [2]),
    ([2**31 - 1], [[0, 1, 2]], [1]), ([2], [[0, 2**31 - 1, 1]], [2])])
def test_compact_leaves_a_bad_sequence_and_reports_it(lens, path, accepted):
    c = cache((2, 2, 8), 4)
    good_path, good_lens = [0, 2, 1], 3
    want = compacted(c, [0, good_lens], [[], good_path], [0, 3])
    new = K.kv_compact_i8(**c, lens=dev(lens + [good_lens]), path=dev(path + [good_path]),
                          accepted=dev(accepted + [3]))
    assert new.tolist() == [lens[0], 6]
    for n in want:
        assert torch.equal(c[n], want[n]), n
    with pytest.raises(_lib.ReefError, match="0x201"):
        K.check_device_error()


@pytest.mark.parametrize("first", ["k", "v"])
def test_compact_writes_no_row_that_is_in_its_place(first):
    """Codes and scales.  K's and V's scales lie in one array, one a step behind the
    other, so that a scale written back where the one has it would undo the other's move."""
    t, max_len = 4, 16
    c = cache((1, 1, max_len), 5)
    both = torch.rand(max_len + 1, device="cuda")
    k, v = both[:max_len].view(1, 1, max_len), both[1:].view(1, 1, max_len)
    if first == "v":
        k, v = v, k
    want = both.clone()
    want[1], want[2] = both[2], both[3]  # row 1 := row 2; row 0 stays
    rows = c["k_cache"].clone()
    K.kv_compact_i8(c["k_cache"], k, c["v_cache"], v, dev([0]), dev([[0, 2, -1, -1]]), dev([2]))
    assert torch.equal(both, want)
    rows[:, :, 1] = rows[:, :, 2]
    assert torch.equal(c["k_cache"], rows)


def test_compact_past_32_bits():
    """The last layer's rows lie past 2^32 bytes."""
    layers, b, hkv, max_len = 66, 4, 8, 16384
    c = cache((layers, b, hkv, 4), 2)
    big = {n: torch.zeros((layers, b, hkv, max_len) + v.shape[4:], dtype=v.dtype, device="cuda")
           for n, v in c.items()}
    assert big["k_cache"].numel() > 1 << 32
    for n in c:
        big[n][:, :, :, -4:] = c[n]
    want = compacted(c, [0] * b, [[2, 3]] * b, [2] * b)
    K.kv_compact_i8(**big, lens=dev([max_len - 4] * b), path=dev([[2, 3, -1, -1]] * b),
                    accepted=dev([2] * b))
    for n in c:
        assert torch.equal(big[n][:, :, :, -4:], want[n])
        assert not big[n][:, :, :, :-4].any()


# ---- add_rmsnorm_quant -----------------------------------------------------------


def two_calls(x, res, gain, eps):
    rows, width = x.shape
    st = torch.cuda.current_stream().cuda_stream
    h = torch.empty_like(x)
    _lib.call("reef_b200_add_f32", x.numel(), x.data_ptr(), res.data_ptr(), h.data_ptr(), st)
    q = torch.empty((rows, width), dtype=torch.int8, device="cuda")
    s = torch.empty(rows, device="cuda")
    _lib.call("reef_b200_rmsnorm_quant", rows, width, eps, h.data_ptr(), gain.data_ptr(),
              q.data_ptr(), s.data_ptr(), st)
    return h, q, s


@pytest.mark.parametrize("rows,width", [(1, 32), (3, 96), (129, 1024), (2, 4096), (65, 4128),
                                        (7, 8192), (5, 11008), (2, 16384), (1500, 512)])
def test_add_rmsnorm_is_the_two_operators(rows, width):
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    x, res = (torch.randn((rows, width), generator=g, device="cuda") * s for s in (1.0, 3.0))
    gain = torch.rand(width, generator=g, device="cuda") + 0.5
    if rows > 2:
        res[1] = -x[1]  # a row of zeros: scale 1
        x[2] *= 1e-20
        res[2] *= 1e-20
    want = two_calls(x, res, gain, 1e-5)
    for got, w in zip(K.add_rmsnorm_quant(x, res, gain, 1e-5), want):
        assert torch.equal(got, w)
    for alias in ("x", "res"):  # in place
        a, b = x.clone(), res.clone()
        got = K.add_rmsnorm_quant(a, b, gain, 1e-5, h=a if alias == "x" else b)
        assert all(torch.equal(p, w) for p, w in zip(got, want))
        assert torch.equal(b if alias == "x" else a, res if alias == "x" else x)


def test_add_rmsnorm_against_64_bits():
    """h within half a step; a code within one of y / scale in 64 bits, and off
    the nearest only where that lies within 1e-4 of a half (y and scale are each
    off by a few 2^-24, a code is at most 127)."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x, res = (torch.randn((50, 4096), generator=g, device="cuda") for _ in range(2))
    gain = torch.rand(4096, generator=g, device="cuda") + 0.5
    h, q, s = K.add_rmsnorm_quant(x, res, gain, 1e-5)
    hd = x.double() + res.double()
    assert bool(((h.double() - hd).abs() <= 2.0**-24 * hd.abs()).all())
    y = hd * gain.double() / torch.sqrt((hd * hd).mean(1, keepdim=True) + 1e-5)
    scale = y.abs().amax(1) / 127
    assert bool(((s.double() - scale).abs() <= 1e-6 * scale).all())
    assert bool(((q.double() - y / scale[:, None]).abs() <= 0.5 + 1e-4).all())


# ---- a run of them together --------------------------------------------------------


@pytest.mark.parametrize("graph", [False, True])
def test_a_step_that_checks_drafts(graph):
    """Attention over the tree, a choice per node, the walk, the compaction: the
    next step's attention over the compacted cache equals that over a cache
    that held the accepted tokens alone."""
    b, t, hq, hkv, max_len, vocab = 4, 8, 8, 2, 256, 500
    g = torch.Generator(device="cuda").manual_seed(77)
    r = np.random.RandomState(77)
    i8 = lambda *s: torch.randint(-127, 128, s, generator=g, device="cuda", dtype=torch.int8)
    f32 = lambda *s: torch.rand(s, generator=g, device="cuda") * 0.02 + 0.005
    c = dict(k_cache=i8(b, hkv, max_len, 128), k_scale=f32(b, hkv, max_len),
             v_cache=i8(b, hkv, max_len, 128), v_scale=f32(b, hkv, max_len))
    q8, qs = i8(b, t, hq, 128), f32(b, t, hq)
    head = torch.randn((hq * 128, vocab), generator=g, device="cuda") * 3.0
    lens = dev([130, 7, 0, 120])
    parents = np.floor(r.random_sample((b, t)) * np.arange(t)).astype(np.int32)
    parents[:, 0] = -1
    parents = dev(parents)
    u = torch.rand(b * t, generator=g, device="cuda")
    top_p = torch.full((b * t,), 0.8, device="cuda")
    tokens = dev(r.randint(0, vocab, (b, t)))
    was = {n: v.clone() for n, v in c.items()}

    def step():
        att = K.tree_attn_i8(q8, qs, **c, lens=lens, parents=parents)
        logits = att.view(b * t, -1) @ head
        chosen, prob = K.sample_f32(logits, u, top_p=top_p)
        chosen = chosen.view(b, t)
        path, accepted, following = K.tree_accept(tokens, chosen, parents=parents)
        new = K.kv_compact_i8(**c, lens=lens, path=path, accepted=accepted)
        return att, chosen, path, accepted, following, new

    # drafts that the model agrees with: every node's token is what its parent chose
    chosen = step()[1]
    up = parents.long().clamp(min=0)
    tokens.copy_(chosen.gather(1, up))
    for n in c:
        c[n].copy_(was[n])
    if graph:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        for n in c:
            c[n].copy_(was[n])
        gr.replay()
    else:
        out = step()
    att, chosen, path, accepted, following, new = out
    torch.cuda.synchronize()
    for i in range(b):
        p = path[i, : int(accepted[i])].tolist()
        assert p == walk(parents[i].tolist(), tokens[i].tolist(), chosen[i].tolist(), t)[0][: len(p)]
        n, m = int(lens[i]), int(new[i])
        assert m == n + len(p) and int(following[i]) == int(chosen[i, p[-1]])
        alone = {k: torch.cat([v[i:i + 1, :, :n], v[i:i + 1, :, [n + j for j in p]],
                               v[i:i + 1, :, m:]], 2).contiguous() for k, v in was.items()}
        one = dict(q8=q8[i:i + 1, :1].contiguous(), q_scale=qs[i:i + 1, :1].contiguous())
        now = {k: v[i:i + 1].contiguous() for k, v in c.items()}
        # the next root stands in row m of both
        assert torch.equal(K.tree_attn_i8(**one, **now, lens=new[i:i + 1].contiguous()),
                           K.tree_attn_i8(**one, **alone, lens=dev([m])))
    assert int(accepted.max()) > 1
    assert math.isfinite(float(att.sum()))
