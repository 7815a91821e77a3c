"""The Llama layer on drafted tokens (reef_b200_llama_verify_forward) against its
own decode step, and sampled GPT-Neo generation.

A drafted token's key and value depend on its own input and its depth alone, so
their cache rows must be the decode step's bit for bit.  The outputs differ by the
attention kernels (the decode head rounds P to f16, this one does not): the
tolerances are those of the decode step against the prefill layer, whose
attentions differ in the same way.
"""
import numpy as np
import pytest
import torch

from reef_b200 import kernels as K
from reef_b200 import layer as RL
from tests import blob_fixture as BF
from tests.test_sample_gpu import plain

pytestmark = pytest.mark.gpu
SHAPE = RL.LlamaShape(hidden=512, heads_q=8, heads_kv=2, ffn=1024)


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_lib):
    yield
    K.check_device_error()


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def decoded(layer, cache, x, lens):
    """x [batch][steps][hidden] one token at a time from `lens`; y alike."""
    ys = []
    for t in range(x.shape[1]):
        ys.append(layer.decode(x[:, t].contiguous(), i32([n + t for n in lens]), cache))
    return torch.stack(ys, 1)


def close(got, want):
    err = (got - want).abs()
    assert float(err.max()) < 5e-2 and float(err.mean()) < 5e-3, (float(err.max()), float(err.mean()))


def history(layer, lens, max_len, seed):
    """A cache with `lens` committed rows, filled by the decode step."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = layer.alloc_cache(max_len)
    for t in range(max(lens)):
        x = torch.randn((layer.batch, 512), generator=g, device="cuda")
        # rows past a sequence's length are overwritten by what follows
        layer.decode(x, i32([min(t, n) for n in lens]), cache)
    return cache


def copy_of(cache):
    return {k: v.clone() if torch.is_tensor(v) else v for k, v in cache.items()}


@pytest.mark.parametrize("drafts,lens", [(1, [30, 7, 0]), (2, [5, 40, 38]), (9, [0, 31, 3]),
                                         (20, [12, 1, 40])])
def test_a_chain_is_that_many_decode_steps(drafts, lens):
    max_len = 64
    layer = RL.LlamaLayer(SHAPE, len(lens), 8, seed=5)
    cache = history(layer, lens, max_len, 1)
    x = torch.randn((len(lens), drafts, 512), device="cuda",
                    generator=torch.Generator(device="cuda").manual_seed(drafts))
    other = copy_of(cache)
    want = decoded(layer, other, x, lens)
    got = layer.verify(x.view(-1, 512), i32(lens), cache).view(len(lens), drafts, 512)
    for b, n in enumerate(lens):
        for c in ("k", "ks", "v", "vs"):
            assert torch.equal(cache[c][b, :, : n + drafts], other[c][b, :, : n + drafts]), (b, c)
    close(got, want)


def test_a_tree_is_its_paths():
    """Each root-to-leaf path of a tree against the decode steps of its inputs; the
    accepted path's cache, compacted, against theirs."""
    lens, t, max_len = [21, 4], 7, 64
    parents = [[-1, 0, 0, 1, 2, 4, 0], [-1, 0, 1, 1, 3, 2, 5]]
    layer = RL.LlamaLayer(SHAPE, 2, 8, seed=6)
    cache = history(layer, lens, max_len, 2)
    x = torch.randn((2, t, 512), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    start = copy_of(cache)
    got = layer.verify(x.view(-1, 512), i32(lens), cache, parents=i32(parents)).view(2, t, 512)
    paths = [[0, 2, 4, 5], [0, 1, 3, 4]]
    steps = torch.stack([x[b, paths[b]] for b in range(2)])
    other = copy_of(start)
    want = decoded(layer, other, steps, lens)
    close(torch.stack([got[b, paths[b]] for b in range(2)]), want)
    # the walk takes these paths when the model chooses their tokens
    tokens = i32([[10 + i for i in range(t)] for _ in range(2)])
    chosen = torch.full((2, t), 999, dtype=torch.int32, device="cuda")
    for b in range(2):
        for a, n in zip(paths[b], paths[b][1:]):
            chosen[b, a] = 10 + n
    path, accepted, following = K.tree_accept(tokens, chosen, parents=i32(parents))
    assert [path[b, :4].tolist() for b in range(2)] == paths and following.tolist() == [999, 999]
    new = K.kv_compact_i8(cache["k"], cache["ks"], cache["v"], cache["vs"], i32(lens), path, accepted)
    assert new.tolist() == [n + 4 for n in lens]
    for b, n in enumerate(lens):
        for c in ("k", "ks", "v", "vs"):
            assert torch.equal(cache[c][b, :, : n + 4], other[c][b, :, : n + 4]), (b, c)


def test_fewer_drafts_and_sequences_that_do_not_fit():
    lens, max_len = [10, 62, 3], 64
    layer = RL.LlamaLayer(SHAPE, 3, 8, seed=7)
    cache = history(layer, [10, 40, 3], max_len, 4)
    x = torch.randn((3, 4, 512), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    was = copy_of(cache)
    got = layer.verify(x.view(-1, 512), i32(lens), cache, draft_lens=i32([4, 3, 0])).view(3, 4, 512)
    for c in ("k", "ks", "v", "vs"):
        assert torch.equal(cache[c][1:], was[c][1:])  # 62 + 3 > 64; no drafts
    with pytest.raises(Exception, match="0x201"):
        K.check_device_error()
    one = RL.LlamaLayer(SHAPE, 1, 8, seed=7)
    close(got[:1], decoded(one, {k: v[:1].contiguous() if torch.is_tensor(v) else v
                                 for k, v in was.items()}, x[:1], [10]))


def test_captured_and_replayed():
    lens = i32([9, 33])
    layer = RL.LlamaLayer(SHAPE, 2, 8, seed=8)
    cache = history(layer, [9, 33], 64, 6)
    x = torch.randn((10, 512), device="cuda")
    want = layer.verify(x, lens, cache).clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer.verify(x, lens, cache)
    y.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)


def test_a_capture_as_the_first_call_and_other_drafts_between_replays():
    """Nothing that a captured call uses goes away or is still to be made."""
    lens = i32([9, 33])
    layer, other = (RL.LlamaLayer(SHAPE, 2, 8, seed=8) for _ in range(2))
    cache = history(other, [9, 33], 64, 6)
    gen = torch.Generator(device="cuda").manual_seed(9)
    x, x2 = (torch.randn((n, 512), device="cuda", generator=gen) for n in (10, 6))
    want, want2 = (other.verify(v, lens, cache).clone() for v in (x, x2))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer.verify(x, lens, cache)
    assert torch.equal(layer.verify(x2, lens, cache), want2)
    assert torch.equal(layer.verify(x2, lens, cache | {"max_len": 64}), want2)
    junk = [torch.full((1 << 20,), 0xff, dtype=torch.uint8, device="cuda") for _ in range(64)]
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want) and all(int(j[0]) == 0xff for j in junk)


def test_the_layers_caches_in_one_stack():
    """Each layer's cache a part of one tensor, which one call compacts."""
    lens, t, max_len, n = [21, 4], 5, 64, 2
    layers = [RL.LlamaLayer(SHAPE, 2, 8, seed=20 + i) for i in range(n)]
    apart = [history(layer, lens, max_len, 30 + i) for i, layer in enumerate(layers)]
    stack = {c: torch.stack([a[c] for a in apart]) for c in ("k", "ks", "v", "vs")}
    parts = [{c: v[i] for c, v in stack.items()} | {"max_len": max_len} for i in range(n)]
    x = torch.randn((2 * t, 512), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    parents = i32([[-1, 0, 0, 2, 1], [-1, 0, 1, 1, 3]])
    path, accepted = i32([[0, 2, 3, -1, -1], [0, 1, 3, 4, -1]]), i32([3, 4])
    a = b = x
    for layer, one, part in zip(layers, apart, parts):
        a, b = layer.verify(a, i32(lens), one, parents), layer.verify(b, i32(lens), part, parents)
    assert torch.equal(a, b)
    new = K.kv_compact_i8(*stack.values(), i32(lens), path, accepted)
    for one in apart:
        K.kv_compact_i8(one["k"], one["ks"], one["v"], one["vs"], i32(lens), path, accepted)
    assert new.tolist() == [24, 8]
    for i, one in enumerate(apart):
        for c in stack:
            assert torch.equal(stack[c][i], one[c]), (i, c)


def test_refusals():
    layer = RL.LlamaLayer(SHAPE, 2, 8, seed=8)
    cache = layer.alloc_cache(64)
    x = torch.zeros((4, 512), device="cuda")
    with pytest.raises(ValueError, match="same number"):
        layer.verify(x[:3], i32([1, 1]), cache)
    with pytest.raises(ValueError, match="drafted tokens"):
        layer.verify(torch.zeros((130, 512), device="cuda"), i32([1, 1]), cache)  # 65 drafts
    with pytest.raises(ValueError, match="lens"):
        layer.verify(x, i32([1, 1, 1]), cache)
    with pytest.raises(ValueError, match="x must be"):
        layer.verify(torch.zeros((4, 256), device="cuda"), i32([1, 1]), cache)
    with pytest.raises(TypeError, match="x must be"):
        layer.verify(x.half(), i32([1, 1]), cache)
    with pytest.raises(ValueError, match="out must be"):
        layer.verify(x, i32([1, 1]), cache, out=x[:2])
    with pytest.raises(ValueError, match="drafted tokens"):
        layer.verify(x, i32([1, 1]), layer.alloc_cache(62))


@pytest.mark.parametrize("precision", ["w8a8", "fp32"])
@pytest.mark.parametrize("how", [dict(), dict(temperature=0.7, top_k=8),
                                 dict(temperature=1.4, top_p=0.7, min_p=0.02)])
def test_sampled_generation(precision, how):
    """Every token is the draw from its own logits; u fixed, the tokens are."""
    blob, prompt, tokens, _ = BF.golden_model(precision)
    u = np.random.RandomState(3).rand(tokens.size).astype(np.float32)
    new = lambda: RL.GptNeoModel(blob, max_tokens=prompt.size + tokens.size)  # noqa: E731
    got, logits = new().generate(prompt, tokens.size, u=u, **how)
    for i in range(tokens.size):
        assert int(got[i]) == plain(logits[i].numpy(), u[i], np.float32(how.get("temperature", 1.0)),
                                    how.get("top_k", 0), np.float32(how.get("top_p", 1.0)),
                                    np.float32(how.get("min_p", 0.0)))[0]
    assert torch.equal(new().generate(prompt, tokens.size, u=u, **how)[0], got)
    greedy = new().generate(prompt, tokens.size, u=u, temperature=0.0)[0]
    assert greedy.tolist() == tokens.tolist()
    with pytest.raises(ValueError, match="u must"):
        new().generate(prompt, 3, u=u)
