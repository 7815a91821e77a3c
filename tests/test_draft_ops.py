"""Refusals of the sampling, drafted-token and residual-norm entry points: they
come back before any CUDA call (no GPU needed)."""
import ctypes as C

import pytest
import torch

from reef_b200 import _lib
from reef_b200 import kernels as K
from reef_b200 import layer as RL

INVALID, ALIGNMENT, TOO_LARGE = 1, 2, 7


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


P, Q = C.c_void_p(4096), C.c_void_p(8192)  # never dereferenced


def test_sample_refusals(L):
    f = L.reef_b200_sample_f32
    assert f(0, 0, *[None] * 9) == 0  # no rows: a no-op
    assert f(1, 0, P, None, None, None, None, P, P, None, None) == INVALID
    for bad in range(3):
        a = [P, P, P]
        a[bad] = None
        assert f(1, 8, a[0], None, None, None, None, a[1], a[2], None, None) == INVALID
    assert f(1, (1 << 20) + 1, P, None, None, None, None, P, P, None, None) == TOO_LARGE
    assert f((1 << 24) + 1, 8, P, None, None, None, None, P, P, None, None) == TOO_LARGE


def test_add_rmsnorm_refusals(L):
    f = L.reef_b200_add_rmsnorm_quant
    assert f(0, 0, 1e-5, *[None] * 7) == 0
    assert f(1, 0, 1e-5, *[P] * 6, None) == INVALID
    assert f(1, 16416, 1e-5, *[P] * 6, None) == INVALID
    assert f(1, 48, 1e-5, *[P] * 6, None) == ALIGNMENT
    for i in range(6):
        a = [P] * 6
        a[i] = None
        assert f(1, 64, 1e-5, *a, None) == INVALID
    for i in range(5):  # x, residual, gain, h: 16 bytes; x_q: 4
        a = [P] * 6
        a[i] = C.c_void_p(4096 + (8 if i < 4 else 2))
        assert f(1, 64, 1e-5, *a, None) == ALIGNMENT


def tree(L, b=1, t=2, hq=4, hkv=2, d=128, n=64, lens=P, ws=P, out=P, q=P, k=P, ks=P, v=P, vs=P,
         nbytes=1 << 40):
    return L.reef_b200_tree_attn_i8(b, t, hq, hkv, d, n, lens, None, None, 1.0, q, P, k, ks, v, vs,
                                    ws, nbytes, out, None)


def test_tree_attn_refusals(L):
    assert tree(L, b=0) == 0 and tree(L, t=0) == 0
    for bad in (dict(hq=0), dict(hkv=0), dict(hq=5), dict(d=64), dict(n=0), dict(hq=8192),
                dict(lens=None), dict(ws=None), dict(out=None), dict(q=None), dict(k=None),
                dict(ks=None), dict(v=None), dict(vs=None)):
        assert tree(L, **bad) == INVALID, bad
    for bad in (dict(t=65), dict(b=2049), dict(b=2048, hq=64, hkv=64), dict(n=(1 << 24) + 4)):
        assert tree(L, **bad) == TOO_LARGE, bad
    off = C.c_void_p(4096 + 4)
    for bad in (dict(n=62), dict(k=off), dict(v=off), dict(ks=off), dict(vs=off), dict(ws=off),
                dict(out=off), dict(q=off)):
        assert tree(L, **bad) == ALIGNMENT, bad
    need = L.reef_b200_tree_attn_workspace_bytes
    for bad in ((0, 1, 1, 1, 4), (2049, 1, 1, 1, 4), (1, 0, 1, 1, 4), (1, 65, 1, 1, 4),
                (1, 1, 0, 1, 4), (1, 1, 3, 2, 4), (1, 1, 1, 0, 4), (1, 1, 1, 1, 0)):
        assert need(*bad) == 0


def test_accept_refusals(L):
    f = L.reef_b200_tree_accept
    assert f(0, 0, *[None] * 8) == 0
    assert f(1, 0, None, None, *[P] * 5, None) == INVALID
    for i in range(5):
        a = [P] * 5
        a[i] = None
        assert f(1, 4, None, None, *a, None) == INVALID
    assert f(1, 65, None, None, *[P] * 5, None) == TOO_LARGE


def compact(L, layers=1, b=1, hkv=2, d=128, n=64, t=4, a=None, new=Q):
    return L.reef_b200_kv_compact_i8(layers, b, hkv, d, n, t, *(a or [P] * 7), new, None)


def test_compact_refusals(L):
    assert compact(L, layers=0) == 0 and compact(L, b=0) == 0
    for bad in (dict(hkv=0), dict(d=64), dict(n=0), dict(t=0), dict(new=None), dict(new=P)):
        assert compact(L, **bad) == INVALID, bad
    for i in range(7):
        a = [P] * 7
        a[i] = None
        assert compact(L, a=a) == INVALID
    for bad in (dict(t=65), dict(layers=65537), dict(n=(1 << 24) + 1),
                dict(layers=65536, b=1 << 20)):
        assert compact(L, **bad) == TOO_LARGE, bad
    for i in (3, 5):
        a = [P] * 7
        a[i] = C.c_void_p(4096 + 8)
        assert compact(L, a=a) == ALIGNMENT


def test_compact_refuses_new_lens_in_what_it_reads(L):
    """The new length of a sequence is written by one CTA while the others read lens,
    path and accepted: no overlap, not even of one element."""
    far = [C.c_void_p(1 << 20), C.c_void_p(2 << 20), C.c_void_p(3 << 20)] + [P] * 4
    base, b, t = 1 << 30, 8, 4
    for i, n in ((0, b), (1, b * t), (2, b)):  # lens, path, accepted at `base`
        a = list(far)
        a[i] = C.c_void_p(base)
        for at in (base, base + 4, base + 4 * (n - 1), base - 4 * (b - 1)):
            assert compact(L, b=b, t=t, a=a, new=C.c_void_p(at)) == INVALID, (i, at)
        for at in (base + 4 * n, base - 4 * b):  # next to it: refused for what comes after
            off = list(a)
            off[3] = C.c_void_p(4096 + 8)
            assert compact(L, b=b, t=t, a=off, new=C.c_void_p(at)) == ALIGNMENT, (i, at)


def test_wrappers_refuse_tensors_before_any_call():
    f, i = torch.zeros, torch.int32
    with pytest.raises(ValueError, match="CUDA"):
        K.sample_f32(f(2, 5), f(2))
    with pytest.raises(TypeError, match="logits"):
        K.sample_f32(f(2, 5, dtype=torch.bfloat16), f(2))
    with pytest.raises(ValueError, match="CUDA"):
        K.add_rmsnorm_quant(f(2, 32), f(2, 32), f(32))
    with pytest.raises(TypeError, match="lens"):
        K.kv_compact_i8(f(1, 1, 4, 128, dtype=torch.int8), f(1, 1, 4),
                        f(1, 1, 4, 128, dtype=torch.int8), f(1, 1, 4), f(1), f(1, 2, dtype=i),
                        f(1, dtype=i))
    with pytest.raises(ValueError, match="CUDA"):
        K.tree_accept(f(1, 2, dtype=i), f(1, 2, dtype=i))
    with pytest.raises(TypeError, match="lens"):
        K.tree_attn_i8(f(1, 2, 4, 128, dtype=torch.int8), f(1, 2, 4),
                       f(1, 2, 8, 128, dtype=torch.int8), f(1, 2, 8),
                       f(1, 2, 8, 128, dtype=torch.int8), f(1, 2, 8), f(1))


def test_verify_refusals(L):
    """The layer description is checked like the decode step's; sizes by arithmetic."""
    need = L.reef_b200_llama_verify_workspace_bytes
    d = _lib.LlamaLayerDesc(batch=2, seq=8, hidden=512, heads_q=4, heads_kv=2, head_dim=128,
                            ffn=1024, rms_eps=1e-5, rope_base=1e4)
    ref = C.byref(d)
    assert need(None, 2, 64) == 0 and need(ref, 0, 64) == 0 and need(ref, 65, 64) == 0
    assert need(ref, 2, 62) == 0
    f = L.reef_b200_llama_verify_forward
    args = [P, P, P, None, None, P, P, P, P]
    assert f(None, 2, *args, 64, P, 1 << 40, None) == INVALID
    assert f(ref, 0, *args, 64, P, 1 << 40, None) == INVALID
    assert f(ref, 65, *args, 64, P, 1 << 40, None) == INVALID
    for i in (0, 1, 2, 5, 6, 7, 8):
        a = list(args)
        a[i] = None
        assert f(ref, 2, *a, 64, P, 1 << 40, None) == INVALID
    assert f(ref, 2, *args, 64, None, 1 << 40, None) == INVALID
    assert f(ref, 2, *args, 62, P, 1 << 40, None) == ALIGNMENT
    assert f(ref, 2, *args, 64, C.c_void_p(4096 + 16), 1 << 40, None) == ALIGNMENT
    for i in (5, 6, 7, 8):
        a = list(args)
        a[i] = C.c_void_p(4096 + 4)
        assert f(ref, 2, *a, 64, P, 1 << 40, None) == ALIGNMENT


def host_layer(batch=2, heads_kv=2, hidden=64, **kw):
    """A layer's wrapper whose tensors are on the host: its operands are refused as on
    the GPU, and one with nothing else wrong for lying there."""
    layer = object.__new__(RL.LlamaLayer)
    layer.__dict__.update(dict(batch=batch, heads_kv=heads_kv, _tiles={}, world=1,
                               tp_mode=RL.TP_ALLREDUCE, w_qkv=torch.zeros(1),
                               attn_norm=torch.zeros(hidden)) | kw)
    return layer


def host_cache(batch=2, heads_kv=2, rows=64, max_len=None):
    shape = (batch, heads_kv, rows)
    c = {n: torch.zeros(shape + (128,), dtype=torch.int8) for n in ("k", "v")}
    return c | {"ks": torch.zeros(shape), "vs": torch.zeros(shape),
                "max_len": rows if max_len is None else max_len}


def test_verify_refuses_a_cache_that_is_not_the_layers(monkeypatch):
    layer, x, lens = host_layer(), torch.zeros((4, 64)), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        layer.verify(x, lens, host_cache())
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)  # (shapes are what is looked at below)
    for bad in (dict(batch=1), dict(batch=3), dict(heads_kv=1), dict(max_len=128), dict(max_len=32)):
        with pytest.raises(ValueError, match="cache's k must be"):
            layer.verify(x, lens, host_cache(**bad))
    for name in ("k", "ks", "v", "vs"):
        c = host_cache()
        for bad in (c[name][:1], c[name][:, :, :32].contiguous(), c[name][None]):
            with pytest.raises(ValueError, match=f"cache's {name} must be"):
                layer.verify(x, lens, c | {name: bad})
        with pytest.raises(TypeError, match=f"cache's {name} must be"):
            layer.verify(x, lens, c | {name: c[name].half()})
    with pytest.raises(ValueError, match="contiguous"):
        layer.verify(x, lens, host_cache() | {"vs": host_cache(rows=128)["vs"][:, :, :64]})


def test_verify_refuses_a_shard_of_the_all_gather_plan():
    """Also without a communicator, where the library cannot know."""
    x, lens = torch.zeros((4, 64)), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="TP_ALLREDUCE"):
        host_layer(world=2, tp_mode=RL.TP_ALLGATHER).verify(x, lens, host_cache())
    with pytest.raises(ValueError, match="TP_ALLREDUCE"):
        host_layer(world=2, tp_mode=RL.TP_ALLGATHER).decode(x, lens, host_cache())
    for fine in (dict(world=2), dict(tp_mode=RL.TP_ALLGATHER)):
        with pytest.raises(ValueError, match="CUDA"):
            host_layer(**fine).verify(x, lens, host_cache())


def test_verify_prepares_on_the_layers_device(monkeypatch):
    """Tiles and workspace of a layer whose device is not the current one: every CUDA call
    of the preparation is made with it current, and once."""
    current, made = [], []

    class Device:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            current.append(self.dev)

        def __exit__(self, *_):
            current.pop()

    class Stream:
        def synchronize(self):
            made.append(("synchronize", list(current)))

    class Lib:
        def reef_b200_llama_verify_workspace_bytes(self, *_):
            made.append(("workspace", list(current)))
            return 256

    layer = host_layer(desc=_lib.LlamaLayerDesc(), _tiles=None)

    def tiles():
        made.append(("tiles", list(current)))
        layer._tiles = {}

    def capturing():
        made.append(("capturing", list(current)))
        return False

    layer._decode_tiles = tiles
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *_: Stream())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", capturing)
    monkeypatch.setattr(_lib, "lib", Lib)
    calls = []
    monkeypatch.setattr(K, "_call_on", lambda dev, name, *a: calls.append((dev, name)))
    dev = layer.w_qkv.device
    x, lens = torch.zeros((4, 64)), torch.zeros(2, dtype=torch.int32)
    for _ in range(2):
        layer.verify(x, lens, host_cache())
    assert made == [(n, [dev]) for n in ("capturing", "tiles", "synchronize", "workspace")]
    layer.verify(torch.zeros((6, 64)), lens, host_cache())
    assert made[4:] == [("workspace", [dev])]
    assert calls == [(dev, "reef_b200_llama_verify_forward")] * 3
