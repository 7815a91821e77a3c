"""Host mirror of reef's operator API (namespace reef_kernels,
inference-engine/coral/include/reef_kernels/kernels.hpp) over CUDA tensors.

Same names and argument meaning as the Coral kernels, batched over rows, on
device memory.  Every function calls into libreef_b200.so through the C ABI
(include/reef_b200.h); none has a CPU path.  torch is used only to hold device
memory and the current stream.  Weights are K-major [out][kpad(in)] int8 (see
:func:`pack_weight_i8` for Coral's transposed [in][out] layout).
"""
from __future__ import annotations

import functools

import torch

from . import _lib


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: torch.Tensor | None) -> int | None:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("reef_b200 entry points take CUDA tensors")
    if not t.is_contiguous():
        raise ValueError("reef_b200 entry points take contiguous tensors")
    return t.data_ptr()


def _take(t: torch.Tensor | None, name: str, dtype, shape, device, other=None) -> int | None:
    """The address of an argument that must be a contiguous CUDA tensor of
    this type (or the other) and shape on this device (None passes as NULL)."""
    if t is None:
        return None
    if t.dtype is dtype and t.shape == shape and t.device == device and t.is_cuda and \
            t.is_contiguous():
        return t.data_ptr()
    if t.dtype is not dtype and t.dtype is not other:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    return _ptr(t)


def _call_on(device: torch.device, name: str, *args) -> None:
    """An entry point on `device` and its current stream (the last argument),
    whichever device is current."""
    # (the raw handle: torch.cuda.current_stream() makes a Stream object, 3 us of
    # a call that takes 4)
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if device.index == torch.cuda.current_device():
        _lib.call(name, *args, stream)
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, stream)


def kpad(n: int) -> int:
    return (n + 15) // 16 * 16


def check_device_error() -> None:
    """Raise when a bounded device wait gave up since the last check."""
    import ctypes as C
    code = C.c_int(0)
    _lib.call("reef_b200_device_error", C.addressof(code))
    if code.value != 0:
        raise _lib.ReefError(f"device wait (code {code.value:#x})", 6)


# ---- quantization --------------------------------------------------------------

def quantize_rows(x: torch.Tensor):
    """quantize_rows (quant.hpp:112-133): returns (x_q [rows][kpad], x_scale)."""
    rows, k = x.shape
    x_q = torch.empty((rows, kpad(k)), dtype=torch.int8, device=x.device)
    xs = torch.empty((rows,), dtype=torch.float32, device=x.device)
    _lib.call("reef_b200_quantize_rows", rows, k, _ptr(x), _ptr(x_q), _ptr(xs), _stream())
    return x_q, xs


def matvec_rows_f32(w: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """reef_kernels::matvec_rows_f32 (kernels.hpp:48-52): y[c] = sum over k, in
    order, of x[k] * w[c][k] (GPT-Neo's lm_head), bit-identical to the engine."""
    out, k = w.shape
    y = torch.empty((out,), dtype=torch.float32, device=w.device)
    _lib.call("reef_b200_matvec_rows_f32", out, k, _ptr(w), _ptr(x), _ptr(y), _stream())
    return y


def argmax_f32(x: torch.Tensor) -> torch.Tensor:
    """reef_kernels::argmax_f32 (kernels.hpp:89-90): index of the first largest
    value, as one device int32 element holding the uint32 index."""
    idx = torch.empty((1,), dtype=torch.int32, device=x.device)
    _lib.call("reef_b200_argmax_f32", x.numel(), _ptr(x), _ptr(idx), _stream())
    return idx


def sample_f32(logits: torch.Tensor, u: torch.Tensor, temperature: torch.Tensor | None = None,
               top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
               min_p: torch.Tensor | None = None, index: torch.Tensor | None = None):
    """One token per row of logits [rows][n] fp32 from the uniform numbers u
    [rows]: softmax at `temperature` (not above 0: greedy), cut by top_k, then
    top_p, then min_p, drawn in index order.  The parameters are per row
    (fp32 [rows]; top_k int32) or None (off); index may be given.  Returns (index [rows] int32
    holding uint32 ids, prob [rows] fp32 under the cut distribution); a row
    without a logit above -inf gives -1 (REEF_B200_NO_TOKEN) and 0."""
    rows, n = logits.shape
    dev = logits.device
    f32, one = torch.float32, (rows,)
    args = (_take(logits, "logits", f32, (rows, n), dev),
            _take(temperature, "temperature", f32, one, dev),
            _take(top_k, "top_k", torch.int32, one, dev), _take(top_p, "top_p", f32, one, dev),
            _take(min_p, "min_p", f32, one, dev), _take(u, "u", f32, one, dev))
    prob = torch.empty_like(u)
    if index is None:
        index = torch.empty_like(u, dtype=torch.int32)
    _call_on(dev, "reef_b200_sample_f32", rows, n, *args,
             _take(index, "index", torch.int32, one, dev, torch.uint32), prob.data_ptr())
    return index, prob


def pack_weight_i8(wt: torch.Tensor) -> torch.Tensor:
    """Coral weight [in][out] -> K-major [out][kpad(in)]."""
    k, n = wt.shape
    w = torch.empty((n, kpad(k)), dtype=torch.int8, device=wt.device)
    _lib.call("reef_b200_pack_weight_i8", k, n, _ptr(wt), _ptr(w), _stream())
    return w


def pad_rows_i8(x: torch.Tensor) -> torch.Tensor:
    rows, k = x.shape
    if k == kpad(k):
        return x
    y = torch.empty((rows, kpad(k)), dtype=torch.int8, device=x.device)
    _lib.call("reef_b200_pad_rows_i8", rows, k, _ptr(x), _ptr(y), _stream())
    return y


# ---- linear layers -------------------------------------------------------------

def linear_w8a8(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                bias: torch.Tensor | None = None, in_features: int | None = None):
    """reef_kernels::linear_w8a8 / linear_w8a8_bias (kernels.hpp:38-46)."""
    rows, k = x.shape
    n = w.shape[0]
    x_q = torch.empty((rows, kpad(k)), dtype=torch.int8, device=x.device)
    xs = torch.empty((rows,), dtype=torch.float32, device=x.device)
    y = torch.empty((rows, n), dtype=torch.float32, device=x.device)
    if bias is None:
        _lib.call("reef_b200_linear_w8a8", rows, k, n, _ptr(x), _ptr(w), _ptr(w_scale),
                  _ptr(x_q), _ptr(xs), _ptr(y), _stream())
    else:
        _lib.call("reef_b200_linear_w8a8_bias", rows, k, n, _ptr(x), _ptr(w),
                  _ptr(w_scale), _ptr(bias), _ptr(x_q), _ptr(xs), _ptr(y), _stream())
    return y


def gemm_w8a8(x_q, x_scale, w, w_scale, bias=None, in_features: int | None = None):
    rows = x_q.shape[0]
    k = in_features if in_features is not None else x_q.shape[1]
    n = w.shape[0]
    y = torch.empty((rows, n), dtype=torch.float32, device=x_q.device)
    _lib.call("reef_b200_gemm_w8a8", rows, k, n, _ptr(x_q), _ptr(x_scale), _ptr(w),
              _ptr(w_scale), _ptr(bias), _ptr(y), _stream())
    return y


def linear_w8a8_swiglu(x_q, x_scale, w_gu, w_scale, in_features: int | None = None):
    """Gate/up projection with SwiGLU in the GEMM epilogue: returns
    (h [rows][ffn] = silu(gate) * up, row_max [rows] = max |h|)."""
    rows = x_q.shape[0]
    k = in_features if in_features is not None else x_q.shape[1]
    ffn = w_gu.shape[0] // 2
    h = torch.empty((rows, ffn), dtype=torch.float32, device=x_q.device)
    row_max = torch.empty(rows, dtype=torch.float32, device=x_q.device)
    _lib.call("reef_b200_linear_w8a8_swiglu", rows, k, ffn, _ptr(x_q), _ptr(x_scale), _ptr(w_gu),
              _ptr(w_scale), _ptr(h), _ptr(row_max), _stream())
    return h, row_max


def linear_int8(x: torch.Tensor, w: torch.Tensor, shift: int,
                bias: torch.Tensor | None = None, in_features: int | None = None):
    """reef_kernels::linear_int8 / linear_bias_int8 (kernels.hpp:101-108).
    x is [rows][kpad(in)] (see :func:`pad_rows_i8`)."""
    rows = x.shape[0]
    k = in_features if in_features is not None else x.shape[1]
    n = w.shape[0]
    y = torch.empty((rows, n), dtype=torch.int8, device=x.device)
    if bias is None:
        _lib.call("reef_b200_linear_int8", rows, k, n, _ptr(x), _ptr(w), shift, _ptr(y),
                  _stream())
    else:
        _lib.call("reef_b200_linear_bias_int8", rows, k, n, _ptr(x), _ptr(w), _ptr(bias),
                  shift, _ptr(y), _stream())
    return y


def gemm_i8_i32(a: torch.Tensor, b: torch.Tensor, k: int | None = None) -> torch.Tensor:
    """matmul<int8,int32>(a, b^T); a [m][kpad], b [n][kpad]."""
    m = a.shape[0]
    n = b.shape[0]
    k = k if k is not None else a.shape[1]
    c = torch.empty((m, n), dtype=torch.int32, device=a.device)
    _lib.call("reef_b200_gemm_i8_i32", m, n, k, _ptr(a), _ptr(b), _ptr(c), _stream())
    return c


# ---- integer softmax and attention heads ---------------------------------------

def exp_table_device(table) -> torch.Tensor:
    """A 256-entry exp_table (int8.hpp:156-164, uint16 values) on the device.
    The bits are held in an int16 tensor; the kernels read them as uint16."""
    import numpy as np
    bits16 = np.ascontiguousarray(np.asarray(table, dtype=np.uint16)).view(np.int16)
    return torch.from_numpy(bits16.copy()).cuda()


def softmax_int8(scores: torch.Tensor, shift: int, table: torch.Tensor) -> torch.Tensor:
    """reef_kernels::softmax_int8 (kernels.hpp:114-117), every row of scores."""
    rows, n = scores.shape
    probs = torch.empty((rows, n), dtype=torch.uint8, device=scores.device)
    _lib.call("reef_b200_softmax_int8", rows, n, _ptr(scores), shift, _ptr(table),
              _ptr(probs), _stream())
    return probs


def attention_head_int8(q, k, v, query_start: int, window: int, score_shift: int,
                        table: torch.Tensor, out_shift: int = 8) -> torch.Tensor:
    """reef_kernels::attention_head_int8 (kernels.hpp:122-129), one head."""
    ql, d = q.shape
    kl = k.shape[0]
    out = torch.empty((ql, d), dtype=torch.int8, device=q.device)
    _lib.call("reef_b200_attention_head_int8", ql, kl, d, query_start, window, _ptr(q), d,
              _ptr(k), _ptr(v), score_shift, _ptr(table), out_shift, None, None, _ptr(out),
              d, _stream())
    return out


def attention_head_f32(q, k, v, query_start: int, window: int) -> torch.Tensor:
    """reef_kernels::attention_head_f32 (kernels.hpp:75-79), one head."""
    ql, d = q.shape
    kl = k.shape[0]
    out = torch.empty((ql, d), dtype=torch.float32, device=q.device)
    _lib.call("reef_b200_attention_head_f32", ql, kl, d, query_start, window, _ptr(q), d,
              _ptr(k), _ptr(v), None, _ptr(out), d, _stream())
    return out


def attention_heads_f32(q, k, v, heads: int, query_start: int = 0, window: int = 0):
    """Attention::context over all heads of [len][d_model] q/k/v."""
    ql, dm = q.shape
    kl = k.shape[0]
    hd = dm // heads
    out = torch.empty((ql, dm), dtype=torch.float32, device=q.device)
    _lib.call("reef_b200_attention_heads_f32", heads, ql, kl, hd, query_start, window,
              _ptr(q), dm, hd, _ptr(k), _ptr(v), dm, hd, _ptr(out), dm, hd, _stream())
    return out


def gemm_w8a8_skinny(x_q, x_scale, w, w_scale, bias=None, in_features: int | None = None):
    """The W8A8 GEMM for rows <= 128 (decode), swap-AB + split-K."""
    rows = x_q.shape[0]
    k = in_features if in_features is not None else x_q.shape[1]
    n = w.shape[0]
    nbytes = _lib.lib().reef_b200_gemm_skinny_workspace_bytes(rows, k, n)
    ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=x_q.device)
    y = torch.empty((rows, n), dtype=torch.float32, device=x_q.device)
    _lib.call("reef_b200_gemm_w8a8_skinny", rows, k, n, _ptr(x_q), _ptr(x_scale), _ptr(w),
              _ptr(w_scale), _ptr(bias), _ptr(ws), ws.numel(), _ptr(y), _stream())
    return y


def add_rmsnorm_quant(x: torch.Tensor, residual: torch.Tensor, gain: torch.Tensor,
                      eps: float = 1e-5, h: torch.Tensor | None = None):
    """h = x + residual, then the Llama pre-norm of h in int8: returns (h
    [rows][width] fp32, x_q [rows][width] int8, x_scale [rows]); h may be given,
    x or residual among them.  The bits of add_f32 and rmsnorm_quant."""
    rows, width = x.shape
    dev, f32 = x.device, torch.float32
    h = torch.empty_like(x) if h is None else h
    args = (_take(x, "x", f32, (rows, width), dev),
            _take(residual, "residual", f32, (rows, width), dev),
            _take(gain, "gain", f32, (width,), dev), _take(h, "h", f32, (rows, width), dev))
    x_q = torch.empty_like(x, dtype=torch.int8)
    xs = x.new_empty(rows)
    _call_on(dev, "reef_b200_add_rmsnorm_quant", rows, width, eps, *args, x_q.data_ptr(),
             xs.data_ptr())
    return h, x_q, xs


# ---- drafted tokens over the int8 KV cache ---------------------------------------


@functools.lru_cache(maxsize=256)
def _tree_attn_workspace(b: int, t: int, hq: int, hkv: int, max_len: int, device: int) -> int:
    with torch.cuda.device(device):
        return max(16, _lib.lib().reef_b200_tree_attn_workspace_bytes(b, t, hq, hkv, max_len))


def tree_attn_i8(q8: torch.Tensor, q_scale: torch.Tensor, k_cache: torch.Tensor,
                 k_scale: torch.Tensor, v_cache: torch.Tensor, v_scale: torch.Tensor,
                 lens: torch.Tensor, parents: torch.Tensor | None = None,
                 draft_lens: torch.Tensor | None = None, sm_scale: float | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of drafted tokens over the int8 KV cache.  q8 [batch][drafts]
    [heads_q][128] int8 + q_scale; caches [batch][heads_kv][max_len][128] int8
    + scales [batch][heads_kv][max_len]; lens [batch] int32 committed rows, the
    drafted tokens' own rows right behind them.  Token t of a sequence sees the
    committed rows, itself and its ancestors under parents [batch][drafts] (None:
    a chain).  Returns out [batch][drafts][heads_q][128] fp32; rows past
    draft_lens are left as they are (zeros in an out made here)."""
    b, t, hq, d = q8.shape
    _, hkv, max_len, _ = k_cache.shape
    dev, f32, i8, i32 = q8.device, torch.float32, torch.int8, torch.int32
    if out is None:
        make = q_scale.new_empty if draft_lens is None else q_scale.new_zeros
        out = make((b, t, hq, d))
    cache, rows = (b, hkv, max_len, d), (b, hkv, max_len)
    before = (_take(lens, "lens", i32, (b,), dev),
              _take(draft_lens, "draft_lens", i32, (b,), dev),
              _take(parents, "parents", i32, (b, t), dev))
    after = (_take(q8, "q8", i8, (b, t, hq, d), dev),
             _take(q_scale, "q_scale", f32, (b, t, hq), dev),
             _take(k_cache, "k_cache", i8, cache, dev), _take(k_scale, "k_scale", f32, rows, dev),
             _take(v_cache, "v_cache", i8, cache, dev), _take(v_scale, "v_scale", f32, rows, dev))
    o = _take(out, "out", f32, (b, t, hq, d), dev)
    ws = q8.new_empty(_tree_attn_workspace(b, t, hq, hkv, max_len, dev.index))
    _call_on(dev, "reef_b200_tree_attn_i8", b, t, hq, hkv, d, max_len, *before,
             d ** -0.5 if sm_scale is None else sm_scale, *after, ws.data_ptr(), ws.numel(), o)
    return out


def tree_accept(tokens: torch.Tensor, chosen: torch.Tensor, parents: torch.Tensor | None = None,
                draft_lens: torch.Tensor | None = None):
    """The path of each tree that the model's own choices follow: tokens /
    chosen [batch][drafts] (the drafted ids; the id chosen after each node), node
    0 the root.  Returns (path [batch][drafts] int32, -1 behind it, accepted
    [batch] int32, next [batch], the id that follows the path, in chosen's
    type)."""
    b, t = tokens.shape
    dev, i32 = tokens.device, torch.int32
    args = (_take(draft_lens, "draft_lens", i32, (b,), dev),
            _take(parents, "parents", i32, (b, t), dev),
            _take(tokens, "tokens", i32, (b, t), dev, torch.uint32),
            _take(chosen, "chosen", i32, (b, t), dev, torch.uint32))
    path = torch.empty_like(tokens, dtype=i32)
    accepted = path.new_empty(b)
    following = chosen.new_empty(b)
    _call_on(dev, "reef_b200_tree_accept", b, t, *args, path.data_ptr(), accepted.data_ptr(),
             following.data_ptr())
    return path, accepted, following


def kv_compact_i8(k_cache: torch.Tensor, k_scale: torch.Tensor, v_cache: torch.Tensor,
                  v_scale: torch.Tensor, lens: torch.Tensor, path: torch.Tensor,
                  accepted: torch.Tensor) -> torch.Tensor:
    """Moves the accepted drafted rows (tree_accept's path) right behind the
    committed ones, in place: row lens + i becomes row lens + path[i].  Caches
    [batch][heads_kv][max_len][128], or [layers][batch]... for every layer's at
    once.  Returns the new lens (lens + accepted)."""
    n = 1 if k_cache.dim() == 4 else k_cache.shape[0]
    b, hkv, max_len, d = k_cache.shape[-4:]
    t = path.shape[1]
    dev, f32, i8, i32 = k_cache.device, torch.float32, torch.int8, torch.int32
    cache = (b, hkv, max_len, d) if k_cache.dim() == 4 else (n, b, hkv, max_len, d)
    args = (_take(lens, "lens", i32, (b,), dev), _take(path, "path", i32, (b, t), dev),
            _take(accepted, "accepted", i32, (b,), dev), _take(k_cache, "k_cache", i8, cache, dev),
            _take(k_scale, "k_scale", f32, cache[:-1], dev),
            _take(v_cache, "v_cache", i8, cache, dev),
            _take(v_scale, "v_scale", f32, cache[:-1], dev))
    new_lens = torch.empty_like(lens)
    _call_on(dev, "reef_b200_kv_compact_i8", n, b, hkv, d, max_len, t, *args,
             new_lens.data_ptr())
    return new_lens
