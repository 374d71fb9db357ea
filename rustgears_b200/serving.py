"""Decoder-serving operators on CUDA tensors: what one attention block of an INT8 decoder
chains between its norms.

    y   = linear_i8_token(x, w, w_scale)                    # x W^T, i8 with a scale per token
    q   = kv_append(k, v, k_cache, v_cache, slots, ...)     # rotate q and k, store k and v
    out = attention_paged(q, k_cache, v_cache, ...)         # new tokens against the cache

``rope`` rotates without a cache, ``rope_table`` builds the cos / sin rows both use, and
:class:`PagedKvCache` hands out pages and holds the index tensors of a batch.

Every operator runs on the current stream of its tensors' device, neither waits nor
copies to the host, and can be captured in a CUDA graph (after one call outside of a
capture on that device).  Shapes, dtypes and strides are checked here and in the library
before anything is launched.  What only the device can see (a slot, position, page or
length out of range, a bounded wait that gave up) sets the device's error words, which
:func:`check` reads: call it where the program synchronises anyway.  An out-of-range
index is never followed; its token, page or sequence is skipped.

The reference has no counterpart (no cache, no rotary positions; its Linears quantize a
whole batch with one scale, src/inference/npu.rs:312).
"""
from __future__ import annotations

import ctypes as C
import math
import struct

import torch

from . import _native
from .spec import Activation

_DTYPE = {torch.float32: _native.RG_DTYPE_F32, torch.float16: _native.RG_DTYPE_F16,
          torch.bfloat16: _native.RG_DTYPE_BF16}
_ACT = {"none": 0, "relu": 1, "sigmoid": 2, "tanh": 3, "gelu": 4, "leaky_relu": 5, "silu": 6}
_SCALING = {"plain": _native.RG_ROPE_PLAIN, "linear": _native.RG_ROPE_LINEAR, "bands": _native.RG_ROPE_BANDS}

# The library's argument structs, packed: one bytes object per call instead of a ctypes
# structure filled field by field (a third of its time; a decode step is made of such calls).
_LINEAR = struct.Struct("@5P6q3if")      # rg_linear_token_args
_ROPE = struct.Struct("@2P4q2P2q5i")     # rg_rope_args
_CACHE = struct.Struct("@2P4i4q")        # rg_kv_cache
_APPEND = struct.Struct("@4P8q3P2q4i")   # rg_kv_append_args
_ATTENTION = struct.Struct("@2P4qPq2Pq6if")  # rg_paged_attention_args

# The current stream's handle without making a Stream object (1.2 us less per call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)

_lib = None
_words: dict[int, torch.Tensor] = {}   # device ordinal -> its two error words
_word_at: dict[int, int] = {}          # ... and their address


def _library():
    global _lib
    if _lib is None:
        _lib = _native.lib()
    return _lib


def _error_words(device: int) -> int:
    """Address of the device's error words, made (zeroed) by its first call."""
    at = _word_at.get(device)
    if at is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call a serving operator once on this device before capturing a graph")
        w = torch.zeros(2, dtype=torch.int32, device=torch.device("cuda", device))
        torch.cuda.current_stream(device).synchronize()   # zeroed before any stream's kernel sets it
        _words[device] = w
        at = _word_at[device] = w.data_ptr()
    return at


def check(device: int | None = None) -> None:
    """Waits for ``device`` (default: the current one) and raises what its serving calls
    reported since the last check (``RgError``), clearing it."""
    if device is None:
        device = torch.cuda.current_device()
    elif not isinstance(device, int):
        device = torch.device(device).index or 0
    w = _words.get(device)
    if w is None:
        return
    torch.cuda.synchronize(device)
    host = w.tolist()
    if host != [0, 0]:
        w.zero_()
        torch.cuda.synchronize(device)
        _native.check(_native.lib().rg_status_from_error_words((C.c_int32 * 2)(*host)))


def _device(first: torch.Tensor, *others) -> int:
    """The common CUDA device of the tensors (None entries are skipped)."""
    dev = first.get_device()
    if dev < 0:
        raise ValueError("serving operators need CUDA tensors")
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensors on {first.device} and {t.device}")
    return dev


def _call(device: int, fn, *args) -> None:
    """fn(*args, stream) with ``device`` current, on its current stream."""
    if torch.cuda.current_device() != device:
        with torch.cuda.device(device):
            return _call(device, fn, *args)
    st = fn(*args, _raw_stream(device))
    if st:
        _native.check(st)


def _vector(t: torch.Tensor, name: str, dtype, n: int) -> None:
    if t.dtype != dtype or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous {dtype} vector of {n} is needed, got {t.dtype} {tuple(t.shape)}")


def _act(act) -> tuple[int, float]:
    if isinstance(act, Activation):
        return act.code, act.param
    if act not in _ACT:
        raise ValueError(f"unknown activation {act!r}")
    return _ACT[act], 0.01 if act == "leaky_relu" else 0.0


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [..., k] as rows [m, k], the last dimension contiguous (a copy only if it has to be)."""
    if x.dtype not in _DTYPE:
        raise ValueError(f"x: float32, float16 or bfloat16 is needed, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x: [..., k] with k > 0 is needed, got {tuple(x.shape)}")
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if not x.is_contiguous():
        (m, k), (sm, sk) = x.shape, x.stride()
        if (sk != 1 and k > 1) or (sm < k and m > 1):
            x = x.contiguous()
    return x


def _ldx(x: torch.Tensor, k: int) -> int:
    return x.stride(0) if x.shape[0] > 1 else k


def quantize_weight_i8(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """weight [n, k] (one row per output channel) -> (i8 [n, ld], f32 scales [n]) for
    ``linear_i8_token``; ld is k rounded up to 16, the tail zero.  Done once per weight."""
    if weight.dim() != 2:
        raise ValueError("weight: [out_features, in_features] is needed")
    return quantize_token_i8(weight)


def quantize_token_i8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., k] -> (i8 [m, ld], f32 scales [m]): every row with its own scale."""
    x = _rows(x)
    m, k = x.shape
    dev = _device(x)
    ld = (k + 15) // 16 * 16
    q = torch.empty((m, ld), dtype=torch.int8, device=x.device)
    scale = torch.empty(m, dtype=torch.float32, device=x.device)
    _call(dev, _library().rg_quantize_token_i8, x.data_ptr(), _DTYPE[x.dtype], m, k, _ldx(x, k), q.data_ptr(), ld,
          scale.data_ptr())
    return q, scale


def linear_i8_token(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor | None = None,
                    act="none", out_dtype: torch.dtype | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """act(x W^T + bias) with x [..., k] quantized to i8 row by row and w [n, ld], w_scale [n]
    from ``quantize_weight_i8`` (ld >= k).  The product is exact in 32-bit integers; its scale
    is row scale * channel scale; the result is rounded once to ``out_dtype`` (default: x's).
    ``act``: an activation name or :class:`Activation`."""
    rows = _rows(x)
    m, k = rows.shape
    if w.dim() != 2 or w.dtype != torch.int8 or not w.is_contiguous() or w.shape[1] < k or w.shape[1] % 16:
        raise ValueError(f"w: contiguous int8 [n, ld] with ld >= {k}, a multiple of 16, is needed, got {w.dtype} "
                         f"{tuple(w.shape)}")
    n, ld = w.shape
    _vector(w_scale, "w_scale", torch.float32, n)
    if bias is not None:
        _vector(bias, "bias", torch.float32, n)
    dt = x.dtype if out_dtype is None else out_dtype
    code = _DTYPE.get(dt)
    if code is None:
        raise ValueError(f"out_dtype: float32, float16 or bfloat16 is needed, got {dt}")
    act_code, act_param = _act(act)
    if out is not None and (out.dtype != dt or out.shape != x.shape[:-1] + (n,) or not out.is_contiguous()):
        raise ValueError(f"out: contiguous {dt} {tuple(x.shape[:-1]) + (n,)} is needed, got {out.dtype} "
                         f"{tuple(out.shape)}")
    dev = _device(rows, w, w_scale, bias, out)
    if out is None:
        out = torch.empty((m, n) if x is rows else x.shape[:-1] + (n,), dtype=dt, device=x.device)
    if m == 0:
        return out
    lib = _lib or _library()
    need = lib.rg_linear_i8_token_workspace_size(m, ld)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    _call(dev, lib.rg_linear_i8_token,
          _LINEAR.pack(rows.data_ptr(), w.data_ptr(), w_scale.data_ptr(), 0 if bias is None else bias.data_ptr(),
                       out.data_ptr(), m, k, _ldx(rows, k), n, ld, n, _DTYPE[rows.dtype], code, act_code, act_param),
          ws.data_ptr() if need else None, _word_at.get(dev) or _error_words(dev))
    return out


def rope_table(positions: int, rot_dim: int, base: float = 10000.0, scaling: str = "plain", factor: float = 1.0,
               gain: float = 1.0, old_context: int = 0, fast_turns: float = 32.0, slow_turns: float = 1.0,
               device="cuda") -> torch.Tensor:
    """cos / sin rows [positions, rot_dim] (rot_dim / 2 cosines, then the sines), f32 from 64-bit
    angles.  ``scaling``: "plain", "linear" (positions / factor), or "bands" (dimensions that
    turn at least ``fast_turns`` times within ``old_context`` keep their frequency, those that
    turn at most ``slow_turns`` times are slowed by ``factor``, a ramp between).  ``gain``
    multiplies every entry."""
    if scaling not in _SCALING:
        raise ValueError(f"unknown scaling {scaling!r}")
    t = torch.empty((positions, rot_dim), dtype=torch.float32, device=device)
    s = _native.RopeScaling(_SCALING[scaling], base, factor, gain, old_context, fast_turns, slow_turns)
    _call(_device(t), _library().rg_rope_table_f32, C.byref(s), positions, rot_dim, t.data_ptr())
    return t


def _heads(t: torch.Tensor, name: str, written: bool = False) -> tuple[int, int, int, int, int]:
    """[tokens, heads, head_dim] with head_dim contiguous: its sizes, then its token and head
    strides (0 for a dimension of one, whose stride in torch may be anything)."""
    if t.dim() != 3 or t.stride(2) != 1:
        raise ValueError(f"{name}: [tokens, heads, head_dim] with contiguous head_dim is needed, got shape "
                         f"{tuple(t.shape)}, strides {t.stride()}")
    n, h, d = t.shape
    ts, hs, _ = t.stride()
    if n == 1:
        ts = 0
    elif ts == 0 and written:
        raise ValueError(f"{name}: an expanded tensor cannot be written")
    if h == 1:
        hs = 0
    elif hs == 0 and written:
        raise ValueError(f"{name}: an expanded tensor cannot be written")
    return n, h, d, ts, hs


def _table(table: torch.Tensor, head_dim: int) -> tuple[int, int]:
    if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous():
        raise ValueError("table: contiguous float32 [positions, rot_dim] is needed")
    rows, rot = table.shape
    if rot > head_dim:
        raise ValueError(f"table: rot_dim {rot} exceeds head_dim {head_dim}")
    return rows, rot


def rope(x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, interleaved: bool = False,
         out: torch.Tensor | None = None) -> torch.Tensor:
    """x [tokens, heads, head_dim] with the first ``table.shape[1]`` dimensions of every head
    rotated by their token's position (int32); the rest is copied.  Pairs are (i, i + rot / 2),
    or (2 i, 2 i + 1) when ``interleaved``.  ``out`` may be ``x``."""
    n, h, d, xt, xh = _heads(x, "x")
    dt = _DTYPE.get(x.dtype)
    if dt is None:
        raise ValueError(f"x: float32, float16 or bfloat16 is needed, got {x.dtype}")
    _vector(positions, "positions", torch.int32, n)
    rows, rot = _table(table, d)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        ot, oh = h * d, d
    else:
        if out.dtype != x.dtype or out.shape != x.shape:
            raise ValueError("out: x's shape and dtype are needed")
        _, _, _, ot, oh = _heads(out, "out", written=True)
    dev = _device(x, positions, table, out)
    if n == 0 or h == 0:
        return out
    _call(dev, (_lib or _library()).rg_rope,
          _ROPE.pack(x.data_ptr(), out.data_ptr(), xt, xh, ot, oh, positions.data_ptr(), table.data_ptr(), rows, n,
                     dt, h, d, rot, interleaved), _word_at.get(dev) or _error_words(dev))
    return out


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple[bytes, int, int, int]:
    """The packed cache, its page size, heads and head_dim."""
    shape, strides = k_cache.shape, k_cache.stride()
    dt = k_cache.dtype
    if len(shape) != 4 or v_cache.shape != shape or v_cache.dtype != dt or strides[3] != 1:
        raise ValueError("caches: two [pages, page_size, kv_heads, head_dim] tensors of one dtype with the same "
                         "strides and contiguous head_dim are needed")
    if v_cache.stride() != strides and any(n > 1 and a != b for n, a, b in zip(shape, strides, v_cache.stride())):
        raise ValueError("caches: the key and value tensors have different strides")
    if dt is not torch.float16 and dt is not torch.bfloat16:
        raise ValueError(f"caches: float16 or bfloat16 is needed, got {dt}")
    pages, page, heads, dim = shape
    sp, st, sh, _ = strides
    return (_CACHE.pack(k_cache.data_ptr(), v_cache.data_ptr(), _DTYPE[dt], page, heads, dim, pages,
                        sp if pages > 1 else 0, st if page > 1 else 0, sh if heads > 1 else 0), page, heads, dim)


def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
              positions: torch.Tensor | None = None, table: torch.Tensor | None = None, interleaved: bool = False,
              q: torch.Tensor | None = None, q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Stores k and v [tokens, kv_heads, head_dim] in the caches (logical shape [pages,
    page_size, kv_heads, head_dim], any strides with contiguous head_dim), token t at
    ``slots[t]`` = page * page_size + offset (int64; negative: not stored).  With ``table``
    the keys are rotated by ``positions`` (int32) on the way.  With ``q`` [tokens, heads,
    head_dim] returns q rotated, in the cache's dtype.  k, v and q are views of any strides
    (one fused projection's output), f32 or of the cache's dtype."""
    n, hk, d, kt, kh = _heads(k, "k")
    nv, hv, dv, vt, vh = _heads(v, "v")
    cache, _, heads_c, dim_c = _cache(k_cache, v_cache)
    if nv != n or hv != hk or dv != d or hk != heads_c or d != dim_c:
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)} do not fit {tuple(k_cache.shape)}")
    dt, ct = k.dtype, k_cache.dtype
    if (dt is not torch.float32 and dt != ct) or v.dtype != dt:
        raise ValueError(f"k and v: float32 or {ct} is needed, got {dt} and {v.dtype}")
    _vector(slots, "slots", torch.int64, n)
    pos_at = table_at = rows = rot = 0
    if table is not None:
        if positions is None:
            raise ValueError("positions are needed with a table")
        _vector(positions, "positions", torch.int32, n)
        rows, rot = _table(table, d)
        pos_at, table_at = positions.data_ptr(), table.data_ptr()
    q_at = out_at = h = qt = qh = ot = oh = 0
    if q is not None:
        nq, h, dq, qt, qh = _heads(q, "q")
        if q.dtype != dt or nq != n or dq != d or h == 0:
            raise ValueError(f"q: {dt} [{n}, heads, {d}] is needed, got {q.dtype} {tuple(q.shape)}")
        if q_out is None:
            q_out = torch.empty((n, h, d), dtype=ct, device=q.device)
            ot, oh = h * d, d
        else:
            if q_out.dtype != ct or q_out.shape != q.shape:
                raise ValueError(f"q_out: {ct} of q's shape is needed")
            _, _, _, ot, oh = _heads(q_out, "q_out", written=True)
        q_at, out_at = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    dev = _device(k, v, k_cache, v_cache, slots, positions, table, q, q_out)
    if n == 0:
        return q_out
    _call(dev, (_lib or _library()).rg_kv_append, cache,
          _APPEND.pack(k.data_ptr(), v.data_ptr(), q_at, out_at, kt, kh, vt, vh, qt, qh, ot, oh, slots.data_ptr(),
                       pos_at, table_at, rows, n, _DTYPE[dt], h, rot, interleaved),
          _word_at.get(dev) or _error_words(dev))
    return q_out


def attention_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    kv_len: torch.Tensor, cu_q: torch.Tensor, max_q_len: int, max_kv_len: int | None = None,
                    scale: float | None = None, causal: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of new tokens q [tokens, heads, head_dim] over a paged cache.

    Sequence b owns tokens ``cu_q[b]`` .. ``cu_q[b + 1]`` - 1 and ``kv_len[b]`` keys (its new
    ones included: append first), in the pages ``block_table[b]`` names ([batch, max_pages],
    all int32).  ``causal``: its tokens are the last of its keys, each seeing itself and what
    is before it.  A row that sees no key is zeros.  heads is a multiple of the cache's heads
    (shared in order).  ``max_q_len`` and ``max_kv_len`` (default: what the table can hold)
    bound the lengths; ``scale`` defaults to 1 / sqrt(head_dim)."""
    n, h, d, qt, qh = _heads(q, "q")
    cache, page, heads_c, dim_c = _cache(k_cache, v_cache)
    if q.dtype != k_cache.dtype or d != dim_c or h == 0 or h % heads_c:
        raise ValueError(f"q {q.dtype} {tuple(q.shape)} does not fit {k_cache.dtype} {tuple(k_cache.shape)}")
    batch = kv_len.numel()
    _vector(kv_len, "kv_len", torch.int32, batch)
    _vector(cu_q, "cu_q", torch.int32, batch + 1)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != batch or \
            (block_table.stride(1) != 1 and block_table.shape[1] > 1):
        raise ValueError(f"block_table: int32 [{batch}, max_pages] with contiguous rows is needed")
    pages = block_table.shape[1]
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        ot, oh = h * d, d
    else:
        if out.dtype != q.dtype or out.shape != q.shape:
            raise ValueError("out: q's shape and dtype are needed")
        _, _, _, ot, oh = _heads(out, "out", written=True)
    dev = _device(q, k_cache, v_cache, block_table, kv_len, cu_q, out)
    args = _ATTENTION.pack(
        q.data_ptr(), out.data_ptr(), qt, qh, ot, oh, block_table.data_ptr(), block_table.stride(0), kv_len.data_ptr(),
        cu_q.data_ptr(), n, batch, h, max_q_len, pages * page if max_kv_len is None else max_kv_len, pages, causal,
        1.0 / math.sqrt(d) if scale is None else scale)
    lib = _lib or _library()
    need = lib.rg_attention_paged_workspace_size(cache, args)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    _call(dev, lib.rg_attention_paged, cache, args, ws.data_ptr() if need > 0 else None,
          _word_at.get(dev) or _error_words(dev))
    return out
