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

import torch

from . import _native
from .spec import Activation

_DTYPE = {torch.float32: _native.RG_DTYPE_F32, torch.float16: _native.RG_DTYPE_F16,
          torch.bfloat16: _native.RG_DTYPE_BF16}
_ACT = {"none": 0, "relu": 1, "sigmoid": 2, "tanh": 3, "gelu": 4, "leaky_relu": 5, "silu": 6}
_SCALING = {"plain": _native.RG_ROPE_PLAIN, "linear": _native.RG_ROPE_LINEAR, "bands": _native.RG_ROPE_BANDS}

_words: dict[int, torch.Tensor] = {}   # device ordinal -> its two error words


def _error_words(device: int) -> torch.Tensor:
    w = _words.get(device)
    if w is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call a serving operator once on this device before capturing a graph")
        w = torch.zeros(2, dtype=torch.int32, device=torch.device("cuda", device))
        torch.cuda.current_stream(device).synchronize()   # zeroed before any stream's kernel sets it
        _words[device] = w
    return w


def check(device: int | None = None) -> None:
    """Waits for ``device`` (default: the current one) and raises what its serving calls
    reported since the last check (``RgError``), clearing it."""
    device = torch.cuda.current_device() if device is None else torch.device("cuda", device).index
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
    if not first.is_cuda:
        raise ValueError("serving operators need CUDA tensors")
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            raise ValueError(f"tensors on {dev} and {t.device}")
    return dev.index


def _call(device: int, fn, *args) -> None:
    """fn(*args, stream) with ``device`` current."""
    if torch.cuda.current_device() == device:
        st = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            st = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if st:
        _native.check(st)


def _need(t: torch.Tensor, name: str, dtype, shape) -> None:
    if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous {dtype} tensor of shape {shape} is needed, got {t.dtype} "
                         f"{tuple(t.shape)}")


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
    if x.stride(1) != 1 and x.shape[1] > 1 or (x.stride(0) < x.shape[1] and x.shape[0] > 1):
        x = x.contiguous()
    return x


def quantize_weight_i8(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """weight [n, k] (one row per output channel) -> (i8 [n, ld], f32 scales [n]) for
    ``linear_i8_token``; ld is k rounded up to 16, the tail zero.  Done once per weight."""
    if weight.dim() != 2:
        raise ValueError("weight: [out_features, in_features] is needed")
    return quantize_token_i8(weight.contiguous())


def quantize_token_i8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., k] -> (i8 [m, ld], f32 scales [m]): every row with its own scale."""
    x = _rows(x)
    m, k = x.shape
    dev = _device(x)
    ld = (k + 15) // 16 * 16
    q = torch.empty((m, ld), dtype=torch.int8, device=x.device)
    scale = torch.empty(m, dtype=torch.float32, device=x.device)
    _call(dev, _native.lib().rg_quantize_token_i8, x.data_ptr(), _DTYPE[x.dtype], m, k, max(x.stride(0), k),
          q.data_ptr(), ld, scale.data_ptr())
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
    _need(w_scale, "w_scale", torch.float32, (n,))
    if bias is not None:
        _need(bias, "bias", torch.float32, (n,))
    dt = x.dtype if out_dtype is None else out_dtype
    if dt not in _DTYPE:
        raise ValueError(f"out_dtype {dt}")
    shape = x.shape[:-1] + (n,)
    if out is None:
        out = torch.empty(shape, dtype=dt, device=x.device)
    else:
        _need(out, "out", dt, tuple(shape))
    dev = _device(rows, w, w_scale, bias, out)
    if m == 0:
        return out
    code, param = _act(act)
    lib = _native.lib()
    ws = torch.empty(lib.rg_linear_i8_token_workspace_size(m, ld), dtype=torch.uint8, device=x.device)
    _call(dev, lib.rg_linear_i8_token, rows.data_ptr(), _DTYPE[rows.dtype], m, k, max(rows.stride(0), k),
          w.data_ptr(), w_scale.data_ptr(), n, ld, None if bias is None else bias.data_ptr(), code, param,
          out.data_ptr(), _DTYPE[dt], n, ws.data_ptr(), _error_words(dev).data_ptr())
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
    _call(_device(t), _native.lib().rg_rope_table_f32, C.byref(s), positions, rot_dim, t.data_ptr())
    return t


def _strides(t: torch.Tensor) -> list[int]:
    """The strides, 0 for a dimension of one (whose stride in torch may be anything)."""
    return [0 if n == 1 else s for n, s in zip(t.shape, t.stride())]


def _heads(t: torch.Tensor, name: str, written: bool = False) -> tuple[int, int]:
    """The token and head strides of [tokens, heads, head_dim] with head_dim contiguous."""
    if t.dim() != 3 or t.stride(2) != 1:
        raise ValueError(f"{name}: [tokens, heads, head_dim] with contiguous head_dim is needed, got shape "
                         f"{tuple(t.shape)}, strides {t.stride()}")
    ts, hs, _ = _strides(t)
    if written and (ts == 0 and t.shape[0] > 1 or hs == 0 and t.shape[1] > 1):
        raise ValueError(f"{name}: an expanded tensor cannot be written")
    return ts, hs


def _index(t: torch.Tensor, name: str, dtype, n: int) -> None:
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous {dtype} vector of {n} is needed, got {t.dtype} {tuple(t.shape)}")


def _table(table: torch.Tensor, head_dim: int) -> None:
    if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous():
        raise ValueError("table: contiguous float32 [positions, rot_dim] is needed")
    if table.shape[1] > head_dim:
        raise ValueError(f"table: rot_dim {table.shape[1]} exceeds head_dim {head_dim}")


def rope(x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, interleaved: bool = False,
         out: torch.Tensor | None = None) -> torch.Tensor:
    """x [tokens, heads, head_dim] with the first ``table.shape[1]`` dimensions of every head
    rotated by their token's position (int32); the rest is copied.  Pairs are (i, i + rot / 2),
    or (2 i, 2 i + 1) when ``interleaved``.  ``out`` may be ``x``."""
    xt, xh = _heads(x, "x")
    if x.dtype not in _DTYPE:
        raise ValueError(f"x: float32, float16 or bfloat16 is needed, got {x.dtype}")
    n, h, d = x.shape
    _index(positions, "positions", torch.int32, n)
    _table(table, d)
    if out is None:
        out = torch.empty((n, h, d), dtype=x.dtype, device=x.device)
    elif out.dtype != x.dtype or out.shape != x.shape:
        raise ValueError("out: x's shape and dtype are needed")
    ot, oh = _heads(out, "out", written=True)
    dev = _device(x, positions, table, out)
    if n == 0 or h == 0:
        return out
    _call(dev, _native.lib().rg_rope, x.data_ptr(), _DTYPE[x.dtype], n, h, d, xt, xh,
          positions.data_ptr(), table.data_ptr(), table.shape[0], table.shape[1], interleaved, out.data_ptr(),
          ot, oh, _error_words(dev).data_ptr())
    return out


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor) -> _native.KvCacheC:
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype or \
            k_cache.stride(3) != 1 or v_cache.stride(3) != 1 or _strides(k_cache) != _strides(v_cache):
        raise ValueError("caches: two [pages, page_size, kv_heads, head_dim] tensors of one dtype with the same "
                         "strides and contiguous head_dim are needed")
    if k_cache.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"caches: float16 or bfloat16 is needed, got {k_cache.dtype}")
    pages, page, heads, dim = k_cache.shape
    sp, st, sh, _ = _strides(k_cache)
    return _native.KvCacheC(k_cache.data_ptr(), v_cache.data_ptr(), _DTYPE[k_cache.dtype], page, heads, dim, pages,
                            sp, st, sh)


def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
              positions: torch.Tensor | None = None, table: torch.Tensor | None = None, interleaved: bool = False,
              q: torch.Tensor | None = None, q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Stores k and v [tokens, kv_heads, head_dim] in the caches (logical shape [pages,
    page_size, kv_heads, head_dim], any strides with contiguous head_dim), token t at
    ``slots[t]`` = page * page_size + offset (int64; negative: not stored).  With ``table``
    the keys are rotated by ``positions`` (int32) on the way.  With ``q`` [tokens, heads,
    head_dim] returns q rotated, in the cache's dtype.  k, v and q are views of any strides
    (one fused projection's output), f32 or of the cache's dtype."""
    a = _native.KvAppendArgs()
    a.k_token_stride, a.k_head_stride = _heads(k, "k")
    a.v_token_stride, a.v_head_stride = _heads(v, "v")
    cache = _cache(k_cache, v_cache)
    n, hk, d = k.shape
    if v.shape != k.shape or (hk, d) != (cache.kv_heads, cache.head_dim):
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)} do not fit {tuple(k_cache.shape)}")
    if k.dtype not in (torch.float32, k_cache.dtype) or v.dtype != k.dtype:
        raise ValueError(f"k and v: float32 or {k_cache.dtype} is needed, got {k.dtype} and {v.dtype}")
    _index(slots, "slots", torch.int64, n)
    if table is not None:
        if positions is None:
            raise ValueError("positions are needed with a table")
        _index(positions, "positions", torch.int32, n)
        _table(table, d)
        a.positions, a.table = positions.data_ptr(), table.data_ptr()
        a.table_rows, a.rot_dim = table.shape
    if q is not None:
        a.q_token_stride, a.q_head_stride = _heads(q, "q")
        if q.dtype != k.dtype or q.shape[0] != n or q.shape[2] != d or q.shape[1] == 0:
            raise ValueError(f"q: {k.dtype} [{n}, heads, {d}] is needed, got {q.dtype} {tuple(q.shape)}")
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=k_cache.dtype, device=q.device)
        elif q_out.dtype != k_cache.dtype or q_out.shape != q.shape:
            raise ValueError(f"q_out: {k_cache.dtype} of q's shape is needed")
        a.q_out_token_stride, a.q_out_head_stride = _heads(q_out, "q_out", written=True)
        a.q, a.q_out, a.heads = q.data_ptr(), q_out.data_ptr(), q.shape[1]
    elif q_out is not None:
        raise ValueError("q_out without q")
    dev = _device(k, v, k_cache, v_cache, slots, positions, table, q, q_out)
    if n == 0:
        return q_out
    a.k, a.v, a.slots = k.data_ptr(), v.data_ptr(), slots.data_ptr()
    a.tokens, a.x_dtype, a.interleaved = n, _DTYPE[k.dtype], interleaved
    _call(dev, _native.lib().rg_kv_append, C.byref(cache), C.byref(a), _error_words(dev).data_ptr())
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
    qt, qh = _heads(q, "q")
    cache = _cache(k_cache, v_cache)
    n, h, d = q.shape
    if q.dtype != k_cache.dtype or d != cache.head_dim or h == 0 or h % cache.kv_heads:
        raise ValueError(f"q {q.dtype} {tuple(q.shape)} does not fit {k_cache.dtype} {tuple(k_cache.shape)}")
    batch = kv_len.shape[0]
    _index(kv_len, "kv_len", torch.int32, batch)
    _index(cu_q, "cu_q", torch.int32, batch + 1)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != batch or \
            (block_table.stride(1) != 1 and block_table.shape[1] > 1):
        raise ValueError(f"block_table: int32 [{batch}, max_pages] with contiguous rows is needed")
    if out is None:
        out = torch.empty((n, h, d), dtype=q.dtype, device=q.device)
    elif out.dtype != q.dtype or out.shape != q.shape:
        raise ValueError("out: q's shape and dtype are needed")
    ot, oh = _heads(out, "out", written=True)
    dev = _device(q, k_cache, v_cache, block_table, kv_len, cu_q, out)
    pages = block_table.shape[1]
    a = _native.PagedAttentionArgs(
        q.data_ptr(), out.data_ptr(), qt, qh, ot, oh,
        block_table.data_ptr(), block_table.stride(0), kv_len.data_ptr(), cu_q.data_ptr(), n, batch, h, max_q_len,
        pages * cache.page_size if max_kv_len is None else max_kv_len, pages, causal,
        1.0 / math.sqrt(d) if scale is None else scale)
    lib = _native.lib()
    need = lib.rg_attention_paged_workspace_size(C.byref(cache), C.byref(a))
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    _call(dev, lib.rg_attention_paged, C.byref(cache), C.byref(a), None if ws is None else ws.data_ptr(),
          _error_words(dev).data_ptr())
    return out
