"""Decoder-serving operators on CUDA tensors: what one attention block of an INT8 decoder
chains between its norms.

    y   = linear_i8_token(x, w, w_scale)                    # x W^T, i8 with a scale per token
    q   = kv_append(k, v, k_cache, v_cache, slots, ...)     # rotate q and k, store k and v
    out = attention_paged(q, k_cache, v_cache, ...)         # new tokens against the cache

``rope`` rotates without a cache, ``rope_table`` builds the cos / sin rows both use, and
:class:`PagedKvCache` hands out pages and holds the index tensors of a batch.

Every operator runs on the current stream of its tensors' device, neither waits nor
copies to the host, and can be captured in a CUDA graph (after one call outside of a
capture on that device).  Shapes, dtypes, strides and devices are checked here
(``ValueError``) and in the library (``RgError``) before anything is launched.  What only
the device can see (a slot, position, page or length out of range, a bounded wait that
gave up) sets the device's error words, which :func:`check` reads: call it where the
program synchronises anyway.  An out-of-range index is never followed; its token, page
or sequence is skipped.

Two limits of masks: keys past a sequence's ``kv_len`` may hold anything, NaN included;
but a NaN or an infinity in the *values* of a key that only later tokens of the same
sequence see reaches earlier ones too (a probability of 0 times it).

The reference has no counterpart (no cache, no rotary positions; its Linears quantize a
whole batch with one scale, src/inference/npu.rs:312).
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _native
from .spec import Activation

_native.lib()
try:
    from . import _serving_bind as _bind
except ImportError as e:
    raise ImportError(f"{e}: build it with `python -m rustgears_b200.build` (a CUDA torch is needed)") from e
if _bind.torch_version != torch.__version__:
    raise ImportError(f"_serving_bind was built for torch {_bind.torch_version}, this is {torch.__version__}: build it "
                      "again with `python -m rustgears_b200.build`")
_bind.set_check(_native.check)

_ACT = {"none": (0, 0.0), "relu": (1, 0.0), "sigmoid": (2, 0.0), "tanh": (3, 0.0), "gelu": (4, 0.0),
        "leaky_relu": (5, 0.01), "silu": (6, 0.0)}
_SCALING = {"plain": _native.RG_ROPE_PLAIN, "linear": _native.RG_ROPE_LINEAR, "bands": _native.RG_ROPE_BANDS}


def check(device: int | torch.device | str | None = None) -> None:
    """Waits for ``device`` (default: the current one) and raises what its serving calls
    reported since the last check (``RgError``), clearing it.  The report is the device's: it
    covers the calls of every thread and stream, and one check takes it for all of them."""
    if device is None:
        device = torch.cuda.current_device()
    elif not isinstance(device, int):
        index = torch.device(device).index
        device = torch.cuda.current_device() if index is None else index
    words = _bind.words(device)
    if words is None:
        return
    torch.cuda.synchronize(device)
    with torch.cuda.device(device):
        taken = torch.empty_like(words)
        _native.check(_native.lib().rg_take_error_words(words.data_ptr(), taken.data_ptr(),
                                                        torch.cuda.current_stream().cuda_stream))
        host = taken.tolist()
    if host != [0, 0]:
        _native.check(_native.lib().rg_status_from_error_words((C.c_int32 * 2)(*host)))


def quantize_weight_i8(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """weight [n, k] (one row per output channel) -> (i8 [n, ld], f32 scales [n]) for
    ``linear_i8_token``; ld is k rounded up to 16, the tail zero.  Done once per weight."""
    if weight.dim() != 2:
        raise ValueError("weight: [out_features, in_features] is needed")
    return _bind.quantize(weight)


def quantize_token_i8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., k] -> (i8 [m, ld], f32 scales [m]): every row with its own scale."""
    return _bind.quantize(x)


def linear_i8_token(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor | None = None,
                    act: str | Activation = "none", out_dtype: torch.dtype | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """act(x W^T + bias) with x [..., k] quantized to i8 row by row and w [n, ld], w_scale [n]
    from ``quantize_weight_i8`` (ld >= k).  The product is exact in 32-bit integers; its scale
    is row scale * channel scale; the result is rounded once to ``out_dtype`` (default: x's).
    ``out`` may be ``x`` or overlap it.  ``act``: an activation name or :class:`Activation`.  f32 results follow the framework's
    activations bit for bit; 16-bit GELU and SiLU are within their own rounding of them."""
    if isinstance(act, Activation):
        code, param = act.code, act.param
    else:
        try:
            code, param = _ACT[act]
        except (KeyError, TypeError):
            raise ValueError(f"unknown activation {act!r}") from None
    return _bind.linear(x, w, w_scale, bias, code, param, out_dtype, out)


def rope_table(positions: int, rot_dim: int, base: float = 10000.0, scaling: str = "plain", factor: float = 1.0,
               gain: float = 1.0, old_context: float = 0, fast_turns: float = 32.0, slow_turns: float = 1.0,
               device="cuda") -> torch.Tensor:
    """cos / sin rows [positions, rot_dim] (rot_dim / 2 cosines, then the sines), f32 from 64-bit
    angles.  ``scaling``: "plain", "linear" (positions / factor), or "bands" (dimensions that
    turn at least ``fast_turns`` times within ``old_context`` keep their frequency, those that
    turn at most ``slow_turns`` times are slowed by ``factor``, a ramp between).  ``gain``
    multiplies every entry."""
    if scaling not in _SCALING:
        raise ValueError(f"unknown scaling {scaling!r}")
    t = torch.empty((positions, rot_dim), dtype=torch.float32, device=device)
    if not t.is_cuda:
        raise ValueError("serving operators need CUDA tensors")
    s = _native.RopeScaling(_SCALING[scaling], base, factor, gain, old_context, fast_turns, slow_turns)
    with torch.cuda.device(t.device):
        _native.check(_native.lib().rg_rope_table_f32(C.byref(s), positions, rot_dim, t.data_ptr(),
                                                      torch.cuda.current_stream(t.device).cuda_stream))
    return t


def rope(x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, interleaved: bool = False,
         out: torch.Tensor | None = None) -> torch.Tensor:
    """x [tokens, heads, head_dim] with the first ``table.shape[1]`` dimensions of every head
    rotated by their token's position (int32); the rest is copied.  Pairs are (i, i + rot / 2),
    or (2 i, 2 i + 1) when ``interleaved``.  x: any strides with contiguous head_dim; ``out``
    may be ``x``."""
    return _bind.rope(x, positions, table, interleaved, out)


def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
              positions: torch.Tensor | None = None, table: torch.Tensor | None = None, interleaved: bool = False,
              q: torch.Tensor | None = None, q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Stores k and v [tokens, kv_heads, head_dim] in the caches (logical shape [pages,
    page_size, kv_heads, head_dim], any strides with contiguous head_dim), token t at
    ``slots[t]`` = page * page_size + offset (int64; negative: not stored).  With ``table``
    the keys are rotated by ``positions`` (int32) on the way.  With ``q`` [tokens, heads,
    head_dim] returns q rotated, in the cache's dtype.  k, v and q are views of any strides
    (one fused projection's output), f32 or of the cache's dtype."""
    return _bind.append(k, v, k_cache, v_cache, slots, positions, table, interleaved, q, q_out)


def attention_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    kv_len: torch.Tensor, cu_q: torch.Tensor, max_q_len: int, max_kv_len: int | None = None,
                    scale: float | None = None, causal: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of new tokens q [tokens, heads, head_dim] over a paged cache.

    Sequence b owns tokens ``cu_q[b]`` .. ``cu_q[b + 1]`` - 1 and ``kv_len[b]`` keys (its new
    ones included: append first), in the pages ``block_table[b]`` names ([batch, max_pages],
    all int32).  ``causal``: its tokens are the last of its keys, each seeing itself and what
    is before it.  A row that sees no key is zeros.  heads is a multiple of the cache's heads
    (shared in order); head_dim 64, 96, 128 or 256.  ``max_q_len`` and ``max_kv_len`` (default:
    what the table can hold) bound the lengths: a sequence beyond them is reported by
    :func:`check` and skipped.  Rows of the result that no sequence owns (padding behind
    ``cu_q[-1]``), and a skipped sequence's, are not written: they keep what ``out`` held, or
    hold anything when the result is allocated here.  ``scale`` defaults to
    1 / sqrt(head_dim)."""
    return _bind.attention(q, k_cache, v_cache, block_table, kv_len, cu_q, max_q_len, max_kv_len, scale, causal, out)


@dataclass
class Step:
    """The index tensors of one batch of new tokens, in the order of the sequences given to
    :meth:`PagedKvCache.extend`; every layer of a model uses the same ones."""
    positions: torch.Tensor     # int32 [tokens]
    slots: torch.Tensor         # int64 [tokens]
    block_table: torch.Tensor   # int32 [batch, max_pages]
    kv_len: torch.Tensor        # int32 [batch], the new tokens included
    cu_q: torch.Tensor          # int32 [batch + 1]
    max_q_len: int
    max_kv_len: int


class PagedKvCache:
    """The pages of a model's layers and which sequence holds which.  ``k[layer]`` and
    ``v[layer]`` are [pages, page_size, kv_heads, head_dim]; a page index means the same page in
    every layer.  The bookkeeping is on the host; :meth:`extend` makes one step's index tensors
    with one copy to the device."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if min(layers, pages, page_size, kv_heads, head_dim) <= 0:
            raise ValueError("layers, pages, page_size, kv_heads and head_dim have to be positive")
        self.page_size = page_size
        self.k = [torch.zeros((pages, page_size, kv_heads, head_dim), dtype=dtype, device=device) for _ in range(layers)]
        self.v = [torch.zeros_like(k) for k in self.k]
        self._free = list(range(pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}
        self._len: dict[int, int] = {}

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, sequence: int) -> int:
        """Tokens of ``sequence`` (0 when it is unknown)."""
        return self._len.get(sequence, 0)

    def release(self, sequence: int) -> None:
        """Gives the sequence's pages back.  Work that reads them has to be ordered before work
        that a later step gives them to (one stream does)."""
        self._free.extend(reversed(self._pages.pop(sequence, [])))
        self._len.pop(sequence, None)

    def extend(self, new_tokens: dict[int, int]) -> Step:
        """Room for ``new_tokens[sequence]`` more tokens of each sequence (made when unknown), and
        the step's index tensors.  Nothing changes when the pages do not suffice (``MemoryError``)."""
        page = self.page_size
        if not new_tokens or any(n < 0 for n in new_tokens.values()):
            raise ValueError("new_tokens: a count >= 0 for one sequence at least is needed")
        need = {s: -(-(self.length(s) + n) // page) - len(self._pages.get(s, ())) for s, n in new_tokens.items()}
        if sum(need.values()) > len(self._free):
            raise MemoryError(f"{sum(need.values())} pages are needed, {len(self._free)} are free")
        positions, slots, kv_len, cu_q = [], [], [], [0]
        for s, n in new_tokens.items():
            mine = self._pages.setdefault(s, [])
            mine += [self._free.pop() for _ in range(need[s])]
            first = self.length(s)
            self._len[s] = first + n
            positions += range(first, first + n)
            slots += [mine[p // page] * page + p % page for p in range(first, first + n)]
            kv_len.append(first + n)
            cu_q.append(cu_q[-1] + n)
        batch, tokens = len(kv_len), len(slots)
        width = max(1, max(len(self._pages[s]) for s in new_tokens))
        table = [x for s in new_tokens for x in self._pages[s] + [0] * (width - len(self._pages[s]))]
        # one buffer, the 64-bit slots first
        host = torch.empty(2 * tokens + tokens + 2 * batch + 1 + len(table), dtype=torch.int32,
                           pin_memory=self.k[0].is_cuda)
        host[:2 * tokens].view(torch.int64).copy_(torch.tensor(slots, dtype=torch.int64))
        host[2 * tokens:].copy_(torch.tensor(positions + kv_len + cu_q + table, dtype=torch.int32))
        dev = host.to(self.k[0].device, non_blocking=True)
        slots_t, rest = dev[:2 * tokens].view(torch.int64), dev[2 * tokens:]
        pos_t, kv_t, cu_t, table_t = rest.split([tokens, batch, batch + 1, len(table)])
        return Step(pos_t, slots_t, table_t.view(batch, width), kv_t, cu_t,
                    max(new_tokens.values()), max(kv_len))


class DecoderAttention:
    """Causal multi-head attention of a decoder with i8 projections: the reference's
    MultiHeadAttention (src/nn/attention.rs:162-196) given rotary positions, a paged cache,
    query heads that share key heads, and a quantization scale per token and channel.

    ``wqkv`` [(heads + 2 kv_heads) head_dim, d] (query, key, value rows) and ``wo``
    [d, heads head_dim] are float tensors on the device, quantized once here."""

    def __init__(self, wqkv: torch.Tensor, wo: torch.Tensor, heads: int, kv_heads: int, table: torch.Tensor,
                 bqkv: torch.Tensor | None = None, bo: torch.Tensor | None = None, interleaved: bool = False):
        total = heads + 2 * kv_heads
        if heads <= 0 or kv_heads <= 0 or heads % kv_heads or wqkv.shape[0] % total:
            raise ValueError(f"wqkv {tuple(wqkv.shape)} does not split into {heads} + 2 x {kv_heads} heads")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, wqkv.shape[0] // total
        if wo.shape[1] != heads * self.head_dim:
            raise ValueError(f"wo {tuple(wo.shape)} does not take {heads} heads of {self.head_dim}")
        self.wqkv, self.sqkv = quantize_weight_i8(wqkv)
        self.wo, self.so = quantize_weight_i8(wo)
        self.bqkv, self.bo, self.table, self.interleaved = bqkv, bo, table, interleaved

    def __call__(self, x: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, step: Step) -> torch.Tensor:
        """x [tokens, d] of the step's new tokens -> [tokens, d]; their keys and values are appended."""
        h, hk = self.heads, self.kv_heads
        y = linear_i8_token(x, self.wqkv, self.sqkv, bias=self.bqkv, out_dtype=k_cache.dtype)
        y = y.view(x.shape[0], h + 2 * hk, self.head_dim)
        q = kv_append(y[:, h:h + hk], y[:, h + hk:], k_cache, v_cache, step.slots, positions=step.positions,
                      table=self.table, interleaved=self.interleaved, q=y[:, :h])
        o = attention_paged(q, k_cache, v_cache, step.block_table, step.kv_len, step.cu_q, step.max_q_len,
                            step.max_kv_len)
        return linear_i8_token(o.view(x.shape[0], h * self.head_dim), self.wo, self.so, bias=self.bo, out_dtype=x.dtype)
