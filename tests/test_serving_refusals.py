"""What the decoder-serving entry points refuse, before any device work: every call here
returns its status without a GPU (the pointers are never followed)."""
import ctypes as C

import pytest

from rustgears_b200 import _native

A, U = 0x10000, 0x10008          # an aligned address, and one that is not 16-byte aligned
INVALID, UNSUPPORTED = _native.RG_ERR_INVALID_ARG, _native.RG_ERR_UNSUPPORTED


def refused(name, status, match, *args):
    L = _native.lib()
    assert getattr(L, name)(*args) == status, _native.last_error()
    assert match in _native.last_error(), _native.last_error()


QUANT = dict(x=A, dt=0, rows=4, k=30, ldx=30, q=A, ldq=32, scale=A)


@pytest.mark.parametrize("change,match", [
    (dict(dt=3), "dtype"), (dict(rows=-1), "rows"), (dict(k=0), "k 0"), (dict(ldx=29), "ldx"), (dict(ldq=40), "16"),
    (dict(ldq=16), "ld"), (dict(x=None), "null"), (dict(q=None), "null"), (dict(scale=None), "null"),
    (dict(x=A + 2), "aligned"), (dict(q=U), "aligned")])
def test_quantize(change, match):
    a = {**QUANT, **change}
    refused("rg_quantize_token_i8", INVALID, match, a["x"], a["dt"], a["rows"], a["k"], a["ldx"], a["q"], a["ldq"],
            a["scale"], None)


GEMM = dict(a=A, sa=A, w=A, sw=A, m=4, n=8, ld=32, bias=A, act=0, out=A, dt=0, ldo=8, err=A)


@pytest.mark.parametrize("change,match,status", [
    (dict(dt=5), "dtype", INVALID), (dict(act=7), "activation", INVALID), (dict(act=-1), "activation", INVALID),
    (dict(m=-1), "m -1", INVALID), (dict(n=0), "n 0", INVALID), (dict(ld=24), "16", INVALID), (dict(ld=0), "ld", INVALID),
    (dict(ldo=7), "ldo", INVALID), (dict(ld=1 << 18), "i32", UNSUPPORTED), (dict(a=None), "null", INVALID),
    (dict(sa=None), "null", INVALID), (dict(w=None), "null", INVALID), (dict(sw=None), "null", INVALID),
    (dict(out=None), "null", INVALID), (dict(err=None), "null", INVALID), (dict(a=U), "aligned", INVALID),
    (dict(w=U), "aligned", INVALID), (dict(out=A + 2), "aligned", INVALID)])
def test_gemm(change, match, status):
    a = {**GEMM, **change}
    refused("rg_gemm_i8_token", status, match, a["a"], a["sa"], a["w"], a["sw"], a["m"], a["n"], a["ld"], a["bias"],
            a["act"], C.c_float(0), a["out"], a["dt"], a["ldo"], a["err"], None)


def linear(**change):
    return _native.LinearTokenArgs(**{**dict(x=A, w=A, w_scale=A, bias=A, out=A, m=4, k=30, ldx=30, n=8, ld=32, ldo=8,
                                             x_dtype=0, out_dtype=0, act=0, act_param=0.0), **change})


@pytest.mark.parametrize("change,match,ws", [
    (dict(k=33), "ld", A), (dict(ldx=3), "ldx", A), (dict(x_dtype=9), "dtype", A), (dict(x=None), "null", A),
    (dict(w=None), "null", A), (dict(act=9), "activation", A), (dict(ld=40), "16", A), (dict(ldo=7), "ldo", A)])
def test_linear(change, match, ws):
    refused("rg_linear_i8_token", INVALID, match, C.byref(linear(**change)), ws, A, None)


@pytest.mark.parametrize("change", [
    dict(out=A), dict(out=A + 29 * 4), dict(out=A + 3 * 30 * 4 + 29 * 4), dict(x=A + 16, out=A),
    dict(x=A + 3 * 32 + 28, out=A), dict(ldx=64, ldo=64, out=A + 26 * 4), dict(k=16, ldx=16, ld=16, x_dtype=1, out=A + 96)])
def test_linear_in_one_launch_refuses_an_overlap(change):
    """Few tokens run in one launch that reads x while it writes out."""
    assert _native.lib().rg_linear_i8_token_workspace_size(4, 8, 32) == 0
    args = linear(**change)
    refused("rg_linear_i8_token", INVALID, "overlap", C.byref(args), None, A, None)


def test_linear_needs_its_workspace():
    big = linear(m=300)
    for ws in (None, U):
        refused("rg_linear_i8_token", INVALID, "workspace", C.byref(big), ws, A, None)
    refused("rg_linear_i8_token", INVALID, "null", None, A, A, None)


def test_linear_workspace_holds_rows_and_scales():
    L = _native.lib()
    assert L.rg_linear_i8_token_workspace_size(0, 8, 32) == 0
    assert L.rg_linear_i8_token_workspace_size(300, 8, 32) >= 300 * 32 + 300 * 4


@pytest.mark.parametrize("change,match", [
    (dict(kind=3), "scaling"), (dict(base=1.0), "base"), (dict(base=float("nan")), "base"), (dict(gain=0.0), "gain"),
    (dict(kind=1, factor=0.0), "factor"), (dict(kind=2, factor=2.0), "bands"),
    (dict(kind=2, factor=2.0, old_context=100.0, fast_turns=1.0, slow_turns=2.0), "bands")])
def test_rope_table(change, match):
    s = {**dict(kind=0, base=1e4, factor=1.0, gain=1.0, old_context=0.0, fast_turns=32.0, slow_turns=1.0), **change}
    refused("rg_rope_table_f32", INVALID, match, C.byref(_native.RopeScaling(**s)), 10, 64, A, None)


@pytest.mark.parametrize("n,rot,table,match", [(-1, 64, A, "-1"), (4, 63, A, "even"), (4, 0, A, "rot_dim"),
                                               (4, 64, None, "null")])
def test_rope_table_sizes(n, rot, table, match):
    refused("rg_rope_table_f32", INVALID, match, C.byref(_native.RopeScaling(0, 1e4, 1, 1, 0, 32, 1)), n, rot, table,
            None)


@pytest.mark.parametrize("change,match", [
    (dict(dtype=3), "dtype"), (dict(tokens=-1), "tokens"), (dict(heads=0), "heads"), (dict(head_dim=63), "even"),
    (dict(token_stride=-1), "stride"), (dict(x=None), "null"), (dict(out=None), "null"), (dict(positions=None), "table"),
    (dict(table=None), "table"), (dict(table_rows=0), "table"), (dict(rot_dim=66), "rot_dim"), (dict(rot_dim=3), "even"),
    (dict(x=A + 1), "misaligned")])
def test_rope(change, match):
    a = _native.RopeArgs(**{**dict(x=A, out=A, token_stride=128, head_stride=64, out_token_stride=128,
                                   out_head_stride=64, positions=A, table=A, table_rows=10, tokens=3, dtype=2, heads=2,
                                   head_dim=64, rot_dim=64, interleaved=0), **change})
    refused("rg_rope", INVALID, match, C.byref(a), A, None)


def test_rope_needs_error_words():
    a = _native.RopeArgs(x=A, out=A, token_stride=128, head_stride=64, positions=A, table=A, table_rows=10, tokens=3,
                         dtype=2, heads=2, head_dim=64, rot_dim=64)
    refused("rg_rope", INVALID, "null", C.byref(a), None, None)
    refused("rg_rope", INVALID, "null", None, A, None)


@pytest.mark.parametrize("words,taken,match", [(None, A, "null"), (A, None, "null"), (A + 2, A, "misaligned")])
def test_take_error_words(words, taken, match):
    refused("rg_take_error_words", INVALID, match, words, taken, None)


def cache(**change):
    return _native.KvCacheC(**{**dict(k=A, v=A, dtype=1, page_size=16, kv_heads=2, head_dim=64, pages=10,
                                      page_stride=2048, token_stride=128, head_stride=64), **change})


def append(**change):
    return _native.KvAppendArgs(**{**dict(k=A, v=A, q=A, q_out=A, k_token_stride=128, k_head_stride=64,
                                          v_token_stride=128, v_head_stride=64, q_token_stride=256, q_head_stride=64,
                                          q_out_token_stride=256, q_out_head_stride=64, slots=A, positions=A, table=A,
                                          table_rows=100, tokens=5, x_dtype=0, heads=4, rot_dim=64), **change})


@pytest.mark.parametrize("change,match,status", [
    (dict(dtype=0), "f16 or bf16", UNSUPPORTED), (dict(page_size=0), "pages", INVALID), (dict(pages=0), "pages", INVALID),
    (dict(kv_heads=0), "heads", INVALID), (dict(k=None), "null", INVALID), (dict(v=None), "null", INVALID),
    (dict(token_stride=-1), "stride", INVALID), (dict(k=A + 1), "misaligned", INVALID)])
def test_cache(change, match, status):
    refused("rg_kv_append", status, match, C.byref(cache(**change)), C.byref(append()), A, None)
    refused("rg_attention_paged", status, match, C.byref(cache(**change)), C.byref(attention()), A, A, None)


@pytest.mark.parametrize("change,match,status", [
    (dict(x_dtype=2), "dtype", UNSUPPORTED), (dict(tokens=-1), "tokens", INVALID), (dict(k=None), "null", INVALID),
    (dict(v=None), "null", INVALID), (dict(slots=None), "null", INVALID), (dict(q_out=None), "null", INVALID),
    (dict(heads=0), "heads", INVALID), (dict(positions=None), "table", INVALID), (dict(rot_dim=65), "even", INVALID),
    (dict(rot_dim=66), "rot_dim", INVALID), (dict(table_rows=0), "table", INVALID),
    (dict(k_token_stride=-4), "stride", INVALID), (dict(q_head_stride=-4), "stride", INVALID),
    (dict(slots=A + 4), "misaligned", INVALID)])
def test_append(change, match, status):
    refused("rg_kv_append", status, match, C.byref(cache()), C.byref(append(**change)), A, None)


def test_append_needs_error_words():
    refused("rg_kv_append", INVALID, "null", C.byref(cache()), C.byref(append()), None, None)
    refused("rg_kv_append", INVALID, "null", C.byref(cache()), None, A, None)
    refused("rg_kv_append", INVALID, "null", None, C.byref(append()), A, None)


def attention(**change):
    return _native.PagedAttentionArgs(**{**dict(q=A, out=A, q_token_stride=256, q_head_stride=64,
                                                out_token_stride=256, out_head_stride=64, block_table=A,
                                                block_table_stride=8, kv_len=A, cu_q=A, tokens=9, batch=2, heads=4,
                                                max_q_len=5, max_kv_len=100, max_pages=8, causal=1, scale=0.125),
                                         **change})


@pytest.mark.parametrize("change,match", [
    (dict(batch=-1), "batch"), (dict(batch=65536), "batch"), (dict(tokens=-1), "tokens"), (dict(heads=0), "heads"),
    (dict(heads=3), "heads"), (dict(max_q_len=-1), "max_q_len"), (dict(max_kv_len=-1), "max_kv_len"),
    (dict(max_kv_len=129), "hold"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(kv_len=None), "null"), (dict(cu_q=None), "null"),
    (dict(block_table=None), "null"), (dict(q=U), "aligned"), (dict(out=U), "aligned"), (dict(q_token_stride=12), "multiples"),
    (dict(out_head_stride=-8), "stride"), (dict(cu_q=A + 2), "misaligned")])
def test_attention(change, match):
    refused("rg_attention_paged", INVALID, match, C.byref(cache()), C.byref(attention(**change)), A, A, None)


@pytest.mark.parametrize("dim", [8, 32, 72, 512])
def test_attention_head_dims(dim):
    c = cache(head_dim=dim)
    refused("rg_attention_paged", UNSUPPORTED, "head_dim", C.byref(c), C.byref(attention()), A, A, None)
    assert _native.lib().rg_attention_paged_workspace_size(C.byref(c), C.byref(attention())) == -1


def test_attention_needs_aligned_cache_strides_and_error_words():
    refused("rg_attention_paged", INVALID, "multiples", C.byref(cache(token_stride=129)), C.byref(attention()), A, A, None)
    refused("rg_attention_paged", INVALID, "null", C.byref(cache()), C.byref(attention()), A, None, None)


def test_python_layer_refuses_before_the_library():
    torch = pytest.importorskip("torch")
    from rustgears_b200 import serving as sv
    x, w, s = torch.zeros(2, 32), torch.zeros(8, 32, dtype=torch.int8), torch.zeros(8)
    with pytest.raises(ValueError, match="CUDA"):
        sv.linear_i8_token(x, w, s)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        sv.linear_i8_token(x.double(), w, s)
    with pytest.raises(ValueError, match="w:"):
        sv.linear_i8_token(x, w[:, :16], s)
    with pytest.raises(ValueError, match="w_scale"):
        sv.linear_i8_token(x, w, s[:4])
    with pytest.raises(ValueError, match="bias"):
        sv.linear_i8_token(x, w, s, bias=s[:3])
    with pytest.raises(ValueError, match="out"):
        sv.linear_i8_token(x, w, s, out=torch.zeros(2, 7))
    h, pos, table = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32), torch.zeros(5, 64)
    for bad in (h[0], h.transpose(1, 2)):
        with pytest.raises(ValueError, match="head_dim"):
            sv.rope(bad, pos, table)
    with pytest.raises(ValueError, match="positions"):
        sv.rope(h, pos.long(), table)
    with pytest.raises(ValueError, match="rot_dim"):
        sv.rope(h, pos, torch.zeros(5, 66))
    with pytest.raises(ValueError, match="expanded"):
        sv.rope(h, pos, table, out=torch.zeros(1, 2, 64).expand(3, 2, 64))
    with pytest.raises(ValueError, match="scaling"):
        sv.rope_table(4, 64, scaling="cubic", device="cpu")
    kc = torch.zeros(4, 8, 2, 64, dtype=torch.float16)
    slots = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="caches"):
        sv.kv_append(h, h, kc, kc.bfloat16(), slots)
    with pytest.raises(ValueError, match="caches"):
        sv.kv_append(h, h, kc.float(), kc.float(), slots)
    with pytest.raises(ValueError, match="caches"):
        sv.kv_append(h, h, kc, kc.transpose(1, 2).contiguous().transpose(1, 2), slots)
    with pytest.raises(ValueError, match="fit"):
        sv.kv_append(h[:, :1], h[:, :1], kc, kc, slots)
    with pytest.raises(ValueError, match="k and v"):
        sv.kv_append(h.bfloat16(), h.bfloat16(), kc, kc, slots)
    with pytest.raises(ValueError, match="positions"):
        sv.kv_append(h, h, kc, kc, slots, table=table)
    with pytest.raises(ValueError, match="slots"):
        sv.kv_append(h, h, kc, kc, slots.int())
    with pytest.raises(ValueError, match="q_out"):
        sv.kv_append(h, h, kc, kc, slots, q_out=kc[0])
    bt, kl, cu = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q = h.half()
    with pytest.raises(ValueError, match="fit"):
        sv.attention_paged(h, kc, kc, bt, kl, cu, 3)
    with pytest.raises(ValueError, match="fit"):
        sv.attention_paged(q[:, :1], kc, kc, bt, kl, cu, 3)
    with pytest.raises(ValueError, match="cu_q"):
        sv.attention_paged(q, kc, kc, bt, kl, cu[:1], 3)
    with pytest.raises(ValueError, match="block_table"):
        sv.attention_paged(q, kc, kc, bt.long(), kl, cu, 3)
    with pytest.raises(ValueError, match="CUDA"):
        sv.attention_paged(q, kc, kc, bt, kl, cu, 3)
