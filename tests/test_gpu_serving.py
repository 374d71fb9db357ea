"""The decoder-serving operators (rustgears_b200.serving) on the device.

The i8 product, the rotation and the append are defined operation by operation, so they
are compared bit for bit with numpy / the oracle.  Attention is compared with 64-bit
softmax attention under a bound derived from its roundings (see attention_bound)."""
import ctypes as C
import math

import numpy as np
import pytest

from oracle import oracle
from rustgears_b200 import _native

pytestmark = pytest.mark.gpu

DT = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


def dtype(torch, name):
    return getattr(torch, DT[name])


@pytest.fixture(scope="module")
def sv():
    from rustgears_b200 import serving
    return serving


@pytest.fixture(autouse=True)
def nothing_reported(gpu, sv):
    """Every test ends with clean error words."""
    yield
    sv.check()


# ---------------------------------------------------------------------------
# i8 product with a scale per token and channel
# ---------------------------------------------------------------------------
def quantized_rows(x):
    """The framework's quantizer with one scale per row, operation by operation in f32."""
    a = np.abs(x)
    amax = np.where(np.isnan(a), np.float32(0), a).max(axis=1).astype(np.float32)
    with np.errstate(all="ignore"):
        scale = np.where(amax < np.float32(1e-12), np.float32(1), amax / np.float32(127)).astype(np.float32)
        t = (x * (np.float32(1) / scale)[:, None]).astype(np.float32)
        r = np.trunc(t)
        r = r + np.sign(t) * (np.abs(t - r) >= 0.5)
    return np.where(np.isnan(r), 0, np.clip(r, -127, 127)).astype(np.int8), scale


def linear_reference(x, wq, w_scale, bias, act, param=0.0):
    q, sa = quantized_rows(x)
    acc = q.astype(np.int64) @ wq.astype(np.int64).T
    with np.errstate(all="ignore"):
        cs = (sa[:, None] * w_scale[None, :]).astype(np.float32)
        y = (acc.astype(np.float32) * cs).astype(np.float32)
        y = (y + (bias[None, :] if bias is not None else np.float32(0))).astype(np.float32)
    return oracle.activation(y, act, param)


def rounded(torch, y, name):
    return torch.from_numpy(np.ascontiguousarray(y)).to(dtype(torch, name))


def same(torch, got, want):
    """Bit-identical, any NaN equal to any NaN."""
    got, want = got.detach().cpu(), want.cpu()
    assert got.dtype == want.dtype and got.shape == want.shape
    gn, wn = torch.isnan(got), torch.isnan(want)
    assert torch.equal(gn, wn)
    bad = ~gn & (got != want)
    assert not bad.any(), f"{int(bad.sum())} of {got.numel()} differ, first at {bad.nonzero()[0].tolist()}: " \
                          f"{got[bad][0].item()} != {want[bad][0].item()}"


def linear_case(m, k, n, seed=0, outlier=True):
    r = np.random.default_rng(seed)
    x = r.standard_normal((m, k)).astype(np.float32)
    if outlier and m:
        x[m // 2] *= 100.0        # one loud token must not cost the others their bits
    wq = r.integers(-127, 128, (n, k)).astype(np.int8)
    return x, wq, (r.random(n).astype(np.float32) + 0.1) * 1e-3, r.standard_normal(n).astype(np.float32)


def run_linear(torch, sv, x, wq, sw, bias, act, xt, ot, **kw):
    ld = (x.shape[-1] + 15) // 16 * 16
    w = torch.zeros((wq.shape[0], ld), dtype=torch.int8, device="cuda")
    w[:, :wq.shape[1]] = torch.from_numpy(wq).cuda()
    xd = torch.from_numpy(x).to(dtype(torch, xt)).cuda()
    return sv.linear_i8_token(xd, w, torch.from_numpy(sw).cuda(),
                              bias=None if bias is None else torch.from_numpy(bias).cuda(), act=act,
                              out_dtype=dtype(torch, ot), **kw)


SHAPES = [(1, 1, 1), (1, 16, 8), (1, 1024, 2816), (2, 100, 33), (7, 4096, 130), (8, 513, 256), (9, 2000, 17),
          (16, 8192, 64), (17, 640, 1000), (33, 129, 500), (64, 1568, 128), (65, 4100, 96), (127, 256, 255),
          (128, 1024, 1024), (129, 1000, 257), (200, 9000, 40), (300, 384, 4096), (513, 2048, 520), (1000, 32, 16),
          (250, 3000, 700), (2100, 300, 130), (1700, 700, 2000), (20, 6000, 130), (100, 2048, 9000)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("xt,ot", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
def test_linear_shapes(gpu, sv, m, k, n, xt, ot):
    torch = gpu
    x, wq, sw, b = linear_case(m, k, n, seed=m + k + n)
    x = torch.from_numpy(x).to(dtype(torch, xt)).float().numpy()      # what the operator is given
    got = run_linear(torch, sv, x, wq, sw, b, "none", xt, ot)
    same(torch, got, rounded(torch, linear_reference(x, wq, sw, b, 0), ot))


@pytest.mark.parametrize("act,code,param", [("none", 0, 0.0), ("relu", 1, 0.0), ("sigmoid", 2, 0.0), ("tanh", 3, 0.0),
                                            ("gelu", 4, 0.0), ("leaky_relu", 5, 0.01), ("silu", 6, 0.0)])
@pytest.mark.parametrize("m,k,n,bias", [(3, 300, 90, True), (260, 512, 384, True), (260, 512, 250, False),
                                        (40, 512, 384, False), (512, 256, 512, False)])
def test_linear_activations(gpu, sv, act, code, param, m, k, n, bias):
    torch = gpu
    x, wq, sw, b = linear_case(m, k, n, seed=m + code, outlier=False)
    b = b if bias else None
    for ot in ("f32", "f16", "bf16"):
        got = run_linear(torch, sv, x, wq, sw, b, act, "f32", ot)
        want = linear_reference(x, wq, sw, b, code, param)
        if act in ("gelu", "silu") and ot != "f32":
            # the smooth ones are not bit-defined in 16 bits: one rounding of u, 2^-5 of it for
            # the f32 evaluations of both sides, the step of f16's subnormals, and what the f32
            # reference itself loses in 1 + tanh
            u = 2.0 ** (-11 if ot == "f16" else -8)
            pre = np.abs(linear_reference(x, wq, sw, b, 0)).astype(np.float64)
            off = np.abs(got.double().cpu().numpy() - want.astype(np.float64))
            assert (off <= u * (1 + 2.0 ** -5) * np.abs(want) + 2.0 ** -25 + 1.2e-7 * pre).all()
        else:
            same(torch, got, rounded(torch, want, ot))


def smooth_exact(act, y):
    """GELU (tanh form, the framework's f32 constant) and SiLU of f32 values in 64 bits."""
    y = y.astype(np.float64)
    a = -y if act == "silu" else -2.0 * float(np.float32(0.7978846)) * (y + 0.044715 * y ** 3)
    with np.errstate(over="ignore"):
        return y / (1.0 + np.exp(a))


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("ot", ["f16", "bf16"])
@pytest.mark.parametrize("m", [3, 40, 300])
def test_linear_smooth_activations_of_large_values(gpu, sv, act, ot, m):
    """Finite pre-activations of any size: the value itself (or the type's infinity) above, 0 below."""
    torch = gpu
    x, wq, _, _ = linear_case(m, 64, 48, seed=m, outlier=False)
    # |pre-activation| of a channel about 3 * 64 * 40 times its scale
    sw = np.logspace(-4, 34, 48).astype(np.float32)
    pre = linear_reference(x, wq, sw, None, 0)
    assert np.isfinite(pre).all() and pre.max() > 1e36 and pre.min() < -1e36
    got = run_linear(torch, sv, x, wq, sw, None, act, "f32", ot).double().cpu().numpy()
    want = smooth_exact(act, pre)
    assert (got[pre < -120.0] == 0).all()
    # one rounding to the type, 2^-5 of it for the f32 evaluation, the type's smallest step
    u, step, most = (2.0 ** -11, 2.0 ** -25, 65504.0) if ot == "f16" else (2.0 ** -8, 2.0 ** -134, 3.38e38)
    assert np.isposinf(got[want > most * (1 + 2 * u)]).all()
    near = (pre > (-9.0 if act == "gelu" else -80.0)) & (want < most * (1 - 2 * u))
    assert near.sum() > 10 and (np.abs(got - want)[near] <= (u * (1 + 2.0 ** -5) * np.abs(want) + step)[near]).all()


@pytest.mark.parametrize("act,lowest", [("gelu", -12.0), ("silu", -110.0)])
@pytest.mark.parametrize("ot", ["f16", "bf16"])
@pytest.mark.parametrize("m", [3, 40, 300])
def test_linear_smooth_activations_vanish_late(gpu, sv, act, lowest, ot, m):
    """The negative tails, down to the type's smallest numbers: rows of zeros leave the bias."""
    torch = gpu
    pre = np.concatenate([np.linspace(lowest, 1.0, 3000), -np.logspace(-44, 0, 500)]).astype(np.float32)
    x, wq, sw, _ = linear_case(m, 32, len(pre), seed=m, outlier=False)
    got = run_linear(torch, sv, x * 0, wq, sw, pre, act, "f32", ot).double().cpu().numpy()
    want = smooth_exact(act, pre)[None, :]
    # one rounding to the type, 2^-5 of it for the f32 evaluation; the type's smallest step
    u, step = (2.0 ** -11, 2.0 ** -24) if ot == "f16" else (2.0 ** -8, 2.0 ** -133)
    assert (np.abs(got - want) <= u * (1 + 2.0 ** -5) * np.abs(want) + step).all()


@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_linear_special_rows(gpu, sv, m):
    """Rows of zeros, tiny rows, NaN and infinities touch no other row."""
    torch = gpu
    x, wq, sw, b = linear_case(m, 200, 70, seed=9)
    rows = {0: 0.0, 1: 1e-20, 2: np.nan, 3: np.inf, 4: 3e38}
    for r, v in rows.items():
        if r < m:
            if r in (0, 1):
                x[r] = v
            else:
                x[r, 5] = v
    got = run_linear(torch, sv, x, wq, sw, b, "none", "f32", "f32")
    same(torch, got, rounded(torch, linear_reference(x, wq, sw, b, 0), "f32"))


@pytest.mark.parametrize("k", [7, 96, 1000])
@pytest.mark.parametrize("xt", ["f32", "f16", "bf16"])
def test_linear_strided_rows(gpu, sv, k, xt):
    """Rows of a wider tensor, at an odd offset and stride; leading dimensions kept."""
    torch = gpu
    x, wq, sw, b = linear_case(6, k, 48, seed=k)
    wide = torch.zeros((6, 2 * k + 5), dtype=dtype(torch, xt), device="cuda")
    wide[:, 3:3 + k] = torch.from_numpy(x).cuda()
    view = wide[:, 3:3 + k]
    x = view.float().cpu().numpy()
    w, ws = torch.zeros((48, (k + 15) // 16 * 16), dtype=torch.int8, device="cuda"), torch.from_numpy(sw).cuda()
    w[:, :k] = torch.from_numpy(wq).cuda()
    want = rounded(torch, linear_reference(x, wq, sw, None, 0), "f32")
    same(torch, sv.linear_i8_token(view, w, ws, out_dtype=torch.float32), want)
    three = sv.linear_i8_token(view.reshape(2, 3, k), w, ws, out_dtype=torch.float32)
    assert three.shape == (2, 3, 48)
    same(torch, three.view(6, 48), want)


@pytest.mark.parametrize("m,k", [(1, 4096), (4, 2048), (8, 1024), (3, 96), (40, 512), (300, 512)])
@pytest.mark.parametrize("xt", ["f32", "bf16"])
def test_linear_in_place(gpu, sv, m, k, xt):
    """out = x, and out one row further in the same memory, at every kernel's sizes."""
    torch = gpu
    x, wq, sw, b = linear_case(m, k, k, seed=m)
    w, ws, bias = torch.from_numpy(wq).cuda(), torch.from_numpy(sw).cuda(), torch.from_numpy(b).cuda()
    memory = torch.zeros((m + 1, k), dtype=dtype(torch, xt), device="cuda")
    x = torch.from_numpy(x).to(memory.dtype)
    want = rounded(torch, linear_reference(x.float().numpy(), wq, sw, b, 1), xt)
    for first in (0, 1):
        memory[:m] = x.cuda()
        out = memory[first:first + m]
        assert sv.linear_i8_token(memory[:m], w, ws, bias=bias, act="relu", out=out) is out
        same(torch, out, want)


def test_linear_wider_weight_rows(gpu, sv):
    """ld beyond k rounded up: the tail columns of x count as zeros."""
    torch = gpu
    x, wq, sw, b = linear_case(20, 100, 64, seed=2)
    w = torch.full((64, 256), 77, dtype=torch.int8, device="cuda")
    w[:, :100] = torch.from_numpy(wq).cuda()
    got = sv.linear_i8_token(torch.from_numpy(x).cuda(), w, torch.from_numpy(sw).cuda())
    same(torch, got, rounded(torch, linear_reference(x, wq, sw, None, 0), "f32"))


def test_calls_see_what_ran_just_before(gpu, sv):
    """Launches start early but read nothing before their predecessors are over: inputs, weights,
    lengths and caches rewritten right before each call, on one stream, eagerly and in a graph,
    and from another stream through an event."""
    torch = gpu
    n, h, d = 64, 4, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    table = sv.rope_table(512, d)
    kc, vc = (torch.zeros(8, 64, h, d, dtype=torch.float16, device="cuda") for _ in range(2))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    slots = torch.arange(n, device="cuda") + 64
    bt = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    data = [(torch.randn(n, 512, device="cuda", generator=g), torch.randn(3 * h * d, 512, device="cuda", generator=g))
            for _ in range(6)]
    x, w = torch.empty_like(data[0][0]), torch.empty_like(data[0][1])
    big = torch.zeros(1 << 26, device="cuda")
    kv_len = torch.zeros(1, dtype=torch.int32, device="cuda")

    def chain():
        kv_len.fill_(n)
        q, s = sv.quantize_weight_i8(w)
        y = sv.linear_i8_token(x, q, s, out_dtype=torch.float16).view(n, 3 * h, d)
        q = sv.kv_append(y[:, h:2 * h], y[:, 2 * h:], kc, vc, slots, positions=pos, table=table, q=y[:, :h])
        o = sv.attention_paged(q, kc, vc, bt, kv_len, cu, max_q_len=n, max_kv_len=n)
        one = sv.attention_paged(q[-1:], kc, vc, bt, kv_len, cu[:2] // n, max_q_len=1, max_kv_len=n)
        kc.zero_()
        vc.zero_()
        kv_len.zero_()
        return torch.cat([o, one])

    def load(i):
        big.add_(1.0)             # long enough that the launches behind it queue up
        x.copy_(data[i][0])
        w.copy_(data[i][1])

    want = []
    for i in range(6):
        load(i)
        torch.cuda.synchronize()
        want.append(chain())
        torch.cuda.synchronize()
    got = []
    for i in range(6):
        load(i)
        got.append(chain())
    for a, b in zip(got, want):
        same(torch, a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain()
    side = torch.cuda.Stream()
    for i in range(6):
        ready = torch.cuda.Event()
        with torch.cuda.stream(side):
            load(i)
            ready.record()
        torch.cuda.current_stream().wait_event(ready)
        if i % 2:
            graph.replay()
            copy = out.clone()
        else:
            copy = chain()
        side.wait_stream(torch.cuda.current_stream())
        same(torch, copy, want[i])


def test_mixed_batches_see_what_ran_just_before(gpu, sv):
    """Chunks beside decoding sequences: queries, keys, lengths and pages written right before the
    call, by an early launch and by copies, with other values in the same memory each time."""
    torch = gpu
    lens = [[(200, 640), (1, 600), (40, 90), (1, 33)], [(90, 500), (1, 610), (150, 150), (1, 7)]]
    heads, hk, d, page = 4, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(5)
    n = max(sum(q for q, _ in ls) for ls in lens)
    batches = [make_batch(torch, ls, heads, hk, d, torch.float16, page, "token", seed=i) for i, ls in enumerate(lens)]
    pages, width = max(b[1].shape[0] for b in batches), max(b[3].shape[1] for b in batches)
    kc, vc = (torch.zeros(pages, page, hk, d, dtype=torch.float16, device="cuda") for _ in range(2))
    q_out = torch.zeros(n, heads, d, dtype=torch.float16, device="cuda")
    bt = torch.zeros(4, width, dtype=torch.int32, device="cuda")
    kv_len, cu = (torch.zeros(k, dtype=torch.int32, device="cuda") for k in (4, 5))
    big = torch.zeros(1 << 26, device="cuda")
    table = sv.rope_table(8, d)
    pos = torch.arange(n, dtype=torch.int32, device="cuda") % 8
    none = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    raw = torch.randn(2, n, heads, d, device="cuda", generator=g)
    kv = torch.zeros(n, hk, d, device="cuda")

    def step(i):
        _, k, v, t, length, first = batches[i]
        kc[:k.shape[0]] = k
        vc[:v.shape[0]] = v
        bt[:, :t.shape[1]] = t
        kv_len.copy_(length)
        cu.copy_(first)
        sv.kv_append(kv, kv, kc, vc, none, positions=pos, table=table, q=raw[i], q_out=q_out)
        return sv.attention_paged(q_out, kc, vc, bt, kv_len, cu, max_q_len=200, max_kv_len=640)

    used = [sum(q for q, _ in ls) for ls in lens]
    want = []
    for i in range(2):
        torch.cuda.synchronize()
        want.append(step(i)[:used[i]].clone())
        torch.cuda.synchronize()
    got = []
    for r in range(12):
        if r % 4 == 0:
            big.add_(1.0)         # long enough that the launches behind it queue up
        got.append(step(r % 2))
    for r, o in enumerate(got):
        same(torch, o[:used[r % 2]], want[r % 2])


def test_linear_kernel_level_calls(gpu, sv):
    """Quantizer and product called apart, the output a column block of a wider tensor."""
    torch, L = gpu, _native.lib()
    x, wq, sw, b = linear_case(150, 320, 200, seed=4)
    q, s = sv.quantize_token_i8(torch.from_numpy(x).cuda())
    qr, sr = quantized_rows(x)
    assert np.array_equal(q.cpu().numpy()[:, :320], qr) and np.array_equal(s.cpu().numpy(), sr)
    w, wsc, bias = torch.from_numpy(wq).cuda(), torch.from_numpy(sw).cuda(), torch.from_numpy(b).cuda()
    err = torch.zeros(2, dtype=torch.int32, device="cuda")
    for name, n0 in (("f32", 0), ("f16", 0), ("bf16", 3)):
        wide = torch.full((150, 260), 5.0, dtype=dtype(torch, name), device="cuda")
        view = wide[:, n0:n0 + 200]
        _native.check(L.rg_gemm_i8_token(q.data_ptr(), s.data_ptr(), w.data_ptr(), wsc.data_ptr(), 150, 200, 320,
                                         bias.data_ptr(), 1, C.c_float(0), view.data_ptr(),
                                         {"f32": 0, "f16": 1, "bf16": 2}[name], 260, err.data_ptr(), None))
        torch.cuda.synchronize()
        same(torch, view.contiguous(), rounded(torch, linear_reference(x, wq, sw, b, 1), name))
        assert (wide[:, :n0] == 5).all() and (wide[:, n0 + 200:] == 5).all()
    assert err.tolist() == [0, 0]


def test_quantized_weight(gpu, sv):
    torch = gpu
    w = torch.randn(33, 50, device="cuda")
    q, s = sv.quantize_weight_i8(w)
    qr, sr = quantized_rows(w.cpu().numpy())
    assert q.shape == (33, 64) and np.array_equal(q.cpu().numpy()[:, :50], qr) and (q[:, 50:] == 0).all()
    assert np.array_equal(s.cpu().numpy(), sr)


# ---------------------------------------------------------------------------
# rotary positions and the append
# ---------------------------------------------------------------------------
def table_reference(positions, rot, base=10000.0, kind="plain", factor=1.0, gain=1.0, old=0, fast=32.0, slow=1.0):
    i = np.arange(rot // 2, dtype=np.float64)
    f = base ** (-2 * i / rot)
    if kind == "linear":
        f = f / factor
    if kind == "bands":
        dim = lambda turns: rot * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(0, math.floor(dim(fast))), min(rot - 1, math.ceil(dim(slow)))
        ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        f = f / factor * ramp + f * (1 - ramp)
    a = np.arange(positions)[:, None] * f
    return np.concatenate([np.cos(a) * gain, np.sin(a) * gain], 1)


@pytest.mark.parametrize("rot,kw", [(2, {}), (64, {}), (128, dict(base=500000.0)),
                                    (96, dict(kind="linear", factor=4.0)),
                                    (128, dict(kind="bands", factor=8.0, old=4096, gain=1.2)),
                                    (64, dict(kind="bands", factor=2.0, old=1024, fast=16.0, slow=2.0))])
def test_rope_table(gpu, sv, rot, kw):
    n = 20001
    names = dict(kind="scaling", old="old_context", fast="fast_turns", slow="slow_turns")
    t = sv.rope_table(n, rot, **{names.get(k, k): v for k, v in kw.items()}).cpu().numpy()
    ref = table_reference(n, rot, **kw)
    # one rounding to f32 of a value of magnitude <= gain, and 64-bit angles up to 2e4
    assert np.abs(t - ref).max() <= 2.0 ** -24 * 1.2 + 1e-10


def rotate_reference(x, positions, table, inter):
    """f32, operation by operation: two products and one sum per element."""
    rot = table.shape[1]
    c, s = table[positions][:, None, :rot // 2], table[positions][:, None, rot // 2:]
    y = x.copy()
    i0, i1 = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if inter else (np.arange(rot // 2), np.arange(rot // 2, rot))
    a, b = x[..., i0], x[..., i1]
    y[..., i0] = a * c - b * s
    y[..., i1] = b * c + a * s
    return y


ROPE = [(1, 32, 128, 128), (1, 1, 2, 2), (3, 5, 64, 16), (7, 3, 96, 24), (33, 4, 80, 40), (5, 2, 10, 6),
        (300, 8, 128, 64), (17, 1, 256, 256), (2, 70, 256, 64)]


@pytest.mark.parametrize("n,h,d,rot", ROPE)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("xt", ["f32", "f16", "bf16"])
def test_rope(gpu, sv, n, h, d, rot, inter, xt):
    torch = gpu
    r = np.random.default_rng(n + d)
    x = torch.from_numpy(r.standard_normal((n, h, d)).astype(np.float32)).to(dtype(torch, xt))
    pos = r.integers(0, 5000, n).astype(np.int32)
    table = sv.rope_table(5000, rot)
    want = rounded(torch, rotate_reference(x.float().numpy(), pos, table.cpu().numpy(), inter), xt)
    xd, pd = x.cuda(), torch.from_numpy(pos).cuda()
    same(torch, sv.rope(xd, pd, table, interleaved=inter), want)
    # a view of a wider tensor at an odd offset, rotated in place
    wide = torch.zeros((n, h * d + 7), dtype=x.dtype, device="cuda")
    view = wide[:, 5:5 + h * d].view(n, h, d)
    view.copy_(xd)
    assert sv.rope(view, pd, table, interleaved=inter, out=view) is view
    same(torch, view.contiguous(), want)
    assert (wide[:, :5] == 0).all() and (wide[:, 5 + h * d:] == 0).all()
    # heads outermost
    turned = xd.transpose(0, 1).contiguous().transpose(0, 1)
    same(torch, sv.rope(turned, pd, table, interleaved=inter), want)


def make_cache(torch, pages, page, heads, dim, dt, layout, fill=float("nan")):
    shape = (pages, page, heads, dim) if layout == "token" else (pages, heads, page, dim)
    t = torch.full(shape, fill, dtype=dt, device="cuda")
    return t if layout == "token" else t.transpose(1, 2)


APPEND = [  # tokens, heads, kv_heads, dim, rot, page
    (1, 32, 8, 128, 128, 16), (5, 4, 4, 64, 32, 16), (64, 8, 2, 128, 128, 1), (130, 6, 3, 96, 24, 24),
    (9, 1, 1, 10, 4, 7), (300, 14, 2, 64, 64, 64), (40, 2, 1, 256, 64, 128)]


@pytest.mark.parametrize("n,h,hk,d,rot,page", APPEND)
@pytest.mark.parametrize("xt,ct", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("layout,inter", [("token", False), ("head", True)])
def test_append(gpu, sv, n, h, hk, d, rot, page, xt, ct, layout, inter):
    torch = gpu
    r = np.random.default_rng(n + d)
    qkv = torch.from_numpy(r.standard_normal((n, (h + 2 * hk) * d)).astype(np.float32)).to(dtype(torch, xt)).cuda()
    q = qkv[:, :h * d].view(n, h, d)
    k = qkv[:, h * d:(h + hk) * d].view(n, hk, d)
    v = qkv[:, (h + hk) * d:].view(n, hk, d)
    pages = n // page + 3
    slots = r.permutation(pages * page)[:n].astype(np.int64)
    if n > 2:
        slots[1] = -1            # padding
    pos = r.integers(0, 3000, n).astype(np.int32)
    table = sv.rope_table(3000, rot)
    kc = make_cache(torch, pages, page, hk, d, dtype(torch, ct), layout)
    vc = make_cache(torch, pages, page, hk, d, dtype(torch, ct), layout)
    got_q = sv.kv_append(k, v, kc, vc, torch.from_numpy(slots).cuda(), positions=torch.from_numpy(pos).cuda(),
                         table=table, interleaved=inter, q=q)
    tab = table.cpu().numpy()
    rot_of = lambda t: rounded(torch, rotate_reference(t.float().cpu().numpy(), pos, tab, inter), ct)  # noqa: E731
    same(torch, got_q, rot_of(q))
    for cache, values in ((kc, rot_of(k)), (vc, v.to(dtype(torch, ct)).cpu())):
        want = torch.full((pages * page, hk, d), float("nan"), dtype=dtype(torch, ct))
        keep = slots >= 0
        want[torch.from_numpy(slots[keep])] = values[torch.from_numpy(np.nonzero(keep)[0])]
        same(torch, cache.reshape(pages * page, hk, d), want)
    # without a table: stored as they are, q not asked for
    assert sv.kv_append(k, v, kc, vc, torch.from_numpy(slots).cuda()) is None
    got = kc.reshape(pages * page, hk, d)[torch.from_numpy(slots[slots >= 0]).cuda()]
    same(torch, got, k[torch.from_numpy(np.nonzero(slots >= 0)[0]).cuda()].to(dtype(torch, ct)))


def test_append_reports_indices_out_of_range(gpu, sv):
    """A slot or position out of range is skipped and reported, the other tokens are stored."""
    torch = gpu
    k = torch.randn(4, 2, 64, device="cuda").half()
    kc, vc = (make_cache(torch, 3, 8, 2, 64, torch.float16, "token", 0.0) for _ in range(2))
    table = sv.rope_table(10, 64)
    slots = torch.tensor([0, 24, 2, 3], dtype=torch.int64, device="cuda")
    pos = torch.tensor([0, 1, 10, 0], dtype=torch.int32, device="cuda")
    sv.kv_append(k, k, kc, vc, slots, positions=pos, table=table)
    with pytest.raises(_native.RgError, match="slot") as e:
        sv.check()
    assert e.value.status == _native.RG_ERR_INVALID_ARG
    sv.check()                                  # cleared
    flat = vc.reshape(24, 2, 64)
    same(torch, flat[0], k[0])
    same(torch, flat[3], k[3])
    assert (flat[1:3] == 0).all() and (flat[4:] == 0).all()
    x = torch.randn(2, 1, 64, device="cuda")
    bad = torch.tensor([-1, 3], dtype=torch.int32, device="cuda")
    out = torch.full_like(x, 7.0)
    sv.rope(x, bad, table, out=out)
    assert (out[0] == 7).all() and not (out[1] == 7).any()
    with pytest.raises(_native.RgError):
        sv.check()


# ---------------------------------------------------------------------------
# attention over the paged cache
# ---------------------------------------------------------------------------
def make_batch(torch, lens, heads, kv_heads, dim, dt, page, layout, seed=0, mul=1.0):
    """A batch whose unused cache cells (page tails, spare pages) hold NaN and infinities."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-kv // page) for _, kv in lens]
    pages = sum(need) + 2
    kc, vc = (make_cache(torch, pages, page, kv_heads, dim, dt, layout) for _ in range(2))
    vc[-1] = float("inf")
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).cpu().tolist()
    table = torch.full((len(lens), max(max(need), 1)), -7, dtype=torch.int32)
    for b, (_, kv) in enumerate(lens):
        mine, order = order[:need[b]], order[need[b]:]
        table[b, :need[b]] = torch.tensor(mine, dtype=torch.int32)
        for c in (kc, vc):
            vals = (torch.randn((kv, kv_heads, dim), device="cuda", generator=g) * mul).to(dt)
            for j, pg in enumerate(mine):
                part = vals[j * page:(j + 1) * page]
                c[pg, :part.shape[0]] = part
    n = sum(q for q, _ in lens)
    q = (torch.randn((n, heads, dim), device="cuda", generator=g) * mul).to(dt)
    kv_len = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda")
    cu = torch.tensor(np.cumsum([0] + [ql for ql, _ in lens]), dtype=torch.int32, device="cuda")
    return q, kc, vc, table.cuda(), kv_len, cu


def attention_reference(torch, q, kc, vc, table, lens, scale, causal):
    """(output, sum p |v|, sum |v|) in 64 bits."""
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    spread, total = torch.zeros_like(out), torch.zeros_like(out)
    page, hk = kc.shape[1], kc.shape[2]
    at = 0
    for b, (ql, kv) in enumerate(lens):
        pg = table[b, :-(-kv // page)].long()
        k = kc[pg].reshape(-1, *kc.shape[2:])[:kv].double()
        v = vc[pg].reshape(-1, *vc.shape[2:])[:kv].double()
        rep = q.shape[1] // hk
        s = torch.einsum("qhd,khd->hqk", q[at:at + ql].double(), k.repeat_interleave(rep, 1)) * scale
        if causal:
            i = torch.arange(ql, device="cuda")[:, None] + (kv - ql)
            s = s.masked_fill(torch.arange(kv, device="cuda")[None, :] > i, -math.inf)
        p = torch.nan_to_num(torch.softmax(s, -1)) if kv else s
        vr = v.repeat_interleave(rep, 1)
        out[at:at + ql] = torch.einsum("hqk,khd->qhd", p, vr)
        spread[at:at + ql] = torch.einsum("hqk,khd->qhd", p, vr.abs())
        total[at:at + ql] = vr.abs().sum(0)
        at += ql
    return out, spread, total


def attention_bound(q, ref, spread, total, score_error):
    """u |o| for the output's rounding, (u + e) sum p |v| for the probabilities' rounding to the
    cache's type and the f32 error e of a score, and f16's smallest step for tiny ones."""
    u = 2.0 ** -8 if q.dtype.itemsize == 2 and "bfloat16" in str(q.dtype) else 2.0 ** -11
    return u * ref.abs() + (u + score_error) * spread + 2.0 ** -25 * total + 1e-30


def check_attention(torch, sv, lens, heads, kv_heads, dim, dt, page, layout, causal=True, scale=None, seed=0, mul=1.0,
                    slack=0):
    q, kc, vc, table, kv_len, cu = make_batch(torch, lens, heads, kv_heads, dim, dt, page, layout, seed, mul)
    most_q, most_kv = max(ql for ql, _ in lens), max(kv for _, kv in lens)
    room = table.shape[1] * page
    got = sv.attention_paged(q, kc, vc, table, kv_len, cu, max_q_len=most_q + slack,
                             max_kv_len=min(most_kv + slack, room), scale=scale, causal=causal)
    sc = 1.0 / math.sqrt(dim) if scale is None else scale
    ref, spread, total = attention_reference(torch, q, kc, vc, table, lens, sc, causal)
    # f32 score of dim products: dim 2^-24 sum |q k| scale, |q k| <= 16 mul^2 nearly always on
    # average 0.64; twice for the difference to the maximum
    err = 2 * dim * 2.0 ** -24 * dim * mul * mul * abs(sc) + 1e-5
    off = (got.double() - ref).abs() - attention_bound(q, ref, spread, total, err)
    assert not torch.isnan(got).any()
    assert off.max().item() <= 0, f"off by {off.max().item()} at {(off == off.max()).nonzero()[0].tolist()}"
    for ql, kv, at in [(ql, kv, int(cu[b])) for b, (ql, kv) in enumerate(lens)]:
        empty = ql if kv == 0 else max(0, ql - kv) if causal else 0
        assert (got[at:at + empty] == 0).all()
    return got


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("page,layout", [(16, "token"), (128, "head"), (24, "token"), (1, "head")])
def test_attention_decode(gpu, sv, dim, dt, page, layout):
    lens = [(1, 1), (1, 2), (1, 31), (1, 64), (1, 65), (1, 700), (1, 1025)]
    for heads, kv_heads in ((8, 2), (3, 3), (7, 1), (16, 1), (40, 2)):
        check_attention(gpu, sv, lens, heads, kv_heads, dim, dtype(gpu, dt), page, layout, seed=heads)


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("page,layout", [(8, "head"), (64, "token"), (48, "head"), (256, "token")])
def test_attention_chunks(gpu, sv, dim, dt, page, layout):
    lens = [(5, 5), (1, 130), (33, 200), (128, 128), (129, 513), (200, 1000), (3, 64)]
    for heads, kv_heads in ((4, 2), (2, 2), (6, 2)):
        check_attention(gpu, sv, lens, heads, kv_heads, dim, dtype(gpu, dt), page, layout, seed=heads)


@pytest.mark.parametrize("lens", [[(300, 300)], [(257, 1300), (1, 40)], [(64, 64)], [(2, 3000)], [(17, 17)] * 20,
                                  [(1, 1)], [(700, 701)]])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 8, 2), (64, 4, 4), (128, 5, 5), (64, 12, 4)])
def test_attention_lengths(gpu, sv, lens, dim, heads, kv_heads):
    check_attention(gpu, sv, lens, heads, kv_heads, dim, gpu.bfloat16, 32, "token", seed=len(lens))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_empty_rows_and_sequences(gpu, sv, dim, causal):
    """No keys, fewer keys than queries (the first queries see none), no queries."""
    lens = [(3, 0), (0, 50), (10, 4), (0, 0), (200, 130), (1, 0), (150, 1)]
    check_attention(gpu, sv, lens, 4, 2, dim, gpu.float16, 16, "token", causal=causal)
    check_attention(gpu, sv, [(2, 0), (1, 0)], 4, 2, dim, gpu.float16, 16, "token", causal=causal)


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_not_causal_scaled(gpu, sv, dim):
    lens = [(70, 333), (1, 90), (300, 77)]
    check_attention(gpu, sv, lens, 6, 3, dim, gpu.bfloat16, 64, "head", causal=False, scale=0.3)
    check_attention(gpu, sv, lens, 6, 3, dim, gpu.bfloat16, 64, "head", causal=True, scale=-0.05)
    check_attention(gpu, sv, lens, 6, 3, dim, gpu.float16, 64, "head", causal=True, scale=0.0)


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_loud_scores(gpu, sv, dim):
    """Scores of a few hundred: the running maximum carries the sum."""
    check_attention(gpu, sv, [(1, 900), (150, 700), (40, 333)], 4, 1, dim, gpu.float16, 16, "token", mul=6.0, scale=0.1)


def test_attention_loose_bounds_and_wide_table(gpu, sv):
    """max_q_len and max_kv_len above the real lengths; a block table that is a view."""
    torch = gpu
    lens = [(1, 300), (20, 77)]
    check_attention(torch, sv, lens, 8, 2, 128, torch.bfloat16, 16, "token", slack=3)
    q, kc, vc, table, kv_len, cu = make_batch(torch, lens, 8, 2, 128, torch.bfloat16, 16, "token")
    a = sv.attention_paged(q, kc, vc, table, kv_len, cu, max_q_len=20, max_kv_len=300)
    wide = torch.full((2, 400), -3, dtype=torch.int32, device="cuda")
    wide[:, 9:9 + table.shape[1]] = table
    b = sv.attention_paged(q, kc, vc, wide[:, 9:], kv_len, cu, max_q_len=2000)
    # another bound may split the keys elsewhere: equal up to the probabilities' rounding
    assert (a.float() - b.float()).abs().max().item() <= 2.0 ** -6


def test_attention_strided_q_and_out(gpu, sv):
    """q a slice of a fused projection's output, out heads-outermost."""
    torch = gpu
    for lens in ([(1, 200), (1, 33)], [(150, 200), (7, 90)]):
        q, kc, vc, table, kv_len, cu = make_batch(torch, lens, 6, 2, 64, torch.float16, 32, "head", seed=1)
        most = max(a for a, _ in lens)
        want = sv.attention_paged(q, kc, vc, table, kv_len, cu, max_q_len=most, max_kv_len=200)
        wide = torch.full((q.shape[0], 8 + 6 * 64 + 16), float("nan"), dtype=torch.float16, device="cuda")
        view = wide[:, 8:8 + 384].view(-1, 6, 64)
        view.copy_(q)
        out = torch.empty((6, q.shape[0], 64), dtype=torch.float16, device="cuda").transpose(0, 1)
        got = sv.attention_paged(view, kc, vc, table, kv_len, cu, max_q_len=most, max_kv_len=200, out=out)
        assert got is out
        same(torch, out.contiguous(), want)


@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("lens", [[(1, 900), (1, 333)], [(200, 700), (1, 450)], [(300, 1000)]])
def test_attention_cache_of_other_strides(gpu, sv, dim, lens):
    """Caches that are views: padded heads, tokens and pages; keys and values of one page side by side."""
    torch = gpu
    q, kc, vc, table, kv_len, cu = make_batch(torch, lens, 6, 3, dim, torch.bfloat16, 16, "token", seed=8)
    most = dict(max_q_len=max(a for a, _ in lens), max_kv_len=max(b for _, b in lens))
    want = sv.attention_paged(q, kc, vc, table, kv_len, cu, **most)
    n = kc.shape[0]
    kp, vp = (torch.full((n, 19, 4, dim + 8), float("nan"), dtype=q.dtype, device="cuda")[:, 2:18, :3, :dim] for _ in range(2))
    both = torch.full((n, 2, 16, 3, dim), float("nan"), dtype=q.dtype, device="cuda")
    turned = torch.full((3, n, 2, 16, dim), float("nan"), dtype=q.dtype, device="cuda")
    for k, v in ((kp, vp), (both[:, 0], both[:, 1]), (turned[:, :, 0].permute(1, 2, 0, 3), turned[:, :, 1].permute(1, 2, 0, 3))):
        k.copy_(kc)
        v.copy_(vc)
        same(torch, sv.attention_paged(q, k, v, table, kv_len, cu, **most), want)


def test_attention_repeats_bit_for_bit(gpu, sv):
    torch = gpu
    for lens in ([(1, 5000)], [(300, 900), (1, 2000), (77, 77)]):
        args = make_batch(torch, lens, 16, 4, 128, torch.bfloat16, 64, "token", seed=3)
        most = max(a for a, _ in lens)
        first = sv.attention_paged(*args, max_q_len=most, max_kv_len=5000 if most == 1 else 2000)
        for _ in range(3):
            same(torch, sv.attention_paged(*args, max_q_len=most, max_kv_len=5000 if most == 1 else 2000), first)


def test_attention_reports_lengths_and_pages_out_of_range(gpu, sv):
    """A bad page's keys count as zeros, a bad sequence is left alone; the others are right."""
    torch = gpu
    for most, dim in ((1, 128), (200, 128), (200, 64), (1, 256)):
        lens = [(most, 400), (most, 300), (most, 350)]
        q, kc, vc, table, kv_len, cu = make_batch(torch, lens, 4, 2, dim, torch.bfloat16, 16, "token", seed=5)
        good = sv.attention_paged(q, kc, vc, table, kv_len, cu, max_q_len=most, max_kv_len=400)
        bad = table.clone()
        bad[1, 3] = kc.shape[0]
        bad[1, 5] = -1
        got = sv.attention_paged(q, kc, vc, bad, kv_len, cu, max_q_len=most, max_kv_len=400)
        with pytest.raises(_native.RgError, match="page"):
            sv.check()
        same(torch, got[:most], good[:most])
        same(torch, got[2 * most:], good[2 * most:])
        assert torch.isfinite(got).all()
        long = kv_len.clone()
        long[1] = 401
        out = torch.full_like(q, 3.0)
        sv.attention_paged(q, kc, vc, table, long, cu, max_q_len=most, max_kv_len=400, out=out)
        with pytest.raises(_native.RgError, match="length"):
            sv.check()
        same(torch, out[:most], good[:most])
        same(torch, out[2 * most:], good[2 * most:])
        assert (out[most:2 * most] == 3).all()


@pytest.mark.parametrize("dim,heads", [(64, 4), (128, 160)])
def test_attention_without_tokens_by_its_bound(gpu, sv, dim, heads):
    """max_q_len 0 is a bound like any other: sequences that have tokens are reported, empty ones
    (all rows padding) are not; no row is written."""
    torch = gpu
    q, kc, vc, table, kv_len, cu = make_batch(torch, [(3, 40), (2, 9)], heads, 2, dim, torch.bfloat16, 16, "token")
    out = torch.full_like(q, 3.0)
    sv.attention_paged(q, kc, vc, table, kv_len, cu, max_q_len=0, max_kv_len=40, out=out)
    with pytest.raises(_native.RgError, match="length"):
        sv.check()
    sv.attention_paged(q, kc, vc, table, kv_len, cu * 0, max_q_len=0, max_kv_len=40, out=out)
    sv.check()
    assert (out == 3).all()


def test_attention_leaves_rows_of_no_sequence_alone(gpu, sv):
    """Padding before and behind the sequences' tokens is not written."""
    torch = gpu
    for most in (1, 150):
        lens = [(most, 200), (most, 170)]
        q, kc, vc, table, kv_len, cu = make_batch(torch, lens, 4, 2, 64, torch.float16, 16, "token", seed=4)
        want = sv.attention_paged(q, kc, vc, table, kv_len, cu, max_q_len=most, max_kv_len=200)
        wide = torch.full((q.shape[0] + 7, 4, 64), 5.0, dtype=q.dtype, device="cuda")
        wide[2:2 + 2 * most] = q
        out = torch.full_like(wide, 3.0)
        sv.attention_paged(wide, kc, vc, table, kv_len, cu + 2, max_q_len=most, max_kv_len=200, out=out)
        same(torch, out[2:2 + 2 * most], want)
        assert (out[:2] == 3).all() and (out[2 + 2 * most:] == 3).all()


def test_attention_cache_beyond_32_bit_offsets(gpu, sv):
    """Pages whose element offset exceeds 2^32 (the same tensor serves as keys and values)."""
    torch = gpu
    pages, page, hk, d = 17000, 256, 8, 128            # 4.46e9 elements
    cache = torch.empty((pages, page, hk, d), dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([pages - 1, 3, pages - 2, 9000], dtype=torch.int32, device="cuda")
    k = torch.randn((1000, hk, d), device="cuda").bfloat16()
    i = torch.arange(1000, device="cuda")
    slots = ids.long()[i // page] * page + i % page
    sv.kv_append(k, k, cache, cache, slots)
    for ql in (1, 130):
        q = torch.randn((ql, 16, d), device="cuda").bfloat16()
        kv_len = torch.tensor([1000], dtype=torch.int32, device="cuda")
        cu = torch.tensor([0, ql], dtype=torch.int32, device="cuda")
        got = sv.attention_paged(q, cache, cache, ids[None], kv_len, cu, max_q_len=ql, max_kv_len=1000)
        small = cache[ids.long()]
        ref, spread, total = attention_reference(torch, q, small, small, torch.arange(4, device="cuda")[None],
                                                 [(ql, 1000)], 1 / math.sqrt(d), True)
        assert ((got.double() - ref).abs() <= attention_bound(q, ref, spread, total, 1e-3)).all()


# ---------------------------------------------------------------------------
# streams and graphs
# ---------------------------------------------------------------------------
def test_other_streams_and_graph_capture(gpu, sv):
    """A block's four calls on a side stream, captured and replayed on changed inputs."""
    torch = gpu
    n, h, hk, d, page = 3, 4, 2, 64, 16
    x = torch.randn(n, 256, device="cuda").bfloat16()
    w, ws = sv.quantize_weight_i8(torch.randn((h + 2 * hk) * d, 256, device="cuda") * 0.05)
    table = sv.rope_table(64, d)
    kc, vc = (make_cache(torch, 8, page, hk, d, torch.bfloat16, "token", 0.0) for _ in range(2))
    pos = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    slots = torch.tensor([32, 33, 34], dtype=torch.int64, device="cuda")
    bt = torch.tensor([[2]], dtype=torch.int32, device="cuda")
    kv_len = torch.tensor([3], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")

    def block():
        y = sv.linear_i8_token(x, w, ws).view(n, h + 2 * hk, d)
        q = sv.kv_append(y[:, h:h + hk], y[:, h + hk:], kc, vc, slots, positions=pos, table=table, q=y[:, :h])
        return sv.attention_paged(q, kc, vc, bt, kv_len, cu, max_q_len=3, max_kv_len=3)

    want = block()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = block()
    side.synchronize()
    same(torch, other, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = block()
    x.copy_(torch.randn(n, 256, device="cuda").bfloat16())
    g.replay()
    torch.cuda.synchronize()
    replayed = out.clone()
    same(torch, replayed, block())


@pytest.mark.parametrize("m", [40, 300, 1500])
def test_linear_bounded_waits_are_reported(gpu, sv, m):
    """Without operand loads the product's waits run out: reported, and the next call is right."""
    torch, L = gpu, _native.lib()
    x, wq, sw, b = linear_case(m, 512, 400, seed=1)
    try:
        L.rg_debug_set_tc_wait(1000000, 1)
        run_linear(torch, sv, x, wq, sw, b, "none", "f32", "f32")
        with pytest.raises(_native.RgError, match="bounded wait") as e:
            sv.check()
        assert e.value.status == _native.RG_ERR_TIMEOUT
    finally:
        L.rg_debug_set_tc_wait(0, 0)
    got = run_linear(torch, sv, x, wq, sw, b, "none", "f32", "f32")
    same(torch, got, rounded(torch, linear_reference(x, wq, sw, b, 0), "f32"))


@pytest.mark.parametrize("act,code", [("none", 0), ("gelu", 4)])
@pytest.mark.parametrize("k", [256, 4096])
def test_linear_few_tokens_leave_together(gpu, sv, k, act, code):
    """9 to 96 tokens, K whole and split: a warp whose wait runs out leaves as one, also where the
    f32 GELU votes inside the loop over the tokens."""
    torch, L = gpu, _native.lib()
    x, wq, sw, b = linear_case(50, k, 300, seed=2)
    for wait in (1, 1000, 1000000):
        try:
            L.rg_debug_set_tc_wait(wait, 1)
            run_linear(torch, sv, x, wq, sw, b, act, "f32", "f32")
            with pytest.raises(_native.RgError, match="bounded wait"):
                sv.check()
        finally:
            L.rg_debug_set_tc_wait(0, 0)
    got = run_linear(torch, sv, x, wq, sw, b, act, "f32", "f32")
    same(torch, got, rounded(torch, linear_reference(x, wq, sw, b, code), "f32"))


@pytest.mark.parametrize("m,k,n", [(64, 4096, 400), (40, 256, 400), (96, 9000, 300)])
def test_linear_given_up_with_copies_on_their_way(gpu, sv, m, k, n):
    """The products are given up while, or after, the last copies are issued: those land before
    their blocks leave, the call is reported, and calls that take over their SMs are right."""
    torch, L = gpu, _native.lib()
    x, wq, sw, b = linear_case(m, k, n, seed=3)
    want = rounded(torch, linear_reference(x, wq, sw, b, 0), "f32")
    same(torch, run_linear(torch, sv, x, wq, sw, b, "none", "f32", "f32"), want)
    for _ in range(3):
        try:
            L.rg_debug_set_tc_wait(1000000, 2)
            run_linear(torch, sv, x, wq, sw, b, "none", "f32", "f32")
        finally:
            L.rg_debug_set_tc_wait(0, 0)
        got = run_linear(torch, sv, x, wq, sw, b, "none", "f32", "f32")
        with pytest.raises(_native.RgError, match="bounded wait") as e:
            sv.check()
        assert e.value.status == _native.RG_ERR_TIMEOUT
        same(torch, got, want)


def test_attention_bounded_waits_are_reported(gpu, sv):
    """Without loads the chunk kernel's waits run out: reported, and the next call is right."""
    torch, L = gpu, _native.lib()
    args = make_batch(torch, [(100, 300)], 4, 2, 64, torch.float16, 16, "token")
    try:
        L.rg_debug_set_tc_wait(1000000, 1)
        sv.attention_paged(*args, max_q_len=100, max_kv_len=300)
        with pytest.raises(_native.RgError, match="bounded wait") as e:
            sv.check()
        assert e.value.status == _native.RG_ERR_TIMEOUT
    finally:
        L.rg_debug_set_tc_wait(0, 0)
    check_attention(torch, sv, [(100, 300)], 4, 2, 64, torch.float16, 16, "token")


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("lens", [[(100, 300)], [(600, 5000)], [(300, 1500), (1, 700)]])
def test_attention_given_up_with_copies_on_their_way(gpu, sv, dim, page, lens):
    """The products of chunks are given up while, or after, the last copies are issued: those land
    before their blocks leave, the call is reported, and the call that takes over their SMs is right."""
    torch, L = gpu, _native.lib()
    args = make_batch(torch, lens, 4, 2, dim, torch.bfloat16, page, "token")
    most = dict(max_q_len=max(a for a, _ in lens), max_kv_len=max(b for _, b in lens))
    want = sv.attention_paged(*args, **most)
    for _ in range(3):
        try:
            L.rg_debug_set_tc_wait(1000000, 2)
            sv.attention_paged(*args, **most)
        finally:
            L.rg_debug_set_tc_wait(0, 0)
        got = sv.attention_paged(*args, **most)
        with pytest.raises(_native.RgError, match="bounded wait") as e:
            sv.check()
        assert e.value.status == _native.RG_ERR_TIMEOUT
        same(torch, got, want)
    check_attention(torch, sv, lens, 4, 2, dim, torch.bfloat16, page, "token")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 384])
def test_attention_long_chunks(gpu, sv, dim, page):
    """Several tiles of rows and keys, pages of every size the tensor-core kernel takes."""
    for lens, heads, kv_heads in (([(700, 2100), (90, 640), (1, 1500)], 6, 2), ([(333, 333), (257, 1024)], 3, 3),
                                  ([(60, 4000)], 16, 2)):
        check_attention(gpu, sv, lens, heads, kv_heads, dim, gpu.bfloat16, page, "head" if page < 64 else "token",
                        seed=page)


def test_check_loses_no_report(gpu, sv, monkeypatch):
    """What another caller's kernel reports while a check is under way is raised by the next one."""
    torch = gpu
    table = sv.rope_table(4, 64)
    x, far = torch.zeros(1, 1, 64, device="cuda"), torch.tensor([99], dtype=torch.int32, device="cuda")
    read = torch.Tensor.tolist

    def read_then_report(t):
        host = read(t)
        monkeypatch.setattr(torch.Tensor, "tolist", read)
        sv.rope(x, far, table)
        torch.cuda.synchronize()
        return host

    sv.rope(x, far, table)
    monkeypatch.setattr(torch.Tensor, "tolist", read_then_report)
    for _ in range(2):
        with pytest.raises(_native.RgError, match="position"):
            sv.check()
    sv.check()


def test_zero_sizes(gpu, sv):
    torch = gpu
    w, ws = sv.quantize_weight_i8(torch.randn(8, 32, device="cuda"))
    assert sv.linear_i8_token(torch.empty(0, 32, device="cuda"), w, ws).shape == (0, 8)
    table = sv.rope_table(4, 64)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert sv.rope(torch.empty(0, 3, 64, device="cuda"), none, table).shape == (0, 3, 64)
    kc = make_cache(torch, 2, 4, 1, 64, torch.float16, "token", 0.0)
    e = torch.empty(0, 1, 64, device="cuda")
    assert sv.kv_append(e, e, kc, kc, none.long(), q=e).shape == (0, 1, 64)
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = sv.attention_paged(e.half(), kc, kc, torch.empty((0, 1), dtype=torch.int32, device="cuda"), none, one,
                             max_q_len=1)
    assert out.shape == (0, 1, 64)


# ---------------------------------------------------------------------------
# the block, the cache's bookkeeping and the example
# ---------------------------------------------------------------------------
def test_decoder_attention_block(gpu, sv):
    """The block against its parts: exact projections, the rotation, 64-bit attention."""
    torch = gpu
    d, h, hk, dim = 256, 6, 2, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    table = sv.rope_table(512, dim)
    block = sv.DecoderAttention(rand((h + 2 * hk) * dim, d) * 0.06, rand(d, h * dim) * 0.05, h, hk, table, bo=rand(d))
    cache = sv.PagedKvCache(1, 40, 16, hk, dim)
    x = {0: rand(150, d).bfloat16(), 1: rand(40, d).bfloat16()}
    got = {s: [] for s in x}
    for sizes in ({0: 100, 1: 3}, {0: 1, 1: 37}, {0: 49}):        # chunks and single tokens mixed
        at = {s: cache.length(s) for s in sizes}
        step = cache.extend(sizes)
        out = block(torch.cat([x[s][at[s]:at[s] + n] for s, n in sizes.items()]), cache.k[0], cache.v[0], step)
        for s, part in zip(sizes, out.split(list(sizes.values()))):
            got[s].append(part)
    sv.check()
    for s, xs in x.items():
        y = sv.linear_i8_token(xs, block.wqkv, block.sqkv).view(-1, h + 2 * hk, dim)
        pos = np.arange(xs.shape[0])
        turn = lambda t: torch.from_numpy(rotate_reference(t.float().cpu().numpy(), pos, table.cpu().numpy(),  # noqa: E731
                                                           False)).bfloat16().cuda()
        q, k, v = turn(y[:, :h]), turn(y[:, h:h + hk]), y[:, h + hk:]
        o, _, _ = attention_reference(torch, q, k[None], v[None], torch.zeros((1, 1), dtype=torch.int32, device="cuda"),
                                      [(len(pos), len(pos))], dim ** -0.5, True)
        want = sv.linear_i8_token(o.bfloat16().view(len(pos), -1), block.wo, block.so, bias=block.bo).float()
        off = (torch.cat(got[s]).float() - want).norm() / want.norm()
        # attention within about 2^-8 of its reference, a step of 1 / 127 of its largest value where
        # that changes a rounding, and the result's own 2^-9
        assert off <= 0.01, float(off)


def test_paged_cache_bookkeeping(gpu, sv):
    torch = gpu
    cache = sv.PagedKvCache(2, 5, 4, 1, 64, dtype=torch.float16)
    step = cache.extend({7: 6, 9: 1})
    assert step.positions.tolist() == [0, 1, 2, 3, 4, 5, 0] and step.cu_q.tolist() == [0, 6, 7]
    assert step.kv_len.tolist() == [6, 1] and (step.max_q_len, step.max_kv_len) == (6, 6)
    pages = [s // 4 for s in step.slots.tolist()]
    assert pages[0] == pages[3] != pages[4] == pages[5] and len(set(pages)) == 3
    assert step.block_table[0].tolist() == [pages[0], pages[4]] and step.block_table[1, 0] == pages[6]
    with pytest.raises(MemoryError):
        cache.extend({9: 20})
    assert cache.length(9) == 1 and cache.free_pages == 2
    step = cache.extend({9: 3, 7: 0})
    assert [s // 4 for s in step.slots.tolist()] == [pages[6]] * 3 and step.positions.tolist() == [1, 2, 3]
    cache.release(7)
    assert cache.free_pages == 4 and cache.length(7) == 0
    with pytest.raises(ValueError):
        cache.extend({})


def test_example_decodes_as_it_prefills(gpu, sv):
    """The logits of decoded tokens are those of the same tokens prefilled as a prompt."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve_decoder.py")
    spec = importlib.util.spec_from_file_location("serve_decoder", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    torch = gpu
    model = m.Decoder(2, vocab=500, positions=512)
    prompts = [[3, 1, 4, 1, 5], list(range(90)), [2] * 300]
    tokens, logits = m.generate(model, prompts, 5, chunk=64)
    longer = [p + t[:-1] for p, t in zip(prompts, tokens.tolist())]
    _, again = m.generate(model, longer, 1, chunk=400)
    # i8 steps that fall the other way after a 16-bit rounding: within a few percent
    off = (logits[:, -1] - again[:, 0]).norm() / again[:, 0].norm()
    assert off < 0.05, float(off)
