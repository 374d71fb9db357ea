"""Performance cases of the decoder-serving operators (``rustgears_b200.serving``).

Four operators that one attention block of an INT8 decoder chains:

* ``linear``     x W^T in 8-bit integers, one scale per token and one per output channel;
* ``rope``       rotary positions from a cos / sin table, half or interleaved pairs;
* ``append``     rotation of q and k and the write of k and v into a paged cache;
* ``attention``  a chunk of new tokens (one token when decoding) against a paged cache.

``run`` computes an operator in its plain form (elementary torch operations in 32
bits, rounded once at the end), or with ``own`` set calls the framework.  Lengths
inside a batch come from the case itself; values and the order of the pages from the
seed.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTS = ("none", "gelu", "silu", "relu")

# What no drawn case exceeds: the largest listed case of each operator.
MAX_MACS = 16384 * 8192 * 8192
MAX_ROPE = 16384 * 32 * 128
MAX_APPEND = 8192 * 32 * 64
MAX_SCORES = 2048 * 16384 * 32
MAX_CACHE = 64 * 6144 * 8 * 128


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one token through a 1024 -> 2816 projection (the transformer configuration's widths)
        dict(name="linear 1x1024x2816", op="linear", m=1, k=1024, n=2816, x="bf16", out="bf16", bias=False, act="none"),
        # a small batch of tokens, rows and reduction not whole tiles, f32 in and out
        dict(name="linear 37x2810x1030 gelu", op="linear", m=37, k=2810, n=1030, x="f32", out="f32", bias=True,
             act="gelu"),
        # a prompt chunk through the 4096 x 14336 Linear + GELU of the benchmark
        dict(name="linear 2048x4096x14336 gelu", op="linear", m=2048, k=4096, n=14336, x="f16", out="f16", bias=True,
             act="gelu"),
        # the benchmark's second Linear shape
        dict(name="linear 16384x8192x8192", op="linear", m=16384, k=8192, n=8192, x="bf16", out="bf16", bias=False,
             act="none"),
        # the query heads of one decoded token
        dict(name="rope 1x32x128", op="rope", tokens=1, heads=32, dim=128, rot=128, inter=False, x="bf16", scaling="none"),
        # a long batch of prompts: f32, half of each head rotated in interleaved pairs, positions far out
        dict(name="rope 16384x32x128 part", op="rope", tokens=16384, heads=32, dim=128, rot=64, inter=True, x="f32",
             scaling="bands"),
        # one decode step of 64 sequences
        dict(name="append 64 tokens", op="append", tokens=64, heads=32, kv_heads=8, dim=128, rot=128, inter=False,
             x="bf16", cache="bf16", page=16, layout="token", scaling="none"),
        # a prompt batch from f32 projections into an f16 cache, one head of every head its own (no sharing)
        dict(name="append 8192 tokens", op="append", tokens=8192, heads=16, kv_heads=16, dim=64, rot=32, inter=True,
             x="f32", cache="f16", page=64, layout="head", scaling="linear"),
        # one decoded token over a context of 4001 keys
        dict(name="attention 1 token", op="attention", mix="one", batch=1, q_len=1, kv_len=4001, heads=32, kv_heads=8,
             dim=128, x="bf16", page=16, layout="token"),
        # one decode step of 64 sequences with contexts of up to 6144 keys
        dict(name="attention 64 decodes", op="attention", mix="ragged", batch=64, q_len=1, kv_len=6144, heads=32,
             kv_heads=8, dim=128, x="bf16", page=64, layout="head"),
        # a batch where some sequences decode and others bring chunks, heads of 64
        dict(name="attention mixed chunks", op="attention", mix="mixed", batch=12, q_len=509, kv_len=2777, heads=16,
             kv_heads=16, dim=64, x="f16", page=128, layout="token"),
        # one chunk of 2048 new tokens on a context of 16384
        dict(name="attention chunk 2048", op="attention", mix="one", batch=1, q_len=2048, kv_len=16384, heads=32,
             kv_heads=8, dim=128, x="bf16", page=64, layout="token"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("linear", "linear", "rope", "append", "attention", "attention", "attention"))
    if op == "linear":
        while True:
            m, k, n = _log(rng, 1, 16384), _log(rng, 256, 8192), _log(rng, 64, 14336)
            if rng.random() < 0.5:
                k, n = max(256, k // 320 * 320), max(64, n // 320 * 320)
            if m * k * n <= MAX_MACS:
                break
        x = rng.choice(("f32", "f16", "bf16"))
        return dict(op=op, m=m, k=k, n=n, x=x, out=rng.choice((x, "f32")), bias=rng.random() < 0.5,
                    act=rng.choice(ACTS))
    dim = rng.choice((64, 64, 96, 128, 128, 128, 256))
    rot = rng.choice((dim, dim, dim // 2, dim // 4))
    scaling = rng.choice(("none", "linear", "bands"))
    inter = rng.random() < 0.5
    if op == "rope":
        heads = rng.randint(1, 64)
        tokens = _log(rng, 1, max(1, min(16384, MAX_ROPE // (heads * dim))))
        return dict(op=op, tokens=tokens, heads=heads, dim=dim, rot=rot, inter=inter,
                    x=rng.choice(("f32", "f16", "bf16")), scaling=scaling)
    kv_heads = rng.choice((1, 2, 3, 4, 8, 8, 16))
    heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 4, 7, 8))
    page = rng.choice((8, 16, 16, 24, 32, 64, 128, 256))
    layout = rng.choice(("token", "head"))
    if op == "append":
        cache = rng.choice(("f16", "bf16"))
        tokens = _log(rng, 1, max(1, min(8192, MAX_APPEND // (heads * dim))))
        return dict(op=op, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, inter=inter,
                    x=rng.choice(("f32", cache)), cache=cache, page=page, layout=layout, scaling=scaling)
    x = rng.choice(("f16", "bf16"))
    while True:
        mix = rng.choice(("one", "ragged", "mixed"))
        batch = 1 if mix == "one" else _log(rng, 2, 64)
        q_len = rng.choice((1, 1, rng.randint(2, 9), _log(rng, 10, 2048)))
        kv_len = max(q_len, _log(rng, 16, 16384))
        if batch * heads * q_len * kv_len <= MAX_SCORES and batch * kv_len * kv_heads * dim <= MAX_CACHE:
            break
    return dict(op=op, mix=mix, batch=batch, q_len=q_len, kv_len=kv_len, heads=heads, kv_heads=kv_heads, dim=dim, x=x,
                page=page, layout=layout)


def _lengths(case):
    """(new tokens, keys) of each sequence of an attention case; the longest is the case's own."""
    b, q, kv = case["batch"], case["q_len"], case["kv_len"]
    r = random.Random(b * 1000003 + q * 1009 + kv)
    out = [(q, kv)]
    for i in range(1, b):
        if case["mix"] == "mixed" and i % 2:
            qi = 1                                          # this sequence decodes
        else:
            qi = q if case["mix"] == "ragged" else r.randint(1, q)
        out.append((qi, r.randint(min(kv, max(qi, kv // 8)), kv)))
    return out


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return dict(bytes=m * k * size[case["x"]] + n * k + 4 * n * (2 if case["bias"] else 1) +
                    m * n * size[case["out"]], flops=2 * m * n * k)
    if case["op"] == "rope":
        e = case["tokens"] * case["heads"] * case["dim"]
        return dict(bytes=2 * e * size[case["x"]] + case["tokens"] * (4 + 4 * case["rot"]),
                    flops=3 * case["tokens"] * case["heads"] * case["rot"])
    if case["op"] == "append":
        e = case["tokens"] * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return dict(bytes=e * (size[case["x"]] + size[case["cache"]]) + case["tokens"] * (12 + 4 * case["rot"]),
                    flops=3 * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["rot"])
    h, hk, d, s = case["heads"], case["kv_heads"], case["dim"], size[case["x"]]
    lens = _lengths(case)
    tokens, keys = sum(q for q, _ in lens), sum(kv for _, kv in lens)
    pairs = sum(q * (kv - q) + q * (q + 1) // 2 for q, kv in lens)
    return dict(bytes=2 * tokens * h * d * s + 2 * keys * hk * d * s +
                4 * sum(-(-kv // case["page"]) for _, kv in lens) + 8 * len(lens), flops=4 * pairs * h * d)


# ---------------------------------------------------------------------------
# what a user's program holds before the call
# ---------------------------------------------------------------------------
def _table(positions, rot, scaling, device):
    """cos / sin rows [positions, rot] (cosines first), f32, from angles in 64 bits."""
    i = torch.arange(rot // 2, device=device, dtype=torch.float64)
    freq = 10000.0 ** (-2.0 * i / rot)
    gain = 1.0
    if scaling == "linear":          # positions interpolated by 4
        freq = freq / 4.0
    elif scaling == "bands":         # low frequencies interpolated by 8, high ones kept, a ramp between
        def edge(turns):
            return rot * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))
        lo, hi = max(0.0, math.floor(edge(32.0))), min(rot - 1.0, math.ceil(edge(1.0)))
        keep = 1.0 - ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        freq = freq / 8.0 * (1.0 - keep) + freq * keep
        gain = 0.1 * math.log(8.0) + 1.0
    a = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * freq
    return torch.cat([a.cos() * gain, a.sin() * gain], 1).float()


def _pool(case, pages, gen):
    """A page pool full of earlier keys, seen as [pages, page, kv_heads, dim]."""
    hk, d, p = case["kv_heads"], case["dim"], case["page"]
    shape = (pages, p, hk, d) if case["layout"] == "token" else (pages, hk, p, d)
    t = torch.randn(shape, device="cuda", generator=gen, dtype=DTYPES[case.get("cache", case["x"])])
    return t if case["layout"] == "token" else t.transpose(1, 2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dev = "cuda"
    s = dict(case=case)
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        x = torch.randn(m, k, device=dev, generator=gen)
        # a few channels much larger than the rest, as activations have them
        x *= 1.0 + 15.0 * (torch.rand(k, device=dev, generator=gen) < 0.005)
        s["x"] = x.to(DTYPES[case["x"]])
        w = torch.randn(n, k, device=dev, generator=gen) * 0.02
        s["w_scale"] = w.abs().amax(1) / 127.0
        ld = (k + 15) // 16 * 16
        s["w"] = torch.zeros(n, ld, device=dev, dtype=torch.int8)
        s["w"][:, :k] = (w / s["w_scale"][:, None]).round().clamp(-127, 127).to(torch.int8)
        s["bias"] = torch.randn(n, device=dev, generator=gen) * 0.01 if case["bias"] else None
        return s
    if case["op"] in ("rope", "append"):
        far = 32768
        t = case["tokens"]
        s["table"] = _table(far, case["rot"], case["scaling"], dev)
        if t >= 512:   # prompts: runs of consecutive positions
            start = torch.randint(0, far - t, (1,), device=dev, generator=gen, dtype=torch.int32)
            s["positions"] = start + torch.arange(t, device=dev, dtype=torch.int32)
        else:
            s["positions"] = torch.randint(0, far, (t,), device=dev, generator=gen, dtype=torch.int32)
    if case["op"] == "rope":
        s["x"] = torch.randn(case["tokens"], case["heads"], case["dim"], device=dev,
                             generator=gen).to(DTYPES[case["x"]])
        return s
    h, hk, d, p = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if case["op"] == "append":
        # one projection's output [tokens, (h + 2 hk) d]: q, k and v are views of it
        qkv = torch.randn(t, (h + 2 * hk) * d, device=dev, generator=gen).to(DTYPES[case["x"]])
        s["q"] = qkv[:, : h * d].view(t, h, d)
        s["k"] = qkv[:, h * d: (h + hk) * d].view(t, hk, d)
        s["v"] = qkv[:, (h + hk) * d:].view(t, hk, d)
        if t >= 512:   # prompts fill pages from their start, the pages lying anywhere
            pages = -(-t // p) + 2
            order = torch.randperm(pages, device=dev, generator=gen)
            i = torch.arange(t, device=dev)
            s["slots"] = order[i // p] * p + i % p
        else:          # decoding: every token in a page of its own
            pages = t + 2
            order = torch.randperm(pages, device=dev, generator=gen)[:t]
            s["slots"] = order * p + torch.randint(0, p, (t,), device=dev, generator=gen)
        s["k_cache"], s["v_cache"] = _pool(case, pages, gen), _pool(case, pages, gen)
        return s
    lens = _lengths(case)
    need = [-(-kv // p) for _, kv in lens]
    pages = sum(need) + 3
    s["k_cache"], s["v_cache"] = _pool(case, pages, gen), _pool(case, pages, gen)
    order = torch.randperm(pages, device=dev, generator=gen).to(torch.int32).cpu()
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(need):
        table[b, :c] = order[at: at + c]
        at += c
    s["block_table"] = table.to(dev)
    s["kv_len"] = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=dev)
    s["cu_q"] = torch.tensor(np.cumsum([0] + [q for q, _ in lens]), dtype=torch.int32, device=dev)
    s["max_q"], s["max_kv"] = max(q for q, _ in lens), max(kv for _, kv in lens)
    tokens = sum(q for q, _ in lens)
    s["q"] = torch.randn(tokens, h, d, device=dev, generator=gen).to(DTYPES[case["x"]])
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _act(y, act):
    if act == "gelu":
        return 0.5 * y * (1.0 + torch.tanh(0.7978846 * (y + 0.044715 * y * y * y)))
    if act == "silu":
        return y * (1.0 / (1.0 + torch.exp(-y)))
    return torch.clamp(y, min=0.0) if act == "relu" else y


def _linear(s):
    c, x = s["case"], s["x"].float()
    amax = x.abs().amax(1, keepdim=True)
    # divided by a tensor: torch multiplies by the reciprocal of a plain number
    scale = torch.where(amax < 1e-12, torch.ones_like(amax), amax / torch.full_like(amax, 127.0))
    t = x * (1.0 / scale)
    whole = torch.trunc(t)
    q = (whole + torch.sign(t) * ((t - whole).abs() >= 0.5)).clamp(-127.0, 127.0)
    acc = q @ s["w"][:, : c["k"]].float().t()
    y = acc * (scale * s["w_scale"])
    if s["bias"] is not None:
        y = y + s["bias"]
    return _act(y, c["act"]).to(DTYPES[c["out"]])


def _rotate(x, positions, table, inter):
    rot = table.shape[1]
    row = table[positions.long()]
    cos, sin = row[:, None, : rot // 2], row[:, None, rot // 2:]
    x = x.float()
    r, rest = x[..., :rot], x[..., rot:]
    a, b = (r[..., 0::2], r[..., 1::2]) if inter else (r[..., : rot // 2], r[..., rot // 2:])
    y, z = a * cos - b * sin, b * cos + a * sin
    both = torch.stack([y, z], -1).flatten(-2) if inter else torch.cat([y, z], -1)
    return torch.cat([both, rest], -1)


def _append(s):
    c = s["case"]
    kind = DTYPES[c["cache"]]
    page, off = s["slots"] // c["page"], s["slots"] % c["page"]
    s["k_cache"][page, off] = _rotate(s["k"], s["positions"], s["table"], c["inter"]).to(kind)
    s["v_cache"][page, off] = s["v"].to(kind)
    return _rotate(s["q"], s["positions"], s["table"], c["inter"]).to(kind), s["k_cache"], s["v_cache"]


def _attention(s):
    c, q = s["case"], s["q"]
    h, hk, d, p = c["heads"], c["kv_heads"], c["dim"], c["page"]
    batch, most_q, most_kv = s["kv_len"].numel(), s["max_q"], s["max_kv"]
    token = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(s["cu_q"][1:].long(), token, right=True)
    at = token - s["cu_q"].long()[seq]
    qp = torch.zeros(batch, most_q, h, d, device=q.device)
    qp[seq, at] = q.float()
    pages = s["block_table"].long().clamp(min=0)
    k = s["k_cache"][pages].reshape(batch, -1, hk, d)[:, :most_kv].float()
    v = s["v_cache"][pages].reshape(batch, -1, hk, d)[:, :most_kv].float()
    # [batch, hk, group * most_q, d]: the query heads that share a key head side by side
    qp = qp.view(batch, most_q, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(batch, hk, -1, d)
    score = (qp @ k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
    kv, ql = s["kv_len"].long(), s["cu_q"].long().diff()
    key = torch.arange(most_kv, device=q.device)
    last = torch.arange(most_q, device=q.device)[None, :] + (kv - ql)[:, None]
    seen = (key[None, None, :] <= last[:, :, None]) & (key[None, None, :] < kv[:, None, None])
    seen = seen[:, None, None]
    score = score.view(batch, hk, h // hk, most_q, most_kv).masked_fill_(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    o = (e.view(batch, hk, -1, most_kv) @ v.permute(0, 2, 1, 3)).view(batch, hk, h // hk, most_q, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(batch, most_q, h, d)[seq, at].to(q.dtype)


def _own(s):
    from rustgears_b200 import serving
    c = s["case"]
    if c["op"] == "linear":
        return serving.linear_i8_token(s["x"], s["w"], s["w_scale"], bias=s["bias"], act=c["act"],
                                       out_dtype=DTYPES[c["out"]])
    if c["op"] == "rope":
        return serving.rope(s["x"], s["positions"], s["table"], interleaved=c["inter"])
    if c["op"] == "append":
        q = serving.kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], positions=s["positions"],
                              table=s["table"], interleaved=c["inter"], q=s["q"])
        return q, s["k_cache"], s["v_cache"]
    return serving.attention_paged(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["kv_len"], s["cu_q"],
                                   max_q_len=s["max_q"], max_kv_len=s["max_kv"])


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "rope":
        c = state["case"]
        return _rotate(state["x"], state["positions"], state["table"], c["inter"]).to(DTYPES[c["x"]])
    return {"linear": _linear, "append": _append, "attention": _attention}[op](state)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _exact_rotation(x, positions, table, inter):
    """Each pair (a, b) as the complex number a + ib times the table's cos + i sin."""
    rot = table.shape[1]
    turn = torch.complex(*table.double()[positions.long()].chunk(2, 1))[:, None]
    out = x.double().clone()
    head = out[..., :rot]
    pairs = head.unflatten(-1, (rot // 2, 2)) if inter else head.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    pairs.copy_(turned)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        # The quantized rows are defined in 32 bits (scale = absmax / 127, its reciprocal,
        # products rounded to the nearest integer, halves away from zero); the rest is exact.
        x = s["x"].float()
        amax = torch.linalg.vector_norm(x, float("inf"), dim=1)
        scale = torch.div(amax, amax.new_full((), 127.0).expand_as(amax)).masked_fill(amax < 1e-12, 1.0)
        t = (x * scale.reciprocal()[:, None]).double()
        q = torch.where(t < 0, (t - 0.5).ceil(), (t + 0.5).floor()).clamp_(-127, 127)
        del t
        y = torch.nn.functional.pad(q, (0, s["w"].shape[1] - q.shape[1])) @ s["w"].double().t()
        y *= scale.double()[:, None]
        y *= s["w_scale"].double()
        if s["bias"] is not None:
            y += s["bias"].double()
        if case["act"] == "gelu":    # the tanh form, its constant the f32 nearest sqrt(2 / pi)
            return 0.5 * y * (1.0 + torch.tanh(float(np.float32(0.7978846)) * (y + 0.044715 * y ** 3)))
        if case["act"] == "silu":
            return y * torch.sigmoid(y)
        return torch.relu(y) if case["act"] == "relu" else y
    if case["op"] == "rope":
        return _exact_rotation(s["x"], s["positions"], s["table"], case["inter"])
    if case["op"] == "append":
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        k = _exact_rotation(s["k"], s["positions"], s["table"], case["inter"])
        slots, p = s["slots"], case["page"]
        where = (torch.div(slots, p, rounding_mode="floor"), torch.remainder(slots, p))
        k_cache = k_cache.index_put(where, k)
        v_cache = v_cache.index_put(where, s["v"].double())
        return _exact_rotation(s["q"], s["positions"], s["table"], case["inter"]), k_cache, v_cache
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    start = 0
    for b, (ql, kv) in enumerate(_lengths(case)):
        pages = s["block_table"][b, : -(-kv // case["page"])].long()
        k = s["k_cache"][pages].flatten(0, 1)[:kv].double()
        v = s["v_cache"][pages].flatten(0, 1)[:kv].double()
        hidden = torch.ones(ql, kv, dtype=torch.bool, device="cuda").triu(kv - ql + 1)
        for g in range(hk):
            q = s["q"][start: start + ql, g * (h // hk): (g + 1) * (h // hk)].double()
            score = torch.einsum("qhd,kd->hqk", q, k[:, g]) / math.sqrt(d)
            prob = torch.softmax(score.masked_fill_(hidden, -math.inf), -1)
            out[start: start + ql, g * (h // hk): (g + 1) * (h // hk)] = torch.einsum("hqk,kd->qhd", prob, v[:, g])
        start += ql
    return out
