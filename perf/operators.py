"""Performance cases of the operators behind a step of drafted tokens: norms and rotation of queries and keys, a
K/V cache held in few bits, attention of a tree of drafts over that cache, and the move of the accepted rows.

``run`` gives each operator's plain form in torch, or, with ``own``, the package's calls.  ``exact`` repeats a case
in 64 bits.  Sizes are those of the package's 8B and 1.5B layer shapes and of odd ones beside them.

A cache buffer holds [positions][KV heads][head_dim] values as F32 or F16, or their codes followed by one f16 scale
per 32 values (Q8_0: a byte, the code plus 128; Q4_0: two codes plus 8 in a byte, the even element low)."""
from __future__ import annotations

import math

import torch

own = False

EPS, THETA = 1e-6, 1e6  # of models that norm their queries and keys
BITS = {"F32": 32, "F16": 16, "Q8_0": 8, "Q4_0": 4}


def listed():
    return [
        # one decoded token of an 8B layer: launch latency
        {"name": "rope_token", "kind": "rope", "tokens": 1, "heads": 32, "kv_heads": 8, "head_dim": 128, "past": 8191},
        # a prompt's chunk of the same layer, written into an F16 cache on the way
        {"name": "rope_prompt", "kind": "rope_store", "type": "F16", "tokens": 2048, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "past": 100},
        # a draft's rows, as each layer of a step writes them
        {"name": "cache_draft", "kind": "cache", "type": "Q8_0", "tokens": 16, "kv_heads": 8, "head_dim": 128,
         "past": 1000},
        # a long ragged document's rows into four bits
        {"name": "cache_prompt", "kind": "cache", "type": "Q4_0", "tokens": 8191, "kv_heads": 8, "head_dim": 128,
         "past": 0},
        # plain decoding: one token over two thousand positions
        {"name": "tree_one", "kind": "tree", "type": "Q8_0", "tokens": 1, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "past": 2047},
        # a usual draft at a full context
        {"name": "tree_draft", "kind": "tree", "type": "Q8_0", "tokens": 16, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "past": 8176},
        # seven query heads per KV head, short rows, an odd length
        {"name": "tree_seven", "kind": "tree", "type": "F16", "tokens": 7, "heads": 14, "kv_heads": 2, "head_dim": 64,
         "past": 1501},
        # the cache as the model keeps it now, a 1.5B model's heads
        {"name": "tree_f32", "kind": "tree", "type": "F32", "tokens": 37, "heads": 12, "kv_heads": 2, "head_dim": 128,
         "past": 600},
        # a wide tree, or the last chunk of a prompt that branches: matrix cores
        {"name": "tree_wide", "kind": "tree", "type": "Q8_0", "tokens": 256, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "past": 8000},
        # a draft at the end of a book held in four bits
        {"name": "tree_long", "kind": "tree", "type": "Q4_0", "tokens": 16, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "past": 131056},
        # the accepted path of a draft in all layers of an 8B model
        {"name": "move_path", "kind": "move", "type": "F16", "layers": 32, "tokens": 16, "accepted": 5, "kv_heads": 8,
         "head_dim": 128, "past": 40},
        # a long path of a wide tree in the f32 cache of a small model
        {"name": "move_wide", "kind": "move", "type": "F32", "layers": 28, "tokens": 256, "accepted": 100,
         "kv_heads": 2, "head_dim": 128, "past": 3},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("rope", "rope_store", "cache", "cache", "tree", "tree", "tree", "tree", "move"))
    kv, hd = rng.choice((1, 2, 3, 4, 8, 8)), rng.choice((64, 64, 96, 128, 128, 128, 256))
    case = {"kind": kind, "kv_heads": kv, "head_dim": hd}
    if kind == "rope":
        return {**case, "heads": kv * rng.randint(1, 8), "tokens": _log(rng, 1, 1500), "past": _log(rng, 1, 100000)}
    if kind == "rope_store":
        return {**case, "heads": kv * rng.randint(1, 8), "tokens": _log(rng, 1, 1500), "past": _log(rng, 1, 500),
                "type": rng.choice(("F32", "F16"))}
    if kind == "cache":
        return {**case, "tokens": _log(rng, 1, 4000), "past": rng.randint(0, 300),
                "type": rng.choice(("F16", "Q8_0", "Q8_0", "Q4_0", "Q4_0"))}
    if kind == "move":
        n = _log(rng, 2, 256)
        return {**case, "layers": rng.randint(1, 40), "tokens": n, "accepted": rng.randint(1, n),
                "past": rng.randint(0, 50), "type": rng.choice(("F32", "F16"))}
    n = rng.choice((1, _log(rng, 1, 64), _log(rng, 1, 64), _log(rng, 32, 256)))
    heads, most = kv * rng.randint(1, 8), 16000 if n < 65 else 4000
    return {**case, "heads": heads, "tokens": n, "past": _log(rng, 1, min(most, 2 ** 33 // (n * heads * hd))),
            "type": rng.choice(("F32", "F16", "Q8_0", "Q8_0", "Q4_0"))}


# ------------------------------------------------------------------- prepare

class _State:
    pass


def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + salt)


def _normal(seed, salt, *shape):
    return torch.randn(*shape, generator=_gen(seed, salt), device="cuda")


def _power(e):
    """2 ** e of whole numbers, exactly (a device's exp2 may be off by a bit, which a tie of the codes shows)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _scales(x, t):
    """One scale per 32 values of x [..., blocks, 32], in 64 bits: the least f16 of 3 (Q8_0) or 8 (Q4_0) significant
    bits that reaches the block's extreme with its largest code; of Q4_0 signed so that the extreme is -8."""
    low, high = x.amin(-1).double(), x.amax(-1).double()
    top = torch.maximum(high, -low)
    bits, want, most = (3, top / 127, 512.0) if t == "Q8_0" else (8, top / 8, 8160.0)
    step = _power((torch.frexp(want)[1] - bits).clamp(min=-24))
    d = (torch.ceil(want / step) * step).clamp(max=most)
    return torch.where(high > -low, -d, d) if t == "Q4_0" else d


def _codes(x, d, t):
    q = torch.where(d[..., None] == 0, 0.0, torch.round(x.double() / d[..., None]))
    return q.clamp(-127, 127) if t == "Q8_0" else q.clamp(-8, 7)


def _encode(x, t):
    """The buffer's bytes of x [positions, KV heads, head_dim] in type t."""
    if t == "F32":
        return x.contiguous().view(torch.uint8).reshape(-1)
    if t == "F16":
        return x.half().view(torch.uint8).reshape(-1)
    b = x.reshape(*x.shape[:2], -1, 32)
    d = _scales(b, t)
    q = (_codes(b, d, t) + (128 if t == "Q8_0" else 8)).to(torch.uint8)
    if t == "Q4_0":
        q = q[..., 0::2] | q[..., 1::2] << 4
    return torch.cat([q.reshape(-1), d.half().view(torch.uint8).reshape(-1)])


def _size(c, positions):
    n = positions * c["kv_heads"] * c["head_dim"]
    return n * BITS[c["type"]] // 8 + (n // 16 if c["type"][0] == "Q" else 0)


def _cache(c, seed, salt, positions):
    """Bytes of a cache buffer of normal rows, encoded in pieces that are put in place."""
    kv, hd, t = c["kv_heads"], c["head_dim"], c["type"]
    g, out, at = _gen(seed, salt), torch.empty(_size(c, positions), dtype=torch.uint8, device="cuda"), 0
    sat = positions * kv * hd * BITS[t] // 8
    for p in range(0, positions, 8192):
        m = min(8192, positions - p)
        piece = _encode(torch.randn(m, kv, hd, generator=g, device="cuda"), t)
        codes = m * kv * hd * BITS[t] // 8
        out[at:at + codes] = piece[:codes]
        at += codes
        out[sat:sat + piece.numel() - codes] = piece[codes:]
        sat += piece.numel() - codes
    return out


def _parents(seed, n):
    """A tree of drafts: each node under an earlier one (most often a late one), or under the history (-1)."""
    at = torch.rand(n, generator=torch.Generator().manual_seed(int(seed) * 7 + 3), dtype=torch.float64)
    i = torch.arange(n)
    return torch.clamp((at.sqrt() * (i + 1)).long(), max=n) - 1


def _mask(parents):
    """[n, words] int64: bit j of row i where j is i or one of its ancestors."""
    n = len(parents)
    rows, words = [], (n + 63) // 64
    for i, p in enumerate(parents.tolist()):
        rows.append((rows[p] if p >= 0 else 0) | 1 << i)
    flat = [r >> 64 * w & (1 << 64) - 1 for r in rows for w in range(words)]
    return torch.tensor([v - (1 << 64) if v >> 63 else v for v in flat], dtype=torch.int64).reshape(n, words)


def _inputs(c, seed):
    """The tensors of a case, from the seed alone."""
    s, n, kv, hd, kind = _State(), c["tokens"], c["kv_heads"], c["head_dim"], c["kind"]
    total = c["past"] + n
    if kind in ("rope", "rope_store"):
        # one projection's output: a token's queries, keys and values in one row
        s.qkv = _normal(seed, 1, n, (c["heads"] + 2 * kv) * hd)
        s.wq, s.wk = (1 + 0.2 * _normal(seed, k, hd) for k in (2, 3))
        s.positions = torch.arange(c["past"], total, device="cuda", dtype=torch.int32)
    if kind == "cache":
        s.x = [_normal(seed, k, n, kv, hd) * torch.exp(_normal(seed, k + 2, n, kv, 1)) for k in (1, 2)]
    if kind == "tree":
        s.q = _normal(seed, 1, n, c["heads"], hd)
        s.parents = _parents(seed, n)
    if kind == "move":
        s.src = (c["past"] + torch.randperm(n, generator=torch.Generator().manual_seed(int(seed) + 5))
                 [:c["accepted"]].sort()[0]).to(torch.int32).cuda()
        s.k, s.v = (_normal(seed, k, c["layers"], total, kv, hd).to(_dtype(c)) for k in (1, 2))
    return s


def _dtype(c):
    return torch.float16 if c["type"] == "F16" else torch.float32


def prepare(case, seed):
    c, s = case, _inputs(case, seed)
    n, kv, hd, total = c["tokens"], c["kv_heads"], c["head_dim"], c["past"] + c["tokens"]
    s.case, s.handle = c, None
    if c["kind"] == "rope":
        s.q_out, s.k_out = torch.empty(n, c["heads"], hd, device="cuda"), torch.empty(n, kv, hd, device="cuda")
    elif c["kind"] == "rope_store":
        s.q_out = torch.empty(n, c["heads"], hd, device="cuda")
        s.k, s.v = (torch.zeros(total, kv, hd, dtype=_dtype(c), device="cuda") for _ in range(2))
    elif c["kind"] == "cache":
        s.k, s.v = (torch.zeros(_size(c, total), dtype=torch.uint8, device="cuda") for _ in range(2))
        s.k_out, s.v_out = (torch.empty(n, kv, hd, device="cuda") for _ in range(2))
    elif c["kind"] == "tree":
        s.k, s.v = _cache(c, seed, 2, total), _cache(c, seed, 3, total)
        s.mask = _mask(s.parents).cuda()
        s.out = torch.empty(n, c["heads"], hd, device="cuda")
    torch.cuda.synchronize()  # the library's own stream does not wait for torch's
    return s


# ----------------------------------------------------------------------- run

_CTX = None


def _context(rf):
    global _CTX
    if _CTX is None:
        _CTX = rf.Context(0)
    return _CTX


def _own_handle(s):
    """The context and the caches' handles, which a program keeps with its buffers."""
    import ramforge_amd as rf

    c, ctx = s.case, _context(rf)
    if c["kind"] == "rope":
        caches = None
    elif c["kind"] == "move":
        caches = rf.KvCacheList([rf.KvCache(ctx, getattr(rf.GGML, c["type"]), k.shape[0], c["kv_heads"],
                                            c["head_dim"], k.data_ptr(), v.data_ptr()) for k, v in zip(s.k, s.v)])
    else:
        caches = rf.KvCache(ctx, getattr(rf.GGML, c["type"]), c["past"] + c["tokens"], c["kv_heads"], c["head_dim"],
                            s.k.data_ptr(), s.v.data_ptr())
    return rf, ctx, caches


def _run_own(s):
    if s.handle is None:
        s.handle = _own_handle(s)
    rf, ctx, cache = s.handle
    c, kind = s.case, s.case["kind"]
    n, kv, hd, past = c["tokens"], c["kv_heads"], c["head_dim"], c["past"]
    if kind in ("rope", "rope_store"):
        qh, row = c["heads"], s.qkv.shape[1]
        q = s.qkv.data_ptr()
        k, v = q + 4 * qh * hd, q + 4 * (qh + kv) * hd
        if kind == "rope":
            rf.qk_norm_rope(ctx, q, k, s.wq.data_ptr(), s.wk.data_ptr(), EPS, s.positions.data_ptr(), n, qh, kv, hd,
                            THETA, s.q_out.data_ptr(), s.k_out.data_ptr(), q_stride=row, k_stride=row)
            return s.q_out, s.k_out
        rf.qk_norm_rope_store(ctx, q, k, v, s.wq.data_ptr(), s.wk.data_ptr(), EPS, s.positions.data_ptr(), n, qh,
                              THETA, s.q_out.data_ptr(), cache, past, q_stride=row, k_stride=row, v_stride=row)
        return s.q_out, s.k, s.v
    if kind == "cache":
        rf.kv_store(ctx, cache, s.x[0].data_ptr(), s.x[1].data_ptr(), past, n)
        rf.kv_load(ctx, cache, past, n, s.k_out.data_ptr(), s.v_out.data_ptr())
        return s.k_out, s.v_out
    if kind == "tree":
        rf.attention_tree(ctx, s.q.data_ptr(), cache, past, n, c["heads"], mask=s.mask.data_ptr(),
                          out=s.out.data_ptr())
        return s.out
    rf.kv_move(ctx, cache, s.src.data_ptr(), past, c["accepted"])
    return s.k, s.v


def _norm_rope(x, w, cos, sin):
    """x [tokens, heads, head_dim]; cos, sin [tokens, 1, head_dim / 2]"""
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    a, b = y.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _decode(buf, c, first, n):
    """Rows first .. first + n - 1 of a cache buffer as f32 [n, KV heads, head_dim]."""
    kv, hd, t = c["kv_heads"], c["head_dim"], c["type"]
    total = c["past"] + c["tokens"]
    row = kv * hd * BITS[t] // 8
    codes = buf[:total * row].reshape(total, row)[first:first + n]
    if t == "F32":
        return codes.view(torch.float32).reshape(n, kv, hd)
    if t == "F16":
        return codes.view(torch.float16).reshape(n, kv, hd).float()
    d = buf[total * row:].view(torch.float16).reshape(total, kv, hd // 32, 1)[first:first + n].float()
    if t == "Q8_0":
        return ((codes.reshape(n, kv, hd // 32, 32).float() - 128) * d).reshape(n, kv, hd)
    u = codes.reshape(n, kv, hd // 32, 16)
    return ((torch.stack([u & 15, u >> 4], -1).reshape(n, kv, hd // 32, 32).float() - 8) * d).reshape(n, kv, hd)


def _run_plain(s):
    c, kind = s.case, s.case["kind"]
    n, kv, hd, past = c["tokens"], c["kv_heads"], c["head_dim"], c["past"]
    if kind in ("rope", "rope_store"):
        qh = c["heads"]
        x = s.qkv.reshape(n, qh + 2 * kv, hd)
        freq = THETA ** (torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / -hd)
        angle = s.positions.double()[:, None, None] * freq
        cos, sin = angle.cos().float(), angle.sin().float()
        q = _norm_rope(x[:, :qh], s.wq, cos, sin)
        k = _norm_rope(x[:, qh:qh + kv], s.wk, cos, sin)
        if kind == "rope":
            return q, k
        s.k[past:past + n] = k.to(s.k.dtype)
        s.v[past:past + n] = x[:, qh + kv:].to(s.v.dtype)
        return q, s.k, s.v
    if kind == "cache":
        total, row = past + n, kv * hd * BITS[c["type"]] // 8
        for buf, x in ((s.k, s.x[0]), (s.v, s.x[1])):
            new = _encode(x, c["type"])
            buf[past * row:total * row] = new[:n * row]
            if c["type"][0] == "Q":
                buf[total * row + past * kv * hd // 16:] = new[n * row:]
        return _decode(s.k, c, past, n), _decode(s.v, c, past, n)
    if kind == "tree":
        total, g = past + n, c["heads"] // kv
        k, v = _decode(s.k, c, 0, total), _decode(s.v, c, 0, total)
        q = s.q.reshape(n, kv, g, hd).permute(1, 0, 2, 3).reshape(kv, n * g, hd)
        scores = torch.bmm(q, k.permute(1, 2, 0).contiguous()) / math.sqrt(hd)
        j = torch.arange(n, device="cuda")
        hidden = (s.mask[:, j // 64] >> j % 64 & 1) == 0
        scores.reshape(kv, n, g, total)[..., past:].masked_fill_(hidden[None, :, None], -math.inf)
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        out = torch.bmm(p, v.permute(1, 0, 2).contiguous()) / p.sum(-1, keepdim=True)
        return out.reshape(kv, n, g, hd).permute(1, 0, 2, 3).reshape(n, kv * g, hd)
    src, m = s.src.long(), c["accepted"]
    s.k[:, past:past + m] = s.k[:, src]
    s.v[:, past:past + m] = s.v[:, src]
    return s.k, s.v


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------- work

def work(case):
    c, kind = case, case["kind"]
    n, kv, hd = c["tokens"], c["kv_heads"], c["head_dim"]
    if kind in ("rope", "rope_store"):
        heads = c["heads"] + kv
        b = 8 * n * heads * hd
        if kind == "rope_store":
            b = 4 * n * (heads + kv) * hd + 4 * n * c["heads"] * hd + 2 * _size(c, n)
        return {"bytes": b, "flops": 10 * n * heads * hd}
    if kind == "cache":  # rows written, then read back
        return {"bytes": 16 * n * kv * hd + 4 * _size(c, n), "flops": 10 * n * kv * hd}
    if kind == "tree":
        total = c["past"] + n
        return {"bytes": 2 * _size(c, total) + 8 * n * c["heads"] * hd, "flops": 4 * n * c["heads"] * total * hd}
    return {"bytes": 4 * c["layers"] * _size(c, c["accepted"]), "flops": 0}


# --------------------------------------------------------------------- exact

def _exact_values(x, t):
    """What a cache of type t gives back for x [..., 32] f64, by integers: the scale's significand is counted up."""
    top = x.abs().amax(-1, keepdim=True)
    levels, bits, most = (127.0, 3, 2.0 ** 9) if t == "Q8_0" else (8.0, 8, 8160.0)
    powers = torch.tensor([2.0 ** k for k in range(-60, 60)], dtype=torch.float64, device=x.device)
    e = torch.floor(torch.log2(torch.clamp(top / levels, min=2.0 ** -40))).long() + 60
    e = e - (powers[e] > top / levels).long() + (powers[e + 1] <= top / levels).long()
    unit = powers[torch.clamp(e - (bits - 1), min=60 - 24)]
    count = torch.floor(top / (levels * unit))
    count = torch.where(count * unit * levels < top, count + 1, count)
    d = torch.clamp(count * unit, max=most)
    if t == "Q4_0":
        d = torch.where(x.amax(-1, keepdim=True) > -x.amin(-1, keepdim=True), -d, d)
    q = x / torch.where(d == 0, torch.ones_like(d), d)
    near = torch.floor(q)
    rest = q - near
    near = torch.where((rest > 0.5) | ((rest == 0.5) & (near % 2 != 0)), near + 1, near)
    return torch.clamp(near, -levels, 127.0 if t == "Q8_0" else 7.0) * d


def _exact_cache(c, seed, salt, positions):
    g, kv, hd, t = _gen(seed, salt), c["kv_heads"], c["head_dim"], c["type"]
    parts = []
    for p in range(0, positions, 8192):
        x = torch.randn(min(8192, positions - p), kv, hd, generator=g, device="cuda")
        if t == "F16":
            x = x.half()
        if t[0] == "Q":
            x = _exact_values(x.double().reshape(-1, 32), t).reshape(x.shape)
        parts.append(x.double())
    return torch.cat(parts)


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    n, kv, hd, past, kind = c["tokens"], c["kv_heads"], c["head_dim"], c["past"], c["kind"]
    if kind in ("rope", "rope_store"):
        qh = c["heads"]
        x = s.qkv.double().reshape(n, -1, hd)
        i = torch.arange(hd // 2, device="cuda").double()
        turn = torch.polar(torch.ones(n, 1, hd // 2, device="cuda", dtype=torch.float64),
                           (past + torch.arange(n, device="cuda").double())[:, None, None]
                           * torch.exp(i * (-2 / hd * math.log(THETA))))

        def rotate(y, w):
            y = y / (y.square().sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
            z = torch.complex(y[..., :hd // 2].contiguous(), y[..., hd // 2:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        q, k = rotate(x[:, :qh], s.wq), rotate(x[:, qh:qh + kv], s.wk)
        if kind == "rope":
            return q, k
        pad = torch.zeros(past, kv, hd, dtype=torch.float64, device="cuda")
        return q, torch.cat([pad, k]), torch.cat([pad, x[:, qh + kv:]])
    if kind == "cache":
        if c["type"][0] != "Q":
            return tuple(x.to(_dtype(c)).double() for x in s.x)
        return tuple(_exact_values(x.double().reshape(-1, 32), c["type"]).reshape(x.shape) for x in s.x)
    if kind == "tree":
        k, v = (_exact_cache(c, seed, salt, past + n) for salt in (2, 3))
        sees = torch.zeros(n, past + n, dtype=torch.bool)
        sees[:, :past] = True
        for i, p in enumerate(s.parents.tolist()):
            if p >= 0:
                sees[i] = sees[p]
            sees[i, past + i] = True
        hide = ~sees.cuda()
        out = torch.empty(n, c["heads"], hd, dtype=torch.float64, device="cuda")
        for h in range(c["heads"]):
            kh, vh = (x[:, h * kv // c["heads"]].contiguous() for x in (k, v))
            z = (s.q[:, h].double() @ kh.T / math.sqrt(hd)).masked_fill(hide, -math.inf)
            out[:, h] = torch.softmax(z, -1) @ vh
        return out
    k, v = s.k.double(), s.v.double()
    for x in (k, v):
        x[:, past:past + c["accepted"]] = torch.stack([x[:, r] for r in s.src.tolist()], 1)
    return k, v
