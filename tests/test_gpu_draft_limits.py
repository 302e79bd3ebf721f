"""The draft-step calls at their far ends: shapes of every kernel that the attention chooses between, positions past 2^32
bytes of a cache, fixed workspaces, other streams, and a whole step captured and replayed.

Attention against its definition in 64 bits, with the tolerance of test_gpu_attention_tree.py (1e-5 of
sum_p softmax_p |v_p|: its derivation does not depend on the number of positions, whose sum's errors are at random)."""
import numpy as np
import pytest

import ramforge_amd as rf
from ramforge_amd import GGML
from test_gpu_attention_tree import TOL, TYPES, bits_of, check, sees_of, tree

pytestmark = pytest.mark.gpu

QUANT = [GGML.F16, GGML.Q8_0, GGML.Q4_0]


def big_cache(ctx, rng, t, cap, kvh, hd):
    """A cache of normal rows (a block of them over and over, no multiple of a row) and the values it gives back."""
    w = kvh * hd
    block = rng.standard_normal(1000003, np.float32)
    cache = rf.KvCache(ctx, t, cap, kvh, hd)
    kd, vd = ctx.array(np.resize(block, (cap, w))), ctx.array(np.resize(block[::-1], (cap, w)))
    rf.kv_store(ctx, cache, kd, vd, 0, cap)
    rf.kv_load(ctx, cache, 0, cap, kd, vd)
    k, v = (x.numpy().reshape(cap, kvh, hd) for x in (kd, vd))
    kd.free()
    vd.free()
    return cache, k, v


def some_rows(q, k, v, hist, sees, pairs):
    """The definition for (token, query head) pairs: result, sum softmax |v|, sum |v|."""
    n, qh, hd = q.shape
    kvh = k.shape[1]
    res = [np.zeros((len(pairs), hd)) for _ in range(3)]
    by = {}
    for e, (i, h) in enumerate(pairs):
        by.setdefault(h * kvh // qh, []).append((e, i, h))
    for g, rows in by.items():
        kk, vv = k[:hist + n, g].astype(np.float64), v[:hist + n, g].astype(np.float64)
        s = np.stack([q[i, h] for _, i, h in rows]).astype(np.float64) @ kk.T / np.sqrt(hd)
        s[:, hist:][~np.stack([sees[i] for _, i, _ in rows])] = -np.inf
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        at = [e for e, _, _ in rows]
        res[0][at], res[1][at], res[2][at] = p @ vv, p @ np.abs(vv), (p > 0) @ np.abs(vv)
    return res


# tokens, history, query heads, KV heads, head_dim: rows of a KV head and positions enough that the wavefronts of a
# workgroup split the rows, two row tiles a wavefront (the first three) or one; and the other kernel with two
FAR = [(1024, 42000, 1, 1, 64), (1000, 32000, 2, 1, 96), (999, 20500, 4, 1, 128), (1024, 22001, 8, 1, 256),
       (60, 41777, 16, 16, 64), (64, 170003, 8, 8, 128), (50, 131009, 8, 8, 96), (64, 4097, 4, 1, 64),
       (61, 4100, 4, 1, 96), (24, 4097, 8, 8, 128)]


# (an F32 cache has the other kernel alone)
@pytest.mark.parametrize("t, n, hist, qh, kvh, hd", [(t, *f) for f in FAR for t in (TYPES if f[1] < 5000 else QUANT)])
def test_shapes_of_every_kernel(ctx, t, n, hist, qh, kvh, hd):
    rng = np.random.default_rng(n + hist + hd)
    cache, k, v = big_cache(ctx, rng, t, hist + n + 1, kvh, hd)
    q = rng.standard_normal((n, qh, hd), np.float32)
    sees = sees_of(tree(rng, n))
    out = rf.attention_tree(ctx, ctx.array(q), cache, hist, n, qh, mask=ctx.array(bits_of(sees))).numpy()
    out = out.reshape(n, qh, hd)
    assert np.isfinite(out).all()
    every = [(i, h) for i in range(n) for h in range(qh)]
    pairs = every[:40] + every[-40:] + [every[j] for j in rng.integers(0, len(every), 80)]
    check(np.stack([out[i, h] for i, h in pairs]), *some_rows(q, k, v, hist, sees, pairs))
    cache.free()


@pytest.mark.parametrize("t, kvh, hd, cap", [(GGML.F32, 1, 128, (1 << 23) + 700), (GGML.Q8_0, 8, 128, (1 << 22) + 700),
                                             (GGML.F16, 2, 160, 6720000)], ids=["F32", "Q8_0", "any_dim"])
def test_positions_past_4_gib(ctx, t, kvh, hd, cap):
    """Stores, loads, moves and attention at rows whose bytes lie past 2^32 of their buffer.  Rows of zeros score 0 and
    weigh 1 each, so the few that are not give the result.  Sums of equal weights round the same way each time: up to
    2^-24 for each of the tiles of 32 that a wavefront adds up (a quarter of 1 / (256 / kvh) of all; in 64 bits where
    head_dim is no matrix instruction's)."""
    rng = np.random.default_rng(kvh)
    w, step, n, qh = kvh * hd, 1 << 15, 6, 2 * kvh
    cache = rf.KvCache(ctx, t, cap, kvh, hd)
    zeros = ctx.array(np.zeros((step, w), np.float32))
    for at in range(0, cap, step):
        rf.kv_store(ctx, cache, zeros, zeros, at, min(step, cap - at))
    hist = cap - 500
    assert hist * w * (4 if t == GGML.F32 else 2 if t == GGML.F16 else 1) > 1 << 32
    near, far = (rng.standard_normal((2, 40, w), np.float32) * 2 for _ in range(2))
    for (a, b), at in ((near, 100), (far, hist - 40 + n)):  # the last n are the drafts
        rf.kv_store(ctx, cache, ctx.array(a), ctx.array(b), at, 40)
    got = []
    for at in (100, hist - 40 + n):
        a, b = ctx.empty((40, w)), ctx.empty((40, w))
        rf.kv_load(ctx, cache, at, 40, a, b)
        got.append([x.numpy().reshape(40, kvh, hd) for x in (a, b)])
    assert np.abs(got[1][0].reshape(40, w) - far[0]).max() <= (0 if t == GGML.F32 else 0.07)  # half a step of 8 / 127
    q = rng.standard_normal((n, qh, hd), np.float32)
    out = rf.attention_tree(ctx, ctx.array(q), cache, hist, n, qh).numpy().reshape(n, qh, hd)
    k, v = (np.concatenate([got[0][i], got[1][i]]).astype(np.float64) for i in range(2))
    want, mag, plain = (np.zeros((n, qh, hd)) for _ in range(3))
    for i in range(n):
        seen = 80 - n + i + 1
        for h in range(qh):
            e = np.exp(k[:seen, h // 2] @ q[i, h].astype(np.float64) / np.sqrt(hd))
            p = e / (e.sum() + (hist + i + 1 - seen))
            want[i, h], mag[i, h], plain[i, h] = p @ v[:seen, h // 2], p @ np.abs(v[:seen, h // 2]), np.abs(v[:seen, h // 2]).sum(0)
    tiles = 0 if hd == 160 else cap / 32 / (4 * 256 / kvh)
    check(out, want, mag, plain, TOL + tiles * 2.0 ** -24)
    # the far rows move to the near ones' place and back
    rf.kv_move(ctx, [cache], ctx.array(np.arange(hist - 40 + n, hist + n, dtype=np.uint32)), 100, 40)
    a, b = ctx.empty((40, w)), ctx.empty((40, w))
    rf.kv_load(ctx, cache, 100, 40, a, b)
    assert np.array_equal(a.numpy().reshape(40, kvh, hd), got[1][0])
    rf.kv_move(ctx, [cache], ctx.array(np.full(1, 100, np.uint32)), cap - 1, 1)
    rf.kv_load(ctx, cache, cap - 1, 1, a, b)
    assert np.array_equal(b.numpy()[0].reshape(kvh, hd), got[1][1][0])
    zeros.free()
    cache.free()


def test_fixed_workspaces():
    """A reservation for the longest context and most tokens serves every shorter call; a smaller one refuses."""
    ctx = rf.Context(0)
    rng = np.random.default_rng(3)
    t, kvh, hd, qh, cap = GGML.Q8_0, 2, 64, 8, 6000
    need = ctx.attention_tree_workspace_bytes(cap, 40, t, qh, kvh, hd)
    assert need
    cache, k, v = big_cache(ctx, rng, t, cap, kvh, hd)
    q = rng.standard_normal((40, qh, hd), np.float32)
    qd, out = ctx.array(q), ctx.empty((40, qh * hd))
    ctx.reserve(attention_bytes=1024, fixed=True)
    with pytest.raises(rf.RamforgeError, match="reserved"):
        rf.attention_tree(ctx, qd, cache, cap - 40, 40, qh, out=out)
    ctx.reserve(attention_bytes=need, fixed=True)
    for n in (1, 2, 3, 5, 8, 9, 16, 17, 32, 33, 40):
        for hist in (0, 100, 127, 128, 1000, 3001, cap - n):
            rf.attention_tree(ctx, qd, cache, hist, n, qh, out=out)
        pairs = [(i, h) for i in range(n) for h in range(qh)]
        got = out.numpy().reshape(40, qh, hd)[:n]
        check(got.reshape(-1, hd), *some_rows(q[:n], k, v, cap - n, np.tri(n, dtype=bool), pairs))
    ctx.close()


def test_another_stream(ctx):
    """Calls on a stream of the caller's give what the context's own gives."""
    rng = np.random.default_rng(4)
    t, kvh, hd, qh, n, hist = GGML.Q4_0, 2, 128, 8, 12, 3000
    cache, k, v = big_cache(ctx, rng, t, hist + 40, kvh, hd)
    row = (qh + 2 * kvh) * hd
    qkv = ctx.array(rng.standard_normal((n, row), np.float32))
    parents, mask, pos = ctx.array(tree(rng, n)), ctx.empty((n, 1), np.uint64), ctx.empty((n,), np.uint32)
    src = ctx.array(np.arange(hist + 2, hist + 7, dtype=np.uint32))
    before = cache.k.numpy(), cache.v.numpy()
    got = []
    for stream in (None, ctx.copy_stream):
        cache.k.upload(before[0])
        cache.v.upload(before[1])
        q, out = ctx.array(np.zeros((n, qh * hd), np.float32)), ctx.array(np.zeros((n, qh * hd), np.float32))
        ctx.synchronize()
        rf.tree_mask(ctx, parents, n, hist, mask, pos, stream=stream)
        rf.qk_norm_rope_store(ctx, qkv.ptr, qkv.ptr + 4 * qh * hd, qkv.ptr + 4 * (qh + kvh) * hd, None, None, 1e-6, pos,
                              n, qh, 1e4, q, cache, hist, q_stride=row, k_stride=row, v_stride=row, stream=stream)
        rf.attention_tree(ctx, q, cache, hist, n, qh, mask=mask, out=out, stream=stream)
        rf.kv_move(ctx, [cache], src, hist, 5, stream=stream)
        ctx.synchronize()
        got.append((q.numpy(), out.numpy(), cache.k.numpy(), cache.v.numpy()))
    for a, b in zip(*got):
        assert np.array_equal(a, b)
    cache.free()


@pytest.mark.parametrize("t", TYPES, ids=lambda t: GGML.NAMES[t])
def test_a_step_captured(ctx, t):
    """Two steps of drafts captured into graphs that share the attention workspace, replayed in turn with eager work
    between them; every replay is the eager step, bit for bit, as the length word grows."""
    rng = np.random.default_rng(6)
    kvh, hd, qh, cap, layers = 2, 64, 8, 4000, 3
    row = (qh + 2 * kvh) * hd
    length = ctx.array(np.array([0], np.uint32))
    made = [big_cache(ctx, rng, t, cap, kvh, hd)[0] for _ in range(layers)]
    caches = [rf.KvCache(ctx, t, cap, kvh, hd, c.k, c.v, length=length) for c in made]
    both = rf.KvCacheList(caches)
    start = [(c.k.numpy(), c.v.numpy()) for c in made]

    def step(n, s):
        parents, mask, pos, q, outs, src = s
        rf.tree_mask(ctx, parents, n, 0, mask, pos, length=length)
        for c, qkv, o in zip(caches, s_qkv[n], outs):
            rf.qk_norm_rope_store(ctx, qkv.ptr, qkv.ptr + 4 * qh * hd, qkv.ptr + 4 * (qh + kvh) * hd, None, None, 1e-6,
                                  pos, n, qh, 1e4, q, c, 0, q_stride=row, k_stride=row, v_stride=row)
            rf.attention_tree(ctx, q, c, 0, n, qh, mask=mask, out=o)
        rf.kv_move(ctx, both, src, 0, 2)

    s_qkv, state, graphs = {}, {}, {}
    for n in (5, 70):
        s_qkv[n] = [ctx.array(rng.standard_normal((n, row), np.float32)) for _ in range(layers)]
        state[n] = (ctx.array(tree(rng, n)), ctx.empty((n, (n + 63) // 64), np.uint64), ctx.empty((n,), np.uint32),
                    ctx.empty((n, qh * hd)), [ctx.empty((n, qh * hd)) for _ in range(layers)],
                    ctx.array(np.array([1, 4], np.uint32)))
        step(n, state[n])
    for n in (5, 70):
        with ctx.capture() as c:
            step(n, state[n])
        graphs[n] = c.graph

    def outcome(n, at, run):
        for c, (k, v) in zip(made, start):
            c.k.upload(k)
            c.v.upload(v)
        length.upload(np.array([at], np.uint32))
        for o in state[n][4]:
            o.upload(np.full((n, qh * hd), np.nan, np.float32))
        run()
        ctx.synchronize()
        return [o.numpy() for o in state[n][4]] + [x.numpy() for c in made for x in (c.k, c.v)]

    for at in (0, 31, 3900, 700):
        for n in (70, 5):
            want = outcome(n, at, lambda: step(n, state[n]))
            for _ in range(2):
                got = outcome(n, at, graphs[n].replay)
                assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(got, want))
    for g in graphs.values():
        g.close()
    for c in made:
        c.free()


@pytest.mark.parametrize("t", TYPES, ids=lambda t: GGML.NAMES[t])
@pytest.mark.parametrize("n, hist, kvh, hd", [(6, 700, 2, 128), (40, 64, 1, 64), (9, 50, 1, 160), (64, 4097, 1, 64),
                                              (1024, 42000, 1, 64)])
def test_queries_that_are_not_finite(ctx, t, n, hist, kvh, hd):
    """A NaN or infinity in a query makes its own row's output NaN and reaches no other row."""
    rng = np.random.default_rng(n)
    qh = kvh if n > 1000 else 4 * kvh
    cache, k, v = big_cache(ctx, rng, t, hist + n, kvh, hd)
    q = rng.standard_normal((n, qh, hd), np.float32)
    q[1, 0, 5], q[4, qh - 1, hd - 1], q[n - 2, 0, 0] = np.nan, np.inf, -np.inf
    q[3, 0] = 0
    out = rf.attention_tree(ctx, ctx.array(q), cache, hist, n, qh).numpy().reshape(n, qh, hd)
    bad = {(1, 0), (4, qh - 1), (n - 2, 0)}
    assert all(np.isnan(out[i, h]).all() for i, h in bad)
    every = [(i, h) for i in range(n) for h in range(qh) if (i, h) not in bad]
    pairs = every[:60] + every[-60:]
    check(np.stack([out[i, h] for i, h in pairs]), *some_rows(q, k, v, hist, np.tri(n, dtype=bool), pairs))
    cache.free()


def test_many_steps_on_two_streams_in_order(ctx):
    """Calls that alternate between two streams, ordered by waiting for each, share the attention workspace."""
    rng = np.random.default_rng(9)
    t, kvh, hd, qh, n, hist = GGML.Q8_0, 2, 64, 8, 8, 2500
    cache, k, v = big_cache(ctx, rng, t, hist + n, kvh, hd)
    q = [rng.standard_normal((n, qh, hd), np.float32) for _ in range(4)]
    dev, outs = [ctx.array(x) for x in q], [ctx.empty((n, qh * hd)) for _ in q]
    for _ in range(3):
        for i in range(4):
            rf.attention_tree(ctx, dev[i], cache, hist, n, qh, out=outs[i], stream=ctx.copy_stream if i % 2 else None)
            ctx.synchronize()
    pairs = [(i, h) for i in range(n) for h in range(qh)]
    for x, o in zip(q, outs):
        check(o.numpy().reshape(-1, hd), *some_rows(x, k, v, hist, np.tri(n, dtype=bool), pairs))
    cache.free()


@pytest.mark.parametrize("n, offset", [(8500000, 0), (2100003, 1)], ids=["vector", "any"])
def test_more_rows_than_one_grid(ctx, n, offset):
    """Stores and loads of more rows than 65536 workgroups take at once, by both kernels: every row comes back."""
    w = 32
    block = np.random.default_rng(n).standard_normal(1000003, np.float32)
    x = np.resize(block, n * w + offset)
    d = ctx.array(x)
    cache = rf.KvCache(ctx, GGML.F32, n, 1, w)
    rf.kv_store(ctx, cache, d.ptr + 4 * offset, d.ptr + 4 * offset, 0, n)
    d.upload(np.zeros_like(x))
    rf.kv_load(ctx, cache, 0, n, d.ptr + 4 * offset, d.ptr + 4 * offset)
    assert np.array_equal(d.numpy()[offset:], x[offset:])
    d.free()
    cache.free()


def test_more_tokens_than_one_grid(ctx):
    """Norm and rotation of 70001 tokens: the last equal a call of their own."""
    rng = np.random.default_rng(1)
    n, qh, kvh, hd, m = 70001, 2, 1, 16, 4500
    q, k = rng.standard_normal((n, qh * hd), np.float32), rng.standard_normal((n, kvh * hd), np.float32)
    pos = rng.integers(0, 1 << 17, n).astype(np.uint32)
    got = []
    for at in (0, n - m):
        c = n - at
        qo, ko = ctx.empty((c, qh * hd)), ctx.empty((c, kvh * hd))
        rf.qk_norm_rope(ctx, ctx.array(q[at:]), ctx.array(k[at:]), None, None, 1e-6, ctx.array(pos[at:]), c, qh, kvh,
                        hd, 1e4, qo, ko)
        got.append((qo.numpy(), ko.numpy()))
    for a, b in zip(*got):
        assert np.array_equal(a[n - m:], b)
