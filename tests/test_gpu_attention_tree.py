"""Attention of drafted tokens over a cache in few bits (rf_attention_tree, rf_tree_mask) against its definition in
64 bits (numpy), on the values that the cache gives back.

Tolerance, before any run: relative to sum_p softmax_p |v_p| per output.  A score is a sum of head_dim products in
f32 (or in two f16 pieces, 2^-22 each): at most head_dim roundings, at random about sqrt(head_dim) 2^-24 of
|q| |k| / sqrt(head_dim); with unit normal q and k scores reach about 6 and sum |q k| / sqrt(head_dim) about
sqrt(head_dim), so a score is off by less than 16 * 2^-24 * 4 = 4e-6 and a weight by as much, relatively; the weights'
own pieces, exp and the sums over positions add about as much again.  1e-5 is asked for.

Weights are two f16 pieces of w * 2^e with the largest between 2^12 and 2^15: below 2^-14 the pieces are subnormal
halves, whole multiples of 2^-24, so a weight is off by up to 2^-25 / 2^12 = 2^-37 of the row's largest however small
it is, and an output by 2^-37 sum_p |v_p| more.  (It shows only where the largest weights meet values of zero.)"""
import numpy as np
import pytest

import ramforge_amd as rf
from ramforge_amd import GGML

pytestmark = pytest.mark.gpu

TOL = 1e-5
TYPES = [GGML.F32, GGML.F16, GGML.Q8_0, GGML.Q4_0]


def tree(rng, n):
    return np.array([int(rng.integers(-1, i)) if rng.random() < 0.4 else i - 1 for i in range(n)], np.int32)


def sees_of(parents):
    n = len(parents)
    sees = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            sees[i] = sees[p]
        sees[i, i] = True
    return sees


def bits_of(sees):
    """[n][ceil(n / 64)] uint64"""
    n = len(sees)
    out = np.zeros((n, (n + 63) // 64), np.uint64)
    for i, j in zip(*np.nonzero(sees)):
        out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out


def definition(q, k, v, hist, sees):
    """q [n, qh, hd], k, v [hist + n, kvh, hd]; returns the result, sum softmax |v| and sum |v|, f64."""
    n, qh, hd = q.shape
    kvh = k.shape[1]
    every = np.concatenate([np.ones((n, hist), bool), sees], 1)
    out, mag, plain = (np.zeros((n, qh, hd)) for _ in range(3))
    for h in range(qh):
        kk, vv = k[:, h * kvh // qh].astype(np.float64), v[:, h * kvh // qh].astype(np.float64)
        for i in range(n):
            at = every[i]
            if not at.any():
                continue
            s = kk[at] @ q[i, h].astype(np.float64) / np.sqrt(hd)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h], mag[i, h], plain[i, h] = p @ vv[at], p @ np.abs(vv[at]), np.abs(vv[at]).sum(0)
    return out, mag, plain


def filled(ctx, rng, t, cap, kvh, hd, rows=None, scale=1.0):
    """A cache of normal rows and the values it gives back."""
    rows = cap if rows is None else rows
    w = kvh * hd
    cache = rf.KvCache(ctx, t, cap, kvh, hd)
    k, v = ((scale * rng.normal(0, 1, (rows, w))).astype(np.float32) for _ in range(2))
    kd, vd = ctx.array(k), ctx.array(v)
    rf.kv_store(ctx, cache, kd, vd, 0, rows)
    rf.kv_load(ctx, cache, 0, rows, kd, vd)
    got = [x.numpy().reshape(rows, kvh, hd) for x in (kd, vd)]
    kd.free()
    vd.free()
    return (cache, *got)


def check(got, want, mag, plain, tol=TOL):
    err = np.maximum(np.abs(got - want) - 2.0 ** -37 * plain, 0) / np.maximum(mag, 1e-30)
    ok, worst = bool(np.isfinite(got).all()), float(err.max())
    assert ok and worst <= tol, worst


SHAPES = [  # tokens, history, query heads, KV heads, head_dim
    (1, 0, 8, 2, 128), (1, 1, 8, 8, 64), (1, 2047, 32, 8, 128), (16, 1000, 32, 8, 128), (7, 1501, 14, 2, 64),
    (37, 600, 12, 2, 128), (5, 31, 6, 3, 96), (70, 333, 4, 1, 128), (33, 64, 4, 2, 256), (130, 90, 2, 2, 64),
    (200, 500, 8, 1, 128), (3, 5000, 8, 1, 64), (64, 0, 8, 4, 96), (9, 4097, 16, 1, 256), (2, 33, 40, 1, 128),
    (1, 9000, 8, 8, 128), (4, 700, 3, 1, 32), (11, 100, 2, 1, 160),
]


@pytest.mark.parametrize("t", TYPES, ids=lambda t: GGML.NAMES[t])
@pytest.mark.parametrize("n, hist, qh, kvh, hd", SHAPES)
def test_tree_attention(ctx, t, n, hist, qh, kvh, hd):
    rng = np.random.default_rng(n * 7 + hist + qh + hd + t)
    cache, k, v = filled(ctx, rng, t, hist + n + 3, kvh, hd)
    q = rng.normal(0, 1, (n, qh, hd)).astype(np.float32)
    parents = tree(rng, n)
    sees = sees_of(parents)
    mask, pos = ctx.empty((n, (n + 63) // 64), np.uint64), ctx.empty((n,), np.uint32)
    rf.tree_mask(ctx, ctx.array(parents), n, hist, mask, pos)
    assert np.array_equal(mask.numpy(), bits_of(sees))
    assert np.array_equal(pos.numpy(), hist + sees.sum(1) - 1)
    out = rf.attention_tree(ctx, ctx.array(q), cache, hist, n, qh, mask=mask)
    check(out.numpy().reshape(n, qh, hd), *definition(q, k[:hist + n], v[:hist + n], hist, sees))
    # without a mask: a chain
    out = rf.attention_tree(ctx, ctx.array(q), cache, hist, n, qh)
    check(out.numpy().reshape(n, qh, hd), *definition(q, k[:hist + n], v[:hist + n], hist, np.tri(n, dtype=bool)))
    cache.free()


@pytest.mark.parametrize("kvh, hd", [(3, 10), (1, 7), (2, 1), (1, 300)])
def test_any_head_dim(ctx, kvh, hd):
    rng = np.random.default_rng(hd)
    for t in (GGML.F32, GGML.F16):
        n, hist, qh = 6, 300, 2 * kvh
        cache, k, v = filled(ctx, rng, t, hist + n, kvh, hd)
        q = rng.normal(0, 1, (n, qh, hd)).astype(np.float32)
        sees = sees_of(tree(rng, n))
        out = rf.attention_tree(ctx, ctx.array(q), cache, hist, n, qh, mask=ctx.array(bits_of(sees)))
        check(out.numpy().reshape(n, qh, hd), *definition(q, k, v, hist, sees))
        cache.free()


@pytest.mark.parametrize("t", TYPES, ids=lambda t: GGML.NAMES[t])
@pytest.mark.parametrize("hd", [64, 128, 160])
def test_rows_that_see_nothing(ctx, t, hd):
    """Without a history, rows of zero masks give zeros, the others theirs; bits past the last token are no tokens."""
    rng = np.random.default_rng(hd)
    n, qh, kvh = 70, 4, 2
    cache, k, v = filled(ctx, rng, t, n, kvh, hd)
    q = rng.normal(0, 1, (n, qh, hd)).astype(np.float32)
    sees = rng.random((n, n)) < 0.1
    sees[[0, 17, 40, 69]] = False
    sees[:, 33] = False
    bits = bits_of(sees)
    bits[:, 1] |= np.uint64(0xFFFFFFFFFFFFFFFF) << np.uint64(n - 64)
    out = rf.attention_tree(ctx, ctx.array(q), cache, 0, n, qh, mask=ctx.array(bits)).numpy().reshape(n, qh, hd)
    assert (out[[0, 17, 40, 69]] == 0).all()
    check(out, *definition(q, k, v, 0, sees))
    cache.free()


@pytest.mark.parametrize("t", TYPES, ids=lambda t: GGML.NAMES[t])
@pytest.mark.parametrize("hd, hist", [(128, 100), (64, 0), (160, 40), (256, 31), (96, 1000)])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf, 3e38])
def test_masked_infinities_and_nan(ctx, t, hd, hist, what):
    """What a token does not see cannot reach it: a drafted row of infinities or NaN, and rows behind the last."""
    rng = np.random.default_rng(hd + hist)
    n, qh, kvh = 20, 6, 2
    cap, w = hist + n + 50, 2 * hd
    cache, k, v = filled(ctx, rng, t, cap, kvh, hd)
    bad = ctx.array(np.full((50, w), what, np.float32))
    rf.kv_store(ctx, cache, bad, bad, hist + n, 50)
    rf.kv_store(ctx, cache, bad, bad, hist + 7, 1)
    rf.kv_store(ctx, cache, bad, bad, hist + 13, 1)
    q = rng.normal(0, 1, (n, qh, hd)).astype(np.float32)
    sees = sees_of(tree(rng, n))
    sees[:, 7] = sees[:, 13] = False
    sees[19, 13] = True  # one row sees one of them
    out = rf.attention_tree(ctx, ctx.array(q), cache, hist, n, qh, mask=ctx.array(bits_of(sees))).numpy()
    out = out.reshape(n, qh, hd)
    check(out[:19], *definition(q[:19], k[:hist + n], v[:hist + n], hist, sees[:19]))
    if not (what == 3e38 and t not in (GGML.F16,)):
        assert not np.isfinite(out[19]).any()
    cache.free()


@pytest.mark.parametrize("t", TYPES, ids=lambda t: GGML.NAMES[t])
@pytest.mark.parametrize("scale, qscale", [(1e-3, 1.0), (30.0, 1.0), (1.0, 1e-6), (1.0, 40.0), (300.0, 0.01)])
def test_magnitudes(ctx, t, scale, qscale):
    """Small and large rows and queries: sharp softmaxes, flat ones, values near the formats' ends.  A score's error
    grows with its size, so the tolerance does where scores are large."""
    rng = np.random.default_rng(int(scale * 7 + qscale))
    n, hist, qh, kvh, hd = 9, 700, 8, 2, 128
    cache, k, v = filled(ctx, rng, t, hist + n, kvh, hd, scale=scale)
    q = (qscale * rng.normal(0, 1, (n, qh, hd))).astype(np.float32)
    sees = sees_of(tree(rng, n))
    out = rf.attention_tree(ctx, ctx.array(q), cache, hist, n, qh, mask=ctx.array(bits_of(sees)))
    check(out.numpy().reshape(n, qh, hd), *definition(q, k, v, hist, sees), tol=TOL * max(1.0, scale * qscale))
    cache.free()


@pytest.mark.parametrize("t", TYPES, ids=lambda t: GGML.NAMES[t])
def test_uneven_weights_and_rows(ctx, t):
    """The largest score late, values that span nine orders between positions, one query much larger than the rest."""
    rng = np.random.default_rng(21)
    n, hist, qh, kvh, hd = 5, 900, 4, 2, 128
    w = kvh * hd
    k = rng.normal(0, 1, (hist + n, w)).astype(np.float32)
    v = (rng.normal(0, 1, (hist + n, w)) * 10.0 ** rng.uniform(-3, 3, (hist + n, 1))).astype(np.float32)
    q = rng.normal(0, 1, (n, qh, hd)).astype(np.float32)
    q[2] *= 30
    q[3] = 0
    k[-n - 1] = 3 * np.tile(q[0, 0], kvh)
    cache = rf.KvCache(ctx, t, hist + n, kvh, hd)
    kd, vd = ctx.array(k), ctx.array(v)
    rf.kv_store(ctx, cache, kd, vd, 0, hist + n)
    rf.kv_load(ctx, cache, 0, hist + n, kd, vd)
    k, v = kd.numpy().reshape(-1, kvh, hd), vd.numpy().reshape(-1, kvh, hd)
    out = rf.attention_tree(ctx, ctx.array(q), cache, hist, n, qh).numpy().reshape(n, qh, hd)
    want = definition(q, k, v, hist, np.tri(n, dtype=bool))
    # scores of the scaled query reach 30 times the others'
    check(out[[0, 1, 3, 4]], *(x[[0, 1, 3, 4]] for x in want), 2 * TOL)
    check(out[[2]], *(x[[2]] for x in want), 30 * TOL)
    cache.free()


def test_strides_and_alignment(ctx):
    """q inside a wider row at 4 bytes' alignment, out rows with gaps that stay."""
    rng = np.random.default_rng(8)
    for t, hd in ((GGML.Q8_0, 128), (GGML.F16, 64), (GGML.F32, 96), (GGML.F32, 33)):
        n, hist, qh, kvh = 6, 200, 4, 2
        cache, k, v = filled(ctx, rng, t, hist + n, kvh, hd)
        wide = rng.normal(0, 1, (n, qh * hd + 9)).astype(np.float32)
        q = wide[:, 5:5 + qh * hd].reshape(n, qh, hd)
        d, o = ctx.array(wide), ctx.array(np.full((n, qh * hd + 3), 9, np.float32))
        rf.attention_tree(ctx, d.ptr + 20, cache, hist, n, qh, out=o.ptr + 4, q_stride=qh * hd + 9,
                          out_stride=qh * hd + 3)
        got = o.numpy()
        assert (got[:, 0] == 9).all() and (got[:, qh * hd + 1:] == 9).all()
        check(got[:, 1:1 + qh * hd].reshape(n, qh, hd), *definition(q, k, v, hist, np.tri(n, dtype=bool)))
        cache.free()


@pytest.mark.parametrize("t", TYPES, ids=lambda t: GGML.NAMES[t])
def test_captured_over_a_growing_cache(ctx, t):
    """A captured call follows the length word; replays with work between them equal the eager calls."""
    rng = np.random.default_rng(17)
    n, cap, qh, kvh, hd = 4, 1200, 8, 2, 128
    cache, k, v = filled(ctx, rng, t, cap, kvh, hd)
    length = ctx.array(np.array([500], np.uint32))
    moving = rf.KvCache(ctx, t, cap, kvh, hd, cache.k, cache.v, length=length)
    q = rng.normal(0, 1, (n, qh, hd)).astype(np.float32)
    qd, out = ctx.array(q), ctx.empty((n, qh * hd))
    mask = ctx.array(bits_of(sees_of(np.array([-1, 0, 0, 2]))))
    rf.attention_tree(ctx, qd, moving, 0, n, qh, mask=mask, out=out)
    with ctx.capture() as c:
        rf.attention_tree(ctx, qd, moving, 0, n, qh, mask=mask, out=out)
    for at in (0, 1, 63, 900, 1196, 500):
        length.upload(np.array([at], np.uint32))
        out.upload(np.full((n, qh * hd), np.nan, np.float32))
        c.graph.replay()
        ctx.synchronize()
        got = out.numpy().reshape(n, qh, hd)
        check(got, *definition(q, k[:at + n], v[:at + n], at, sees_of(np.array([-1, 0, 0, 2]))))
        rf.attention_tree(ctx, qd, moving, 0, n, qh, mask=mask, out=out)
        assert np.array_equal(out.numpy().reshape(n, qh, hd), got)
    # past the capacity: what lies inside is seen, and nothing else is read
    for at in (1198, 1200, 0xFFFFFFF0):
        length.upload(np.array([at], np.uint32))
        rf.attention_tree(ctx, qd, moving, 0, n, qh, mask=mask, out=out)
        h = min(at, cap)
        m = cap - h
        sees = sees_of(np.array([-1, 0, 0, 2]))[:, :m]
        got = out.numpy().reshape(n, qh, hd)
        check(got, *definition(q, k, v, h, sees))
    c.graph.close()
    cache.free()


def test_mask_of_bad_parents(ctx):
    """A parent that is no earlier token counts as the history."""
    for parents in ([5, 0, 1], [0, 1, 2, 3], [-7, 2 ** 31 - 1, 0], [-1], [-1] * 200, list(range(-1, 1023))):
        p = np.array(parents, np.int32)
        n = len(p)
        mask, pos = ctx.empty((n, (n + 63) // 64), np.uint64), ctx.empty((n,), np.uint32)
        rf.tree_mask(ctx, ctx.array(p), n, 10, mask, pos, length=ctx.array(np.array([90], np.uint32)))
        sees = sees_of(p)
        assert np.array_equal(mask.numpy(), bits_of(sees))
        assert np.array_equal(pos.numpy(), 100 + sees.sum(1) - 1)


@pytest.mark.parametrize("t", [GGML.F32, GGML.Q8_0], ids=["F32", "Q8_0"])
def test_a_step_of_drafts(ctx, t):
    """Mask, norm and rotation into the cache, attention, and the move of the accepted path, as a step uses them:
    the next step's tokens see the accepted rows as their history."""
    rng = np.random.default_rng(2)
    n, hist, qh, kvh, hd, layers = 8, 40, 8, 2, 64, 2
    cap, theta = 128, 1e4
    parents = np.array([-1, 0, 0, 1, 1, 2, 3, 6], np.int32)
    path = [0, 1, 3, 6]
    wq, wk = (1 + 0.2 * rng.normal(0, 1, hd).astype(np.float32) for _ in range(2))
    dwq, dwk = ctx.array(wq), ctx.array(wk)
    state = [filled(ctx, rng, t, cap, kvh, hd, rows=hist) for _ in range(layers)]
    mask, pos = ctx.empty((n, 1), np.uint64), ctx.empty((n,), np.uint32)
    rf.tree_mask(ctx, ctx.array(parents), n, hist, mask, pos)
    sees = sees_of(parents)
    q_out, out = ctx.empty((n, qh * hd)), ctx.empty((n, qh * hd))
    ko, vo = ctx.empty((cap, kvh * hd)), ctx.empty((cap, kvh * hd))
    kept = []
    for cache, k, v in state:
        qkv = rng.normal(0, 1, (n, qh + 2 * kvh, hd)).astype(np.float32)
        d = ctx.array(qkv)
        row = (qh + 2 * kvh) * hd
        rf.qk_norm_rope_store(ctx, d.ptr, d.ptr + 4 * qh * hd, d.ptr + 4 * (qh + kvh) * hd, dwq, dwk, 1e-6, pos, n,
                              qh, theta, q_out, cache, hist, q_stride=row, k_stride=row, v_stride=row)
        rf.attention_tree(ctx, q_out, cache, hist, n, qh, mask=mask, out=out)
        rf.kv_load(ctx, cache, 0, cap, ko, vo)
        kk, vv = (x.numpy().reshape(cap, kvh, hd)[:hist + n] for x in (ko, vo))
        assert np.array_equal(kk[:hist], k) and np.array_equal(vv[:hist], v)
        check(out.numpy().reshape(n, qh, hd), *definition(q_out.numpy().reshape(n, qh, hd), kk, vv, hist, sees))
        kept.append((np.concatenate([kk[:hist], kk[hist:][path]]), np.concatenate([vv[:hist], vv[hist:][path]])))
    rf.kv_move(ctx, [s[0] for s in state], ctx.array(np.array([hist + i for i in path], np.uint32)), hist, len(path))
    hist += len(path)
    for (cache, _, _), (k, v) in zip(state, kept):
        new = rng.normal(0, 1, (1, 2, kvh * hd)).astype(np.float32)
        d = ctx.array(new)
        rf.kv_store(ctx, cache, d.ptr, d.ptr + 4 * kvh * hd, hist, 1)
        q = rng.normal(0, 1, (1, qh, hd)).astype(np.float32)
        got = rf.attention_tree(ctx, ctx.array(q), cache, hist, 1, qh)
        rf.kv_load(ctx, cache, 0, cap, ko, vo)
        kk, vv = (x.numpy().reshape(cap, kvh, hd)[:hist + 1] for x in (ko, vo))
        assert np.array_equal(kk[:hist], k) and np.array_equal(vv[:hist], v)
        check(got.numpy().reshape(1, qh, hd), *definition(q, kk, vv, hist, np.ones((1, 1), bool)))
        cache.free()
