"""The K/V cache in few bits (rf_kv_store, rf_kv_load, rf_kv_move) and the norm and rotation that write into it,
against definitions in 64 bits (numpy).

Tolerances, before any run: what a Q8_0 or Q4_0 cache gives back of given rows is defined exactly, and equal.
A norm over h values and a rotation in f32: the sum of squares, the root, two products and the rotation's two
products and sum are at most h / 2 + 8 roundings of 2^-24 on the longest chain, the cosines' error 2^-22; each
relative to the pair's length.  2e-6 covers h = 512 with its sums taken in 8 to 64 parallel chains.  An angle of
position p is rounded in 64 bits about three times on either side: p * 2^-52 * 3 radians more."""
import numpy as np
import pytest

import ramforge_amd as rf
from ramforge_amd import GGML

pytestmark = pytest.mark.gpu

TYPES = [GGML.F32, GGML.F16, GGML.Q8_0, GGML.Q4_0]
LEVELS = {GGML.Q8_0: 127, GGML.Q4_0: 8}


def quantised(x, t):
    """What a cache of type t gives back for x: per 32 values, by the definition in ramforge_hip.h."""
    if t == GGML.F32:
        return x.astype(np.float32)
    if t == GGML.F16:
        return x.astype(np.float16).astype(np.float32)
    with np.errstate(all="ignore"):
        b = x.astype(np.float64).reshape(-1, 32)
        whole = np.isfinite(b).all(1)
        b = np.where(whole[:, None], b, 0)
        top, lv, bits, most = np.abs(b).max(1), LEVELS[t], 3 if t == GGML.Q8_0 else 8, 512 if t == GGML.Q8_0 else 8160
        want = top / lv  # f64: no multiple of the grid lies between it and the quotient
        step = np.ldexp(1.0, np.maximum(np.frexp(want)[1] - bits, -24))
        d = np.minimum(np.ceil(want / step) * step, most)
        if t == GGML.Q4_0:
            d = np.where(b.max(1) > -b.min(1), -d, d)
        q = np.clip(np.rint(b / np.where(d == 0, 1, d)[:, None]), -lv, 127 if t == GGML.Q8_0 else 7)
        return np.where(whole[:, None], q * d[:, None], np.nan).astype(np.float32).reshape(x.shape)


def rows(rng, n, width):
    """Values of many magnitudes, with zeros, ties and blocks of one sign."""
    x = rng.normal(0, 1, (n, width)) * np.exp(rng.normal(0, 2, (n, 1)))
    x[rng.random((n, width)) < 0.02] = 0
    if n > 2:
        x[1] = np.round(x[1] * 4) / 8  # multiples that meet half steps
        x[2] = np.abs(x[2])
    return x.astype(np.float32)


def equal(a, b):
    assert np.array_equal(a, b, equal_nan=True), np.nanmax(np.abs(a - b))


@pytest.mark.parametrize("t", TYPES, ids=lambda t: GGML.NAMES[t])
@pytest.mark.parametrize("n, kvh, hd", [(1, 8, 128), (17, 8, 128), (5, 1, 64), (3, 3, 96), (700, 2, 256), (2, 5, 32),
                                        (4, 1, 512), (9, 24, 128), (1, 1, 32)])
def test_store_and_load(ctx, t, n, kvh, hd):
    rng = np.random.default_rng(n * 1000 + hd + t)
    w, first, cap = kvh * hd, 3, n + 5
    cache = rf.KvCache(ctx, t, cap, kvh, hd)
    before = rng.integers(0, 255, cache.k.nbytes, dtype=np.uint8)
    cache.k.upload(before)
    cache.v.upload(before)
    k, v = rows(rng, n, w), rows(rng, n, w)
    rf.kv_store(ctx, cache, ctx.array(k), ctx.array(v), first, n)
    ko, vo = ctx.empty((n, w)), ctx.empty((n, w))
    rf.kv_load(ctx, cache, first, n, ko, vo)
    equal(ko.numpy(), quantised(k, t))
    equal(vo.numpy(), quantised(v, t))
    # nothing outside the rows was written
    codes = w * {GGML.F32: 4, GGML.F16: 2, GGML.Q8_0: 1, GGML.Q4_0: 0.5}[t]
    scales = w // 16 if t in LEVELS else 0
    for buf in (cache.k, cache.v):
        after = buf.numpy()
        kept = np.ones(len(after), bool)
        kept[int(first * codes):int((first + n) * codes)] = False
        at = int(cap * codes)
        kept[at + first * scales:at + (first + n) * scales] = False
        assert np.array_equal(after[kept], before[kept])
    cache.free()


@pytest.mark.parametrize("t", [GGML.F32, GGML.F16], ids=["F32", "F16"])
def test_any_head_dim(ctx, t):
    """Rows that are no whole number of 16-byte pieces."""
    rng = np.random.default_rng(3)
    for kvh, hd in ((3, 10), (1, 7), (5, 1)):
        w = kvh * hd
        cache = rf.KvCache(ctx, t, 9, kvh, hd)
        k, v = rows(rng, 6, w), rows(rng, 6, w)
        rf.kv_store(ctx, cache, ctx.array(k), ctx.array(v), 2, 6)
        ko, vo = ctx.empty((6, w)), ctx.empty((6, w))
        rf.kv_load(ctx, cache, 2, 6, ko, vo)
        equal(ko.numpy(), quantised(k, t))
        equal(vo.numpy(), quantised(v, t))
        cache.free()


@pytest.mark.parametrize("t", [GGML.Q8_0, GGML.Q4_0], ids=["Q8_0", "Q4_0"])
def test_edges_of_the_formats(ctx, t):
    """Zeros, the smallest and largest magnitudes, signs, ties, infinities and NaN, one block each."""
    lv = LEVELS[t]
    b = np.zeros((16, 32), np.float32)
    b[1, 5] = 1e-45
    b[2, :] = 2.0 ** -24 * np.arange(32)
    b[3, :] = 1e-7 * np.linspace(-1, 1, 32)
    b[4, 0] = lv * 0.25
    b[5, :] = 0.25 * (np.arange(32) - 15.5)
    b[5, 0] = -lv * 0.25  # the scale is 0.25 and every other value a tie
    b[6, :] = [lv * 1.0, -lv * 1.0] * 16
    b[7, 3] = 3e38
    b[7, 4] = -12345
    b[8, 9] = np.inf
    b[9, 31] = np.nan
    b[10, :] = -np.abs(np.linspace(0.001, 1, 32))
    b[11, :] = np.abs(np.linspace(0.001, 1, 32))
    b[12, 0] = np.nextafter(np.float32(lv * 0.25), np.float32(1e9))
    b[13, 0] = np.nextafter(np.float32(lv * 0.25), np.float32(0))
    b[14, 0] = -np.inf
    b[15, :] = 65504.0 * np.linspace(-1, 1, 32)
    x = b.reshape(1, -1)
    cache = rf.KvCache(ctx, t, 1, 4, 128)
    rf.kv_store(ctx, cache, ctx.array(x), ctx.array(-x), 0, 1)
    ko, vo = ctx.empty((1, 512)), ctx.empty((1, 512))
    rf.kv_load(ctx, cache, 0, 1, ko, vo)
    equal(ko.numpy(), quantised(x, t))
    equal(vo.numpy(), quantised(-x, t))
    cache.free()


def test_strided_and_misaligned_rows(ctx):
    """Rows inside a wider projection output, at addresses of 4 bytes' alignment."""
    rng = np.random.default_rng(11)
    n, kvh, hd, stride = 13, 2, 64, 401
    w = kvh * hd
    for t in TYPES:
        src = rng.normal(0, 1, (n, stride)).astype(np.float32)
        d = ctx.array(src)
        cache = rf.KvCache(ctx, t, n, kvh, hd)
        rf.kv_store(ctx, cache, d.ptr + 4 * 7, d.ptr + 4 * 201, 0, n, k_stride=stride, v_stride=stride)
        out = ctx.array(np.full((n, stride), 7, np.float32))
        rf.kv_load(ctx, cache, 0, n, out.ptr + 4 * 3, out.ptr + 4 * 203, k_stride=stride, v_stride=stride)
        o = out.numpy()
        equal(o[:, 3:3 + w], quantised(np.ascontiguousarray(src[:, 7:7 + w]), t))
        equal(o[:, 203:203 + w], quantised(np.ascontiguousarray(src[:, 201:201 + w]), t))
        assert (o[:, :3] == 7).all() and (o[:, 203 + w:] == 7).all() and (o[:, 3 + w:203] == 7).all()
        cache.free()


@pytest.mark.parametrize("t", TYPES, ids=lambda t: GGML.NAMES[t])
@pytest.mark.parametrize("layers, n, kvh, hd", [(32, 5, 8, 128), (3, 1, 1, 32), (70, 9, 2, 64), (2, 1024, 1, 128),
                                                (4, 300, 3, 96)])
def test_move(ctx, t, layers, n, kvh, hd):
    """Targets that are sources too, the same source twice, a source past the capacity."""
    rng = np.random.default_rng(layers + n)
    cap = n + 40
    caches = [rf.KvCache(ctx, t, cap, kvh, hd) for _ in range(layers)]
    w = kvh * hd
    values = []
    for c in caches:
        k, v = rng.normal(0, 1, (cap, w)).astype(np.float32), rng.normal(0, 1, (cap, w)).astype(np.float32)
        rf.kv_store(ctx, c, ctx.array(k), ctx.array(v), 0, cap)
        values.append((quantised(k, t), quantised(v, t)))
    first = 20
    src = rng.integers(0, cap, n).astype(np.uint32)
    if n > 4:
        src[3] = src[1]
        src[2] = cap + 5
        src[4] = 0xFFFFFFFF
    rf.kv_move(ctx, rf.KvCacheList(caches), ctx.array(src), first, n)
    ko, vo = ctx.empty((cap, w)), ctx.empty((cap, w))
    for c, kv in zip(caches, values):
        rf.kv_load(ctx, c, 0, cap, ko, vo)
        for got, x in zip((ko.numpy(), vo.numpy()), kv):
            want = x.copy()
            for j, r in enumerate(src):
                if r < cap:
                    want[first + j] = x[r]
            equal(got, want)
        c.free()


def norm_rope(x, w, eps, pos, theta):
    """x [n, heads, hd] f64."""
    hd = x.shape[-1]
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    angle = pos.astype(np.float64)[:, None, None] * theta ** (-np.arange(0, hd, 2) / hd)
    c, s = np.cos(angle), np.sin(angle)
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def close(y, ref, pos):
    """Errors relative to the length of each rotated pair."""
    h = ref.shape[-1] // 2
    pair = np.sqrt(ref[..., :h] ** 2 + ref[..., h:] ** 2)
    err = np.abs(y - ref) / np.maximum(np.concatenate([pair, pair], -1), 1e-30)
    tol = 2e-6 + 3 * 2.0 ** -52 * pos.astype(np.float64)
    assert (err.max((1, 2)) <= tol).all(), (err.max((1, 2)) / tol).max()


@pytest.mark.parametrize("n, qh, kvh, hd", [(1, 32, 8, 128), (37, 14, 2, 64), (3, 6, 3, 96), (1100, 8, 2, 128),
                                            (2, 4, 4, 256), (5, 3, 1, 10), (2, 2, 1, 512), (4, 5, 5, 2), (3, 2, 2, 32),
                                            (2, 1, 1, 508)])
@pytest.mark.parametrize("norms", ["both", "q", "none"])
def test_norm_and_rotation(ctx, n, qh, kvh, hd, norms):
    rng = np.random.default_rng(hd + n)
    eps, theta = 1e-6, 1e6
    q, k = (rng.normal(0, 2, (n, h, hd)).astype(np.float32) for h in (qh, kvh))
    wq, wk = (1 + 0.3 * rng.normal(0, 1, hd).astype(np.float32) for _ in range(2))
    wq = wq if norms != "none" else None
    wk = wk if norms == "both" else None
    # far and near positions, in no order
    pos = rng.integers(0, 1 << 20, n).astype(np.uint32)
    pos[0] = 0xFFFFFFFF if n > 1 else 131071
    qo, ko = ctx.empty((n, qh, hd)), ctx.empty((n, kvh, hd))
    dev = [None if a is None else ctx.array(a) for a in (q, k, wq, wk, pos)]
    rf.qk_norm_rope(ctx, dev[0], dev[1], dev[2], dev[3], eps, dev[4], n, qh, kvh, hd, theta, qo, ko)
    close(qo.numpy(), norm_rope(q.astype(np.float64), wq, eps, pos, theta), pos)
    close(ko.numpy(), norm_rope(k.astype(np.float64), wk, eps, pos, theta), pos)
    # in place
    rf.qk_norm_rope(ctx, dev[0], dev[1], dev[2], dev[3], eps, dev[4], n, qh, kvh, hd, theta, dev[0], dev[1])
    equal(dev[0].numpy(), qo.numpy())
    equal(dev[1].numpy(), ko.numpy())


@pytest.mark.parametrize("t", TYPES, ids=lambda t: GGML.NAMES[t])
@pytest.mark.parametrize("n, qh, kvh, hd, offset", [(1, 32, 8, 128, 0), (21, 14, 2, 64, 0), (6, 6, 3, 96, 0),
                                                    (1030, 4, 2, 128, 0), (5, 2, 1, 256, 1), (7, 3, 3, 32, 0)])
def test_norm_rotation_and_store(ctx, t, n, qh, kvh, hd, offset):
    """The cache holds what kv_store writes of the separately rotated rows, bit for bit; q is the same."""
    rng = np.random.default_rng(n + hd + t)
    row = (qh + 2 * kvh) * hd + offset
    qkv = rng.normal(0, 2, (n, row)).astype(np.float32)
    wq, wk = (ctx.array(1 + 0.3 * rng.normal(0, 1, hd).astype(np.float32)) for _ in range(2))
    d = ctx.array(qkv)
    q, k, v = d.ptr, d.ptr + 4 * qh * hd, d.ptr + 4 * (qh + kvh) * hd
    first, cap = 4, n + 6
    pos = ctx.array(np.arange(first, first + n, dtype=np.uint32))
    q1, k1, q2 = ctx.empty((n, qh * hd)), ctx.empty((n, kvh * hd)), ctx.empty((n, qh * hd))
    rf.qk_norm_rope(ctx, q, k, wq, wk, 1e-6, pos, n, qh, kvh, hd, 1e4, q1, k1, q_stride=row, k_stride=row)
    got = []
    for fused in (False, True):
        cache = rf.KvCache(ctx, t, cap, kvh, hd)
        fill = np.full(cache.k.nbytes, 0x5A, np.uint8)
        cache.k.upload(fill)
        cache.v.upload(fill)
        if fused:
            rf.qk_norm_rope_store(ctx, q, k, v, wq, wk, 1e-6, None, n, qh, 1e4, q2, cache, first, q_stride=row,
                                  k_stride=row, v_stride=row)
        else:
            rf.kv_store(ctx, cache, k1, v, first, n, v_stride=row)
        got.append((cache.k.numpy(), cache.v.numpy()))
        cache.free()
    equal(q1.numpy(), q2.numpy())
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])


def test_length_word(ctx):
    """A cache's length word moves every call's rows, inside a replayed graph too; rows past the capacity are left."""
    rng = np.random.default_rng(5)
    n, kvh, hd, cap = 3, 2, 64, 8
    w = kvh * hd
    length = ctx.array(np.array([0], np.uint32))
    cache = rf.KvCache(ctx, GGML.F32, cap, kvh, hd, length=length)
    k, v = rows(rng, n, w), rows(rng, n, w)
    kd, vd = ctx.array(k), ctx.array(v)
    plain = rf.KvCache(ctx, GGML.F32, cap, kvh, hd, cache.k, cache.v)
    zeros = np.zeros((cap, w), np.float32)
    with ctx.capture() as cap_:
        rf.kv_store(ctx, cache, kd, vd, 0, n)
    for at in (0, 4, 6, 5, 0xFFFFFFFF):
        cache.k.upload(zeros)
        cache.v.upload(zeros)
        length.upload(np.array([at], np.uint32))
        cap_.graph.replay()
        ctx.synchronize()
        ko, vo = ctx.empty((cap, w)), ctx.empty((cap, w))
        rf.kv_load(ctx, plain, 0, cap, ko, vo)
        want = zeros.copy()
        m = max(0, min(n, cap - at))
        want[at:at + m] = k[:m]
        equal(ko.numpy(), want)
        out = ctx.array(np.full((n, w), 3, np.float32))
        rf.kv_load(ctx, cache, 0, n, out, ctx.empty((n, w)))
        equal(out.numpy(), np.concatenate([k[:m], np.full((n - m, w), 3, np.float32)]))
    cap_.graph.close()
    cache.free()
