"""Refusals of the draft-step calls (rf_kv_*, rf_qk_norm_rope*, rf_tree_mask, rf_attention_tree): arguments are
checked before any device work, so these run without a GPU, on a context that is never dereferenced."""
import ctypes as C

import pytest

from ramforge_amd import _lib

CTX = 1 << 20  # not null; no refused call reads it
INVALID, UNSUPPORTED = 1, 4
P = 1 << 24    # an aligned device address that nothing reads


def cache(**kw):
    f = dict(type=8, kv_heads=2, head_dim=64, reserved=0, capacity=100, k=P, v=P, length=None)
    f.update(kw)
    s = _lib.KvCacheStruct(**f)
    cache.keep = s
    return C.addressof(s)


BAD_CACHES = [
    (dict(type=10), UNSUPPORTED, "does not support a cache of tensor type Q2_K"),
    (dict(type=77), UNSUPPORTED, "does not support"),
    (dict(kv_heads=0), INVALID, "non-zero"),
    (dict(head_dim=0), INVALID, "non-zero"),
    (dict(capacity=0), INVALID, "non-zero"),
    (dict(head_dim=544), UNSUPPORTED, "does not cover"),
    (dict(kv_heads=65536), UNSUPPORTED, "does not cover"),
    (dict(kv_heads=8193, head_dim=128), UNSUPPORTED, "does not cover"),
    (dict(head_dim=80), INVALID, "not divisible by 32"),
    (dict(type=2, head_dim=16), INVALID, "Q4_0 cache head_dim 16 not divisible by 32"),
    (dict(capacity=1 << 32), UNSUPPORTED, "2^32 - 1"),
    (dict(k=None), INVALID, "null buffer"),
    (dict(v=None), INVALID, "null buffer"),
    (dict(k=P + 8), INVALID, "16-byte aligned"),
]


def calls(ref):
    lib = _lib.load()
    return {
        "store": lambda: lib.rf_kv_store(CTX, ref, P, 0, P, 0, 0, 1, None),
        "load": lambda: lib.rf_kv_load(CTX, ref, 0, 1, P, 0, P, 0, None),
        "move": lambda: lib.rf_kv_move(CTX, ref, 1, P, 0, 1, None),
        "rope_store": lambda: lib.rf_qk_norm_rope_store(CTX, P, 0, P, 0, P, 0, None, None, 1e-6, None, 1, 4, 1e4, P, 0,
                                                        ref, 0, None),
        "attention": lambda: lib.rf_attention_tree(CTX, P, 0, ref, 0, None, 1, 4, P, 0, None),
    }


@pytest.mark.parametrize("fields, code, text", BAD_CACHES)
@pytest.mark.parametrize("call", ["store", "load", "move", "rope_store", "attention"])
def test_bad_caches(call, fields, code, text):
    assert calls(cache(**fields))[call]() == code
    assert text in _lib.last_error()


@pytest.mark.parametrize("call", ["store", "load", "rope_store", "attention"])
def test_null_cache(call):
    assert calls(None)[call]() == INVALID
    assert "null cache" in _lib.last_error()


def refused(rc, code, text):
    assert rc == code, _lib.last_error()
    assert text in _lib.last_error()


def test_store_and_load_arguments():
    lib, c = _lib.load(), cache()
    refused(lib.rf_kv_store(None, c, P, 0, P, 0, 0, 1, None), INVALID, "null context")
    refused(lib.rf_kv_store(CTX, c, None, 0, P, 0, 0, 1, None), INVALID, "null pointer")
    refused(lib.rf_kv_load(CTX, c, 0, 1, P, 0, None, 0, None), INVALID, "null pointer")
    refused(lib.rf_kv_store(CTX, c, P, 0, P, 0, 90, 11, None), INVALID, "exceeds the cache's 100")
    refused(lib.rf_kv_load(CTX, c, 101, 0, P, 0, P, 0, None), INVALID, "exceeds the cache's 100")
    refused(lib.rf_kv_store(CTX, c, P, 0, P, 0, 2 ** 64 - 1, 2, None), INVALID, "exceeds the cache's 100")
    refused(lib.rf_kv_store(CTX, c, P, 127, P, 0, 0, 1, None), INVALID, "k stride 127 is below the row's 128")
    refused(lib.rf_kv_load(CTX, c, 0, 1, P, 0, P, 1, None), INVALID, "v stride 1 is below the row's 128")
    refused(lib.rf_kv_store(CTX, c, P, 2 ** 62, P, 0, 0, 2, None), INVALID, "overflows 64 bits")
    assert lib.rf_kv_store(CTX, c, None, 0, None, 0, 100, 0, None) == 0
    assert lib.rf_kv_load(CTX, c, 0, 0, None, 0, None, 0, None) == 0


def test_move_arguments():
    lib = _lib.load()
    one = cache
    refused(lib.rf_kv_move(None, one(), 1, P, 0, 1, None), INVALID, "null context")
    refused(lib.rf_kv_move(CTX, None, 1, P, 0, 1, None), INVALID, "null pointer")
    refused(lib.rf_kv_move(CTX, one(), 1, None, 0, 1, None), INVALID, "null pointer")
    refused(lib.rf_kv_move(CTX, one(), 1, P, 99, 2, None), INVALID, "exceeds the cache's 100")
    refused(lib.rf_kv_move(CTX, one(capacity=5000), 1, P, 0, 1025, None), UNSUPPORTED, "exceeds 1024")
    fields = dict(type=8, kv_heads=2, head_dim=64, reserved=0, capacity=100, k=P, v=P, length=None)
    for other in (dict(type=1), dict(kv_heads=4), dict(head_dim=128), dict(capacity=99), dict(length=P)):
        two = (_lib.KvCacheStruct * 2)(_lib.KvCacheStruct(**fields), _lib.KvCacheStruct(**{**fields, **other}))
        refused(lib.rf_kv_move(CTX, C.addressof(two), 2, P, 0, 1, None), INVALID, "cache 1 differs from the first")
    assert lib.rf_kv_move(CTX, None, 0, None, 0, 1, None) == 0
    assert lib.rf_kv_move(CTX, one(), 1, None, 0, 0, None) == 0


def test_rope_arguments():
    lib = _lib.load()

    def rope(ctx=CTX, q=P, qs=0, k=P, ks=0, eps=1e-6, pos=P, n=1, qh=4, kvh=2, hd=64, theta=1e4, qo=P, qos=0, ko=P,
             kos=0):
        return lib.rf_qk_norm_rope(ctx, q, qs, k, ks, None, None, eps, pos, n, qh, kvh, hd, theta, qo, qos, ko, kos,
                                   None)

    refused(rope(ctx=None), INVALID, "null context")
    for kw in (dict(q=None), dict(k=None), dict(pos=None), dict(qo=None), dict(ko=None)):
        refused(rope(**kw), INVALID, "null pointer")
    for hd in (0, 7):
        refused(rope(hd=hd), INVALID, "non-zero and even")
    refused(rope(qh=0), INVALID, "non-zero query and KV head counts")
    refused(rope(kvh=0), INVALID, "non-zero query and KV head counts")
    refused(rope(hd=514), UNSUPPORTED, "does not cover")
    refused(rope(qh=65536), UNSUPPORTED, "does not cover")
    for theta in (0.0, -1.0, float("inf"), float("nan")):
        refused(rope(theta=theta), INVALID, "frequency base")
    for eps in (-1e-9, float("inf"), float("nan")):
        refused(rope(eps=eps), INVALID, "epsilon")
    refused(rope(qs=255), INVALID, "q stride 255 is below")
    refused(rope(ks=127), INVALID, "k stride 127 is below")
    refused(rope(qos=3), INVALID, "q_out stride 3 is below")
    refused(rope(kos=3), INVALID, "k_out stride 3 is below")
    refused(rope(n=2 ** 60), INVALID, "overflows 64 bits")
    assert rope(n=0, q=None, k=None, qo=None, ko=None, pos=None) == 0
    c = cache()
    args = (P, 0, P, 0, P, 0, None, None, 1e-6, None)
    refused(lib.rf_qk_norm_rope_store(CTX, *args, 5, 4, 1e4, P, 0, c, 96, None), INVALID, "exceeds the cache's 100")
    refused(lib.rf_qk_norm_rope_store(CTX, P, 0, P, 0, P, 5, None, None, 1e-6, None, 5, 4, 1e4, P, 0, c, 0, None),
            INVALID, "v stride 5 is below")
    refused(lib.rf_qk_norm_rope_store(CTX, P, 0, P, 0, None, 0, None, None, 1e-6, None, 5, 4, 1e4, P, 0, c, 0, None),
            INVALID, "null pointer")


def test_mask_and_attention_arguments():
    lib, c = _lib.load(), cache()
    refused(lib.rf_tree_mask(None, P, 1, 0, None, P, None, None), INVALID, "null context")
    refused(lib.rf_tree_mask(CTX, None, 1, 0, None, P, None, None), INVALID, "null pointer")
    refused(lib.rf_tree_mask(CTX, P, 1, 0, None, None, None, None), INVALID, "null pointer")
    refused(lib.rf_tree_mask(CTX, P, 1025, 0, None, P, None, None), UNSUPPORTED, "exceeds 1024")
    refused(lib.rf_tree_mask(CTX, P, 2, 2 ** 32 - 2, None, P, None, None), UNSUPPORTED, "2^32 - 1")
    assert lib.rf_tree_mask(CTX, None, 0, 0, None, None, None, None) == 0

    def attention(ctx=CTX, q=P, qs=0, ref=c, hist=0, n=1, qh=4, out=P, os=0):
        return lib.rf_attention_tree(ctx, q, qs, ref, hist, None, n, qh, out, os, None)

    refused(attention(ctx=None), INVALID, "null context")
    refused(attention(q=None), INVALID, "null pointer")
    refused(attention(out=None), INVALID, "null pointer")
    refused(attention(qh=0), INVALID, "non-zero query heads")
    refused(attention(qh=3), INVALID, "GQA requires query_heads 3 to be divisible by kv_heads 2")
    refused(attention(qh=65536), UNSUPPORTED, "does not cover")
    refused(attention(n=1025), UNSUPPORTED, "at most 1024")
    refused(attention(hist=100), INVALID, "exceeds the cache's 100")
    refused(attention(hist=2 ** 64 - 1), INVALID, "exceeds the cache's 100")
    refused(attention(qs=255), INVALID, "q stride 255 is below")
    refused(attention(os=255), INVALID, "out stride 255 is below")
    assert attention(n=0, q=None, out=None) == 0


def test_cache_bytes():
    lib = _lib.load()
    assert lib.rf_kv_cache_bytes(0, 10, 2, 7) == 10 * 14 * 4
    assert lib.rf_kv_cache_bytes(1, 10, 2, 7) == 10 * 14 * 2
    assert lib.rf_kv_cache_bytes(8, 10, 2, 64) == 10 * 128 * 34 // 32
    assert lib.rf_kv_cache_bytes(2, 10, 2, 64) == 10 * 128 * 18 // 32
    for bad in ((10, 10, 2, 64), (8, 10, 2, 63), (0, 1 << 32, 1, 1), (0, 1, 1, 513), (0, 1, 65536, 1), (0, 0, 1, 1)):
        assert lib.rf_kv_cache_bytes(*bad) == 0


def test_tree_workspace_bytes():
    lib = _lib.load()
    for bad in ((0, 1, 8, 32, 8, 128), (100, 0, 8, 32, 8, 128), (100, 1025, 8, 32, 8, 128), (100, 1, 8, 30, 8, 128),
                (100, 1, 10, 32, 8, 128), (1 << 32, 1, 8, 32, 8, 128), (100, 1, 8, 32, 0, 128)):
        assert lib.rf_attention_tree_workspace_bytes(*bad) == 0
    # never less for a longer context or more tokens: a reservation serves every shorter call
    for t in (0, 1, 2, 8):
        last = 0
        for total in (1, 64, 100, 1000, 5000, 8192, 20000, 131072, 1 << 20):
            now = lib.rf_attention_tree_workspace_bytes(total, 16, t, 32, 8, 128)
            assert now >= last
            last = now
        last = 0
        for n in (1, 2, 4, 5, 8, 16, 17, 33, 64, 65, 200, 256, 500, 1024):
            now = lib.rf_attention_tree_workspace_bytes(9000, n, t, 32, 8, 128)
            assert now >= last
            last = now


def test_widest_positions():
    lib = _lib.load()
    assert lib.rf_kv_cache_bytes(1, 10, 8192, 128) == 10 * 2 ** 20 * 2
    assert lib.rf_kv_cache_bytes(1, 10, 8193, 128) == 0
    one = cache(type=1, kv_heads=1, head_dim=64, capacity=5000)
    refused(lib.rf_attention_tree(CTX, P, 0, one, 0, None, 1024, 1024, P, 0, None), UNSUPPORTED,
            "does not cover 1024 tokens of 1024 query heads a KV head")
    assert lib.rf_attention_tree_workspace_bytes(5000, 1024, 1, 1024, 1, 64) == 0


def test_a_freed_cache_is_refused():
    import ramforge_amd as rf

    class Ctx:
        handle, lib = CTX, _lib.load()

    class Buffer(rf.DeviceArray):
        def free(self):
            self.ptr = 0

    k, v = (Buffer(Ctx, P, 1 << 20, (1 << 20,), "uint8", "") for _ in range(2))
    c = rf.KvCache(Ctx, 8, 100, 2, 64, k, v)
    c.owned = [k, v]
    c.free()
    with pytest.raises(rf.RamforgeError, match="null buffer"):
        rf.kv_store(Ctx, c, P, P, 0, 1)
    with pytest.raises(rf.RamforgeError, match="null buffer"):
        rf.kv_move(Ctx, [c], P, 0, 1)
