// rf_draft.hip — entry points of a step of drafted tokens: rf_kv_*,
// rf_qk_norm_rope*, rf_tree_mask, rf_attention_tree.
#include <cmath>

#include "rf_kv.h"
#include "rf_runtime.h"

using namespace rf;

namespace {

typedef unsigned long long ull;

bool mul_ok(uint64_t a, uint64_t b, uint64_t* out) { return !__builtin_mul_overflow(a, b, out); }

// Makes the context's device current for the call's launches.
struct OnDevice {
  int before = -1;
  bool ok = true;
  explicit OnDevice(const rf_ctx* ctx) {
    if (hipGetDevice(&before) != hipSuccess) before = -1;
    if (before != ctx->device) ok = hipSetDevice(ctx->device) == hipSuccess;
    else before = -1;
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

const char* cache_type_name(uint32_t t) {
  return t == RF_TYPE_F32 ? "F32" : t == RF_TYPE_F16 ? "F16" : t == RF_TYPE_Q8_0 ? "Q8_0" : t == RF_TYPE_Q4_0 ? "Q4_0" : nullptr;
}

// A cache's fields, and the K and V buffers it describes.
int32_t check_cache(const char* op, const rf_kv_cache* c, KvView* out) {
  if (!c) return set_error(RF_ERR_INVALID, "%s received a null cache", op);
  if (!cache_type_name(c->type))
    return set_error(RF_ERR_UNSUPPORTED, "%s does not support a cache of tensor type %s (%u)", op, type_name(c->type), c->type);
  if (c->kv_heads == 0 || c->head_dim == 0 || c->capacity == 0)
    return set_error(RF_ERR_INVALID, "%s requires a cache of non-zero positions, KV heads and head dimension", op);
  if (c->head_dim > KV_MAX_HEAD_DIM || c->kv_heads > 65535u || (uint64_t)c->kv_heads * c->head_dim > KV_MAX_WIDTH)
    return set_error(RF_ERR_UNSUPPORTED, "%s does not cover %u KV heads of %u", op, c->kv_heads, c->head_dim);
  if (c->type >= RF_TYPE_Q4_0 && c->head_dim % 32)
    return set_error(RF_ERR_INVALID, "%s cache head_dim %u not divisible by 32", cache_type_name(c->type), c->head_dim);
  if (c->capacity > 0xFFFFFFFFull) return set_error(RF_ERR_UNSUPPORTED, "%s over more than 2^32 - 1 positions", op);
  if (!c->k || !c->v) return set_error(RF_ERR_INVALID, "%s received a cache with a null buffer", op);
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15u)
    return set_error(RF_ERR_INVALID, "%s cache buffers must be 16-byte aligned", op);
  *out = KvView{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), c->length, c->capacity, c->type, c->kv_heads,
                c->head_dim};
  return RF_OK;
}

// Rows first .. first + n - 1 lie in the cache (with a length word the device checks each row).
int32_t check_rows(const char* op, const KvView& c, uint64_t first, uint64_t n) {
  if (first > c.cap || n > c.cap - first)
    return set_error(RF_ERR_INVALID, "%s of positions %llu + %llu exceeds the cache's %llu", op, (ull)first, (ull)n, (ull)c.cap);
  return RF_OK;
}

int32_t check_stride(const char* op, const char* what, uint64_t* stride, uint64_t width, uint64_t n) {
  if (*stride == 0) *stride = width;
  uint64_t all = 0;
  if (*stride < width) return set_error(RF_ERR_INVALID, "%s %s stride %llu is below the row's %llu", op, what, (ull)*stride, (ull)width);
  if (!mul_ok(n, *stride, &all) || !mul_ok(all, 4, &all))
    return set_error(RF_ERR_INVALID, "%s of %llu rows of %llu overflows 64 bits", op, (ull)n, (ull)*stride);
  return RF_OK;
}

int32_t launched(hipError_t e, const char* what) { return e == hipSuccess ? RF_OK : hip_error(e, what); }

}  // namespace

#define RF_TRY(call)       \
  do {                     \
    int32_t _rc = (call);  \
    if (_rc) return _rc;   \
  } while (0)
#define RF_ON_DEVICE(ctx) \
  OnDevice on(ctx);       \
  if (!on.ok) return hip_error(hipErrorInvalidDevice, "hipSetDevice")

extern "C" {

uint64_t rf_kv_cache_bytes(uint32_t type, uint64_t capacity, uint32_t kv_heads, uint32_t head_dim) {
  uint64_t all = 0;
  if (!cache_type_name(type) || (type >= RF_TYPE_Q4_0 && head_dim % 32) || kv_heads > 65535u ||
      head_dim > KV_MAX_HEAD_DIM || (uint64_t)kv_heads * head_dim > KV_MAX_WIDTH || capacity > 0xFFFFFFFFull)
    return 0;
  return mul_ok(capacity, kv_row_bytes(type, (uint64_t)kv_heads * head_dim), &all) ? all : 0;
}

int32_t rf_kv_store(rf_ctx* ctx, const rf_kv_cache* cache, const float* k, uint64_t k_stride, const float* v,
                    uint64_t v_stride, uint64_t first, uint64_t n, rf_stream_t s) {
  if (!ctx) return set_error(RF_ERR_INVALID, "null context");
  KvView c;
  RF_TRY(check_cache("KV store", cache, &c));
  RF_TRY(check_rows("KV store", c, first, n));
  const uint64_t width = (uint64_t)c.kvh * c.hd;
  RF_TRY(check_stride("KV store", "k", &k_stride, width, n));
  RF_TRY(check_stride("KV store", "v", &v_stride, width, n));
  if (n == 0) return RF_OK;
  if (!k || !v) return set_error(RF_ERR_INVALID, "KV store received a null pointer");
  RF_ON_DEVICE(ctx);
  return launched(launch_kv_store(c, k, k_stride, v, v_stride, first, n, pick_stream(ctx, s)), "KV store launch");
}

int32_t rf_kv_load(rf_ctx* ctx, const rf_kv_cache* cache, uint64_t first, uint64_t n, float* k, uint64_t k_stride,
                   float* v, uint64_t v_stride, rf_stream_t s) {
  if (!ctx) return set_error(RF_ERR_INVALID, "null context");
  KvView c;
  RF_TRY(check_cache("KV load", cache, &c));
  RF_TRY(check_rows("KV load", c, first, n));
  const uint64_t width = (uint64_t)c.kvh * c.hd;
  RF_TRY(check_stride("KV load", "k", &k_stride, width, n));
  RF_TRY(check_stride("KV load", "v", &v_stride, width, n));
  if (n == 0) return RF_OK;
  if (!k || !v) return set_error(RF_ERR_INVALID, "KV load received a null pointer");
  RF_ON_DEVICE(ctx);
  return launched(launch_kv_load(c, first, n, k, k_stride, v, v_stride, pick_stream(ctx, s)), "KV load launch");
}

int32_t rf_kv_move(rf_ctx* ctx, const rf_kv_cache* caches, uint32_t n_caches, const uint32_t* src, uint64_t first,
                   uint64_t n, rf_stream_t s) {
  if (!ctx) return set_error(RF_ERR_INVALID, "null context");
  if (n_caches == 0 || n == 0) return RF_OK;
  if (n > KV_MOVE_MAX)
    return set_error(RF_ERR_UNSUPPORTED, "KV move of %llu rows exceeds %u", (ull)n, KV_MOVE_MAX);
  if (!caches || !src) return set_error(RF_ERR_INVALID, "KV move received a null pointer");
  for (uint32_t i = 0; i < n_caches; ++i) {
    KvView c;
    RF_TRY(check_cache("KV move", &caches[i], &c));
    if (c.type != caches[0].type || c.kvh != caches[0].kv_heads || c.hd != caches[0].head_dim ||
        c.cap != caches[0].capacity || c.length != caches[0].length)
      return set_error(RF_ERR_INVALID, "KV move shape mismatch: cache %u differs from the first", i);
    RF_TRY(check_rows("KV move", c, first, n));
  }
  RF_ON_DEVICE(ctx);
  for (uint32_t at = 0; at < n_caches; at += KV_MOVE_CACHES) {
    const uint32_t m = n_caches - at < KV_MOVE_CACHES ? n_caches - at : KV_MOVE_CACHES;
    KvView views[KV_MOVE_CACHES];
    for (uint32_t i = 0; i < m; ++i) (void)check_cache("KV move", &caches[at + i], &views[i]);
    RF_TRY(launched(launch_kv_move(views, m, src, first, (uint32_t)n, pick_stream(ctx, s)), "KV move launch"));
  }
  return RF_OK;
}

// Arguments that both forms share; widths and strides in floats.
static int32_t rope_args(const char* op, QkRopeArgs* a, float theta) {
  if (a->hd == 0 || a->hd % 2 != 0) return set_error(RF_ERR_INVALID, "%s head dimension must be non-zero and even", op);
  if (a->qh == 0 || a->kvh == 0) return set_error(RF_ERR_INVALID, "%s requires non-zero query and KV head counts", op);
  if (a->hd > KV_MAX_HEAD_DIM || a->qh > 65535u || a->kvh > 65535u)
    return set_error(RF_ERR_UNSUPPORTED, "%s does not cover %u query and %u KV heads of %u", op, a->qh, a->kvh, a->hd);
  if (!std::isfinite(theta) || theta <= 0.f)
    return set_error(RF_ERR_INVALID, "%s frequency base must be finite and positive", op);
  if (!std::isfinite(a->eps) || a->eps < 0.f)
    return set_error(RF_ERR_INVALID, "%s epsilon must be finite and non-negative", op);
  a->log2_theta = std::log2((double)theta);
  const uint64_t qw = (uint64_t)a->qh * a->hd, kw = (uint64_t)a->kvh * a->hd;
  RF_TRY(check_stride(op, "q", &a->q_stride, qw, a->n));
  RF_TRY(check_stride(op, "k", &a->k_stride, kw, a->n));
  RF_TRY(check_stride(op, "q_out", &a->q_out_stride, qw, a->n));
  return RF_OK;
}

int32_t rf_qk_norm_rope(rf_ctx* ctx, const float* q, uint64_t q_stride, const float* k, uint64_t k_stride,
                        const float* q_norm, const float* k_norm, float eps, const uint32_t* positions,
                        uint64_t n_tokens, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, float theta,
                        float* q_out, uint64_t q_out_stride, float* k_out, uint64_t k_out_stride, rf_stream_t s) {
  if (!ctx) return set_error(RF_ERR_INVALID, "null context");
  QkRopeArgs a{};
  a.q = q; a.q_stride = q_stride; a.k = k; a.k_stride = k_stride; a.q_norm = q_norm; a.k_norm = k_norm; a.eps = eps;
  a.positions = positions; a.n = n_tokens; a.qh = q_heads; a.kvh = kv_heads; a.hd = head_dim;
  a.q_out = q_out; a.q_out_stride = q_out_stride; a.k_out = k_out; a.k_out_stride = k_out_stride;
  RF_TRY(rope_args("QK norm and RoPE", &a, theta));
  RF_TRY(check_stride("QK norm and RoPE", "k_out", &a.k_out_stride, (uint64_t)kv_heads * head_dim, n_tokens));
  if (n_tokens == 0) return RF_OK;
  if (!q || !k || !q_out || !k_out || !positions)
    return set_error(RF_ERR_INVALID, "QK norm and RoPE received a null pointer");
  RF_ON_DEVICE(ctx);
  return launched(launch_qk_norm_rope(a, pick_stream(ctx, s)), "QK norm and RoPE launch");
}

int32_t rf_qk_norm_rope_store(rf_ctx* ctx, const float* q, uint64_t q_stride, const float* k, uint64_t k_stride,
                              const float* v, uint64_t v_stride, const float* q_norm, const float* k_norm, float eps,
                              const uint32_t* positions, uint64_t n_tokens, uint32_t q_heads, float theta,
                              float* q_out, uint64_t q_out_stride, const rf_kv_cache* cache, uint64_t first,
                              rf_stream_t s) {
  if (!ctx) return set_error(RF_ERR_INVALID, "null context");
  QkRopeArgs a{};
  RF_TRY(check_cache("QK norm and RoPE store", cache, &a.cache));
  a.q = q; a.q_stride = q_stride; a.k = k; a.k_stride = k_stride; a.v = v; a.v_stride = v_stride;
  a.q_norm = q_norm; a.k_norm = k_norm; a.eps = eps; a.positions = positions; a.n = n_tokens;
  a.qh = q_heads; a.kvh = a.cache.kvh; a.hd = a.cache.hd;
  a.q_out = q_out; a.q_out_stride = q_out_stride; a.first = first;
  RF_TRY(rope_args("QK norm and RoPE store", &a, theta));
  RF_TRY(check_stride("QK norm and RoPE store", "v", &a.v_stride, (uint64_t)a.kvh * a.hd, n_tokens));
  RF_TRY(check_rows("QK norm and RoPE store", a.cache, first, n_tokens));
  if (n_tokens == 0) return RF_OK;
  if (!q || !k || !v || !q_out) return set_error(RF_ERR_INVALID, "QK norm and RoPE store received a null pointer");
  RF_ON_DEVICE(ctx);
  return launched(launch_qk_norm_rope(a, pick_stream(ctx, s)), "QK norm and RoPE store launch");
}

int32_t rf_tree_mask(rf_ctx* ctx, const int32_t* parents, uint64_t n, uint64_t base, const uint32_t* length,
                     uint64_t* mask, uint32_t* positions, rf_stream_t s) {
  if (!ctx) return set_error(RF_ERR_INVALID, "null context");
  if (n > TREE_MAX_NODES)
    return set_error(RF_ERR_UNSUPPORTED, "tree mask of %llu tokens exceeds %u", (ull)n, TREE_MAX_NODES);
  if (base > 0xFFFFFFFFull - n) return set_error(RF_ERR_UNSUPPORTED, "tree mask positions exceed 2^32 - 1");
  if (n == 0) return RF_OK;
  if (!parents || !mask) return set_error(RF_ERR_INVALID, "tree mask received a null pointer");
  RF_ON_DEVICE(ctx);
  return launched(launch_tree_mask(parents, (uint32_t)n, (uint32_t)base, length, mask, positions, pick_stream(ctx, s)),
                  "tree mask launch");
}

uint64_t rf_attention_tree_workspace_bytes(uint64_t max_positions, uint64_t n, uint32_t type, uint32_t qh, uint32_t kvh,
                                           uint32_t hd) {
  if (max_positions == 0 || n == 0 || qh == 0 || kvh == 0 || hd == 0 || n > TREE_MAX_NODES || qh % kvh ||
      !cache_type_name(type) || max_positions > 0xFFFFFFFFull || qh > 65535u || hd > KV_MAX_HEAD_DIM ||
      n * (qh / kvh) > TREE_MAX_ROWS)
    return 0;
  return tree_ws_floats_upto(max_positions, (uint32_t)n, qh, kvh, hd, type) * 4;
}

int32_t rf_attention_tree(rf_ctx* ctx, const float* q, uint64_t q_stride, const rf_kv_cache* cache, uint64_t hist_len,
                          const uint64_t* mask, uint64_t n, uint32_t q_heads, float* out, uint64_t out_stride,
                          rf_stream_t s) {
  if (!ctx) return set_error(RF_ERR_INVALID, "null context");
  TreeArgs a{};
  RF_TRY(check_cache("tree attention", cache, &a.cache));
  if (q_heads == 0) return set_error(RF_ERR_INVALID, "tree attention requires non-zero query heads");
  if (q_heads % a.cache.kvh != 0)
    return set_error(RF_ERR_INVALID, "GQA requires query_heads %u to be divisible by kv_heads %u", q_heads, a.cache.kvh);
  if (n > TREE_MAX_NODES || q_heads > 65535u)
    return set_error(RF_ERR_UNSUPPORTED, "tree attention does not cover %llu tokens of %u query heads (at most %u)",
                     (ull)n, q_heads, TREE_MAX_NODES);
  if (n * (q_heads / a.cache.kvh) > TREE_MAX_ROWS)
    return set_error(RF_ERR_UNSUPPORTED, "tree attention does not cover %llu tokens of %u query heads a KV head",
                     (ull)n, q_heads / a.cache.kvh);
  RF_TRY(check_rows("tree attention", a.cache, hist_len, n));
  const uint64_t width = (uint64_t)q_heads * a.cache.hd;
  RF_TRY(check_stride("tree attention", "q", &q_stride, width, n));
  RF_TRY(check_stride("tree attention", "out", &out_stride, width, n));
  if (n == 0) return RF_OK;
  if (!q || !out) return set_error(RF_ERR_INVALID, "tree attention received a null pointer");
  a.q = q; a.q_stride = q_stride; a.out = out; a.out_stride = out_stride; a.mask = mask;
  a.hist = hist_len; a.n = (uint32_t)n; a.qh = q_heads;
  a.q_vec = (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && q_stride % 4 == 0;
  // with a length word the context may grow to the whole cache under a captured call
  a.total = a.cache.length ? a.cache.cap : hist_len + n;
  a.nsplit = tree_splits(a.total, a.n, q_heads, a.cache.kvh, a.cache.hd, a.cache.type);
  hipStream_t st = pick_stream(ctx, s);
  RF_ON_DEVICE(ctx);
  const uint64_t ws = tree_ws_floats(a.nsplit, a.n, q_heads, a.cache.hd) * 4;
  if (ws) {
    RF_TRY(ensure_workspace(ctx, ctx->attn_ws, "workspace:attention", ws, st));
    a.ws = static_cast<float*>(ctx->attn_ws.ptr);
  }
  return launched(launch_attention_tree(a, st), "tree attention launch");
}

}  // extern "C"
