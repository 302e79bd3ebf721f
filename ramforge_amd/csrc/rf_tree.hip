// rf_tree.hip — attention of drafted tokens over a cache in few bits.
//
// n tokens whose K / V rows are positions hist .. hist + n - 1 of the cache
// attend the whole history and, of one another, what the mask allows (a tree:
// a token's ancestors and itself).  out = softmax(q K^T / sqrt(hd)) V per query
// head, query head h reading KV head h * kvh / qh.  Rows that see nothing are
// zeros.
#include "rf_device.h"
#include "rf_kernels.h"
#include "rf_kv.h"

namespace rf {

// Bit j of row i: j is i or an ancestor of i.  A thread makes one word by
// walking up from i; parents are earlier, so it stops below its word.
__global__ __launch_bounds__(256) void tree_mask(const int32_t* parents, uint32_t n, uint32_t base,
                                                 const uint32_t* length, uint64_t* mask, uint32_t* positions) {
  __shared__ int32_t par[TREE_MAX_NODES];
  for (uint32_t i = threadIdx.x; i < n; i += 256u) {
    const int32_t p = parents[i];
    par[i] = p >= 0 && p < (int32_t)i ? p : -1;
  }
  __syncthreads();
  const uint32_t words = (n + 63u) / 64u, t = blockIdx.x * 256u + threadIdx.x;
  if (t >= n * words) return;
  const uint32_t i = t / words, w = t % words;
  uint64_t bits = 0;
  for (int32_t j = (int32_t)i; j >= (int32_t)(64u * w); j = par[j])
    if ((uint32_t)j < 64u * w + 64u) bits |= 1ull << (j & 63);
  mask[t] = bits;
  if (positions && w == 0) {
    uint32_t depth = 0;
    for (int32_t j = par[i]; j >= 0; j = par[j]) ++depth;
    positions[i] = base + depth + (length ? *length : 0u);
  }
}

hipError_t launch_tree_mask(const int32_t* parents, uint32_t n, uint32_t base, const uint32_t* length, uint64_t* mask,
                            uint32_t* positions, hipStream_t st) {
  const uint32_t words = (n + 63u) / 64u;
  RF_KLAUNCH(tree_mask, dim3((n * words + 255u) / 256u), dim3(256), 0, st, parents, n, base, length, mask, positions);
  return hipGetLastError();
}

// ------------------------------------------------------------- any shape

// One value of a cache buffer.
__device__ __forceinline__ float kv_value(const uint8_t* b, const KvView& c, uint64_t row, uint32_t col) {
  const uint64_t width = (uint64_t)c.kvh * c.hd, at = row * width + col;
  if (c.type == T_F32) return reinterpret_cast<const float*>(b)[at];
  if (c.type == T_F16) return (float)reinterpret_cast<const _Float16*>(b)[at];
  const bool q8 = c.type == T_Q8_0;
  const uint64_t codes = q8 ? c.cap * width : c.cap * width / 2;
  const float d = (float)reinterpret_cast<const _Float16*>(b + codes)[at / 32];
  return (q8 ? (float)b[at] - 128.f : (float)((b[at / 2] >> 4 * (at & 1u)) & 15u) - 8.f) * d;
}

// History and end of the keys of a call, inside the cache whatever *length says.
__device__ __forceinline__ void tree_range(const TreeArgs& a, uint64_t& hist, uint64_t& total) {
  hist = min(a.hist + (a.cache.length ? *a.cache.length : 0u), a.cache.cap);
  total = min(hist + a.n, a.cache.cap);
}

__device__ __forceinline__ bool tree_sees(const TreeArgs& a, uint32_t words, uint32_t i, uint32_t j) {
  return a.mask ? (a.mask[(uint64_t)i * words + j / 64u] >> (j & 63u)) & 1u : j <= i;
}

// Head dimensions outside the matrix-core kernel: a workgroup per (token,
// query head), 256 positions at a time, a thread per position for the scores
// and per dim for V.  Positions the token does not see are skipped, not
// weighted with zero: what they hold cannot reach it.
__global__ __launch_bounds__(256) void tree_plain(TreeArgs a) {
  __shared__ float qs[KV_MAX_HEAD_DIM], p[256], red[4];
  __shared__ bool seen[256];
  const uint32_t i = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, hd = a.cache.hd;
  const uint32_t g = (uint32_t)((uint64_t)h * a.cache.kvh / a.qh), words = (a.n + 63u) / 64u;
  uint64_t hist, total;
  tree_range(a, hist, total);
  for (uint32_t d = tid; d < hd; d += 256u) qs[d] = a.q[(uint64_t)i * a.q_stride + (uint64_t)h * hd + d];
  float o[2] = {0.f, 0.f}, m = -INFINITY, l = 0.f;
  const float denom = sqrtf((float)hd);
  for (uint64_t p0 = 0; p0 < total; p0 += 256u) {
    const uint64_t pos = p0 + tid;
    const bool see = pos < total && (pos < hist || tree_sees(a, words, i, (uint32_t)(pos - hist)));
    __syncthreads();
    float s = -INFINITY;
    if (see) {
      float acc = 0.f;
      for (uint32_t d = 0; d < hd; ++d) acc = fmaf(qs[d], kv_value(a.cache.k, a.cache, pos, g * hd + d), acc);
      s = acc / denom;
    }
    const float wm = rf_wave_max(s);
    if ((tid & 63u) == 0u) red[tid >> 6] = wm;
    __syncthreads();
    const float mn = fmaxf(fmaxf(m, fmaxf(red[0], red[1])), fmaxf(red[2], red[3]));
    const float base = mn == -INFINITY ? 0.f : mn;  // nothing seen yet
    const float al = expf(m - base), e = see ? expf(s - base) : 0.f;
    m = mn;
    p[tid] = e;
    seen[tid] = see;
    const float ws = rf_wave_sum(e);
    __syncthreads();
    if ((tid & 63u) == 0u) red[tid >> 6] = ws;
    __syncthreads();
    l = l * al + ((red[0] + red[1]) + (red[2] + red[3]));
    const uint32_t np = (uint32_t)min((uint64_t)256u, total - p0);
    for (uint32_t r = 0, d = tid; d < hd; d += 256u, ++r) {
      float acc = o[r] * al;
      for (uint32_t j = 0; j < np; ++j)
        if (seen[j]) acc = fmaf(p[j], kv_value(a.cache.v, a.cache, p0 + j, g * hd + d), acc);
      o[r] = acc;
    }
  }
  for (uint32_t r = 0, d = tid; d < hd; d += 256u, ++r)
    a.out[(uint64_t)i * a.out_stride + (uint64_t)h * hd + d] = l == 0.f ? 0.f : o[r] / l;
}

uint32_t tree_splits(uint64_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) { return 1; }
uint64_t tree_ws_floats(uint32_t nsplit, uint32_t n, uint32_t qh, uint32_t hd) {
  return nsplit > 1 ? (uint64_t)nsplit * n * qh * (hd + 4) : 0;
}

hipError_t launch_attention_tree(const TreeArgs& a, hipStream_t st) {
  RF_KLAUNCH(tree_plain, dim3(a.n, a.qh), dim3(256), 0, st, a);
  return hipGetLastError();
}

hipError_t load_module_tree() {
  hipFuncAttributes fa;
  return hipFuncGetAttributes(&fa, reinterpret_cast<const void*>(&tree_plain));
}

}  // namespace rf
