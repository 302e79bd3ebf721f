// rf_kv.hip — the K/V cache's writers and readers: norm and rotation of
// queries and keys (into the cache if wanted), quantised stores and loads, and
// the move of accepted rows.  The layout and its reasons: rf_kv.h.
//
// All of these are bound by HBM (or by launch latency for a token or two):
// each input is read and each output written once, 16 bytes per lane where
// addresses allow.
#include "rf_device.h"
#include "rf_kernels.h"
#include "rf_kv.h"

namespace rf {

// ------------------------------------------------------------ quantisation

// Max over the 8 lanes of a block (lanes 8 b .. 8 b + 7 hold its 32 values).
__device__ __forceinline__ float row8_max(float v) {
  v = fmaxf(v, rf_xchg16<1>(v));
  v = fmaxf(v, rf_xchg16<2>(v));
  return fmaxf(v, rf_xchg16<4>(v));
}

// The least float of BITS significant bits (none below 2^-24) that is >= t >= 0.
template <int BITS>
__device__ __forceinline__ float scale_up(float t) {
  constexpr uint32_t LOW = (1u << (24 - BITS)) - 1u;
  // 2^(BITS - 25) and above: BITS bits of significand are multiples of 2^-24
  return t >= (BITS == 3 ? 0x1p-22f : 0x1p-17f) ? __uint_as_float((__float_as_uint(t) + LOW) & ~LOW)
                                                : ceilf(t * 0x1p24f) * 0x1p-24f;
}

// The nearest whole number to x / d, ties to even: the remainder x - q d is
// exact (q d has at most 15 bits) and says on which side of the half step x
// lies.
__device__ __forceinline__ float nearest_code(float x, float d) {
  x = fminf(fmaxf(x, -8192.f * fabsf(d)), 8192.f * fabsf(d));  // past every clamp; keeps the remainder finite
  float q = rintf(x / d);
  const float r = fmaf(-q, d, x), h = 0.5f * fabsf(d), a = fabsf(r);
  if (a > h || (a == h && ((int)q & 1))) q += (r > 0.f) == (d > 0.f) ? 1.f : -1.f;
  return q;
}

// Scale and codes (with their offset) of one lane's four values of a block.
//
// A code is the nearest to x / d.  y = x * (1 / d) is off by less than
// |y| 2^-22 < 4e-5, so its nearest is that of the quotient unless y is that
// close to a half: then, or where the scale is cut at its largest, the
// wavefront takes the exact way (nearest_code).  Random values do so once in
// about 40 wavefronts; with the exact way alone the stores are bound by vector
// instructions (8191 x 1024 rows into Q4_0: 25.8 us, 3.0 TB/s).
template <bool Q8>
__device__ __forceinline__ uint32_t quantise4(const float (&x)[4], uint32_t* scale_bits) {
  constexpr float LEVELS = Q8 ? 127.f : 8.f, LARGEST = Q8 ? 512.f : 8160.f;
  constexpr int BITS = Q8 ? 3 : 8;
  float hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
  float lo = fmaxf(fmaxf(-x[0], -x[1]), fmaxf(-x[2], -x[3]));
  // an infinity or NaN: 0 * x is NaN
  float odd = fmaf(0.f, x[0], fmaf(0.f, x[1], fmaf(0.f, x[2], 0.f * x[3]))) == 0.f ? 0.f : 1.f;
  hi = row8_max(hi);
  lo = row8_max(lo);
  odd = row8_max(odd);
  const float top = odd == 0.f ? fmaxf(hi, lo) : 0.f;
  float d;
  if constexpr (Q8) {
    // from just below top / 127, so that the scale is at most one step low
    d = scale_up<BITS>(top * 0x1.0204p-7f);
    if (d * LEVELS < top) d = scale_up<BITS>(__uint_as_float(__float_as_uint(d) + 1u));
  } else {
    d = scale_up<BITS>(top * 0.125f);
    if (d * LEVELS < top) d = 0x1p-24f;  // top / 8 was no float
  }
  bool exact = d > LARGEST;
  d = fminf(d, LARGEST);
  if (!Q8 && hi > lo) d = -d;
  const float inv = d != 0.f ? __builtin_amdgcn_rcpf(d) : 0.f;
  // the sum's low bits are the nearest whole number (|y| <= 128)
  constexpr float MAGIC = 12582912.f;
  float r[4], far = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float y = x[i] * inv;
    r[i] = y + MAGIC;
    far = fmaxf(far, fabsf(y - (r[i] - MAGIC)));
  }
  exact |= far > 0.5f - 5e-5f;
  if (__any(exact)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float q = d != 0.f ? nearest_code(x[i], d) : 0.f;
      q = fminf(fmaxf(q, -LEVELS), LEVELS);
      r[i] = q + MAGIC;
    }
  }
  uint32_t w;
  if constexpr (Q8) {
    const uint32_t ab = __builtin_amdgcn_perm(__float_as_uint(r[1]), __float_as_uint(r[0]), 0x0C0C0400u);
    const uint32_t cd = __builtin_amdgcn_perm(__float_as_uint(r[3]), __float_as_uint(r[2]), 0x04000C0Cu);
    w = (ab | cd) ^ 0x80808080u;
    if (odd != 0.f) w = 0x80808080u;
  } else {
    uint32_t n[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = __float_as_uint(fminf(r[i], MAGIC + 7.f)) + 8u & 15u;
    w = n[0] | n[1] << 4 | n[2] << 8 | n[3] << 12;
    if (odd != 0.f) w = 0x8888u;
  }
  *scale_bits = odd != 0.f ? 0x7E00u : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)d);
  return w;
}

// Four values (of the 8 lanes of a block) at value index `at` of buffer b:
// codes at at, scale at at / 32 of the region behind cap_values codes.  Lanes
// of a block are all active or all inactive.
__device__ __forceinline__ void put4(uint8_t* b, uint32_t type, uint64_t cap_values, uint64_t at, const float (&x)[4],
                                     uint32_t lane, bool write) {
  if (type == T_Q8_0 || type == T_Q4_0) {
    uint32_t s;
    if (type == T_Q8_0) {
      const uint32_t w = quantise4<true>(x, &s);
      if (write) *reinterpret_cast<uint32_t*>(b + at) = w;
    } else {
      const uint32_t w = quantise4<false>(x, &s);
      if (write) *reinterpret_cast<uint16_t*>(b + at / 2) = (uint16_t)w;
    }
    if (write && (lane & 7u) == 0u)
      reinterpret_cast<uint16_t*>(b + (type == T_Q8_0 ? cap_values : cap_values / 2))[at / 32] = (uint16_t)s;
  } else if (write && type == T_F32) {
    *reinterpret_cast<float4*>(b + at * 4) = make_float4(x[0], x[1], x[2], x[3]);
  } else if (write) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<h4*>(b + at * 2) = h4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
  }
}

__device__ __forceinline__ void put1(uint8_t* b, uint32_t type, uint64_t at, float x) {
  if (type == T_F32) reinterpret_cast<float*>(b)[at] = x;
  else reinterpret_cast<_Float16*>(b)[at] = (_Float16)x;
}

__device__ __forceinline__ void get4(const uint8_t* b, uint32_t type, uint64_t cap_values, uint64_t at, float (&x)[4]) {
  if (type == T_F32) {
    const float4 f = *reinterpret_cast<const float4*>(b + at * 4);
    x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
  } else if (type == T_F16) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    const h4 h = *reinterpret_cast<const h4*>(b + at * 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)h[i];
  } else {
    const bool q8 = type == T_Q8_0;
    const uint16_t* sc = reinterpret_cast<const uint16_t*>(b + (q8 ? cap_values : cap_values / 2));
    const float d = (float)__builtin_bit_cast(_Float16, sc[at / 32]);
    const uint32_t w = q8 ? *reinterpret_cast<const uint32_t*>(b + at) : *reinterpret_cast<const uint16_t*>(b + at / 2);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = (q8 ? (float)((w >> 8 * i) & 255u) - 128.f : (float)((w >> 4 * i) & 15u) - 8.f) * d;
  }
}

// ------------------------------------------------------------- store, load

// Where a thread's four values of a row lie.  Threads map to (row, 4 values): a
// row takes tpr threads, a workgroup holds 256 / tpr rows, or 1024 values of
// one wide row.
struct RowMap {
  uint32_t width, rpw, row, col;
  bool ok;
};
__device__ __forceinline__ RowMap row_map(const KvView& c) {
  RowMap m;
  m.width = c.kvh * c.hd;
  const uint32_t tpr = (m.width + 3u) / 4u, tid = threadIdx.x;
  m.rpw = tpr < 256u ? 256u / tpr : 1u;
  m.row = tpr < 256u ? tid / tpr : 0u;
  m.col = 4u * (tpr < 256u ? tid % tpr : blockIdx.y * 256u + tid);
  m.ok = m.col < m.width && m.row < m.rpw;
  return m;
}

// Rows of 16-byte pieces.  Bound by HBM once the loads are many enough in
// flight: a thread asks for U rows before it uses the first, with addresses
// clamped instead of branches (a load in a branch is waited for there).  8191
// rows of 1024 values into Q4_0, 76 MB: 25.8 us with the exact rounding for
// every value, 21.4 us without it and one row a thread, 19.2 us as it is (4.0
// TB/s); back to floats 13.2 us.
template <bool LOAD, uint32_t T, int U>
__global__ __launch_bounds__(256) void kv_rows(KvView c, float* k, uint64_t k_stride, float* v, uint64_t v_stride,
                                               uint64_t first, uint64_t n) {
  const RowMap m = row_map(c);
  const uint32_t col = m.ok ? m.col : 0u, lane = threadIdx.x;
  float* const x = (blockIdx.z ? v : k) + col;
  const uint64_t stride = blockIdx.z ? v_stride : k_stride, cap_values = c.cap * m.width;
  uint8_t* const b = blockIdx.z ? c.v : c.k;
  const uint64_t base = first + (c.length ? *c.length : 0u);
  for (uint64_t i0 = (uint64_t)blockIdx.x * (m.rpw * U); i0 < n; i0 += (uint64_t)gridDim.x * (m.rpw * U)) {
    float f[U][4];
    bool ok[U];
    uint64_t i[U], at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t want = i0 + u * m.rpw + m.row;
      i[u] = min(want, n - 1u);
      ok[u] = m.ok && want < n && base + want < c.cap;
      at[u] = min(base + i[u], c.cap - 1u) * m.width + col;
      if constexpr (LOAD) {
        get4(b, T, cap_values, at[u], f[u]);
      } else {
        const float4 t = *reinterpret_cast<const float4*>(x + i[u] * stride);
        f[u][0] = t.x; f[u][1] = t.y; f[u][2] = t.z; f[u][3] = t.w;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (!LOAD) put4(b, T, cap_values, at[u], f[u], lane, ok[u]);
      else if (ok[u]) *reinterpret_cast<float4*>(x + i[u] * stride) = make_float4(f[u][0], f[u][1], f[u][2], f[u][3]);
    }
  }
}

// Any width, stride and alignment, by value.
template <bool LOAD>
__global__ __launch_bounds__(256) void kv_rows_any(KvView c, float* k, uint64_t k_stride, float* v, uint64_t v_stride,
                                                   uint64_t first, uint64_t n) {
  const RowMap m = row_map(c);
  float* const x = blockIdx.z ? v : k;
  const uint64_t stride = blockIdx.z ? v_stride : k_stride, cap_values = c.cap * m.width;
  uint8_t* const b = blockIdx.z ? c.v : c.k;
  const uint64_t base = first + (c.length ? *c.length : 0u);
  const bool quant = c.type == T_Q8_0 || c.type == T_Q4_0;  // width is then a multiple of 32
  for (uint64_t i0 = (uint64_t)blockIdx.x * m.rpw; i0 < n; i0 += (uint64_t)gridDim.x * m.rpw) {
    const uint64_t i = i0 + m.row, row = base + i;
    const bool ok = m.ok && i < n && row < c.cap;
    const uint64_t at = ok ? row * m.width + m.col : 0u;
    const uint32_t ne = ok ? min(4u, m.width - m.col) : 0u;
    float* const xp = x + (ok ? i * stride + m.col : 0u);
    float f[4] = {0.f, 0.f, 0.f, 0.f};
    if constexpr (LOAD) {
      if (quant) get4(b, c.type, cap_values, at, f);
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e)
        if (e < ne)
          xp[e] = quant ? f[e] : c.type == T_F32 ? reinterpret_cast<const float*>(b)[at + e]
                                                 : (float)reinterpret_cast<const _Float16*>(b)[at + e];
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e)
        if (e < ne) f[e] = xp[e];
      if (quant) {
        put4(b, c.type, cap_values, at, f, threadIdx.x, ok);
      } else {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
          if (e < ne) put1(b, c.type, at + e, f[e]);
      }
    }
  }
}

template <bool LOAD, uint32_t T>
static void launch_rows_vec(bool ahead, dim3 grid, const KvView& c, float* k, uint64_t ks, float* v, uint64_t vs,
                            uint64_t first, uint64_t n, hipStream_t st) {
  if (ahead) RF_KLAUNCH((kv_rows<LOAD, T, 4>), grid, dim3(256), 0, st, c, k, ks, v, vs, first, n);
  else RF_KLAUNCH((kv_rows<LOAD, T, 1>), grid, dim3(256), 0, st, c, k, ks, v, vs, first, n);
}

template <bool LOAD>
static hipError_t launch_rows(const KvView& c, float* k, uint64_t ks, float* v, uint64_t vs, uint64_t first,
                              uint64_t n, hipStream_t st) {
  const uint32_t width = c.kvh * c.hd, tpr = (width + 3u) / 4u, rpw = tpr < 256u ? 256u / tpr : 1u;
  const bool vec = width % 4u == 0u && ks % 4u == 0u && vs % 4u == 0u &&
                   ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0u;
  // four rows a thread where that leaves 8 workgroups a CU
  const uint32_t wide = (tpr + 255u) / 256u;
  const bool ahead = vec && n * 2 * wide >= (uint64_t)rpw * 4 * 2048;
  const uint64_t per = (uint64_t)rpw * (ahead ? 4 : 1), wgs = (n + per - 1) / per;
  const dim3 grid((uint32_t)(wgs < 65536 ? wgs : 65536), wide, 2);
  if (!vec) {
    RF_KLAUNCH((kv_rows_any<LOAD>), grid, dim3(256), 0, st, c, k, ks, v, vs, first, n);
    return hipGetLastError();
  }
  switch (c.type) {
    case T_F32: launch_rows_vec<LOAD, T_F32>(ahead, grid, c, k, ks, v, vs, first, n, st); break;
    case T_F16: launch_rows_vec<LOAD, T_F16>(ahead, grid, c, k, ks, v, vs, first, n, st); break;
    case T_Q8_0: launch_rows_vec<LOAD, T_Q8_0>(ahead, grid, c, k, ks, v, vs, first, n, st); break;
    default: launch_rows_vec<LOAD, T_Q4_0>(ahead, grid, c, k, ks, v, vs, first, n, st);
  }
  return hipGetLastError();
}

hipError_t launch_kv_store(const KvView& c, const float* k, uint64_t ks, const float* v, uint64_t vs, uint64_t first,
                           uint64_t n, hipStream_t st) {
  return launch_rows<false>(c, const_cast<float*>(k), ks, const_cast<float*>(v), vs, first, n, st);
}

hipError_t launch_kv_load(const KvView& c, uint64_t first, uint64_t n, float* k, uint64_t ks, float* v, uint64_t vs,
                          hipStream_t st) {
  return launch_rows<true>(c, k, ks, v, vs, first, n, st);
}

// -------------------------------------------------------------------- move

struct MoveArgs {
  uint8_t *k[KV_MOVE_CACHES], *v[KV_MOVE_CACHES];
  const uint32_t *src, *length;
  uint64_t cap, first, code_row, scale_row, scale_base;  // bytes
  uint32_t n, code_units, units, slice;                  // units of U bytes in a row: codes, all; log2 of a workgroup's
};

// A workgroup takes `slice` units of every row of one buffer: all its reads
// are in LDS before its first write, so a row may be source and target, in
// any order.  Bound by its launch and one round trip to HBM: 32 layers of 5 F16
// rows 4.0 us, 28 layers of 100 F32 rows (11.5 MB) 6.4 us.
template <typename U>
__global__ __launch_bounds__(256) void kv_move(MoveArgs a) {
  __shared__ U held[KV_MOVE_MAX];
  const uint32_t cache = blockIdx.y >> 1;
  uint8_t* const b = blockIdx.y & 1u ? a.v[cache] : a.k[cache];
  const uint32_t u0 = blockIdx.x << a.slice, mask = (1u << a.slice) - 1u, items = a.n << a.slice;  // <= KV_MOVE_MAX
  const uint64_t base = a.length ? *a.length : 0u, first = a.first + base;
  auto addr = [&](uint64_t row, uint32_t u) {
    return u < a.code_units ? b + row * a.code_row + (uint64_t)u * sizeof(U)
                            : b + a.scale_base + row * a.scale_row + (uint64_t)(u - a.code_units) * sizeof(U);
  };
  constexpr uint32_t PER = KV_MOVE_MAX / 256u;
  uint64_t row[PER];
  bool moves[PER];
  U x[PER];
#pragma unroll
  for (uint32_t i = 0; i < PER; ++i) {
    const uint32_t t = threadIdx.x + 256u * i;
    row[i] = t < items ? base + a.src[t >> a.slice] : ~0ull;
  }
#pragma unroll
  for (uint32_t i = 0; i < PER; ++i) {
    const uint32_t t = threadIdx.x + 256u * i, u = u0 + (t & mask);
    moves[i] = t < items && u < a.units && row[i] < a.cap && first + (t >> a.slice) < a.cap;
    if (moves[i]) x[i] = *reinterpret_cast<const U*>(addr(row[i], u));
  }
#pragma unroll
  for (uint32_t i = 0; i < PER; ++i)
    if (moves[i]) held[threadIdx.x + 256u * i] = x[i];
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < PER; ++i) {
    const uint32_t t = threadIdx.x + 256u * i;
    if (moves[i]) *reinterpret_cast<U*>(addr(first + (t >> a.slice), u0 + (t & mask))) = held[t];
  }
}

hipError_t launch_kv_move(const KvView* caches, uint32_t n_caches, const uint32_t* src, uint64_t first, uint32_t n,
                          hipStream_t st) {
  const KvView& c = caches[0];
  const uint64_t values = (uint64_t)c.kvh * c.hd;
  MoveArgs a{};
  a.src = src; a.length = c.length; a.cap = c.cap; a.first = first; a.n = n;
  a.code_row = kv_code_bytes(c.type, values);
  a.scale_row = kv_row_bytes(c.type, values) - a.code_row;
  a.scale_base = c.cap * a.code_row;
  const uint64_t bits = a.code_row | a.scale_row;
  const uint32_t unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 2;
  a.code_units = (uint32_t)(a.code_row / unit);
  a.units = (uint32_t)((a.code_row + a.scale_row) / unit);
  while ((n << (a.slice + 1)) <= KV_MOVE_MAX && (1u << a.slice) < a.units) ++a.slice;
  for (uint32_t at = 0; at < n_caches; at += KV_MOVE_CACHES) {
    const uint32_t m = n_caches - at < KV_MOVE_CACHES ? n_caches - at : KV_MOVE_CACHES;
    for (uint32_t i = 0; i < m; ++i) { a.k[i] = caches[at + i].k; a.v[i] = caches[at + i].v; }
    const dim3 grid((a.units + (1u << a.slice) - 1) >> a.slice, 2 * m);
    if (unit == 16) RF_KLAUNCH(kv_move<uint4>, grid, dim3(256), 0, st, a);
    else if (unit == 4) RF_KLAUNCH(kv_move<uint32_t>, grid, dim3(256), 0, st, a);
    else RF_KLAUNCH(kv_move<uint16_t>, grid, dim3(256), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// ------------------------------------------------- norms, rotation, storing

constexpr uint32_t ROPE_THREADS = 256;

// A group of gs lanes owns one head row; lane j of it the pairs (i, hd / 2 + i)
// of VEC consecutive i (VEC = 1: up to four such).  The cosines and sines of a
// token are made once per workgroup, in LDS, and serve all its heads; the first
// head's row is requested before them, the next one's before a head is worked
// on.  Angles are position * theta^(-2 i / hd) in 64 bits, reduced to a part of
// a turn before they are rounded to 32: at position 10^6 an f32 product would be
// off by 0.03 rad.
//
// Bound by HBM: 2048 tokens of 32 + 8 heads of 128 into an F16 cache, 92 MB, 18
// us, 5.1 TB/s.
template <int VEC>
__global__ __launch_bounds__(ROPE_THREADS) void qk_norm_rope(QkRopeArgs a, uint32_t gs, uint32_t heads_per_wg) {
  constexpr int PP = VEC == 4 ? 1 : 4;
  extern __shared__ float lds[];
  const uint32_t half = a.hd / 2u, tid = threadIdx.x;
  float2* const cs = reinterpret_cast<float2*>(lds);                 // [half]
  float* const stage = lds + a.hd + (size_t)(tid / gs) * a.hd;       // this group's row, for the cache
  const uint32_t lane = tid % gs, group = tid / gs, groups = ROPE_THREADS / gs;
  const bool to_cache = a.cache.k != nullptr;
  const uint32_t all = a.qh + a.kvh + (to_cache ? a.kvh : 0u);
  const uint32_t h0 = blockIdx.y * heads_per_wg, h1 = min(all, h0 + heads_per_wg);
  const uint64_t base = a.first + (a.cache.length ? *a.cache.length : 0u);
  const uint32_t width = a.kvh * a.hd;
  for (uint64_t t = blockIdx.x; t < a.n; t += gridDim.x) {
    float next_lo[PP][VEC], next_hi[PP][VEC];
    auto fetch = [&](uint32_t want) {  // heads and pairs past the last are the last's, so that no load is in a branch
      const uint32_t h = min(want, h1 - 1u);
      const float* const x = h < a.qh ? a.q + t * a.q_stride + (size_t)h * a.hd
                             : h < a.qh + a.kvh ? a.k + t * a.k_stride + (size_t)(h - a.qh) * a.hd
                                                : a.v + t * a.v_stride + (size_t)(h - a.qh - a.kvh) * a.hd;
#pragma unroll
      for (int p = 0; p < PP; ++p) {
        const uint32_t i = min((lane + gs * p) * VEC, half - VEC);
        if constexpr (VEC == 4) {
          const float4 l4 = *reinterpret_cast<const float4*>(x + i), h4 = *reinterpret_cast<const float4*>(x + half + i);
          next_lo[p][0] = l4.x; next_lo[p][1] = l4.y; next_lo[p][2] = l4.z; next_lo[p][3] = l4.w;
          next_hi[p][0] = h4.x; next_hi[p][1] = h4.y; next_hi[p][2] = h4.z; next_hi[p][3] = h4.w;
        } else {
          next_lo[p][0] = x[i];
          next_hi[p][0] = x[half + i];
        }
      }
    };
    fetch(h0 + group);
    const uint64_t pos = a.positions ? a.positions[t] : base + t;
    __syncthreads();  // the last token's readers of cs
    for (uint32_t i = tid; i < half; i += ROPE_THREADS) {
      const double turns = (double)pos * (exp2(a.log2_theta * (-2.0 * i / a.hd)) * 0.15915494309189533577);
      float s, c;
      sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
      cs[i] = make_float2(c, s);
    }
    __syncthreads();
    for (uint32_t h = h0 + group; h < h1; h += groups) {
      const uint32_t kind = h < a.qh ? 0u : h < a.qh + a.kvh ? 1u : 2u;
      const uint32_t hl = kind == 0u ? h : kind == 1u ? h - a.qh : h - a.qh - a.kvh;
      const float* const w = kind == 0u ? a.q_norm : kind == 1u ? a.k_norm : nullptr;
      float lo[PP][VEC], hi[PP][VEC];
      float sum = 0.f;
#pragma unroll
      for (int p = 0; p < PP; ++p) {
        const bool mine = (lane + gs * p) * VEC < half;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          lo[p][e] = mine ? next_lo[p][e] : 0.f;
          hi[p][e] = mine ? next_hi[p][e] : 0.f;
          sum = fmaf(lo[p][e], lo[p][e], fmaf(hi[p][e], hi[p][e], sum));
        }
      }
      fetch(h + groups);
      if (w) {
        for (uint32_t o = 1; o < gs; o <<= 1) sum += __shfl_xor(sum, o);
        const float r = 1.f / sqrtf(sum / (float)a.hd + a.eps);
#pragma unroll
        for (int p = 0; p < PP; ++p) {
          const uint32_t i = (lane + gs * p) * VEC;
          if (i < half) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              lo[p][e] = lo[p][e] * r * w[i + e];
              hi[p][e] = hi[p][e] * r * w[half + i + e];
            }
          }
        }
      }
      if (kind != 2u) {
#pragma unroll
        for (int p = 0; p < PP; ++p) {
          const uint32_t i = (lane + gs * p) * VEC;
          if (i < half) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const float2 r = cs[i + e];
              const float l = lo[p][e], u = hi[p][e];
              lo[p][e] = l * r.x - u * r.y;
              hi[p][e] = u * r.x + l * r.y;
            }
          }
        }
      }
      if (kind == 0u || !to_cache) {
        float* const y = kind == 0u ? a.q_out + t * a.q_out_stride + (size_t)hl * a.hd
                                    : a.k_out + t * a.k_out_stride + (size_t)hl * a.hd;
#pragma unroll
        for (int p = 0; p < PP; ++p) {
          const uint32_t i = (lane + gs * p) * VEC;
          if (i < half) {
            if constexpr (VEC == 4) {
              *reinterpret_cast<float4*>(y + i) = make_float4(lo[p][0], lo[p][1], lo[p][2], lo[p][3]);
              *reinterpret_cast<float4*>(y + half + i) = make_float4(hi[p][0], hi[p][1], hi[p][2], hi[p][3]);
            } else {
              y[i] = lo[p][0];
              y[half + i] = hi[p][0];
            }
          }
        }
        continue;
      }
      // into the cache: through LDS, so that a block's 32 values lie in 8 lanes
      const uint64_t row = base + t;
      uint8_t* const b = kind == 1u ? a.cache.k : a.cache.v;
      const uint64_t at0 = row * width + (uint64_t)hl * a.hd;
#pragma unroll
      for (int p = 0; p < PP; ++p) {
        const uint32_t i = (lane + gs * p) * VEC;
        if (i < half) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            stage[i + e] = lo[p][e];
            stage[half + i + e] = hi[p][e];
          }
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      const bool ok = row < a.cache.cap;
      if (a.hd % 4u == 0u) {
        for (uint32_t s = lane; s < a.hd / 4u; s += gs) {
          const float f[4] = {stage[4 * s], stage[4 * s + 1], stage[4 * s + 2], stage[4 * s + 3]};
          put4(b, a.cache.type, a.cache.cap * width, ok ? at0 + 4u * s : 0u, f, lane, ok);
        }
      } else if (ok) {
        for (uint32_t s = lane; s < a.hd; s += gs) put1(b, a.cache.type, at0 + s, stage[s]);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
}

hipError_t launch_qk_norm_rope(const QkRopeArgs& a, hipStream_t st) {
  const uint32_t half = a.hd / 2u;
  auto al = [](const void* p, uint64_t stride) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride % 4 == 0; };
  const bool vec = a.hd % 8u == 0u && al(a.q, a.q_stride) && al(a.k, a.k_stride) && al(a.q_out, a.q_out_stride) &&
                   (a.cache.k ? al(a.v, a.v_stride) : al(a.k_out, a.k_out_stride));
  const uint32_t per = vec ? half / 4u : half;
  uint32_t gs = 8;
  while (gs < 64u && gs < per) gs *= 2;
  const uint32_t groups = ROPE_THREADS / gs, all = a.qh + a.kvh * (a.cache.k ? 2u : 1u);
  // few tokens: the heads of one are spread over workgroups
  const uint32_t per_wg = a.n >= 1024 ? all : groups;
  const dim3 grid((uint32_t)(a.n < 65536 ? a.n : 65536), (all + per_wg - 1) / per_wg);
  const uint32_t lds = 4u * (a.hd + (a.cache.k ? groups * a.hd : 0u));
  if (vec) RF_KLAUNCH(qk_norm_rope<4>, grid, dim3(ROPE_THREADS), lds, st, a, gs, per_wg);
  else RF_KLAUNCH(qk_norm_rope<1>, grid, dim3(ROPE_THREADS), lds, st, a, gs, per_wg);
  return hipGetLastError();
}

hipError_t load_module_kv() {
  hipFuncAttributes fa;
  return hipFuncGetAttributes(&fa, reinterpret_cast<const void*>(&kv_move<uint4>));
}

}  // namespace rf
