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

// The least float of BITS significant bits (none below 2^-24) that is >= t > 0.
template <int BITS>
__device__ __forceinline__ float scale_up(float t) {
  constexpr uint32_t LOW = (1u << (24 - BITS)) - 1u;
  // 2^(BITS - 25) and above: BITS bits of significand are multiples of 2^-24
  if (t >= (BITS == 3 ? 0x1p-22f : 0x1p-17f)) return __uint_as_float((__float_as_uint(t) + LOW) & ~LOW);
  return ceilf(t * 0x1p24f) * 0x1p-24f;
}

// The nearest whole number to x / d, ties to even.  x * (1 / d) is off by an
// ulp or two; the remainder x - q d is exact (q d has at most 15 bits) and
// says on which side of the half step x lies.
__device__ __forceinline__ float nearest_code(float x, float d, float inv) {
  float q = rintf(x * inv);
  const float r = fmaf(-q, d, x), h = 0.5f * fabsf(d), a = fabsf(r);
  if (a > h || (a == h && ((int)q & 1))) q += (r > 0.f) == (d > 0.f) ? 1.f : -1.f;
  return q;
}

// Scale and codes (with their offset) of one lane's four values of a block.
template <bool Q8>
__device__ __forceinline__ uint32_t quantise4(const float (&x)[4], uint32_t* scale_bits) {
  float hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
  float lo = fmaxf(fmaxf(-x[0], -x[1]), fmaxf(-x[2], -x[3]));
  bool odd = false;  // an infinity or NaN
#pragma unroll
  for (int i = 0; i < 4; ++i) odd |= !(fabsf(x[i]) <= 3.402823466e38f);
  hi = row8_max(hi);
  lo = row8_max(lo);
  odd = row8_max(odd ? 1.f : 0.f) != 0.f;
  const float top = fmaxf(hi, lo);
  constexpr float LEVELS = Q8 ? 127.f : 8.f;
  float d = scale_up<Q8 ? 3 : 8>(top / LEVELS);
  // the division may have rounded down to a scale that does not reach the top
  if (d * LEVELS < top) d = scale_up<Q8 ? 3 : 8>(__uint_as_float(__float_as_uint(d) + 1u));
  d = fminf(d, Q8 ? 512.f : 8160.f);
  if (top == 0.f) d = 0.f;
  if (!Q8 && hi > lo) d = -d;
  const float inv = d != 0.f ? 1.f / d : 0.f;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // 8192 codes are past every clamp; it keeps far values' remainders finite
    const float xi = odd ? 0.f : fminf(fmaxf(x[i], -8192.f * fabsf(d)), 8192.f * fabsf(d));
    float q = d != 0.f ? nearest_code(xi, d, inv) : 0.f;
    q = Q8 ? fminf(fmaxf(q, -127.f), 127.f) + 128.f : fminf(fmaxf(q, -8.f), 7.f) + 8.f;
    w |= (uint32_t)q << (Q8 ? 8 * i : 4 * i);
  }
  *scale_bits = odd ? 0x7E00u : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)d);
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

// Threads map to (row, 4 values): a row takes tpr threads, a workgroup holds
// 256 / tpr rows (or 1024 values of one wide row).  VEC: all rows and widths
// allow 16-byte accesses; else (F32 / F16 only, or strided rows) by value.
template <bool LOAD, bool VEC>
__global__ __launch_bounds__(256) void kv_rows(KvView c, float* k, uint64_t k_stride, float* v, uint64_t v_stride,
                                               uint64_t first, uint64_t n) {
  const uint32_t width = c.kvh * c.hd, tpr = (width + 3u) / 4u, rpw = tpr < 256u ? 256u / tpr : 1u;
  const uint32_t tid = threadIdx.x, r = tpr < 256u ? tid / tpr : 0u;
  const uint32_t col = 4u * (tpr < 256u ? tid % tpr : blockIdx.y * 256u + tid);
  float* const x = blockIdx.z ? v : k;
  const uint64_t stride = blockIdx.z ? v_stride : k_stride, cap_values = c.cap * width;
  uint8_t* const b = blockIdx.z ? c.v : c.k;
  const uint64_t base = first + (c.length ? *c.length : 0u);
  const bool lane_ok = col < width && r < rpw;
  for (uint64_t i0 = (uint64_t)blockIdx.x * rpw; i0 < n; i0 += (uint64_t)gridDim.x * rpw) {
    const uint64_t i = i0 + r, row = base + i;
    const bool ok = lane_ok && i < n && row < c.cap;
    const uint64_t at = ok ? row * width + col : 0u;
    float* const xp = x + (ok ? i * stride + col : 0u);
    float f[4] = {0.f, 0.f, 0.f, 0.f};
    if constexpr (LOAD) {
      if (!ok) continue;
      if (c.type == T_Q8_0 || c.type == T_Q4_0 || width % 4u == 0u) {
        get4(b, c.type, cap_values, at, f);
      } else {
        for (uint32_t e = 0; e < min(4u, width - col); ++e)
          f[e] = c.type == T_F32 ? reinterpret_cast<const float*>(b)[at + e]
                                 : (float)reinterpret_cast<const _Float16*>(b)[at + e];
      }
      if constexpr (VEC) {
        *reinterpret_cast<float4*>(xp) = make_float4(f[0], f[1], f[2], f[3]);
      } else {
        for (uint32_t e = 0; e < min(4u, width - col); ++e) xp[e] = f[e];
      }
    } else {
      if (ok) {
        if constexpr (VEC) {
          const float4 t = *reinterpret_cast<const float4*>(xp);
          f[0] = t.x; f[1] = t.y; f[2] = t.z; f[3] = t.w;
        } else {
          for (uint32_t e = 0; e < min(4u, width - col); ++e) f[e] = xp[e];
        }
      }
      if (width % 4u == 0u) {
        put4(b, c.type, cap_values, at, f, tid, ok);
      } else if (ok) {
        for (uint32_t e = 0; e < min(4u, width - col); ++e) put1(b, c.type, at + e, f[e]);
      }
    }
  }
}

template <bool LOAD>
static hipError_t launch_rows(const KvView& c, float* k, uint64_t ks, float* v, uint64_t vs, uint64_t first,
                              uint64_t n, hipStream_t st) {
  const uint32_t width = c.kvh * c.hd, tpr = (width + 3u) / 4u, rpw = tpr < 256u ? 256u / tpr : 1u;
  const bool vec = width % 4u == 0u && ks % 4u == 0u && vs % 4u == 0u &&
                   ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0u;
  const uint64_t wgs = (n + rpw - 1) / rpw;
  const dim3 grid((uint32_t)(wgs < 65536 ? wgs : 65536), (tpr + 255u) / 256u, 2);
  if (vec) RF_KLAUNCH((kv_rows<LOAD, true>), grid, dim3(256), 0, st, c, k, ks, v, vs, first, n);
  else RF_KLAUNCH((kv_rows<LOAD, false>), grid, dim3(256), 0, st, c, k, ks, v, vs, first, n);
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
  uint32_t n, code_units, units, slice;                  // units of U bytes in a row: codes, all; per workgroup
};

// A workgroup takes `slice` units of every row of one buffer: all its reads
// are in LDS before its first write, so a row may be source and target, in
// any order.
template <typename U>
__global__ __launch_bounds__(256) void kv_move(MoveArgs a) {
  __shared__ U held[KV_MOVE_MAX];
  const uint32_t cache = blockIdx.y >> 1;
  uint8_t* const b = blockIdx.y & 1u ? a.v[cache] : a.k[cache];
  const uint32_t u0 = blockIdx.x * a.slice, un = min(a.slice, a.units - u0), items = a.n * un;
  const uint64_t base = a.length ? *a.length : 0u;
  const uint64_t first = a.first + base;
  auto addr = [&](uint64_t row, uint32_t u) {
    return u < a.code_units ? b + row * a.code_row + (uint64_t)u * sizeof(U)
                            : b + a.scale_base + row * a.scale_row + (uint64_t)(u - a.code_units) * sizeof(U);
  };
  for (uint32_t t = threadIdx.x; t < items; t += 256u) {
    const uint64_t row = base + a.src[t / un];
    if (row < a.cap) held[t] = *reinterpret_cast<const U*>(addr(row, u0 + t % un));
  }
  __syncthreads();
  for (uint32_t t = threadIdx.x; t < items; t += 256u) {
    const uint64_t row = first + t / un;
    if (base + a.src[t / un] < a.cap && row < a.cap) *reinterpret_cast<U*>(addr(row, u0 + t % un)) = held[t];
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
  a.slice = KV_MOVE_MAX / n < a.units ? KV_MOVE_MAX / n : a.units;
  for (uint32_t at = 0; at < n_caches; at += KV_MOVE_CACHES) {
    const uint32_t m = n_caches - at < KV_MOVE_CACHES ? n_caches - at : KV_MOVE_CACHES;
    for (uint32_t i = 0; i < m; ++i) { a.k[i] = caches[at + i].k; a.v[i] = caches[at + i].v; }
    const dim3 grid((a.units + a.slice - 1) / a.slice, 2 * m);
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

// A group of GS lanes owns one head row; lane j of it the pairs (i, hd / 2 + i)
// of VEC consecutive i (VEC = 1: up to four such).  The cosines and sines of a
// token are made once per workgroup, in LDS, and serve all its heads.  Angles
// are position * theta^(-2 i / hd) in 64 bits, reduced to a part of a turn
// before they are rounded to 32: at position 10^6 an f32 product would be off
// by 0.03 rad.
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
      const float* const x = (kind == 0u ? a.q + t * a.q_stride : kind == 1u ? a.k + t * a.k_stride
                                                                             : a.v + t * a.v_stride) + (size_t)hl * a.hd;
      const float* const w = kind == 0u ? a.q_norm : kind == 1u ? a.k_norm : nullptr;
      float lo[PP][VEC], hi[PP][VEC];
      float sum = 0.f;
#pragma unroll
      for (int p = 0; p < PP; ++p) {
        const uint32_t i = (lane + gs * p) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) lo[p][e] = hi[p][e] = 0.f;
        if (i < half) {
          if constexpr (VEC == 4) {
            const float4 l4 = *reinterpret_cast<const float4*>(x + i), h4 = *reinterpret_cast<const float4*>(x + half + i);
            lo[p][0] = l4.x; lo[p][1] = l4.y; lo[p][2] = l4.z; lo[p][3] = l4.w;
            hi[p][0] = h4.x; hi[p][1] = h4.y; hi[p][2] = h4.z; hi[p][3] = h4.w;
          } else {
            lo[p][0] = x[i];
            hi[p][0] = x[half + i];
          }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum = fmaf(lo[p][e], lo[p][e], fmaf(hi[p][e], hi[p][e], sum));
      }
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
