// rf_tree.hip — attention of drafted tokens over a cache in few bits.
//
// n tokens whose K / V rows are positions hist .. hist + n - 1 of the cache
// attend the whole history and, of one another, what the mask allows (a tree:
// a token's ancestors and itself).  out = softmax(q K^T / sqrt(hd)) V per query
// head, query head h reading KV head h * kvh / qh.  Rows that see nothing are
// zeros.
#include <type_traits>

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

// The same for 32 positions at once: bit b is position d0 + b of the drafts
// (d0 < 0: those below 0 are the history), of which there are nd.
__device__ __forceinline__ uint32_t tree_window(const TreeArgs& a, uint32_t words, uint32_t i, int64_t d0, uint32_t nd) {
  const uint32_t shift = d0 < 0 ? (uint32_t)-d0 : 0u, first = d0 < 0 ? 0u : (uint32_t)d0;  // shift <= 31
  if (first >= nd) return shift ? (1u << shift) - 1u : 0u;
  uint64_t bits;
  if (a.mask) {
    const uint64_t* const m = a.mask + (uint64_t)i * words + first / 64u;
    bits = m[0] >> (first & 63u);
    if ((first & 63u) > 32u && first / 64u + 1u < words) bits |= m[1] << (64u - (first & 63u));
  } else {
    const uint32_t n = i >= first ? i - first + 1u : 0u;
    bits = n >= 32u ? 0xFFFFFFFFull : (1ull << n) - 1ull;
  }
  if (nd - first < 32u) bits &= (1ull << (nd - first)) - 1ull;
  return (uint32_t)(bits << shift | ((1ull << shift) - 1ull));
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
  double o[2] = {0., 0.}, l = 0.;
  float m = -INFINITY;
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
    l = l * al + (double)((red[0] + red[1]) + (red[2] + red[3]));
    const uint32_t np = (uint32_t)min((uint64_t)256u, total - p0);
    for (uint32_t r = 0, d = tid; d < hd; d += 256u, ++r) {
      float acc = 0.f;
      for (uint32_t j = 0; j < np; ++j)
        if (seen[j]) acc = fmaf(p[j], kv_value(a.cache.v, a.cache, p0 + j, g * hd + d), acc);
      o[r] = o[r] * al + acc;
    }
  }
  for (uint32_t r = 0, d = tid; d < hd; d += 256u, ++r)
    a.out[(uint64_t)i * a.out_stride + (uint64_t)h * hd + d] = l == 0. ? 0.f : (float)(o[r] / l);
}

// ---------------------------------------------------------- matrix cores

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// S^T = K Q^T and O^T = V^T P^T on 16x16 matrix instructions, 32 positions at
// a time.  A row is one (token, query head) of a KV head: row r of a head is
// token r / G, head r % G.  Lane l of a wavefront, with c = l % 16 and
// g = l / 16:
//   * K^: A operand of S^T, position c of a half tile, HD / 4 consecutive dims
//     from g HD / 4 (so a lane loads 16-byte pieces); Q: B operand, row c, the
//     same dims in the same order.
//   * S^T comes back as row c at positions 4 g + v of each half tile: all of a
//     lane's eight scores are of one row, so maximum, sum and rescaling are
//     per lane, and P is already the B operand of O^T, with position
//     16 t + 4 g + v in place 4 t + v.
//   * V: A operand of O^T, eight positions in that order for the dims that c
//     owns (HD / 16 consecutive ones, so a lane loads whole words of a row);
//     pairs of positions are interleaved by byte permutes.
// Nothing passes through LDS until a workgroup's wavefronts join, and each
// cached byte is decoded once per M row tiles.
//
// Precision: cached values are exact in f16.  q (scaled by a power of two per
// row to 2^10 .. 2^11) and P (up to 2^15) are taken as two f16 pieces, 22 bits
// together, products and sums in f32.  An f32 cache takes f32 matrix
// instructions, 1/16 of the f16 rate (1/8 for the two pieces).
//
// Bound by vector issue where positions are many (a matrix instruction keeps a
// SIMD's vector issue for about half its 16 cycles, and a tile of Q4_0 with two
// row tiles takes 344 vector instructions beside 64 of them): 1024 rows over
// 8256 Q8_0 positions 82 us, 0.84 PFLOP/s of matrix work; 64 over 131072 Q4_0
// 88 us.  By the start, the first tile's loads and the join where they are few:
// 64 rows over 8192 Q8_0 positions 17.1 us with tree_join.
template <int HD> struct TreeDims {
  static constexpr int STEPS = HD / 32;   // matrix instructions of a half tile's scores
  static constexpr int TILES = HD / 16;   // 16-dim tiles of the output
  // the dims of lane c: W0 from c W0 and, behind the 16 W0 first, W1 from c W1
  static constexpr int W0 = HD == 96 ? 4 : HD / 16, W1 = HD == 96 ? 2 : 0;
  static __device__ __forceinline__ uint32_t dim(int tile, uint32_t c) {
    return tile < W0 ? c * W0 + tile : 16u * W0 + c * W1 + (tile - W0);
  }
};

typedef __amdgpu_buffer_rsrc_t TreeRsrc;
__device__ __forceinline__ TreeRsrc tree_rsrc(const uint8_t* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, (int32_t)bytes, 0x00020000);
}

// N words at byte offset off (a multiple of 4); past the end they are zeros.
template <int N>
__device__ __forceinline__ void tree_words(uint32_t* w, TreeRsrc r, uint32_t off) {
  if constexpr (N >= 4) {
    const u32x4 v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
    w[0] = v[0]; w[1] = v[1]; w[2] = v[2]; w[3] = v[3];
    if constexpr (N > 4) tree_words<N - 4>(w + 4, r, off + 16u);
  } else if constexpr (N >= 2) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
    w[0] = v[0]; w[1] = v[1];
    if constexpr (N > 2) tree_words<N - 2>(w + 2, r, off + 8u);
  } else {
    w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
  }
}
__device__ __forceinline__ uint32_t tree_u16(TreeRsrc r, uint32_t off) {
  return (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
}
// BYTES (1, 2 or whole words) of a row.
template <int BYTES>
__device__ __forceinline__ void tree_bytes(uint32_t* w, TreeRsrc r, uint32_t off) {
  if constexpr (BYTES == 1) w[0] = (uint32_t)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, off, 0, 0);
  else if constexpr (BYTES == 2) w[0] = tree_u16(r, off);
  else tree_words<BYTES / 4>(w, r, off);
}

__device__ __forceinline__ uint32_t pk_mul(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, a) * __builtin_bit_cast(half2_t, b));
}
// What decoding takes: (x & mask) | magic is an f16 pair of `one` + codes with
// their offset, and minus that it is the codes.  The masks are scalars and the
// magics vector registers that the compiler does not know to be constants: as
// literals the two operations would not be one instruction (64 of the 408 of a
// tile of Q4_0 with two row tiles).
struct TreeMagic {
  uint32_t low = 0x000F000Fu, high = 0x00F000F0u, m64 = 0x64006400u, m54 = 0x54005400u;
  __device__ __forceinline__ TreeMagic() {
    asm("" : "+s"(low));
    asm("" : "+s"(high));
    asm("" : "+v"(m64));
    asm("" : "+v"(m54));
  }
};
__device__ __forceinline__ uint32_t pk_minus(uint32_t x, float off) {
  const half2_t o = {(_Float16)off, (_Float16)off};
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, x) - o);
}
// Nibble k (0..3) of both halves of x.
template <int K>
__device__ __forceinline__ uint32_t pk_q4(uint32_t x, const TreeMagic& mg) {
  if constexpr (K >= 2) x >>= 8;
  return K % 2 ? pk_minus((x & mg.high) | mg.m54, 72.f) : pk_minus((x & mg.low) | mg.m64, 1032.f);
}

// One tile of 32 positions as a lane holds it, and its decoding.
template <uint32_t T, int HD> struct TreeTile {
  using D = TreeDims<HD>;
  static constexpr int BITS = T == T_F16 ? 16 : T == T_Q8_0 ? 8 : 4;
  static constexpr bool QUANT = T != T_F16;
  static constexpr int KW = HD * BITS / 128;              // words of a lane's K dims
  static constexpr int B0 = D::W0 * BITS / 8, B1 = D::W1 * BITS / 8;  // bytes of a lane's V dims
  static constexpr int VW0 = B0 < 4 ? 1 : B0 / 4, VW1 = B1 == 0 ? 0 : B1 < 4 ? 1 : B1 / 4;
  static constexpr int VW = VW0 + VW1;
  static constexpr int KS = QUANT ? (HD == 96 ? 3 : HD <= 128 ? 1 : HD / 128) : 0;  // scales of a lane's K dims
  static constexpr int VS = QUANT ? (D::W1 ? 2 : 1) : 0;
  uint32_t k[2][KW], v[8][VW];
  uint32_t ks[2][KS ? KS : 1], vs[8][VS ? VS : 1];

  // kr, vr: the tile's rows of codes; ksr, vsr: of scales.  row, srow: bytes of a position.
  __device__ __forceinline__ void load_k(TreeRsrc kr, TreeRsrc ksr, uint32_t row, uint32_t srow, uint32_t head,
                                         uint32_t c, uint32_t g) {
    const uint32_t hb = head * (HD * BITS / 8), hs = head * (HD / 16);
#pragma unroll
    for (uint32_t t = 0; t < 2; ++t) tree_words<KW>(k[t], kr, (16u * t + c) * row + hb + g * (KW * 4u));
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (QUANT) {
#pragma unroll
      for (uint32_t t = 0; t < 2; ++t) {
        const uint32_t p = 16u * t + c;
#pragma unroll
        for (uint32_t i = 0; i < (uint32_t)KS; ++i) {
          const uint32_t b = HD == 96 ? (g * 24u + 8u * i) / 32u : HD == 64 ? g / 2u : g * (HD / 128) + i;
          ks[t][i] = tree_u16(ksr, p * srow + hs + 2u * b);
        }
      }
    }
  }
  __device__ __forceinline__ void load_v(TreeRsrc vr, TreeRsrc vsr, uint32_t row, uint32_t srow, uint32_t head,
                                         uint32_t c, uint32_t g) {
    const uint32_t hb = head * (HD * BITS / 8), hs = head * (HD / 16);
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      const uint32_t p = 16u * (j / 4u) + 4u * g + j % 4u;
      tree_bytes<B0>(v[j], vr, p * row + hb + c * B0);
      if constexpr (B1 > 0) tree_bytes<B1>(v[j] + VW0, vr, p * row + hb + 16u * B0 + c * B1);
      if constexpr (QUANT) {
        vs[j][0] = tree_u16(vsr, p * srow + hs + 2u * (c * D::W0 / 32u));
        if constexpr (VS == 2) vs[j][1] = tree_u16(vsr, p * srow + hs + 2u * 2u);
      }
    }
  }
  // Element i of a lane's Q for step s goes with dim 8 s + order(i) of its HD / 4.
  static __device__ __forceinline__ constexpr int order(int i) { return T == T_Q4_0 ? (i / 2) + 4 * (i % 2) : i; }

  // The eight halves of a step's K words.
  static __device__ __forceinline__ void decode_k(const uint32_t* k, uint32_t scale, const TreeMagic& mg, u32x4& w) {
    const uint32_t s2 = scale | scale << 16;
    if constexpr (T == T_Q8_0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        w[2 * i] = pk_mul(pk_minus(__builtin_amdgcn_perm(mg.m64, k[i], 0x05010500u), 1152.f), s2);
        w[2 * i + 1] = pk_mul(pk_minus(__builtin_amdgcn_perm(mg.m64, k[i], 0x05030502u), 1152.f), s2);
      }
    } else {
      w[0] = pk_mul(pk_q4<0>(k[0], mg), s2);
      w[1] = pk_mul(pk_q4<1>(k[0], mg), s2);
      w[2] = pk_mul(pk_q4<2>(k[0], mg), s2);
      w[3] = pk_mul(pk_q4<3>(k[0], mg), s2);
    }
  }
  __device__ __forceinline__ half8_t kfrag(int t, int s, const TreeMagic& mg) const {
    u32x4 w;
    if constexpr (T == T_F16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = k[t][4 * s + i];
    } else {
      decode_k(k[t] + s * (BITS / 4), ks[t][HD == 96 ? s : s / 4], mg, w);
    }
    return __builtin_bit_cast(half8_t, w);
  }
  // The halves of two positions a, b at dim TILE of the lane's
  template <int TILE>
  static __device__ __forceinline__ uint32_t pair(const uint32_t* va, const uint32_t* vb, const uint32_t* sa,
                                                  const uint32_t* sb, const TreeMagic& mg) {
    constexpr int seg = TILE < D::W0 ? 0 : 1, e = seg ? TILE - D::W0 : TILE, per = 32 / BITS;  // element e of the lane's dims
    constexpr int word = (seg ? VW0 : 0) + e / per, in = e % per;
    const uint32_t a = va[word], b = vb[word];
    if constexpr (T == T_F16) {
      return __builtin_amdgcn_perm(b, a, in ? 0x07060302u : 0x05040100u);
    } else {
      const uint32_t s2 = sa[seg] | sb[seg] << 16;
      if constexpr (T == T_Q8_0) {
        return pk_mul(pk_minus(__builtin_amdgcn_perm(b, a, 0x0C040C00u + 0x00010001u * in) | mg.m64, 1152.f), s2);
      } else {
        const uint32_t x = __builtin_amdgcn_perm(b, a, in < 4 ? 0x05040100u : 0x07060302u);
        return pk_mul(pk_q4<in % 4>(x, mg), s2);
      }
    }
  }
  // V^T's tile of 16 dims
  template <int TILE>
  __device__ __forceinline__ half8_t vfrag(const TreeMagic& mg) const {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pair<TILE>(v[2 * i], v[2 * i + 1], vs[2 * i], vs[2 * i + 1], mg);
    return __builtin_bit_cast(half8_t, w);
  }
  // One word of all tiles' operands, from two positions
  template <int TILE = 0>
  static __device__ __forceinline__ void decode_v(const uint32_t* va, const uint32_t* vb, const uint32_t* sa,
                                                  const uint32_t* sb, const TreeMagic& mg, uint32_t (&w)[D::TILES]) {
    if constexpr (TILE < D::TILES) {
      w[TILE] = pair<TILE>(va, vb, sa, sb, mg);
      decode_v<TILE + 1>(va, vb, sa, sb, mg, w);
    }
  }
};

// The f32 cache's tile.
template <int HD> struct TreeTile<T_F32, HD> {
  using D = TreeDims<HD>;
  static constexpr bool QUANT = false;
  uint32_t k[2][HD / 4], v[8][HD / 16];
  __device__ __forceinline__ void load_k(TreeRsrc kr, TreeRsrc, uint32_t row, uint32_t, uint32_t head, uint32_t c,
                                         uint32_t g) {
#pragma unroll
    for (uint32_t t = 0; t < 2; ++t) tree_words<HD / 4>(k[t], kr, (16u * t + c) * row + head * (HD * 4u) + g * HD);
  }
  __device__ __forceinline__ void load_v(TreeRsrc vr, TreeRsrc, uint32_t row, uint32_t, uint32_t head, uint32_t c,
                                         uint32_t g) {
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      const uint32_t off = (16u * (j / 4u) + 4u * g + j % 4u) * row + head * (HD * 4u);
      tree_words<D::W0>(v[j], vr, off + c * (D::W0 * 4u));
      if constexpr (D::W1 > 0) tree_words<D::W1>(v[j] + D::W0, vr, off + 16u * D::W0 * 4u + c * (D::W1 * 4u));
    }
  }
  static __device__ __forceinline__ constexpr int order(int i) { return i; }
};

constexpr float TREE_FLOOR = -3e38f;  // reference of a row that has seen nothing
// A row's reference is set 2^12 below its largest score and moves once a weight
// would pass 2^15: weights stay inside f16, and as far as can be above its
// subnormals, which a weight 2^-26 of the largest meets.
constexpr float TREE_BELOW = 12.f, TREE_MOST = 15.f;
constexpr uint32_t TREE_WAVES = 4, TREE_KEYS = 32;

__device__ __forceinline__ void tree_lds_order() {  // within a wavefront
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Two f16 pieces of x and y: the nearest halves, and the nearest of what they
// leave.  minus: -1 that the compiler cannot see through, so that the rest is
// one mixed-precision fma each and no conversion back.
__device__ __forceinline__ float tree_minus() {
  float m = -1.f;
  asm volatile("" : "+v"(m));
  return m;
}
__device__ __forceinline__ void tree_pieces(float x, float y, float minus, uint32_t& hi, uint32_t& lo) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const half2_t h = __builtin_convertvector((f32x2{x, y}), half2_t);
  hi = __builtin_bit_cast(uint32_t, h);
  lo = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{fmaf((float)h[0], minus, x), fmaf((float)h[1], minus, y)}), half2_t));
}

// Shared memory of a workgroup: Q's operands (all its wavefronts have the same
// rows) and where odd values are added, and, once the positions are done, the
// rows of sums in their place.
constexpr uint32_t TREE_ODD = 36;
// Wavefronts of a workgroup of tree_mfma: eight (two a SIMD, one decoding under
// the other's matrix instructions) where two row tiles keep a CU to itself, four
// where workgroups are many and small (1024 rows over 8256 positions 93 us with
// four, 83 with eight; one token over 2048 9.8 and 10.2).
constexpr int tree_wide(uint32_t type, int hd, int m) { return m == 2 && !(type == T_F32 && hd == 128) ? 8 : 4; }
template <uint32_t T, int HD, int M> struct TreeShared {
  static constexpr int W = tree_wide(T, HD, M);
  static constexpr uint32_t OP = HD + 4;  // floats of a row of sums
  union {
    struct {
      u32x4 q[M][HD / 16][64];
      float odd[W][16 * TREE_ODD];
    };
    float sum[W][M * 16 * OP];
  };
  float scale[M][16];
  float m[W][M * 16], l[W][M * 16];
};

// A lane's HD / 4 values of a row of q.
template <int HD>
__device__ __forceinline__ void tree_get_q(float (&x)[HD / 4], const float* qp, bool vec) {
  if (vec) {
#pragma unroll
    for (int e = 0; e < HD / 16; ++e) {
      const float4 v = reinterpret_cast<const float4*>(qp)[e];
      x[4 * e] = v.x; x[4 * e + 1] = v.y; x[4 * e + 2] = v.z; x[4 * e + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < HD / 4; ++e) x[e] = qp[e];
  }
}

// Their two pieces of every step, put(step, piece, eight halves), piece 1 the
// first and 0 the rest, scaled to 2^10 .. 2^11 by a power of two; the scale
// that takes the scores to powers of two is returned.
template <uint32_t T, int HD, typename Put>
__device__ __forceinline__ float tree_split_q(const float (&x)[HD / 4], Put put) {
  const float minus = tree_minus();
  float scale = 1.44269504088896340736f / sqrtf((float)HD), top = 0.f, up = 1.f;
#pragma unroll
  for (int i = 0; i < HD / 4; ++i) top = fmaxf(top, fabsf(x[i]));
  top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  if (top > 0x1p-100f && top <= 3.402823466e38f) {
    const uint32_t e = __float_as_uint(top) >> 23;  // biased
    up = __uint_as_float((264u - e) << 23);         // 2^(10 - (e - 127))
    scale *= __uint_as_float((e - 10u) << 23);
  }
#pragma unroll
  for (int s = 0; s < HD / 32; ++s) {
    u32x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      using Tile = TreeTile<T, HD>;
      uint32_t h, r;
      tree_pieces(x[8 * s + Tile::order(2 * i)] * up, x[8 * s + Tile::order(2 * i + 1)] * up, minus, h, r);
      hi[i] = h;
      lo[i] = r;
    }
    put(s, 0, lo);
    put(s, 1, hi);
  }
  return scale;
}

// Q's operands of row tile m, by one wavefront.  f16 caches: word 2 s + piece of lane l is its eight halves of step s.
// An f32 cache: word i is four floats.
template <uint32_t T, int HD, int M>
__device__ __forceinline__ void tree_put_q(TreeShared<T, HD, M>& sh, int m, float (&x)[HD / 4], uint32_t lane) {
  float scale = 1.44269504088896340736f / sqrtf((float)HD);  // of the scores, to powers of two
  if constexpr (T == T_F32) {
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = __float_as_uint(x[4 * i + e]);
      sh.q[m][i][lane] = w;
    }
  } else {
    scale = tree_split_q<T, HD>(x, [&](int s, int piece, u32x4 w) { sh.q[m][2 * s + piece][lane] = w; });
  }
  if (lane < 16u) sh.scale[m][lane] = scale;
}

// Non-finite values of the tile's drafted V rows must not meet the zero
// weights of rows that do not see them: they are taken out of the operand and
// added, by value, to the rows that do.  Rare, so plain and slow; the sums go
// through 16 x TREE_ODD floats of LDS, 32 dims at a time, so that no register
// array is indexed.
template <int HD, int M>
__device__ __forceinline__ void tree_odd_rows(const TreeArgs& a, const float (&p)[M][8], const uint32_t (&see)[M],
                                              uint64_t p0, uint64_t total, uint32_t head, uint32_t c, uint32_t g,
                                              float* lds, f32x4 (&o)[M][TreeDims<HD>::TILES]) {
  using D = TreeDims<HD>;
  const uint32_t np = (uint32_t)min((uint64_t)TREE_KEYS, total - p0);
  float* const mine = lds + c * TREE_ODD;
#pragma unroll
  for (int m = 0; m < M; ++m) {
#pragma unroll 1
    for (uint32_t part = 0; part < (uint32_t)HD / 32u; ++part) {
#pragma unroll 1
      for (uint32_t d = g; d < 32u; d += 4u) mine[d] = 0.f;
#pragma unroll 1
      for (uint32_t k = 0; k < np; ++k) {
        const uint32_t j = 4u * (k / 16u) + k % 4u;
        const int from = (int)((k % 16u / 4u) * 16u + c);  // the lane that holds row c's weight of position k
        float w = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) w = i == j ? p[m][i] : w;
        w = __shfl(w, from);
        const bool sees = (uint32_t)__shfl((int)see[m], from) >> j & 1u;
#pragma unroll 1
        for (uint32_t d = g; d < 32u; d += 4u) {
          const float x = kv_value(a.cache.v, a.cache, p0 + k, head * HD + part * 32u + d);
          if (sees && !(fabsf(x) <= 3.402823466e38f)) mine[d] += w * x;
        }
      }
      tree_lds_order();
#pragma unroll
      for (int d = 0; d < D::TILES; ++d)
#pragma unroll
        for (uint32_t v = 0; v < 4; ++v) {
          const uint32_t dim = D::dim(d, 4u * g + v);
          if (dim / 32u == part) o[m][d][v] += mine[dim % 32u];
        }
      tree_lds_order();
    }
  }
}

// What a row tile's scores do to its state: masked ones out, the reference,
// weights, their sum.  s comes in as raw sums of products.
template <int HD, bool DRAFTS>
__device__ __forceinline__ void tree_soften(f32x4 (&s)[2], uint32_t see, float scale, float& ref, float& l,
                                            f32x4 (&o)[TreeDims<HD>::TILES], float (&p)[8]) {
  if constexpr (DRAFTS) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j / 4][j % 4] = see >> j & 1u ? s[j / 4][j % 4] : -INFINITY;
  }
  // exponents against the reference, and the largest of them
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    p[j] = fmaf(s[j / 4][j % 4], scale, -ref);
    top = fmaxf(top, p[j]);
  }
  // The reference stays until a weight would pass 2^15: few tiles rescale.
  if (__any(top > TREE_MOST)) {
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    // against the old reference; a row that has seen nothing starts from its scores
    const bool first = ref == TREE_FLOOR;
    float best = -INFINITY;
    if (first) {
#pragma unroll
      for (int j = 0; j < 8; ++j) best = fmaxf(best, s[j / 4][j % 4]);
    }
    best = fmaxf(best, __shfl_xor(best, 16));
    best = fmaxf(best, __shfl_xor(best, 32));
    const float now = first ? fmaxf(ref, fmaf(best, scale, -TREE_BELOW)) : ref + fmaxf(0.f, top - TREE_BELOW);
    const float al = first ? 0.f : __builtin_amdgcn_exp2f(ref - now);
    ref = now;
    l *= al;
#pragma unroll
    for (int d = 0; d < TreeDims<HD>::TILES; ++d)
#pragma unroll
      for (int v = 0; v < 4; ++v) o[d][v] *= al;
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = fmaf(s[j / 4][j % 4], scale, -ref);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(p[j]);
  l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
}

// The places of a lane (4 t + v: position p0 + 16 t + 4 g + v) that token i sees.
__device__ __forceinline__ uint32_t tree_places(const TreeArgs& a, uint32_t words, uint32_t i, uint64_t p0,
                                                uint64_t hist, uint64_t total, uint32_t g) {
  const uint32_t w = tree_window(a, words, i, (int64_t)(p0 - hist), (uint32_t)(total - hist)) >> 4u * g;
  return (w & 15u) | (w >> 12 & 0xF0u);
}

// A tile of V^T without its non-finite values.
__device__ __forceinline__ half8_t tree_finite(half8_t v, bool& odd) {
  u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t keep =
        ((w[k] & 0x7C00u) == 0x7C00u ? 0u : 0xFFFFu) | ((w[k] & 0x7C000000u) == 0x7C000000u ? 0u : 0xFFFF0000u);
    odd |= keep != 0xFFFFFFFFu;
    w[k] &= keep;
  }
  return __builtin_bit_cast(half8_t, w);
}

// O^T += V^T P^T for the f16 forms, N dim tiles at a time: the first of the
// pieces for all of them, then the other, so that no instruction waits for the
// sum before it.  DRAFTS: non-finite values are taken out (see above).
template <uint32_t T, int HD, int M, bool DRAFTS, int TILE>
__device__ __forceinline__ void tree_tiles(const TreeTile<T, HD>& x, const u32x4 (&ph)[M], const u32x4 (&pl)[M],
                                           const TreeMagic& mg, bool& odd, f32x4 (&o)[M][TreeDims<HD>::TILES]) {
  constexpr int N = M == 1 ? 4 : 2;
  static_assert(TreeDims<HD>::TILES % 2 == 0, "whole groups");
  if constexpr (TILE < TreeDims<HD>::TILES) {
    half8_t vf[N];
    auto decode = [&](auto i) {
      constexpr int I = decltype(i)::value;
      if constexpr (I < N && TILE + I < TreeDims<HD>::TILES) {
        vf[I] = x.template vfrag<TILE + I>(mg);
        if constexpr (DRAFTS) vf[I] = tree_finite(vf[I], odd);
      }
    };
    decode(std::integral_constant<int, 0>());
    decode(std::integral_constant<int, 1>());
    decode(std::integral_constant<int, 2>());
    decode(std::integral_constant<int, 3>());
#pragma unroll
    for (int piece = 0; piece < 2; ++piece)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (TILE + i < TreeDims<HD>::TILES) {
#pragma unroll
          for (int m = 0; m < M; ++m)
            o[m][TILE + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                vf[i], __builtin_bit_cast(half8_t, piece ? ph[m] : pl[m]), o[m][TILE + i], 0, 0, 0);
        }
    tree_tiles<T, HD, M, DRAFTS, TILE + N>(x, ph, pl, mg, odd, o);
  }
}

// Two wavefronts per SIMD where the registers allow it: one's decoding and
// exponentials run under the other's matrix instructions.
constexpr int tree_waves_per_simd(uint32_t type, int hd, int m) {
  return (type == T_F32 && hd * m >= 256) || (hd == 256 && (type == T_F16 || type == T_Q8_0)) || hd * m > 256 ? 1 : 2;
}
template <uint32_t T, int HD, int M>
__global__ __launch_bounds__(64 * tree_wide(T, HD, M), tree_wide(T, HD, M) == 8 ? 1 : tree_waves_per_simd(T, HD, M)) void tree_mfma(
    const float* q, uint64_t q_stride, const uint8_t* k_codes, const uint32_t* length, uint32_t rows, uint32_t G,
    uint32_t row, uint32_t all_tiles, uint32_t all_per, uint32_t all_total, TreeArgs a) {
  using D = TreeDims<HD>;
  using Tile = TreeTile<T, HD>;
  using S = TreeShared<T, HD, M>;
  constexpr bool F32 = T == T_F32;
  constexpr uint32_t W = S::W;
  __shared__ S sh;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, c = lane & 15u, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // uniform: the tiles' descriptors are scalars
  const uint32_t split = blockIdx.x, head = blockIdx.z, row0 = blockIdx.y * (M * 16u);
  const uint32_t words = a.words;

  // this lane's Q: wavefront w has row tiles w, w + 4, ..; requested before the cache's rows
  float x[HD / 4];
  auto ask_q = [&](int m) {
    const uint32_t r = min(row0 + 16u * m + c, rows - 1u), i = r / G;
    const float* const qp = q + (uint64_t)i * q_stride + ((uint64_t)head * G + (r - i * G)) * HD + g * (HD / 4);
    tree_get_q<HD>(x, qp, a.q_vec);
  };
  static_assert(M <= (int)W, "a row tile per wavefront");
  if (wave < (uint32_t)M) ask_q((int)wave);
  __builtin_amdgcn_sched_barrier(0);

  uint64_t hist = a.hist, total = all_total;
  uint32_t tiles = all_tiles, per = all_per;
  if (length) {
    tree_range(a, hist, total);
    tiles = (uint32_t)((total + TREE_KEYS - 1u) / TREE_KEYS);
    per = (tiles + a.nsplit - 1u) / a.nsplit;
  }
  const uint32_t t0 = min(tiles, split * per), t1 = min(tiles, t0 + per);
  const uint32_t srow = a.scale_row;
  const uint64_t sbase = a.scale_base;
  Tile cur;
  // Bounded descriptors: rows behind the last read as zeros, and nothing is
  // read for a tile behind the last.  The loads are in no branch and in this
  // order, here and in the loop, so that a wait for one of them (they return
  // in order) is a wait for no later one.
  auto rows_of = [&](uint32_t tile) { return tile < t1 ? (uint32_t)min((uint64_t)TREE_KEYS, total - (uint64_t)tile * TREE_KEYS) : 0u; };
  auto fetch_k = [&](uint32_t tile) {
    const uint64_t p = (uint64_t)tile * TREE_KEYS;
    const uint32_t np = rows_of(tile);
    cur.load_k(tree_rsrc(k_codes + p * row, np * row), tree_rsrc(a.cache.k + sbase + p * srow, np * srow), row, srow,
               head, c, g);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto fetch_v = [&](uint32_t tile) {
    const uint64_t p = (uint64_t)tile * TREE_KEYS;
    const uint32_t np = rows_of(tile);
    cur.load_v(tree_rsrc(a.cache.v + p * row, np * row), tree_rsrc(a.cache.v + sbase + p * srow, np * srow), row, srow,
               head, c, g);
    __builtin_amdgcn_sched_barrier(0);
  };
  uint32_t tile = t0 + wave;
  fetch_k(tile);
  fetch_v(tile);
  if (wave < (uint32_t)M) tree_put_q<T, HD, M>(sh, (int)wave, x, lane);
  __syncthreads();

  uint32_t tok[M];
  float scale[M], ref[M], l[M];
  f32x4 o[M][D::TILES];
  const float minus = tree_minus();
  const TreeMagic mg;
#pragma unroll
  for (int m = 0; m < M; ++m) {
    tok[m] = min(row0 + 16u * m + c, rows - 1u) / G;
    scale[m] = sh.scale[m][c];
    ref[m] = TREE_FLOOR;
    l[m] = 0.f;
#pragma unroll
    for (int d = 0; d < D::TILES; ++d) o[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  auto step = [&](auto drafts) {
    constexpr bool DRAFTS = decltype(drafts)::value;  // the tile has positions that some rows may not see
    __builtin_amdgcn_s_setprio(0);
    const uint64_t p0 = (uint64_t)tile * TREE_KEYS;
    // scores of row c at positions p0 + 16 t + 4 g + v
    f32x4 s[M][2];
#pragma unroll
    for (int m = 0; m < M; ++m) s[m][0] = s[m][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < HD / 16; ++i)
#pragma unroll
        for (int m = 0; m < M; ++m) {
          const u32x4 w = sh.q[m][i][lane];
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int t = 0; t < 2; ++t)
              s[m][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(cur.k[t][4 * i + e]), __uint_as_float(w[e]),
                                                              s[m][t], 0, 0, 0);
        }
    } else {
#pragma unroll
      for (int i = 0; i < D::STEPS; ++i) {
        const half8_t k0 = cur.kfrag(0, i, mg), k1 = cur.kfrag(1, i, mg);
#pragma unroll
        for (int piece = 0; piece < 2; ++piece)
#pragma unroll
          for (int m = 0; m < M; ++m) {
            const half8_t qf = __builtin_bit_cast(half8_t, sh.q[m][2 * i + piece][lane]);
            s[m][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qf, s[m][0], 0, 0, 0);
            s[m][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qf, s[m][1], 0, 0, 0);
          }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    fetch_k(tile + W);  // the old words are spent
    // ahead of a wavefront that is at its scores: the two of a SIMD stay apart,
    // one at vector instructions while the other feeds the matrix cores (1 to 2%)
    __builtin_amdgcn_s_setprio(1);
    float p[M][8];
    uint32_t see[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
      see[m] = DRAFTS ? tree_places(a, words, tok[m], p0, hist, total, g) : 0xFFu;
      tree_soften<HD, DRAFTS>(s[m], see[m], scale[m], ref[m], l[m], o[m], p[m]);
    }
    bool odd = false;
    if constexpr (F32) {
#pragma unroll
      for (int d = 0; d < D::TILES; ++d)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float v = __uint_as_float(cur.v[j][d]);
          if (DRAFTS && !(fabsf(v) <= 3.402823466e38f)) {
            odd = true;
            v = 0.f;
          }
#pragma unroll
          for (int m = 0; m < M; ++m) o[m][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p[m][j], o[m][d], 0, 0, 0);
        }
    } else {
      u32x4 ph[M], pl[M];
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t h, r;
          tree_pieces(p[m][2 * j], p[m][2 * j + 1], minus, h, r);
          ph[m][j] = h;
          pl[m][j] = r;
        }
      tree_tiles<T, HD, M, DRAFTS, 0>(cur, ph, pl, mg, odd, o);
    }
    __builtin_amdgcn_sched_barrier(0);
    fetch_v(tile + W);
    if (DRAFTS && __any(odd)) tree_odd_rows<HD, M>(a, p, see, p0, total, head, c, g, sh.odd[wave], o);
  };
  // the drafts come last
  for (; tile < t1 && (uint64_t)tile * TREE_KEYS + TREE_KEYS <= hist; tile += W) step(std::false_type());
  for (; tile < t1; tile += W) step(std::true_type());

  __builtin_amdgcn_s_setprio(0);
  // Join the wavefronts: all their sums in LDS (in Q's place, so once all are
  // done with it), and what a sum weighs is worked out where it is added.
  __syncthreads();
#pragma unroll
  for (int m = 0; m < M; ++m) {
    l[m] += __shfl_xor(l[m], 16);
    l[m] += __shfl_xor(l[m], 32);
    if (g == 0) {
      sh.m[wave][16 * m + c] = ref[m];
      sh.l[wave][16 * m + c] = l[m];
    }
#pragma unroll
    for (int d = 0; d < D::TILES; ++d)
#pragma unroll
      for (uint32_t v = 0; v < 4; ++v) sh.sum[wave][(16 * m + c) * S::OP + D::dim(d, 4u * g + v)] = o[m][d][v];
  }
  __syncthreads();
#pragma unroll
  for (uint32_t e0 = 0; e0 < M * 16u * HD / 4u; e0 += 64u * W) {
    const uint32_t e = e0 + tid, rr = e / (HD / 4u), d = e % (HD / 4u) * 4u, r = row0 + rr;
    if (e >= M * 16u * HD / 4u || r >= rows) continue;
    float w[W], best = TREE_FLOOR, sum = 0.f;
#pragma unroll
    for (uint32_t k = 0; k < W; ++k) best = fmaxf(best, w[k] = sh.m[k][rr]);
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t k = 0; k < W; ++k) {
      w[k] = __builtin_amdgcn_exp2f(w[k] - best);
      sum = fmaf(sh.l[k][rr], w[k], sum);
      const f32x4 z = *reinterpret_cast<const f32x4*>(&sh.sum[k][rr * S::OP + d]);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = fmaf(z[i], w[k], y[i]);
    }
    const uint32_t i = r / G, h = head * G + (r - i * G);
    if (a.nsplit == 1) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      float* const out = a.out + (uint64_t)i * a.out_stride + (uint64_t)h * HD + d;
#pragma unroll
      for (int k = 0; k < 4; ++k) out[k] = y[k] * inv;
    } else {
      float* const rec = a.ws + (((uint64_t)split * a.n + i) * a.qh + h) * (HD + 4);
      *reinterpret_cast<f32x4*>(rec + d) = y;
      if (d == 0) { rec[HD] = best; rec[HD + 1] = sum; }
    }
  }
}

// ------------------------------------------- rows over the wavefronts

// With many rows the decoding is what a wavefront does most: here the four
// wavefronts of a workgroup have rows of their own (M tiles of 16 each) and the
// same positions, each decodes a quarter of a tile into LDS as the matrix
// instructions take it, and all read it from there.  Tiles are double-buffered:
// one barrier each; the words of the next but one are in flight.
// 512 rows over 32128 Q8_0 positions 141 us, 0.96 PFLOP/s; bound by the chain of
// a tile (LDS reads, scores, softmax, sums) with two wavefronts a SIMD.
//   Wavefront w decodes, of K, half tile w % 2 and steps from w / 2 (STEPS / 2
//   rounded up), and of V its positions 4 t + v = 2 w, 2 w + 1 for all dims:
//   word w of every tile's operand.
template <uint32_t T, int HD> struct TreePart {
  using Tile = TreeTile<T, HD>;
  using D = TreeDims<HD>;
  static constexpr int KSTEPS = (D::STEPS + 1) / 2, SW = Tile::BITS / 4;  // steps, words of a step
  uint32_t k[KSTEPS * SW], ks[KSTEPS], v[2][Tile::VW], vs[2][2];

  __device__ __forceinline__ void load_k(TreeRsrc kr, TreeRsrc ksr, uint32_t row, uint32_t srow, uint32_t head,
                                         uint32_t c, uint32_t g, uint32_t wave) {
    const uint32_t p = 16u * (wave & 1u) + c, s0 = (wave >> 1) * KSTEPS;
    tree_words<KSTEPS * SW>(k, kr, p * row + head * (HD * Tile::BITS / 8) + g * (D::STEPS * SW * 4u) + s0 * (SW * 4u));
    if constexpr (Tile::QUANT) {
#pragma unroll
      for (int i = 0; i < KSTEPS; ++i)
        if (i == 0 || HD == 96)  // elsewhere a wavefront's steps lie in one block
          ks[i] = tree_u16(ksr, p * srow + head * (HD / 16) + 2u * ((g * (HD / 4) + 8u * (s0 + i)) / 32u));
    }
  }
  __device__ __forceinline__ void load_v(TreeRsrc vr, TreeRsrc vsr, uint32_t row, uint32_t srow, uint32_t head,
                                         uint32_t c, uint32_t g, uint32_t wave) {
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      const uint32_t j = 2u * wave + i, p = 16u * (j / 4u) + 4u * g + j % 4u, hb = head * (HD * Tile::BITS / 8);
      tree_bytes<Tile::B0>(v[i], vr, p * row + hb + c * Tile::B0);
      if constexpr (Tile::B1 > 0) tree_bytes<Tile::B1>(v[i] + Tile::VW0, vr, p * row + hb + 16u * Tile::B0 + c * Tile::B1);
      if constexpr (Tile::QUANT) {
        vs[i][0] = tree_u16(vsr, p * srow + head * (HD / 16) + 2u * (c * D::W0 / 32u));
        if constexpr (Tile::VS == 2) vs[i][1] = tree_u16(vsr, p * srow + head * (HD / 16) + 4u);
      }
    }
  }
  __device__ __forceinline__ half8_t kfrag(int s, const TreeMagic& mg) const {
    u32x4 w;
    if constexpr (T == T_F16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = k[4 * s + i];
    } else {
      Tile::decode_k(k + s * SW, ks[HD == 96 ? s : 0], mg, w);
    }
    return __builtin_bit_cast(half8_t, w);
  }
};

template <int HD> struct TreeRowsShared {
  u32x4 k[2][2][TreeDims<HD>::STEPS][64];  // buffer, half tile, step, lane
  u32x4 v[2][TreeDims<HD>::TILES][64];
  float odd[TREE_WAVES][16 * TREE_ODD];
};

template <uint32_t T, int HD, int M>
__global__ __launch_bounds__(64 * TREE_WAVES, 2) void tree_rows(TreeArgs a) {
  using D = TreeDims<HD>;
  using Tile = TreeTile<T, HD>;
  using Part = TreePart<T, HD>;
  __shared__ TreeRowsShared<HD> sh;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, c = lane & 15u, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t split = blockIdx.x, head = blockIdx.z, row0 = (blockIdx.y * TREE_WAVES + wave) * (M * 16u);
  const uint32_t G = a.group, rows = a.rows, words = a.words;
  uint64_t hist = a.hist, total = a.total;
  uint32_t tiles = a.tiles, per = a.per;
  if (a.cache.length) {
    tree_range(a, hist, total);
    tiles = (uint32_t)((total + TREE_KEYS - 1u) / TREE_KEYS);
    per = (tiles + a.nsplit - 1u) / a.nsplit;
  }
  const uint32_t t0 = min(tiles, split * per), t1 = min(tiles, t0 + per);
  const uint32_t row = a.code_row, srow = a.scale_row;
  const uint64_t sbase = a.scale_base;
  Part part;
  auto fetch = [&](uint32_t tile) {  // as in tree_mfma: in no branch
    const uint64_t p = (uint64_t)tile * TREE_KEYS;
    const uint32_t np = tile < t1 ? (uint32_t)min((uint64_t)TREE_KEYS, total - p) : 0u;
    part.load_k(tree_rsrc(a.cache.k + p * row, np * row), tree_rsrc(a.cache.k + sbase + p * srow, np * srow), row, srow,
                head, c, g, wave);
    part.load_v(tree_rsrc(a.cache.v + p * row, np * row), tree_rsrc(a.cache.v + sbase + p * srow, np * srow), row, srow,
                head, c, g, wave);
    __builtin_amdgcn_sched_barrier(0);
  };
  const TreeMagic mg;
  auto put = [&](uint32_t buf) {
    const uint32_t t = wave & 1u, s0 = (wave >> 1) * Part::KSTEPS;
#pragma unroll
    for (int i = 0; i < Part::KSTEPS; ++i)
      if (D::STEPS % 2 == 0 || s0 + i < (uint32_t)D::STEPS) sh.k[buf][t][s0 + i][lane] = __builtin_bit_cast(u32x4, part.kfrag(i, mg));
    uint32_t w[D::TILES];
    Tile::decode_v(part.v[0], part.v[1], part.vs[0], part.vs[1], mg, w);
#pragma unroll
    for (int d = 0; d < D::TILES; ++d) reinterpret_cast<uint32_t*>(&sh.v[buf][d][lane])[wave] = w[d];
  };

  half8_t qh[M][D::STEPS], ql[M][D::STEPS];
  uint32_t tok[M];
  float scale[M], ref[M], l[M];
  f32x4 o[M][D::TILES];
  const float minus = tree_minus();
  float x[M][HD / 4];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const uint32_t r = min(row0 + 16u * m + c, rows - 1u);
    tok[m] = r / G;
    const float* const qp = a.q + (uint64_t)tok[m] * a.q_stride + ((uint64_t)head * G + (r - tok[m] * G)) * HD + g * (HD / 4);
    tree_get_q<HD>(x[m], qp, a.q_vec);
  }
  __builtin_amdgcn_sched_barrier(0);
  fetch(t0);
#pragma unroll
  for (int m = 0; m < M; ++m) {
    scale[m] = tree_split_q<T, HD>(x[m], [&](int s, int piece, u32x4 w) {
      (piece ? qh : ql)[m][s] = __builtin_bit_cast(half8_t, w);
    });
    ref[m] = TREE_FLOOR;
    l[m] = 0.f;
#pragma unroll
    for (int d = 0; d < D::TILES; ++d) o[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  put(0);
  fetch(t0 + 1);
  __syncthreads();

  auto step = [&](auto drafts, uint32_t tile, uint32_t buf) {
    constexpr bool DRAFTS = decltype(drafts)::value;
    __builtin_amdgcn_s_setprio(0);
    const uint64_t p0 = (uint64_t)tile * TREE_KEYS;
    f32x4 s[M][2];
#pragma unroll
    for (int m = 0; m < M; ++m) s[m][0] = s[m][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D::STEPS; ++i) {
      const half8_t k0 = __builtin_bit_cast(half8_t, sh.k[buf][0][i][lane]), k1 = __builtin_bit_cast(half8_t, sh.k[buf][1][i][lane]);
#pragma unroll
      for (int piece = 0; piece < 2; ++piece)
#pragma unroll
        for (int m = 0; m < M; ++m) {
          s[m][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, piece ? qh[m][i] : ql[m][i], s[m][0], 0, 0, 0);
          s[m][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, piece ? qh[m][i] : ql[m][i], s[m][1], 0, 0, 0);
        }
    }
    __builtin_amdgcn_s_setprio(1);  // as in tree_mfma
    float p[M][8];
    uint32_t see[M];
    u32x4 ph[M], pl[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
      see[m] = DRAFTS ? tree_places(a, words, tok[m], p0, hist, total, g) : 0xFFu;
      tree_soften<HD, DRAFTS>(s[m], see[m], scale[m], ref[m], l[m], o[m], p[m]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t h, r;
        tree_pieces(p[m][2 * j], p[m][2 * j + 1], minus, h, r);
        ph[m][j] = h;
        pl[m][j] = r;
      }
    }
    bool odd = false;
    constexpr int N = M == 1 ? 4 : 2;
#pragma unroll
    for (int d = 0; d < D::TILES; d += N) {
      half8_t vf[N];
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (d + i < D::TILES) {
          vf[i] = __builtin_bit_cast(half8_t, sh.v[buf][d + i][lane]);
          if (DRAFTS) vf[i] = tree_finite(vf[i], odd);
        }
#pragma unroll
      for (int piece = 0; piece < 2; ++piece)
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (d + i < D::TILES) {
#pragma unroll
            for (int m = 0; m < M; ++m)
              o[m][d + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[i], __builtin_bit_cast(half8_t, piece ? ph[m] : pl[m]),
                                                                    o[m][d + i], 0, 0, 0);
          }
    }
    if (DRAFTS && __any(odd)) tree_odd_rows<HD, M>(a, p, see, p0, total, head, c, g, sh.odd[wave], o);
    put(buf ^ 1u);
    fetch(tile + 2u);
    __syncthreads();
  };
  uint32_t buf = 0, tile = t0;
  for (; tile < t1 && (uint64_t)tile * TREE_KEYS + TREE_KEYS <= hist; ++tile, buf ^= 1u) step(std::false_type(), tile, buf);
  for (; tile < t1; ++tile, buf ^= 1u) step(std::true_type(), tile, buf);

  // each wavefront has its rows alone
#pragma unroll
  for (int m = 0; m < M; ++m) {
    l[m] += __shfl_xor(l[m], 16);
    l[m] += __shfl_xor(l[m], 32);
    const uint32_t r = row0 + 16u * m + c;
    if (r >= rows) continue;
    const uint32_t h = head * G + (r - tok[m] * G);
    const bool whole = a.nsplit == 1;
    const float inv = whole ? (l[m] == 0.f ? 0.f : 1.f / l[m]) : 1.f;
    float* const rec = a.ws + (((uint64_t)split * a.n + tok[m]) * a.qh + h) * (HD + 4);
    float* const out = whole ? a.out + (uint64_t)tok[m] * a.out_stride + (uint64_t)h * HD : rec;
#pragma unroll
    for (int d = 0; d < D::TILES; d += D::W1 ? 2 : 4)
#pragma unroll
      for (uint32_t v = 0; v < 4; ++v) {
        constexpr int N = D::W1 ? 2 : 4;  // consecutive tiles are consecutive dims
        float* const to = out + D::dim(d, 4u * g + v);
        if (whole) {
#pragma unroll
          for (int i = 0; i < N; ++i) to[i] = o[m][d + i][v] * inv;
        } else if constexpr (N == 4) {
          *reinterpret_cast<float4*>(to) = make_float4(o[m][d][v], o[m][d + 1][v], o[m][d + 2][v], o[m][d + 3][v]);
        } else {
          *reinterpret_cast<float2*>(to) = make_float2(o[m][d][v], o[m][d + 1][v]);
        }
      }
    if (!whole && g == 0) {
      rec[HD] = ref[m];
      rec[HD + 1] = l[m];
    }
  }
}

// Joins a row's records: HD / 4 lanes of 4 dims take every JOIN-th split, and
// their sums meet in LDS, so that a row of many splits is a few loads deep.  2.4
// us for 32 rows, 4.8 for 512 of 16 splits.
template <int HD>
__global__ __launch_bounds__(256) void tree_join(const float* ws, float* to, uint64_t out_stride,
                                                 uint32_t n_rows, uint32_t qh, uint32_t nsplit) {
  constexpr uint32_t LANES = HD / 4, JOIN = 256u / LANES;
  __shared__ __align__(16) float y[JOIN][HD + 4];
  const uint64_t rows = n_rows, r = blockIdx.x;
  const uint32_t part = threadIdx.x / LANES, d = threadIdx.x % LANES * 4u;
  const float* const rec = ws + r * (HD + 4);
  const uint64_t step = rows * (HD + 4);
  if (part < JOIN) {
    float top = TREE_FLOOR, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (uint32_t s = part; s < nsplit; s += JOIN) {
      const float* const at = rec + s * step;
      const float4 z = *reinterpret_cast<const float4*>(at + d);
      const float m = at[HD], now = fmaxf(top, m), al = __builtin_amdgcn_exp2f(top - now), w = __builtin_amdgcn_exp2f(m - now);
      top = now;
      sum = fmaf(sum, al, at[HD + 1] * w);
      o[0] = fmaf(o[0], al, z.x * w); o[1] = fmaf(o[1], al, z.y * w);
      o[2] = fmaf(o[2], al, z.z * w); o[3] = fmaf(o[3], al, z.w * w);
    }
    *reinterpret_cast<float4*>(&y[part][d]) = make_float4(o[0], o[1], o[2], o[3]);
    if (d == 0) { y[part][HD] = top; y[part][HD + 1] = sum; }
  }
  __syncthreads();
  if (part != 0) return;
  float top = TREE_FLOOR, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (uint32_t p = 0; p < JOIN; ++p) top = fmaxf(top, y[p][HD]);
#pragma unroll
  for (uint32_t p = 0; p < JOIN; ++p) {
    const float w = __builtin_amdgcn_exp2f(y[p][HD] - top);
    const float4 z = *reinterpret_cast<const float4*>(&y[p][d]);
    sum = fmaf(y[p][HD + 1], w, sum);
    o[0] = fmaf(z.x, w, o[0]); o[1] = fmaf(z.y, w, o[1]); o[2] = fmaf(z.z, w, o[2]); o[3] = fmaf(z.w, w, o[3]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  float* const out = to + r / qh * out_stride + r % qh * HD + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = o[e] * inv;
}

// ---------------------------------------------------------------- launches

static bool tree_on_matrix_cores(uint32_t hd) { return hd == 64 || hd == 96 || hd == 128 || hd == 256; }

// The kernel of a shape.  tree_mfma, whose wavefronts split the positions, has
// few records to join; tree_rows, whose wavefronts split the rows, decodes less
// and reads the cache fewer times.  The first is ahead until every CU has 5 hd
// pairs of a row tile and a tile of positions (us in the first and the second,
// 8 KV heads of 128: 64 rows over 8192 Q8_0 positions 18.3 and 27.2, 256 over
// 8192 31.0 and 47.8, 1024 over 8256 84 and 95, 512 over 16128 85.9 and 87.8,
// 64 over 131072 Q4_0 positions 89.7 and 96.1, 256 over 65600 155 and 144, 512
// over 32128 Q8_0 positions 160 and 141; 2 of 64, 1400 rows over 8200 F16
// positions 30.8 and 33.4, over 16200 51.4 and 45.6).  An f32 cache has nothing
// to decode and stays with it.
//
// Row tiles of a wavefront in the first: two where that leaves a workgroup for
// every CU, one otherwise (37 tokens over 637 f32 positions: 12.3 us with one,
// 16.7 with two; 1024 rows over 8256 Q8_0 positions 133 and 83).
struct TreePlan {
  bool rows_apart;
  uint32_t tiles, block_rows;  // row tiles of a wavefront, rows of a workgroup
};
constexpr uint32_t TREE_CUS = 256, TREE_LEAST = 4;  // tiles of a split at least
static TreePlan tree_plan(uint64_t rows, uint32_t kvh, uint64_t total, uint32_t hd, uint32_t type) {
  const uint64_t tiles = (total + TREE_KEYS - 1) / TREE_KEYS, work = tiles * kvh * ((rows + 15) / 16);
  TreePlan p{type != T_F32 && rows > 32 && work > 5ull * hd * TREE_CUS, 1, 16};
  if (p.rows_apart) {
    p.tiles = rows > 64 && hd != 256 ? 2 : 1;
    p.block_rows = 16 * TREE_WAVES * p.tiles;
  } else {
    const uint64_t splits = (tiles + TREE_LEAST - 1) / TREE_LEAST;
    p.tiles = rows > 16 && hd != 256 && kvh * ((rows + 15) / 16) * splits > TREE_CUS ? 2 : 1;
    p.block_rows = 16 * p.tiles;
  }
  return p;
}

// Splits for at most one workgroup a CU (tree_mfma, whose records grow with the
// splits: 64 rows over 8192 positions 18.0 us, 26.3 with two a CU) or two
// (tree_rows: 141 us against 160 with one at 512 rows over 32128).  At most: one
// workgroup too many is a second round for all (80 rows over 8192 positions
// 20.4 us with 240 workgroups, 28.2 with 264).
uint32_t tree_splits(uint64_t total, uint32_t n, uint32_t qh, uint32_t kvh, uint32_t hd, uint32_t type) {
  if (!tree_on_matrix_cores(hd)) return 1;
  const uint64_t rows = (uint64_t)n * (qh / kvh);
  const TreePlan p = tree_plan(rows, kvh, total, hd, type);
  const uint64_t units = kvh * ((rows + p.block_rows - 1) / p.block_rows), tiles = (total + TREE_KEYS - 1) / TREE_KEYS;
  const uint64_t want = (p.rows_apart ? 2 : 1) * TREE_CUS / units;
  const uint64_t most = (tiles + TREE_LEAST - 1) / TREE_LEAST, s = want < most ? want : most;
  return (uint32_t)(s ? s : 1);
}
uint64_t tree_ws_floats(uint32_t nsplit, uint32_t n, uint32_t qh, uint32_t hd) {
  return nsplit > 1 ? (uint64_t)nsplit * n * qh * (hd + 4) : 0;
}

// A longer context or more tokens may go another way: the most over the ways
// and over every smaller n (fewer rows, more splits).
uint64_t tree_ws_floats_upto(uint64_t total, uint32_t n, uint32_t qh, uint32_t kvh, uint32_t hd, uint32_t type) {
  if (!tree_on_matrix_cores(hd)) return 0;
  uint64_t most = 0;
  const uint64_t tiles = (total + TREE_KEYS - 1) / TREE_KEYS, cut = (tiles + TREE_LEAST - 1) / TREE_LEAST;
  for (uint32_t m = 1; m <= n; ++m) {
    const uint64_t rows = (uint64_t)m * (qh / kvh);
    for (uint32_t block : {16u, 32u, 64u, 128u}) {  // rows of a workgroup; two a CU from 64
      const uint64_t units = kvh * ((rows + block - 1) / block), want = (block < 64 ? 1 : 2) * TREE_CUS / units;
      const uint64_t s = want < cut ? want : cut, need = tree_ws_floats((uint32_t)s, m, qh, hd);
      most = need > most ? need : most;
    }
  }
  return most;
}

// What a workgroup needs before its first load goes in front of the rest, as
// scalars: the kernels of this file are built with their first 14 words of
// arguments preloaded into registers, and do not wait for them (64 rows over
// 8192 positions: tree_mfma 15.9 -> 14.9 us; the join of 32 rows 3.0 -> 2.4).
#define TREE_FIRST \
  a.q, a.q_stride, a.cache.k, a.cache.length, a.rows, a.group, a.code_row, a.tiles, a.per, (uint32_t)a.total
template <uint32_t T, int HD>
static void launch_tree(const TreeArgs& a, hipStream_t st) {
  const TreePlan p = tree_plan(a.rows, a.cache.kvh, a.total, HD, T);
  const dim3 grid(a.nsplit, (a.rows + p.block_rows - 1) / p.block_rows, a.cache.kvh), wg(64 * TREE_WAVES);
  if (p.rows_apart) {
    if constexpr (T != T_F32) {
      if constexpr (HD <= 128) {
        if (p.tiles == 2) RF_KLAUNCH((tree_rows<T, HD, 2>), grid, wg, 0, st, a);
      }
      if (p.tiles == 1) RF_KLAUNCH((tree_rows<T, HD, 1>), grid, wg, 0, st, a);
    }
  } else {
    if constexpr (HD <= 128) {
      if (p.tiles == 2) RF_KLAUNCH((tree_mfma<T, HD, 2>), grid, dim3(64 * tree_wide(T, HD, 2)), 0, st, TREE_FIRST, a);
    }
    if (p.tiles == 1) RF_KLAUNCH((tree_mfma<T, HD, 1>), grid, wg, 0, st, TREE_FIRST, a);
  }
  if (a.nsplit > 1)
    RF_KLAUNCH(tree_join<HD>, dim3(a.n * a.qh), dim3(256), 0, st, a.ws, a.out, a.out_stride, a.n * a.qh, a.qh, a.nsplit);
}

template <uint32_t T>
static void launch_tree_type(const TreeArgs& a, hipStream_t st) {
  switch (a.cache.hd) {
    case 64: launch_tree<T, 64>(a, st); break;
    case 96: launch_tree<T, 96>(a, st); break;
    case 128: launch_tree<T, 128>(a, st); break;
    default: launch_tree<T, 256>(a, st);
  }
}

hipError_t launch_attention_tree(const TreeArgs& args, hipStream_t st) {
  TreeArgs a = args;
  const uint64_t width = (uint64_t)a.cache.kvh * a.cache.hd;
  a.group = a.qh / a.cache.kvh;
  a.rows = a.n * a.group;
  a.words = (a.n + 63u) / 64u;
  a.code_row = (uint32_t)kv_code_bytes(a.cache.type, width);
  a.scale_row = (uint32_t)(kv_row_bytes(a.cache.type, width) - a.code_row);
  a.scale_base = a.cache.cap * a.code_row;
  a.tiles = (uint32_t)((a.total + TREE_KEYS - 1) / TREE_KEYS);
  a.per = (a.tiles + a.nsplit - 1) / a.nsplit;
  if (!tree_on_matrix_cores(a.cache.hd)) {
    RF_KLAUNCH(tree_plain, dim3(a.n, a.qh), dim3(256), 0, st, a);
    return hipGetLastError();
  }
  switch (a.cache.type) {
    case T_F32: launch_tree_type<T_F32>(a, st); break;
    case T_F16: launch_tree_type<T_F16>(a, st); break;
    case T_Q8_0: launch_tree_type<T_Q8_0>(a, st); break;
    default: launch_tree_type<T_Q4_0>(a, st);
  }
  return hipGetLastError();
}

hipError_t load_module_tree() {
  hipFuncAttributes fa;
  return hipFuncGetAttributes(&fa, reinterpret_cast<const void*>(&tree_plain));
}

}  // namespace rf
