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
// (x | magic) is an f16 pair of `one` + codes with their offset; minus that it is the codes.
__device__ __forceinline__ uint32_t pk_code(uint32_t x, uint32_t mask, uint32_t magic, float off) {
  const half2_t o = {(_Float16)off, (_Float16)off};
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, (x & mask) | magic) - o);
}
__device__ __forceinline__ uint32_t pk_q8(uint32_t x) { return pk_code(x, 0x00FF00FFu, 0x64006400u, 1152.f); }
// Nibble k (0..3) of both halves of x.
template <int K>
__device__ __forceinline__ uint32_t pk_q4(uint32_t x) {
  if constexpr (K >= 2) x >>= 8;
  return K % 2 ? pk_code(x, 0x00F000F0u, 0x54005400u, 72.f) : pk_code(x, 0x000F000Fu, 0x64006400u, 1032.f);
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
  __device__ __forceinline__ void load(TreeRsrc kr, TreeRsrc ksr, TreeRsrc vr, TreeRsrc vsr, uint32_t row,
                                       uint32_t srow, uint32_t head, uint32_t c, uint32_t g) {
    const uint32_t hb = head * (HD * BITS / 8), hs = head * (HD / 16);
#pragma unroll
    for (uint32_t t = 0; t < 2; ++t) {
      const uint32_t p = 16u * t + c;
      tree_words<KW>(k[t], kr, p * row + hb + g * (KW * 4u));
      if constexpr (QUANT) {
#pragma unroll
        for (uint32_t i = 0; i < (uint32_t)KS; ++i) {
          const uint32_t b = HD == 96 ? (g * 24u + 8u * i) / 32u : HD == 64 ? g / 2u : g * (HD / 128) + i;
          ks[t][i] = tree_u16(ksr, p * srow + hs + 2u * b);
        }
      }
    }
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

  __device__ __forceinline__ half8_t kfrag(int t, int s) const {
    u32x4 w;
    if constexpr (T == T_F16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = k[t][4 * s + i];
    } else {
      const uint32_t sc = ks[t][HD == 96 ? s : s / 4], sc2 = sc | sc << 16;
      if constexpr (T == T_Q8_0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t x = k[t][2 * s + i];
          w[2 * i] = pk_mul(pk_q8(__builtin_amdgcn_perm(0u, x, 0x0C010C00u)), sc2);
          w[2 * i + 1] = pk_mul(pk_q8(__builtin_amdgcn_perm(0u, x, 0x0C030C02u)), sc2);
        }
      } else {
        const uint32_t x = k[t][s];
        w[0] = pk_mul(pk_q4<0>(x), sc2);
        w[1] = pk_mul(pk_q4<1>(x), sc2);
        w[2] = pk_mul(pk_q4<2>(x), sc2);
        w[3] = pk_mul(pk_q4<3>(x), sc2);
      }
    }
    return __builtin_bit_cast(half8_t, w);
  }
  // V^T's tile of 16 dims
  template <int TILE>
  __device__ __forceinline__ half8_t vfrag() const {
    constexpr int seg = TILE < D::W0 ? 0 : 1, e = seg ? TILE - D::W0 : TILE, per = 32 / BITS;  // element e of the lane's dims
    constexpr int word = (seg ? VW0 : 0) + e / per, in = e % per;
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = v[2 * i][word], b = v[2 * i + 1][word];
      if constexpr (T == T_F16) {
        w[i] = __builtin_amdgcn_perm(b, a, in ? 0x07060302u : 0x05040100u);
      } else {
        const uint32_t s2 = vs[2 * i][seg] | vs[2 * i + 1][seg] << 16;
        if constexpr (T == T_Q8_0) {
          w[i] = pk_mul(pk_q8(__builtin_amdgcn_perm(b, a, 0x0C040C00u + 0x00010001u * in)), s2);
        } else {
          const uint32_t x = __builtin_amdgcn_perm(b, a, in < 4 ? 0x05040100u : 0x07060302u);
          w[i] = pk_mul(pk_q4<in % 4>(x), s2);
        }
      }
    }
    return __builtin_bit_cast(half8_t, w);
  }
};

// The f32 cache's tile.
template <int HD> struct TreeTile<T_F32, HD> {
  using D = TreeDims<HD>;
  static constexpr bool QUANT = false;
  uint32_t k[2][HD / 4], v[8][HD / 16];
  __device__ __forceinline__ void load(TreeRsrc kr, TreeRsrc, TreeRsrc vr, TreeRsrc, uint32_t row, uint32_t,
                                       uint32_t head, uint32_t c, uint32_t g) {
#pragma unroll
    for (uint32_t t = 0; t < 2; ++t) tree_words<HD / 4>(k[t], kr, (16u * t + c) * row + head * (HD * 4u) + g * HD);
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      const uint32_t off = (16u * (j / 4u) + 4u * g + j % 4u) * row + head * (HD * 4u);
      tree_words<D::W0>(v[j], vr, off + c * (D::W0 * 4u));
      if constexpr (D::W1 > 0) tree_words<D::W1>(v[j] + D::W0, vr, off + 16u * D::W0 * 4u + c * (D::W1 * 4u));
    }
  }
  static __device__ __forceinline__ constexpr int order(int i) { return i; }
};

constexpr float TREE_FLOOR = -1e30f;  // reference of a row that has seen nothing
// A row's reference is set 2^12 below its largest score and moves once a weight
// would pass 2^15: weights stay inside f16, and as far as can be above its
// subnormals, which a weight 2^-26 of the largest meets.
constexpr float TREE_BELOW = 12.f, TREE_MOST = 15.f;
constexpr uint32_t TREE_WAVES = 4, TREE_KEYS = 32;

template <uint32_t T, int HD, int M, int TILE>
__device__ __forceinline__ void tree_tiles(const TreeTile<T, HD>& x, const half8_t (&ph)[M], const half8_t (&pl)[M],
                                           bool drafts, bool& odd, f32x4 (&o)[M][TreeDims<HD>::TILES]) {
  if constexpr (TILE < TreeDims<HD>::TILES) {
    half8_t vf = x.template vfrag<TILE>();
    if (drafts) {
      u32x4 w = __builtin_bit_cast(u32x4, vf);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t keep = ((w[i] & 0x7C00u) == 0x7C00u ? 0u : 0xFFFFu) | ((w[i] & 0x7C000000u) == 0x7C000000u ? 0u : 0xFFFF0000u);
        odd |= keep != 0xFFFFFFFFu;
        w[i] &= keep;
      }
      vf = __builtin_bit_cast(half8_t, w);
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
      o[m][TILE] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[m], o[m][TILE], 0, 0, 0);
      o[m][TILE] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[m], o[m][TILE], 0, 0, 0);
    }
    tree_tiles<T, HD, M, TILE + 1>(x, ph, pl, drafts, odd, o);
  }
}

// Non-finite values of the tile's drafted V rows must not meet the zero
// weights of rows that do not see them: they are taken out of the operand and
// added, by value, to the rows that do.  Rare, so plain and slow; the sums go
// through this wavefront's LDS rows so that no register array is indexed.
template <uint32_t T, int HD, int M>
__device__ __forceinline__ void tree_odd_rows(const TreeArgs& a, const float (&p)[M][8], const uint32_t (&see)[M],
                                              uint64_t p0, uint64_t total, uint32_t head, uint32_t c, uint32_t g,
                                              float* lds, f32x4 (&o)[M][TreeDims<HD>::TILES]) {
  using D = TreeDims<HD>;
  const uint32_t np = (uint32_t)min((uint64_t)TREE_KEYS, total - p0);
  float* const mine = lds + c * (HD + 4);
#pragma unroll
  for (int m = 0; m < M; ++m) {
#pragma unroll 1
    for (uint32_t d = g; d < (uint32_t)HD; d += 4u) mine[d] = 0.f;
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
      for (uint32_t d = g; d < (uint32_t)HD; d += 4u) {
        const float x = kv_value(a.cache.v, a.cache, p0 + k, head * HD + d);
        if (sees && !(fabsf(x) <= 3.402823466e38f)) mine[d] += w * x;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int d = 0; d < D::TILES; ++d)
#pragma unroll
      for (uint32_t v = 0; v < 4; ++v) o[m][d][v] += mine[D::dim(d, 4u * g + v)];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// O^T += V^T P^T
template <uint32_t T, int HD, int M>
__device__ __forceinline__ void tree_weigh(const TreeArgs& a, const TreeTile<T, HD>& x, const float (&p)[M][8],
                                           const uint32_t (&see)[M], bool drafts, uint64_t p0, uint64_t total,
                                           uint32_t head, uint32_t c, uint32_t g, float* lds,
                                           f32x4 (&o)[M][TreeDims<HD>::TILES]) {
  using D = TreeDims<HD>;
  bool odd = false;
  if constexpr (T == T_F32) {
#pragma unroll
    for (int d = 0; d < D::TILES; ++d)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float v = __uint_as_float(x.v[j][d]);
        if (drafts && !(fabsf(v) <= 3.402823466e38f)) {
          odd = true;
          v = 0.f;
        }
#pragma unroll
        for (int m = 0; m < M; ++m) o[m][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p[m][j], o[m][d], 0, 0, 0);
      }
  } else {
    half8_t ph[M], pl[M];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ph[m][j] = (_Float16)p[m][j];
        pl[m][j] = (_Float16)(p[m][j] - (float)ph[m][j]);
      }
    tree_tiles<T, HD, M, 0>(x, ph, pl, drafts, odd, o);
  }
  if (drafts && __any(odd)) tree_odd_rows<T, HD, M>(a, p, see, p0, total, head, c, g, lds, o);
}

template <uint32_t T, int HD, int M>
__global__ __launch_bounds__(64 * TREE_WAVES) void tree_mfma(TreeArgs a, uint32_t row_blocks) {
  using D = TreeDims<HD>;
  using Tile = TreeTile<T, HD>;
  constexpr bool F32 = T == T_F32;
  constexpr uint32_t OP = HD + 4;  // LDS row of an output tile
  __shared__ float so[TREE_WAVES][16 * OP];
  __shared__ float sm[TREE_WAVES][M * 16], sl[TREE_WAVES][M * 16];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, c = lane & 15u, g = lane >> 4;
  const uint32_t split = blockIdx.x, head = blockIdx.y / row_blocks, row0 = blockIdx.y % row_blocks * (M * 16u);
  const uint32_t G = a.qh / a.cache.kvh, rows = a.n * G, words = (a.n + 63u) / 64u;
  uint64_t hist, total;
  tree_range(a, hist, total);
  const uint64_t tiles = (total + TREE_KEYS - 1u) / TREE_KEYS, per = (tiles + a.nsplit - 1u) / a.nsplit;
  const uint64_t t0 = split * per, t1 = min(tiles, t0 + per);

  // this lane's rows
  uint32_t tok[M];
  const float* qp[M];
  float scale[M];  // score = scale * S, in powers of two
  half8_t qh[M][D::STEPS], ql[M][D::STEPS];
  float qf[M][F32 ? HD / 4 : 1];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const uint32_t r = min(row0 + 16u * m + c, rows - 1u);
    tok[m] = r / G;
    qp[m] = a.q + (uint64_t)tok[m] * a.q_stride + ((uint64_t)head * G + r % G) * HD + g * (HD / 4);
    float x[HD / 4], top = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) {
      x[i] = qp[m][i];
      top = fmaxf(top, fabsf(x[i]));
    }
    float up = 1.f;
    scale[m] = 1.44269504088896340736f / sqrtf((float)HD);
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < HD / 4; ++i) qf[m][i] = x[i];
    } else {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      if (top > 0x1p-100f && top <= 3.402823466e38f) {  // to 2^10 .. 2^11
        const uint32_t e = __float_as_uint(top) >> 23;  // biased
        up = __uint_as_float((264u - e) << 23);         // 2^(10 - (e - 127))
        scale[m] *= __uint_as_float((e - 10u) << 23);
      }
#pragma unroll
      for (int s = 0; s < D::STEPS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = x[8 * s + Tile::order(i)] * up;
          qh[m][s][i] = (_Float16)y;
          ql[m][s][i] = (_Float16)(y - (float)qh[m][s][i]);
        }
    }
  }

  f32x4 o[M][D::TILES];
  float ref[M], l[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    ref[m] = TREE_FLOOR;
    l[m] = 0.f;
#pragma unroll
    for (int d = 0; d < D::TILES; ++d) o[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const uint32_t width = a.cache.kvh * HD;
  const uint32_t row = T == T_F32 ? width * 4u : T == T_F16 ? width * 2u : T == T_Q8_0 ? width : width / 2u, srow = width / 16u;
  const uint64_t sbase = a.cache.cap * (uint64_t)row;
  auto fetch = [&](Tile& x, uint64_t tile) {
    const uint64_t p = tile * TREE_KEYS;
    const uint32_t np = (uint32_t)min((uint64_t)TREE_KEYS, total - p);
    x.load(tree_rsrc(a.cache.k + p * row, np * row), tree_rsrc(a.cache.k + sbase + p * srow, np * srow),
           tree_rsrc(a.cache.v + p * row, np * row), tree_rsrc(a.cache.v + sbase + p * srow, np * srow), row, srow,
           head, c, g);
  };
  // A tile ahead of the one at work; the f32 cache's long rows leave no registers for two.
  constexpr bool AHEAD = !(F32 && HD >= 128);
  Tile cur, nxt;
  uint64_t tile = t0 + wave;
  if (AHEAD && tile < t1) fetch(cur, tile);
  for (; tile < t1; tile += TREE_WAVES) {
    if (!AHEAD) fetch(cur, tile);
    else if (tile + TREE_WAVES < t1) fetch(nxt, tile + TREE_WAVES);
    __builtin_amdgcn_sched_barrier(0);
    const uint64_t p0 = tile * TREE_KEYS;
    // scores of row c at positions p0 + 16 t + 4 g + v
    f32x4 s[M][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int m = 0; m < M; ++m) s[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < HD / 4; ++i)
#pragma unroll
          for (int m = 0; m < M; ++m)
            s[m][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(cur.k[t][i]), qf[m][i], s[m][t], 0, 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < D::STEPS; ++i) {
          const half8_t kf = cur.kfrag(t, i);
#pragma unroll
          for (int m = 0; m < M; ++m) {
            s[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[m][i], s[m][t], 0, 0, 0);
            s[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[m][i], s[m][t], 0, 0, 0);
          }
        }
      }
    }
    const bool drafts = p0 + TREE_KEYS > hist;  // uniform
    float p[M][8];
    uint32_t see[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
      see[m] = 0xFFu;
      if (drafts) {
        // bits g of each half: position p0 + 16 t + 4 g + v in place 4 t + v
        const uint32_t w = tree_window(a, words, tok[m], (int64_t)(p0 - hist), (uint32_t)(total - hist)) >> 4u * g;
        see[m] = (w & 15u) | (w >> 12 & 0xF0u);
      }
      float x[8], top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = s[m][j / 4][j % 4] * scale[m];
        if (drafts && !(see[m] >> j & 1u)) x[j] = -INFINITY;
        top = fmaxf(top, x[j]);
      }
      // The reference stays until a weight would pass 2^15: few tiles rescale.
      if (__any(top > ref[m] + TREE_MOST)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float now = fmaxf(ref[m], top - TREE_BELOW), al = exp2f(ref[m] - now);
        ref[m] = now;
        l[m] *= al;
#pragma unroll
        for (int d = 0; d < D::TILES; ++d)
#pragma unroll
          for (int v = 0; v < 4; ++v) o[m][d][v] *= al;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) p[m][j] = __builtin_amdgcn_exp2f(x[j] - ref[m]);
      l[m] += ((p[m][0] + p[m][1]) + (p[m][2] + p[m][3])) + ((p[m][4] + p[m][5]) + (p[m][6] + p[m][7]));
    }
    tree_weigh<T, HD, M>(a, cur, p, see, drafts, p0, total, head, c, g, so[wave], o);
    if (AHEAD) cur = nxt;
  }

  // join the wavefronts, a row tile at a time
#pragma unroll
  for (int m = 0; m < M; ++m) {
    l[m] += __shfl_xor(l[m], 16);
    l[m] += __shfl_xor(l[m], 32);
    if (g == 0) {
      sm[wave][16 * m + c] = ref[m];
      sl[wave][16 * m + c] = l[m];
    }
  }
#pragma unroll
  for (int m = 0; m < M; ++m) {
    __syncthreads();
    float top = TREE_FLOOR;
#pragma unroll
    for (uint32_t w = 0; w < TREE_WAVES; ++w) top = fmaxf(top, sm[w][16 * m + c]);
    const float al = exp2f(ref[m] - top);
#pragma unroll
    for (int d = 0; d < D::TILES; ++d)
#pragma unroll
      for (uint32_t v = 0; v < 4; ++v) so[wave][c * OP + D::dim(d, 4u * g + v)] = o[m][d][v] * al;
    __syncthreads();
    for (uint32_t e = tid; e < 16u * HD / 4u; e += 64u * TREE_WAVES) {
      const uint32_t rr = e / (HD / 4u), d = e % (HD / 4u) * 4u, r = row0 + 16u * m + rr;
      if (r >= rows) continue;
      float best = TREE_FLOOR, sum = 0.f;
#pragma unroll
      for (uint32_t w = 0; w < TREE_WAVES; ++w) best = fmaxf(best, sm[w][16 * m + rr]);
#pragma unroll
      for (uint32_t w = 0; w < TREE_WAVES; ++w) sum += sl[w][16 * m + rr] * exp2f(sm[w][16 * m + rr] - best);
      float4 y = *reinterpret_cast<const float4*>(&so[0][rr * OP + d]);
#pragma unroll
      for (uint32_t w = 1; w < TREE_WAVES; ++w) {
        const float4 z = *reinterpret_cast<const float4*>(&so[w][rr * OP + d]);
        y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
      }
      const uint32_t i = r / G, h = head * G + r % G;
      if (a.nsplit == 1) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        float* const out = a.out + (uint64_t)i * a.out_stride + (uint64_t)h * HD + d;
        out[0] = y.x * inv; out[1] = y.y * inv; out[2] = y.z * inv; out[3] = y.w * inv;
      } else {
        float* const rec = a.ws + (((uint64_t)split * a.n + i) * a.qh + h) * (HD + 4);
        *reinterpret_cast<float4*>(rec + d) = y;
        if (d == 0) { rec[HD] = best; rec[HD + 1] = sum; }
      }
    }
  }
}

// Joins a row's records: HD / 4 lanes of 4 dims per row.
template <int HD>
__global__ __launch_bounds__(256) void tree_join(TreeArgs a) {
  constexpr uint32_t LANES = HD / 4, PER = 256u / LANES;
  const uint64_t rows = (uint64_t)a.n * a.qh, r = (uint64_t)blockIdx.x * PER + threadIdx.x / LANES;
  const uint32_t d = threadIdx.x % LANES * 4u;
  if (threadIdx.x >= LANES * PER || r >= rows) return;
  const float* const rec = a.ws + r * (HD + 4);
  const uint64_t step = rows * (HD + 4);
  float top = TREE_FLOOR;
  for (uint32_t s = 0; s < a.nsplit; ++s) top = fmaxf(top, rec[s * step + HD]);
  float sum = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (uint32_t s = 0; s < a.nsplit; ++s) {
    const float w = exp2f(rec[s * step + HD] - top);
    sum = fmaf(rec[s * step + HD + 1], w, sum);
    const float4 z = *reinterpret_cast<const float4*>(rec + s * step + d);
    y[0] = fmaf(z.x, w, y[0]); y[1] = fmaf(z.y, w, y[1]); y[2] = fmaf(z.z, w, y[2]); y[3] = fmaf(z.w, w, y[3]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  float* const out = a.out + r / a.qh * a.out_stride + r % a.qh * HD + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = y[e] * inv;
}

// ---------------------------------------------------------------- launches

static bool tree_on_matrix_cores(uint32_t hd) { return hd == 64 || hd == 96 || hd == 128 || hd == 256; }

// Row tiles of a wavefront: a decoded tile serves more rows with two.  With
// head_dim 256 the second tile's registers do not fit.
static uint32_t tree_row_tiles(uint64_t rows, uint32_t hd) { return rows > 16 && hd <= 128 ? 2 : 1; }

uint32_t tree_splits(uint64_t total, uint32_t n, uint32_t qh, uint32_t kvh, uint32_t hd, uint32_t) {
  if (!tree_on_matrix_cores(hd)) return 1;
  const uint64_t rows = (uint64_t)n * (qh / kvh), per = 16u * tree_row_tiles(rows, hd);
  const uint64_t units = kvh * ((rows + per - 1) / per), tiles = (total + TREE_KEYS - 1) / TREE_KEYS;
  const uint64_t want = (512 + units - 1) / units, most = (tiles + TREE_WAVES - 1) / TREE_WAVES;
  const uint64_t s = want < most ? want : most;
  return (uint32_t)(s ? s : 1);
}
uint64_t tree_ws_floats(uint32_t nsplit, uint32_t n, uint32_t qh, uint32_t hd) {
  return nsplit > 1 ? (uint64_t)nsplit * n * qh * (hd + 4) : 0;
}

template <uint32_t T, int HD, int M>
static void launch_tree(const TreeArgs& a, hipStream_t st) {
  const uint64_t rows = (uint64_t)a.n * (a.qh / a.cache.kvh);
  const uint32_t blocks = (uint32_t)((rows + 16 * M - 1) / (16 * M));
  RF_KLAUNCH((tree_mfma<T, HD, M>), dim3(a.nsplit, a.cache.kvh * blocks), dim3(64 * TREE_WAVES), 0, st, a, blocks);
  if (a.nsplit > 1) {
    const uint64_t all = (uint64_t)a.n * a.qh;
    constexpr uint32_t PER = 256 / (HD / 4);
    RF_KLAUNCH(tree_join<HD>, dim3((uint32_t)((all + PER - 1) / PER)), dim3(256), 0, st, a);
  }
}

template <uint32_t T>
static void launch_tree_type(const TreeArgs& a, hipStream_t st) {
  const bool two = tree_row_tiles((uint64_t)a.n * (a.qh / a.cache.kvh), a.cache.hd) == 2;
  switch (a.cache.hd) {
    case 64: two ? launch_tree<T, 64, 2>(a, st) : launch_tree<T, 64, 1>(a, st); break;
    case 96: two ? launch_tree<T, 96, 2>(a, st) : launch_tree<T, 96, 1>(a, st); break;
    case 128: two ? launch_tree<T, 128, 2>(a, st) : launch_tree<T, 128, 1>(a, st); break;
    default: launch_tree<T, 256, 1>(a, st);
  }
}

hipError_t launch_attention_tree(const TreeArgs& a, hipStream_t st) {
  if (!tree_on_matrix_cores(a.cache.hd)) {
    RF_KLAUNCH(tree_plain, dim3(a.n, a.qh), dim3(256), 0, st, a);
  } else {
    switch (a.cache.type) {
      case T_F32: launch_tree_type<T_F32>(a, st); break;
      case T_F16: launch_tree_type<T_F16>(a, st); break;
      case T_Q8_0: launch_tree_type<T_Q8_0>(a, st); break;
      default: launch_tree_type<T_Q4_0>(a, st);
    }
  }
  return hipGetLastError();
}

hipError_t load_module_tree() {
  hipFuncAttributes fa;
  return hipFuncGetAttributes(&fa, reinterpret_cast<const void*>(&tree_plain));
}

}  // namespace rf
