// rf_kv.h — K/V cache in few bits: layout and launchers (internal).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rf {

// Layer caches are K and V buffers of [cap][kvh][hd] values.  F32 and F16 hold
// them as they are.  Q8_0 and Q4_0 hold codes [cap][kvh * hd] and, behind them,
// one f16 scale per 32 values [cap][kvh * hd / 32]:
//   Q8_0: a byte per value, code + 128, code in -127..127.  The scale is the
//         least f16 of at most 3 significant bits with 127 d >= max |x|: a
//         code has at most 7 bits and a sign, so code * d has at most 10
//         significant bits and is an f16 exactly.  The matrix cores then take
//         the cached values themselves, and no scale is left for the scores.
//         (Rounding the scale up costs 11% of a step on average, 25% at most;
//         one scale per 128 values would cost 28%.)
//   Q4_0: two values per byte (the even one low), code + 8, code in -8..7.
//         |d| is the least f16 of at most 8 significant bits with
//         8 |d| >= max |x| (3 bits of code and 8 of scale: exact in f16), its
//         sign such that the extreme value's code is -8.
// Codes are the nearest to x / d, ties to even.  A block that holds an
// infinity or NaN has scale NaN and reads back as NaN.  Magnitudes above
// 127 * 512 (Q8_0) or 8 * 8160 (Q4_0) are cut there.
struct KvView {
  uint8_t *k, *v;
  const uint32_t* length;  // device word added to every position of a call, or null
  uint64_t cap;
  uint32_t type, kvh, hd;
};

constexpr uint32_t KV_MOVE_MAX = 1024;   // rows of one move
constexpr uint32_t KV_MOVE_CACHES = 64;  // caches of one launch (pointers are kernel arguments)
constexpr uint32_t TREE_MAX_NODES = 1024;
constexpr uint32_t KV_MAX_HEAD_DIM = 512;
// Values of a position, and rows (tokens times query heads) of a KV head: grids
// and byte offsets within a tile stay inside 32 bits, grid y inside 16.
constexpr uint32_t KV_MAX_WIDTH = 1u << 20, TREE_MAX_ROWS = 65535u * 16u;

inline uint64_t kv_code_bytes(uint32_t type, uint64_t values) {
  return type == 0u ? values * 4 : type == 1u ? values * 2 : type == 8u ? values : values / 2;
}
inline uint64_t kv_row_bytes(uint32_t type, uint64_t values) {
  return kv_code_bytes(type, values) + (type >= 2u ? values / 16 : 0);
}

struct QkRopeArgs {
  const float *q, *k, *v;  // v: null without a cache
  uint64_t q_stride, k_stride, v_stride;
  const float *q_norm, *k_norm;
  float eps;
  const uint32_t* positions;  // null: the row's own position in the cache
  uint64_t n;
  uint32_t qh, kvh, hd;
  double log2_theta;
  float *q_out, *k_out;
  uint64_t q_out_stride, k_out_stride;
  KvView cache;  // k null: none
  uint64_t first;
};

hipError_t launch_qk_norm_rope(const QkRopeArgs& a, hipStream_t st);
hipError_t launch_kv_store(const KvView& c, const float* k, uint64_t k_stride, const float* v, uint64_t v_stride,
                           uint64_t first, uint64_t n, hipStream_t st);
hipError_t launch_kv_load(const KvView& c, uint64_t first, uint64_t n, float* k, uint64_t k_stride, float* v,
                          uint64_t v_stride, hipStream_t st);
// All caches share type, kvh, hd; length is caches[0]'s.
hipError_t launch_kv_move(const KvView* caches, uint32_t n_caches, const uint32_t* src, uint64_t first, uint32_t n,
                          hipStream_t st);
hipError_t launch_tree_mask(const int32_t* parents, uint32_t n, uint32_t base, const uint32_t* length, uint64_t* mask,
                            uint32_t* positions, hipStream_t st);

struct TreeArgs {
  const float* q;  // [n][q_stride]
  uint64_t q_stride;
  float* out;
  uint64_t out_stride;
  KvView cache;
  const uint64_t* mask;  // [n][ceil(n / 64)] or null: token i sees drafts 0..i
  uint64_t hist, total;  // keys before the drafts, and in all (with a length word: at most, nsplit is chosen for it)
  uint32_t n, qh;
  uint32_t nsplit;  // position splits; > 1: records in ws
  uint32_t q_vec;   // q rows are 16-byte aligned
  float* ws;
  // what a kernel would otherwise work out before its first load (launch_attention_tree)
  uint32_t group, rows, words;        // query heads and rows of a KV head, words of a mask row
  uint32_t code_row, scale_row;       // bytes of a position
  uint64_t scale_base;                // of the scales, from the codes
  uint32_t tiles, per;                // tiles of 32 positions in all and of a split, without a length word
};
// Splits of a call over `total` positions, and the workspace floats they need.
uint32_t tree_splits(uint64_t total, uint32_t n, uint32_t qh, uint32_t kvh, uint32_t hd, uint32_t type);
uint64_t tree_ws_floats(uint32_t nsplit, uint32_t n, uint32_t qh, uint32_t hd);
hipError_t launch_attention_tree(const TreeArgs& a, hipStream_t st);
// Workspace floats of every call of up to `total` positions and n tokens.
uint64_t tree_ws_floats_upto(uint64_t total, uint32_t n, uint32_t qh, uint32_t kvh, uint32_t hd, uint32_t type);
hipError_t load_module_kv();
hipError_t load_module_tree();

}  // namespace rf
