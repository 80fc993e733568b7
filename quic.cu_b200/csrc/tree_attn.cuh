// What the two kernels of the tree attention and their merge share: the call's
// arguments, the place of a position in the blocks, a request's part of the batch and its split into CTAs.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace quic {

struct TreeArgs {
  const void* q;                     // [rows][heads][dim] by strides, in elements
  const void *k, *v;                 // [n_blocks][kv heads][block][dim] by strides, in elements
  void* out;                         // [rows][heads][dim]
  int64_t q_row, q_head, k_block, k_head, k_tok, v_block, v_head, v_tok, table_row, mask_row;
  const int32_t *tables, *lengths, *row_start;
  const uint32_t* mask;              // [rows][mask_words] by mask_row, or nullptr: node i sees nodes 0 .. i
  float4* part_o;                    // partial results [parts][dim / 4][tile_rows]
  float2* part_ml;                   // [parts][tile_rows]: maximum (base 2), sum
  int64_t* first;                    // tcgen05 form: key tiles (with gaps) of the requests before each and of all, then a CTA's share
  FastDiv block, group;              // tokens per block, query heads per KV head
  int32_t rows, requests, heads, kv_heads, n_blocks, max_blocks, mask_words, max_new;
  int32_t tiles, tile_rows;          // row tiles of a request and KV head at most, rows of one
  int32_t splits, chunk;             // mma.sync form: CTAs per request, KV head and row tile at most; the tokens of one at least
  int32_t line_gap;                  // tcgen05 form: key tiles' worth of time that a segment costs
  int32_t cluster;                   // mma.sync form: these CTAs are a cluster and merge their results themselves
  float scale_log2;
};

// A request's rows [start, start + n), its cached tokens before them and the end of its keys, all within the tensors
// whatever the tables hold.
struct TreeRequest {
  int start, n, len, end;
};
__device__ __forceinline__ TreeRequest tree_request(const TreeArgs& a, int b) {
  TreeRequest r;
  const int s = a.row_start[b], e = a.row_start[b + 1];
  r.start = min(max(s, 0), a.rows);
  r.n = max(min(e, a.rows) - r.start, 0);
  const int64_t room = (int64_t)a.max_blocks * a.block.d;
  r.len = (int)min((int64_t)max(a.lengths[b], 0), room);
  r.end = (int)min((int64_t)r.len + r.n, room);
  return r;
}
// mma.sync form: how many CTAs share a request's keys, and the keys of each: equal parts, whole tiles of 64.
__device__ __forceinline__ int tree_parts(const TreeArgs& a, int end, int& per) {
  const int parts = max(1, min(a.splits, (end + a.chunk - 1) / a.chunk));
  per = ((end + parts - 1) / parts + 63) & ~63;
  return per > 0 ? (end + per - 1) / per : 1;
}

// ... and the first part of a row tile in the partial results.
__device__ __forceinline__ int64_t tree_part(const TreeArgs& a, int b, int kvh, int tile) {
  return (((int64_t)b * a.kv_heads + kvh) * a.tiles + tile) * a.splits;
}

// tcgen05 form: the work is a line of key tiles (64 keys of one row tile), request after request, KV head after KV head, row
// tile after row tile; every CTA has an equal share of the line.  A row tile's tiles that one CTA has are a segment.  Behind each row
// tile's last tile lie some (line_gap) that are no work, for the time that the end of a segment and the beginning of the next take.
constexpr int kTreeTcRows = 256, kTreeTcKeys = 64, kTreeTcCtas = 148;
struct TreeUnits {   // of a request
  int rows;          // (node, head) pairs per KV head
  int row_tiles;
  int key_tiles;     // of each row tile; one without keys writes zeros
  int line_tiles;    // ... and the gap
  __device__ __forceinline__ int64_t all(const TreeArgs& a) const { return (int64_t)row_tiles * a.kv_heads * line_tiles; }
};
__device__ __forceinline__ TreeUnits tree_units(const TreeArgs& a, const TreeRequest& r) {
  TreeUnits u;
  u.rows = min(r.n, a.max_new) * (int)a.group.d;
  u.row_tiles = (u.rows + kTreeTcRows - 1) / kTreeTcRows;
  u.key_tiles = max(1, (r.end + kTreeTcKeys - 1) / kTreeTcKeys);
  u.line_tiles = u.key_tiles + a.line_gap;
  return u;
}

// Which of the 32 positions from t on node `node` sees, the positions up to `end` taken for present: bit j for t + j.
__device__ __forceinline__ uint32_t tree_visible32(const TreeArgs& a, const TreeRequest& r, int node, int t) {
  const int first = t - r.len;  // number of the node at position t
  if (first + 32 <= 0) return 0xffffffffu;
  uint32_t seen;
  if (a.mask == nullptr) {
    const int last = node - first;  // the last bit
    seen = last >= 31 ? 0xffffffffu : (last < 0 ? 0u : (2u << last) - 1u);
    return first < 0 ? seen | ((1u << -first) - 1u) : seen;
  }
  const uint32_t* row = a.mask + (int64_t)(r.start + node) * a.mask_row;
  const int w = first >> 5;  // (rounds down)
  const uint32_t lo = w < 0 ? 0xffffffffu : (w < a.mask_words ? row[w] : 0u);
  const uint32_t hi = w + 1 < a.mask_words ? row[w + 1] : 0u;
  return __funnelshift_r(lo, hi, first & 31);
}

__device__ __forceinline__ float tree_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t pair2(float x, float y) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
__device__ __forceinline__ void unpair2(uint64_t d, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(d)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two values in a word of the tensors' type.
template <typename T>
__device__ __forceinline__ uint32_t tree_pack(float x, float y);
template <>
__device__ __forceinline__ uint32_t tree_pack<half>(float x, float y) {
  const half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t tree_pack<__nv_bfloat16>(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ float2 tree_unpack(uint32_t w);
template <>
__device__ __forceinline__ float2 tree_unpack<half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const half2*>(&w));
}
template <>
__device__ __forceinline__ float2 tree_unpack<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// The exponent of an infinity or NaN, and the sign bits of those of the two values in a word that have it (the sum of exponent and
// fraction reaches the sign then, and never the next value).
template <typename T>
constexpr uint32_t kTreeExponent = 0;
template <>
constexpr uint32_t kTreeExponent<half> = 0x7c00u;
template <>
constexpr uint32_t kTreeExponent<__nv_bfloat16> = 0x7f80u;
template <typename T>
__device__ __forceinline__ uint32_t tree_not_finite(uint32_t w) {
  constexpr uint32_t one = 0x8000u - kTreeExponent<T>;
  return ((w & 0x7fff7fffu) + (one << 16 | one)) & 0x80008000u;
}
template <typename T>
__device__ __forceinline__ bool tree_not_finite(const uint4& w) {
  return (tree_not_finite<T>(w.x) | tree_not_finite<T>(w.y) | tree_not_finite<T>(w.z) | tree_not_finite<T>(w.w)) != 0u;
}
// The word with what is not finite replaced by zero.
template <typename T>
__device__ __forceinline__ uint32_t tree_finite(uint32_t w) {
  return w & ~((tree_not_finite<T>(w) >> 15) * 0xffffu);
}

// The reference point of a row's exponentials moves only when its maximum has grown by more than 2^8: P and the sums stay far within
// their types' ranges.
constexpr float kTreeGrowth = 8.f;
// P = 2^(score - reference + shift), the scores to base 2: fp16 weights reach 2^15 and stay normal down to 2^-21 of the reference.  bf16
// has fp32's range.
template <typename T>
constexpr float kTreeShift = 0.f;
template <>
constexpr float kTreeShift<half> = 7.f;

// The throughput form (tree_attn_tc.cu) takes what TMA can fetch.
bool tree_attn_tc_takes(int block_size, int64_t k_block, int64_t k_head, int64_t k_tok, int64_t v_block, int64_t v_head, int64_t v_tok);
int tree_attn_tc_launch(const TreeArgs& a, bool bf16, int dim, cudaStream_t stream);

}  // namespace quic
