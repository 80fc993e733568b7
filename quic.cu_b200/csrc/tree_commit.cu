// Keeps the branch of every drafted tree that the target model agrees with.
//
// path[0] = 0; path[j + 1] is the first child of path[j] whose token is the target's choice at path[j]; the walk ends where
// there is none.  Parents lie before their children, so paths ascend and path[j] >= j: the rows of K and V that move, from
// position len + path[j] to len + j, do so towards the front, and taken in ascending j no row is overwritten before it has
// been read (a later row's source lies behind every earlier row's target).
//
// A CTA walks the tree of one request (one warp, 32 nodes a look, from shared memory) and moves the path in eight of its
// (layer, K or V, KV head) planes at a time, a warp each, 16 bytes a lane, up to four loads in flight before the first store.
// The walk is repeated by every CTA of a request: it costs less than a second launch.  Bound: the latency of a launch, two
// rounds of loads and the walk; the bytes of a step are few.
#include "common.cuh"

namespace quic {
namespace {

constexpr int kThreads = 256, kMostNodes = 1024;

__global__ void __launch_bounds__(kThreads) tree_commit_kernel(const quic_tree_commit_t t) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.y;
  int64_t* const token_s = reinterpret_cast<int64_t*>(smem);  // later: where a row moves from
  int64_t* const target_s = token_s + t.max_new;              // later: where it moves to
  int32_t* const parent_s = reinterpret_cast<int32_t*>(target_s + t.max_new);
  int32_t* const path_s = parent_s + t.max_new;
  __shared__ int accepted_s;
  pdl_launch_dependents();
  pdl_wait();
  const int start = min(max(t.row_start[b], 0), t.rows), end = min(t.row_start[b + 1], t.rows);
  const int len = t.lengths[b];
  int n = end - start;
  if (n < 0 || n > t.max_new) n = 0;
  auto read = [&](const void* p, int i) {
    return t.token_bytes == 8 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
  };
  for (int i = tid; i < n; i += kThreads) {
    parent_s[i] = t.parents[start + i];
    token_s[i] = read(t.tokens, start + i);
    target_s[i] = read(t.targets, start + i);
  }
  __syncthreads();
  if (warp == 0) {
    int count = 0, at = 0;
    while (n > 0) {
      if (lane == 0) path_s[count] = at;
      ++count;
      const int64_t want = target_s[at];
      int next = -1;
      for (int i0 = (at + 1) & ~31; i0 < n; i0 += 32) {  // (a parent lies before its children)
        const int i = i0 + lane;
        const uint32_t hit = __ballot_sync(0xffffffffu, i > at && i < n && parent_s[i] == at && token_s[i] == want);
        if (hit) {
          next = i0 + __ffs(hit) - 1;
          break;
        }
      }
      if (next < 0) break;
      at = next;
    }
    __syncwarp();
    if (blockIdx.x == 0) {
      for (int j = lane; j < t.max_new; j += 32) t.path[(int64_t)b * t.max_new + j] = j < count ? path_s[j] : -1;
      if (lane == 0) {
        const int64_t next = n > 0 ? target_s[at] : -1;
        if (t.token_bytes == 8) reinterpret_cast<int64_t*>(t.next_token)[b] = next;
        else reinterpret_cast<int32_t*>(t.next_token)[b] = (int32_t)next;
        t.accepted[b] = count;
        t.new_lengths[b] = len + count;
      }
    }
    if (lane == 0) accepted_s = count;
  }
  __syncthreads();
  const int accepted = accepted_s;

  // ---- the rows that move: a suffix of the path
  auto place = [&](int node) {
    const int64_t p = (int64_t)len + node;
    const int64_t j = p / t.block_size;
    if (p < 0 || j >= t.max_blocks) return (int64_t)-1;
    const int id = t.tables[(int64_t)b * t.table_row + j];
    return id < 0 || id >= t.n_blocks ? (int64_t)-1 : id * t.kv_block + (p - j * t.block_size) * t.kv_tok;
  };
  int stay = 0;
  while (stay < accepted && path_s[stay] == stay) ++stay;
  const int moves = accepted - stay;
  if (moves == 0) return;
  for (int j = tid; j < moves; j += kThreads) {
    const int64_t from = place(path_s[stay + j]), to = place(stay + j);
    token_s[j] = from < 0 || to < 0 ? -1 : from;
    target_s[j] = to;
  }
  __syncthreads();
  const int pieces = t.dim / 8, planes = t.layers * 2 * t.kv_heads;
  for (int plane = blockIdx.x * (kThreads / 32) + warp; plane < planes; plane += gridDim.x * (kThreads / 32)) {
    const int head = plane % t.kv_heads, kind = plane / t.kv_heads & 1, layer = plane / t.kv_heads >> 1;
    uint16_t* const kv = reinterpret_cast<uint16_t*>(t.kv) + layer * t.kv_layer + kind * t.kv_kind + head * t.kv_head;
    for (int i0 = 0; i0 < moves * pieces; i0 += 128) {
      uint4 v[4];
      int64_t to[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + 32 * u + lane, row = i / pieces, piece = i - row * pieces;
        to[u] = -1;
        if (i < moves * pieces && token_s[row] >= 0) {
          to[u] = target_s[row] + 8 * piece;
          v[u] = *reinterpret_cast<const uint4*>(kv + token_s[row] + 8 * piece);
        }
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (to[u] >= 0) *reinterpret_cast<uint4*>(kv + to[u]) = v[u];
      __syncwarp();
    }
  }
}

}  // namespace
}  // namespace quic

using namespace quic;

extern "C" int quic_tree_commit(const quic_tree_commit_t* t, void* stream) {
  QUIC_REQUIRE(t != nullptr, QUIC_E_ARG, "tree_commit: null arguments");
  QUIC_REQUIRE(t->token_bytes == 4 || t->token_bytes == 8, QUIC_E_SHAPE, "tree_commit: tokens are int32 or int64");
  QUIC_REQUIRE(t->layers >= 1 && t->n_blocks >= 1 && t->kv_heads >= 1 && t->block_size >= 1 && t->max_blocks >= 1 && t->dim >= 8 &&
                   t->dim % 8 == 0 && (int64_t)t->layers * 2 * t->kv_heads < (1 << 24) && t->dim <= 4096,
               QUIC_E_SHAPE, "tree_commit: bad cache geometry");
  QUIC_REQUIRE(t->rows >= 0 && t->requests >= 0, QUIC_E_SHAPE, "tree_commit: bad row or request count");
  QUIC_REQUIRE(t->max_new >= 1 && t->max_new <= kMostNodes && t->requests <= 65535, QUIC_E_LIMIT,
               "tree_commit: at most 1024 rows of a request and 65535 requests");
  if (t->requests == 0) return QUIC_OK;
  QUIC_REQUIRE(t->kv && t->tables && t->lengths && t->row_start && t->path && t->accepted && t->next_token && t->new_lengths &&
                   (t->rows == 0 || (t->parents && t->tokens && t->targets)),
               QUIC_E_ARG, "tree_commit: null tensor");
  QUIC_REQUIRE(t->new_lengths != t->lengths, QUIC_E_ARG, "tree_commit: new_lengths must not be lengths");
  QUIC_REQUIRE((uintptr_t)t->kv % 16 == 0 && ((t->kv_layer | t->kv_kind | t->kv_block | t->kv_head | t->kv_tok) & 7) == 0, QUIC_E_ARG,
               "tree_commit: the cache must be 16-byte aligned, its strides multiples of 8 elements");
  const int64_t planes = (int64_t)t->layers * 2 * t->kv_heads;
  const int64_t ctas = (planes + kThreads / 32 - 1) / (kThreads / 32);
  QUIC_CUDA(launch(tree_commit_kernel, dim3((unsigned)(ctas > 256 ? 256 : ctas), t->requests), dim3(kThreads), (size_t)t->max_new * 24,
                   (cudaStream_t)stream, true, *t));
  return QUIC_OK;
}
