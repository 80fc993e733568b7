// Attention of drafted trees over a blocked KV cache.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i . k_j)
//
// for node i of a request's tree over the request's cached positions 0 .. len - 1 and those of the nodes (position
// len + a for node a) that it sees: its ancestors and itself by bit mask, or without masks nodes 0 .. i.  A chain, the next
// chunk of a prompt and a single decode token are trees too.  The R = nodes x (query heads per KV head) rows of a
// request and KV head share their keys; K and V are read once per tile of those rows.  (A tile walks the keys to the end of its
// request, those behind its last node as well: a prompt's chunk without cached tokens costs twice what it must.)
//
// This file: the form for few rows (mma.sync), the merge of many parts of a request, and the entry point; tree_attn_tc.cu has the form
// for more rows.
// A CTA has 16 or 32 rows and a part of the keys, which its four warps walk 32 (16 of 128 dims) at a time, each through a ring of
// its own (cp.async, no barrier between warps), one pass with a running maximum and sum per row; the warps' results meet in
// shared memory at the end, those of up to eight CTAs as well, which are a cluster then and each sum a share of the rows' dims (over
// distributed shared memory), those of more CTAs in the merge kernel.  Bound: the bytes of K and V (16 x 1 x 8192, fp16, 14:2 heads
// of 64: 16.7 us, 4.0 TB/s; 9 x 13 x 7247..14495, 8:8 heads: 40.6 us, 4.9 TB/s); with 32 rows what a warp's steps wait for of their own
// results, two warps a scheduler (64 x 8 x 200..1500: 18.8 us); for small calls the launch and what depends
// on one another: lengths, table, keys, results (1 x 1 x 300: 5.0 us).  Moving the reference point for every larger maximum, sums of
// the rounded weights and separate exponents cost 64 x 8 x 200..1500 25.5 instead of 22.2 us; places of keys computed by the
// lane of the key, and the masks of the rows kept in shared memory, cost more than they saved (+0.2 to +1 us).
#include <math.h>

#include <type_traits>

#include "tree_attn.cuh"

namespace quic {
namespace {

constexpr int kWarps = 4, kMostCluster = 8, kByRowsTile = 32 * kWarps;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {  // zeros beyond `bytes`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
// d += a b (kFirst: d = a b)
template <typename T, bool kFirst = false>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (kFirst) d[0] = d[1] = d[2] = d[3] = 0.f;
  if constexpr (kTreeExponent<T> == kTreeExponent<half>)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Keys of a warp's tile (8 KB of K and V) and tiles of its ring: two CTAs an SM with two tiles a warp under way.  With tiles of 32
// keys for 128 dims too, one CTA fitted an SM: 48 requests x 2 nodes x 11707 tokens, 16:1 heads, 65 -> 85 us; with rings of two
// tiles 16 x 1 x 8192, 14:2 heads of 64, 19 -> 21 us, of four (one CTA an SM) 27.  Eight warps a CTA are ahead by 1 us where
// there are fewer row tiles than SMs, and behind by 3 us where there are more.
template <int D>
constexpr int kTileKeys = D == 64 ? 32 : 16;
constexpr int kStages = 3;
constexpr uint32_t kRowsBytes = 32 * 64 * 2;  // K (or V) of a tile
template <int D, int MT>
constexpr uint32_t kSmem = kWarps * kStages * 2 * kRowsBytes > kWarps * MT * 16 * (D + 4) * 4 ? kWarps * kStages * 2 * kRowsBytes
                                                                                              : kWarps * MT * 16 * (D + 4) * 4;

// Tile element (row, 16-byte chunk): chunks swapped by row so that eight rows of a chunk lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t tile_at(int row, int chunk) {
  return row * (D * 2) + ((chunk ^ (row & 7)) << 4);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// What CTA `rank` of the cluster has at this CTA's shared-memory address `at`.
__device__ __forceinline__ uint32_t in_cta(uint32_t at, int rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(rank));
  return remote;
}
__device__ __forceinline__ float2 cluster_ld2(uint32_t at) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float4 cluster_ld4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}

// The result of dims 4 c4 .. of a row of a request and KV head: sum x by 1 / l.
template <typename T, int D>
__device__ __forceinline__ void write_out(const TreeArgs& a, const TreeRequest& r, int kvh, int row, int c4, const float4& x, float l) {
  const int node = (int)a.group.div(row), head = kvh * (int)a.group.d + row - node * (int)a.group.d;
  const float inv = l != 0.f ? 1.f / l : 0.f;  // (NaN stays)
  *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + ((int64_t)(r.start + node) * a.heads + head) * D + 4 * c4) =
      make_uint2(tree_pack<T>(x.x * inv, x.y * inv), tree_pack<T>(x.z * inv, x.w * inv));
}

// kByRows: a warp has rows of its own and all keys, else the rows of the CTA and every fourth tile of the keys.
template <typename T, int D, int MT, bool kByRows>
__global__ void __launch_bounds__(kWarps * 32) tree_attn_kernel(const TreeArgs a) {
  constexpr int kKeys = kTileKeys<D>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint32_t valid_s[kWarps][kStages];
  __shared__ float2 ml_s[MT * 16];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int split = blockIdx.x, kvh = blockIdx.y % a.kv_heads, tile = blockIdx.y / a.kv_heads;
  pdl_wait();
  const TreeRequest r = tree_request(a, blockIdx.z);
  const int all = min(r.n, a.max_new) * (int)a.group.d;  // row = node x group + head of the group
  if (tile * 16 * MT * (kByRows ? kWarps : 1) >= all) return;  // (a cluster as one)
  const int r0 = (kByRows ? tile * kWarps + warp : tile) * 16 * MT;
  int per;
  const int parts = tree_parts(a, r.end, per);
  if (split >= parts && !a.cluster) return;
  const int t_begin = split * per, t_end = kByRows && r0 >= all ? 0 : min(t_begin + per, r.end);
  const int32_t* table = a.tables + (int64_t)blockIdx.z * a.table_row;

  // ---- queries: A fragments of every 16 rows
  uint32_t qf[MT][D / 16][4];
  int node[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = r0 + 16 * m + 8 * h + g;
      node[m][h] = (int)a.group.div(row);
      const int head = kvh * (int)a.group.d + row - node[m][h] * (int)a.group.d;
      const uint32_t* q = reinterpret_cast<const uint32_t*>(reinterpret_cast<const T*>(a.q) + (int64_t)(r.start + node[m][h]) * a.q_row +
                                                            (int64_t)head * a.q_head);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qf[m][ks][h] = row < all ? __ldg(q + 8 * ks + c) : 0u;
        qf[m][ks][2 + h] = row < all ? __ldg(q + 8 * ks + 4 + c) : 0u;
      }
      if (row >= all) node[m][h] = 0;
    }

  // ---- the warp's ring
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * kStages * 2 * kRowsBytes;
  constexpr int kPer = D / 8, kAtOnce = 32 / kPer;  // chunks of a row, rows of one instruction
  constexpr int step = (kByRows ? 1 : kWarps) * kKeys;
  constexpr uint32_t kAllKeys = 0xffffffffu >> (32 - kKeys);
  // the block of position t + lane, or -1 where there is none
  auto fetch = [&](int t) {
    const int p = t + (lane & (kKeys - 1));
    const int id = p < t_end ? __ldg(table + a.block.div(p)) : -1;
    return id < a.n_blocks ? id : -1;
  };
  const T* const k_lane = reinterpret_cast<const T*>(a.k) + kvh * a.k_head + lane % kPer * 8;
  const T* const v_lane = reinterpret_cast<const T*>(a.v) + kvh * a.v_head + lane % kPer * 8;
  const int run = a.max_blocks == 1 || a.block.d % 16 == 0 ? 16 : (a.block.d % 8 == 0 ? 8 : 0);
  auto request = [&](int t, int stage, int id) {
    const uint32_t ok = __ballot_sync(0xffffffffu, id >= 0) & kAllKeys;
    if (lane == 0) valid_s[warp][stage] = ok;
    const uint32_t dst = ring + stage * 2 * kRowsBytes;
    const int chunk = lane % kPer;
    // Keys that lie in one block, one after the other: their place is looked up once (once a row, 64 x 8 x 200..1500 takes 22.2
    // instead of 18.8 us, 9 x 13 x 14495 in blocks of 24, 42.3 instead of 40.6).
    auto runs = [&](auto length) {
      constexpr int kRun = decltype(length)::value;
#pragma unroll
      for (int h = 0; h < kKeys / kRun; ++h) {
        const int64_t at = max(__shfl_sync(0xffffffffu, id, kRun * h), 0);
        const int p = t + kRun * h, off = p - (int)a.block.div(p) * (int)a.block.d + lane / kPer;
        const T* kp = k_lane + at * a.k_block + off * a.k_tok;
        const T* vp = v_lane + at * a.v_block + off * a.v_tok;
#pragma unroll
        for (int i = 0; i < kRun / kAtOnce; ++i) {
          const int row = kRun * h + i * kAtOnce + lane / kPer;
          const uint32_t bytes = ok >> row & 1u ? 16u : 0u, to = dst + tile_at<D>(row, chunk);
          cp_async16(to, kp, bytes);
          cp_async16(to + kRowsBytes, vp, bytes);
          kp += kAtOnce * a.k_tok, vp += kAtOnce * a.v_tok;
        }
      }
    };
    if (run == 16) return runs(std::integral_constant<int, 16>{});
    if (run == 8) return runs(std::integral_constant<int, 8>{});
    const int p = t + (lane & (kKeys - 1)), off = p - (int)a.block.div(p) * (int)a.block.d;
#pragma unroll 1
    for (int i = 0; i < kKeys / kAtOnce; ++i) {
      const int row = i * kAtOnce + lane / kPer;
      const int bid = __shfl_sync(0xffffffffu, id, row), boff = __shfl_sync(0xffffffffu, off, row);
      const int64_t at = max(bid, 0), o = bid >= 0 ? boff : 0;
      const uint32_t bytes = bid >= 0 ? 16u : 0u, to = dst + tile_at<D>(row, chunk);
      cp_async16(to, k_lane + at * a.k_block + o * a.k_tok, bytes);
      cp_async16(to + kRowsBytes, v_lane + at * a.v_block + o * a.v_tok, bytes);
    }
  };

  float o[MT][D / 8][4], m_run[MT][2];  // m_run: the reference point
  uint64_t l_run[MT][2];                // two sums each
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.f;
    m_run[m][0] = m_run[m][1] = -INFINITY;
    l_run[m][0] = l_run[m][1] = 0ull;
  }

  const uint64_t scale2 = pair2(a.scale_log2, a.scale_log2);
  const int t_warp = t_begin + (kByRows ? 0 : warp * kKeys);
  int id = fetch(t_warp);
#pragma unroll(D == 64 && MT == 1 ? kStages - 1 : 1)  // (else code that is read once: 57.9 -> 54.3 us at 48 x 2 x 11707, 16:1 heads of 128)
  for (int s = 0; s < kStages - 1; ++s) {
    if (t_warp + s * step < t_end) request(t_warp + s * step, s, id);
    asm volatile("cp.async.commit_group;" ::: "memory");
    id = fetch(t_warp + (s + 1) * step);
  }
  int stage = 0;
  for (int t = t_warp; t < t_end; t += step) {
    {
      const int ahead = t + (kStages - 1) * step;
      const int to = stage == 0 ? kStages - 1 : stage - 1;
      if (ahead < t_end) request(ahead, to, id);
      asm volatile("cp.async.commit_group;" ::: "memory");
      id = fetch(ahead + step);
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();
    const uint32_t k_at = ring + stage * 2 * kRowsBytes, v_at = k_at + kRowsBytes;
    const uint32_t valid = valid_s[warp][stage];

    // S = Q K^T
    float s[MT][kKeys / 8][4];
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
      for (int n = 0; n < kKeys / 8; ++n) {
        uint32_t b[4];
        ldsm4(b, k_at + tile_at<D>(n * 8 + (lane & 7), kk * 4 + (lane >> 3)));
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if (kk == 0) mma<T, true>(s[m][n], qf[m][2 * kk], b[0], b[1]);
          else mma<T>(s[m][n], qf[m][2 * kk], b[0], b[1]);
          mma<T>(s[m][n], qf[m][2 * kk + 1], b[2], b[3]);
        }
      }

    // what each row sees
    const bool tree = t + kKeys > r.len, masked = tree || valid != kAllKeys;
    uint32_t seen[MT][2];
    if (masked) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          seen[m][h] = valid & tree_visible32(a, r, node[m][h], t);
#pragma unroll
          for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (!(seen[m][h] >> (8 * n + 2 * c + e) & 1u)) s[m][n][2 * h + e] = -INFINITY;
        }
    }

    // reference points: moved when a score is far above (from -inf: by any)
    bool grown = false;
    float top[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = fmaxf(s[m][0][2 * h], s[m][0][2 * h + 1]);
#pragma unroll
        for (int n = 1; n < kKeys / 8; ++n) mx = max3(mx, s[m][n][2 * h], s[m][n][2 * h + 1]);
        top[m][h] = mx * a.scale_log2;  // (the scale is positive)
        grown |= top[m][h] > m_run[m][h] + kTreeGrowth;
      }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = top[m][h];  // of the row: four lanes have eight keys each
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          if (mx > m_run[m][h] + kTreeGrowth) {
            const float alpha = tree_ex2(m_run[m][h] - mx);
            m_run[m][h] = mx;
            float x, y;
            unpair2(l_run[m][h], x, y);
            l_run[m][h] = pair2(x * alpha, y * alpha);
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
              o[m][n][2 * h] *= alpha;
              o[m][n][2 * h + 1] *= alpha;
            }
          }
        }
    }

    // weights and their sums
    uint32_t p[MT][kKeys / 16][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float shifted = kTreeShift<T> - (m_run[m][h] == -INFINITY ? 0.f : m_run[m][h]);
        const uint64_t shifted2 = pair2(shifted, shifted);
#pragma unroll
        for (int n = 0; n < kKeys / 8; ++n) {
          float x, y;
          unpair2(fma2(pair2(s[m][n][2 * h], s[m][n][2 * h + 1]), scale2, shifted2), x, y);
          x = tree_ex2(x);  // 2^-inf = 0 for keys that are not seen
          y = tree_ex2(y);
          p[m][n >> 1][2 * (n & 1) + h] = tree_pack<T>(x, y);
          l_run[m][h] = add2(l_run[m][h], pair2(x, y));
        }
      }

    // A node's infinity or NaN reaches the rows that see the node only: weight zero times it would be NaN in all others.
    if (tree) {
      bool odd = false;
#pragma unroll
      for (int i = 0; i < kKeys / kAtOnce; ++i) {
        const uint4 w = *reinterpret_cast<const uint4*>(smem + (v_at - (uint32_t)__cvta_generic_to_shared(smem)) +
                                                        tile_at<D>(i * kAtOnce + lane / kPer, lane % kPer));
        odd |= tree_not_finite<T>(w);
      }
      if (__any_sync(0xffffffffu, odd)) {
        unsigned char* v_tile = smem + (v_at - (uint32_t)__cvta_generic_to_shared(smem));
        for (int key = 0; key < kKeys; ++key) {
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(v_tile + tile_at<D>(key, n) + 4 * c);
            if (tree_not_finite<T>(w)) {
              const float2 f = tree_unpack<T>(w), z = tree_unpack<T>(tree_finite<T>(w));
#pragma unroll
              for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                  if (seen[m][h] >> key & 1u) {
                    o[m][n][2 * h] += f.x - z.x;  // (x - x = 0 for what is finite)
                    o[m][n][2 * h + 1] += f.y - z.y;
                  }
            }
          }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kKeys / kAtOnce; ++i) {
          uint4* const at = reinterpret_cast<uint4*>(v_tile + tile_at<D>(i * kAtOnce + lane / kPer, lane % kPer));
          uint4 w = *at;
          w.x = tree_finite<T>(w.x), w.y = tree_finite<T>(w.y), w.z = tree_finite<T>(w.z), w.w = tree_finite<T>(w.w);
          *at = w;
        }
        __syncwarp();
      }
    }

    // O += P V
#pragma unroll
    for (int jk = 0; jk < kKeys / 16; ++jk)
#pragma unroll
      for (int cc = 0; cc < D / 16; ++cc) {
        uint32_t b[4];
        ldsm4_t(b, v_at + tile_at<D>(jk * 16 + (lane >> 3 & 1) * 8 + (lane & 7), 2 * cc + (lane >> 4)));
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          mma<T>(o[m][2 * cc], p[m][jk], b[0], b[1]);
          mma<T>(o[m][2 * cc + 1], p[m][jk], b[2], b[3]);
        }
      }
    __syncwarp();  // (the stage is requested anew in the next round)
    stage = stage == kStages - 1 ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  pdl_launch_dependents();

  // ---- the four warps' parts, or rows
  constexpr int kRows = MT * 16, kLine = D + 4;  // a row: D values, maximum, sum
  float* const mine = reinterpret_cast<float*>(smem) + warp * kRows * kLine;
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float* line = mine + (16 * m + 8 * h + g) * kLine;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(line + 8 * n + 2 * c) = make_float2(o[m][n][2 * h], o[m][n][2 * h + 1]);
      float l, l1;
      unpair2(l_run[m][h], l, l1);
      l += l1;
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (c == 0) line[D] = l != l ? INFINITY : m_run[m][h], line[D + 1] = l;  // (a maximum passes over NaN)
    }
  if constexpr (kByRows) {
    __syncwarp();
#pragma unroll 4
    for (int i = lane; i < kRows * (D / 4); i += 32) {
      const int row = i / (D / 4), c4 = i % (D / 4);
      if (r0 + row >= all) break;
      write_out<T, D>(a, r, kvh, r0 + row, c4, *reinterpret_cast<const float4*>(mine + row * kLine + 4 * c4), mine[row * kLine + D + 1]);
    }
    return;
  }
  __syncthreads();
  const int64_t part = tree_part(a, blockIdx.z, kvh, tile) + split;
  for (int i = tid; i < kRows * (D / 4); i += kWarps * 32) {
    const int row = i % kRows, c4 = i / kRows;
    if (r0 + row >= all) continue;
    const float* line = reinterpret_cast<const float*>(smem) + row * kLine;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, line[w * kRows * kLine + D]);
    const float ref = top == -INFINITY ? 0.f : top;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float* at = line + w * kRows * kLine;
      const float f = tree_ex2(at[D] - ref);
      if (f != 0.f) {
        const float4 y = *reinterpret_cast<const float4*>(at + 4 * c4);
        x.x += f * y.x, x.y += f * y.y, x.z += f * y.z, x.w += f * y.w;
        l += f * at[D + 1];
      }
    }
    if (parts == 1) {
      if (split == 0) write_out<T, D>(a, r, kvh, r0 + row, c4, x, l);
    } else if (a.cluster) {  // (in the place of the first warp's part, which nobody else reads)
      *reinterpret_cast<float4*>(smem + ((row * kLine) + 4 * c4) * 4) = x;
      if (c4 == 0) ml_s[row] = make_float2(top, l);
    } else {
      a.part_o[(part * (D / 4) + c4) * a.tile_rows + row] = x;
      if (c4 == 0) a.part_ml[part * a.tile_rows + row] = make_float2(top, l);
    }
  }
  if (!a.cluster || parts == 1) return;

  // ---- the cluster's parts: every CTA sums its share of the rows' dims
  __syncwarp();
  cluster_sync();
  const int share = (kRows * (D / 4) + a.splits - 1) / a.splits, last = min((split + 1) * share, kRows * (D / 4));
  for (int i = split * share + tid; i < last; i += kWarps * 32) {
    const int row = i / (D / 4), c4 = i % (D / 4);
    if (r0 + row >= all) break;
    const uint32_t ml_at = (uint32_t)__cvta_generic_to_shared(&ml_s[row]), at = (uint32_t)__cvta_generic_to_shared(smem) + (row * kLine + 4 * c4) * 4;
    float2 ml[kMostCluster];
    float4 y[kMostCluster], x = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, l = 0.f;
#pragma unroll
    for (int s = 0; s < kMostCluster; ++s)
      if (s < parts) ml[s] = cluster_ld2(in_cta(ml_at, s)), y[s] = cluster_ld4(in_cta(at, s));
#pragma unroll
    for (int s = 0; s < kMostCluster; ++s)
      if (s < parts) top = fmaxf(top, ml[s].x);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int s = 0; s < kMostCluster; ++s)
      if (s < parts) {
        const float f = tree_ex2(ml[s].x - ref);
        if (f != 0.f) l += f * ml[s].y, x.x += f * y[s].x, x.y += f * y[s].y, x.z += f * y[s].z, x.w += f * y[s].w;
      }
    write_out<T, D>(a, r, kvh, r0 + row, c4, x, l);
  }
  __syncwarp();
  cluster_sync();  // (nobody leaves while its shared memory is read)
}

// Rows whose keys several CTAs shared: sum of the parts, each by 2^(its maximum - the largest).  A CTA has 32 rows of a tile
// (a row a lane, so that parts are read in whole lines).  kFewParts: and all head dimensions, an eighth a warp, which reads all parts;
// else 16 of them and a warp every eighth part, and the warps meet in shared memory.  Bound by two rounds of loads (17 parts a warp
// 22 us).
template <typename T, int D, bool kTc, bool kFewParts>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeArgs a) {
  constexpr int kChunks = kFewParts ? D / 32 : 4;  // of four dims, a thread
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kvh = blockIdx.y;
  const int rows32 = kFewParts ? blockIdx.x : blockIdx.x / (D / 16), chunk0 = kFewParts ? kChunks * warp : 4 * (blockIdx.x % (D / 16));
  const int per_tile = a.tile_rows / 32, tile = rows32 / per_tile, row = rows32 % per_tile * 32 + lane;
  pdl_launch_dependents();
  pdl_wait();
  const TreeRequest r = tree_request(a, blockIdx.z);
  const int all = min(r.n, a.max_new) * (int)a.group.d, number = tile * a.tile_rows + row;
  if (number - lane >= all) return;
  int parts;
  int64_t part0, part, step;  // the parts are part0, then part + step, part + 2 step, ...
  if constexpr (kTc) {  // the CTA where the row tile begins has it as its last segment, the others as their first
    const TreeUnits u = tree_units(a, r);
    const int64_t share = a.first[a.requests + 1], t0 = a.first[blockIdx.z] + ((int64_t)kvh * u.row_tiles + tile) * u.line_tiles;
    const int64_t t1 = t0 + u.key_tiles - 1;
    const bool narrow = t1 <= 0xffffffffll;  // (a division of 64 bits takes as long as a round of loads)
    const int64_t c0 = narrow ? (int64_t)((uint32_t)t0 / (uint32_t)share) : t0 / share;
    const int64_t c1 = narrow ? (int64_t)((uint32_t)t1 / (uint32_t)share) : t1 / share;
    parts = (int)(c1 - c0) + 1;
    part0 = 2 * c0 + 1, part = 2 * c0, step = 2;
  } else {
    int per;
    parts = tree_parts(a, r.end, per);
    part0 = part = tree_part(a, blockIdx.z, kvh, tile), step = 1;
  }
  if (parts == 1) return;
  float top = -INFINITY, l = 0.f;
  float4 o[kChunks] = {};
#pragma unroll 4
  for (int s = kFewParts ? 0 : warp; s < parts; s += kFewParts ? 1 : 8) {  // running maximum and sum
    const int64_t at = s == 0 ? part0 : part + s * step;
    const float2 x = a.part_ml[at * a.tile_rows + row];
    float4 y[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) y[c] = a.part_o[(at * (D / 4) + chunk0 + c) * a.tile_rows + row];
    const float m = fmaxf(top, x.x), ref = m == -INFINITY ? 0.f : m, f = tree_ex2(top - ref), g = tree_ex2(x.x - ref);
    top = m;
    l = (f != 0.f ? f * l : 0.f) + (g != 0.f ? g * x.y : 0.f);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      o[c].x = (f != 0.f ? f * o[c].x : 0.f) + (g != 0.f ? g * y[c].x : 0.f);
      o[c].y = (f != 0.f ? f * o[c].y : 0.f) + (g != 0.f ? g * y[c].y : 0.f);
      o[c].z = (f != 0.f ? f * o[c].z : 0.f) + (g != 0.f ? g * y[c].z : 0.f);
      o[c].w = (f != 0.f ? f * o[c].w : 0.f) + (g != 0.f ? g * y[c].w : 0.f);
    }
  }
  if constexpr (kFewParts) {
    if (number < all) {
#pragma unroll
      for (int c = 0; c < kChunks; ++c) write_out<T, D>(a, r, kvh, number, chunk0 + c, o[c], l);
    }
  } else {
    __shared__ float4 o_s[8][4][32];
    __shared__ float2 ml_s[8][32];
#pragma unroll
    for (int c = 0; c < 4; ++c) o_s[warp][c][lane] = o[c];
    ml_s[warp][lane] = make_float2(top, l);
    __syncthreads();
    if (warp >= 4 || number >= all) return;  // a warp four dims
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < 8; ++w) m = fmaxf(m, ml_s[w][lane].x);
    const float ref = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const float2 x = ml_s[w][lane];
      const float4 y = o_s[w][warp][lane];
      const float f = tree_ex2(x.x - ref);
      if (f != 0.f) sum += f * x.y, v.x += f * y.x, v.y += f * y.y, v.z += f * y.z, v.w += f * y.w;
    }
    write_out<T, D>(a, r, kvh, number, chunk0 + warp, v, sum);
  }
}

template <typename T, int D, int MT, bool kByRows>
int launch_few(const TreeArgs& a, cudaStream_t st) {
  QUIC_CUDA((allow_smem<tree_attn_kernel<T, D, MT, kByRows>>(kSmem<D, MT>)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.splits, a.kv_heads * a.tiles, a.requests);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = kSmem<D, MT>;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  if (a.cluster) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  if (pdl_enabled()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  QUIC_CUDA(cudaLaunchKernelEx(&cfg, tree_attn_kernel<T, D, MT, kByRows>, a));
  return QUIC_OK;
}

// What the end of a segment and the beginning of the next cost a CTA of the tcgen05 form, in key tiles.  us with 0 / 3 / 5 / 6 / 7 / 9:
// 64 x 8 x 200..1500 (14:2) 25.4 / 22.8 / 21.7 / 21.3 / 20.9 / 21.7, 27 x 25 x 5074..10148 (16:1) 67.4 / 66.9 / 65.2 / 65.0 / 64.8 / 65.2,
// 8 x 64 x 12000..16384 132.5 / 131.4 / 131.1 / 130.9 / 131.1 / 131.3, 10 x 38 x 4..23 (16:1) 21.8 / 14.6 / 14.4 / 14.5 / 14.3 / 14.3.
constexpr int kLineGap = 6;
constexpr int64_t kMostTokens = 1 << 29;  // of a request: sums of two counts stay within an int
// Which form takes a call, by the rows of a request and KV head and by the work of the mma.sync form, in tiles of 32 rows x keys of
// 64 dims (for all requests, of the longest's keys).  The tcgen05 form has three times its throughput where it has the rows for it,
// but 6 us more of launch and merge, and 3 us for every row tile of a CTA.  requests x nodes x tokens, us mma.sync / tcgen05:
//   heads 14:2, dim 64:  5 x 23 x 388..777 9.2 / 12.8 (work 48,000), 1 x 48 x 4096 13.1 / 15.3 (91,000), 2 x 32 x 8192 17.4 / 18.0
//                        (230,000), 64 x 5 x 500..1000 15.3 / 19.8 (257,000), 16 x 16 x 1024..2048 17.1 / 14.5 (264,000),
//                        64 x 8 x 750..1500 21.8 / 23.0 (386,000), 16 x 8 x 4096..8192 28.4 / 22.3 (525,000)
//   heads 32:8, dim 128: 20 x 28 x 7..15 15.3 / 17.2 (55,000), 4 x 16 x 512..1024 15.9 / 14.3 (133,000), 8 x 9 x 512..1024 21.6 / 20.6
//                        (264,000), 16 x 9 x 256..512 20.0 / 22.0 (267,000), 4 x 9 x 2048..4096 31.4 / 21.0 (525,000)
//   heads 16:1, dim 128: 16 x 2 x 1024..2048 15.4 / 14.3 (66,000), 4 x 8 x 2048..4096 16.4 / 14.8 (131,000), 32 x 2 x 4096..8192 32.4 /
//                        30.0 (524,000)
// Of up to 32 rows and 64 dims 9 x 13 x 7247..14495 (8:8) 41.9 / 53.1, 64 x 3 x 2000..4000 (14:2) 29.9 / 35.0.  Of 89 calls drawn over
// these ranges the rule's form is 1.2 % behind the faster one on average: even with it for 84, and behind near the line by 46 % (51 x 20 x
// 107, 32:8: 41.6 / 28.5), 33 % (1 x 13 x 17767, 16:1: 23.5 / 31.2), 17 % (22 x 33 x 7..14, 16:1: 14.4 / 12.3) and 7 %; of the calls above by
// 18 % at 16 x 16 x 1024..2048, 11 % at 4 x 16 x 512..1024, 8 % at 16 x 2 x 1024..2048.
bool tensor_pays(int64_t rows, int64_t units, int64_t bound, int dim) {
  const int64_t work = units * ((rows + 31) / 32) * bound * (dim / 64);
  return (rows > 32 || (rows > 16 && dim == 128)) &&
         work > (dim == 64 ? 225000 : 112500) + 1500 * units * ((rows + kTreeTcRows - 1) / kTreeTcRows);
}

// CTAs of the mma.sync form that run at once, by the size of their clusters (148 SMs of two, as the GPU's groups of SMs allow)
constexpr int kSlots[kMostCluster] = {296, 296, 279, 284, 280, 270, 259, 264};
struct Plan {
  bool tc, cluster;
  int64_t tiles;                   // row tiles of a request and KV head
  int tile_rows, splits, chunk;    // rows of one (a multiple of 32); mma.sync form: CTAs that share its keys, the keys of one
  int64_t parts;                   // partial results
};
// `bound`: keys of a request at most.
Plan make_plan(int requests, int kv_heads, int heads, int max_new, int64_t bound, int dim, bool tc) {
  Plan p = {};
  p.tc = tc;
  const int64_t rows = (int64_t)max_new * (heads / kv_heads);
  bound = bound < kMostTokens ? bound : kMostTokens;
  p.tile_rows = p.tc ? (int)(rows < kTreeTcRows ? (rows + 31) / 32 * 32 : kTreeTcRows) : 32;
  p.tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  p.splits = 1;
  if (p.tc) {
    p.parts = 2 * kTreeTcCtas;
    return p;
  }
  p.chunk = 64;
  // Parts by their cost in keys: waves of CTAs, each with 256 keys' worth of beginning and end; then the merge, by the cluster (64)
  // or by a kernel of its own (192 and 4 a part).  us with the best number of parts, cluster / kernel / one part, 14:2 heads of 64:
  // 1 x 1 x 300 4.8 / 5.8 / 4.6, 1 x 1 x 4000 7.6 / 7.8 (17 parts) / 24.7, 32 x 1 x 500..1000 6.8 / 8.4 / 8.9, 16 x 1 x 8192 16.7 /
  // 18.2 / 60, 5 x 23 x 0..777 8.7 / 10.0 / 11.1, 1 x 48 x 4096 12.5 (6) / 13.2 (12) / 39, 64 x 8 x 200..1500 25.1 / 22.1 / 18.6;
  // 32:8 heads of 128: 8 x 3 x 2000..4000 23.3 / 27.5 / 52; 8:8 of 64: 9 x 13 x 7247..14495 41.3 / 40.7 / 94.  The costs, fitted to loops
  // that took up to a third longer, take the best within 0.1 us but at 1 x 1 x 300 (4.9) and 1 x 48 x 4096 (13.1).  The most parts of
  // every number of waves are looked at.  (Equal shares of all requests' keys instead, which ragged requests would call for, cost a CTA two
  // row tiles one after the other: 64 x 8 x 200..1500 34 where the loop of that time took 25.6.)
  const int64_t units = (int64_t)requests * kv_heads * p.tiles, slots = kSlots[0];
  const int64_t most = bound < 256 ? 1 : (bound < 128 * 256 ? (bound + 255) / 256 : 128);
  int64_t best = 1, least = INT64_MAX;
  for (int64_t waves = 0; waves <= 4; ++waves) {
    int64_t s = waves == 0 ? 1 : waves * slots / units;
    s = s < 1 ? 1 : (s > most ? most : s);
    const int64_t part = ((bound + s - 1) / s + 63) / 64 * 64;
    const int64_t cost = (units * s + slots - 1) / slots * (part + 256) + (s > 1 ? 192 + 4 * s : 0);
    if (cost < least) least = cost, best = s;
  }
  for (int64_t s = 2; s <= kMostCluster && 64 * (s - 1) < bound; ++s) {
    const int64_t part = ((bound + s - 1) / s + 63) / 64 * 64;
    const int64_t cost = (units * s + kSlots[s - 1] - 1) / kSlots[s - 1] * (part + 256) + 64;
    if (cost < least) least = cost, best = s, p.cluster = true;
  }
  // ... or each warp has 32 rows of its own and all keys, with a quarter of the CTAs and no merge: for many rows and few keys, where
  // the warps have rows.  us keys by warps / rows by warps: 14:2 heads of 64, 64 x 16 x 15..30 12.4 / 9.0, x 50..100 12.6 / 10.6 (the
  // rule takes the former), x 200..400 17.8 / 19.2; 32:8 of 128, 20 x 28 x 7..15 19.6 / 15.4, x 50..100 21.9 / 21.5, 64 x 16 x 10..20 35.3 /
  // 24.0; 8:8 of 64, 20 x 40 x 25..50 (40 rows) 7.5 / 9.8.
  const int64_t wide = (rows + kByRowsTile - 1) / kByRowsTile, wide_units = (int64_t)requests * kv_heads * wide;
  if (best == 1 && rows > 32 && 2 * rows >= wide * kByRowsTile &&
      192 + (wide_units + slots - 1) / slots * ((dim == 64 ? 4 : 6) * bound + 96) <
          256 + (units + slots - 1) / slots * ((bound + 63) / 64 * 64 + 96)) {
    p.tile_rows = kByRowsTile, p.tiles = wide;
    return p;
  }
  p.chunk = (int)(((bound + best - 1) / best + 63) / 64 * 64);
  if (p.chunk < 64) p.chunk = 64;
  p.splits = (int)((bound + p.chunk - 1) / p.chunk);
  if (p.splits < 1) p.splits = 1;
  if (p.cluster) p.chunk = 64;  // (shorter requests: all CTAs of the cluster are there)
  p.parts = p.splits > 1 && !p.cluster ? units * p.splits : 0;
  return p;
}
int64_t first_bytes(const Plan& p, int requests) { return p.tc ? ((int64_t)requests + 2 + 1) / 2 * 16 : 0; }

template <typename T, int D>
int launch_typed(const TreeArgs& a, const Plan& p, cudaStream_t st) {
  const int rc = p.tc                             ? tree_attn_tc_launch(a, kTreeExponent<T> == kTreeExponent<__nv_bfloat16>, D, st)
                 : p.tile_rows == kByRowsTile     ? launch_few<T, D, 2, true>(a, st)
                 : a.max_new * (int64_t)a.group.d <= 16 ? launch_few<T, D, 1, false>(a, st)
                                                        : launch_few<T, D, 2, false>(a, st);
  if (rc != QUIC_OK || p.parts == 0) return rc;
  // few parts, and more CTAs of 16 dims than 148 SMs take at four each: us with a part a warp / with all of them, 8 x 64 x 16384 139 / 133
  // (4096 CTAs), 27 x 25 x 10148 (16:1) 66.7 / 64.9, 64 x 8 x 1500 on tcgen05 21.6 / 21.4 (1024), 16 x 1 x 8192 on it 25.4 / 27.1 (128), 8 x 48 x 2048 20 / 22 (1024, of six parts)
  const int64_t units = (int64_t)a.requests * a.kv_heads * a.tiles, narrow = units * (a.tile_rows / 32) * (D / 16);
  const bool few = narrow > 4 * 148 && (p.tc ? kTreeTcCtas / units + 2 : a.splits) <= 4;
  const dim3 grid((unsigned)(a.tiles * (a.tile_rows / 32) * (few ? 1 : D / 16)), a.kv_heads, a.requests);
  if (p.tc)
    QUIC_CUDA(launch(few ? tree_merge_kernel<T, D, true, true> : tree_merge_kernel<T, D, true, false>, grid, dim3(256), 0, st, true, a));
  else
    QUIC_CUDA(launch(few ? tree_merge_kernel<T, D, false, true> : tree_merge_kernel<T, D, false, false>, grid, dim3(256), 0, st, true, a));
  return QUIC_OK;
}

}  // namespace
}  // namespace quic

using namespace quic;

static int g_tensor_mode = -1;
extern "C" void quic_set_tree_attn_tensor(int mode) { g_tensor_mode = mode; }

extern "C" int64_t quic_tree_attn_scratch_bytes(int32_t requests, int32_t heads, int32_t kv_heads, int32_t dim, int32_t max_new,
                                                int64_t max_len) {
  if (requests < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || (dim != 64 && dim != 128) || max_new < 1 || max_len < 0) return 0;
  int64_t most = 0;  // (of either form: strides decide too)
  for (int tc = 0; tc < 2; ++tc) {
    const Plan p = make_plan(requests, kv_heads, heads, max_new, max_len + max_new, dim, tc != 0);
    const int64_t need = first_bytes(p, requests) + p.parts * p.tile_rows * (dim + 2) * 4;
    most = need > most ? need : most;
  }
  return most;
}

extern "C" int quic_tree_attn(const quic_tree_attn_t* t, void* scratch, void* stream) {
  QUIC_REQUIRE(t != nullptr, QUIC_E_ARG, "tree_attn: null arguments");
  QUIC_REQUIRE(t->dtype == QUIC_DTYPE_F16 || t->dtype == QUIC_DTYPE_BF16, QUIC_E_SHAPE, "tree_attn: unknown element type");
  QUIC_REQUIRE(t->dim == 64 || t->dim == 128, QUIC_E_SHAPE, "tree_attn: the head dimension is 64 or 128");
  QUIC_REQUIRE(t->rows >= 0 && t->requests >= 0 && t->heads >= 1 && t->kv_heads >= 1 && t->heads % t->kv_heads == 0, QUIC_E_SHAPE,
               "tree_attn: bad row, request or head count");
  QUIC_REQUIRE(t->n_blocks >= 1 && t->block_size >= 1 && t->max_blocks >= 1 && (int64_t)t->block_size * t->max_blocks <= kMostTokens,
               QUIC_E_SHAPE, "tree_attn: bad block geometry");
  QUIC_REQUIRE(t->max_new >= 1 && t->max_len >= 0, QUIC_E_SHAPE, "tree_attn: bad bounds of a request's rows or tokens");
  if (t->rows == 0 || t->requests == 0) return QUIC_OK;
  QUIC_REQUIRE(t->q && t->k && t->v && t->out && t->tables && t->lengths && t->row_start, QUIC_E_ARG, "tree_attn: null tensor");
  QUIC_REQUIRE(t->mask == nullptr || t->mask_words >= 1, QUIC_E_SHAPE, "tree_attn: a mask has at least one word a row");
  QUIC_REQUIRE(((uintptr_t)t->q | (uintptr_t)t->k | (uintptr_t)t->v | (uintptr_t)t->out) % 16 == 0, QUIC_E_ARG,
               "tree_attn: tensors must be 16-byte aligned");
  QUIC_REQUIRE(((t->q_row | t->q_head | t->k_block | t->k_head | t->k_tok | t->v_block | t->v_head | t->v_tok) & 7) == 0, QUIC_E_ARG,
               "tree_attn: strides must be multiples of 8 elements");
  QUIC_REQUIRE((int64_t)t->rows * t->heads < (1ll << 31), QUIC_E_LIMIT, "tree_attn: rows times heads reach 2^31");
  const int max_new = t->max_new < t->rows ? t->max_new : t->rows;
  const int64_t room = (int64_t)t->max_blocks * t->block_size, max_len = t->max_len < room ? t->max_len : room;
  const int mode = g_tensor_mode;
  const bool tc = mode != 0 && tree_attn_tc_takes(t->block_size, t->k_block, t->k_head, t->k_tok, t->v_block, t->v_head, t->v_tok) &&
                  (mode == 1 || tensor_pays((int64_t)max_new * (t->heads / t->kv_heads), (int64_t)t->requests * t->kv_heads,
                                            max_len + max_new, t->dim));
  const Plan p = make_plan(t->requests, t->kv_heads, t->heads, max_new, max_len + max_new, t->dim, tc);
  QUIC_REQUIRE(t->requests <= 65535 && t->kv_heads * p.tiles <= 65535, QUIC_E_LIMIT,
               "tree_attn: more than 65535 requests, or row tiles of one");
  TreeArgs a = {};
  a.splits = p.splits, a.chunk = p.chunk, a.cluster = p.cluster, a.line_gap = kLineGap, a.tiles = (int)p.tiles, a.tile_rows = p.tile_rows;
  QUIC_REQUIRE(p.parts == 0 || (scratch != nullptr && (uintptr_t)scratch % 16 == 0), QUIC_E_ARG,
               "tree_attn: scratch missing or not 16-byte aligned");
  a.q = t->q, a.k = t->k, a.v = t->v, a.out = t->out;
  a.q_row = t->q_row, a.q_head = t->q_head;
  a.k_block = t->k_block, a.k_head = t->k_head, a.k_tok = t->k_tok;
  a.v_block = t->v_block, a.v_head = t->v_head, a.v_tok = t->v_tok;
  a.table_row = t->table_row, a.mask_row = t->mask_row;
  a.tables = t->tables, a.lengths = t->lengths, a.row_start = t->row_start;
  a.mask = (const uint32_t*)t->mask, a.mask_words = t->mask_words;
  a.first = (int64_t*)scratch;
  a.part_o = (float4*)((char*)scratch + first_bytes(p, t->requests));
  a.part_ml = (float2*)(a.part_o + p.parts * p.tile_rows * (t->dim / 4));
  a.block = FastDiv::of((uint32_t)t->block_size);
  a.group = FastDiv::of((uint32_t)(t->heads / t->kv_heads));
  a.rows = t->rows, a.requests = t->requests, a.heads = t->heads, a.kv_heads = t->kv_heads;
  a.n_blocks = t->n_blocks, a.max_blocks = t->max_blocks, a.max_new = max_new;
  a.scale_log2 = (t->scale > 0.f ? t->scale : 1.f / sqrtf((float)t->dim)) * 1.4426950408889634f;
  cudaStream_t st = (cudaStream_t)stream;
  if (t->dtype == QUIC_DTYPE_F16)
    return t->dim == 64 ? launch_typed<half, 64>(a, p, st) : launch_typed<half, 128>(a, p, st);
  return t->dim == 64 ? launch_typed<__nv_bfloat16, 64>(a, p, st) : launch_typed<__nv_bfloat16, 128>(a, p, st);
}
