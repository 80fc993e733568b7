// Tree attention of many rows on tcgen05: the throughput form of tree_attn.cu.
//
// A CTA owns 128 rows (row = node x heads per KV head + head) of one request and KV head and a part of its keys, and walks
// those 64 at a time:
//   S = Q K^T      A = Q (128 x dim, loaded once), B = K tile, both K-major in the 128-byte swizzle; S (128 x 64 fp32) in
//                  tensor memory;
//   softmax        four warps, a thread owns a row (TMEM lane): running maximum, P = exp2(..) rounded to the tensors'
//                  type, which replaces the scores as the A operand of the second product; warps without rows rest;
//   O += P V       B = the V tile as it lies in the cache (token-major, the transposed form), 64 dims a product.
// K and V come by cp.async from two warps, a key of the tile a lane: that takes blocks and strides of any size, and leaves
// zeros where there is no key.  They signal a stage after their copies have landed and a proxy fence; while the next
// stage is not yet free they wait for the oldest copy under way, so that no more than that is ever held back.
// Only tiles that reach beyond the cached tokens look at masks.  A V row of a node may hold infinities or NaN that most rows
// must not see: such values are zeroed in shared memory and added, at the end, to the rows that see them.
//
// Roles: warps 0-3 softmax and epilogue, warp 4 MMA issuer, warps 5-6 loaders.  Every wait is bounded; a wait that runs out
// sets word 0 of the tensor path's error words and the CTA leaves with its MMAs and copies complete and its tensor memory
// released.
#include "tc_common.cuh"
#include "tree_attn.cuh"

namespace quic {
namespace {

constexpr int kRows = 128, kKeys = 64, kSoftmaxWarps = 4, kLoaders = 2;
constexpr int kThreads = (kSoftmaxWarps + 1 + kLoaders) * 32;
constexpr uint32_t kHalfQ = kRows * 128, kHalfK = kKeys * 128;  // 64 dims of Q, of a K or V tile

struct TreeTcArgs {
  TreeArgs t;
  int32_t tiles;          // 128-row tiles of a request and KV head
  uint32_t wait_limit_us;
  int32_t skip_tile;      // test hook: this key tile never comes; below -1, all come late (-1: none)
};

__device__ __forceinline__ void mbar_arrive_cta(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {  // zeros beyond `bytes`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_landed_but(int n) {  // all groups of this thread but the last n
  if (n == 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
  else if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 2;" ::: "memory");
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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// D[tmem] (+)= A[tmem] . B, A 16-bit values packed two to a column
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Whether the phase is complete, at once (a try_wait may sleep).
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

template <int D>
constexpr uint32_t kTcSmem = (D / 64) * (kHalfQ + 2 * 2 * kHalfK) + 1024;  // Q, two stages of K and V

// kAhead: the scores of tile i + 1 are computed while the softmax of tile i runs; two score buffers.
template <typename T, int D, bool kAhead>
__global__ void __launch_bounds__(kThreads, (D == 64 && !kAhead) ? 4 : 2)
    tree_attn_tc_kernel(const __grid_constant__ TreeTcArgs args, int* status) {
  constexpr int kHalves = D / 64;
  constexpr uint32_t kColS1 = kAhead ? 64 : 0, kColO = kAhead ? 128 : 64, kTmemCols = (kColO + D) <= 128 ? 128 : 256;
  constexpr uint32_t kK = kHalves * kHalfQ, kV = kK + 2 * kHalves * kHalfK, kStage = kHalves * kHalfK;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[2], bar_empty[2], bar_s[2], bar_p, bar_drain;
  __shared__ uint32_t valid_s[2][kLoaders];
  __shared__ uint32_t tmem_base_s;
  __shared__ int fail_s, odd_s;  // odd_s: the first tile in which V held what is not finite

  const TreeArgs& a = args.t;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tile = blockIdx.x % args.tiles, split = blockIdx.x / args.tiles, kvh = blockIdx.y;
  const TreeRequest r = tree_request(a, blockIdx.z);
  const int all = min(r.n, a.max_new) * (int)a.group.d, r0 = tile * kRows;
  if (r0 >= all) return;
  int per;
  const int parts = tree_parts(a, r.end, per);
  if (split >= parts) return;
  const int t_begin = split * per, t_end = min(t_begin + per, r.end);
  const int n_tiles = (t_end - t_begin + kKeys - 1) / kKeys;
  const int active = min((all - r0 + 31) / 32, kSoftmaxWarps);  // softmax warps with rows
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* const smem = smem_raw + (base - smem_u32(smem_raw));

  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&bar_full[s]), kLoaders);
      mbar_init(smem_u32(&bar_empty[s]), 1);
      mbar_init(smem_u32(&bar_s[s]), 1);
    }
    mbar_init(smem_u32(&bar_p), active);
    mbar_init(smem_u32(&bar_drain), 1);
    fail_s = 0;
    odd_s = 0x7fffffff;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp < kSoftmaxWarps + 1) {  // queries; rows that are none are zero
    for (int i = tid; i < kRows * (D / 8); i += (kSoftmaxWarps + 1) * 32) {
      const int row = i / (D / 8), chunk = i % (D / 8);
      uint4 w = make_uint4(0u, 0u, 0u, 0u);
      if (r0 + row < all) {
        const int node = (int)a.group.div(r0 + row), head = kvh * (int)a.group.d + (r0 + row) - node * (int)a.group.d;
        w = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (int64_t)(r.start + node) * a.q_row +
                                                 (int64_t)head * a.q_head) + chunk);
      }
      *reinterpret_cast<uint4*>(smem + (chunk >> 3) * kHalfQ + sw128_offset(row, chunk & 7)) = w;
    }
    fence_proxy_async();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_s = tmem_base_s, tmem_o = tmem_base_s + kColO;

  bool issuer = false;
  if (warp > kSoftmaxWarps) {
    // ---------------- loaders ----------------
    const int me = warp - kSoftmaxWarps - 1;
    const int32_t* table = a.tables + (int64_t)blockIdx.z * a.table_row;
    auto fetch = [&](int i) {  // the block of this lane's key of tile i, -1 where there is none
      const int p = t_begin + i * kKeys + 32 * me + lane;
      const int id = p < t_end ? __ldg(table + a.block.div(p)) : -1;
      return id < a.n_blocks ? id : -1;
    };
    int landed = 0, id = fetch(0);  // tiles that have been signalled
    auto signal = [&](int issued) {
      copies_landed_but(issued - landed - 1);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0 && landed != args.skip_tile) mbar_arrive_cta(smem_u32(&bar_full[landed & 1]));
      ++landed;
    };
    bool ok = true;
    for (int i = 0; ok && i < n_tiles; ++i) {
      const int st = i & 1;
      if (i >= 2) {
        const uint32_t bar = smem_u32(&bar_empty[st]), parity = ((i >> 1) - 1) & 1;
        while (landed < i && !__all_sync(0xffffffffu, mbar_test(bar, parity))) signal(i);
        ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, args.wait_limit_us));
        if (!ok) {
          fail_s = 2;
          break;
        }
      }
      if (args.skip_tile < -1) pause_us(-args.skip_tile);
      const uint32_t there = __ballot_sync(0xffffffffu, id >= 0);
      if (lane == 0) valid_s[st][me] = there;
      const int p = t_begin + i * kKeys + 32 * me + lane;
      const int off = p - (int)a.block.div(p) * (int)a.block.d;
      const int chunk = lane & 7;  // four rows of eight 16-byte chunks an instruction
#pragma unroll 4
      for (int j = 0; j < 8; ++j) {
        const int key = 4 * j + (lane >> 3);
        const int bid = __shfl_sync(0xffffffffu, id, key), boff = __shfl_sync(0xffffffffu, off, key);
        const uint32_t bytes = bid >= 0 ? 16u : 0u;
        const int64_t at = max(bid, 0), o = bid >= 0 ? boff : 0;
        const T* k = reinterpret_cast<const T*>(a.k) + at * a.k_block + kvh * a.k_head + o * a.k_tok + chunk * 8;
        const T* v = reinterpret_cast<const T*>(a.v) + at * a.v_block + kvh * a.v_head + o * a.v_tok + chunk * 8;
        const uint32_t dst = base + st * kStage + sw128_offset(32 * me + key, chunk);
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          copy16(dst + kK + h * kHalfK, k + 64 * h, bytes);
          copy16(dst + kV + h * kHalfK, v + 64 * h, bytes);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      id = fetch(i + 1);
    }
    while (ok && landed < n_tiles) signal(n_tiles);
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == kSoftmaxWarps) {
    // ---------------- MMA issuer ----------------
    issuer = elect_one();
    if (issuer) {
      const uint64_t q0 = umma_desc_sw128(base), k0 = umma_desc_sw128(base + kK), v0 = umma_desc_sw128(base + kV);
      constexpr uint32_t kType = sizeof(T) == 2 && kTreeExponent<T> == 0x7f80u ? (1u << 7) | (1u << 10) : 0u;  // bf16 x bf16
      const uint32_t idesc = umma_idesc_f16(kKeys) | kType;  // M = 128, N = 64
      const uint32_t idesc_v = idesc | (1u << 16);           // B transposed: N (the head dims) contiguous
      auto scores = [&](int i) {
        const int st = i & 1;
        if (!mbar_wait(smem_u32(&bar_full[st]), (i >> 1) & 1, args.wait_limit_us)) return false;
        // the columns' last P has been multiplied
        if (kAhead && i >= 2 && !mbar_wait(smem_u32(&bar_empty[st]), ((i >> 1) - 1) & 1, args.wait_limit_us)) return false;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_f16(tmem_s + kColS1 * st, q0 + (uint64_t)((k >> 2) * (kHalfQ / 16)) + 2 * (k & 3),
                   k0 + (uint64_t)((st * kHalves + (k >> 2)) * (kHalfK / 16)) + 2 * (k & 3), idesc, k > 0 ? 1u : 0u);
        umma_commit(smem_u32(&bar_s[st]));
        return true;
      };
      bool ok = n_tiles == 0 || scores(0);
      for (int i = 0; ok && i < n_tiles; ++i) {
        const int st = i & 1;
        if (kAhead && i + 1 < n_tiles) ok = scores(i + 1);
        if (!ok || !mbar_wait(smem_u32(&bar_p), i & 1, args.wait_limit_us)) {  // P(i) is in tensor memory, O rescaled where need be
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
          for (int k = 0; k < 4; ++k)  // sixteen tokens a step: two groups of eight rows of the V tile, eight columns of P
            umma_ts(tmem_o + 64u * h, tmem_s + kColS1 * st + 8u * k,
                    v0 + (uint64_t)((st * kHalves + h) * (kHalfK / 16)) + k * (2048 / 16), idesc_v, (i > 0 || k > 0) ? 1u : 0u);
        umma_commit(smem_u32(&bar_empty[st]));
        if (!kAhead && i + 1 < n_tiles)  // P(i) shares S's columns: its product has to be complete
          ok = mbar_wait(smem_u32(&bar_empty[st]), (i >> 1) & 1, args.wait_limit_us) && scores(i + 1);
      }
      if (!ok) fail_s = 3;
    }
  } else if (warp < active) {
    // ---------------- softmax, epilogue ----------------
    const int row = 32 * warp + lane;  // TMEM lane
    const int mine = min(r0 + row, all - 1), node = (int)a.group.div(mine), head = kvh * (int)a.group.d + mine - node * (int)a.group.d;
    const uint32_t lane_addr = (uint32_t)(32 * warp) << 16;
    const uint32_t limit = 4 * args.wait_limit_us;  // (the issuer waits up to three times between two tiles' scores)
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    for (int i = 0; i < n_tiles; ++i) {
      const int st = i & 1, t = t_begin + i * kKeys;
      const uint32_t at_s = tmem_s + kColS1 * st + lane_addr;
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_s[st]), (i >> 1) & 1, limit));
      // (complete: for what the loaders wrote, which this thread reads itself)
      ok = ok && __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_full[st]), (i >> 1) & 1, limit));
      if (!ok) break;
      tc_fence_after();
      const uint32_t valid[2] = {valid_s[st][0], valid_s[st][1]};
      const bool tree = t + kKeys > r.len, masked = tree || (valid[0] & valid[1]) != 0xffffffffu;
      if (tree) {  // (the same for all the CTA's rows)
        unsigned char* const v_tile = smem + kV + st * kStage;
        bool odd = false;
        for (int c = tid; c < (int)kStage / 16; c += 32 * active) {
          uint4 w = reinterpret_cast<const uint4*>(v_tile)[c];
          if (tree_not_finite<T>(w.x) || tree_not_finite<T>(w.y) || tree_not_finite<T>(w.z) || tree_not_finite<T>(w.w)) {
            w.x = tree_finite<T>(w.x), w.y = tree_finite<T>(w.y), w.z = tree_finite<T>(w.z), w.w = tree_finite<T>(w.w);
            reinterpret_cast<uint4*>(v_tile)[c] = w;
            odd = true;
          }
        }
        if (odd) {
          fence_proxy_async();
          atomicMin(&odd_s, i);
        }
        __syncwarp();
      }
      uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
      if (masked) {
        seen[0] = valid[0] & tree_visible32(a, r, node, t);
        seen[1] = valid[1] & tree_visible32(a, r, node, t + 32);
      }
      float s[kAhead ? 64 : 32];  // with registers to spare the scores stay for the second pass
      auto load = [&](int h) {
        float (&part)[32] = *reinterpret_cast<float(*)[32]>(&s[kAhead ? 32 * h : 0]);
        tmem_ld32(at_s + 32u * h, part);
        if (masked) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (!(seen[h] >> j & 1u)) part[j] = -INFINITY;
        }
      };
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // independent chains
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        load(h);
        const float* part = &s[kAhead ? 32 * h : 0];
#pragma unroll
        for (int j = 0; j < 32; j += 2) mx[(j >> 1) & 3] = max3(mx[(j >> 1) & 3], part[j], part[j + 1]);
      }
      const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;  // (the scale is positive)
      if (i == 0) {
        m_run = mt;
      } else if (__any_sync(0xffffffffu, mt > m_run)) {
        const float m_new = fmaxf(m_run, mt), alpha = m_new == m_run ? 1.f : tree_ex2(m_run - m_new);
        l_run *= alpha;
        m_run = m_new;
        if (kAhead) {  // O has its last product (else the scores waited for it)
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_empty[(i - 1) & 1]), ((i - 1) >> 1) & 1, limit));
          if (!ok) break;
          tc_fence_after();
        }
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          float v[16];
          uint32_t w[16];
          tmem_ld_cols<16>(tmem_o + lane_addr + 16u * c, v);
#pragma unroll
          for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(v[j] * alpha);
          tmem_st16(tmem_o + lane_addr + 16u * c, w);
        }
      }
      const float ref = kTreeShift<T> - (m_run == -INFINITY ? 0.f : m_run);
      const uint64_t scale2 = pair2(a.scale_log2, a.scale_log2), ref2 = pair2(ref, ref);
      uint64_t l2[2] = {0ull, 0ull};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t w[16];
        if (!kAhead) load(h);
        const float* part = &s[kAhead ? 32 * h : 0];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float p0, p1;
          unpair2(fma2(pair2(part[2 * j], part[2 * j + 1]), scale2, ref2), p0, p1);
          p0 = tree_ex2(p0);  // 2^-inf = 0 for keys that are not seen
          p1 = tree_ex2(p1);
          w[j] = tree_pack<T>(p0, p1);
          l2[j & 1] = add2(l2[j & 1], pair2(p0, p1));
        }
        tmem_st16(at_s + 16u * h, w);  // (P in the scores' own columns, behind those that are still to be read)
      }
      float la, lb;
      unpair2(add2(l2[0], l2[1]), la, lb);
      l_run += la + lb;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cta(smem_u32(&bar_p));
    }
    if (ok && n_tiles > 0)
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_empty[(n_tiles - 1) & 1]), ((n_tiles - 1) >> 1) & 1, limit));
    tc_fence_after();
    ok = __all_sync(0xffffffffu, ok && !fail_s);
    if (!ok && fail_s == 0) fail_s = 1;
    if (ok) {
      const int odd_from = odd_s;  // (all softmax warps are through with the last tile)
      const int64_t line = (int64_t)(r.start + node) * a.heads + head;
      if (l_run != l_run) m_run = INFINITY;  // (a maximum passes over NaN)
      const float inv = parts > 1 ? 1.f : (l_run != 0.f ? 1.f / l_run : 0.f);
      const bool write = r0 + row < all;
      if (parts > 1 && write) a.part_ml[line * a.splits + split] = make_float2(m_run, l_run);
#pragma unroll 1
      for (int c = 0; c < D / 16; ++c) {
        float o[16] = {};
        __syncwarp();
        if (n_tiles > 0) tmem_ld_cols<16>(tmem_o + lane_addr + 16u * c, o);
        if (odd_from < n_tiles) {
          for (int p = t_begin + odd_from * kKeys; p < t_end; ++p) {
            const int j = (int)a.block.div(p), id = a.tables[(int64_t)blockIdx.z * a.table_row + j];
            if (id < 0 || id >= a.n_blocks || !(tree_visible32(a, r, node, p) & 1u)) continue;
            const uint32_t* v = reinterpret_cast<const uint32_t*>(reinterpret_cast<const T*>(a.v) + (int64_t)id * a.v_block +
                                                                  kvh * a.v_head + (int64_t)(p - j * (int)a.block.d) * a.v_tok + 16 * c);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const float2 f = tree_unpack<T>(v[x]), z = tree_unpack<T>(tree_finite<T>(v[x]));
              o[2 * x] += f.x - z.x;  // (x - x = 0 for what is finite)
              o[2 * x + 1] += f.y - z.y;
            }
          }
        }
        if (write && parts > 1) {
          float4* const to = reinterpret_cast<float4*>(a.part_o + (line * a.splits + split) * D + 16 * c);
#pragma unroll
          for (int x = 0; x < 4; ++x) to[x] = make_float4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
        } else if (write) {
          uint4* const to = reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + line * D + 16 * c);
#pragma unroll
          for (int x = 0; x < 2; ++x)
            to[x] = make_uint4(tree_pack<T>(o[8 * x] * inv, o[8 * x + 1] * inv), tree_pack<T>(o[8 * x + 2] * inv, o[8 * x + 3] * inv),
                               tree_pack<T>(o[8 * x + 4] * inv, o[8 * x + 5] * inv), tree_pack<T>(o[8 * x + 6] * inv, o[8 * x + 7] * inv));
        }
      }
    }
  }
  __syncwarp();
  pdl_launch_dependents();
  tc_fence_before();
  __syncthreads();
  if (fail_s != 0) {
    if (tid == 0) tc_report(status, (fail_s << 16) | 0x3000 | ((int)blockIdx.x & 0xfff));
    drain_failed(issuer, smem_u32(&bar_drain));
  }
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base_s), "r"(kTmemCols) : "memory");
}

template <typename T, int D, bool kAhead>
int launch_tc(const TreeTcArgs& a, cudaStream_t stream, int* status) {
  QUIC_CUDA((allow_smem<tree_attn_tc_kernel<T, D, kAhead>>(kTcSmem<D>)));
  QUIC_CUDA(launch(tree_attn_tc_kernel<T, D, kAhead>, dim3((unsigned)(a.tiles * a.t.splits), a.t.kv_heads, a.t.requests), dim3(kThreads),
                   kTcSmem<D>, stream, false, a, status));
  return QUIC_OK;
}

}  // namespace

int tree_attn_tc_launch(const TreeArgs& t, bool bf16, int dim, cudaStream_t stream) {
  int* status = tc_status_words();
  QUIC_REQUIRE(status != nullptr, QUIC_E_CUDA, "tree_attn: no address for the tensor path's error words");
  TreeTcArgs a = {};
  a.t = t;
  a.tiles = (int)(((int64_t)t.max_new * t.group.d + kRows - 1) / kRows);
  tc_test_hook(&a.wait_limit_us, &a.skip_tile);
  const bool ahead = (int64_t)a.tiles * t.splits * t.kv_heads * t.requests <= 4 * 148;
  if (dim == 128) return bf16 ? launch_tc<__nv_bfloat16, 128, true>(a, stream, status) : launch_tc<half, 128, true>(a, stream, status);
  if (bf16)
    return ahead ? launch_tc<__nv_bfloat16, 64, true>(a, stream, status) : launch_tc<__nv_bfloat16, 64, false>(a, stream, status);
  return ahead ? launch_tc<half, 64, true>(a, stream, status) : launch_tc<half, 64, false>(a, stream, status);
}

}  // namespace quic
