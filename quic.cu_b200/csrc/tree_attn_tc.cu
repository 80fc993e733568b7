// Tree attention of many rows on tcgen05: the throughput form of tree_attn.cu.
//
// A CTA, alone on its SM, owns up to 256 rows (row = node x heads per KV head + head) of one request and KV head and a part
// of its keys, and walks those 64 at a time in two streams, each with 128 rows, a softmax group of four warps, two score buffers
// and an accumulator in tensor memory.  With more than 128 rows the streams are the two halves of the rows and share every
// key tile; with fewer they are the even and the odd key tiles of the same rows, and meet at the end.  Per tile and stream:
//   S = Q K^T      A = Q (128 x dim, loaded once), B = K tile, both K-major in the 128-byte swizzle; S (128 x 64 fp32) in
//                  tensor memory, a tile ahead of the softmax;
//   softmax        a thread owns a row (TMEM lane): P = exp2(..) rounded to the tensors' type, which replaces the scores as
//                  the A operand of the second product; warps without rows rest;
//   O += P V       B = the V tile as it lies in the cache (token-major, the transposed form), N = the head dims.
// O is rescaled in tensor memory when a row's reference point moves (kTreeGrowth).
// K and V come by TMA, in boxes of as many tokens as lie together in a block for sure (the largest power of two that divides
// the block size, 8 to 64); positions without a block are fetched from beyond the planes, as zeros.  (By cp.async, which takes
// any block size, the loaders had to fence every stage for the tensor cores, and the fence waited for all copies under way:
// 8 requests x 64 nodes x 12000..16384 tokens, bf16, 32:8 heads of 128, 215 us instead of 193.)
// Only tiles that reach beyond the cached tokens look at masks.  A V row of a node may hold infinities or NaN that most rows
// must not see: such values are zeroed in shared memory and added, at the end, to the rows that see them.
//
// The CTAs have equal shares of the line of key tiles of all requests (tree_attn.cuh): the same case 193 -> 143 us, with an issuer
// per stream instead of one for both.  126 to 132 us now (3.6 to 3.8 TB/s, 750 to 780 TFLOP/s) at the 1.8 GHz that it has after a rest, 152 to
// 156 at the 1.53 GHz that calls one after the other settle at (power limit): 2170 clocks a tile by stamps in both.  Of the 143, K and V alone
// took 101, with the products 112.  A softmax warp's clocks: 1150 to 1550 from complete scores to stored weights (1550 the slowest of a
// stream's four, which sets the pace), 150 to 500 until the scores are complete, 450 for the way round; two of them share a scheduler.  With all exponentials on their unit (512 clocks a warp
// and tile, 54 % busy) it was 143; three in eight are polynomials.  Tried and behind: scores fetched during the last exponentials 153, weights by the
// old maximum before the new one is known 157, two threads a row 187, one lane of a warp waiting for all 170, two CTAs an SM with a
// stream each 27 -> 31 us at 4 x 15 x 6146.
//
// Roles: warps 0-7 queries, softmax and epilogue, warps 8 and 9 MMA issuers of the two streams, warps 10 and 11
// TMA of K and V.  Every wait is bounded; a wait that runs out sets word 0 of the tensor path's error words and the CTA leaves with
// its MMAs and copies complete and its tensor memory released.
#include "tc_common.cuh"
#include "tree_attn.cuh"

namespace quic {
namespace {

constexpr int kRows = 128, kKeys = 64, kGroupWarps = 4, kSoftmaxWarps = 2 * kGroupWarps;
constexpr int kTmaWarp = kSoftmaxWarps + 2, kThreads = (kTmaWarp + 2) * 32;
constexpr int kLeastShare = 2;  // key tiles of a CTA
static_assert(2 * kRows == kTreeTcRows && kKeys == kTreeTcKeys, "two streams of rows");
constexpr uint32_t kHalfQ = kRows * 128, kHalfK = kKeys * 128;  // 64 dims of Q, of a K or V tile

struct TreeTcArgs {
  TreeArgs t;
  int32_t box, log_boxes; // tokens of a TMA box, log2 of the boxes of a tile
  uint32_t wait_limit_us;
  int32_t skip_tile;      // test hook: this key tile never comes; below -1, all come late, and issuers without a step (-1: none)
};

__device__ __forceinline__ void mbar_arrive_cta(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {  // zeros beyond `bytes`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// 2^x of two x up to 127, without the unit for exponentials: x = n + f with n the nearest whole number (the low bits of x + 1.5 2^23),
// 2^f = 1 + f (c1 + c2 f + c3 f^2 + c4 f^3) on [-1/2, 1/2], fitted to the least largest relative error, 2^-18.4, and 2^n put together
// from its exponent.  Below -127: 0.  NaN stays.
__device__ __forceinline__ void ex2_fma(uint64_t x2, float& p0, float& p1) {
  float x, y;
  unpair2(x2, x, y);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(y) : "f"(-127.f));
  const uint64_t q = pair2(x, y), n = add2(q, pair2(12582912.f, 12582912.f));
  const uint64_t f = fma2(add2(n, pair2(-12582912.f, -12582912.f)), pair2(-1.f, -1.f), q);
  uint64_t p = fma2(pair2(0.00958285f, 0.00958285f), f, pair2(0.05590642f, 0.05590642f));
  p = fma2(p, f, pair2(0.24024099f, 0.24024099f));
  p = fma2(p, f, pair2(0.69312419f, 0.69312419f));
  p = fma2(p, f, pair2(1.f, 1.f));
  unpair2(n, x, y);
  unpair2(mul2(p, pair2(__int_as_float((__float_as_int(x) << 23) + 0x3f800000), __int_as_float((__float_as_int(y) << 23) + 0x3f800000))),
          p0, p1);
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
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
__device__ __forceinline__ void tmem_st2(uint32_t taddr, uint32_t a, uint32_t b) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1,%2};" ::"r"(taddr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Barrier 1: the softmax warps.
__device__ __forceinline__ void softmax_barrier() { asm volatile("barrier.cta.sync 1, %0;" ::"n"(kSoftmaxWarps * 32) : "memory"); }

template <int D>
constexpr int kStages = D == 64 ? 8 : 5;
template <int D>
constexpr uint32_t kTcSmem = (D / 64) * (2 * kHalfQ + kStages<D> * 2 * kHalfK) + 1024;  // Q of both streams, stages of K and V
static_assert(kTcSmem<128> + 1024 <= 232448 && kTcSmem<64> > 115 * 1024, "one CTA fills an SM: it takes all tensor memory");

// A CTA's way through its share of the line of key tiles.
struct Segment {
  TreeRequest r;
  int b, kvh, r0, rows;             // request, KV head, first row of the row tile, rows of the request
  int tile0, n_tiles, key_tiles;    // key tiles of the row tile: the first of the segment, their number, all
  bool halves;                      // two streams of rows, or of key tiles
  __device__ __forceinline__ int steps(int g) const { return halves ? n_tiles : (n_tiles + 1 - g) / 2; }
  __device__ __forceinline__ int step_tile(int g, int k) const { return halves ? k : 2 * k + g; }
  __device__ __forceinline__ int warps(int g) const {  // of a stream that have rows
    return max(0, min((rows - r0 - (halves ? g * kRows : 0) + 31) / 32, kGroupWarps));
  }
  __device__ __forceinline__ int begin() const { return tile0 * kKeys; }
  __device__ __forceinline__ int end() const { return min((tile0 + n_tiles) * kKeys, r.end); }
};
struct Walk {
  int b;
  int64_t at, left;  // tile of the request, tiles still to do
  __device__ __forceinline__ bool next(const TreeArgs& a, Segment& s) {
    while (left > 0) {
      s.r = tree_request(a, b);
      const TreeUnits u = tree_units(a, s.r);
      s.b = b;
      if (u.rows == 0) {
        ++b;
        continue;
      }
      // (a division of 64 bits takes longer than a key tile's products)
      const uint32_t unit = at <= 0xffffffffll ? (uint32_t)at / (uint32_t)u.line_tiles : (uint32_t)(at / u.line_tiles);
      s.tile0 = (int)(at - (int64_t)unit * u.line_tiles);
      s.n_tiles = (int)min(left, (int64_t)(u.key_tiles - s.tile0));
      const int step = s.tile0 + max(s.n_tiles, 0) >= u.key_tiles ? u.line_tiles - s.tile0 : s.n_tiles;  // with the gap behind the last
      at += step;
      left -= step;
      if (at == u.all(a)) ++b, at = 0;
      if (s.n_tiles <= 0) continue;  // (began in a gap)
      s.kvh = (int)(unit / (uint32_t)u.row_tiles);
      s.r0 = (int)(unit - (uint32_t)s.kvh * u.row_tiles) * kTreeTcRows;
      s.rows = u.rows;
      s.halves = u.rows - s.r0 > kRows;
      s.key_tiles = u.key_tiles;
      return true;
    }
    return false;
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) tree_attn_tc_kernel(const __grid_constant__ CUtensorMap tm_k,
                                                                   const __grid_constant__ CUtensorMap tm_v,
                                                                   const __grid_constant__ TreeTcArgs args, int* status) {
  constexpr int kHalves = D / 64, kRing = kStages<D>;
  constexpr uint32_t kColO = 256, kTmemCols = 512;  // scores of stream g, buffer x: 128 g + 64 x; O of stream g: 256 + 128 g
  constexpr uint32_t kQ = kHalves * kHalfQ, kK = 2 * kQ, kTile = kHalves * kHalfK, kStage = 2 * kTile;  // a stage: K, V
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kRing], bar_empty[kRing], bar_s[2][2], bar_p[2][2], bar_o[2][2], bar_q, bar_drain;
  __shared__ uint32_t valid_s[kRing];  // which boxes of the stage have a block
  __shared__ int64_t sums_s[kThreads / 32];
  __shared__ Walk walk_s;
  __shared__ Segment segment_s;
  __shared__ uint32_t tmem_base_s;
  __shared__ int fail_s, odd_s[2];  // odd_s: the first tile of an even, odd segment in which V held what is not finite

  const TreeArgs& a = args.t;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* const smem = smem_raw + (base - smem_u32(smem_raw));

  // ---- barriers and tensor memory, before the kernels in front have ended
  if (warp == kTmaWarp && lane == 0) {
    for (int s = 0; s < kRing; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 2);
      mbar_init(smem_u32(&bar_empty[s]), 2);
    }
    for (int g = 0; g < 2; ++g)
      for (int x = 0; x < 2; ++x) {
        mbar_init(smem_u32(&bar_s[g][x]), 2);
        mbar_init(smem_u32(&bar_p[g][x]), kGroupWarps);
        mbar_init(smem_u32(&bar_o[g][x]), 1);
      }
    mbar_init(smem_u32(&bar_q), kSoftmaxWarps + 2);
    mbar_init(smem_u32(&bar_drain), 2);
    fail_s = 0;
    odd_s[0] = odd_s[1] = 0x7fffffff;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kSoftmaxWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();

  // ---- the line of key tiles, and where in it this CTA begins
  uint32_t tmem;
  {
    const int each = (a.requests + kThreads - 1) / kThreads, b0 = min(tid * each, a.requests), b1 = min(b0 + each, a.requests);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += tree_units(a, tree_request(a, b)).all(a);
    int64_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += y;
    }
    if (lane == 31) sums_s[warp] = before;
    before -= mine;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    tmem = tmem_base_s;
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += sums_s[w];
      total += sums_s[w];
    }
    const int64_t share = max((int64_t)kLeastShare, (total + kTreeTcCtas - 1) / kTreeTcCtas), start = blockIdx.x * share;
    if (blockIdx.x == 0) {  // for the merge
      int64_t sum = before;
      for (int b = b0; b < b1; ++b) {
        a.first[b] = sum;
        sum += tree_units(a, tree_request(a, b)).all(a);
      }
      if (tid == 0) a.first[a.requests] = total, a.first[a.requests + 1] = share;
    }
    if (start >= total) {
      if (warp == kSoftmaxWarps)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
      return;
    }
    if (before <= start && start < before + mine) {
      int b = b0;
      for (int64_t n; (n = tree_units(a, tree_request(a, b)).all(a)) <= start - before; ++b) before += n;
      Walk first = {b, start - before, min(share, total - start)};
      if (!first.next(a, segment_s)) segment_s.n_tiles = 0;
      walk_s = first;
    }
    __syncthreads();
    if (segment_s.n_tiles == 0) {  // the share is all gap
      if (warp == kSoftmaxWarps)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
      return;
    }
  }
  Walk walk = walk_s;
  Segment s = segment_s, later;  // this one and the next, whose numbers are fetched ahead
  bool more = true, more_later = false;
  int ring = 0;  // tiles of the segments before
  bool issuer = false;

  if (warp >= kTmaWarp) {
    // ---------------- TMA, K and V: a lane a box of 64 dims.  (A warp's copies go out one after the other, 80 clocks each) ----------------
    const int what = warp - kTmaWarp, boxes = 1 << args.log_boxes, box = lane & (boxes - 1), half = lane >> args.log_boxes;
    const bool copies = half < kHalves;
    const CUtensorMap* const map = what ? &tm_v : &tm_k;
    const uint32_t dst = base + kK + what * kTile + half * kHalfK + box * args.box * 128;
    if (lane == 0) tma_prefetch_desc(map);
    bool ok = true;
    for (; ok && more; s = later, more = more_later) {
      const int32_t* table = a.tables + (int64_t)s.b * a.table_row;
      const int t_begin = s.begin(), t_end = s.end();
      // the blocks of 32 boxes, n_blocks (beyond the planes) where there is none; those of the next 32 are under way meanwhile
      const int at_once = 32 >> args.log_boxes;
      auto fetch = [&](int i) {
        const int p = t_begin + i * kKeys + lane * args.box, id = p < t_end ? __ldg(table + a.block.div(p)) : -1;
        return id >= 0 && id < a.n_blocks ? id : a.n_blocks;
      };
      int ids = 0, next = fetch(0);
      for (int i = 0; i < s.n_tiles; ++i, ++ring) {
        const int st = ring % kRing;
        if ((i & (at_once - 1)) == 0) {
          ids = next;
          next = fetch(i + at_once);
        }
        const int id = __shfl_sync(0xffffffffu, ids, ((i & (at_once - 1)) << args.log_boxes) + box);
        if (ring >= kRing && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_empty[st]), (ring / kRing - 1) & 1, args.wait_limit_us))) {
          fail_s = 2;
          ok = false;
          break;
        }
        if (args.skip_tile < -1) pause_us(-args.skip_tile);
        const uint32_t there = __ballot_sync(0xffffffffu, id < a.n_blocks) & (0xffffffffu >> (32 - boxes));
        const uint32_t full = smem_u32(&bar_full[st]);
        if (lane == 0) {
          if (what == 0) valid_s[st] = there;
          mbar_expect_tx(full, kTile);
        }
        __syncwarp();
        const int p = t_begin + i * kKeys + box * args.box;
        if (copies && (ring != args.skip_tile || what))
          tma_load_4d(dst + st * kStage, map, 64 * half, p - (int)a.block.div(p) * (int)a.block.d, s.kvh, id, full);
        if (i == min(2, s.n_tiles - 1)) more_later = walk.next(a, later);
      }
    }
  } else if (warp >= kSoftmaxWarps) {
    // ---------------- MMA issuers, one per stream: a warp in step, one lane of which issues ----------------
    const int g = warp - kSoftmaxWarps;
    issuer = elect_one();
    const uint64_t q0 = umma_desc_sw128(base), k0 = umma_desc_sw128(base + kK);
    // V: head dims contiguous, the two halves of 128 dims kHalfK apart (leading byte offset)
    const uint64_t v0 = umma_desc_sw128(base + kK + kTile) + ((uint64_t)(kHalfK / 16 - 1) << 16);
    constexpr uint32_t kType = kTreeExponent<T> == kTreeExponent<__nv_bfloat16> ? (1u << 7) | (1u << 10) : 0u;  // bf16 x bf16
    const uint32_t idesc = umma_idesc_f16(kKeys) | kType;             // M = 128, N = 64
    const uint32_t idesc_v = umma_idesc_f16(D) | kType | (1u << 16);  // N = the head dims, B transposed
    const uint32_t at_s = tmem + 128u * g, at_o = tmem + kColO + 128u * g;
    auto wait = [&](uint64_t* bar, int parity) {
      return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, args.wait_limit_us)) != 0;
    };
    int u = 0;  // steps of the segments before
    bool ok = true;
    for (int seg = 0; ok && more; s = later, more = more_later, ++seg) {
      const int steps = s.steps(g);
      // Through with the segment before.  In a segment without a step for its stream nothing else waits for an issuer, which waits for a
      // parity: two segments behind the others it would wait for a phase that has passed.
      if (lane == 0) mbar_arrive_cta(smem_u32(&bar_q));
      if (args.skip_tile < -1 && steps == 0) pause_us(min(-2 * args.skip_tile, (int)(args.wait_limit_us / 2)));
      const uint64_t q = q0 + (uint64_t)((s.halves ? g : 0) * (kQ / 16));
      auto scores = [&](int k) {
        const int n = ring + s.step_tile(g, k), st = n % kRing, x = (u + k) & 1;
        if (!wait(&bar_full[st], (n / kRing) & 1)) return false;
        // the product that read the buffer's last P is complete
        if (u + k >= 2 && !wait(&bar_o[g][x], (((u + k) >> 1) - 1) & 1)) return false;
        tc_fence_after();
        const uint64_t kt = k0 + (uint64_t)(st * (kStage / 16));
        const uint32_t to = at_s + 64u * x, bar = smem_u32(&bar_s[g][x]);
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < D / 16; ++c)
            umma_f16(to, q + (uint64_t)((c >> 2) * (kHalfQ / 16)) + 2 * (c & 3), kt + (uint64_t)((c >> 2) * (kHalfK / 16)) + 2 * (c & 3),
                     idesc, c > 0 ? 1u : 0u);
          umma_commit(bar);
          mbar_arrive_cta(bar);  // (hands on what it has seen of the stage: which boxes are there)
        }
        __syncwarp();
        return true;
      };
      more_later = walk.next(a, later);
      ok = wait(&bar_q, seg & 1) && (steps == 0 || scores(0));
      for (int k = 0; ok && k < steps; ++k) {
        const int n = ring + s.step_tile(g, k), st = n % kRing, x = (u + k) & 1;
        ok = (k + 1 == steps || scores(k + 1)) && wait(&bar_p[g][x], ((u + k) >> 1) & 1);  // P is there, O rescaled where need be
        if (!ok) break;
        tc_fence_after();
        const uint64_t vt = v0 + (uint64_t)(st * (kStage / 16));
        const uint32_t from = at_s + 64u * x, bar = smem_u32(&bar_o[g][x]), free = smem_u32(&bar_empty[st]);
        const uint32_t onto = k > 0 ? 1u : 0u;
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < 4; ++c)  // sixteen tokens a step: two groups of eight rows of the V tile, eight columns of P
            umma_ts(at_o, from + 8u * c, vt + c * (2048 / 16), idesc_v, c > 0 ? 1u : onto);
          umma_commit(bar);
          umma_commit(free);
          if (!s.halves) umma_commit(free);  // (nobody else reads the tile)
        }
        __syncwarp();
      }
      u += steps;
      ring += s.n_tiles;
    }
    if (!ok) fail_s = 3;
  } else {
    // ---------------- queries, softmax, epilogue ----------------
    const int group = warp / kGroupWarps, quarter = warp % kGroupWarps;
    const uint32_t lane_addr = (uint32_t)(32 * quarter) << 16;
    const uint32_t at_o = tmem + kColO + 128u * group + lane_addr;
    const uint32_t limit = 2 * args.wait_limit_us;  // (the issuers and the TMA warp give up first)
    const uint64_t scale2 = pair2(a.scale_log2, a.scale_log2);
    int u0 = 0;  // steps of the segments before
    bool ok = true;  // (without it a warp goes on to the end, past all waits, for the barriers of the segments)
    bool ahead = false;  // the segment's queries are on their way already
    auto queries = [&](const Segment& q) {
      if (!q.halves && group != 0) return;
#pragma unroll 4
      for (int i = lane; i < 32 * (D / 8); i += 32) {  // (a warp its own rows: in their place it gathers its results)
        const int row = 32 * quarter + i / (D / 8), chunk = i % (D / 8);
        const int number = q.r0 + group * kRows + row, mine = min(number, q.rows - 1);
        const int node = (int)a.group.div(mine), head = q.kvh * (int)a.group.d + mine - node * (int)a.group.d;
        copy16(base + group * kQ + (chunk >> 3) * kHalfQ + sw128_offset(row, chunk & 7),
               reinterpret_cast<const T*>(a.q) + (int64_t)(q.r.start + node) * a.q_row + (int64_t)head * a.q_head + 8 * chunk,
               number < q.rows ? 16u : 0u);
      }
    };
    for (int seg = 0; more; s = later, more = more_later, ++seg) {
      const int t_begin = s.begin(), t_end = s.end(), steps = s.steps(group);
      // ---- queries of the stream's rows (the first stream's, where they are the same); rows that are none are zero
      if (!ahead) queries(s);
      if (s.halves || group == 0) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_cta(smem_u32(&bar_q));
      // ---- during the first product: the next segment, and what the row sees of the first tile that reaches beyond the cached tokens
      more_later = walk.next(a, later);
      const bool works = quarter < s.warps(group);
      const int number = s.r0 + (s.halves ? group * kRows : 0) + 32 * quarter + lane, mine = min(number, s.rows - 1);
      const int node = (int)a.group.div(mine);
      const int tree_from = max(t_begin, s.r.len & ~(kKeys - 1));
      const uint32_t first0 = tree_visible32(a, s.r, node, tree_from), first1 = tree_visible32(a, s.r, node, tree_from + 32);
      ok = ok && __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_q), seg & 1, limit));
      if (tid == 0) odd_s[(seg + 1) & 1] = 0x7fffffff;  // (all are through with the segment before, none with this)

      // ---- softmax
      float m_run = -INFINITY, l_run = 0.f;
      const int stride = s.halves ? 1 : 2;  // of the stream's tiles
      int i = s.step_tile(group, 0), st = (ring + i) % kRing, t = t_begin + i * kKeys, u = u0;
      for (int k = 0; ok && k < steps; ++k, ++u, i += stride, t += stride * kKeys, st = st + stride < kRing ? st + stride : st + stride - kRing) {
        const uint32_t at_s = tmem + 128u * group + 64u * (u & 1) + lane_addr;
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_s[group][u & 1]), (u >> 1) & 1, limit));
        if (!ok) break;
        const bool tree = t + kKeys > s.r.len;
        if (tree) {  // (the same for all the CTA's rows)
          // (complete: this thread reads itself what the copies brought)
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_full[st]), ((ring + i) / kRing) & 1, limit));
          if (!ok) break;
          unsigned char* const v_tile = smem + kK + st * kStage + kTile;
          bool stored = s.halves;  // (each stream for itself, changed or not: the other's change may be under way)
#pragma unroll 4
          for (int c = 32 * quarter + lane; c < (int)kTile / 16; c += 32 * kGroupWarps) {
            uint4 w = reinterpret_cast<const uint4*>(v_tile)[c];
            const bool odd = tree_not_finite<T>(w);
            if (odd) {
              w.x = tree_finite<T>(w.x), w.y = tree_finite<T>(w.y), w.z = tree_finite<T>(w.z), w.w = tree_finite<T>(w.w);
              if (t + (c % (kKeys * 8)) / 8 < t_end) {  // (rows behind the last key may hold anything)
                atomicMin(&odd_s[seg & 1], i);
                __threadfence_block();  // known before it is gone
              }
              stored = true;
            }
            if (odd || s.halves) reinterpret_cast<uint4*>(v_tile)[c] = w;
          }
          if (stored) fence_proxy_async();
          __syncwarp();
        }
        if (!works) {
          if (lane == 0) mbar_arrive_cta(smem_u32(&bar_p[group][u & 1]));
          continue;
        }
        tc_fence_after();
        float x[64];
        tmem_ld_cols<64>(at_s, x);
        const uint32_t there = valid_s[st], whole = 0xffffffffu >> (32 - (1 << args.log_boxes));
        if (tree || there != whole) {
          uint32_t seen0 = first0, seen1 = first1;
          if (t != tree_from) seen0 = tree_visible32(a, s.r, node, t), seen1 = tree_visible32(a, s.r, node, t + 32);
          const int left = t_end - t;
          if (left < 64) {
            seen0 &= left < 32 ? (1u << max(left, 0)) - 1u : 0xffffffffu;
            seen1 &= left < 32 ? 0u : (1u << (left - 32)) - 1u;
          }
          if (there != whole) {
            const uint64_t tokens = 0xffffffffffffffffull >> (64 - args.box);
            uint64_t have = 0ull;
            for (int j = 0; j < 1 << args.log_boxes; ++j)
              if (there >> j & 1u) have |= tokens << (j * args.box);
            seen0 &= (uint32_t)have;
            seen1 &= (uint32_t)(have >> 32);
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (!(seen0 >> j & 1u)) x[j] = -INFINITY;
            if (!(seen1 >> j & 1u)) x[32 + j] = -INFINITY;
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // independent chains
#pragma unroll
        for (int j = 0; j < 64; j += 2) mx[(j >> 1) & 3] = max3(mx[(j >> 1) & 3], x[j], x[j + 1]);
        const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;  // (the scale is positive)
        const bool grown = mt > m_run + kTreeGrowth;  // (from -inf: by any score)
        if (k == 0) {
          m_run = mt;
        } else if (__any_sync(0xffffffffu, grown)) {
          const float alpha = grown ? tree_ex2(m_run - mt) : 1.f;
          if (grown) m_run = mt;
          l_run *= alpha;
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_o[group][(u - 1) & 1]), ((u - 1) >> 1) & 1, limit));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            float v[16];
            uint32_t w[16];
            tmem_ld_cols<16>(at_o + 16u * c, v);
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(v[j] * alpha);
            tmem_st16(at_o + 16u * c, w);
          }
        }
        const float ref = kTreeShift<T> - (m_run == -INFINITY ? 0.f : m_run);
        const uint64_t ref2 = pair2(ref, ref);
        uint64_t l2[2] = {0ull, 0ull};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t w[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float p0, p1;
            const uint64_t e = fma2(pair2(x[32 * h + 2 * j], x[32 * h + 2 * j + 1]), scale2, ref2);
            if (j % 8 == 1 || j % 8 == 4 || j % 8 == 6) {  // three in eight: none 143 us, two 134.8, three 133.9, four 139 (with a slower merge)
              ex2_fma(e, p0, p1);
            } else {
              unpair2(e, p0, p1);
              p0 = tree_ex2(p0);  // 2^-inf = 0 for keys that are not seen
              p1 = tree_ex2(p1);
            }
            w[j] = tree_pack<T>(p0, p1);
            l2[j & 1] = add2(l2[j & 1], pair2(p0, p1));
          }
          tmem_st16(at_s + 16u * h, w);  // (P in the scores' own columns: they have all been read)
        }
        float la, lb;
        unpair2(add2(l2[0], l2[1]), la, lb);
        l_run += la + lb;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cta(smem_u32(&bar_p[group][u & 1]));
      }
      u0 += steps;
      ring += s.n_tiles;
      if (ok && steps > 0)  // the last product
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_o[group][(u0 - 1) & 1]), ((u0 - 1) >> 1) & 1, limit));
      tc_fence_after();
      if (l_run != l_run) m_run = INFINITY;  // (a maximum passes over NaN)

      // ---- epilogue; streams that share their rows meet here: both accumulators are in reach of both streams' warps, which
      // have half of the head dims each
      if (!s.halves) {
        tmem_st2(tmem + 128u * group + lane_addr, __float_as_uint(m_run), __float_as_uint(l_run));  // (the scores have been used)
        tmem_wait_st();
        tc_fence_before();
        softmax_barrier();
        tc_fence_after();
      }
      // The next segment's queries, while the results are written, where their place is free: in a segment of two streams of rows the
      // stream's own, unless its results are gathered there; else the first stream's (the results are gathered in the second's).
      ahead = more_later && (s.halves ? s.n_tiles != s.key_tiles : group == 0);
      if (ahead) queries(later);
      if (ok && works) {
        const bool both = s.steps(1) > 0 && !s.halves, alone = s.n_tiles == s.key_tiles;
        const int c_begin = s.halves ? 0 : group * (D / 32), c_end = s.halves ? D / 16 : (group + 1) * (D / 32);
        const uint32_t at_o0 = tmem + kColO + (s.halves ? 128u * group : 0u) + lane_addr;
        float f0 = 1.f, f1 = 0.f;
        if (!s.halves) {
          float one[2], two[2];
          tmem_ld_cols<2>(tmem + lane_addr, one);
          tmem_ld_cols<2>(tmem + 128u + lane_addr, two);
          const float top = fmaxf(one[0], two[0]), ref = top == -INFINITY ? 0.f : top;
          f0 = tree_ex2(one[0] - ref);
          f1 = tree_ex2(two[0] - ref);
          l_run = (f0 != 0.f ? f0 * one[1] : 0.f) + (f1 != 0.f ? f1 * two[1] : 0.f);
          m_run = top;
        }
        const float inv = !alone ? 1.f : (l_run != 0.f ? 1.f / l_run : 0.f);
        const bool write = number < s.rows;
        const int64_t part = 2 * blockIdx.x + (s.tile0 == 0 ? 1 : 0);
        const int odd_from = odd_s[seg & 1];
        // (the queries' place: the stream's own, or that of the stream without)
        unsigned char* const lines = smem + (s.halves ? group : 1) * kQ;
        auto line_at = [&](int row, int chunk) { return (chunk >> 3) * kHalfQ + sw128_offset(32 * quarter + row, chunk & 7); };
        if (!alone && write && c_begin == 0) a.part_ml[part * a.tile_rows + number - s.r0] = make_float2(m_run, l_run);
#pragma unroll 1
        for (int c = c_begin; c < c_end; ++c) {
          float o[16];
          __syncwarp();
          tmem_ld_cols<16>(at_o0 + 16u * c, o);
          if (both) {
            float y[16];
            tmem_ld_cols<16>(at_o0 + 128u + 16u * c, y);
#pragma unroll
            for (int z = 0; z < 16; ++z) o[z] = (f0 != 0.f ? f0 * o[z] : 0.f) + (f1 != 0.f ? f1 * y[z] : 0.f);
          }
          if (odd_from < s.n_tiles) {
            for (int p = t_begin + odd_from * kKeys; p < t_end; ++p) {
              const int j = (int)a.block.div(p), id = a.tables[(int64_t)s.b * a.table_row + j];
              if (id < 0 || id >= a.n_blocks || !(tree_visible32(a, s.r, node, p) & 1u)) continue;
              const uint32_t* v = reinterpret_cast<const uint32_t*>(reinterpret_cast<const T*>(a.v) + (int64_t)id * a.v_block +
                                                                    s.kvh * a.v_head + (int64_t)(p - j * (int)a.block.d) * a.v_tok + 16 * c);
#pragma unroll
              for (int z = 0; z < 8; ++z) {
                const float2 f = tree_unpack<T>(v[z]), w = tree_unpack<T>(tree_finite<T>(v[z]));
                o[2 * z] += f.x - w.x;  // (x - x = 0 for what is finite)
                o[2 * z + 1] += f.y - w.y;
              }
            }
          }
          if (!alone) {
            if (write) {
#pragma unroll
              for (int z = 0; z < 4; ++z)
                a.part_o[(part * (D / 4) + 4 * c + z) * a.tile_rows + number - s.r0] =
                    make_float4(o[4 * z], o[4 * z + 1], o[4 * z + 2], o[4 * z + 3]);
            }
          } else {
#pragma unroll
            for (int z = 0; z < 2; ++z)
              *reinterpret_cast<uint4*>(lines + line_at(lane, 2 * c + z)) =
                  make_uint4(tree_pack<T>(o[8 * z] * inv, o[8 * z + 1] * inv), tree_pack<T>(o[8 * z + 2] * inv, o[8 * z + 3] * inv),
                             tree_pack<T>(o[8 * z + 4] * inv, o[8 * z + 5] * inv), tree_pack<T>(o[8 * z + 6] * inv, o[8 * z + 7] * inv));
          }
        }
        __syncwarp();
        if (alone) {  // whole rows, from shared memory
          const int first = number - lane;
#pragma unroll 4
          for (int i = lane; i < 32 * 2 * (c_end - c_begin); i += 32) {
            const int at = s.halves ? i / (D / 8) : i / (D / 16), chunk = 2 * c_begin + (s.halves ? i % (D / 8) : i % (D / 16));
            if (first + at < s.rows) {
              const int nd = (int)a.group.div(first + at), head = s.kvh * (int)a.group.d + first + at - nd * (int)a.group.d;
              reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + ((int64_t)(s.r.start + nd) * a.heads + head) * D)[chunk] =
                  *reinterpret_cast<const uint4*>(lines + line_at(at, chunk));
            }
          }
          __syncwarp();
        }
        tc_fence_before();
      }
      if (!s.halves) softmax_barrier();  // the second stream's accumulator and the queries' place are free
    }
    if (!ok && fail_s == 0) fail_s = 1;
  }
  __syncwarp();
  pdl_launch_dependents();
  tc_fence_before();
  __syncthreads();
  if (fail_s != 0) {
    if (tid == 0) tc_report(status, (fail_s << 16) | 0x3000 | (blockIdx.x & 0xfff));
    drain_failed(issuer, smem_u32(&bar_drain));
  }
  if (warp == kSoftmaxWarps)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

template <typename T, int D>
int launch_tc(const TreeTcArgs& a, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t stream, int* status) {
  QUIC_CUDA((allow_smem<tree_attn_tc_kernel<T, D>>(kTcSmem<D>)));
  QUIC_CUDA(launch(tree_attn_tc_kernel<T, D>, dim3(kTreeTcCtas), dim3(kThreads),
                   kTcSmem<D>, stream, true, tm_k, tm_v, a, status));
  return QUIC_OK;
}

int box_tokens(int block_size) {
  int box = block_size & -block_size;
  return box < kKeys ? box : kKeys;
}

// [n_blocks][kv heads][block][dim] by strides, 64 dims of `box` tokens at a time
int plane_map(CUtensorMap* map, const TreeArgs& t, const void* base, int64_t block, int64_t head, int64_t tok, int dim, int box, bool bf16) {
  const cuuint64_t dims[4] = {(cuuint64_t)dim, t.block.d, (cuuint64_t)t.kv_heads, (cuuint64_t)t.n_blocks};
  const cuuint64_t strides[3] = {(cuuint64_t)tok * 2, (cuuint64_t)head * 2, (cuuint64_t)block * 2};
  const cuuint32_t shape[4] = {64, (cuuint32_t)box, 1, 1};
  return make_tiled_map(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims, strides, shape,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
}

}  // namespace

// Boxes of whole groups of eight rows (the swizzle's period) and strides that a tensor map can have.
bool tree_attn_tc_takes(int block_size, int64_t k_block, int64_t k_head, int64_t k_tok, int64_t v_block, int64_t v_head, int64_t v_tok) {
  if (block_size % 8 != 0) return false;
  for (int64_t s : {k_block, k_head, k_tok, v_block, v_head, v_tok})
    if (s <= 0 || s >= (1ll << 39)) return false;
  return true;
}

int tree_attn_tc_launch(const TreeArgs& t, bool bf16, int dim, cudaStream_t stream) {
  int* status = tc_status_words();
  QUIC_REQUIRE(status != nullptr, QUIC_E_CUDA, "tree_attn: no address for the tensor path's error words");
  TreeTcArgs a = {};
  a.t = t;
  a.box = box_tokens((int)t.block.d);
  while ((a.box << a.log_boxes) < kKeys) ++a.log_boxes;
  tc_test_hook(&a.wait_limit_us, &a.skip_tile);
  CUtensorMap tm_k, tm_v;
  int rc = plane_map(&tm_k, t, t.k, t.k_block, t.k_head, t.k_tok, dim, a.box, bf16);
  if (rc == QUIC_OK) rc = plane_map(&tm_v, t, t.v, t.v_block, t.v_head, t.v_tok, dim, a.box, bf16);
  if (rc != QUIC_OK) return rc;
  if (dim == 128)
    return bf16 ? launch_tc<__nv_bfloat16, 128>(a, tm_k, tm_v, stream, status) : launch_tc<half, 128>(a, tm_k, tm_v, stream, status);
  return bf16 ? launch_tc<__nv_bfloat16, 64>(a, tm_k, tm_v, stream, status) : launch_tc<half, 64>(a, tm_k, tm_v, stream, status);
}

}  // namespace quic
