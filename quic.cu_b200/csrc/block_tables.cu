// The block tables, slot maps, positions and tree masks of a step, from the lengths of its requests.
//
// With take_b = max(n_new_b, 0):  need_b = max(0, ceil((len_b + take_b) / block) - held_b), 0 without rows;
// first row = exclusive sum of take, first block = exclusive sum of need, both in the order of the requests.  New block k
// of the call is ring[(head + k) % n]; what ended requests held goes to ring[(head + count + k) % n], and since free and
// held blocks are n together, the two ranges of the ring do not meet.
//
// One launch.  Every CTA takes the sums over all requests by itself (three numbers each, at most 4096 requests) and writes
// its share of rows, table entries and returned blocks, each found by bisection in the sums; nothing that another CTA may
// still read is written before the last CTA has arrived at the pool's counter, which then updates held and pool.  No CTA
// waits.  A warp builds the masks of one request's tree, 32 nodes at a time: in-chunk ancestors by pointer doubling (five
// rounds of shuffles), those of earlier chunks from the masks already written.  Bound: the latency of one launch with
// three rounds of loads; the bytes are the rows' 12 and their masks'.  With a walk along the parents per row, sums by
// shared-memory atomics and a bisection per row it took 13.8 us at 64 requests with trees of 16, and 17 us at 390,000 rows.
#include "common.cuh"

namespace quic {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kMostRequests = 4096, kWarpRows = 128;
constexpr int64_t kMostPositions = 1 << 29;

struct TablesArgs {
  int32_t *tables, *held, *pool, *row_start, *positions, *mask;
  int64_t* slot_map;
  const int32_t *lengths, *n_new, *parents;
  int64_t table_row;
  FastDiv block;
  int32_t max_blocks, n_blocks, requests, mask_words, max_rows, most_rows;
};

// The last i with first[i] <= x among 0 .. n - 1 (first[0] <= x): the request that x belongs to, since those without a
// share have the next one's beginning.
__device__ __forceinline__ int owner(const uint32_t* first, int n, uint32_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads) block_tables_kernel(const TablesArgs a) {
  extern __shared__ uint32_t sums[];  // first row, first new block, first returned block of every request, and the ends
  uint32_t *const row0 = sums, *const new0 = sums + a.requests + 1, *const old0 = sums + 2 * (a.requests + 1);
  __shared__ uint32_t part_s[3][kWarps];
  __shared__ uint64_t rows_s[kWarps], need_s[kWarps];
  __shared__ int wrong_s[kWarps], last_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const int pool_head = a.pool[0], pool_count = a.pool[1];

  // ---- the requests' rows and blocks; a thread has `each` of them, one after the other
  const int each = (a.requests + kThreads - 1) / kThreads, b0 = min(tid * each, a.requests), b1 = min(b0 + each, a.requests);
  auto share = [&](int b, uint32_t& take, uint32_t& need, uint32_t& gone, bool& too_long) {
    const int n = a.n_new[b], held = min(max(a.held[b], 0), a.max_blocks);
    const int64_t end = (int64_t)max(a.lengths[b], 0) + n;
    take = (uint32_t)max(n, 0);
    gone = n < 0 ? (uint32_t)held : 0u;
    need = 0u;
    too_long = false;
    if (n > 0) {
      too_long = end > (int64_t)a.max_blocks * a.block.d;
      const uint32_t want = too_long ? 0u : a.block.div((uint32_t)end + a.block.d - 1);
      need = want > (uint32_t)held ? want - held : 0u;
    }
  };
  uint32_t v[3] = {0u, 0u, 0u};
  uint64_t rows64 = 0ull, need64 = 0ull;
  int wrong = 0;  // 1: a request is too long, 2: it has more rows than its masks have bits
  for (int b = b0; b < b1; ++b) {
    uint32_t take, need, gone;
    bool too_long;
    share(b, take, need, gone, too_long);
    v[0] += take, v[1] += need, v[2] += gone;  // (sums that wrap belong to calls that are refused)
    rows64 += take, need64 += need;
    wrong |= (too_long ? 1 : 0) | (a.parents != nullptr && take > 32u * (uint32_t)a.mask_words ? 2 : 0);
  }
  uint32_t base[3], total[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    uint32_t x = v[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    base[i] = x - v[i];
    if (lane == 31) part_s[i][warp] = x;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    rows64 += __shfl_xor_sync(0xffffffffu, rows64, o);
    need64 += __shfl_xor_sync(0xffffffffu, need64, o);
  }
  wrong = __reduce_or_sync(0xffffffffu, wrong);
  if (lane == 0) rows_s[warp] = rows64, need_s[warp] = need64, wrong_s[warp] = wrong;
  __syncthreads();
  rows64 = need64 = 0ull;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) rows64 += rows_s[w], need64 += need_s[w], wrong |= wrong_s[w];
  const int n_ring = a.n_blocks, count = min(max(pool_count, 0), n_ring);
  const int head = n_ring > 0 ? (int)((uint32_t)pool_head % (uint32_t)n_ring) : 0;
  int status = 0;
  if (wrong & 1) status = -1;
  else if ((wrong & 2) || rows64 > (uint64_t)a.most_rows) status = -2;
  else if (need64 > (uint64_t)count) status = (int)min(need64 - (uint64_t)count, (uint64_t)0x7fffffff);
  const bool fine = status == 0;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    total[i] = 0u;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) base[i] += part_s[i][w];
      total[i] += part_s[i][w];
    }
    if (i < 2 && !fine) base[i] = total[i] = 0u;
  }
  for (int b = b0; b < b1; ++b) {
    uint32_t take = v[0], need = v[1], gone = v[2];
    bool too_long;
    if (each > 1) share(b, take, need, gone, too_long);
    row0[b] = base[0], new0[b] = base[1], old0[b] = base[2];
    if (fine) base[0] += take, base[1] += need;
    base[2] += gone;
  }
  if (tid == 0) row0[a.requests] = total[0], new0[a.requests] = total[1], old0[a.requests] = total[2];
  __syncthreads();

  // ---- this CTA's share of everything
  const int32_t* const ring = a.pool + 4;
  const int at = blockIdx.x * kThreads + tid, stride = gridDim.x * kThreads;
  auto in_ring = [&](uint32_t k) {  // (k is at most twice their number)
    if (k >= (uint32_t)n_ring) k -= n_ring;
    return k >= (uint32_t)n_ring ? k - n_ring : k;
  };
  for (int b = at; b <= a.requests; b += stride) a.row_start[b] = (int)row0[b];
  for (uint32_t k = at; k < total[1]; k += stride) {
    const int b = owner(new0, a.requests, k);
    a.tables[b * a.table_row + min(max(a.held[b], 0), a.max_blocks) + (k - new0[b])] = ring[in_ring((uint32_t)head + k)];
  }
  for (uint32_t k = at; k < total[2] && k < (uint32_t)n_ring; k += stride) {
    const int b = owner(old0, a.requests, k);
    a.pool[4 + in_ring((uint32_t)head + (uint32_t)count + k)] = a.tables[b * a.table_row + (k - old0[b])];
  }
  // rows: a warp has kWarpRows that follow one another
  for (int64_t first = (int64_t)(blockIdx.x * kWarps + warp) * kWarpRows; first < a.max_rows; first += (int64_t)gridDim.x * kWarps * kWarpRows) {
    int b = first < total[0] ? owner(row0, a.requests, (uint32_t)first) : 0;
#pragma unroll
    for (int i = 0; i < kWarpRows / 32; ++i) {
      const int64_t row = first + 32 * i + lane;
      if (row >= a.max_rows) break;
      if (row >= (int64_t)total[0]) {
        a.slot_map[row] = -1;
        a.positions[row] = 0;
        continue;
      }
      while (row0[b + 1] <= (uint32_t)row) ++b;
      const int place = max(a.lengths[b], 0) + (int)row - (int)row0[b];
      const int j = (int)a.block.div(place), held = min(max(a.held[b], 0), a.max_blocks);
      const int id = j < held ? a.tables[b * a.table_row + j] : ring[in_ring((uint32_t)head + new0[b] + (uint32_t)(j - held))];
      a.slot_map[row] = (int64_t)id * a.block.d + (place - j * (int)a.block.d);
      if (a.parents == nullptr) a.positions[row] = place;
    }
  }
  if (a.parents != nullptr) {
    for (int b = blockIdx.x * kWarps + warp; b < a.requests; b += gridDim.x * kWarps) {  // a warp a tree
      const int start = (int)row0[b], n = (int)(row0[b + 1] - row0[b]), len = n > 0 ? max(a.lengths[b], 0) : 0;
      for (int c = 0; 32 * c < n; ++c) {
        const int node = 32 * c + lane;
        int up = node < n ? a.parents[start + node] : -1;
        if (up >= node) up = -1;
        int out = up < 32 * c ? max(up, -1) : -1;  // the ancestor in an earlier chunk, of those without one in this
        up = up < 32 * c ? -1 : up - 32 * c;
        uint32_t own = 1u << lane;  // the node and its ancestors, up to but without `up`
#pragma unroll
        for (int i = 0; i < 5; ++i) {
          const uint32_t m = __shfl_sync(0xffffffffu, own, up & 31);
          const int o = __shfl_sync(0xffffffffu, out, up & 31), u = __shfl_sync(0xffffffffu, up, up & 31);
          if (up >= 0) own |= m, out = o, up = u;
        }
        int depth = len + __popc(own) - 1;
        if (node < n) {
          int32_t* const row = a.mask + (int64_t)(start + node) * a.mask_words;
          for (int w = 0; w < a.mask_words; ++w) {
            const uint32_t bits = w < c && out >= 0 ? (uint32_t)a.mask[(int64_t)(start + out) * a.mask_words + w] : (w == c ? own : 0u);
            row[w] = (int)bits;
            if (w < c) depth += __popc(bits);
          }
          a.positions[start + node] = depth;
        }
        __threadfence_block();
        __syncwarp();  // (the next chunk reads these masks)
      }
    }
    const int64_t words = (int64_t)a.max_rows * a.mask_words;
    for (int64_t i = (int64_t)total[0] * a.mask_words + at; i < words; i += stride) a.mask[i] = 0;
  }

  // ---- the last CTA: held and pool
  __threadfence();
  __syncthreads();
  if (tid == 0) last_s = atomicAdd(&a.pool[2], 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (!last_s) return;
  __threadfence();
  for (int b = tid; b < a.requests; b += kThreads) {
    const uint32_t more = new0[b + 1] - new0[b];
    if (old0[b + 1] != old0[b]) a.held[b] = 0;
    else if (more != 0u) a.held[b] = min(max(a.held[b], 0), a.max_blocks) + (int)more;
  }
  if (tid == 0) {
    if (n_ring > 0) a.pool[0] = (int)in_ring((uint32_t)head + total[1]);
    a.pool[1] = (int)min((uint32_t)count - total[1] + total[2], (uint32_t)n_ring);
    a.pool[2] = 0;
    a.pool[3] = status;
  }
}

}  // namespace
}  // namespace quic

using namespace quic;

extern "C" int quic_block_tables(const quic_block_tables_t* t, void* stream) {
  QUIC_REQUIRE(t != nullptr && t->tables && t->held && t->pool && t->lengths && t->n_new && t->row_start, QUIC_E_ARG,
               "block_tables: null tensor");
  QUIC_REQUIRE(t->max_rows >= 0 && (t->max_rows == 0 || (t->slot_map && t->positions)), QUIC_E_ARG, "block_tables: null tensor");
  QUIC_REQUIRE(t->parents == nullptr || (t->mask_words >= 1 && t->parent_rows >= 0 && (t->mask || t->max_rows == 0)), QUIC_E_ARG,
               "block_tables: parents without a mask");
  QUIC_REQUIRE(t->requests >= 1 && t->max_blocks >= 1 && t->n_blocks >= 0 && t->block_size >= 1 && t->n_blocks < (1 << 30) &&
                   (int64_t)t->max_blocks * t->block_size <= kMostPositions,
               QUIC_E_SHAPE, "block_tables: bad request count or block geometry");
  QUIC_REQUIRE(t->requests <= kMostRequests && t->max_rows <= 65535 * 256, QUIC_E_LIMIT,
               "block_tables: more than 4096 requests, or too many rows");
  const int32_t requests = t->requests, max_rows = t->max_rows, mask_words = t->mask_words;
  const int32_t* const parents = t->parents;
  const TablesArgs a = {t->tables, t->held, t->pool, t->row_start, t->positions, t->mask, t->slot_map, t->lengths, t->n_new, parents,
                        t->table_row, FastDiv::of((uint32_t)t->block_size), t->max_blocks, t->n_blocks, requests, mask_words, max_rows,
                        parents != nullptr && t->parent_rows < max_rows ? t->parent_rows : max_rows};
  // a warp's rows, or a tree, per warp at most
  int64_t ctas = ((int64_t)max_rows + kWarps * kWarpRows - 1) / (kWarps * kWarpRows);
  if (parents != nullptr && ctas < (requests + kWarps - 1) / kWarps) ctas = (requests + kWarps - 1) / kWarps;
  ctas = ctas < 1 ? 1 : (ctas > 148 * 4 ? 148 * 4 : ctas);
  const size_t smem = 3 * (size_t)(requests + 1) * 4;
  if (smem > 48000) QUIC_CUDA(allow_smem<block_tables_kernel>(3 * (kMostRequests + 1) * 4));
  QUIC_CUDA(launch(block_tables_kernel, dim3((unsigned)ctas), dim3(kThreads), smem, (cudaStream_t)stream, true, a));
  return QUIC_OK;
}
