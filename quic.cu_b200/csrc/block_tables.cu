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
// waits.  Bound: the latency of one launch with two rounds of loads; the bytes are the rows' 12 and their masks'.
#include "common.cuh"

namespace quic {
namespace {

constexpr int kThreads = 256, kMostRequests = 4096;
constexpr int64_t kMostPositions = 1 << 29;

struct TablesArgs {
  int32_t *tables, *held, *pool, *row_start, *positions, *mask;
  int64_t* slot_map;
  const int32_t *lengths, *n_new, *parents;
  int64_t table_row;
  int32_t max_blocks, n_blocks, requests, block_size, mask_words, max_rows, most_rows;
};

__device__ __forceinline__ uint32_t warp_exclusive(uint32_t v, uint32_t& total, int lane) {
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  total = __shfl_sync(0xffffffffu, x, 31);
  return x - v;
}
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
  __shared__ uint32_t part_s[3][kThreads / 32];
  __shared__ unsigned long long rows_s, need_s;
  __shared__ int short_s, many_s, last_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) rows_s = need_s = 0ull, short_s = many_s = 0;
  __syncthreads();

  // ---- the requests' rows and blocks; a thread has `each` of them, one after the other
  const int each = (a.requests + kThreads - 1) / kThreads, b0 = min(tid * each, a.requests), b1 = min(b0 + each, a.requests);
  auto share = [&](int b, uint32_t& take, uint32_t& need, uint32_t& gone, bool& too_long) {
    const int n = a.n_new[b], held = min(max(a.held[b], 0), a.max_blocks);
    take = (uint32_t)max(n, 0);
    gone = n < 0 ? (uint32_t)held : 0u;
    need = 0u;
    too_long = false;
    if (n > 0) {
      const int64_t want = ((int64_t)max(a.lengths[b], 0) + n + a.block_size - 1) / a.block_size;
      too_long = want > a.max_blocks;
      need = want > held ? (uint32_t)(want - held) : 0u;
    }
  };
  uint32_t v[3] = {0u, 0u, 0u};
  unsigned long long rows64 = 0ull, need64 = 0ull;
  for (int b = b0; b < b1; ++b) {
    uint32_t take, need, gone;
    bool too_long;
    share(b, take, need, gone, too_long);
    v[0] += take, v[1] += need, v[2] += gone;  // (sums that wrap belong to calls that are refused)
    rows64 += take, need64 += need;
    if (too_long) short_s = 1;
    if (a.parents != nullptr && take > 32u * (uint32_t)a.mask_words) many_s = 1;
  }
  if (rows64) atomicAdd(&rows_s, rows64);
  if (need64) atomicAdd(&need_s, need64);
  uint32_t base[3], total[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    uint32_t sum;
    base[i] = warp_exclusive(v[i], sum, lane);
    if (lane == 0) part_s[i][warp] = sum;
  }
  __syncthreads();
  const int n_ring = a.n_blocks;
  const int count = min(max(a.pool[1], 0), n_ring), head = n_ring > 0 ? (int)((uint32_t)a.pool[0] % (uint32_t)n_ring) : 0;
  int status = 0;
  if (short_s) status = -1;
  else if (many_s || rows_s > (unsigned long long)a.most_rows) status = -2;
  else if (need_s > (unsigned long long)count) status = (int)min(need_s - count, 0x7fffffffull);
  const bool fine = status == 0;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    total[i] = 0u;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) base[i] += part_s[i][w];
      total[i] += part_s[i][w];
    }
    if (i < 2 && !fine) base[i] = total[i] = 0u;
  }
  for (int b = b0; b < b1; ++b) {
    uint32_t take, need, gone;
    bool too_long;
    share(b, take, need, gone, too_long);
    row0[b] = base[0], new0[b] = base[1], old0[b] = base[2];
    if (fine) base[0] += take, base[1] += need;
    base[2] += gone;
  }
  if (tid == 0) row0[a.requests] = total[0], new0[a.requests] = total[1], old0[a.requests] = total[2];
  __syncthreads();

  // ---- this CTA's share of everything
  const int32_t* const ring = a.pool + 4;
  const int at = blockIdx.x * kThreads + tid, stride = gridDim.x * kThreads;
  for (int b = at; b <= a.requests; b += stride) a.row_start[b] = (int)row0[b];
  auto new_block = [&](uint32_t k) { return ring[((uint32_t)head + k) % (uint32_t)n_ring]; };
  for (uint32_t k = at; k < total[1]; k += stride) {
    const int b = owner(new0, a.requests, k);
    a.tables[b * a.table_row + min(max(a.held[b], 0), a.max_blocks) + (k - new0[b])] = new_block(k);
  }
  for (uint32_t k = at; k < total[2] && n_ring > 0; k += stride) {
    const int b = owner(old0, a.requests, k);
    a.pool[4 + ((uint32_t)head + (uint32_t)count + k) % (uint32_t)n_ring] = a.tables[b * a.table_row + (k - old0[b])];
  }
  for (int row = at; row < a.max_rows; row += stride) {
    if ((uint32_t)row >= total[0]) {
      a.slot_map[row] = -1;
      if (a.parents == nullptr) a.positions[row] = 0;
      continue;
    }
    const int b = owner(row0, a.requests, (uint32_t)row);
    const int place = max(a.lengths[b], 0) + row - (int)row0[b];
    const int j = place / a.block_size, held = min(max(a.held[b], 0), a.max_blocks);
    const int id = j < held ? a.tables[b * a.table_row + j] : new_block(new0[b] + (uint32_t)(j - held));
    a.slot_map[row] = (int64_t)id * a.block_size + (place - j * a.block_size);
    if (a.parents == nullptr) a.positions[row] = place;
  }
  if (a.parents != nullptr) {
    const int64_t words = (int64_t)a.max_rows * a.mask_words;
    for (int64_t i = at; i < words; i += stride) {
      const int row = (int)(i / a.mask_words), w = (int)(i - (int64_t)row * a.mask_words);
      uint32_t bits = 0u;
      int depth = 0;
      if ((uint32_t)row < total[0]) {
        const int b = owner(row0, a.requests, (uint32_t)row), start = (int)row0[b];
        int node = row - start;
        while (true) {  // (each step is to an earlier node)
          if (node >> 5 == w) bits |= 1u << (node & 31);
          const int up = a.parents[start + node];
          if (up < 0 || up >= node) break;
          node = up;
          ++depth;
        }
        depth += max(a.lengths[b], 0);
      }
      a.mask[i] = (int)bits;
      if (w == 0) a.positions[row] = depth;
    }
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
    if (n_ring > 0) a.pool[0] = (int)(((uint32_t)head + total[1]) % (uint32_t)n_ring);
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
                        t->table_row, t->max_blocks, t->n_blocks, requests, t->block_size, mask_words, max_rows,
                        parents != nullptr && t->parent_rows < max_rows ? t->parent_rows : max_rows};
  const int64_t work = (int64_t)max_rows * (parents != nullptr ? mask_words : 1);
  int64_t ctas = (work + 4 * kThreads - 1) / (4 * kThreads);
  ctas = ctas < 1 ? 1 : (ctas > 148 * 4 ? 148 * 4 : ctas);
  const size_t smem = 3 * (size_t)(requests + 1) * 4;
  if (smem > 48000) QUIC_CUDA(allow_smem<block_tables_kernel>(3 * (kMostRequests + 1) * 4));
  QUIC_CUDA(launch(block_tables_kernel, dim3((unsigned)ctas), dim3(kThreads), smem, (cudaStream_t)stream, false, a));
  return QUIC_OK;
}
