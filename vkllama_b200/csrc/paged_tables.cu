// Block tables and slot maps from request lengths, on the device: sequences get from `lengths` to `target` tokens.
//
//   have_i = ceil(length_i / page), want_i = ceil(target_i / page)
//   page j of [want_i, have_i) of sequence i goes back to the pool: entry count + B - k, k = (pages given back by sequences before i)
//     + j - want_i, B all pages given back
//   page j of [have_i, want_i) comes from entry count + B - k, k = (pages taken by sequences before i) + j - have_i
//   new row r of sequence i: position p = length_i + r - starts_i, slot = page of p * page size + p % page size
//
// Taking and giving back are each other's inverse: pages that come and go leave the pool as it was. Pages that are given back in
// a call can be taken in the same call. A call that cannot be carried out whole (pool empty, table full, too few rows) changes
// nothing, gives every row kNoSlot and raises the error word.
//
// One launch. Every CTA scans all sequences for itself (a scan of three counts in shared memory), so that no CTA waits for another; pages and
// rows are then dealt out over the CTAs and find their sequence by bisection. Nothing that a CTA reads is written before the last
// one is through: pages taken are read from entries up to the old count, or straight from the tables of the sequences that give
// them back; entries above the old count are written only, and lengths and count by the CTA that arrives last.
// Bound by latency: one CTA's chain of loads, scan and stores, 6 us on the device for 64 sequences that take a token each as for 256 that take 16,500
// pages (the bytes would take 0.4). A program sees the host's call, 7 us.
#include "common.cuh"
#include "paged.h"

namespace vkl {
namespace {

constexpr uint32_t kThreads = 512, kWarps = kThreads / 32;
constexpr uint32_t kRowsPerCta = 2048, kPagesPerCta = 2048;

struct Counts {
  uint32_t rows, need, give;
};
__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, const Divisor &page) { return tokens ? quotient(tokens - 1, page) + 1 : 0; }

// Sequence of item k: the last i with before[i] <= k (before[0] = 0, ascending, before[n] > k).
__device__ __forceinline__ uint32_t owner(const uint32_t *before, uint32_t n, uint32_t k) {
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (before[mid] <= k) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads) paged_tables_kernel(const PagedTables p) {
  extern __shared__ uint32_t sm[];
  uint32_t *rows_before = sm, *need_before = sm + p.n + 1, *give_before = need_before + p.n + 1;
  __shared__ uint32_t warp_sum_s[3][kWarps];
  __shared__ unsigned long long total_s[3];
  __shared__ uint32_t bad_s, last_s;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  follow();
  stamp_begin(p.stamps);
  const uint32_t count = p.pool[0];
  if (tid == 0) bad_s = 0;
  if (tid < 3) total_s[tid] = 0;
  __syncthreads();

  // totals in 64 bits first: nothing is trusted before it is known that the call can be carried out
  const uint32_t each = (p.n + kThreads - 1) / kThreads, i0 = min(tid * each, p.n), i1 = min(i0 + each, p.n);
  auto counts = [&](uint32_t i, uint32_t &bad) {
    const uint32_t len = p.lengths[i], to = p.target[i];
    if ((len | to) >> 31) bad = PAGED_TABLE_FULL;
    const uint32_t have = pages_of(len, p.page), want = pages_of(to, p.page);
    if (have > p.width || want > p.width) bad = PAGED_TABLE_FULL;
    return Counts{to > len ? to - len : 0, want > have ? want - have : 0, have > want ? have - want : 0};
  };
  Counts mine = {0, 0, 0};
  unsigned long long wide[3] = {0, 0, 0};
  uint32_t bad = 0;
  for (uint32_t i = i0; i < i1; ++i) {
    const Counts c = counts(i, bad);
    mine.rows += c.rows, mine.need += c.need, mine.give += c.give;
    wide[0] += c.rows, wide[1] += c.need, wide[2] += c.give;
  }
  if (bad) bad_s = bad;
  Counts up = mine;  // inclusive scan over the warp
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, up.rows, o), b = __shfl_up_sync(0xffffffffu, up.need, o), c = __shfl_up_sync(0xffffffffu, up.give, o);
    if (lane >= o) up.rows += a, up.need += b, up.give += c;
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) wide[k] += __shfl_xor_sync(0xffffffffu, wide[k], o);
    if (lane == 0 && wide[k]) atomicAdd(&total_s[k], wide[k]);
  }
  if (lane == 31) warp_sum_s[0][warp] = up.rows, warp_sum_s[1][warp] = up.need, warp_sum_s[2][warp] = up.give;
  __syncthreads();
  bad = bad_s;
  if (!bad && total_s[0] > p.rows) bad = PAGED_ROWS;
  if (!bad && p.n && (count > p.capacity || count + total_s[2] > p.capacity)) bad = PAGED_POOL_BAD;
  if (!bad && total_s[1] > count + total_s[2]) bad = PAGED_POOL_EMPTY;
  if (bad) {
    for (uint32_t r = blockIdx.x * kThreads + tid; r < p.rows; r += gridDim.x * kThreads) p.map[r] = kNoSlot, p.map[p.rows + r] = 0;
    if (blockIdx.x == 0) {
      for (uint32_t i = tid; i <= p.n; i += kThreads) p.starts[i] = 0;
      if (tid == 0) raise(p.error, bad);
    }
  } else {
    const uint32_t all_rows = (uint32_t)total_s[0], need = (uint32_t)total_s[1], give = (uint32_t)total_s[2], top = count + give;
    Counts at = {up.rows - mine.rows, up.need - mine.need, up.give - mine.give};
    for (uint32_t w = 0; w < warp; ++w) at.rows += warp_sum_s[0][w], at.need += warp_sum_s[1][w], at.give += warp_sum_s[2][w];
    for (uint32_t i = i0; i < i1; ++i) {
      rows_before[i] = at.rows, need_before[i] = at.need, give_before[i] = at.give;
      if (blockIdx.x == 0) p.starts[i] = at.rows;
      const Counts c = counts(i, bad);
      at.rows += c.rows, at.need += c.need, at.give += c.give;
    }
    if (tid == 0) {
      rows_before[p.n] = all_rows, need_before[p.n] = need, give_before[p.n] = give;
      if (blockIdx.x == 0) p.starts[p.n] = all_rows;
    }
    __syncthreads();
    auto given = [&](uint32_t k) {  // the k-th page that is given back
      const uint32_t i = owner(give_before, p.n, k);
      return p.table[(size_t)i * p.width + pages_of(p.target[i], p.page) + k - give_before[i]];
    };
    auto taken = [&](uint32_t k) {  // the k-th page that is taken
      const uint32_t e = top - k;
      return e <= count ? p.pool[e] : given(top - e);
    };
    const uint32_t t0 = blockIdx.x * kThreads + tid, step = gridDim.x * kThreads;
    for (uint32_t k = t0; k < give; k += step) p.pool[top - k] = given(k);
    for (uint32_t k = t0; k < need; k += step) {
      const uint32_t i = owner(need_before, p.n, k);
      p.table[(size_t)i * p.width + pages_of(p.lengths[i], p.page) + k - need_before[i]] = taken(k);
    }
    for (uint32_t r4 = t0 * 4; r4 < p.rows; r4 += step * 4) {  // four rows: one bisection, mostly one page
      uint32_t i = 0, next = 0, len = 0, have = 0, j_at = 0xffffffffu, page = 0;
      if (r4 < all_rows) i = owner(rows_before, p.n, r4);
#pragma unroll
      for (uint32_t r = r4; r < r4 + 4; ++r) {
        if (r >= p.rows) break;
        uint32_t slot = kNoSlot, pos = 0;
        if (r < all_rows) {
          if (r == r4 || r >= next) {
            while (r >= rows_before[i + 1]) ++i;
            next = rows_before[i + 1];
            len = p.lengths[i];
            have = pages_of(len, p.page);
            j_at = 0xffffffffu;
          }
          pos = len + r - rows_before[i];
          const uint32_t j = quotient(pos, p.page);
          if (j != j_at) page = j < have ? p.table[(size_t)i * p.width + j] : taken(need_before[i] + j - have);
          j_at = j;
          const unsigned long long s = (unsigned long long)page * p.page.d + (pos - j * p.page.d);
          if (s < kNoSlot) slot = (uint32_t)s;
          else raise(p.error, PAGED_BAD_PAGE);
        }
        p.map[r] = slot;
        p.map[p.rows + r] = pos;
      }
    }
  }

  bool last = true;
  if (gridDim.x > 1) {
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      const uint32_t a = atomicAdd(p.arrived, 1u);
      last_s = a + 1 == gridDim.x;
      if (last_s) *p.arrived = 0;
    }
    __syncthreads();
    last = last_s;
  } else {
    __syncthreads();
  }
  if (!last) return;
  stamp_end(p.stamps);
  if (bad) return;
  if (tid == 0 && p.n) p.pool[0] = count + (uint32_t)total_s[2] - (uint32_t)total_s[1];
  for (uint32_t i = i0; i < i1; ++i) p.lengths[i] = p.target[i];
}

size_t tables_smem(uint32_t n) { return (size_t)3 * (n + 1) * 4; }

}  // namespace

cudaError_t setup_paged_tables() {
  return cudaFuncSetAttribute(paged_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)tables_smem(kTablesMaxSequences));
}
cudaError_t launch_paged_tables(const PagedTables &p, uint32_t sms, cudaStream_t s) {
  // Pages that come back are not known here: at most what the tables, and the pool, can hold.
  const uint64_t pages = (uint64_t)p.n * p.width < p.capacity ? (uint64_t)p.n * p.width : p.capacity;
  const uint64_t ctas = ((uint64_t)p.rows + kRowsPerCta - 1) / kRowsPerCta, more = pages / kPagesPerCta;
  uint64_t grid = ctas > more ? ctas : more;
  grid = grid < 1 ? 1 : grid > sms ? sms : grid;
  return launch_following(paged_tables_kernel, dim3((uint32_t)grid), kThreads, tables_smem(p.n), s, p);
}

}  // namespace vkl
