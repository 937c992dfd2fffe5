// What the kernels for several new rows per sequence share: which rows a tile has, and a row computed by itself.
#pragma once
#include "common.cuh"
#include "paged.h"
#include "paged_value.cuh"

namespace vkl {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// A tile of packed rows: which sequence, and its rows.
struct Place {
  uint32_t seq, row0, fresh, len;  // first row of the sequence in q, its new rows, its length
  uint32_t first;                  // first packed row of the tile
};

// Rows of sequence i, 0 where starts, lengths and table do not belong together.
__device__ __forceinline__ uint32_t fresh_rows(const PagedAttention &p, uint32_t i, bool &bad) {
  const uint32_t a = p.starts[i], b = p.starts[i + 1], len = p.lengths[i];
  if (a <= b && b <= p.rows && b - a <= len && len <= p.width * p.page.d) return b - a;
  bad = true;
  return 0;
}

// Which kernel takes a sequence: tcgen05 (part 2) where it has more packed rows than a tile of the other, or a tile of 128 positions to see; the tiles of
// 64 rows on mma.sync (part 1), three CTAs to an SM, else. us, 32 heads of 128, mma.sync / tcgen05: 64 prompts of 32 52 / 65, of 64 67 / 65, of 96
// 119 / 67; 8 prompts of 64 12.3 / 14.4, of 80 22.4 / 14.5; 64 drafts of 2 rows behind 100 63 / 72, behind 400 150 / 128; 8 drafts of 5, 8 key heads,
// behind 100 10.9 / 9.3, behind 600 28.7 / 16.5.
constexpr uint32_t kTensorRows = 65, kTensorLength = 128;
__device__ __forceinline__ uint32_t rows_here(const PagedAttention &p, uint32_t i, uint32_t per, bool &bad) {
  const uint32_t fresh = fresh_rows(p, i, bad);
  if (p.part == 0) return fresh;
  const bool tensor = (uint64_t)fresh * per >= kTensorRows || p.lengths[i] >= kTensorLength;
  return tensor == (p.part == 2) ? fresh : 0;
}

// The place of tile `index` when every sequence has ceil(new * per / rows) of them, by one warp; false beyond the last. What takes longest
// comes first: a sequence's last tiles, which see most, and of up to 32 sequences the longest. A later search for a tile further on goes on where
// this one ended.
struct Walk {
  uint32_t from = 0;    // sequences in front, a multiple of 32
  uint64_t before = 0;  // their tiles
};
__device__ __forceinline__ bool find_tile(const PagedAttention &p, uint32_t per, uint32_t rows, uint32_t index, Place &at, Walk &walk) {
  const uint32_t lane = threadIdx.x & 31;
  bool bad = false;
  uint64_t &before = walk.before;
  for (uint32_t &i0 = walk.from; i0 < p.n; i0 += 32) {
    const uint32_t i = i0 + lane, fresh = i < p.n ? rows_here(p, i, per, bad) : 0;
    const uint64_t mine = ((uint64_t)fresh * per + rows - 1) / rows;
    uint64_t up = mine;  // and all of the chunk's sequences that come before
    if (p.n <= 32) {
      const uint32_t len = fresh ? p.lengths[i] : 0;
      for (uint32_t x = 0; x < p.n; ++x) {
        const uint32_t other = __shfl_sync(0xffffffffu, len, x);
        const uint64_t its = __shfl_sync(0xffffffffu, mine, x);
        if (other > len || (other == len && x < lane)) up += its;
      }
    } else {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t a = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += a;
      }
    }
    const uint32_t it = __ballot_sync(0xffffffffu, before + up > index && before + up - mine <= index);
    if (it) {
      const uint32_t x = __ffs(it) - 1;
      at.seq = i0 + x;
      at.fresh = __shfl_sync(0xffffffffu, fresh, x);
      at.first = ((uint32_t)(__shfl_sync(0xffffffffu, before + up, x) - index) - 1) * rows;
      at.row0 = p.starts[at.seq];
      at.len = p.lengths[at.seq];
      return true;
    }
    if (p.n > 32) before += __shfl_sync(0xffffffffu, up, 31);
  }
  return false;
}
// Starts and lengths that do not belong together are reported by the first CTA's first warp.
__device__ __forceinline__ void check_rows(const PagedAttention &p) {
  bool bad = false;
  for (uint32_t i = threadIdx.x & 31; i < p.n; i += 32) fresh_rows(p, i, bad);
  if (bad) raise(p.error, PAGED_BAD_ROWS);
}

// Dimensions [d0, d1) of one packed row by a warp, from the definition in fp32. In the tiles' second product a position that a row does not see has the
// probability 0, and 0 times an infinity or a NaN in that position's value is NaN: rows that come out of it not finite are computed
// again here, from the positions that they see. (So a value that is not finite costs time, and reaches only the rows that see it.)
template <bool BF> __device__ __noinline__ void row_again(const PagedAttention &p, const Place &at, uint32_t kvh, uint32_t packed, uint32_t d0, uint32_t d1) {
  const uint32_t lane = threadIdx.x & 31, per = p.heads / p.kv_heads, t = packed / per, h = kvh * per + packed - t * per;
  const uint32_t pos = at.len - at.fresh + t, first = p.window && pos + 1 > p.window ? pos + 1 - p.window : 0;
  const uint16_t *q = static_cast<const uint16_t *>(p.q) + (at.row0 + t) * p.q_ld + h * p.dim;
  const uint16_t *k = static_cast<const uint16_t *>(p.kcache), *v = static_cast<const uint16_t *>(p.vcache);
  float m = -INFINITY, l = 0.f;
  float2 o[4] = {};  // dimensions lane * 2 + 64 i
  for (uint32_t j0 = first; j0 <= pos; j0 += 32) {
    const uint32_t j = j0 + lane;
    bool there = j <= pos;
    size_t row = 0;
    float s = -INFINITY;
    if (there) {
      const uint32_t n = quotient(j, p.page), page = p.table[(size_t)at.seq * p.width + n];
      there = page < p.pages;
      if (there) {
        row = ((size_t)page * p.kv_heads + kvh) * p.page.d + j - n * p.page.d;
        s = 0.f;
        for (uint32_t d = 0; d < p.dim; d += 2) {
          const float2 a = unpack2<BF>(*reinterpret_cast<const uint32_t *>(q + d)), b = unpack2<BF>(*reinterpret_cast<const uint32_t *>(k + row * p.dim + d));
          s = fmaf(a.x, b.x, s);
          s = fmaf(a.y, b.y, s);
        }
        s *= p.scale * kLog2e;
      }
    }
    const float now = fmaxf(m, warp_max(s)), ref = now == -INFINITY ? 0.f : now, c = exp2f(m - ref);
    const float w = there ? exp2f(s - ref) : 0.f;
    m = now;
    l = l * c + warp_sum(w);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i].x *= c, o[i].y *= c;
    const uint32_t all = __ballot_sync(0xffffffffu, there);
    for (uint32_t x = 0; x < 32; ++x) {
      if (!(all >> x & 1)) continue;
      const float wx = __shfl_sync(0xffffffffu, w, x);
      const size_t rx = __shfl_sync(0xffffffffu, (unsigned long long)row, x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t d = lane * 2 + 64 * i;
        if (d < p.dim) {
          const float2 b = unpack2<BF>(*reinterpret_cast<const uint32_t *>(v + rx * p.dim + d));
          o[i].x = fmaf(wx, b.x, o[i].x);
          o[i].y = fmaf(wx, b.y, o[i].y);
        }
      }
    }
  }
  const float r = 1.0f / l;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t d = lane * 2 + 64 * i;
    if (d >= d0 && d < d1 && d < p.dim) *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(p.out) + ((size_t)(at.row0 + t) * p.heads + h) * p.dim + d) = pack2<BF>(o[i].x * r, o[i].y * r);
  }
}

}  // namespace
}  // namespace vkl
