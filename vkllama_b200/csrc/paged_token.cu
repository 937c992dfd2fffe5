// Attention of one new token per sequence over a paged cache:
//   out = sum_j softmax_j(scale q.k_j) v_j over the positions max(0, length - window) <= j < length.
//
// Every visible key and value is read once for all query heads of its group (sixteen of them at a time), so HBM bounds it: 4 dim bytes a
// position and key head. The products run on mma.sync (m16n8k16, fp32 sums) because a group's queries share the fragments: its query
// heads are the rows of A, cached rows the columns. Probabilities go into the second product as two 16-bit numbers, p = hi + lo, both
// products exact: relative 2^-16 in bfloat16, 2^-22 in fp16 (half steps of two numbers). fp16 ends at steps of 2^-24, so its probabilities
// are 2^14 times as large, in sums and outputs alike: they keep 2^-22 down to 2^-17 of the row's largest, an output's 2^-11 down to 2^-28, and below each is off by
// 2^-39 of the largest. (As they are, thousands of positions below 2^-25 counted in the sum and not in the output: with one position that outweighs
// 4000 others by 20 nats and has the value 0, nothing was left.) Up to eight heads lo has the upper eight rows of A, which would be empty, and costs
// nothing; beyond, a second product with the same fragment of V.
//
// Work is cut into equal shares, not by sequence: the tiles (of 16 or 32 positions) of all (sequence, head group) pairs stand in one row, with
// a place more for each pair's own cost; every CTA takes a range of it and every warp of the CTA a range of that, however the lengths are spread. Ranges cut pairs: a warp keeps
// running maximum, sum and output of its part; parts meet in shared memory, and those of several CTAs in scratch, where the CTA that
// arrives last adds them up in their order, many of them in two steps (the result does not depend on who that is). Cuts that would leave a small piece of a pair are
// moved to its border.
//
// A warp streams its range through a ring of its own (cp.async, tiles of keys and of values alternating, swizzled for ldmatrix):
// no barrier inside the stream, the next pages are looked up a tile ahead. Maximum and sum run along in one pass (Milakov and Gimelshein, Online normalizer
// calculation for softmax, 2018). Rows that are not visible are not read and count as zeros.
//
// Measured on sequences that hold 0.37 GB together (57 us at the rate of a copy): 70 ... 78 us, 4.9 ... 5.3 TB/s, with up to eight heads to a
// key head whatever the width, the page and the lengths; 76 us with 12 or 16 heads of 128, 93 us with 16 of 256 (shared memory and the
// products are the limit there), 117 us with 32 on one key head, which reads everything twice. What is left up to eight heads is the
// machine's: under full load groups of SMs take 12 % longer for the same bytes, and shares are fixed before anyone knows which.
#include <algorithm>

#include "common.cuh"
#include "paged.h"
#include "paged_rows.cuh"
#include "paged_value.cuh"

namespace vkl {
namespace {

constexpr uint32_t kShareRows = 256;          // a CTA's share is at least this many positions
// A cut this near to a pair's border moves there. A cut costs some 5 us at the end (the parts of several CTAs meet in L2); a tile of 32 more
// for one CTA costs 0.4 us where HBM is the limit, and an eighth of 1 us where the whole call is short.
constexpr uint32_t kSnapRows = 256, kSnapRowsShort = 512, kShortRows = 1024;
// Where a tile has more products (sixteen heads, or heads above 128), shorter pieces are worth their cut. us, these three as above and as below: one sequence of 1151
// positions, 32 heads of 128 on 2 key heads, 21.8 and 14.9; three of 2500, 16 heads of 256 on one, 35 and 26; four of 2000, 16 of 256 on 2, 26 and 19.
constexpr uint32_t kWideRows = 128, kSnapRowsShort256 = 256;
// Parts of a pair that one CTA adds up, and how many it does at a time; of more, every kGroup are added up first (one sequence of 60,000 positions, 16 heads of 128
// on one key head, 148 parts: 55 us by one CTA, this way 26).
constexpr uint32_t kJoin = 32, kGroup = 16, kAtOnce = 8;
constexpr uint32_t kPairCost = 1;             // what a pair costs beside its tiles (queries, output, short rows in the ring), in tiles
constexpr float kRaise = 14.f;                // fp16 probabilities are 2^14 times as large; 2^16 is left for one that its exponent's rounding takes above 1

// DP: padded head width. WIDE: sixteen query heads in the rows of A; else eight, and the low parts of their probabilities in the others.
template <int DP, bool WIDE> struct Cfg {
  static constexpr uint32_t kWarps = DP == 256 && WIDE ? 6 : 8, kThreads = kWarps * 32;
  static constexpr uint32_t kTile = DP == 64 || (DP == 128 && !WIDE) ? 32 : 16;  // positions of a tile
  static constexpr uint32_t kHalf = kTile * DP * 2;                            // bytes of a tile's keys, or values
  static constexpr uint32_t kRing = DP == 64 ? 5 : DP == 128 ? (WIDE ? 4 : 3) : 2;
  static constexpr uint32_t kHeads = WIDE ? 16 : 8;
  static constexpr uint32_t kStash = kHeads * DP * 4;  // a warp's first part, where its range goes on behind it
  static constexpr uint32_t kSmem = kWarps * (kRing * kHalf + kStash + 2 * kHeads * 2 * 4);
  static constexpr uint32_t kShare = (WIDE ? kWideRows : kShareRows) / kTile, kSnap = (WIDE ? kWideRows : kSnapRows) / kTile;
  static constexpr uint32_t kSnapShort = (WIDE ? kWideRows : DP == 256 ? kSnapRowsShort256 : kSnapRowsShort) / kTile, kShort = kShortRows / kTile;
  static_assert(kSmem + 2048 <= 227 * 1024, "shared memory of an SM");
  static_assert(kRing * kHalf >= kStash, "a warp's last part lies in its ring");
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Pair {        // tiles t .. t1 of a sequence and head group
  uint32_t seq, grp;
  uint32_t t, t0, t1;
  uint32_t len, first;  // visible positions
  uint32_t place;       // of tile t in the row of all work
};

// One record per part of a pair that ends inside a CTA.
struct Part {
  uint32_t seq, grp;
  uint8_t there, begins, ends;  // the pair begins, ends in this part
};

template <bool BF, int DP, bool WIDE> __global__ void __launch_bounds__(Cfg<DP, WIDE>::kThreads, 1) paged_token_kernel(const PagedAttention p) {
  using C = Cfg<DP, WIDE>;
  constexpr uint32_t kWarps = C::kWarps, kThreads = C::kThreads;
  constexpr int NR = WIDE ? 2 : 1;           // query heads of a thread's fragments: rows g (and g + 8)
  constexpr uint32_t CH = DP / 8;            // 16-byte pieces of a row
  constexpr uint32_t T = C::kTile, NC = T * CH / 32;  // pieces of a half and lane
  constexpr int KS = DP / 16, NT = DP / 8, SN = T / 8;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ uint32_t before_s[kThreads + 1];  // tiles of one head group's sequences, which fit 31 bits over all groups (the host knows, or p.count)
  __shared__ uint32_t warp_sum_s[kWarps];
  __shared__ uint32_t border_s[2], cut_s[2][2];  // the range's ends, and the first and last cut of the pairs that they cut
  __shared__ Part part_s[kWarps][2];
  __shared__ uint32_t last_s[2];
  unsigned char *ring = smem + threadIdx.x / 32 * C::kRing * C::kHalf;
  float *stash = reinterpret_cast<float *>(smem + kWarps * C::kRing * C::kHalf);       // [warp][head][DP]
  float *ml = reinterpret_cast<float *>(smem + kWarps * (C::kRing * C::kHalf + C::kStash));  // [warp][2][head][2]
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const uint32_t per = p.heads / p.kv_heads, groups = (per + C::kHeads - 1) / C::kHeads, pairs = p.kv_heads * groups;
  const float scale = fabsf(p.scale) * kLog2e;  // maxima are of the plain products; a negative scale turns the queries round
  const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
  const uint32_t room = p.width * p.page.d;  // positions that a table holds (checked by the host to fit 31 bits)

  follow();
  stamp_begin(p.stamps);
  // ---- where this CTA's and this warp's range is ----
  auto length = [&](uint32_t i) { return min(p.lengths[i], room); };
  auto first_of = [&](uint32_t len) { return p.window && len > p.window ? len - p.window : 0u; };
  // A pair's tiles, and the places that it takes up in the row of all work.
  auto tiles = [&](uint32_t len) { return max((len + T - 1) / T, 1u) - first_of(len) / T; };
  auto places = [&](uint32_t len) { return tiles(len) + kPairCost; };
  if (p.count) {
    __shared__ unsigned long long all_s;
    if (tid == 0) all_s = 0;
    __syncthreads();
    unsigned long long all = 0;
    for (uint32_t i = tid; i < p.n; i += kThreads) all += places(length(i));
    atomicAdd(&all_s, all);
    __syncthreads();
    if (all_s > 0x7fffffffu / pairs) {
      if (blockIdx.x == 0 && tid == 0) raise(p.error, PAGED_TOO_MUCH);
      return;
    }
  }
  const uint32_t each = (p.n + kThreads - 1) / kThreads;
  {
    const uint32_t i0 = min(tid * each, p.n), i1 = min(i0 + each, p.n);
    uint32_t mine = 0;
    for (uint32_t i = i0; i < i1; ++i) {
      if (p.lengths[i] > room && blockIdx.x == 0) raise(p.error, PAGED_TABLE_FULL);
      mine += places(length(i));
    }
    uint32_t up = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t a = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += a;
    }
    if (lane == 31) warp_sum_s[warp] = up;
    if (tid < kWarps * 2) part_s[tid >> 1][tid & 1].there = 0;
    __syncthreads();
    uint32_t base = 0;
    for (uint32_t w = 0; w < warp; ++w) base += warp_sum_s[w];
    before_s[tid] = base + up - mine;
    if (tid == kThreads - 1) before_s[kThreads] = base + up;
    __syncthreads();
  }
  const uint32_t total = before_s[kThreads] * pairs, share = max((total + gridDim.x - 1) / gridDim.x, C::kShare);
  const uint32_t snap = share <= C::kShort ? C::kSnapShort : C::kSnap;
  auto find = [&](uint32_t pos) {  // by a warp: the pair at place pos < total; t may lie behind its last tile, in the place that stands for its cost
    uint32_t m = __ballot_sync(0xffffffffu, before_s[lane * kWarps] * pairs <= pos);
    uint32_t lo = (31 - __clz(m)) * kWarps;
    m = __ballot_sync(0xffffffffu, lane < kWarps && before_s[lo + min(lane, kWarps - 1)] * pairs <= pos);
    lo += 31 - __clz(m);
    Pair r;
    r.place = pos;
    r.seq = lo * each;
    uint32_t left = pos - before_s[lo] * pairs, len = length(r.seq), n = places(len);
    while (left >= n * pairs) {
      left -= n * pairs;
      len = length(++r.seq);
      n = places(len);
    }
    r.grp = left / n;
    r.len = len;
    r.first = first_of(len);
    r.t0 = r.first / T;
    r.t1 = r.t0 + n - kPairCost;
    r.t = r.t0 + left - r.grp * n;
    return r;
  };
  if (warp < 2) {  // the range's ends
    uint32_t b = min((uint64_t)(blockIdx.x + warp) * share, (uint64_t)total);
    if (b > 0 && b < total) {
      const Pair r = find(b);
      const uint32_t in = r.t - r.t0, out = r.t1 + kPairCost - r.t, begin = b - in;
      if (min(in, out) <= snap) {
        b = in <= out ? begin : b + out;
      } else if (lane == 0) {  // all cuts of the pair: multiples of the share further than `snap` inside it
        cut_s[warp][0] = (begin + snap) / share + 1;
        cut_s[warp][1] = (begin + in + out - snap - 1) / share;
      }
    }
    if (lane == 0) border_s[warp] = b;
  }
  __syncthreads();
  const uint32_t b0 = border_s[0], b1 = border_s[1];
  if (b0 == b1) return;
  // a warp's places
  const uint32_t part = (b1 - b0) / kWarps, more = (b1 - b0) % kWarps;
  const uint32_t w0 = b0 + part * warp + min(warp, more), w1 = w0 + part + (warp < more);

  auto advance = [&](Pair &r) {
    ++r.place;
    if (++r.t < r.t1) return;
    r.place += kPairCost;
    if (++r.grp == pairs) {
      r.grp = 0;
      if (++r.seq >= p.n) return;
      r.len = length(r.seq);
      r.first = first_of(r.len);
      r.t0 = r.first / T;
      r.t1 = r.t0 + tiles(r.len);
    }
    r.t = r.t0;
  };
  auto write_out = [&](uint32_t seq, uint32_t head, uint32_t d, float a, float b) {
    if (d < p.dim) *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(p.out) + ((size_t)seq * p.heads + head) * p.dim + d) = pack2<BF>(a, b);
  };
  // A row that is not finite, from the definition (paged_rows.cuh): a value that is not may have met a part of a probability that is 0.
  auto redo = [&](uint32_t seq, uint32_t head) {
    const Place one = {seq, seq, 1, length(seq), 0};
    const uint32_t kvh = head / per;
    row_again<BF>(p, one, kvh, head - kvh * per, 0, DP);
  };
  auto first_head = [&](uint32_t grp) { return grp / groups * per + grp % groups * C::kHeads; };
  auto heads_of = [&](uint32_t grp) { return min(per - grp % groups * C::kHeads, C::kHeads); };

  Pair at = {};
  at.place = w1;
  if (w0 < w1) {
    at = find(w0);
    if (at.t >= at.t1) {  // the range begins behind a pair's last tile
      at.place += at.t1 + kPairCost - at.t - 1 - kPairCost;
      at.t = at.t1 - 1;
      advance(at);
    }
  }
  if (at.place < w1) {
    // ---- the stream: tile halves, keys and values in turn, go into the ring's places one after the other ----
    Pair in = at;  // the tile whose page has been looked up
    uint32_t entry = 0, in_page = 0, row_at = 0xffffffffu, slot_in = 0;
    bool values = false, whole = false;
    const uint32_t ring_a = smem_addr(ring);
    auto look_up = [&]() {  // the page of this lane's position of the tile that comes next
      const uint32_t j = in.t * T + lane % T;
      entry = kNoSlot;
      if (j >= in.first && j < in.len) {
        const uint32_t n = quotient(j, p.page);
        entry = p.table[(size_t)in.seq * p.width + n];
        in_page = j - n * p.page.d;
      }
    };
    look_up();
    // Pieces of a half: lane l has piece l % CH of row l / CH of every 32 / CH rows. Piece c of row r lies at piece c ^ (r % 8), and what
    // that exclusive-or takes from i is the same for every lane.
    constexpr uint32_t RS = 32 / CH;
    const uint32_t col = lane % CH, prow = lane / CH;
    const bool col_there = col * 8 < p.dim;
    const uint32_t piece = prow * CH * 16 + ((col ^ prow) << 4);
    const uint64_t step = (uint64_t)RS * p.dim * 2;
    const bool runs = p.page.d % 8 == 0;  // eight rows from a multiple of eight on follow each other in a page
    auto request = [&]() {
      if (values || in.place < w1) {
        if (!values) {
          row_at = 0xffffffffu;
          if (entry < p.pages) row_at = (entry * p.kv_heads + in.grp / groups) * p.page.d + in_page;  // the host has checked that rows fit 32 bits
          else if (entry != kNoSlot) raise(p.error, PAGED_BAD_PAGE);
          whole = runs && in.t * T >= in.first && in.t * T + T <= in.len && __all_sync(0xffffffffu, entry < p.pages);
          advance(in);
          if (in.place < w1) look_up();
        }
        const uint8_t *cache = static_cast<const uint8_t *>(values ? p.vcache : p.kcache);
        const uint32_t dst = ring_a + slot_in * C::kHalf + piece;
        if (whole) {
#pragma unroll
          for (uint32_t h = 0; h < T / 8; ++h) {
            const uint32_t r = __shfl_sync(0xffffffffu, row_at, h * 8);
            const uint8_t *src = cache + ((size_t)(r + prow) * p.dim + (col_there ? col * 8 : 0)) * 2;
#pragma unroll
            for (uint32_t i = h * 8 / RS; i < (h + 1) * 8 / RS; ++i, src += step) copy16((dst ^ (i * RS % 8) << 4) + i * 512, src, col_there);
          }
        } else {
#pragma unroll
          for (uint32_t i = 0; i < NC; ++i) {
            const uint32_t r = __shfl_sync(0xffffffffu, row_at, i * RS + prow);
            const bool there = r != 0xffffffffu && col_there;
            copy16((dst ^ (i * RS % 8) << 4) + i * 512, there ? cache + ((size_t)r * p.dim + col * 8) * 2 : cache, there);
          }
        }
        values = !values;
        slot_in = slot_in + 1 == C::kRing ? 0 : slot_in + 1;
      }
      copy_commit();  // one group per place, also when it is empty
    };
#pragma unroll 1
    for (uint32_t i = 0; i < C::kRing; ++i) request();

    // ---- the sums of the current pair: rows g of every group of eight heads; o's second half holds the low parts ----
    float o[NT][4], mx[NR], sum[NR];
    uint32_t q[KS][2 * NR];
    uint32_t slot = 0;
    bool begins = at.t == at.t0;
    auto start_pair = [&]() {
      const uint32_t h0 = first_head(at.grp), nh = heads_of(at.grp);
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        // every load first, whether its number exists or not: under conditions they waited for one another (sixteen heads of 192: 5.5 us)
        const uint16_t *src = static_cast<const uint16_t *>(p.q) + at.seq * p.q_ld + (h0 + min(r * 8 + g, nh - 1)) * p.dim;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) q[k][e * NR + r] = *reinterpret_cast<const uint32_t *>(src + min(k * 16 + e * 8 + t4 * 2, p.dim - 2));
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) q[k][e * NR + r] = r * 8 + g < nh && k * 16 + e * 8 + t4 * 2 < p.dim ? q[k][e * NR + r] ^ flip : 0u;
        mx[r] = -INFINITY;
        sum[r] = 0.f;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
    };
    // Output e of row r of a pair of dimensions. High and low part lie apart in the narrow form; an infinite high part has no low one (its
    // product there is 0 times infinity).
    auto result = [&](int n, int r, int e) {
      if constexpr (WIDE) return o[n][2 * r + e];
      else return fabsf(o[n][e]) < INFINITY ? o[n][e] + o[n][2 + e] : o[n][e];
    };
    auto keep = [&](float *to, float *to_ml) {  // this part for the ones that join it
#pragma unroll
      for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int n = 0; n < NT; ++n) *reinterpret_cast<float2 *>(to + (r * 8 + g) * DP + n * 8 + t4 * 2) = make_float2(result(n, r, 0), result(n, r, 1));
        if (t4 == 0) to_ml[(r * 8 + g) * 2] = mx[r], to_ml[(r * 8 + g) * 2 + 1] = sum[r];
      }
    };
    start_pair();
    const uint32_t lrow = lane & 7, lsel = lane >> 3;  // ldmatrix: row of a matrix, which of the four
    const uint32_t k_at = (lrow + (lsel >> 1) * 8) * CH * 16 + (((lsel & 1) ^ lrow) << 4);
    const uint32_t v_at = (lrow + (lsel & 1) * 8) * CH * 16 + (((lsel >> 1) ^ lrow) << 4);
#pragma unroll 1
    for (;;) {
      copy_wait<C::kRing - 1>();
      __syncwarp();
      // S = Q K^T: matrices (rows 0-7 | 8-15) x (k low | k high)
      float s[SN][4] = {};
      {
        const uint32_t kt = ring_a + slot * C::kHalf + k_at;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int n = 0; n < SN; n += 2) {
            uint32_t b[4];
            ldmatrix4(b, (kt ^ k << 5) + n * 8 * CH * 16);
            mma2<BF>(s[n], q[k][0], WIDE ? q[k][1] : 0, q[k][NR], WIDE ? q[k][2 * NR - 1] : 0, b[0], b[1]);
            mma2<BF>(s[n + 1], q[k][0], WIDE ? q[k][1] : 0, q[k][NR], WIDE ? q[k][2 * NR - 1] : 0, b[2], b[3]);
          }
      }
      slot = slot + 1 == C::kRing ? 0 : slot + 1;
      __syncwarp();
      request();
      // softmax so far
      if (at.t * T < at.first || at.t * T + T > at.len) {
#pragma unroll
        for (int n = 0; n < SN; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t j = at.t * T + n * 8 + t4 * 2 + e;
            if (j < at.first || j >= at.len) {
#pragma unroll
              for (int r = 0; r < NR; ++r) s[n][2 * r + e] = -INFINITY;
            }
          }
      }
      uint32_t hi[SN][NR], lo[SN][NR];  // the probabilities' high and low parts
      bool grown = false;
      float ref[NR], top[NR];
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        top[r] = mx[r];
#pragma unroll
        for (int n = 0; n < SN; ++n) top[r] = fmaxf(top[r], fmaxf(s[n][2 * r], s[n][2 * r + 1]));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
        ref[r] = top[r] == -INFINITY ? 0.f : top[r] * scale;
        grown |= top[r] != mx[r];
      }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float c = exp2_fast(mx[r] * scale - ref[r]);
          sum[r] *= c;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            o[n][2 * r] *= c, o[n][2 * r + 1] *= c;
            if constexpr (!WIDE) o[n][2] *= c, o[n][3] *= c;
          }
          mx[r] = top[r];
        }
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float raise = BF ? -ref[r] : kRaise - ref[r];
#pragma unroll
        for (int n = 0; n < SN; ++n) {
          const float a = exp2_fast(fmaf(s[n][2 * r], scale, raise)), b = exp2_fast(fmaf(s[n][2 * r + 1], scale, raise));
          sum[r] += a + b;
          hi[n][r] = pack2<BF>(a, b);
          const float2 h = unpack2<BF>(hi[n][r]);
          lo[n][r] = pack2<BF>(a - h.x, b - h.y);
        }
      }
      copy_wait<C::kRing - 1>();
      __syncwarp();
      {
        const uint32_t vt = ring_a + slot * C::kHalf + v_at;
#pragma unroll
        for (int k = 0; k < SN; k += 2)
#pragma unroll
          for (int n = 0; n < NT; n += 2) {
            uint32_t b[4];
            ldmatrix4_t(b, (vt ^ n << 4) + k * 8 * CH * 16);
            if constexpr (WIDE) {
              mma2<BF>(o[n], hi[k][0], hi[k][1], hi[k + 1][0], hi[k + 1][1], b[0], b[1]);
              mma2<BF>(o[n + 1], hi[k][0], hi[k][1], hi[k + 1][0], hi[k + 1][1], b[2], b[3]);
              mma2<BF>(o[n], lo[k][0], lo[k][1], lo[k + 1][0], lo[k + 1][1], b[0], b[1]);
              mma2<BF>(o[n + 1], lo[k][0], lo[k][1], lo[k + 1][0], lo[k + 1][1], b[2], b[3]);
            } else {
              mma2<BF>(o[n], hi[k][0], lo[k][0], hi[k + 1][0], lo[k + 1][0], b[0], b[1]);
              mma2<BF>(o[n + 1], hi[k][0], lo[k][0], hi[k + 1][0], lo[k + 1][0], b[2], b[3]);
            }
          }
      }
      slot = slot + 1 == C::kRing ? 0 : slot + 1;
      __syncwarp();
      request();

      const bool ends = at.t + 1 == at.t1, over = at.place + 1 + (ends ? kPairCost : 0) >= w1;
      if (!ends && !over) {
        ++at.t;
        ++at.place;
        continue;
      }
      // a part is complete
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
      }
      if (begins && ends) {
        const uint32_t h0 = first_head(at.grp), nh = heads_of(at.grp);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float inv = at.len ? 1.0f / sum[r] : 0.f;  // nothing visible: zeros
          float finite = 0.f;
          if (r * 8 + g < nh) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const float a = result(n, r, 0) * inv, b = result(n, r, 1) * inv;
              finite += a * 0.f + b * 0.f;
              write_out(at.seq, h0 + r * 8 + g, n * 8 + t4 * 2, a, b);
            }
          }
          uint32_t again = __ballot_sync(0xffffffffu, finite != 0.f);  // NaN
          __syncwarp();
#pragma unroll 1
          while (again) {
            const uint32_t x = (__ffs(again) - 1) / 4;
            redo(at.seq, h0 + r * 8 + x);
            again &= ~(15u << (x * 4));
          }
        }
      } else {
        if (lane == 0) part_s[warp][over] = {at.seq, at.grp, 1, begins, ends};
        float *to = stash + warp * (C::kStash / 4);
        if (over) {
          copy_wait<0>();
          __syncwarp();
          to = reinterpret_cast<float *>(ring);
        }
        keep(to, ml + (warp * 2 + over) * C::kHeads * 2);
      }
      if (over) break;
      advance(at);
      start_pair();
      begins = true;
    }
    copy_wait<0>();
  }
  __syncthreads();

  // ---- parts meet. They stand in order (warp by warp, a warp's first before its last); a run of them is one pair. ----
  auto part_o = [&](uint32_t i) { return (i & 1) ? reinterpret_cast<const float *>(smem + (i >> 1) * C::kRing * C::kHalf) : stash + (i >> 1) * (C::kStash / 4); };
  float *scratch_o = p.scratch, *scratch_ml = p.scratch + (size_t)gridDim.x * 2 * C::kHeads * DP;
  uint32_t run = 0, open_there = 0;
  uint32_t open_seq[2] = {}, open_grp[2] = {};  // the CTA's pairs that began before it (0), end behind it (1)
  const Part mine = part_s[min(lane >> 1, kWarps - 1)][lane & 1];
  const uint32_t all_there = __ballot_sync(0xffffffffu, lane < 2 * kWarps && mine.there), all_begin = __ballot_sync(0xffffffffu, mine.begins);
  const uint32_t all_end = __ballot_sync(0xffffffffu, lane < 2 * kWarps && mine.there && mine.ends);
  for (uint32_t rest = all_there; rest; ++run) {
    const uint32_t i = __ffs(rest) - 1, end = all_end & -(1u << i), in_run = rest & (end ? (2u << (__ffs(end) - 1)) - 1 : 0xffffu);
    rest &= ~in_run;
    const bool begins = all_begin >> i & 1, whole = begins && end;
    const uint32_t side = begins ? 1 : 0;  // where it goes in scratch
    const uint32_t seq = __shfl_sync(0xffffffffu, mine.seq, i), grp = __shfl_sync(0xffffffffu, mine.grp, i);
    const uint32_t h0 = first_head(grp), nh = heads_of(grp);
    for (uint32_t h = (warp + kWarps - run % kWarps) % kWarps; h < nh; h += kWarps) {
      // lane x has part x's maximum and sum
      float m = -INFINITY, l = 0.f;
      if (in_run >> lane & 1) {
        const float2 v = *reinterpret_cast<const float2 *>(ml + (lane * C::kHeads + h) * 2);
        m = v.x, l = v.y;
      }
      const float top = warp_max(m), ref = top == -INFINITY ? 0.f : top * scale;
      const float c = exp2_fast(m * scale - ref);
      l = warp_sum(l * c);
      m = top;
      float2 acc[DP / 64] = {};
#pragma unroll 1
      for (uint32_t more = in_run; more; more &= more - 1) {
        const uint32_t x = __ffs(more) - 1;
        const float cx = __shfl_sync(0xffffffffu, c, x);
        const float *src = part_o(x) + h * DP;
#pragma unroll
        for (int d = 0; d < DP / 64; ++d) {
          const float2 v = *reinterpret_cast<const float2 *>(src + d * 64 + lane * 2);
          acc[d].x += cx * v.x, acc[d].y += cx * v.y;
        }
      }
      if (whole) {
        const float r = 1.0f / l;
        float finite = 0.f;
#pragma unroll
        for (int d = 0; d < DP / 64; ++d) {
        const float a = acc[d].x * r, b = acc[d].y * r;
        finite += a * 0.f + b * 0.f;
        write_out(seq, h0 + h, d * 64 + lane * 2, a, b);
      }
      if (__any_sync(0xffffffffu, finite != 0.f)) {
        __syncwarp();
        redo(seq, h0 + h);
      }
      } else {
        const size_t rec = ((size_t)blockIdx.x * 2 + side) * C::kHeads + h;
#pragma unroll
        for (int d = 0; d < DP / 64; ++d) *reinterpret_cast<float2 *>(scratch_o + rec * DP + d * 64 + lane * 2) = acc[d];
        if (lane == 0) *reinterpret_cast<float2 *>(scratch_ml + rec * 2) = make_float2(m, l);
      }
    }
    if (!whole) {
      open_there |= 1u << side;
      open_seq[side] = seq, open_grp[side] = grp;
    }
  }
  if (!open_there) {
    stamp_end(p.stamps);
    return;
  }

  // ---- pairs of several CTAs: the last of its CTAs adds up the parts, of more than kJoin the last one of every kGroup does and the last of those ----
  auto rec = [&](uint32_t c, uint32_t c0, uint32_t h) { return ((size_t)c * 2 + (c + 1 == c0 ? 1 : 0)) * C::kHeads + h; };  // the first part ends its CTA's range
  auto add_up = [&](uint32_t side, uint32_t first, uint32_t step, uint32_t parts, bool whole) {  // at most 32 parts: lane x has part x's maximum and sum
    const uint32_t seq = open_seq[side], grp = open_grp[side], h0 = first_head(grp), nh = heads_of(grp), c0 = cut_s[side][0];
#pragma unroll 1
    for (uint32_t h = warp; h < nh; h += kWarps) {
      float2 own = {-INFINITY, 0.f};
      if (lane < parts) own = __ldcg(reinterpret_cast<const float2 *>(scratch_ml + rec(first + lane * step, c0, h) * 2));
      const float m = warp_max(own.x), ref = m == -INFINITY ? 0.f : m * scale, w = exp2_fast(own.x * scale - ref), l = warp_sum(lane < parts ? w * own.y : 0.f);
      float2 acc[DP / 64] = {};
#pragma unroll 1
      for (uint32_t x = 0; x < parts; x += kAtOnce) {
        float2 v[kAtOnce][DP / 64];
#pragma unroll
        for (uint32_t y = 0; y < kAtOnce; ++y)
#pragma unroll
          for (int d = 0; d < DP / 64; ++d)
            v[y][d] = __ldcg(reinterpret_cast<const float2 *>(scratch_o + rec(first + min(x + y, parts - 1) * step, c0, h) * DP + d * 64 + lane * 2));
#pragma unroll
        for (uint32_t y = 0; y < kAtOnce; ++y) {
          const float wy = __shfl_sync(0xffffffffu, w, (x + y) & 31);
          if (x + y >= parts) continue;
#pragma unroll
          for (int d = 0; d < DP / 64; ++d) acc[d].x += wy * v[y][d].x, acc[d].y += wy * v[y][d].y;
        }
      }
      if (!whole) {
        const size_t to = rec(first, c0, h);
        __syncwarp();
#pragma unroll
        for (int d = 0; d < DP / 64; ++d) *reinterpret_cast<float2 *>(scratch_o + to * DP + d * 64 + lane * 2) = acc[d];
        if (lane == 0) *reinterpret_cast<float2 *>(scratch_ml + to * 2) = make_float2(m, l);
        continue;
      }
      const float r = 1.0f / l;
      float finite = 0.f;
#pragma unroll
      for (int d = 0; d < DP / 64; ++d) {
        const float a = acc[d].x * r, b = acc[d].y * r;
        finite += a * 0.f + b * 0.f;
        write_out(seq, h0 + h, d * 64 + lane * 2, a, b);
      }
      if (__any_sync(0xffffffffu, finite != 0.f)) {
        __syncwarp();
        redo(seq, h0 + h);
      }
    }
  };
  __threadfence();
  __syncthreads();
  if (tid < 2) {
    last_s[tid] = 0;
    if (open_there >> tid & 1) {
      const uint32_t c0 = cut_s[tid][0], parts = cut_s[tid][1] - c0 + 2, g = (blockIdx.x + 1 - c0) / kGroup;
      uint32_t *counter = parts <= kJoin ? p.counters + c0 : p.counters + gridDim.x + 1 + c0 + g;  // a pair has fewer groups than cuts
      __threadfence();
      if (atomicAdd(counter, 1u) + 1 == (parts <= kJoin ? parts : min(kGroup, parts - g * kGroup))) {
        *counter = 0;
        last_s[tid] = 1;
      }
    }
  }
  __syncthreads();
#pragma unroll 1
  for (uint32_t side = 0; side < 2; ++side) {
    if (!last_s[side]) continue;
    __threadfence();
    const uint32_t c0 = cut_s[side][0], parts = cut_s[side][1] - c0 + 2;
    if (parts <= kJoin) {
      add_up(side, c0 - 1, 1, parts, true);
      continue;
    }
    const uint32_t g = (blockIdx.x + 1 - c0) / kGroup, groups = (parts + kGroup - 1) / kGroup;
    add_up(side, c0 - 1 + g * kGroup, 1, min(kGroup, parts - g * kGroup), false);
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      __threadfence();
      last_s[side] = 1;
      if (atomicAdd(p.counters + c0, 1u) + 1 == groups) {
        p.counters[c0] = 0;
        last_s[side] = 2;
      }
    }
    __syncthreads();
    if (last_s[side] == 2) {
      __threadfence();
      add_up(side, c0 - 1, kGroup, groups, true);
    }
  }
  stamp_end(p.stamps);
}

template <bool BF, int DP, bool WIDE> cudaError_t setup_one() {
  return cudaFuncSetAttribute(paged_token_kernel<BF, DP, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg<DP, WIDE>::kSmem);
}
template <bool BF, int DP, bool WIDE> cudaError_t run(const PagedAttention &p, uint32_t sms, cudaStream_t s) {
  using C = Cfg<DP, WIDE>;
  // No more CTAs than there can be shares of.
  const uint64_t per = p.heads / p.kv_heads, pairs = (uint64_t)p.kv_heads * ((per + C::kHeads - 1) / C::kHeads);
  const double most = (double)p.n * pairs * (((uint64_t)p.width * p.page.d + C::kTile - 1) / C::kTile + kPairCost), shares = (most + C::kShare - 1) / C::kShare;
  return launch_following(paged_token_kernel<BF, DP, WIDE>, dim3((uint32_t)std::min<double>(sms, shares)), C::kThreads, C::kSmem, s, p);
}
bool wide(uint32_t heads, uint32_t kv_heads) { return heads / kv_heads > 8; }  // more query heads than the narrow form's rows
template <bool BF> cudaError_t pick(const PagedAttention &p, uint32_t sms, cudaStream_t s) {
  const bool w = wide(p.heads, p.kv_heads);
  if (p.dim <= 64) return w ? run<BF, 64, true>(p, sms, s) : run<BF, 64, false>(p, sms, s);
  if (p.dim <= 128) return w ? run<BF, 128, true>(p, sms, s) : run<BF, 128, false>(p, sms, s);
  return w ? run<BF, 256, true>(p, sms, s) : run<BF, 256, false>(p, sms, s);
}

}  // namespace

size_t paged_token_scratch(uint32_t heads, uint32_t kv_heads, uint32_t dim, uint32_t sms) {
  const uint32_t dp = dim <= 64 ? 64 : dim <= 128 ? 128 : 256, most = wide(heads, kv_heads) ? 16 : 8;
  return (size_t)sms * 2 * most * (dp + 2) * 4;
}
cudaError_t setup_paged_token() {
  for (cudaError_t e : {setup_one<false, 64, false>(), setup_one<false, 64, true>(), setup_one<false, 128, false>(), setup_one<false, 128, true>(),
                        setup_one<false, 256, false>(), setup_one<false, 256, true>(), setup_one<true, 64, false>(), setup_one<true, 64, true>(),
                        setup_one<true, 128, false>(), setup_one<true, 128, true>(), setup_one<true, 256, false>(), setup_one<true, 256, true>()})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}
cudaError_t launch_paged_token(const PagedAttention &p, uint32_t sms, cudaStream_t s) { return p.bf ? pick<true>(p, sms, s) : pick<false>(p, sms, s); }

}  // namespace vkl
