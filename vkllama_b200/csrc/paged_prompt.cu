// Attention of several new rows per sequence over a paged cache (prompts, chunks of prompts, drafts): row t of sequence i stands at
// position p = length_i - new_i + t and sees the positions max(0, p + 1 - window) <= j <= p,
//   out = sum_j softmax_j(scale q.k_j) v_j.
//
// The query heads of a key head share its keys and values, so a tile's rows are (row, head of the group) pairs, 64 of them: with
// grouped heads a tile has fewer rows of the sequence and the same use of every key that is fetched. One CTA of four warps has a tile;
// keys and values come through shared memory by cp.async, two tiles ahead, and both products run on mma.sync (m16n8k16, fp32 sums) with
// a running maximum and sum per row (Milakov and Gimelshein, 2018). Probabilities are rounded to 16 bits for the second product, as its operand has to be (relative
// 2^-11 or 2^-8 each, as much as the rounding of the output); their sum is taken before. In fp16 they are 2^14 times as large, in sum and output
// alike, because the format ends at steps of 2^-24: so 2^-11 holds down to 2^-28 of the row's largest, and below each is off by 2^-39 of
// the largest at most. Positions that a row does not see are masked
// only in the tiles that some row of the warp does not see whole; a row whose result is not finite is computed again from its own
// positions (paged_rows.cuh).
//
// It has what the tcgen05 kernel (paged_prompt_tc.cu) would leave mostly empty, and heads above 128: sequences of few rows that see few positions, where
// the start and end of a CTA are what there is, so three of them share an SM. 64 prompts of 64 rows, 32 heads of 128: 67 us, 2.0 TB/s; four of
// 64 rows 10 us. On long prompts its products run at 210 TFLOP/s (fp32 sums of mma.sync; 4096 rows, 32 heads of 128, 658 us, tcgen05 137 on a cool GPU and
// 163 under full load; 16 heads of 200 or 256, which have no other kernel, 570 and 565).
#include <algorithm>

#include "common.cuh"
#include "paged.h"
#include "paged_rows.cuh"
#include "paged_value.cuh"

namespace vkl {
namespace {

constexpr uint32_t kThreads = 128, kRows = 64;
constexpr float kRaise = 14.f;  // of fp16 probabilities' exponents

template <int DP> struct Cfg {
  static constexpr uint32_t kKeys = DP == 256 ? 32 : 64;  // positions of a tile
  static constexpr uint32_t kSmem = 2 * 2 * kKeys * DP * 2;
};

// MANY: tables that hold more than kManyPositions (paged_rows.cuh). The other widths have no more than 128 positions here, or the tcgen05 kernel takes them. (One
// kernel for both: 4096 rows, 16 heads of 256, 574 us instead of 565.)
template <bool BF, int DP, bool MANY = false> __global__ void __launch_bounds__(kThreads, DP == 256 ? 1 : 3) paged_prompt_kernel(const PagedAttention p) {
  using C = Cfg<DP>;
  constexpr uint32_t CH = DP / 8, KT = C::kKeys;
  constexpr int KS = DP / 16, NT = DP / 8, SN = KT / 8;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint32_t row_s[2][KT];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const uint32_t per = p.heads / p.kv_heads, tile = blockIdx.x / p.kv_heads, kvh = blockIdx.x - tile * p.kv_heads;
  __shared__ Place at_s;
  __shared__ bool found_s;
  follow();
  stamp_begin(p.stamps);
  if (warp == 0) {
    Place found = {};
    Walk walk;
    const bool there = find_tile(p, per, kRows, tile, found, walk);
    if (lane == 0) at_s = found, found_s = there;
  } else if (warp == 1 && blockIdx.x == 0) {
    check_rows(p);
  }
  __syncthreads();
  if (!found_s) return;
  const Place at = at_s;
  const uint32_t packed = at.fresh * per, r_end = min(at.first + kRows, packed), past = at.len - at.fresh;
  // positions that the tile's rows see
  const uint32_t lo_pos = past + at.first / per, hi_pos = past + (r_end - 1) / per;
  const uint32_t j_begin = p.window && lo_pos + 1 > p.window ? lo_pos + 1 - p.window : 0;
  const uint32_t t0 = j_begin / KT, t1 = hi_pos / KT + 1;

  const uint32_t smem_a = smem_addr(smem);
  auto look_up = [&](uint32_t t) {  // cache rows of tile t
    if (tid < KT) {
      const uint32_t j = t * KT + tid;
      uint32_t r = 0xffffffffu;
      if (t < t1 && j >= j_begin && j <= hi_pos) {
        const uint32_t n = quotient(j, p.page), page = p.table[(size_t)at.seq * p.width + n];
        if (page < p.pages) r = (page * p.kv_heads + kvh) * p.page.d + j - n * p.page.d;
        else raise(p.error, PAGED_BAD_PAGE);
      }
      row_s[t & 1][tid] = r;
    }
  };
  auto request = [&](uint32_t t) {
    if (t < t1) {
      const uint32_t dst = smem_a + (t & 1) * 2 * KT * DP * 2;
#pragma unroll
      for (uint32_t i = 0; i < KT * CH / kThreads; ++i) {
        const uint32_t c = i * kThreads + tid, row = c / CH, col = c % CH;
        const uint32_t r = row_s[t & 1][row];
        const bool there = r != 0xffffffffu && col * 8 < p.dim;
        const size_t o = there ? (size_t)r * p.dim + col * 8 : 0;
        const uint32_t to = dst + (row * CH + (col ^ (row & 7))) * 16;
        copy16(to, static_cast<const uint16_t *>(p.kcache) + o, there);
        copy16(to + KT * DP * 2, static_cast<const uint16_t *>(p.vcache) + o, there);
      }
    }
    copy_commit();
  };
  look_up(t0);
  look_up(t0 + 1);
  __syncthreads();
  request(t0);
  request(t0 + 1);

  // this thread's rows: g and g + 8 of its warp's sixteen
  uint32_t q[KS][4], pos[2];
  size_t out_at[2];
  bool mine[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t r = at.first + warp * 16 + g + i * 8;
    mine[i] = r < packed;
    const uint32_t t = mine[i] ? r / per : 0, h = kvh * per + (mine[i] ? r - t * per : 0);
    pos[i] = past + (mine[i] ? t : (r_end - 1) / per);
    out_at[i] = ((size_t)(at.row0 + t) * p.heads + h) * p.dim;
    const uint16_t *src = static_cast<const uint16_t *>(p.q) + (at.row0 + t) * p.q_ld + h * p.dim;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t d = k * 16 + e * 8 + t4 * 2;
        q[k][i + 2 * e] = mine[i] && d < p.dim ? *reinterpret_cast<const uint32_t *>(src + d) : 0u;
      }
  }
  const uint32_t wr0 = min(at.first + warp * 16, r_end - 1), wr1 = min(wr0 + 15, r_end - 1);
  const uint32_t w_lo = past + wr0 / per, w_hi = past + wr1 / per;  // least and most position of the warp's rows
  const uint32_t w_first = p.window && w_hi + 1 > p.window ? w_hi + 1 - p.window : 0;  // all of them see [w_first, w_lo]
  float o[NT][4] = {}, mx[2] = {-INFINITY, -INFINITY}, sum[2] = {};
  const float scale = p.scale * kLog2e;
  const uint32_t lrow = lane & 7, lsel = lane >> 3;

#pragma unroll 1
  for (uint32_t t = t0; t < t1; ++t) {
    copy_wait<1>();
    __syncthreads();  // the tile is there, and its rows' places may be looked up anew
    look_up(t + 2);
    const uint32_t kt = smem_a + (t & 1) * 2 * KT * DP * 2, vt = kt + KT * DP * 2;
    float s[SN][4] = {};
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int n = 0; n < SN; n += 2) {
        uint32_t b[4];
        ldmatrix4(b, kt + ((n * 8 + lrow + (lsel >> 1) * 8) * CH + ((2 * k + (lsel & 1)) ^ lrow)) * 16);
        mma2<BF>(s[n], q[k][0], q[k][1], q[k][2], q[k][3], b[0], b[1]);
        mma2<BF>(s[n + 1], q[k][0], q[k][1], q[k][2], q[k][3], b[2], b[3]);
      }
    const bool whole = t * KT >= w_first && t * KT + KT - 1 <= w_lo;
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < SN; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] *= scale;
        if (!whole) {
          const uint32_t j = t * KT + n * 8 + t4 * 2 + (e & 1), at_pos = pos[e >> 1];
          if (j > at_pos || (p.window && j + p.window <= at_pos)) s[n][e] = -INFINITY;
        }
        top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
      }
    float ref[2], from[2];  // what exponents are taken against, of sums so far and of probabilities
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
      const float now = fmaxf(mx[i], top[i]);
      ref[i] = now == -INFINITY ? 0.f : now;
      from[i] = BF ? ref[i] : ref[i] - kRaise;
      const float c = exp2f(mx[i] - ref[i]);
      mx[i] = now;
      sum[i] *= c;
#pragma unroll
      for (int n = 0; n < NT; ++n) o[n][2 * i] *= c, o[n][2 * i + 1] *= c;
    }
#pragma unroll
    for (int n = 0; n < SN; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = exp2f(s[n][e] - from[e >> 1]);
        sum[e >> 1] += s[n][e];
      }
    if (MANY && t1 - t0 > kManyPositions / KT) {
      uint32_t a[KT / 16][4];
#pragma unroll
      for (int k = 0; k < (int)KT / 16; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) a[k][e] = pack2<BF>(s[2 * k + (e >> 1)][2 * (e & 1)], s[2 * k + (e >> 1)][2 * (e & 1) + 1]);
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        float x[4] = {}, y[4] = {};
#pragma unroll
        for (int k = 0; k < (int)KT / 16; ++k) {
          uint32_t b[4];
          ldmatrix4_t(b, vt + ((k * 16 + lrow + (lsel & 1) * 8) * CH + ((n + (lsel >> 1)) ^ lrow)) * 16);
          mma2<BF>(x, a[k][0], a[k][1], a[k][2], a[k][3], b[0], b[1]);
          mma2<BF>(y, a[k][0], a[k][1], a[k][2], a[k][3], b[2], b[3]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] += x[e], o[n + 1][e] += y[e];
      }
    } else {
#pragma unroll
      for (int k = 0; k < (int)KT / 16; ++k) {
        const uint32_t a0 = pack2<BF>(s[2 * k][0], s[2 * k][1]), a1 = pack2<BF>(s[2 * k][2], s[2 * k][3]);
        const uint32_t a2 = pack2<BF>(s[2 * k + 1][0], s[2 * k + 1][1]), a3 = pack2<BF>(s[2 * k + 1][2], s[2 * k + 1][3]);
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          uint32_t b[4];
          ldmatrix4_t(b, vt + ((k * 16 + lrow + (lsel & 1) * 8) * CH + ((n + (lsel >> 1)) ^ lrow)) * 16);
          mma2<BF>(o[n], a0, a1, a2, a3, b[0], b[1]);
          mma2<BF>(o[n + 1], a0, a1, a2, a3, b[2], b[3]);
        }
      }
    }
    __syncthreads();  // everyone is through with the tile
    request(t + 2);
  }
  copy_wait<0>();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
    sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
    const float r = 1.0f / sum[i];
    float finite = 0.f;
    if (mine[i]) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint32_t d = n * 8 + t4 * 2;
        const float a = o[n][2 * i] * r, b = o[n][2 * i + 1] * r;
        finite += a * 0.f + b * 0.f;
        if (d < p.dim) *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(p.out) + out_at[i] + d) = pack2<BF>(a, b);
      }
    }
    const uint32_t again = __ballot_sync(0xffffffffu, finite != 0.f);  // NaN
    __syncwarp();
    for (uint32_t x = 0; x < 8; ++x)
      if (again >> (x * 4) & 15u) row_again<BF>(p, at, kvh, at.first + warp * 16 + i * 8 + x, 0, DP);
  }
  stamp_end(p.stamps);
}

template <bool BF, int DP, bool MANY = false> cudaError_t setup_one() {
  return cudaFuncSetAttribute(paged_prompt_kernel<BF, DP, MANY>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg<DP>::kSmem);
}
template <bool BF> cudaError_t pick(const PagedAttention &p, cudaStream_t s) {
  // tiles are counted on the device; every sequence has at most one that is not full
  const uint64_t per = p.heads / p.kv_heads, tiles = p.rows * per / kRows + std::min<uint64_t>(p.n, p.rows * per);
  const dim3 grid((uint32_t)(tiles * p.kv_heads));  // all heads of a tile, then the next tile
  if (p.dim <= 64) return launch_following(paged_prompt_kernel<BF, 64>, grid, kThreads, Cfg<64>::kSmem, s, p);
  if (p.dim <= 128) return launch_following(paged_prompt_kernel<BF, 128>, grid, kThreads, Cfg<128>::kSmem, s, p);
  return launch_following(p.width * p.page.d > kManyPositions ? paged_prompt_kernel<BF, 256, true> : paged_prompt_kernel<BF, 256>, grid, kThreads, Cfg<256>::kSmem, s, p);
}

}  // namespace

cudaError_t setup_paged_prompt() {
  for (cudaError_t e : {setup_one<false, 64>(), setup_one<false, 128>(), setup_one<false, 256>(), setup_one<false, 256, true>(), setup_one<true, 64>(), setup_one<true, 128>(),
                        setup_one<true, 256>(), setup_one<true, 256, true>()})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}
// The host knows the rows of all sequences together, and how many positions a table can hold. Where that does not say enough, each kernel takes the
// sequences that are its own (the second finds nothing to do in 2 to 3 us).
uint32_t paged_prompt_launches(const PagedAttention &p) {
  const bool many = (uint64_t)p.rows * (p.heads / p.kv_heads) >= (uint64_t)kTensorRows * p.n;
  return (p.dim > 128 || many || p.width * p.page.d < kTensorLength ? 1 : 2) + (p.splits > 1);
}
cudaError_t launch_paged_prompt(const PagedAttention &p, uint32_t sms, cudaStream_t s) {
  const bool many = (uint64_t)p.rows * (p.heads / p.kv_heads) >= (uint64_t)kTensorRows * p.n;
  const uint32_t launches = paged_prompt_launches(p) - (p.splits > 1);
  const bool tensor = p.dim <= 128 && many;
  PagedAttention q = p;
  if (launches == 2) q.part = 1;
  cudaError_t e = cudaSuccess;
  if (launches == 2 || !tensor) e = p.bf ? pick<true>(q, s) : pick<false>(q, s);
  if (launches == 2) q.part = 2;
  if (e == cudaSuccess && (launches == 2 || tensor)) e = launch_paged_prompt_tc(q, sms, s);
  if (e == cudaSuccess && p.splits > 1) e = launch_paged_prompt_join(p, s);
  return e;
}

}  // namespace vkl
