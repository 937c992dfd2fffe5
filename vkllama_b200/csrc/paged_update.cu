// New rows of queries, keys and values, of as many sequences as there are: queries and keys are rotated by the position of their
// row, keys and values go to their slots.
//
//   (x_2k, x_2k+1) -> (x_2k cos a - x_2k+1 sin a, x_2k sin a + x_2k+1 cos a), a = position * theta^(-2k / dim)
//
// The angle is taken in turns, in 64 bits, and only what is left of it after whole turns is rounded to 32: a position of 100,000
// would otherwise cost the fastest pairs 17 bits of their phase. One CTA has (a part of) one row: its threads request their 16-byte
// pieces, work out the row's dim / 2 angles once for all heads meanwhile, and store. Bound by HBM: a row is read and written once; 0.21 GB of queries, keys
// and values in 37 us, 5.7 TB/s (a copy: 6.56). A decode step's 24 rows take 2 us, which the host's call hides.
#include <math.h>

#include "common.cuh"
#include "paged.h"
#include "paged_value.cuh"

namespace vkl {
namespace {

constexpr uint32_t kThreads = 256, kPieces = 4;  // 16-byte pieces of a thread
constexpr uint32_t kMaxPairs = 128;

template <bool BF> __global__ void __launch_bounds__(kThreads) paged_update_kernel(const PagedUpdate p) {
  __shared__ float2 turn_s[kMaxPairs];
  follow();
  stamp_begin(p.stamps);
  const uint32_t row = blockIdx.x, tid = threadIdx.x, per = p.dim / 8;
  const uint32_t nq = p.q ? p.heads * per : 0, nk = p.kv_heads * per, all = nq + 2 * nk, first = blockIdx.y * kThreads * kPieces + tid;
  uint4 x[kPieces];
#pragma unroll
  for (uint32_t i = 0; i < kPieces; ++i) {
    const uint32_t c = first + i * kThreads;
    if (c >= all) break;
    const uint16_t *src = c < nq        ? static_cast<const uint16_t *>(p.q) + row * p.q_ld + c * 8
                          : c < nq + nk ? static_cast<const uint16_t *>(p.k) + row * p.k_ld + (c - nq) * 8
                                        : static_cast<const uint16_t *>(p.v) + row * p.v_ld + (c - nq - nk) * 8;
    x[i] = load_once(src);
  }
  const uint32_t slot = p.map[row], pos = p.map[p.rows + row];
  if (p.turns) {
    if (tid < p.dim / 2) {
      const double turns = (double)pos * p.turns[tid];
      float s, c;
      sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
      turn_s[tid] = make_float2(c, s);
    }
    __syncthreads();
  }
  const uint32_t page = slot / p.page.d, in = slot - page * p.page.d;
  const bool there = slot != kNoSlot && page < p.pages;
  if (slot != kNoSlot && !there && tid == 0) raise(p.error, PAGED_BAD_PAGE);
#pragma unroll
  for (uint32_t i = 0; i < kPieces; ++i) {
    const uint32_t c = first + i * kThreads;
    if (c >= all) break;
    if (c < nq + nk && p.turns) {
      const uint32_t pair = (c < nq ? c : c - nq) % per * 4;
      uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 t = turn_s[pair + e], v = unpack2<BF>(u[e]);
        u[e] = pack2<BF>(v.x * t.x - v.y * t.y, v.x * t.y + v.y * t.x);
      }
      x[i] = make_uint4(u[0], u[1], u[2], u[3]);
    }
    if (c < nq) {
      *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.q_out) + ((size_t)row * nq + c) * 8) = x[i];
    } else if (there) {
      const bool key = c < nq + nk;
      const uint32_t at = c - nq - (key ? 0 : nk), head = at / per;
      const size_t to = ((size_t)page * p.kv_heads + head) * p.page.d + in;
      *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(key ? p.kcache : p.vcache) + (to * per + at - head * per) * 8) = x[i];
    }
  }
  if (blockIdx.x + 1024 >= gridDim.x) stamp_end(p.stamps);  // of the CTAs that may be the last
}

}  // namespace

cudaError_t launch_paged_update(const PagedUpdate &p, cudaStream_t s) {
  const uint32_t pieces = ((p.q ? p.heads : 0) + 2 * p.kv_heads) * (p.dim / 8), parts = (pieces + kThreads * kPieces - 1) / (kThreads * kPieces);
  return launch_following(p.bf ? paged_update_kernel<true> : paged_update_kernel<false>, dim3(p.rows, parts), kThreads, 0, s, p);
}

}  // namespace vkl
