// Attention of several new rows per sequence (paged_prompt.cu) on the 5th-generation tensor cores, for heads up to 128 wide.
//
// A CTA has 256 packed rows of a sequence and key head, as two tiles of 128, and walks over the positions that they see in tiles of
// 128. Per tile of rows i and positions j: S_i = Q_i K_j^T (tcgen05.mma, fp32 in TMEM), P_i = 2^(scale S_i - reference) as 16-bit numbers
// written over S_i in TMEM, O_i += P_i V_j with P as the TMEM operand. The two tiles of rows take turns: while the tensor core works
// for one, the exponentials of the other are computed, which take as long (16 per clock and SM: 1024 cycles for 128 x 128, like the two
// products). Warps:
//   0-3, 4-7  softmax of tile 0, 1: one thread per row, so no exchange between threads. The reference is the row's maximum as of the last time
//             that it grew by more than 2^8: until then the probabilities stay below 2^8 and O as it is; only then O is multiplied. Reads S
//             twice (maximum, exponentials) instead of keeping 128 values.
//   8, 9      fetch Q, then K_j and V_j by cp.async into rings of two stages, in the 128-byte swizzle of the matrix descriptors: K is K-major and
//             V, as it lies in the cache, MN-major (64 dimensions of a position are a row of 128 bytes in both).
//   10        issues the MMAs. They complete in order, so the commit behind S_i(j + 1) also says that P_i(j) V_j is in O_i.
// Every wait is bounded; after one that ran out all warps leave, and the error word is raised.
#include <algorithm>

#include "paged_rows.cuh"
#include "tcgen05.cuh"

namespace vkl {
namespace {

constexpr uint32_t kSoftmaxWarps = 8, kFetchWarps = 2, kMmaWarp = 10, kThreads = 12 * 32;  // the twelfth idles: more than 12 warps would have 128 registers each
constexpr uint32_t kRows = 128, kKeys = 128, kStages = 2;
constexpr uint32_t kWaitCode = 9, kPolls = 1u << 20;

template <int DP> struct Cfg {
  static constexpr uint32_t kTile = 128 * DP * 2;  // bytes of 128 rows
  // One CTA per SM, which takes all of its TMEM: more than half of the shared memory, whatever the head width.
  static constexpr uint32_t kSmem = std::max((2 + 2 * kStages) * kTile, 120u * 1024) + 1024;
};

__device__ __forceinline__ void mma_tmem(uint32_t acc, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, bool accumulate) {
  constexpr uint32_t hi = (1024u >> 4) | 1u << 14 | 2u << 29;  // as mma_f16's
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 b;\n mov.b64 b, {%2, %3};\n setp.ne.b32 p, %5, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}" ::"r"(acc), "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
               "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool BF, int DP> __global__ void __launch_bounds__(kThreads, 1) paged_prompt_tc_kernel(const PagedAttention p) {
  using C = Cfg<DP>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t q_full, k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], s_full[2], p_full[2], o_full[2];
  __shared__ uint32_t tmem_s, row_s[kFetchWarps][2][kKeys];
  __shared__ volatile uint32_t failed_s;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kvh = blockIdx.y, per = p.heads / p.kv_heads;
  follow();
  stamp_begin(p.stamps);
  Place at;
  if (!find_tile<kThreads>(p, per, 2 * kRows, blockIdx.x, at)) return;
  const uint32_t packed = at.fresh * per, past = at.len - at.fresh;
  // per tile of rows: its rows that exist, and the tiles of positions [b, e) that they see
  const bool both = at.first + kRows < packed;
  uint32_t b[2], e[2];
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    const uint32_t r0 = at.first + (both ? i : 0) * kRows, r1 = min(r0 + kRows, packed), lo = past + r0 / per, hi = past + (r1 - 1) / per;
    b[i] = (p.window && lo + 1 > p.window ? lo + 1 - p.window : 0) / kKeys;
    e[i] = hi / kKeys + 1;
  }
  const uint32_t t0 = b[0], t1 = e[1], tiles = both ? 2 : 1;  // b and e grow with the rows
  if (tid == 0) {
    auto init = [](uint64_t *bar, uint32_t n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(sa(bar)), "r"(n) : "memory"); };
    init(&q_full, kFetchWarps);
    for (uint32_t s = 0; s < kStages; ++s) init(&k_full[s], kFetchWarps), init(&v_full[s], kFetchWarps), init(&k_empty[s], 1), init(&v_empty[s], 1);
    for (uint32_t i = 0; i < 2; ++i) init(&s_full[i], 1), init(&p_full[i], 4), init(&o_full[i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    failed_s = 0;
  }
  if (warp == kMmaWarp) tmem_alloc<512>(sa(&tmem_s));
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = tmem_s, q_a = sa(smem), k_a = q_a + 2 * C::kTile, v_a = k_a + kStages * C::kTile;
  // False when the wait ran out, or anyone's did.
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    const uint32_t a = sa(bar);
    for (uint32_t n = 0; n < kPolls / 64; ++n) {
      for (uint32_t k = 0; k < 64; ++k) {
        uint32_t ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(a), "r"(parity) : "memory");
        if (ok) return true;
      }
      if (failed_s) return false;
    }
    failed_s = 1;
    return false;
  };
  auto wait_warp = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };  // the lanes agree

  if (warp < kSoftmaxWarps) {
    // ------------------------------------------------------------------------------------------------------- softmax
    const uint32_t i = warp >> 2, quad = warp & 3;
    if (i < tiles) {
      const uint32_t r = at.first + tid, w0 = min(at.first + warp * 32, packed - 1), w1 = min(w0 + 31, packed - 1);
      const uint32_t pos = past + min(r, packed - 1) / per, w_lo = past + w0 / per, w_hi = past + w1 / per;
      const uint32_t w_first = p.window && w_hi + 1 > p.window ? w_hi + 1 - p.window : 0;  // every row of the warp sees [w_first, w_lo]
      const uint32_t first = p.window && pos + 1 > p.window ? pos + 1 - p.window : 0;
      const float scale = p.scale * kLog2e;
      const uint32_t lanes = (quad * 32u) << 16, s_t = tmem + lanes + i * 128, o_t = tmem + lanes + 256 + i * DP;
      float top = -INFINITY, ref = 0.f, sum = 0.f;  // of scaled scores: reference, and what is subtracted (0 where the reference is -infinity)
      bool ok = true;
      uint32_t phase = 0;
      const uint32_t bi = b[i], ei = e[i];
      for (uint32_t t = bi; t < ei; ++t, phase ^= 1) {
        if (!(ok = wait_warp(&s_full[i], phase))) break;
        tc_after();
        const bool whole = t * kKeys >= w_first && t * kKeys + kKeys - 1 <= w_lo;
        auto take = [&](uint32_t c, float (&v)[32]) {
          uint32_t u[32];
          tmem_ld32(s_t + c * 32, u);
#pragma unroll
          for (int x = 0; x < 32; ++x) v[x] = __uint_as_float(u[x]) * scale;
          if (!whole) {
#pragma unroll
            for (int x = 0; x < 32; ++x) {
              const uint32_t j = t * kKeys + c * 32 + x;
              if (j > pos || j < first) v[x] = -INFINITY;
            }
          }
        };
        float m = -INFINITY;
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) {
          float v[32];
          take(c, v);
#pragma unroll
          for (int x = 0; x < 32; ++x) m = fmaxf(m, v[x]);
        }
        if (t == bi) {
          top = m;
          ref = m == -INFINITY ? 0.f : m;
        } else {
          const bool grown = m - ref > 8.0f || (top == -INFINITY && m != -INFINITY);
          if (__any_sync(0xffffffffu, grown)) {
            float c = 1.0f;
            if (grown) {
              c = exp2_fast(top - m);
              top = ref = m;
            }
            sum *= c;
#pragma unroll 1
            for (uint32_t d = 0; d < DP; d += 32) {
              uint32_t u[32];
              tmem_ld32(o_t + d, u);
#pragma unroll
              for (int x = 0; x < 32; ++x) u[x] = __float_as_uint(__uint_as_float(u[x]) * c);
              tmem_st32(o_t + d, u);
            }
            tmem_stored();
          }
        }
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) {
          float v[32];
          uint32_t u[16];
          take(c, v);
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            v[x] = exp2_fast(v[x] - ref);
            sum += v[x];
          }
#pragma unroll
          for (int x = 0; x < 16; ++x) u[x] = pack2<BF>(v[2 * x], v[2 * x + 1]);
          tmem_st16(s_t + c * 16, u);
        }
        tmem_stored();
        tc_before();
        __syncwarp();
        if (lane == 0) arrive(sa(&p_full[i]));
      }
      if (ok && wait_warp(&o_full[i], 0)) {
        tc_after();
        const float inv = 1.0f / sum;
        const uint32_t row = min(r, packed - 1), rt = row / per, h = kvh * per + row - rt * per;
        uint16_t *out = static_cast<uint16_t *>(p.out) + ((size_t)(at.row0 + rt) * p.heads + h) * p.dim;
        float finite = 0.f;
#pragma unroll 1
        for (uint32_t d = 0; d < DP; d += 32) {
          uint32_t u[32];
          tmem_ld32(o_t + d, u);
#pragma unroll
          for (int x = 0; x < 32; x += 8) {
            float v[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              v[y] = __uint_as_float(u[x + y]) * inv;
              finite += v[y] * 0.f;
            }
            if (r < packed && d + x < p.dim)
              *reinterpret_cast<uint4 *>(out + d + x) = make_uint4(pack2<BF>(v[0], v[1]), pack2<BF>(v[2], v[3]), pack2<BF>(v[4], v[5]), pack2<BF>(v[6], v[7]));
          }
        }
        uint32_t again = __ballot_sync(0xffffffffu, finite != 0.f && r < packed);  // NaN
        __syncwarp();
        for (; again; again &= again - 1) row_again<BF>(p, at, kvh, at.first + warp * 32 + __ffs(again) - 1);
      }
    }
  } else if (warp < kSoftmaxWarps + kFetchWarps) {
    // --------------------------------------------------------------------------------------------------------- fetch
    constexpr uint32_t CH = DP / 8, FT = kFetchWarps * 32, RS = FT / CH;  // pieces of a row; rows that the warps fetch at a time
    const uint32_t ft = tid - kSoftmaxWarps * 32, col = ft % CH, frow = ft / CH;
    const bool col_there = col * 8 < p.dim;
    auto place = [&](uint32_t row) { return (col >> 3) * (128 * 128) + row * 128 + (((col & 7) ^ (row & 7)) << 4); };
    auto landed = [&](uint64_t *bar) {  // this thread's oldest pieces are there: the tensor core may read them
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive(sa(bar));
    };
    const uint32_t j_first = past + at.first / per + 1 > p.window && p.window ? past + at.first / per + 1 - p.window : 0, j_last = past + (min(at.first + 2 * kRows, packed) - 1) / per;
    uint32_t(*rows)[kKeys] = row_s[warp - kSoftmaxWarps];  // each warp looks up for itself: the fetching warps never wait for each other
    auto look_up = [&](uint32_t t) {  // cache rows of the tile's positions
#pragma unroll
      for (uint32_t x = lane; x < kKeys; x += 32) {
        const uint32_t j = t * kKeys + x;
        uint32_t r = 0xffffffffu;
        if (j >= j_first && j <= j_last) {
          const uint32_t n = quotient(j, p.page), page = __ldg(p.table + (size_t)at.seq * p.width + n);
          if (page < p.pages) r = (page * p.kv_heads + kvh) * p.page.d + j - n * p.page.d;
          else raise(p.error, PAGED_BAD_PAGE);
        }
        rows[t & 1][x] = r;
      }
    };
    auto request = [&](const void *cache, uint32_t dst, uint32_t t) {
#pragma unroll 8
      for (uint32_t i = 0; i < kKeys / RS; ++i) {
        const uint32_t row = i * RS + frow, r = rows[t & 1][row];
        const bool there = r != 0xffffffffu && col_there;
        copy16(dst + place(row), static_cast<const uint16_t *>(cache) + (there ? (size_t)r * p.dim + col * 8 : 0), there);
      }
      copy_commit();
    };
    look_up(t0);
#pragma unroll 4
    for (uint32_t i = 0; i < tiles * kRows / RS; ++i) {
      const uint32_t row = i * RS + frow, r = at.first + row;
      const bool there = r < packed && col_there;
      const uint32_t rt = r / per;
      const uint16_t *src = static_cast<const uint16_t *>(p.q);
      copy16(q_a + (row >> 7) * C::kTile + place(row & 127), there ? src + (at.row0 + rt) * p.q_ld + (kvh * per + r - rt * per) * p.dim + col * 8 : src, there);
    }
    copy_commit();
    __syncwarp();
    request(p.kcache, k_a, t0);
    copy_wait<1>();
    landed(&q_full);
    // a tile's values are requested before its keys have landed, the next tile's keys before its values have
    bool ok = true;
    for (uint32_t t = t0; t < t1; ++t) {
      const uint32_t n = t - t0, s = n % kStages, parity = (n / kStages + 1) & 1;  // of the stage's last release
      if (n >= kStages && !(ok = wait_warp(&v_empty[s], parity))) break;
      request(p.vcache, v_a + s * C::kTile, t);
      copy_wait<1>();
      landed(&k_full[s]);
      if (t + 1 < t1) {
        look_up(t + 1);  // its place was last read for tile t - 1
        __syncwarp();
        const uint32_t n1 = n + 1, s1 = n1 % kStages;
        if (n1 >= kStages && !(ok = wait_warp(&k_empty[s1], (n1 / kStages + 1) & 1))) break;
        request(p.kcache, k_a + s1 * C::kTile, t + 1);
        copy_wait<1>();
      } else {
        copy_wait<0>();
      }
      landed(&v_full[s]);
    }
    copy_wait<0>();
  } else if (warp == kMmaWarp) {
    // ----------------------------------------------------------------------------------------------------------- MMA
    if (elect_one()) {
      constexpr uint32_t idesc_s = instr_desc(kRows, kKeys, BF), idesc_o = instr_desc(kRows, DP, BF) | 1u << 16;  // the second: B is MN-major
      const uint32_t q0 = desc_lo(q_a), k0 = desc_lo(k_a);
      const uint32_t v0 = ((v_a & 0x3FFFFu) >> 4) | (128u * 128 >> 4) << 16;  // 64 dimensions are 16 KB from the next 64
      bool ok = wait(&q_full, 0);
      uint32_t p_phase = 0;  // bit i
      // Before tile t's turn: S of t for the tiles of rows that see it.
      auto scores = [&](uint32_t i, uint32_t t) {
        const uint32_t st = ((t - t0) % kStages) * (C::kTile >> 4), qi = q0 + i * (C::kTile >> 4);
#pragma unroll
        for (uint32_t k = 0; k < DP / 16; ++k) {
          const uint32_t off = (k >> 2) * (128 * 128 >> 4) + (k & 3) * 2;
          mma_f16<1>(tmem + i * 128, qi + off, k0 + st + off, idesc_s, k != 0);
        }
        mma_commit(sa(&s_full[i]));
      };
      // t0 - 1 stands for what comes before the first tile
      for (uint32_t n = 0; ok && n <= t1 - t0; ++n) {
        const uint32_t t = t0 + n;  // scores of t, output of t - 1
        bool keys = false;
        if (n > 0 && !(ok = wait(&v_full[(n - 1) % kStages], ((n - 1) / kStages) & 1))) break;
        for (uint32_t i = 0; ok && i < tiles; ++i) {
          if (n > 0 && t - 1 >= b[i] && t - 1 < e[i]) {
            if (!(ok = wait(&p_full[i], p_phase >> i & 1))) break;
            p_phase ^= 1u << i;
            tc_after();
            const uint32_t st = v0 + ((n - 1) % kStages) * (C::kTile >> 4);
#pragma unroll
            for (uint32_t k = 0; k < kKeys / 16; ++k)
              mma_tmem(tmem + 256 + i * DP, tmem + i * 128 + k * 8, st + k * (2048 >> 4), idesc_o, k != 0 || t - 1 > b[i]);
            if (t == e[i]) mma_commit(sa(&o_full[i]));
          }
          if (t < t1 && t >= b[i] && t < e[i]) {
            if (!keys && !(ok = wait(&k_full[n % kStages], (n / kStages) & 1))) break;
            keys = true;
            tc_after();
            scores(i, t);
          }
        }
        if (!ok) break;
        if (n > 0) mma_commit(sa(&v_empty[(n - 1) % kStages]));
        if (t < t1) {
          if (!keys && !(ok = wait(&k_full[n % kStages], (n / kStages) & 1))) break;  // nobody sees it (between windows): still given back
          mma_commit(sa(&k_empty[n % kStages]));
        }
      }
    }
    __syncwarp();
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (tid == 0 && failed_s) raise(p.error, kWaitCode);
  stamp_end(p.stamps);
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <bool BF, int DP> cudaError_t run(const PagedAttention &p, cudaStream_t s) {
  const uint64_t per = p.heads / p.kv_heads, tiles = p.rows * per / (2 * kRows) + std::min<uint64_t>(p.n, p.rows * per);
  return launch_following(paged_prompt_tc_kernel<BF, DP>, dim3((uint32_t)tiles, p.kv_heads), kThreads, Cfg<DP>::kSmem, s, p);
}
template <bool BF, int DP> cudaError_t setup_one() {
  return cudaFuncSetAttribute(paged_prompt_tc_kernel<BF, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg<DP>::kSmem);
}

}  // namespace

cudaError_t setup_paged_prompt_tc() {
  for (cudaError_t e : {setup_one<false, 64>(), setup_one<false, 128>(), setup_one<true, 64>(), setup_one<true, 128>()})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}
cudaError_t launch_paged_prompt_tc(const PagedAttention &p, cudaStream_t s) {
  if (p.dim <= 64) return p.bf ? run<true, 64>(p, s) : run<false, 64>(p, s);
  return p.bf ? run<true, 128>(p, s) : run<false, 128>(p, s);
}

}  // namespace vkl
