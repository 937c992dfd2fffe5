// Attention of several new rows per sequence (paged_prompt.cu) on the 5th-generation tensor cores, for heads up to 128 wide.
//
// A CTA has 256 packed rows of a sequence and key head, as two tiles of 128, and walks over the positions that they see in tiles of
// 128. Per tile of rows i and positions j: S_i = Q_i K_j^T (tcgen05.mma, fp32 in TMEM), P_i = 2^(scale S_i - reference) as 16-bit numbers
// written over S_i in TMEM, O_i += P_i V_j with P as the TMEM operand. The two tiles of rows take turns: while the tensor core works
// for one, the exponentials of the other are computed, which take as long (16 per clock and SM: 1024 cycles for 128 x 128, like the two
// products). A CTA stays on its SM and takes one such item after the other by tickets, what takes longest first: a new CTA per item costs some
// 10 us of start and end, in which nothing else runs (64 prompts of 256: 210 us, this way 106; both on a cool GPU, under full load 123). That a reference
// follows its maximum only after some growth, and that two tiles of rows take turns, are published ways of attention on tensor cores. Warps:
//   0-3, 4-7  softmax of tile 0, 1: one thread per row, so no exchange between threads. The reference is the row's maximum as of the last time
//             that it grew by more than 2^8 (fp16: 2^4): until then the probabilities stay below that and O as it is; only then O is multiplied. In fp16,
//             which ends at steps of 2^-24, they are 2^11 times as large, in sum and O alike: their rounding is relative (2^-11) down to 2^-25
//             of the row's largest, and below each is off by 2^-36 of the largest at most.
//   8, 9      fetch K_j and V_j into a ring, by tensor copies of boxes of rows and, where pages have none, by cp.async; in the 128-byte
//             swizzle of the matrix descriptors: K is K-major and V, as it lies in the cache, MN-major (64 dimensions of a position are a
//             row of 128 bytes in both).
//   10        issues the MMAs. They complete in order, so the commit behind S_i(j + 1) also says that P_i(j) V_j is in O_i.
//   11        takes the tickets and fetches Q, so that queries, keys and values of the next item are there when this one's output is stored.
// Every wait is bounded: a step's after some seconds, an item's, and all of a CTA that computes rows again, after minutes (for items of up to 2^31
// positions, and rows of some ten million), or when another one has run out. Then all warps leave, and the error word is raised.
#include <algorithm>

#include "paged_rows.cuh"
#include "tcgen05.cuh"

namespace vkl {
namespace {

constexpr uint32_t kSoftmaxWarps = 8, kFetchWarps = 2, kMmaWarp = 10, kThreads = 12 * 32;  // more than 12 warps would have 128 registers each
constexpr uint32_t kRows = 128, kKeys = 128;
constexpr uint32_t kWaitCode = 9, kPolls = 1u << 20, kRounds = 64, kLongPolls = 1u << 30;
// Where there are fewer items than SMs, an item's positions are split, into slices of at least kSliceTiles tiles; the sums of a row's slices meet
// in a kernel of their own.
constexpr uint32_t kSliceTiles = 4, kMostSplits = 32;
constexpr uint32_t kAsideTiles = kManyPositions / kKeys;
template <int DP> constexpr uint32_t kAsideRow = DP + 4;  // numbers of a row's sums put aside: outputs, their reference, the sum of probabilities
// Octaves that a maximum grows by before the reference follows, and that probabilities are raised by: together 2^15, of 2^16 that fp16 has. (Of normally
// distributed scores, 32 rows of 4096 positions, 0.1 % of the tiles let O be multiplied; with 2^3 2.4 %, and 4096 rows take 165 us instead of 163.)
template <bool BF> constexpr float kGrown = BF ? 8.0f : 4.0f;
template <bool BF> constexpr float kRaise = BF ? 0.0f : 11.0f;
// Registers of a thread: a softmax thread has a row of scores in registers, the other warps give theirs. The sum has to be below what the launch has.
constexpr uint32_t kSoftmaxRegs = 208, kOtherRegs = 80, kLaunchRegs = kSoftmaxWarps * 32 * kSoftmaxRegs + (kThreads - kSoftmaxWarps * 32) * kOtherRegs;

// What a CTA works on: 256 packed rows of a sequence and key head, as one or two tiles, and the tiles of positions [b, e) that each of them sees.
struct Item {
  Place at;
  uint32_t found, kvh, tiles, b[2], e[2];
  uint32_t slice, slices;  // of the tiles of positions, this one's and how many
};

template <int DP> struct Cfg {
  static constexpr uint32_t kTile = 128 * DP * 2;  // bytes of 128 rows
  // One CTA per SM, which takes all of its TMEM: more than half of the shared memory, whatever the head width. K and V tiles take
  // turns in one ring: with two places each (373 -> 238 us) the MMAs still waited 1000 of 4000 cycles a tile for keys.
  static constexpr uint32_t kStages = DP == 64 ? 8 : 5;
  struct Shared {  // behind the tiles
    uint64_t q_full[2], q_empty[2], full[kStages], empty[kStages], s_full[2], p_full[2][2], o_full[2], turn[2][4], item_full[2], item_empty[2], fetched, drained;
    Item items[2];
    uint32_t tmem;
    // going: 0 once a wait has run out; slow: rows have been computed again. Words that, where they are not 0, make waits long.
    volatile uint32_t going, slow;
  };
  static constexpr uint32_t kSmem = (2 + kStages) * kTile + sizeof(Shared);
  static_assert(kSmem > 114 * 1024 && kSmem <= 227 * 1024, "one CTA per SM");
};

__device__ __forceinline__ void mma_tmem(uint32_t acc, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, bool accumulate) {
  constexpr uint32_t hi = (1024u >> 4) | 1u << 14 | 2u << 29;  // as mma_f16's
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 b;\n mov.b64 b, {%2, %3};\n setp.ne.b32 p, %5, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}" ::"r"(acc), "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
               "r"(r[14]), "r"(r[15])
               : "memory");
}
// A thread's 128 columns. The wait is part of the statement, so that nothing touches the registers before it.
__device__ __forceinline__ void tmem_ld128(uint32_t taddr, uint32_t (&r)[128]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x128.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,"
      "%58,%59,%60,%61,%62,%63,%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,%80,%81,%82,%83,%84,%85,"
      "%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,"
      "%111,%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127"
      "}, [%128];\n tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]),
        "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]),
        "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]),
        "=r"(r[61]), "=r"(r[62]), "=r"(r[63]), "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]),
        "=r"(r[71]), "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]), "=r"(r[80]),
        "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]), "=r"(r[88]), "=r"(r[89]), "=r"(r[90]),
        "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]), "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]),
        "=r"(r[101]), "=r"(r[102]), "=r"(r[103]), "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]),
        "=r"(r[111]), "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]), "=r"(r[120]),
        "=r"(r[121]), "=r"(r[122]), "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ uint64_t pair_of(float a, float b) { return (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a); }
__device__ __forceinline__ float2 of_pair(uint64_t v) { return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void mbar_wait_short(uint32_t bar, uint32_t parity) {
  uint32_t ok = 0;
  for (uint32_t i = 0; !ok && i < 1u << 14; ++i)
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, uint32_t x, uint32_t y, uint32_t z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void store32(void *to, const uint32_t *v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&u)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n tcgen05.wait::ld.sync.aligned;"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]),
                 "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
               : "r"(taddr)
               : "memory");
}
// Sixteen columns times c.
__device__ __forceinline__ void rescale16(uint32_t taddr, float c) {
  uint32_t u[16];
  tmem_ld16(taddr, u);
#pragma unroll
  for (int x = 0; x < 16; ++x) u[x] = __float_as_uint(__uint_as_float(u[x]) * c);
  tmem_st16(taddr, u);
}

// A row's sums, relative to `ref`, out of the way: added to what is there (unless this is the first time), and 0 from here on. Or back, added to what came since.
template <int DP, bool BACK> __device__ __forceinline__ void put_aside(float *there, bool first, uint32_t o_t, float ref, float &sum) {
  if (!first) {  // it has long left the caches
#pragma unroll
    for (uint32_t d = 0; d < DP + 2; d += 32) asm volatile("prefetch.global.L1 [%0];" ::"l"(there + d));
  }
  const float2 ml = first ? make_float2(0.f, 0.f) : *reinterpret_cast<const float2 *>(there + DP);  // reference, sum of probabilities
  const float c = ml.y == 0.f ? 0.f : exp2_fast(ml.x - ref);  // nothing was seen until then, and the reference stands for nothing
  sum += ml.y * c;
#pragma unroll 2
  for (uint32_t d = 0; d < DP; d += 16) {
    uint32_t u[16];
    tmem_ld16(o_t + d, u);
#pragma unroll
    for (int x = 0; x < 16; x += 4) {
      float4 *at = reinterpret_cast<float4 *>(there + d + x), v = first ? make_float4(0.f, 0.f, 0.f, 0.f) : *at;
      v.x = v.x * c + __uint_as_float(u[x]), v.y = v.y * c + __uint_as_float(u[x + 1]);
      v.z = v.z * c + __uint_as_float(u[x + 2]), v.w = v.w * c + __uint_as_float(u[x + 3]);
      if (!BACK) *at = v;
      u[x] = BACK ? __float_as_uint(v.x) : 0, u[x + 1] = BACK ? __float_as_uint(v.y) : 0;
      u[x + 2] = BACK ? __float_as_uint(v.z) : 0, u[x + 3] = BACK ? __float_as_uint(v.w) : 0;
    }
    tmem_st16(o_t + d, u);
  }
  tmem_stored();
  if (!BACK) {
    *reinterpret_cast<float2 *>(there + DP) = make_float2(ref, sum);
    sum = 0.f;
  }
}

// SPLIT: p.splits > 1. (One kernel for both costs 0.4 us an item.) MANY: p.aside, every kAsideTiles tiles a row's sums are added to what
// lies there, in 32 bits as everywhere but rounded (bf16, 1024 rows behind 100,000 positions, 32 heads of 128 over 8: 1.5 % more on a cool GPU).
template <bool BF, int DP, bool SPLIT, bool MANY> __global__ void __launch_bounds__(kThreads, 1)
    paged_prompt_tc_kernel(const PagedAttention p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                           const __grid_constant__ CUtensorMap map_q, const uint32_t box, const bool q_box) {
  using C = Cfg<DP>;
  extern __shared__ __align__(1024) unsigned char smem[];
  typename C::Shared &sh = *reinterpret_cast<typename C::Shared *>(smem + (2 + C::kStages) * C::kTile);
  auto &q_full = sh.q_full, &s_full = sh.s_full, &o_full = sh.o_full;
  auto &full = sh.full, &empty = sh.empty;
  auto &p_full = sh.p_full;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, per = p.heads / p.kv_heads;
  if (tid == 0) {
    auto init = [](uint64_t *bar, uint32_t n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(sa(bar)), "r"(n) : "memory"); };
    for (uint32_t s = 0; s < C::kStages; ++s) init(&full[s], 1), init(&empty[s], 1);
    for (uint32_t i = 0; i < 2; ++i) init(&q_full[i], 1), init(&sh.q_empty[i], 1), init(&s_full[i], 1), init(&p_full[i][0], 4), init(&p_full[i][1], 4), init(&o_full[i], 1);
    for (uint32_t i = 0; i < 2; ++i) init(&sh.item_full[i], 1), init(&sh.item_empty[i], kSoftmaxWarps + kFetchWarps + 1);
    init(&sh.fetched, kFetchWarps);
    init(&sh.drained, 1);
    for (uint32_t i = 0; i < 8; ++i) init(&sh.turn[i >> 2][i & 3], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    sh.going = 1, sh.slow = 0;
  }
  if (warp == kMmaWarp) tmem_alloc<512>(sa(&sh.tmem));
  tc_before();
  __syncthreads();
  tc_after();
  follow();
  if (p.part != 2) stamp_begin(p.stamps);  // else the launch in front of this one did
  const uint32_t tmem = sh.tmem, q_a = sa(smem), ring_a = q_a + 2 * C::kTile;
  // Waits, false when they ran out: after kPolls (4 us each: try_wait sleeps), or after kRounds times as many as long as the word `longer` is not 0.
  // The loop is one statement, with nothing behind a wait that is over: these instructions are between every two steps of a tile (checks in C++
  // behind it: 108 us where 103 are possible).
  auto wait = [&](uint64_t *bar, uint32_t parity, const volatile uint32_t &longer) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p, q;\n .reg .u32 n, m;\n mov.u32 n, %3;\n"
        "again:\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n @p bra there;\n sub.u32 n, n, 1;\n and.b32 m, n, %4;\n setp.ne.u32 q, m, 0;\n @q bra again;\n"
        " ld.volatile.shared.u32 m, [%5];\n setp.eq.u32 q, m, 0;\n @q bra there;\n setp.ne.u32 q, n, 0;\n @q bra again;\n"
        "there:\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(sa(bar)), "r"(parity), "n"(kPolls * kRounds), "n"(kPolls - 1), "r"(sa(const_cast<uint32_t *>(&longer)))
        : "memory");
    if (!ok) sh.going = 0;
    return ok != 0;
  };
  // For waits that are long by design: a warp that polls takes issue slots from the softmax warps of its scheduler (the ticket warp alone
  // cost a third of the rate). That one waits for whole items, which may have millions of positions.
  auto wait_idle = [&](uint64_t *bar, uint32_t parity, uint32_t ns, bool item = false) {
    uint32_t ok = 0;
    for (uint32_t n = 0; !ok && n < ((item ? sh.going : sh.slow) ? kLongPolls : item ? 0 : kPolls); ++n) {
      asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(sa(bar)), "r"(parity) : "memory");
      if (!ok) __nanosleep(ns);
    }
    if (!ok) sh.going = 0;
    return __all_sync(0xffffffffu, ok) != 0;
  };
  auto wait_warp = [&](uint64_t *bar, uint32_t parity, const volatile uint32_t &longer) { return __all_sync(0xffffffffu, wait(bar, parity, longer)) != 0; };  // the lanes agree

  // Item k of this CTA; null when the wait ran out.
  auto item = [&](uint32_t k) { return wait_warp(&sh.item_full[k & 1], k >> 1 & 1, sh.going) ? &sh.items[k & 1] : nullptr; };
  auto item_done = [&](uint32_t k) {
    __syncwarp();
    if (lane == 0) arrive(sa(&sh.item_empty[k & 1]));
  };

  if (warp < kSoftmaxWarps) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));

  if (warp < kSoftmaxWarps) {
    // ------------------------------------------------------------------------------------------------------- softmax
    const uint32_t i = warp >> 2, quad = warp & 3;
    uint32_t scores = 0, output = 0, turn = 0;  // parities of the barriers, over all items
    bool ok = true;
    for (uint32_t k = 0; ok; ++k) {
      const Item *it = item(k);
      if (!it || !it->found) break;
      const Place at = it->at;
      const uint32_t kvh = it->kvh, tiles = it->tiles, both_b = it->b[1], both_e = it->e[0];  // positions of both tiles, where there are two
      if (i < tiles) {
        const uint32_t packed = at.fresh * per, past = at.len - at.fresh, bi = it->b[i], ei = it->e[i];
        const uint32_t r = at.first + tid, w0 = min(at.first + warp * 32, packed - 1), w1 = min(w0 + 31, packed - 1);
        const uint32_t pos = past + quotient(min(r, packed - 1), p.group), w_lo = past + quotient(w0, p.group), w_hi = past + quotient(w1, p.group);
        const uint32_t w_first = p.window && w_hi + 1 > p.window ? w_hi + 1 - p.window : 0;  // every row of the warp sees [w_first, w_lo]
        const uint32_t first = p.window && pos + 1 > p.window ? pos + 1 - p.window : 0;
        const float scale = fabsf(p.scale) * kLog2e;  // a negative scale is the MMA's negated operand
        const uint32_t lanes = (quad * 32u) << 16, s_t = tmem + lanes + i * 128, o_t = tmem + lanes + 256 + i * DP;
        float top = -INFINITY, ref = 0.f, sum = 0.f;  // the reference, and what is subtracted from scaled scores (0 where it is -infinity)
        for (uint32_t t = bi; t < ei; ++t, scores ^= 1) {
          if (!(ok = wait_warp(&s_full[i], scores, sh.slow))) break;
          tc_after();
          uint32_t u[128];
          tmem_ld128(s_t, u);
          if (t * kKeys + kKeys - 1 > w_lo) {  // positions that some row of the warp does not see yet
            const int hi = (int)pos - (int)(t * kKeys);
#pragma unroll
            for (int x = 0; x < 128; ++x)
              if (x > hi) u[x] = 0xff800000u;
          }
          if (t * kKeys < w_first) {  // and no more
            const int lo = (int)first - (int)(t * kKeys);
#pragma unroll
            for (int x = 0; x < 128; ++x)
              if (x < lo) u[x] = 0xff800000u;
          }
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (uint32_t x = 0; x < 128; x += 8)
#pragma unroll
            for (uint32_t y = 0; y < 4; ++y) m4[y] = max3(m4[y], __uint_as_float(u[x + y]), __uint_as_float(u[x + 4 + y]));
          const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
          if (t == bi) {
            top = m;
            ref = m == -INFINITY ? 0.f : m * scale;
          } else {
            const bool grown = m * scale - ref > kGrown<BF> || (top == -INFINITY && m != -INFINITY);
            const bool due = MANY && (t - bi) % kAsideTiles == 0;
            if (__any_sync(0xffffffffu, grown || due)) {
              if (due) put_aside<DP, false>(p.aside + ((size_t)blockIdx.x * kSoftmaxWarps * 32 + tid) * kAsideRow<DP>, t - bi == kAsideTiles, o_t, ref, sum);
              float c = 1.0f;
              if (grown) {
                c = exp2_fast((top - m) * scale);
                top = m;
                ref = m * scale;
              }
              sum *= c;
#pragma unroll 1
              for (uint32_t d = 0; d < DP; d += 16) rescale16(o_t + d, c);
              tmem_stored();
            }
          }
          // The special function unit of a scheduler belongs to one tile's warp at a time: the other's products run meanwhile.
          const bool shared_tile = tiles == 2 && t >= both_b && t < both_e;
          if (shared_tile && (i || t > both_b)) {
            if (!(ok = wait_warp(&sh.turn[i][quad], turn, sh.slow))) break;
            turn ^= 1;
          }
          const uint64_t scale2 = pair_of(scale, scale), ref2 = pair_of(kRaise<BF> - ref, kRaise<BF> - ref);
          uint64_t sum2[2] = {0, 0};
#pragma unroll
          for (uint32_t c = 0; c < 4; ++c) {
            uint32_t w[16];
#pragma unroll
            for (uint32_t x = 0; x < 16; ++x) {
              const uint64_t y = fma_pair(pair_of(__uint_as_float(u[c * 32 + 2 * x]), __uint_as_float(u[c * 32 + 2 * x + 1])), scale2, ref2);
              const float2 v = of_pair(y);
              const float a = exp2_fast(v.x), z = exp2_fast(v.y);
              sum2[x & 1] = add_pair(sum2[x & 1], pair_of(a, z));
              w[x] = pack2<BF>(a, z);
            }
            tmem_st16(s_t + c * 16, w);
            if (c == 1) {  // the product with the first 64 positions' values can begin
              tmem_stored();
              tc_before();
              __syncwarp();
              if (lane == 0) arrive(sa(&p_full[i][0]));
            }
          }
          if (shared_tile && lane == 0) arrive(sa(&sh.turn[i ^ 1][quad]));
          const float2 part = of_pair(add_pair(sum2[0], sum2[1]));
          sum += part.x + part.y;
          tmem_stored();
          tc_before();
          __syncwarp();
          if (lane == 0) arrive(sa(&p_full[i][1]));
        }
        if (ok) ok = wait_warp(&o_full[i], output, sh.slow);
        output ^= 1;
        if (ok) {
          tc_after();
          if (MANY && bi + kAsideTiles < ei)
            put_aside<DP, true>(p.aside + ((size_t)blockIdx.x * kSoftmaxWarps * 32 + tid) * kAsideRow<DP>, false, o_t, ref, sum);
          const float inv = 1.0f / sum;
          const uint32_t row = min(r, packed - 1), rt = quotient(row, p.group);
          const size_t to = (size_t)(at.row0 + rt) * p.heads + kvh * per + row - rt * per;
          uint16_t *out = static_cast<uint16_t *>(p.out) + to * p.dim;
          float finite = 0.f;
          if (SPLIT && it->slices > 1) {  // a part of the row's positions
            const size_t part = (size_t)it->slice * p.rows * p.heads + to;
            if (r < packed) p.part_ml[part] = make_float2(ref, sum == 0.f ? -1.f : sum);  // 0 is a part that there is not
#pragma unroll
            for (uint32_t d = 0; d < DP; d += 32) {
              uint32_t u[32];
              tmem_ld32(o_t + d, u);
              if (r < packed) {
#pragma unroll
                for (uint32_t x = 0; x < 32; x += 8) store32(p.part_o + part * DP + d + x, u + x);
              }
            }
          } else
#pragma unroll
          for (uint32_t d = 0; d < DP; d += 32) {
            uint32_t u[32], w[16];
            tmem_ld32(o_t + d, u);
#pragma unroll
            for (uint32_t x = 0; x < 16; ++x) {
              const float a = __uint_as_float(u[2 * x]) * inv, z = __uint_as_float(u[2 * x + 1]) * inv;
              finite += a * 0.f + z * 0.f;
              w[x] = pack2<BF>(a, z);
            }
            if (r < packed) {
#pragma unroll
              for (uint32_t x = 0; x < 32; x += 16) {  // whole sectors where rows begin at them
                const uint32_t *v = w + x / 2;
                if (p.dim % 16 == 0) {
                  if (d + x < p.dim) store32(out + d + x, v);
                } else {
                  if (d + x < p.dim) *reinterpret_cast<uint4 *>(out + d + x) = make_uint4(v[0], v[1], v[2], v[3]);
                  if (d + x + 8 < p.dim) *reinterpret_cast<uint4 *>(out + d + x + 8) = make_uint4(v[4], v[5], v[6], v[7]);
                }
              }
            }
          }
          uint32_t again = __ballot_sync(0xffffffffu, finite != 0.f && r < packed);  // NaN
          __syncwarp();
          if (again) sh.slow = 1;
          for (; again; again &= again - 1) row_again<BF>(p, at, kvh, at.first + warp * 32 + __ffs(again) - 1, 0, DP);
        }
      }
      if (i == 0 && tiles == 2 && both_e > both_b) turn ^= 1;  // the other tile's last turn, which nobody waits for
      item_done(k);
    }
  } else if (warp < kSoftmaxWarps + kFetchWarps) {
    // ------------------------------------------------------------------------------------- fetch: keys one warp, values the other
    constexpr uint32_t CH = DP / 8, RS = 32 / CH, BLOCKS = DP / 64;  // pieces of a row; rows at a time
    const uint32_t values = warp - kSoftmaxWarps, col = lane % CH, frow = lane / CH;
    const bool col_there = col * 8 < p.dim;
    const uint16_t *cache = static_cast<const uint16_t *>(values ? p.vcache : p.kcache);
    const CUtensorMap *map = values ? &map_v : &map_k;
    // A tile is fetched in boxes of rows that lie in one page, by tensor copies. Scores of positions that a row does not see are masked, so keys are
    // fetched with what lies behind the last position in its box, or left as they are where there are no positions at all. Values meet
    // probabilities of 0 there, which takes finite ones: zeros (of rows behind the cache), and in the last position's box a copy piece by piece.
    // So go all rows of pages of which no eight make a box. (All of a tile with a ragged end piece by piece: 64 prompts of 96 105 us, of 200 149, of 300
    // 276.)
    const uint32_t boxes = box ? kKeys / box : 0, box_log = box ? __ffs(box) - 1 : 0, rows_all = p.pages * p.kv_heads * p.page.d;
    uint64_t *late = nullptr;  // pieces by cp.async are reported behind the next request
    auto landed = [&]() {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the tensor core may read them
      __syncwarp();
      if (lane == 0) arrive(sa(late));
      late = nullptr;
    };
    RingPos<(int)C::kStages> pos;  // an item's tiles make requests in turn: keys, values, keys, ...
    if (values) pos.next();
    uint32_t x = values;
    bool ok = true;
    for (uint32_t k = 0; ok; ++k) {
      const Item *it = item(k);
      if (!it || !it->found) break;
      const uint32_t packed = it->at.fresh * per, past = it->at.len - it->at.fresh, kvh = it->kvh, len = it->at.len, t0 = it->b[0], t1 = it->e[1];
      const uint32_t lo_pos = past + quotient(it->at.first, p.group), j_first = p.window && lo_pos + 1 > p.window ? lo_pos + 1 - p.window : 0;
      const uint32_t j_last = past + quotient(min(it->at.first + 2 * kRows, packed) - 1, p.group);
      const uint32_t *pages = p.table + (size_t)it->at.seq * p.width;
      auto cache_row = [&](uint32_t j) {  // of position j; behind the last one where there is none
        const uint32_t n = quotient(j, p.page), page = pages[n];
        if (page < p.pages) return (page * p.kv_heads + kvh) * p.page.d + j - n * p.page.d;
        raise(p.error, PAGED_BAD_PAGE);
        return 0xffffffffu;
      };
      uint32_t look_row = 0;
      auto look_up = [&](uint32_t t) {  // lane x: box x of a tile
        const uint32_t j = t * kKeys + lane * box;
        look_row = lane < boxes && j + box > j_first && j < len ? cache_row(j) : 0xffffffffu;
      };
      look_up(t0);
      for (uint32_t t = t0; t < t1; ++t, x += 2, pos.next(), pos.next()) {
        const uint32_t my_row = min(look_row, rows_all), j0 = t * kKeys;  // a row behind the cache reads as zeros
        // boxes [lo, hi) hold positions, [lo, whole) nothing else; [first, last) are copied, rows [r0, r1) go piece by piece
        const uint32_t lo = j_first > j0 ? (j_first - j0) >> box_log : 0, left = len > j0 ? min(len - j0, kKeys) : 0;
        const uint32_t hi = box ? (left + box - 1) >> box_log : 0, whole = left >> box_log;
        const uint32_t first = values ? 0 : lo, last = values ? boxes : hi;
        const uint32_t r0 = values ? whole * box : 0, r1 = !box ? kKeys : values ? hi * box : 0;
        const uint32_t copied = last > first ? last - first - (r1 > r0 && box ? 1 : 0) : 0;
        if (t1 - t == min(t1 - t0, 2u) && lane == 0) arrive(sa(&sh.fetched));  // the next ticket may be taken
        if (x >= C::kStages && !(ok = wait_idle(&empty[pos.s], pos.phase ^ 1, 64))) break;
        const uint32_t dst = ring_a + pos.s * C::kTile, bar = sa(&full[pos.s]);
        const bool pieces = r1 > r0;
        if (copied) {
          if (elect_one()) asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(copied * box * DP * 2) : "memory");
          for (uint32_t g = first; g < last; ++g) {
            if (pieces && g == whole) continue;
            const uint32_t row = __shfl_sync(0xffffffffu, my_row, g);
            if (elect_one()) {  // one lane, known to the compiler: copies from several lanes at once became a loop, 2000 cycles a tile
#pragma unroll
              for (uint32_t k = 0; k < BLOCKS; ++k) tma_load_2d(dst + k * (128 * 128) + g * box * 128, map, k * 64, row, bar);
            }
          }
        }
        if (pieces) {
#pragma unroll 4
          for (uint32_t row = r0 + frow; row < r1; row += RS) {
            const uint32_t j = j0 + row, r = j >= j_first && j <= j_last ? cache_row(j) : 0xffffffffu;
            const bool there = r != 0xffffffffu && col_there;
            copy16(dst + (col >> 3) * (128 * 128) + row * 128 + (((col & 7) ^ (row & 7)) << 4), cache + (there ? (size_t)r * p.dim + col * 8 : 0), there);
          }
        }
        copy_commit();
        if (late) {
          copy_wait<1>();
          landed();
        }
        if (pieces) {
          late = &full[pos.s];
        } else {
          __syncwarp();
          if (lane == 0) arrive(bar);
        }
        if (t + 1 < t1) look_up(t + 1);
      }
      copy_wait<0>();
      if (late) landed();
      item_done(k);
    }
    if (!sh.going && lane == 0) {  // nothing may land when the CTA has gone
      for (uint32_t y = x > C::kStages ? x - C::kStages : 0; y < x; ++y)
        if ((y & 1) == values) mbar_wait_short(sa(&full[y % C::kStages]), y / C::kStages & 1);
    }
  } else if (warp == kMmaWarp) {
    // ----------------------------------------------------------------------------------------------------------- MMA
    if (elect_one()) {
      const uint32_t idesc_s = instr_desc(kRows, kKeys, BF) | (p.scale < 0.f ? 1u << 13 : 0u);  // negates A
      constexpr uint32_t idesc_o = instr_desc(kRows, DP, BF) | 1u << 16;  // the second: B is MN-major
      const uint32_t q0 = desc_lo(q_a), k0 = desc_lo(ring_a);
      const uint32_t v0 = ((ring_a & 0x3FFFFu) >> 4) | (128u * 128 >> 4) << 16;  // 64 dimensions are 16 KB from the next 64
      bool ok = true;
      uint32_t p_phase = 0, q_phase = 0;    // bit i, over all items
      RingPos<(int)C::kStages> keys, vals;  // a tile's keys are an even request, its values the one behind
      vals.next();
      for (uint32_t k = 0; ok; ++k) {
        if (!(ok = wait(&sh.item_full[k & 1], k >> 1 & 1, sh.going))) break;
        const Item &it = sh.items[k & 1];
        if (!it.found) break;
        const uint32_t tiles = it.tiles, b[2] = {it.b[0], it.b[1]}, e[2] = {it.e[0], it.e[1]}, t0 = b[0], t1 = e[1];  // registers: the loops over i are unrolled
        // step n: output of tile t - 1, scores of tile t, for one tile of rows after the other
        for (uint32_t n = 0; ok && n <= t1 - t0; ++n) {
          const uint32_t t = t0 + n;
          bool waited = false;
          if (n > 0 && !(ok = wait(&full[vals.s], vals.phase, sh.slow))) break;
#pragma unroll
          for (uint32_t i = 0; i < 2; ++i) {
            if (!ok || i >= tiles) break;
            if (n > 0 && t - 1 >= b[i] && t - 1 < e[i]) {
              const uint32_t st = v0 + vals.s * (C::kTile >> 4), parity = p_phase >> i & 1;
              p_phase ^= 1u << i;
#pragma unroll
              for (uint32_t half = 0; half < 2; ++half) {
                if (!(ok = wait(&p_full[i][half], parity, sh.slow))) break;
                tc_after();
#pragma unroll
                for (uint32_t k = half * 4; k < half * 4 + 4; ++k)
                  mma_tmem(tmem + 256 + i * DP, tmem + i * 128 + k * 8, st + k * (2048 >> 4), idesc_o, k != 0 || t - 1 > b[i]);
              }
              if (!ok) break;
              if (t == e[i]) mma_commit(sa(&o_full[i]));
            }
            if (n > 0 && i + 1 == tiles) mma_commit(sa(&empty[vals.s]));
            if (t < t1 && t >= b[i] && t < e[i]) {
              if (t == b[i]) {
                if (!(ok = wait(&q_full[i], q_phase >> i & 1, sh.slow))) break;
                q_phase ^= 1u << i;
              }
              if (!waited && !(ok = wait(&full[keys.s], keys.phase, sh.slow))) break;
              waited = true;
              tc_after();
              const uint32_t st = k0 + keys.s * (C::kTile >> 4), qi = q0 + i * (C::kTile >> 4);
#pragma unroll
              for (uint32_t k = 0; k < DP / 16; ++k) {
                const uint32_t off = (k >> 2) * (128 * 128 >> 4) + (k & 3) * 2;
                mma_f16<1>(tmem + i * 128, qi + off, st + off, idesc_s, k != 0);
              }
              mma_commit(sa(&s_full[i]));
              if (t + 1 == e[i]) mma_commit(sa(&sh.q_empty[i]));
            }
          }
          if (!ok) break;
          if (t < t1) {
            if (!waited && !(ok = wait(&full[keys.s], keys.phase, sh.slow))) break;  // nobody sees it (between windows): still given back
            mma_commit(sa(&empty[keys.s]));
            keys.next(), keys.next();
          }
          if (n > 0) vals.next(), vals.next();
        }
        arrive(sa(&sh.item_empty[k & 1]));
      }
      if (!ok) {  // nothing may be in work when the TMEM is given back
        mma_commit(sa(&sh.drained));
        mbar_wait_short(sa(&sh.drained), 0);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------- what comes next, once two tiles of this item are left to request: a ticket taken much earlier
    // could have been another CTA's, which has nothing left to do (106 -> 158 us for a few long items)
    if (blockIdx.x == 0) check_rows(p);
    uint32_t used[2] = {};  // how often each tile's place for Q
    Walk walk;
    uint32_t ticket = blockIdx.x;  // the first ones are dealt out
    auto take = [&]() {
      uint32_t next = 0;
      if (lane == 0) next = gridDim.x + atomicAdd(p.tickets, 1u);
      return __shfl_sync(0xffffffffu, next, 0);
    };
    for (uint32_t k = 0;; ++k) {
      if (k >= 1 && !wait_idle(&sh.fetched, k + 1 & 1, 200, true)) break;
      if (k >= 2 && !wait_idle(&sh.item_empty[k & 1], (k >> 1) + 1 & 1, 200, true)) break;
      if (k) ticket = take();
      Item it = {};
      for (;; ticket = take()) {
        const uint32_t head = SPLIT ? ticket / p.splits : ticket, tile = head / p.kv_heads;  // all heads of a tile, then the next tile
        it.found = find_tile(p, per, 2 * kRows, tile, it.at, walk);
        it.kvh = head - tile * p.kv_heads;
        const uint32_t packed = it.at.fresh * per, past = it.at.len - it.at.fresh;
        it.tiles = it.at.first + kRows < packed ? 2 : 1;
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {  // b and e grow with the rows, by one at most; the second tile's stand for both where there is one
          const uint32_t r0 = it.at.first + (it.tiles == 2 ? i : 0) * kRows, lo = past + quotient(r0, p.group), hi = past + quotient(min(r0 + kRows, packed) - 1, p.group);
          it.b[i] = (p.window && lo + 1 > p.window ? lo + 1 - p.window : 0) / kKeys;
          it.e[i] = hi / kKeys + 1;
        }
        if (!SPLIT || !it.found) break;
        const uint32_t t0 = it.b[0], all = it.e[1] - t0;
        it.slice = ticket - head * p.splits;
        it.slices = max(min(p.splits, all / kSliceTiles), 1u);
        if (it.slice >= it.slices) continue;
        const uint32_t s0 = t0 + it.slice * all / it.slices, s1 = t0 + (it.slice + 1) * all / it.slices;
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) it.b[i] = max(it.b[i], s0), it.e[i] = min(it.e[i], s1);
        break;
      }
      const uint32_t packed = it.at.fresh * per;
      if (lane == 0) sh.items[k & 1] = it;
      __syncwarp();
      if (lane == 0) arrive(sa(&sh.item_full[k & 1]));
      if (!it.found) break;
      // its queries: a tensor copy where a tile of packed rows is a box of rows and heads (what follows behind the sequence's rows comes along,
      // and is not stored), else piece by piece
      bool ok = true;
      for (uint32_t i = 0; ok && i < it.tiles; ++i) {
        if (used[i] && !(ok = wait_idle(&sh.q_empty[i], used[i] + 1 & 1, 64, true))) break;
        ++used[i];
        const uint32_t dst = q_a + i * C::kTile, bar = sa(&q_full[i]), r0 = it.at.first + i * kRows;
        if (q_box) {
          if (elect_one()) {
            asm volatile("mbarrier.arrive.expect_tx.relaxed.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(C::kTile) : "memory");
#pragma unroll
            for (uint32_t x = 0; x < DP / 64; ++x) tma_load_3d(dst + x * (128 * 128), &map_q, x * 64, it.kvh * per, it.at.row0 + quotient(r0, p.group), bar);
          }
          __syncwarp();
        } else {
          constexpr uint32_t CH = DP / 8, RS = 32 / CH;  // pieces of a row; rows at a time
          const uint32_t col = lane % CH;
          const uint16_t *src = static_cast<const uint16_t *>(p.q), *mine = src + it.at.row0 * p.q_ld + it.kvh * per * p.dim + col * 8;
#pragma unroll 4
          for (uint32_t row = lane / CH; row < kRows; row += RS) {
            const uint32_t qr = r0 + row, rt = quotient(qr, p.group);
            const bool there = qr < packed && col * 8 < p.dim;
            copy16(dst + (col >> 3) * (128 * 128) + row * 128 + (((col & 7) ^ (row & 7)) << 4), there ? mine + rt * p.q_ld + (qr - rt * per) * p.dim : src, there);
          }
          copy_commit();
          copy_wait<0>();
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) arrive(bar);
        }
      }
      if (!ok) break;
    }
    if (!sh.going && lane == 0) {  // nothing may land when the CTA has gone
      for (uint32_t i = 0; i < 2; ++i)
        if (used[i]) mbar_wait_short(sa(&q_full[i]), used[i] + 1 & 1);
    }
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (tid == 0 && !sh.going) raise(p.error, kWaitCode);
  stamp_end(p.stamps);
  if (tid == 0) {
    __threadfence();
    if (atomicAdd(p.tickets + 1, 1u) + 1 == gridDim.x) p.tickets[0] = p.tickets[1] = 0;
  }
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// One row and head of a call whose positions were split, by a warp: lane s has slice s.
template <bool BF, int DP> __global__ void __launch_bounds__(256) paged_prompt_join_kernel(const PagedAttention p) {
  const uint32_t lane = threadIdx.x & 31, per = p.heads / p.kv_heads;
  const size_t to = (size_t)blockIdx.x * 8 + threadIdx.x / 32, all = (size_t)p.rows * p.heads;
  follow();
  if (to < all) {
    float2 ml = {0.f, 0.f};
    if (lane < p.splits) {
      ml = p.part_ml[lane * all + to];
      if (ml.y != 0.f) p.part_ml[lane * all + to] = make_float2(0.f, 0.f);
    }
    const uint32_t there = __ballot_sync(0xffffffffu, ml.y != 0.f);
    if (there) {  // else the row was not split, or belongs to no sequence
      const bool seen = ml.y != 0.f && ml.y != -1.f;
      const uint32_t use = __ballot_sync(0xffffffffu, seen);
      const float top = warp_max(seen ? ml.x : -INFINITY), w = seen ? exp2f(ml.x - top) : 0.f, inv = 1.0f / warp_sum(seen ? w * ml.y : 0.f);
      float v[DP / 32] = {};  // dimensions lane * DP / 32 ...
#pragma unroll 4
      for (uint32_t s = 0; s < p.splits; ++s) {
        const float ws = __shfl_sync(0xffffffffu, w, s);
        if (!(use >> s & 1)) continue;
        const float *src = p.part_o + (s * all + to) * DP + lane * (DP / 32);
#pragma unroll
        for (int d = 0; d < DP / 32; d += 2) {
          const float2 x = *reinterpret_cast<const float2 *>(src + d);
          v[d] += ws * x.x, v[d + 1] += ws * x.y;
        }
      }
      float finite = 0.f;
      uint16_t *out = static_cast<uint16_t *>(p.out) + to * p.dim + lane * (DP / 32);
#pragma unroll
      for (int d = 0; d < DP / 32; d += 2) {
        if (lane * (DP / 32) + d >= p.dim) continue;
        const float a = v[d] * inv, b = v[d + 1] * inv;
        finite += a * 0.f + b * 0.f;
        *reinterpret_cast<uint32_t *>(out + d) = pack2<BF>(a, b);
      }
      if (__any_sync(0xffffffffu, finite != 0.f)) {  // NaN
        const uint32_t row = (uint32_t)(to / p.heads), head = (uint32_t)(to - (size_t)row * p.heads), kvh = head / per;
        uint32_t lo = 0, hi = p.n;  // the last sequence that begins at or in front of the row: the one that has it, for it was computed
        while (hi - lo > 1) {
          const uint32_t mid = (lo + hi) / 2;
          if (p.starts[mid] <= row) lo = mid;
          else hi = mid;
        }
        bool bad = false;
        const Place at = {lo, p.starts[lo], fresh_rows(p, lo, bad), p.lengths[lo], 0};
        __syncwarp();
        if (row - at.row0 < at.fresh) row_again<BF>(p, at, kvh, (row - at.row0) * per + head - kvh * per, 0, DP);
      }
    }
  }
  stamp_end(p.stamps);
}

uint64_t most_items(const PagedAttention &p) {  // every sequence with rows may have a tile that is not full
  const uint64_t packed = (uint64_t)p.rows * (p.heads / p.kv_heads);
  return (packed + std::min<uint64_t>(p.n, packed) * (2 * kRows - 1)) / (2 * kRows) * p.kv_heads;
}

// Queries as [rows, heads, dim]: boxes of 64 dimensions, a group's heads and as many rows as make up a tile. False where they cannot be mapped.
template <bool BF> bool make_q_map(CUtensorMap *map, const PagedAttention &p, uint32_t per) {
  EncodeTiled enc = encode_tiled();
  const cuuint64_t dims[3] = {p.dim, p.heads, p.rows}, strides[2] = {(cuuint64_t)p.dim * 2, (cuuint64_t)p.q_ld * 2};
  const cuuint32_t boxes[3] = {64, per, kRows / per}, steps[3] = {1, 1, 1};
  return enc && enc(map, BF ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(p.q), dims, strides, boxes, steps,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
template <bool BF, int DP> cudaError_t run(const PagedAttention &p, uint32_t sms, cudaStream_t s) {
  const uint64_t per = p.heads / p.kv_heads;
  const uint64_t cache_rows = (uint64_t)p.pages * p.kv_heads * p.page.d;
  CUtensorMap map_k = {}, map_v = {}, map_q = {};
  uint32_t box = kKeys;  // the most rows, a power of two, of which pages consist; coordinates are signed
  while (p.page.d % box) box /= 2;
  if (box < 8 || cache_rows > 0x7fffffffu || !make_map(&map_k, p.kcache, (uint32_t)cache_rows, p.dim, box, BF) ||
      !make_map(&map_v, p.vcache, (uint32_t)cache_rows, p.dim, box, BF))
    box = 0;
  const bool q_box = kRows % per == 0 && make_q_map<BF>(&map_q, p, (uint32_t)per);
  const dim3 grid((uint32_t)std::min<uint64_t>(sms, most_items(p) * p.splits));
  auto kernel = p.splits > 1 ? (p.aside ? paged_prompt_tc_kernel<BF, DP, true, true> : paged_prompt_tc_kernel<BF, DP, true, false>)
                             : (p.aside ? paged_prompt_tc_kernel<BF, DP, false, true> : paged_prompt_tc_kernel<BF, DP, false, false>);
  return launch_following(kernel, grid, kThreads, Cfg<DP>::kSmem, s, p, map_k, map_v, map_q, box, q_box);
}
template <bool BF, int DP> cudaError_t setup_one() {
  for (auto kernel : {paged_prompt_tc_kernel<BF, DP, false, false>, paged_prompt_tc_kernel<BF, DP, true, false>, paged_prompt_tc_kernel<BF, DP, false, true>,
                      paged_prompt_tc_kernel<BF, DP, true, true>}) {
    cudaFuncAttributes a;
    cudaError_t e = cudaFuncGetAttributes(&a, kernel);
    if (e != cudaSuccess) return e;
    if (a.numRegs * kThreads < kLaunchRegs) return cudaErrorInvalidConfiguration;  // the softmax warps would wait for registers that nobody has
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg<DP>::kSmem);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t setup_paged_prompt_tc() {
  for (cudaError_t e : {setup_one<false, 64>(), setup_one<false, 128>(), setup_one<true, 64>(), setup_one<true, 128>()})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}
// As many slices as make the waves of items shortest, a few slices to an SM at most; more slices only where they gain a sixth. Not where there are
// items for every SM: the longest first, they fill them well enough. us, 32 heads of 128 over 8: a chunk of 128 rows behind 30,000 positions (16
// items, 9 slices) 449 -> 72, two of 300 rows behind 6,000 (80 items, 3 slices) 118 -> 104.
uint32_t paged_prompt_splits(const PagedAttention &p, uint32_t sms) {
  if (p.dim > 128) return 1;
  const uint64_t items = most_items(p), most = std::min<uint64_t>({(uint64_t)p.width * p.page.d / (kKeys * kSliceTiles), kMostSplits, 3 * sms / items});
  uint32_t best = 1;
  if (items >= sms) return best;
  auto waves = [&](uint64_t n) { return (items * n + sms - 1) / sms; };
  for (uint32_t n = 2; n <= most; ++n)
    if (6 * waves(n) * best < 5 * waves(best) * n) best = n;
  return best;
}
size_t paged_prompt_aside(uint32_t dim, uint32_t sms) { return (size_t)sms * kSoftmaxWarps * 32 * (dim <= 64 ? kAsideRow<64> : kAsideRow<128>) * 4; }
cudaError_t launch_paged_prompt_join(const PagedAttention &p, cudaStream_t s) {
  const dim3 grid((uint32_t)(((uint64_t)p.rows * p.heads + 7) / 8));
  if (p.dim <= 64) return launch_following(p.bf ? paged_prompt_join_kernel<true, 64> : paged_prompt_join_kernel<false, 64>, grid, 256, 0, s, p);
  return launch_following(p.bf ? paged_prompt_join_kernel<true, 128> : paged_prompt_join_kernel<false, 128>, grid, 256, 0, s, p);
}
cudaError_t launch_paged_prompt_tc(const PagedAttention &p, uint32_t sms, cudaStream_t s) {
  if (p.dim <= 64) return p.bf ? run<true, 64>(p, sms, s) : run<false, 64>(p, sms, s);
  return p.bf ? run<true, 128>(p, sms, s) : run<false, 128>(p, sms, s);
}

}  // namespace vkl
