// A key-value cache in pages that many sequences share: what its operators' launchers take.
//
// cache   [pages][kv_heads][page][dim], keys and values apart, fp16 or bf16
// table   [sequences][width]: a sequence's pages in order; position j is row j % page of page table[j / page]
// slot    page * page_size + row of a token, or kNoSlot
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace vkl {

constexpr uint32_t kNoSlot = 0xffffffffu;

// What a kernel found on the device that the host could not see, in the command's error word (wait() reports it). Waits inside
// kernels that ran out have codes below 0x100.
enum PagedError : uint32_t {
  PAGED_POOL_EMPTY = 0x101,  // tables: more pages are needed than the pool holds
  PAGED_TABLE_FULL,          // a sequence is longer than a row of its table
  PAGED_ROWS,                // tables: more new rows than the call has room for
  PAGED_POOL_BAD,            // tables: the pool's count and what comes back do not fit it
  PAGED_BAD_PAGE,            // a page that the cache does not have
  PAGED_BAD_ROWS,            // attention: starts and lengths do not belong together
  PAGED_TOO_MUCH,            // attention of one token: tiles of positions beyond 31 bits
};

// n / d for n < 2^31 by a multiplication.
struct Divisor {
  uint32_t d, mul, shift;
};
inline Divisor divisor(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {d, (uint32_t)((((1ull << s) - d) << 32) / d + 1), s};
}
#ifdef __CUDACC__
__device__ __forceinline__ uint32_t quotient(uint32_t n, const Divisor &v) { return (__umulhi(n, v.mul) + n) >> v.shift; }
__device__ __forceinline__ void raise(uint32_t *error, uint32_t code) { atomicCAS(error, 0u, code); }
// Launches may begin before the one in front of them in the stream has ended (launch_following): nothing is read or written before
// follow() returns, when everything in front has ended and is visible, and the launch behind may be prepared from then on. What the launch in
// front may have written is not read-only for the whole of this one, so these kernels have no ld.global.nc (__ldg).
__device__ __forceinline__ void follow() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
}
template <class K, class... P> cudaError_t launch_following(K kernel, dim3 grid, uint32_t threads, size_t smem, cudaStream_t s, const P &...p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p...);
}

// When a launch began and when its last CTA ended, for Op::time(): two events around every launch would cost 5 us of device time.
// The timer only grows, so the later end is the last launch's.
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void stamp_begin(unsigned long long *stamps) {
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) stamps[0] = now_ns();
}
__device__ __forceinline__ void stamp_end(unsigned long long *stamps) {
  if (threadIdx.x == 0) atomicMax(stamps + 1, now_ns());
}
__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
#endif

struct PagedTables {
  uint32_t *lengths;       // [n], becomes target
  const uint32_t *target;  // [n]
  uint32_t *table;         // [n][width]
  uint32_t *pool;          // [0] count, then the free pages, the next one to be taken last
  uint32_t *map;           // [2][rows]: slots, positions of the new rows
  uint32_t *starts;        // [n + 1] first new row of every sequence
  uint32_t *arrived;       // CTAs that are through; 0 between launches
  unsigned long long *stamps;
  uint32_t *error;
  uint32_t n, width, capacity, rows;
  Divisor page;
};
constexpr uint32_t kTablesMaxSequences = 8192;
cudaError_t launch_paged_tables(const PagedTables &p, uint32_t sms, cudaStream_t s);
cudaError_t setup_paged_tables();  // once per device

struct PagedUpdate {
  const void *q, *k, *v;        // [rows] of heads * dim, kv_heads * dim values, apart by q_ld, ... values; q may be null
  void *q_out;                  // [rows][heads * dim]
  void *kcache, *vcache;
  const uint32_t *map;          // [2][rows]
  unsigned long long *stamps;
  uint32_t *error;
  uint64_t q_ld, k_ld, v_ld;
  uint32_t rows, heads, kv_heads, dim, pages;
  Divisor page;
  const double *turns;          // [dim / 2] turns of a pair per position, or null: no rotation
  bool bf;
};
cudaError_t launch_paged_update(const PagedUpdate &p, cudaStream_t s);

// The matrix units cut their fp32 sums off instead of rounding them: what they add up themselves comes out low, by 0.014 % over this many positions of equal
// weight and values of one sign, by 0.65 % over a million. Where a prompt's rows see more, sums of fewer are added up by ordinary additions.
constexpr uint32_t kManyPositions = 32768;

struct PagedAttention {
  const void *q;                // [rows] of heads * dim values, q_ld apart
  const void *kcache, *vcache;
  void *out;                    // [rows][heads * dim]
  const uint32_t *table, *lengths;
  const uint32_t *starts;       // [n + 1], or null: row i is the last token of sequence i
  float *scratch;               // partial results, paged_token_scratch() bytes
  uint32_t *counters;           // [2 (SMs + 1)], 0 between launches
  uint32_t *tickets;            // [2], 0 between launches
  float *part_o;                // prompts whose positions are split: [splits][rows][heads][64 or 128] sums of parts
  float2 *part_ml;              // and [splits][rows][heads] references and sums of probabilities, 0 between calls
  unsigned long long *stamps;
  uint32_t *error;
  uint64_t q_ld;
  uint32_t rows, n, heads, kv_heads, dim, width, pages, window;
  Divisor page, group;          // query heads of a key head
  float scale;                  // on the scores
  bool bf, count;               // count (one token): the tables could hold more tiles than 31 bits count, so the lengths have to be added up first
  uint32_t splits;              // parts of a sequence's positions at most
  uint32_t part;                // of a prompt call's sequences, those that the launch takes: 0 all, 1 or 2 by paged_rows.cuh's rule
  float *aside;                 // prompts, tables beyond kManyPositions: sums so far, paged_prompt_aside() bytes; else null
};
// One new token per sequence.
cudaError_t launch_paged_token(const PagedAttention &p, uint32_t sms, cudaStream_t s);
size_t paged_token_scratch(uint32_t heads, uint32_t kv_heads, uint32_t dim, uint32_t sms);
cudaError_t setup_paged_token();   // once per device
// Any number of rows per sequence; in one launch or two.
uint32_t paged_prompt_launches(const PagedAttention &p);
cudaError_t launch_paged_prompt(const PagedAttention &p, uint32_t sms, cudaStream_t s);
cudaError_t setup_paged_prompt();
// The same on tcgen05, heads up to 128 wide.
uint32_t paged_prompt_splits(const PagedAttention &p, uint32_t sms);
size_t paged_prompt_aside(uint32_t dim, uint32_t sms);
cudaError_t launch_paged_prompt_tc(const PagedAttention &p, uint32_t sms, cudaStream_t s);
cudaError_t launch_paged_prompt_join(const PagedAttention &p, cudaStream_t s);  // where splits > 1, behind it
cudaError_t setup_paged_prompt_tc();

}  // namespace vkl
