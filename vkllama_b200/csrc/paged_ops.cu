// The operators of a key-value cache in pages (paged.h): argument checks, outputs, launches.
#include <math.h>

#include <cmath>
#include <new>

#include "op.h"
#include "paged.h"

using namespace vkl;

namespace {

constexpr uint64_t kMaxTokens = 0x7fffffffu;  // of a sequence, so that positions and their quotients stay in 32 bits

// The op's device is current while it launches, whatever the caller's thread has current.
struct OnDevice {
  int before = -1;
  explicit OnDevice(int ordinal) {
    if (cudaGetDevice(&before) != cudaSuccess || before == ordinal || cudaSetDevice(ordinal) != cudaSuccess) before = -1;
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

// A stream for what has to be done at once, beside the command's.
struct OwnStream {
  cudaStream_t s = nullptr;
  cudaError_t open() { return cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking); }
  ~OwnStream() {
    if (s) cudaStreamDestroy(s);
  }
};

struct PagedOp : vkl_op {
  vkl_tensor *stamps = nullptr;  // of the last launch (paged.h), in the place of the other ops' events
  std::shared_ptr<std::atomic<uint64_t>> waits;  // the command's
  uint64_t run_in = 0;                           // what they were at the last launch
  using vkl_op::vkl_op;
  ~PagedOp() override { vkl_tensor_release(stamps); }
  int paged_init() {
    if (!dev || !cmd) return fail(VKL_INVALID_ARGUMENT, "op: null device or command");
    VKL_OKAY(ensure_tensor(dev, &stamps, 1, 1, 4, VKL_UINT32));
    VKL_CUDA(cudaMemsetAsync(stamps->data(), 0, 16, cmd->stream));
    waits = cmd->waits;
    uint32_t *word;
    VKL_OKAY(command_error_word(cmd, &word));  // allocated here, so that run() does not have to
    inited = true;
    return VKL_OK;
  }
  int begin(const char *who) {
    if (!inited) return fail(VKL_FAILED_PRECONDITION, "%s: init() was not called", who);
    return recording(cmd, who);
  }
  unsigned long long *stamp() {
    timed = true;
    run_in = *waits;
    return (unsigned long long *)stamps->data();
  }
  int elapsed(uint64_t *usec) override {
    *usec = 0;
    if (!timed) return VKL_OK;
    OnDevice here(dev->ordinal);
    if (*waits == run_in) {  // not waited for since (so the command is there): over where its stream has nothing left
      cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;  // a query would end a capture
      if (cudaStreamIsCapturing(cmd->stream, &capturing) != cudaSuccess || capturing != cudaStreamCaptureStatusNone || cudaStreamQuery(cmd->stream) != cudaSuccess) {
        (void)cudaGetLastError();
        return fail(VKL_FAILED_PRECONDITION, "op_time: the op's last run has not finished (wait on its command first)");
      }
    }
    unsigned long long t[2];
    OwnStream own;  // not behind what the command's has, nor in the way of other streams
    VKL_CUDA(own.open());
    VKL_CUDA(cudaMemcpyAsync(t, stamps->data(), 16, cudaMemcpyDeviceToHost, own.s));
    VKL_CUDA(cudaStreamSynchronize(own.s));
    *usec = t[1] > t[0] ? (t[1] - t[0] + 500) / 1000 : 0;
    return VKL_OK;
  }
  int check(const vkl_tensor *t, const char *who, const char *name, int dtype, bool dense = true) {
    if (!t) return fail(VKL_INVALID_ARGUMENT, "%s: null %s", who, name);
    if (t->dev->ordinal != dev->ordinal) return fail(VKL_INVALID_ARGUMENT, "%s: %s is on device %d, the op on device %d", who, name, t->dev->ordinal, dev->ordinal);
    if (t->dtype != dtype) return fail(VKL_INVALID_ARGUMENT, "%s: %s has dtype %d, expected %d", who, name, t->dtype, dtype);
    if (dense && !t->dense()) return fail(VKL_UNIMPLEMENTED, "%s: %s must be dense", who, name);
    return VKL_OK;
  }
  int check_list(const vkl_tensor *t, const char *who, const char *name, size_t n) {
    VKL_OKAY(check(t, who, name, VKL_UINT32));
    if (t->c != 1 || t->h != 1 || t->w != n)
      return fail(VKL_INVALID_ARGUMENT, "%s: %s has shape (%zu, %zu, %zu), expected (1, 1, %zu)", who, name, t->c, t->h, t->w, n);
    return VKL_OK;
  }
  // Rows of `w` values, possibly apart (a view of wider rows).
  int check_rows(const vkl_tensor *t, const char *who, const char *name, int dtype) {
    VKL_OKAY(check(t, who, name, dtype, false));
    if (t->c != 1) return fail(VKL_INVALID_ARGUMENT, "%s: %s has %zu channels, expected 1", who, name, t->c);
    if (t->h > kMaxTokens) return fail(VKL_OUT_OF_RANGE, "%s: %zu rows", who, t->h);
    return VKL_OK;
  }
  int check_apart(const vkl_tensor *t, const char *who, const char *name) {
    if (t->h > 1 && t->hs % 16) return fail(VKL_UNIMPLEMENTED, "%s: rows of %s are %zu bytes apart, which is no multiple of 16", who, name, t->hs);
    return VKL_OK;
  }
  int check_cache(const vkl_tensor *k, const vkl_tensor *v, const char *who, int dtype, size_t kv_heads, size_t page, size_t dim) {
    VKL_OKAY(check(k, who, "key cache", dtype));
    VKL_OKAY(check(v, who, "value cache", dtype));
    if (k->c != v->c || k->h != v->h || k->w != v->w || k->h != kv_heads * page || k->w != dim)
      return fail(VKL_INVALID_ARGUMENT, "%s: caches have shapes (%zu, %zu, %zu) and (%zu, %zu, %zu), expected (pages, %zu, %zu)", who, k->c, k->h, k->w, v->c, v->h,
                  v->w, kv_heads * page, dim);
    if (k->c * k->h >= 0xffffffffu) return fail(VKL_OUT_OF_RANGE, "%s: a cache of %zu rows; at most 2^32 - 2 can be named", who, k->c * k->h);
    return VKL_OK;
  }
  int check_table(const vkl_tensor *t, const char *who, size_t page) {
    VKL_OKAY(check(t, who, "table", VKL_UINT32));
    if (t->c != 1) return fail(VKL_INVALID_ARGUMENT, "%s: the table has %zu channels, expected 1", who, t->c);
    if (t->w * page > kMaxTokens) return fail(VKL_OUT_OF_RANGE, "%s: a table of %zu pages of %zu tokens; a sequence has at most 2^31 - 1", who, t->w, page);
    return VKL_OK;
  }
};

bool good_page(int page) { return page >= 1 && page <= 1 << 20; }
bool good_dim(int dim) { return dim >= 8 && dim <= 256 && dim % 8 == 0; }
bool good_dtype(int dtype) { return dtype == VKL_FP16 || dtype == VKL_BF16; }

// -------------------------------------------------------------- PagedTables
struct PagedTablesOp : PagedOp {
  int page;
  vkl_tensor *map = nullptr, *starts = nullptr, *arrived = nullptr;
  PagedTablesOp(vkl_device *d, vkl_command *c, int pg) : PagedOp(d, c), page(pg) {}
  ~PagedTablesOp() override {
    for (vkl_tensor *t : {map, starts, arrived}) vkl_tensor_release(t);
  }
  int init() override {
    if (inited) return VKL_OK;
    OnDevice here(dev->ordinal);
    if (!good_page(page)) return fail(VKL_INVALID_ARGUMENT, "PagedTables op: a page of %d tokens", page);
    VKL_CUDA(setup_paged_tables());
    VKL_OKAY(ensure_tensor(dev, &arrived, 1, 1, 1, VKL_UINT32));
    VKL_CUDA(cudaMemsetAsync(arrived->data(), 0, 4, cmd->stream));
    return paged_init();
  }
  int run(vkl_tensor *lengths, vkl_tensor *target, vkl_tensor *table, vkl_tensor *pool, size_t rows, vkl_tensor **o_map, vkl_tensor **o_starts) {
    const char *who = "paged_tables";
    OnDevice here(dev->ordinal);
    VKL_OKAY(check_table(table, who, page));
    const size_t n = table->h;
    VKL_OKAY(check_list(lengths, who, "lengths", n));
    VKL_OKAY(check_list(target, who, "target", n));
    VKL_OKAY(check(pool, who, "pool", VKL_UINT32));
    if (pool->c != 1 || pool->h != 1 || pool->w < 1) return fail(VKL_INVALID_ARGUMENT, "%s: the pool has shape (%zu, %zu, %zu), expected (1, 1, 1 + pages)", who, pool->c, pool->h, pool->w);
    if (n > kTablesMaxSequences) return fail(VKL_OUT_OF_RANGE, "%s: %zu sequences, at most %u", who, n, kTablesMaxSequences);
    if (rows > kMaxTokens || pool->w > kMaxTokens) return fail(VKL_OUT_OF_RANGE, "%s: %zu rows, a pool of %zu pages", who, rows, pool->w - 1);
    VKL_OKAY(begin(who));
    VKL_OKAY(ensure_tensor(dev, &map, 1, 2, rows, VKL_UINT32));
    VKL_OKAY(ensure_tensor(dev, &starts, 1, 1, n + 1, VKL_UINT32));
    PagedTables p = {};
    p.lengths = (uint32_t *)lengths->data();
    p.target = (const uint32_t *)target->data();
    p.table = (uint32_t *)table->data();
    p.pool = (uint32_t *)pool->data();
    p.map = (uint32_t *)map->data();
    p.starts = (uint32_t *)starts->data();
    p.arrived = (uint32_t *)arrived->data();
    VKL_OKAY(command_error_word(cmd, &p.error));
    p.stamps = stamp();
    p.n = (uint32_t)n, p.width = (uint32_t)table->w, p.capacity = (uint32_t)pool->w - 1, p.rows = (uint32_t)rows;
    p.page = divisor(page);
    VKL_LAUNCH(1, launch_paged_tables(p, dev->prop.multiProcessorCount, cmd->stream));
    if (o_map) *o_map = map;
    if (o_starts) *o_starts = starts;
    return VKL_OK;
  }
};

// ------------------------------------------------------- UpdatePagedKVCache
struct UpdatePagedOp : PagedOp {
  int dim, page, dtype;
  float theta;
  vkl_tensor *turns = nullptr, *out = nullptr;
  UpdatePagedOp(vkl_device *d, vkl_command *c, int dm, int pg, float th, int dt) : PagedOp(d, c), dim(dm), page(pg), dtype(dt), theta(th) {}
  ~UpdatePagedOp() override {
    vkl_tensor_release(turns);
    vkl_tensor_release(out);
  }
  int init() override {
    if (inited) return VKL_OK;
    OnDevice here(dev->ordinal);
    if (!good_dtype(dtype)) return fail(VKL_INVALID_ARGUMENT, "UpdatePagedKVCache op: only fp16 and bf16 dtypes are supported.");
    if (!good_page(page)) return fail(VKL_INVALID_ARGUMENT, "UpdatePagedKVCache op: a page of %d tokens", page);
    if (!good_dim(dim)) return fail(VKL_INVALID_ARGUMENT, "UpdatePagedKVCache op: head dim %d is no multiple of 8 up to 256", dim);
    if (theta != 0.f && !(theta >= 1.f && theta <= 1e30f)) return fail(VKL_INVALID_ARGUMENT, "UpdatePagedKVCache op: theta is %g", theta);
    if (theta != 0.f) {
      double per[128];
      for (int k = 0; k < dim / 2; ++k) per[k] = std::pow((double)theta, -2.0 * k / dim) / (2.0 * std::acos(-1.0));
      VKL_OKAY(ensure_tensor(dev, &turns, 1, 1, dim, VKL_FP32));
      VKL_CUDA(cudaMemcpyAsync(turns->data(), per, dim / 2 * 8, cudaMemcpyHostToDevice, cmd->stream));
      VKL_CUDA(cudaStreamSynchronize(cmd->stream));
    }
    return paged_init();
  }
  int run(vkl_tensor *kcache, vkl_tensor *vcache, vkl_tensor *k, vkl_tensor *v, vkl_tensor *map, vkl_tensor *q, vkl_tensor **o) {
    const char *who = "update_paged_kvcache";
    OnDevice here(dev->ordinal);
    VKL_OKAY(check_rows(k, who, "keys", dtype));
    VKL_OKAY(check_rows(v, who, "values", dtype));
    if (k->h != v->h || k->w != v->w || k->w == 0 || k->w % dim)
      return fail(VKL_INVALID_ARGUMENT, "%s: keys have shape (%zu, %zu, %zu), values (%zu, %zu, %zu), heads are %d wide", who, k->c, k->h, k->w, v->c, v->h, v->w, dim);
    const size_t rows = k->h, kv_heads = k->w / dim;
    if (q) {
      VKL_OKAY(check_rows(q, who, "queries", dtype));
      if (q->h != rows || q->w == 0 || q->w % dim)
        return fail(VKL_INVALID_ARGUMENT, "%s: queries have shape (%zu, %zu, %zu) beside %zu keys, heads are %d wide", who, q->c, q->h, q->w, rows, dim);
    }
    VKL_OKAY(check_cache(kcache, vcache, who, dtype, kv_heads, page, dim));
    VKL_OKAY(check(map, who, "map", VKL_UINT32));
    if (map->c != 1 || map->h != 2 || map->w != rows)
      return fail(VKL_INVALID_ARGUMENT, "%s: the map has shape (%zu, %zu, %zu), expected (1, 2, %zu)", who, map->c, map->h, map->w, rows);
    VKL_OKAY(check_apart(k, who, "keys"));
    VKL_OKAY(check_apart(v, who, "values"));
    if (q) VKL_OKAY(check_apart(q, who, "queries"));
    if (kcache->data() == vcache->data()) return fail(VKL_INVALID_ARGUMENT, "%s: keys and values have one cache", who);
    if ((q ? q->w : 0) + 2 * k->w > 1u << 24) return fail(VKL_OUT_OF_RANGE, "%s: rows of %zu values", who, (q ? q->w : 0) + 2 * k->w);
    VKL_OKAY(begin(who));
    // queries may be turned in their place; keys and values would be read while other threads store there
    if (q && out && (k->data() == out->data() || v->data() == out->data())) return fail(VKL_INVALID_ARGUMENT, "%s: keys or values are this op's own output", who);
    if (q) VKL_OKAY(ensure_tensor(dev, &out, 1, rows, q->w, dtype));
    if (rows) {
      PagedUpdate p = {};
      p.k = k->data(), p.v = v->data();
      p.k_ld = k->hs / 2, p.v_ld = v->hs / 2;
      if (q) {
        p.q = q->data(), p.q_out = out->data();
        p.q_ld = q->hs / 2;
        p.heads = (uint32_t)(q->w / dim);
      }
      p.kcache = kcache->data(), p.vcache = vcache->data();
      p.map = (const uint32_t *)map->data();
      VKL_OKAY(command_error_word(cmd, &p.error));
      p.stamps = stamp();
      p.rows = (uint32_t)rows, p.kv_heads = (uint32_t)kv_heads, p.dim = (uint32_t)dim, p.pages = (uint32_t)kcache->c;
      p.page = divisor(page);
      p.turns = turns ? (const double *)turns->data() : nullptr;
      p.bf = dtype == VKL_BF16;
      VKL_LAUNCH(1, launch_paged_update(p, cmd->stream));
    }
    if (o) *o = q ? out : nullptr;
    return VKL_OK;
  }
};

// ------------------------------------------------------------ PagedAttention
struct PagedAttentionOp : PagedOp {
  int heads, kv_heads, dim, page, window, dtype;
  float scale;
  vkl_tensor *out = nullptr, *scratch = nullptr, *counters = nullptr, *part_o = nullptr, *part_ml = nullptr, *aside = nullptr;
  vkl_tensor *older[64];  // smaller part_o and part_ml, which captured calls go on using
  int n_older = 0;
  PagedAttentionOp(vkl_device *d, vkl_command *c, int h, int kv, int dm, int pg, float s, int w, int dt)
      : PagedOp(d, c), heads(h), kv_heads(kv), dim(dm), page(pg), window(w), dtype(dt), scale(s) {}
  ~PagedAttentionOp() override {
    for (vkl_tensor *t : {out, scratch, counters, part_o, part_ml, aside}) vkl_tensor_release(t);
    while (n_older) vkl_tensor_release(older[--n_older]);
  }
  int init() override {
    if (inited) return VKL_OK;
    OnDevice here(dev->ordinal);
    if (!good_dtype(dtype)) return fail(VKL_INVALID_ARGUMENT, "PagedAttention op: only fp16 and bf16 dtypes are supported.");
    if (heads < 1 || kv_heads < 1 || heads % kv_heads || heads > 65535)
      return fail(VKL_INVALID_ARGUMENT, "PagedAttention op: %d heads over %d key heads", heads, kv_heads);
    if (!good_dim(dim)) return fail(VKL_INVALID_ARGUMENT, "PagedAttention op: head dim %d is no multiple of 8 up to 256", dim);
    if (!good_page(page)) return fail(VKL_INVALID_ARGUMENT, "PagedAttention op: a page of %d tokens", page);
    if (window < 0) return fail(VKL_INVALID_ARGUMENT, "PagedAttention op: a window of %d positions", window);
    if (scale != 0.f && !(fabsf(scale) >= 1e-20f && fabsf(scale) <= 1e20f)) return fail(VKL_INVALID_ARGUMENT, "PagedAttention op: scale is %g", scale);
    const uint32_t sms = dev->prop.multiProcessorCount;
    VKL_CUDA(setup_paged_token());
    VKL_CUDA(setup_paged_prompt());
    VKL_CUDA(setup_paged_prompt_tc());
    VKL_OKAY(ensure_tensor(dev, &scratch, 1, 1, paged_token_scratch(heads, kv_heads, dim, sms) / 4, VKL_FP32));
    VKL_OKAY(ensure_tensor(dev, &counters, 1, 1, 2 * (sms + 1) + 2, VKL_UINT32));
    VKL_CUDA(cudaMemsetAsync(counters->data(), 0, counters->device_bytes(), cmd->stream));
    return paged_init();
  }
  // Room for n numbers, all 0 if it is new: at once, for a call that is being captured would only put that into its graph. It grows by powers of two.
  int room(vkl_tensor **t, size_t n) {
    if (*t && (*t)->w >= n) return VKL_OK;
    size_t more = 1 << 16;
    while (more < n) more *= 2;
    if (*t) {
      if (n_older == 64) return fail(VKL_RESOURCE_EXHAUSTED, "paged_attention: too many workspaces");
      older[n_older++] = *t;
      *t = nullptr;
    }
    VKL_OKAY(ensure_tensor(dev, t, 1, 1, more, VKL_FP32));
    OwnStream own;
    VKL_CUDA(own.open());
    VKL_CUDA(cudaMemsetAsync((*t)->data(), 0, more * 4, own.s));
    VKL_CUDA(cudaStreamSynchronize(own.s));
    return VKL_OK;
  }
  int run(vkl_tensor *q, vkl_tensor *kcache, vkl_tensor *vcache, vkl_tensor *table, vkl_tensor *lengths, vkl_tensor *starts, vkl_tensor **o) {
    const char *who = "paged_attention";
    OnDevice here(dev->ordinal);
    VKL_OKAY(check_rows(q, who, "queries", dtype));
    if (q->w != (size_t)heads * dim) return fail(VKL_INVALID_ARGUMENT, "%s: queries are %zu wide, expected %d heads of %d", who, q->w, heads, dim);
    VKL_OKAY(check_cache(kcache, vcache, who, dtype, kv_heads, page, dim));
    VKL_OKAY(check_table(table, who, page));
    const size_t n = table->h, rows = q->h, per = heads / kv_heads;
    const uint32_t sms = dev->prop.multiProcessorCount;
    VKL_OKAY(check_list(lengths, who, "lengths", n));
    if (starts) VKL_OKAY(check_list(starts, who, "starts", n + 1));
    if (!starts && rows != n) return fail(VKL_INVALID_ARGUMENT, "%s: %zu queries for %zu sequences of one new token each", who, rows, n);
    VKL_OKAY(check_apart(q, who, "queries"));
    if (rows * per > kMaxTokens || n > kMaxTokens || (rows * per / 64 + n) * kv_heads > kMaxTokens)
      return fail(VKL_OUT_OF_RANGE, "%s: %zu rows, %zu sequences of up to %zu tokens", who, rows, n, table->w * page);
    VKL_OKAY(begin(who));
    if (out && q->data() == out->data()) return fail(VKL_INVALID_ARGUMENT, "%s: the queries are this op's own output", who);
    VKL_OKAY(ensure_tensor(dev, &out, 1, rows, q->w, dtype));
    if (rows && n) {
      PagedAttention p = {};
      p.q = q->data(), p.q_ld = q->hs / 2;
      p.kcache = kcache->data(), p.vcache = vcache->data();
      p.out = out->data();
      p.table = (const uint32_t *)table->data();
      p.lengths = (const uint32_t *)lengths->data();
      p.starts = starts ? (const uint32_t *)starts->data() : nullptr;
      p.scratch = (float *)scratch->data();
      p.counters = (uint32_t *)counters->data();
      p.tickets = p.counters + 2 * (sms + 1);
      VKL_OKAY(command_error_word(cmd, &p.error));
      p.stamps = stamp();
      p.rows = (uint32_t)rows, p.n = (uint32_t)n, p.heads = heads, p.kv_heads = kv_heads, p.dim = dim;
      p.width = (uint32_t)table->w, p.pages = (uint32_t)kcache->c, p.window = window;
      p.page = divisor(page);
      p.group = divisor((uint32_t)per);
      p.scale = scale != 0.f ? scale : 1.0f / sqrtf((float)dim);
      p.bf = dtype == VKL_BF16;
      // the one-token form counts tiles of 16 or 32 positions of all sequences and head groups in 31 bits
      p.count = !starts && table->w * page / 16 + 2 > kMaxTokens / (n * kv_heads * ((per + 7) / 8));
      p.splits = starts ? paged_prompt_splits(p, sms) : 1;
      if (p.splits > 1) {
        const size_t parts = p.splits * rows * heads;
        VKL_OKAY(room(&part_o, parts * (dim <= 64 ? 64 : 128)));
        VKL_OKAY(room(&part_ml, parts * 2));
        p.part_o = (float *)part_o->data(), p.part_ml = (float2 *)part_ml->data();
      }
      if (starts && dim <= 128 && table->w * page > kManyPositions) {
        VKL_OKAY(ensure_tensor(dev, &aside, 1, 1, paged_prompt_aside(dim, sms) / 4, VKL_FP32));
        p.aside = (float *)aside->data();
      }
      VKL_LAUNCH(starts ? paged_prompt_launches(p) : 1, starts ? launch_paged_prompt(p, sms, cmd->stream) : launch_paged_token(p, sms, cmd->stream));
    }
    *o = out;
    return VKL_OK;
  }
};

template <class T, class... A> int make(vkl_op **out, vkl_device *dev, vkl_command *cmd, A... a) {
  if (!out) return fail(VKL_INVALID_ARGUMENT, "op create: null output");
  if (!dev || !cmd) return fail(VKL_INVALID_ARGUMENT, "op create: null device or command");
  if (cmd->dev->ordinal != dev->ordinal) return fail(VKL_INVALID_ARGUMENT, "op create: the command is on device %d, not %d", cmd->dev->ordinal, dev->ordinal);
  *out = new (std::nothrow) T(dev, cmd, a...);
  return *out ? VKL_OK : fail(VKL_RESOURCE_EXHAUSTED, "op create: out of host memory");
}

}  // namespace

extern "C" {

int vkl_paged_tables_create(vkl_device *dev, vkl_command *cmd, int page_size, vkl_op **out) { return make<PagedTablesOp>(out, dev, cmd, page_size); }
int vkl_paged_tables_run(vkl_op *op, vkl_tensor *lengths, vkl_tensor *target, vkl_tensor *table, vkl_tensor *pool, size_t rows, vkl_tensor **map, vkl_tensor **starts) {
  PagedTablesOp *m;
  VKL_OKAY(as(op, &m, "paged_tables_run"));
  if (!map || !starts) return fail(VKL_INVALID_ARGUMENT, "paged_tables_run: null output");
  return m->run(lengths, target, table, pool, rows, map, starts);
}
int vkl_update_paged_kvcache_create(vkl_device *dev, vkl_command *cmd, int dim, int page_size, float theta, int dtype, vkl_op **out) {
  return make<UpdatePagedOp>(out, dev, cmd, dim, page_size, theta, dtype);
}
int vkl_update_paged_kvcache_run(vkl_op *op, vkl_tensor *kcache, vkl_tensor *vcache, vkl_tensor *k, vkl_tensor *v, vkl_tensor *map, vkl_tensor *q, vkl_tensor **out) {
  UpdatePagedOp *m;
  VKL_OKAY(as(op, &m, "update_paged_kvcache_run"));
  if (q && !out) return fail(VKL_INVALID_ARGUMENT, "update_paged_kvcache_run: null output");
  return m->run(kcache, vcache, k, v, map, q, out);
}
int vkl_paged_attention_create(vkl_device *dev, vkl_command *cmd, int heads, int kv_heads, int dim, int page_size, float scale, int window, int dtype, vkl_op **out) {
  return make<PagedAttentionOp>(out, dev, cmd, heads, kv_heads, dim, page_size, scale, window, dtype);
}
int vkl_paged_attention_run(vkl_op *op, vkl_tensor *q, vkl_tensor *kcache, vkl_tensor *vcache, vkl_tensor *table, vkl_tensor *lengths, vkl_tensor *starts, vkl_tensor **out) {
  PagedAttentionOp *m;
  VKL_OKAY(as(op, &m, "paged_attention_run"));
  if (!out) return fail(VKL_INVALID_ARGUMENT, "paged_attention_run: null output");
  return m->run(q, kcache, vcache, table, lengths, starts, out);
}

}  // extern "C"
