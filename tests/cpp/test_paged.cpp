// The paged cache through the header-only class layer (include/vkllama/vkllama.h): prompts of three sequences, then a token each, every
// output against the definition in 64 bits.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#include "vkllama/vkllama.h"

using namespace vkllama;

#define CHECK_OK(expr)                                                  \
  do {                                                                  \
    auto s__ = (expr);                                                  \
    if (!s__.ok()) {                                                    \
      fprintf(stderr, "%s failed: %s\n", #expr, s__.ToString().c_str()); \
      return 1;                                                         \
    }                                                                   \
  } while (0)

static float value(uint16_t u) {
  _Float16 h;
  memcpy(&h, &u, 2);
  return (float)h;
}
static uint16_t bits(double x) {
  const _Float16 h = (_Float16)x;
  uint16_t u;
  memcpy(&u, &h, 2);
  return u;
}
static uint32_t state = 1;
static double draw() {  // -1 .. 1
  state = state * 1664525u + 1013904223u;
  return (state >> 8) / 8388608.0 - 1.0;
}

constexpr int kHeads = 4, kKvHeads = 2, kDim = 64, kPage = 16, kPages = 12, kSequences = 3, kWidth = 4;

int main() {
  GPUDevice gpu(0);
  CHECK_OK(gpu.init());
  Command cmd(&gpu);
  CHECK_OK(cmd.init());

  PagedTables tables(&gpu, &cmd, kPage);
  UpdatePagedKVCache update(&gpu, &cmd, kDim, kPage, 0.0f);  // not rotated, so that the definition stays short
  PagedAttention attention(&gpu, &cmd, kHeads, kKvHeads, kDim, kPage);
  for (Op *op : {(Op *)&tables, (Op *)&update, (Op *)&attention}) CHECK_OK(op->init());

  Tensor kcache(kPages, kKvHeads * kPage, kDim, &gpu, FP16), vcache(kPages, kKvHeads * kPage, kDim, &gpu, FP16);
  Tensor table(1, kSequences, kWidth, &gpu, UINT32), lengths(1, 1, kSequences, &gpu, UINT32), target(1, 1, kSequences, &gpu, UINT32);
  Tensor pool(1, 1, 1 + kPages, &gpu, UINT32);
  std::vector<uint32_t> free_pages = {kPages};
  for (uint32_t i = 0; i < kPages; ++i) free_pages.push_back(i);

  std::vector<std::vector<double>> keys(kSequences), values(kSequences);  // [position][key head][dim]
  const uint32_t prompts[kSequences] = {5, 40, 17};
  uint32_t have[kSequences] = {};
  double worst = 0;
  for (int pass = 0; pass < 3; ++pass) {
    uint32_t rows = 0, want[kSequences];
    for (int i = 0; i < kSequences; ++i) {
      want[i] = have[i] + (pass == 0 ? prompts[i] : 1);
      rows += want[i] - have[i];
    }
    std::vector<uint16_t> q((size_t)rows * kHeads * kDim), k((size_t)rows * kKvHeads * kDim), v(k.size()), got(q.size());
    for (auto *x : {&q, &k, &v})
      for (uint16_t &e : *x) e = bits(draw());
    for (int i = 0, r = 0; i < kSequences; ++i)
      for (uint32_t p = have[i]; p < want[i]; ++p, ++r)
        for (int e = 0; e < kKvHeads * kDim; ++e) {
          keys[i].push_back(value(k[(size_t)r * kKvHeads * kDim + e]));
          values[i].push_back(value(v[(size_t)r * kKvHeads * kDim + e]));
        }

    Tensor tq(1, rows, kHeads * kDim, &gpu, FP16), tk(1, rows, kKvHeads * kDim, &gpu, FP16), tv(1, rows, kKvHeads * kDim, &gpu, FP16);
    CHECK_OK(cmd.begin());
    if (pass == 0) {
      CHECK_OK(cmd.upload(free_pages.data(), free_pages.size(), pool));
      CHECK_OK(cmd.upload(have, kSequences, lengths));
    }
    CHECK_OK(cmd.upload(want, kSequences, target));
    CHECK_OK(cmd.upload(q.data(), q.size(), tq));
    CHECK_OK(cmd.upload(k.data(), k.size(), tk));
    CHECK_OK(cmd.upload(v.data(), v.size(), tv));
    auto at = tables(lengths, target, table, pool, rows);
    CHECK_OK(at.status());
    CHECK_OK(update(kcache, vcache, tk, tv, at->map));
    auto out = pass == 0 ? attention(tq, kcache, vcache, table, lengths, at->starts) : attention(tq, kcache, vcache, table, lengths);
    CHECK_OK(out.status());
    CHECK_OK(cmd.download(*out, got.data(), got.size()));
    CHECK_OK(cmd.end());
    CHECK_OK(cmd.submit_and_wait());

    for (int i = 0, r = 0; i < kSequences; ++i)
      for (uint32_t p = have[i]; p < want[i]; ++p, ++r)
        for (int h = 0; h < kHeads; ++h) {
          const int g = h / (kHeads / kKvHeads);
          double sum = 0, o[kDim] = {};
          for (uint32_t j = 0; j <= p; ++j) {
            const double *kj = &keys[i][((size_t)j * kKvHeads + g) * kDim], *vj = &values[i][((size_t)j * kKvHeads + g) * kDim];
            double s = 0;
            for (int d = 0; d < kDim; ++d) s += value(q[((size_t)r * kHeads + h) * kDim + d]) * kj[d];
            const double w = std::exp(s / std::sqrt((double)kDim));
            sum += w;
            for (int d = 0; d < kDim; ++d) o[d] += w * vj[d];
          }
          for (int d = 0; d < kDim; ++d) worst = std::max(worst, std::fabs(value(got[((size_t)r * kHeads + h) * kDim + d]) - o[d] / sum));
        }
    for (int i = 0; i < kSequences; ++i) have[i] = want[i];
  }
  // |out| < 1: the output's rounding 2^-12, the probabilities' 2^-11 of it, and fp32 sums far below
  printf("largest error %g\n", worst);
  if (worst > 3.0 / 4096) return 1;
  printf("PASS\n");
  return 0;
}
