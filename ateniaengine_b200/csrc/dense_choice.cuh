// Which kernel a dense product takes, from its sizes alone (host arithmetic).
#pragma once
#include <stdint.h>
#ifdef DENSE_TUNE
#include <cstdio>
#include <cstdlib>
#endif

namespace atenia {

struct DenseSize {
  int64_t M, N;  // N: columns of the result
  int kb;        // k-blocks of 64
};
struct DensePlan {
  bool pairs;    // dense_pair.cu; else tiles of 128 x `columns` (dense_gemm.cu), the reduction cut `split` ways
  int columns;
  int split;
};

inline DensePlan dense_plan(const DenseSize* sizes, int problems, bool two_columns, bool full_rows, int num_sms) {
#ifdef DENSE_TUNE
  if (const char* e = getenv("DENSE_PLAN")) {
    int a = 0, c = 128, b = 1;
    const char* q = e;
    if (getenv("DENSE_PLAN2") && sizes[0].kb >= atoi(getenv("DENSE_KB"))) q = getenv("DENSE_PLAN2");
    sscanf(q, "%d,%d,%d", &a, &c, &b);
    for (int i = 0; i < problems; ++i)
      while (sizes[i].kb < b) b /= 2;
    return {a && full_rows, c, b};
  }
#endif
  const int n_out = two_columns ? 128 : 256;
  int64_t pairs = 0, tiles = 0;
  int min_kb = 1 << 30;
  for (int i = 0; i < problems; ++i) {
    pairs += (sizes[i].M + 255) / 256 * ((sizes[i].N + n_out - 1) / n_out);
    tiles += (sizes[i].M + 127) / 128 * ((sizes[i].N + n_out / 2 - 1) / (n_out / 2));
    if (sizes[i].kb < min_kb) min_kb = sizes[i].kb;
  }
  if (full_rows && pairs >= num_sms / 2) return {true, 0, 1};
  // clusters until every SM has a CTA, each with four k-blocks at least
  int split = 1;
  while (split < 8 && tiles * split < num_sms && min_kb >= 8 * split) split *= 2;
  return {false, 128, split};
}

}  // namespace atenia
