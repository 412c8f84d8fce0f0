// Test-only: the choice of dense kernels and the launches' limit, compiled with a host compiler.  Not part of the product library.
#include "../ateniaengine_b200/csrc/dense_choice.cuh"

// sizes: M, N, kb of each problem; result: work items of the launch (tiles, times the CTAs or pairs that share one)
extern "C" long long limits_work_items(const long long* sizes, int problems, int rows, int two_columns, int grad, int adapters) {
  atenia::DenseSize s[3];
  for (int i = 0; i < problems; ++i) s[i] = {sizes[3 * i], sizes[3 * i + 1], (int)sizes[3 * i + 2]};
  const atenia::DensePlan p = atenia::dense_plan(s, problems, rows, two_columns != 0, grad != 0, rows == 128, adapters, 148);
  const int height = p.pairs ? 256 : 128, width = (p.pairs ? 256 : p.columns) / (two_columns ? 2 : 1);
  int64_t tiles = 0;
  for (int i = 0; i < problems; ++i) tiles += atenia::dense_ceil(s[i].M, height) * atenia::dense_ceil(s[i].N, width);
  return tiles * p.split;
}
extern "C" long long limits_most() { return atenia::kDenseMostTiles; }
