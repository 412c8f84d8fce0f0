// Test-only: compiles the choice of dense kernels with a host compiler.  Not part of the product library.
#include "../ateniaengine_b200/csrc/dense_choice.cuh"

// sizes: M, N, kb of each problem; out: pairs, columns, split, tail_split
extern "C" void choice_dense(const long long* sizes, int problems, int rows, int two_columns, int grad, int full_rows, int adapters,
                             int num_sms, int* out) {
  atenia::DenseSize s[3];
  for (int i = 0; i < problems; ++i) s[i] = {sizes[3 * i], sizes[3 * i + 1], (int)sizes[3 * i + 2]};
  const atenia::DensePlan p = atenia::dense_plan(s, problems, rows, two_columns != 0, grad != 0, full_rows != 0, adapters, num_sms);
  out[0] = p.pairs, out[1] = p.columns, out[2] = p.split, out[3] = p.tail_split;
}

// out: pieces, blocks
extern "C" void choice_rows(int groups, int steps, int warps, int places, int* out) {
  const atenia::RowsPlan p = atenia::rows_plan(groups, steps, warps, places);
  out[0] = p.pieces, out[1] = p.blocks;
}

// out: split, lanes
extern "C" void choice_reduce(long long rows, long long tiles, int kb, int n, int per_pass, int num_sms, int* out) {
  const atenia::ReducePlan p = atenia::reduce_plan(rows, tiles, kb, n, per_pass, num_sms);
  out[0] = p.split, out[1] = p.lanes;
}
