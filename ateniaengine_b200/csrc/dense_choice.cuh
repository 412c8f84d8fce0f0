// Which kernel a dense product takes, from its sizes alone (host arithmetic).
//
// Microseconds of each kernel, fitted to 310 products of five shapes (512 x 1408 to 4096 x 14336), 8 to 4096 tokens and each direction,
// run one after another on a B200 with their weights out of L2, every kernel at every split.  The kernel chosen is within 0.8 % of
// the fastest on average and 13 % at most; two rules by tile counts alone were 8 % and 2.2 times off.
//   a wave   : as many CTAs as are resident at once, given how clusters of a size fit the GPU's parts
//   a k-block: 0.32 us of a pair's 256 x 256 tile, 0.35 of 128 x 256 (its MMAs wait for shared memory), 0.30 of 128 x 128 alone on
//              its SM and 0.48 beside another
//   tail     : 2 us for a launch of its own
//   splits   : what adding the sums through distributed shared memory costs
//   adapters : 0.1 us of each on a tile of 128 columns (a batch of few rows may have one per row; up to 512 rows are taken for a decode
//              batch with up to 64 a tile, 300 rows of 90 requests beside 4096 x 4096 50 -> 27 us, of five 29 -> 23; more for prompts, of
//              which a tile has a few: 4000 rows of 90 requests through a block of 2048 x 5632 would go from 247 to 298; what that costs
//              where every row has its own, rank 16 beside 4096 x 4096: 512 rows 70 us, 513 160)
#pragma once
#include <stdint.h>

namespace atenia {

struct DenseSize {
  int64_t M, N;  // N: columns of the result
  int kb;        // k-blocks of 64
};
struct DensePlan {
  bool pairs;    // dense_pair.cu; else tiles of 128 x `columns` (dense_gemm.cu); the reduction cut `split` ways
  int columns;
  int split;
  int tail_split;  // pairs: of the tiles behind the last whole wave
};

// Tiles of a launch, times the CTAs or pairs that share one, at most: grids and tile indices are 32 bits.  No plan of sizes that the entry
// points take has more (2^24 rows of 2^20 columns of gate and up are 2^29 pair tiles).
constexpr int64_t kDenseMostTiles = (int64_t)1 << 29;

inline int64_t dense_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// rows: of A a stage holds (128 = all); two_columns: gate and up of a feature (kDenseSwiGLU); grad: kDenseGateGrad; full_rows: the
// pair kernel can take the call (its A boxes are 128 rows high); adapters: how many there are (0: none in this product)
inline DensePlan dense_plan(const DenseSize* sizes, int problems, int rows, bool two_columns, bool grad, bool full_rows, int adapters,
                            int num_sms) {
  // CTAs of a cluster of 1 .. 8 that are resident at once on 148 SMs, one or two an SM (cudaOccupancyMaxActiveClusters)
  static const int kAlone[9] = {0, 148, 148, 135, 132, 130, 132, 105, 120};
  static const int kTwice[9] = {0, 296, 296, 279, 284, 280, 270, 259, 264};
  const double scale = num_sms / 148.0;
  const int wide = two_columns ? 128 : 256;  // result columns of a tile of 256 MMA columns
  int64_t pairs = 0, tiles256 = 0, tiles128 = 0;
  int kb = 0, least_kb = 1 << 30;
  double bytes = 0;
  for (int i = 0; i < problems; ++i) {
    const DenseSize& s = sizes[i];
    pairs += dense_ceil(s.M, 256) * dense_ceil(s.N, wide);
    tiles256 += dense_ceil(s.M, 128) * dense_ceil(s.N, wide);
    tiles128 += dense_ceil(s.M, 128) * dense_ceil(s.N, wide / 2);
    kb = s.kb > kb ? s.kb : kb;
    least_kb = s.kb < least_kb ? s.kb : least_kb;
    bytes += 128.0 * s.kb * (s.M + (two_columns ? 2 : 1) * s.N) + (grad ? 14.0 : 2.0) * s.M * s.N;
  }
  const int most = sizes[0].M > 512 ? 8 : sizes[0].M > 128 ? 64 : (int)sizes[0].M;
  const double extra = 0.1 * (adapters < most ? adapters : most);
  const double floor = 4.5 + bytes / 5.35e6, f = rows / 128.0;
  DensePlan best{false, 128, 1, 1};
  double best_us = 1e30;
  auto offer = [&](bool p, int columns, int split, double us, int tail = 1) {
    us = (us > floor ? us : floor) + (adapters ? 0.5 : 0.05) * us;  // (of two that the bytes bound, the one with less to do)
    if (us < best_us) {
      best_us = us;
      best = {p, columns, split, tail};
    }
  };
  static const int kSplits[6] = {1, 2, 3, 4, 6, 8};
  for (int s : kSplits) {
    // (clusters of eight beside many adapters: 64 rows of 4096 x 4096 with 80 of rank 16 19.5 us, of six 16.8; 117 rows through a block of
    // 1008 x 1984 with 53 29.0 and 23.7; but with one adapter 23 rows through 352 x 13360 22.6 and 24.1)
    if (s > least_kb || (s == 8 && adapters > 4)) break;
    const double kc = (double)dense_ceil(kb, s);
    const bool cut = s > 1;
    if (full_rows && s <= 4) {
      const double w = (double)dense_ceil(pairs * s, (int64_t)(kAlone[2 * s] * scale) / 2);
      const double wave = 0.322 * kc + 1.6 + (cut ? 3.9 : 0.0) + (grad ? 5.5 : 0.0) + 2.5 * extra / s;
      offer(true, 256, s, 3.2 + w * wave);
      const int64_t room = (int64_t)(kAlone[2] * scale) / 2, whole = pairs / room, rest = pairs - whole * room;
      if (cut && whole > 0 && rest > 0) {
        const double full = 0.322 * kb + 1.6 + (grad ? 5.5 : 0.0) + 2.5 * extra;
        const double tail = (double)dense_ceil(rest * s, (int64_t)(kAlone[2 * s] * scale) / 2);
        offer(true, 256, 1, 5.2 + whole * full + tail * wave, s);
      }
    }
    {
      const double w = (double)dense_ceil(tiles256 * s, (int64_t)(kAlone[s] * scale));
      offer(false, 256, s, -0.4 + w * (0.348 * kc * (0.84 + 0.16 * f) + 5.4 + (cut ? 4.9 * f + 0.2 * s : grad ? 12.6 : 0.0) + 2.0 * extra / s));
    }
    {
      const int64_t n = tiles128 * s, room = (int64_t)(kTwice[s] * scale), w = dense_ceil(n, room);
      const double last = n - (w - 1) * room <= (int64_t)(kAlone[s] * scale) ? 0.30 : 0.477;
      offer(false, 128, s, -0.1 + kc * (0.72 + 0.28 * f) * ((w - 1) * 0.477 + last) + w * (3.6 + (grad && !cut ? 8.7 : 0.0) + extra / s) +
                               (cut ? w * 4.7 * f - 0.8 + 0.2 * s : 0.0));
    }
  }
  return best;
}

// adapters.cu: a tile of 128 token rows takes passes of so many adapters; CTAs side by side take the passes (lanes) or share one's reduction
// (split).  Microseconds: a pass's loads, sums and stores 2, a cluster's two barriers 2.2, a k-block 0.23; measured with clock64.  How many
// passes a tile has only the device knows: one per row in a decode batch, a few in a prompt.
// B200, whole calls: 2000 rows of 90 requests, rank 128 of 1024 inputs beside 4096 outputs 87.5 us with the greatest split, 77.3 so; a block of
// 1024 x 4096 with rank 64, 500 rows of 90 requests 95.1 and 87.8.
struct ReducePlan {
  int split, lanes;
};
inline ReducePlan reduce_plan(int64_t rows, int64_t tiles, int kb, int n, int per_pass, int num_sms) {
  const int64_t most = n < 128 ? (rows < n ? rows : n) : (rows < 128 ? rows : 128);
  const int64_t likely = rows > 512 ? 4 : rows > 128 ? 16 : rows;
  const int64_t passes = dense_ceil(most, per_pass), expected = dense_ceil(most < likely ? most : likely, per_pass);
  const int64_t places = 2 * num_sms;
  ReducePlan best{1, 1};
  double best_us = 1e30;
  for (int split = 1; split <= 8 && (split == 1 || kb >= 2 * split); split *= 2) {
    int64_t lanes = places / (tiles * split);
    lanes = lanes < 1 ? 1 : lanes > passes ? passes : lanes;
    const double waves = (double)dense_ceil(tiles * split * lanes, places), rounds = (double)dense_ceil(expected, lanes);
    const double us = waves * (1.6 + rounds * (0.23 * kb / split + 2.0 + (split > 1 ? 2.2 : 0.0)));
    if (us < best_us) {
      best_us = us;
      best = {split, (int)lanes};
    }
  }
  return best;
}

// dense_rows.cu: row groups, each cut in 1, 2, 4 or 8 pieces of the reduction (of two steps at least), `warps` of them to a block; the
// cut that leaves the fewest of the `places` for blocks empty in the last wave, the least one of equals.
struct RowsPlan {
  int pieces, blocks;
  double used;  // of the places in all waves
};
inline RowsPlan rows_plan(int groups, int steps, int warps, int places) {
  RowsPlan best{1, (int)dense_ceil(groups, warps), 0.0};
  for (int pieces = 1; pieces <= warps && (pieces == 1 || steps >= 2 * pieces); pieces *= 2) {
    const int64_t blocks = dense_ceil(groups, warps / pieces);
    const double used = (double)blocks / (double)(dense_ceil(blocks, places) * places);
    if (used > 1.01 * best.used) best = {pieces, (int)blocks, used};
  }
  return best;
}

}  // namespace atenia
