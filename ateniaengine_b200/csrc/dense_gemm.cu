// Dense products on one CTA per tile (tcgen05 cta_group::1): 128 rows x 128 columns, the reduction cut over a cluster.
//
// D[m, n] = sum_k A[m, k] B[n, k]; a lane of tensor memory holds a row of D, so the epilogue of a row (gate and up of a feature,
// the saved values, 32 contiguous bytes of the result) stays in one thread.
//   k-block: 64; a stage holds the A rows the call has (8 .. 128) and 128 B rows (kDenseSwiGLU: 64 gate and 64 up rows)
//   split  : the CTAs of a cluster (1, 2, 4, 8) take consecutive k ranges of one tile and add their f32 sums through distributed
//            shared memory in rank order, so results do not depend on timing and nothing is kept in global memory
// What bounds it: for few rows the weights' bytes (two CTAs per SM, 80 to 100 KiB of loads in flight each).
//
// Adapters: after its k range a CTA takes its share of the tile's adapters (ascending ids, dealt over the ranks).  For adapter a it
// multiplies the tile's reduced rows v (K = 16 steps) by B_a with the lanes of all other rows disabled, so a row only ever adds
// its own adapter: no row is multiplied by zero for another one's, and infinities or NaN in an adapter stay with its own rows.
#include <type_traits>

#include "dense_gemm.cuh"

namespace atenia {
namespace {
using namespace tc;

constexpr int kTileN = 128;
constexpr int kTileStages = 8;   // at most
constexpr int kTileThreads = 192;
constexpr int kTmemCols = 128;
constexpr int kBBytes = kTileN * BK * 2;
constexpr int kMaxSplit = 8;
constexpr int kRingBytes = 100 * 1024;  // two CTAs per SM
constexpr int kPartPitch = kTileN + 4;         // floats: eight lanes' 16-byte accesses fall into different banks
constexpr int kPartBytes = BM * kPartPitch * 4;  // f32 sums of a tile [row][column]
static_assert(kPartBytes <= kRingBytes, "the sums take the ring's place");

struct __align__(8) TileBars {
  uint64_t full[kTileStages];
  uint64_t empty[kTileStages];
  uint64_t acc_full;
  uint32_t tmem_base;
  int abort_flag;
};

struct TileArgs {
  int problems, a_rows, stages, split, b_early, a_early;
  int tile_end[kMaxDenseProblems];  // tiles of the problems up to and including this one
  DeviceError* err;
};
struct NoAdapters {};
template <int NP>
struct Problems {
  DenseProblem p[NP];
};

constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(128 >> 4) << 24);

// This rank's share of a tile whose sums lie in the shared memory of the S CTAs: four columns a thread, columns fastest, all S loads
// on their way before the first is added; added in rank order.
template <int EPI, int S>
__device__ __forceinline__ void add_parts(const DenseProblem& p, int64_t at0, int rows, int cols, uint32_t part, int rank) {
  constexpr int N_OUT = EPI == kDenseSwiGLU ? kTileN / 2 : kTileN;
  const int quads = cols / 4, total = rows * quads;
  const int begin = total * rank / S, end = total * (rank + 1) / S;
#pragma unroll 1
  for (int i = begin + (int)threadIdx.x; i < end; i += kTileThreads) {
    const int r = i / quads, c = 4 * (i - r * quads);
    const uint32_t at = part + (r * kPartPitch + c) * 4;
    float4 v[S], v1[EPI == kDenseSwiGLU ? S : 1];
#pragma unroll
    for (int q = 0; q < S; ++q) {
      v[q] = ld_cluster_f32x4(at, q);
      if constexpr (EPI == kDenseSwiGLU) v1[q] = ld_cluster_f32x4(at + N_OUT * 4, q);
    }
    float acc[4] = {}, acc1[4] = {};
#pragma unroll
    for (int q = 0; q < S; ++q) {
      acc[0] += v[q].x, acc[1] += v[q].y, acc[2] += v[q].z, acc[3] += v[q].w;
      if constexpr (EPI == kDenseSwiGLU) acc1[0] += v1[q].x, acc1[1] += v1[q].y, acc1[2] += v1[q].z, acc1[3] += v1[q].w;
    }
    dense_emit4<EPI>(p, at0 + (int64_t)r * p.N + c, acc, acc1);
  }
}

template <int EPI, bool A_MN, bool B_MN, int NP, bool AD>
__global__ void __launch_bounds__(kTileThreads)
dense_tile_kernel(const __grid_constant__ Problems<NP> ps, const __grid_constant__ TileArgs ta,
                  const __grid_constant__ std::conditional_t<AD, DenseAdapters, NoAdapters> ad) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ TileBars bars;
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  float* part = reinterpret_cast<float*>(smem_raw + (ring - smem_u32(smem_raw)));
  volatile int* abort_flag = &bars.abort_flag;
  const int warp = uniform_warp();
  const int lane = threadIdx.x & 31;
  const int split = ta.split;
  const int rank = split > 1 ? (int)cluster_rank() : 0;

  int tile = blockIdx.x / split, which = 0;
  if constexpr (NP > 1) {
    while (which + 1 < ta.problems && tile >= ta.tile_end[which]) ++which;
    if (which > 0) tile -= ta.tile_end[which - 1];
  }
  const DenseProblem& p = ps.p[NP > 1 ? which : 0];
  constexpr int N_OUT = EPI == kDenseSwiGLU ? kTileN / 2 : kTileN;
  const int m_tiles = (p.M + BM - 1) / BM;
  const int nt = tile / m_tiles;  // tiles of the same B rows are neighbours
  const int m0 = (tile - nt * m_tiles) * BM, n0 = nt * N_OUT;
  const int rows = min(BM, p.M - m0), cols = min(N_OUT, p.N - n0);
  const int kb_begin = (int)((int64_t)p.kb * rank / split), kb_end = (int)((int64_t)p.kb * (rank + 1) / split);
  const int stages = ta.stages;
  const int a_bytes = A_MN ? BM * BK * 2 : ta.a_rows * BK * 2;
  const int stage_bytes = a_bytes + kBBytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(smem_u32(&bars.full[s]), 1);
      mbar_init(smem_u32(&bars.empty[s]), 1);
    }
    mbar_init(smem_u32(&bars.acc_full), 1);
    bars.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem_base;

  if (warp == 0) {
    // ================= TMA producer =================
    int stage = 0;
    uint32_t phase = 0, armed = 0;
    bool ok = true;
    auto load_b = [&](int kb, uint32_t dst, uint32_t bar) {
      const int seg = EPI != kDenseSwiGLU && kb >= p.kb0;
      const int k = (kb - (seg ? p.kb0 : 0)) * BK;
      if constexpr (EPI == kDenseSwiGLU) {
        tma_load_2d_one(dst, &p.b[0], bar, k, n0);
        tma_load_2d_one(dst + 8192, &p.b[1], bar, k, n0);
      } else if constexpr (B_MN) {
        tma_load_2d_one(dst, &p.b[seg], bar, n0, k);
        tma_load_2d_one(dst + 8192, &p.b[seg], bar, n0 + 64, k);
      } else {
        tma_load_2d_one(dst, &p.b[seg], bar, k, n0);
        tma_load_2d_one(dst + 8192, &p.b[seg], bar, k, n0 + 64);
      }
    };
    auto load_a = [&](int kb, uint32_t dst, uint32_t bar) {
      const int seg = EPI != kDenseSwiGLU && kb >= p.kb0;
      const int k = (kb - (seg ? p.kb0 : 0)) * BK;
      if constexpr (A_MN) {
        tma_load_2d_one(dst, &p.a[seg], bar, m0, k);
        tma_load_2d_one(dst + 8192, &p.a[seg], bar, m0 + 64, k);
      } else {
        tma_load_2d_one(dst, &p.a[seg], bar, k, m0);
      }
    };
    auto free_stage = [&]() {
      if (!mbar_wait(smem_u32(&bars.empty[stage]), phase ^ 1u, abort_flag)) {
        if (lane == 0) report_error(ta.err, ATENIA_ERR_DEVICE_TIMEOUT, 2100 + stage);
        *abort_flag = 1;
        ok = false;
      }
      ok = __all_sync(0xffffffffu, ok);
      return ok;
    };
    auto next_stage = [&]() {
      armed |= 1u << stage;
      if (++stage == stages) {
        stage = 0;
        phase ^= 1u;
      }
    };
    int ahead = 0;
    if (ta.b_early) {
      ahead = min(kb_end - kb_begin, stages);
      for (int i = 0; i < ahead; ++i) {
        const uint32_t bar = smem_u32(&bars.full[i]), dst = ring + i * stage_bytes;
        mbar_expect_tx_one(bar, stage_bytes);
        load_b(kb_begin + i, dst + a_bytes, bar);
        if (ta.a_early) load_a(kb_begin + i, dst, bar);
      }
    }
    if (!(AD && ta.a_early)) chain_wait();
    for (int kb = kb_begin; kb < kb_end; ++kb) {
      const uint32_t bar = smem_u32(&bars.full[stage]), dst = ring + stage * stage_bytes;
      if (kb - kb_begin < ahead) {
        if (!ta.a_early) load_a(kb, dst, bar);
      } else {
        if (!free_stage()) break;
        mbar_expect_tx_one(bar, stage_bytes);
        load_b(kb, dst + a_bytes, bar);
        load_a(kb, dst, bar);
      }
      next_stage();
    }
    if constexpr (AD) {
      chain_wait();  // v is the kernel before's
      int32_t id[4];
      load_ids(id, ad.ids, m0, rows, ad.n, lane);
      int32_t a = -1;
      for (int i = 0; ok && (a = next_adapter(id, a)) != kNoAdapter; ++i) {
        if (i % split != rank) continue;
        for (int seg = 0; ok && seg < (EPI == kDenseSwiGLU ? 2 : 1); ++seg) {
          const int r = ad.seg[seg].rank;
          for (int r0 = 0; ok && r0 < r; r0 += 64) {
            if (!free_stage()) break;
            const int steps = (min(r - r0, 64) + 15) / 16;
            const uint32_t bar = smem_u32(&bars.full[stage]), dst = ring + stage * stage_bytes;
            constexpr int b_step = EPI == kDenseSwiGLU ? 2048 : 4096;
            mbar_expect_tx_one(bar, steps * (ta.a_rows * 32 + b_step));
            for (int c = 0; c < steps; ++c) {
              tma_load_2d_one(dst + c * ta.a_rows * 32, &ad.seg[seg].v, bar, r0 + 16 * c, m0);
              tma_load_3d_one(dst + a_bytes + c * 4096, &ad.seg[seg].b, bar, r0 + 16 * c, n0, a);
              if constexpr (EPI != kDenseSwiGLU)
                tma_load_3d_one(dst + a_bytes + c * 4096 + 2048, &ad.seg[seg].b, bar, r0 + 16 * c, n0 + 64, a);
            }
            next_stage();
          }
        }
      }
    }
    chain_next();  // (every load is on its way: what follows may be launched)
    if (*abort_flag && lane == 0) {
      // let the copies already issued land before the shared memory is released
      for (int s = 0; s < stages; ++s) {
        if (!(armed & (1u << s))) continue;
        const uint32_t par = s < stage ? phase : phase ^ 1u;
        for (int i = 0; i < (1 << 16) && !mbar_try_wait(smem_u32(&bars.full[s]), par); ++i) {}
      }
    }
  } else if (warp == 1) {
    // ================= MMA issuer =================
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    auto filled = [&]() {
      if (!mbar_wait(smem_u32(&bars.full[stage]), phase, abort_flag)) {
        if (lane == 0) report_error(ta.err, ATENIA_ERR_DEVICE_TIMEOUT, 2200 + stage);
        *abort_flag = 1;
        ok = false;
      }
      ok = __all_sync(0xffffffffu, ok);
      if (ok) tc_fence_after();
      return ok;
    };
    auto used = [&]() {
      tc_commit_one(smem_u32(&bars.empty[stage]));
      if (++stage == stages) {
        stage = 0;
        phase ^= 1u;
      }
    };
    constexpr uint32_t idesc = kIdesc | (uint32_t(A_MN) << 15) | (uint32_t(B_MN) << 16) | (uint32_t(kTileN >> 3) << 17);
    for (int kb = kb_begin; kb < kb_end; ++kb) {
      if (!filled()) break;
      const uint32_t sa = ring + stage * stage_bytes;
      const uint64_t da = operand_desc<A_MN>(sa), db = operand_desc<B_MN>(sa + a_bytes);
#pragma unroll
      for (int k = 0; k < BK / UMMA_K; ++k)
        tc_mma_bf16_one(tmem, da + k * kOperandStep<A_MN>, db + k * kOperandStep<B_MN>, idesc, kb > kb_begin || k > 0);
      used();
    }
    if constexpr (AD) {
      int32_t id[4];
      uint32_t off[4];
      load_ids(id, ad.ids, m0, rows, ad.n, lane);
      int32_t a = -1;
      for (int i = 0; ok && (a = next_adapter(id, a)) != kNoAdapter; ++i) {
        if (i % split != rank) continue;
        lanes_off(off, id, a);
        for (int seg = 0; ok && seg < (EPI == kDenseSwiGLU ? 2 : 1); ++seg) {
          const int r = ad.seg[seg].rank;
          for (int r0 = 0; ok && r0 < r; r0 += 64) {
            if (!filled()) break;
            const int steps = (min(r - r0, 64) + 15) / 16;
            const uint32_t sa = ring + stage * stage_bytes;
            constexpr uint32_t idesc_ad = kIdesc | (uint32_t(N_OUT >> 3) << 17);
            for (int c = 0; c < steps; ++c)
              tc_mma_bf16_lanes_one(tmem + seg * N_OUT, make_smem_desc_k16(sa + c * ta.a_rows * 32),
                                    make_smem_desc_k16(sa + a_bytes + c * 4096), idesc_ad, off);
            used();
          }
        }
      }
    }
    if (ok) tc_commit_one(smem_u32(&bars.acc_full));
  } else {
    // ================= epilogue (warps 2..5) =================
    chain_wait();
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const bool ready = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.acc_full), 0, abort_flag));
    if (!ready) {
      if (lane == 0) report_error(ta.err, ATENIA_ERR_DEVICE_TIMEOUT, 2300);
      *abort_flag = 1;
    } else if (quarter * 32 < rows) {
      tc_fence_after();
      const uint32_t taddr = tmem + (uint32_t(quarter * 32) << 16);
      if (split == 1) {
#pragma unroll 1
        for (int c = 0; c < cols; c += 16) {
          uint32_t v[16], v1[16];
          tc_ld16(taddr + c, v);
          if constexpr (EPI == kDenseSwiGLU) tc_ld16(taddr + N_OUT + c, v1);
          tc_ld_wait();
          float f[16], f1[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            f[j] = __uint_as_float(v[j]);
            f1[j] = EPI == kDenseSwiGLU ? __uint_as_float(v1[j]) : 0.f;
          }
          if (row < rows) dense_emit16<EPI>(p, (int64_t)(m0 + row) * p.N + n0 + c, f, f1);
        }
      } else {
#pragma unroll 2
        for (int c = 0; c < kTileN; c += 16) {
          uint32_t v[16];
          tc_ld16(taddr + c, v);
          tc_ld_wait();
          if (row < rows) {
            uint4* dst = reinterpret_cast<uint4*>(part + row * kPartPitch + c);
#pragma unroll
            for (int j = 0; j < 4; ++j) dst[j] = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          }
        }
      }
      tc_fence_before();
    }
  }

  if (split > 1) {
    __syncthreads();
    cluster_barrier();
    if (!*abort_flag) {
      const int64_t at0 = (int64_t)m0 * p.N + n0;
      if (split == 2) add_parts<EPI, 2>(p, at0, rows, cols, smem_u32(part), rank);
      else if (split == 4) add_parts<EPI, 4>(p, at0, rows, cols, smem_u32(part), rank);
      else add_parts<EPI, 8>(p, at0, rows, cols, smem_u32(part), rank);
    }
    __syncthreads();
    cluster_barrier();  // no CTA leaves while another reads its sums
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

template <int EPI, bool A_MN, bool B_MN, int NP, bool AD>
int launch_tiles(const DenseGemm& g, const TileArgs& ta, int grid, int smem, cudaStream_t s) {
  auto kernel = dense_tile_kernel<EPI, A_MN, B_MN, NP, AD>;
  static bool attr_set[kMaxDevices] = {};
  if (first_use_on_current_device(attr_set)) {
    ATENIA_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes + 1024));
  }
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ta.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = g.chained ? 2 : 1;
  Problems<NP> ps;
  for (int i = 0; i < NP; ++i) ps.p[i] = g.p[i];
  std::conditional_t<AD, DenseAdapters, NoAdapters> ad{};
  if constexpr (AD) ad = *g.adapters;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, ps, ta, ad);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return (int)e;
}

}  // namespace

int launch_dense_tiles(const DenseGemm& g, int num_sms, cudaStream_t s) {
  TileArgs ta{};
  int rc = dense_error_word(&ta.err);
  if (rc) return rc;
  const int n_out = g.epilogue == kDenseSwiGLU ? kTileN / 2 : kTileN;
  int64_t tiles = 0;
  int min_kb = 1 << 30;
  for (int i = 0; i < g.problems; ++i) {
    const DenseProblem& p = g.p[i];
    tiles += (int64_t)((p.M + BM - 1) / BM) * ((p.N + n_out - 1) / n_out);
    if (tiles > (1 << 26)) return ATENIA_ERR_SHAPE;
    ta.tile_end[i] = (int)tiles;
    if (p.kb < min_kb) min_kb = p.kb;
  }
  if (tiles == 0) return ATENIA_OK;
  ta.problems = g.problems;
  ta.a_rows = g.a_rows;
  ta.b_early = g.b_early;
  ta.a_early = g.a_early && g.b_early;
  // clusters until every SM has a CTA, each with four k-blocks at least
  ta.split = 1;
  while (ta.split < kMaxSplit && tiles * ta.split < num_sms && min_kb >= 8 * ta.split) ta.split *= 2;
  const int stage_bytes = (g.a_mn ? BM * BK * 2 : g.a_rows * BK * 2) + kBBytes;
  ta.stages = kRingBytes / stage_bytes;
  if (ta.stages > kTileStages) ta.stages = kTileStages;
  const int grid = (int)tiles * ta.split;
  const int smem = kRingBytes + 1024;
  count_launch();
  count_tcgen05_launch();
  const bool ad = g.adapters != nullptr;
  if (g.epilogue == kDenseSwiGLU && !g.a_mn && !g.b_mn && g.problems == 1)
    return ad ? launch_tiles<kDenseSwiGLU, false, false, 1, true>(g, ta, grid, smem, s)
              : launch_tiles<kDenseSwiGLU, false, false, 1, false>(g, ta, grid, smem, s);
  if (g.epilogue == kDensePlain && !g.a_mn && !g.b_mn && g.problems == 1)
    return ad ? launch_tiles<kDensePlain, false, false, 1, true>(g, ta, grid, smem, s)
              : launch_tiles<kDensePlain, false, false, 1, false>(g, ta, grid, smem, s);
  if (ad) return ATENIA_ERR_UNSUPPORTED;
  if (g.epilogue == kDenseGateGrad && !g.a_mn && g.b_mn && g.problems == 1)
    return launch_tiles<kDenseGateGrad, false, true, 1, false>(g, ta, grid, smem, s);
  if (g.epilogue == kDensePlain && !g.a_mn && g.b_mn && g.problems == 1)
    return launch_tiles<kDensePlain, false, true, 1, false>(g, ta, grid, smem, s);
  if (g.epilogue == kDensePlain && g.a_mn && g.b_mn && g.problems == 3)
    return launch_tiles<kDensePlain, true, true, 3, false>(g, ta, grid, smem, s);
  return ATENIA_ERR_UNSUPPORTED;
}

int launch_dense_gemm(const DenseGemm& g, int num_sms, cudaStream_t s) {
  if (dense_gemv_serves(g)) return launch_dense_gemv(g, num_sms, s);
  // pairs where every pair of SMs has a tile
  const int n_out = g.epilogue == kDenseSwiGLU ? 128 : 256;
  int64_t tiles = 0;
  for (int i = 0; i < g.problems; ++i) tiles += (int64_t)((g.p[i].M + 255) / 256) * ((g.p[i].N + n_out - 1) / n_out);
  if ((g.a_mn || g.a_rows == BM) && tiles >= num_sms / 2) return launch_dense_pairs(g, num_sms, s);
  return launch_dense_tiles(g, num_sms, s);
}

}  // namespace atenia
