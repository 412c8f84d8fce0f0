// Dense products on one CTA per tile (tcgen05 cta_group::1): 128 rows x 128 or 256 columns, the reduction cut over a cluster.
//
// D[m, n] = sum_k A[m, k] B[n, k]; a lane of tensor memory holds a row of D, so the epilogue of a row (gate and up of a feature,
// the saved values, 32 contiguous bytes of the result) stays in one thread.
//   k-block: 64; a stage holds the A rows the call has (8 .. 128) and the tile's B rows (kDenseSwiGLU: half gate and half up rows)
//   split  : the CTAs of a cluster (1, 2, 3, 4, 6, 8) take consecutive k ranges of one tile and add their f32 sums through distributed
//            shared memory in rank order, so results do not depend on timing and nothing is kept in global memory
// What bounds it: for few rows the weights' bytes (two CTAs per SM with 100 KiB of loads in flight each, or one with 190: 37 rows, gate and
// up of 4096 x 14336 235 MB in 41 us, 5.7 TB/s); for some hundred rows the MMAs, which wait for shared memory (333 rows, 2048 x 5632: 11 of
// 17 us), and the 5 us before the first and after the last of them.
//
// Adapters: a CTA takes its share of the tile's adapters (in the order of their first rows, dealt over the ranks).  For adapter a it
// multiplies the tile's reduced rows v (K = 16 steps) by B_a with the lanes of all other rows disabled, so a row only ever adds
// its own adapter: no row is multiplied by zero for another one's, and infinities or NaN in an adapter stay with its own rows.
#include <type_traits>

#include "dense_gemm.cuh"

namespace atenia {
namespace {
using namespace tc;

constexpr int kTileStages = 8;   // at most

template <int BN>
struct TileSize {
  static constexpr int kEpiWarps = BN / 32;  // a warp has 128 columns of a quarter of the lanes
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kBBytes = BN * BK * 2;
  static constexpr int kRing = BN == 128 ? 108 * 1024 : 196 * 1024;  // two CTAs per SM, or one
};
constexpr int kTileSmemMax = 200 * 1024;

struct __align__(8) TileBars {
  uint64_t full[kTileStages];
  uint64_t empty[kTileStages];
  uint64_t acc_full;
  uint64_t listed;  // the tile's adapters are in shared memory
  uint64_t v_full;  // ... and their reduced rows
  uint32_t tmem_base;
  int abort_flag;
};

struct TileArgs {
  int problems, a_rows, stages, split, b_early, a_early, next_early;
  int v_bytes;                      // of the reduced rows, ahead of the ring
  int tile_end[kMaxDenseProblems];  // tiles of the problems up to and including this one
  DeviceError* err;
};
struct NoAdapters {};
template <int NP>
struct Problems {
  DenseProblem p[NP];
};

constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(128 >> 4) << 24);

struct TileMasks : TileList {
  int4 off[BM];  // of the listed adapters: bit set where a row has another one
};

template <int EPI, bool B_MN, int NP, bool AD, int BN>
__global__ void __launch_bounds__(TileSize<BN>::kThreads)
dense_tile_kernel(const __grid_constant__ Problems<NP> ps, const __grid_constant__ TileArgs ta,
                  const __grid_constant__ std::conditional_t<AD, DenseAdapters, NoAdapters> ad) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ TileBars bars;
  __shared__ std::conditional_t<AD, TileMasks, NoAdapters> list;
  constexpr int N_OUT = EPI == kDenseSwiGLU ? BN / 2 : BN;
  const uint32_t v_smem = (smem_u32(smem_raw) + 1023u) & ~1023u;  // reduced rows, then the ring; at the end the sums of a cut reduction
  const uint32_t ring = v_smem + (AD ? ta.v_bytes : 0);
  float* part = reinterpret_cast<float*>(smem_raw + (v_smem - smem_u32(smem_raw)));
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
  const int m_tiles = (p.M + BM - 1) / BM;
  const int nt = tile / m_tiles;  // tiles of the same B rows are neighbours
  const int m0 = (tile - nt * m_tiles) * BM, n0 = nt * N_OUT;
  const int rows = min(BM, p.M - m0), cols = min(N_OUT, p.N - n0);
  const int kb_begin = (int)((int64_t)p.kb * rank / split), kb_end = (int)((int64_t)p.kb * (rank + 1) / split);
  // The adapters' steps come before the last quarter of a long k range: their reduced rows are there by then, and the weights go on
  // arriving while their short MMAs are issued (48 tokens with 32 adapters, gate and up of 4096 x 14336: 2.5 us of 78).  Behind a short one,
  // which would wait for the rows half done (64 tokens beside 4096 x 4096, eight k-blocks a CTA: 17.4 / 19.7 us).
  const int kb_adapters = kb_end - kb_begin < 24 ? kb_end : kb_begin + (kb_end - kb_begin) * 3 / 4;
  const int stages = ta.stages;
  constexpr bool A_MN = NP > 1;
  const int a_bytes = ta.a_rows * BK * 2;
  const int stage_bytes = a_bytes + TileSize<BN>::kBBytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(smem_u32(&bars.full[s]), 1);
      mbar_init(smem_u32(&bars.empty[s]), 1);
    }
    mbar_init(smem_u32(&bars.acc_full), 1);
    mbar_init(smem_u32(&bars.listed), 4);
    mbar_init(smem_u32(&bars.v_full), 1);
    bars.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_base)),
                 "r"(BN)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem_base;

  // Adapters: this rank takes every split-th of the list.  A stage holds `group` of them, or (group 0) one chunk of one.
  const std::conditional_t<AD, AdapterChunks<EPI>, NoAdapters> ac(ad);
  int chunk_bytes = 0, v_bytes = 0, group = 0;
  if constexpr (AD) {
    chunk_bytes = N_OUT * ac.widest * 2;
    v_bytes = ta.a_rows * ac.widest * 2;
    group = stage_bytes / (chunk_bytes * ac.chunks);
  }
  auto give_up = [&](int site) {
    if (lane == 0) report_error(ta.err, ATENIA_ERR_DEVICE_TIMEOUT, site);
    *abort_flag = 1;
    return false;
  };
  auto wait_all = [&](uint64_t* bar, uint32_t parity, int site) {
    const bool ok = mbar_wait(smem_u32(bar), parity, abort_flag) || give_up(site);
    return __all_sync(0xffffffffu, ok) != 0;
  };

  if (warp == 0) {
    // ================= TMA producer =================
    int stage = 0;
    uint32_t phase = 0, armed = 0;
    bool ok = true;
    auto load_b = [&](int kb, uint32_t dst, uint32_t bar) {
      const int seg = EPI != kDenseSwiGLU && kb >= p.kb0;
      const int k = (kb - (seg ? p.kb0 : 0)) * BK;
#pragma unroll
      for (int j = 0; j < BN / 64; ++j) {
        if constexpr (EPI == kDenseSwiGLU) tma_load_2d_one(dst + 8192 * j, &p.b[j >= BN / 128], bar, k, n0 + 64 * (j % (BN / 128)));
        else tma_load_2d_one(dst + 8192 * j, &p.b[seg], bar, B_MN ? n0 + 64 * j : k, B_MN ? k : n0 + 64 * j);
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
    auto next_stage = [&]() {
      armed |= 1u << stage;
      if (++stage == stages) {
        stage = 0;
        phase ^= 1u;
      }
    };
    int ahead = 0;
    if (ta.b_early) {
      ahead = min((AD ? kb_adapters : kb_end) - kb_begin, stages);
      for (int i = 0; i < ahead; ++i) {
        const uint32_t bar = smem_u32(&bars.full[i]), dst = ring + i * stage_bytes;
        mbar_expect_tx_one(bar, stage_bytes);
        load_b(kb_begin + i, dst + a_bytes, bar);
        if (ta.a_early) load_a(kb_begin + i, dst, bar);
      }
    }
    if (!ta.a_early) {
      chain_wait();
      if (ta.next_early) chain_next();
    }
    auto load_blocks = [&](int from, int to) {
      for (int kb = from; kb < to; ++kb) {
        const uint32_t bar = smem_u32(&bars.full[stage]), dst = ring + stage * stage_bytes;
        if (kb - kb_begin < ahead) {
          if (!ta.a_early) load_a(kb, dst, bar);
        } else {
          if (!(ok = wait_all(&bars.empty[stage], phase ^ 1u, 2100 + stage))) break;
          mbar_expect_tx_one(bar, stage_bytes);
          load_b(kb, dst + a_bytes, bar);
          load_a(kb, dst, bar);
        }
        next_stage();
      }
    };
    load_blocks(kb_begin, AD ? kb_adapters : kb_end);
    if constexpr (AD) {
      // (B is not written by the kernel before; the reduced rows, which are, come with another warp)
      ok = ok && wait_all(&bars.listed, 0, 2110);
      const int count = ok ? list.count : 0;
      int left = count > rank ? (count - rank + split - 1) / split : 0;
      auto load_chunk = [&](int c, uint32_t dst, uint32_t bar, int adapter) {
        const CUtensorMap* map = &ad.seg[ac.second[c]].b;
#pragma unroll
        for (int j = 0; j < N_OUT / 64; ++j) tma_load_3d_one(dst + j * 128 * ac.width[c], map, bar, ac.column[c], n0 + 64 * j, adapter);
      };
      for (int i = rank; left > 0;) {
        const int here = group > 0 ? min(left, group) : 1;
        if (group > 0) {
          if (!(ok = wait_all(&bars.empty[stage], phase ^ 1u, 2120 + stage))) break;
          const uint32_t bar = smem_u32(&bars.full[stage]);
          uint32_t dst = ring + stage * stage_bytes;
          mbar_expect_tx_one(bar, here * ac.columns * N_OUT * 2);
          for (int s = 0; s < here; ++s, i += split) {
            const int adapter = list.adapter[i];
#pragma unroll
            for (int c = 0; c < kMaxChunks; ++c) {
              if (c >= ac.chunks) break;
              load_chunk(c, dst, bar, adapter);
              dst += chunk_bytes;
            }
          }
          next_stage();
        } else {
          const int adapter = list.adapter[i];
          i += split;
#pragma unroll
          for (int c = 0; c < kMaxChunks; ++c) {
            if (c >= ac.chunks) break;
            if (!(ok = wait_all(&bars.empty[stage], phase ^ 1u, 2120 + stage))) break;
            const uint32_t bar = smem_u32(&bars.full[stage]);
            mbar_expect_tx_one(bar, ac.width[c] * N_OUT * 2);
            load_chunk(c, ring + stage * stage_bytes, bar, adapter);
            next_stage();
          }
          if (!ok) break;
        }
        left -= here;
      }
      if (ok) load_blocks(kb_adapters, kb_end);
    }
    chain_wait();
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
      ok = wait_all(&bars.full[stage], phase, 2200 + stage);
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
    constexpr uint32_t idesc = kIdesc | (uint32_t(A_MN) << 15) | (uint32_t(B_MN) << 16) | (uint32_t(BN >> 3) << 17);
    auto multiply_blocks = [&](int from, int to) {
      for (int kb = from; kb < to; ++kb) {
        if (!filled()) break;
        const uint32_t sa = ring + stage * stage_bytes;
        const uint64_t da = operand_desc<A_MN>(sa), db = operand_desc<B_MN>(sa + a_bytes);
#pragma unroll
        for (int k = 0; k < BK / UMMA_K; ++k)
          tc_mma_bf16_one(tmem, da + k * kOperandStep<A_MN>, db + k * kOperandStep<B_MN>, idesc, kb > kb_begin || k > 0);
        used();
      }
    };
    multiply_blocks(kb_begin, AD ? kb_adapters : kb_end);
    if constexpr (AD) {
      ok = ok && wait_all(&bars.listed, 0, 2210);
      const int count = ok ? list.count : 0;
      int left = count > rank ? (count - rank + split - 1) / split : 0;
      if (left > 0) ok = wait_all(&bars.v_full, 0, 2220);
      uint32_t off[4] = {};
      uint64_t dv[kMaxChunks];
#pragma unroll
      for (int c = 0; c < kMaxChunks; ++c) dv[c] = make_smem_desc_width(v_smem + c * v_bytes, ac.width[c]);
      auto add_chunk = [&](int c, uint32_t at) {
        constexpr uint32_t idesc_ad = kIdesc | (uint32_t(N_OUT >> 3) << 17);
        const uint64_t db = make_smem_desc_width(at, ac.width[c]);
        const uint32_t d = tmem + (ac.second[c] ? N_OUT : 0);
        tc_mma_bf16_lanes_one(d, dv[c], db, idesc_ad, ac.steps[c], off);
        if (ad.parts > 1) tc_mma_bf16_lanes_one(d, dv[c] + (uint32_t)(ac.chunks * v_bytes >> 4), db, idesc_ad, ac.steps[c], off);
      };
      for (int i = rank; ok && left > 0;) {
        const int here = group > 0 ? min(left, group) : 1;
        if (group > 0 && !filled()) break;
        uint32_t at = ring + stage * stage_bytes;
        for (int s = 0; s < here; ++s, i += split) {
          const int4 m = list.off[i];
          off[0] = m.x, off[1] = m.y, off[2] = m.z, off[3] = m.w;
#pragma unroll
          for (int c = 0; c < kMaxChunks; ++c) {
            if (c >= ac.chunks) break;
            if (group == 0) {
              if (!filled()) break;
              at = ring + stage * stage_bytes;
            }
            add_chunk(c, at);
            at += chunk_bytes;
            if (group == 0) used();
          }
        }
        if (group > 0) used();
        left -= here;
      }
      if (ok) multiply_blocks(kb_adapters, kb_end);
    }
    if (ok) tc_commit_one(smem_u32(&bars.acc_full));
  } else {
    // ================= epilogue =================
    if constexpr (AD) {
      if (warp < 6) {
        list_adapters(list, ad.ids, m0, rows, ad.n, warp - 2, lane);
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const int32_t mine = list.id[32 * (warp - 2) + lane];
        for (int i = 0; i < list.count; ++i) {
          const uint32_t off = __ballot_sync(0xffffffffu, mine != list.adapter[i]);
          if (lane == 0) reinterpret_cast<uint32_t*>(&list.off[i])[warp - 2] = off;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bars.listed));
      }
    }
    chain_wait();
    if constexpr (AD) {
      if (warp == 2 && wait_all(&bars.listed, 0, 2310) && list.count > rank) {
        const uint32_t bar = smem_u32(&bars.v_full);
        mbar_expect_tx_one(bar, ad.parts * ta.a_rows * 2 * ac.columns);
        for (int q = 0; q < ad.parts; ++q)
#pragma unroll
          for (int c = 0; c < kMaxChunks; ++c)
            if (c < ac.chunks) tma_load_3d_one(v_smem + (q * ac.chunks + c) * v_bytes, &ad.seg[ac.second[c]].v, bar, ac.column[c], m0, q);
        if (*abort_flag)
          for (int i = 0; i < (1 << 16) && !mbar_try_wait(bar, 0); ++i) {}
      }
    }
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    constexpr int kShares = BN / 128;  // warps of a quarter: each its share of the columns
    constexpr int kCols = N_OUT / kShares;
    const int share = (warp - 2) >> 2;
    const int end = min(cols, (share + 1) * kCols);
    Saved<EPI, 16> kept, next;
    if (split == 1) kept.load(p, m0 + row, n0 + share * kCols, row < rows && share * kCols < end);
    if (!wait_all(&bars.acc_full, 0, 2300)) {
      // (reported)
    } else if (quarter * 32 < rows) {
      tc_fence_after();
      const uint32_t taddr = tmem + (uint32_t(quarter * 32) << 16);
      if (split == 1) {
#pragma unroll 2
        for (int c = share * kCols; c < end; c += 16) {
          next.load(p, m0 + row, n0 + c + 16, row < rows && c + 16 < end);
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
          if (row < rows) dense_emit<EPI, 16>(p, m0 + row, n0 + c, f, f1, kept);
          kept = next;
        }
      } else {
#pragma unroll 2
        for (int c = share * 128; c < share * 128 + 128; c += 16) {
          uint32_t v[16];
          tc_ld16(taddr + c, v);
          tc_ld_wait();
          if (row < rows) {
            uint4* dst = reinterpret_cast<uint4*>(part + row * kSumsPitch<BN> + c);
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
      const uint32_t at = smem_u32(part);
      switch (split) {
        case 2: add_parts<EPI, BN, 2, 1>(p, m0, n0, rows, cols, at, rank, 0); break;
        case 3: add_parts<EPI, BN, 3, 1>(p, m0, n0, rows, cols, at, rank, 0); break;
        case 4: add_parts<EPI, BN, 4, 1>(p, m0, n0, rows, cols, at, rank, 0); break;
        case 6: add_parts<EPI, BN, 6, 1>(p, m0, n0, rows, cols, at, rank, 0); break;
        default: add_parts<EPI, BN, 8, 1>(p, m0, n0, rows, cols, at, rank, 0); break;
      }
    }
    __syncthreads();
    cluster_barrier();  // no CTA leaves while another reads its sums
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(BN) : "memory");
  }
}

// Of the reduced rows of a tile in shared memory
int reduced_row_bytes(const DenseGemm& g) {
  if (!g.adapters) return 0;
  int chunks = 0, width = 0;
  for (int i = 0; i < (g.epilogue == kDenseSwiGLU ? 2 : 1); ++i) {
    const AdapterSegment& seg = g.adapters->seg[i];
    if (seg.rank == 0) continue;
    chunks += (seg.rank + seg.width - 1) / seg.width;
    width = seg.width > width ? seg.width : width;
  }
  return (g.adapters->parts * chunks * g.a_rows * width * 2 + 1023) / 1024 * 1024;
}

template <int EPI, bool B_MN, int NP, bool AD, int BN>
int launch_tiles(const DenseGemm& g, TileArgs ta, int tiles, cudaStream_t s) {
  auto kernel = dense_tile_kernel<EPI, B_MN, NP, AD, BN>;
  static FirstUse ready[kMaxDevices];
  if (const int rc = allow_shared_memory(ready, kernel, kTileSmemMax)) return rc;
  const int rows = g.a_rows;
  const int stage_bytes = rows * BK * 2 + TileSize<BN>::kBBytes;
  std::conditional_t<AD, DenseAdapters, NoAdapters> ad{};
  if constexpr (AD) ad = *g.adapters;
  int ring = TileSize<BN>::kRing - ta.v_bytes;
  if (ring < 2 * stage_bytes) ring = TileSize<256>::kRing - ta.v_bytes;  // (many reduced rows: one CTA per SM)
  ta.stages = ring / stage_bytes;
  if (ta.stages > kTileStages) ta.stages = kTileStages;
  const int sums = ta.split > 1 ? rows * kSumsPitch<BN> * 4 : 0, operands = ta.v_bytes + ta.stages * stage_bytes;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ta.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(tiles * ta.split);
  cfg.blockDim = dim3(TileSize<BN>::kThreads);
  cfg.dynamicSmemBytes = 1024 + (operands > sums ? operands : sums);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = g.chained ? 2 : 1;
  Problems<NP> ps;
  for (int i = 0; i < NP; ++i) ps.p[i] = g.p[i];
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, ps, ta, ad);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return (int)e;
}

template <int BN>
int launch_tiles_of(const DenseGemm& g, const TileArgs& ta, int tiles, cudaStream_t s) {
  const bool ad = g.adapters != nullptr;
  const bool b_mn = g.p[0].b_mn;
  if (g.problems > 1)
    return g.epilogue == kDensePlain && b_mn && !ad ? launch_tiles<kDensePlain, true, kMaxDenseProblems, false, BN>(g, ta, tiles, s) : ATENIA_ERR_UNSUPPORTED;
  if (ad && b_mn) return ATENIA_ERR_UNSUPPORTED;
  if (g.epilogue == kDenseSwiGLU && !b_mn)
    return ad ? launch_tiles<kDenseSwiGLU, false, 1, true, BN>(g, ta, tiles, s) : launch_tiles<kDenseSwiGLU, false, 1, false, BN>(g, ta, tiles, s);
  if (g.epilogue == kDensePlain)
    return ad     ? launch_tiles<kDensePlain, false, 1, true, BN>(g, ta, tiles, s)
           : b_mn ? launch_tiles<kDensePlain, true, 1, false, BN>(g, ta, tiles, s)
                  : launch_tiles<kDensePlain, false, 1, false, BN>(g, ta, tiles, s);
  if (g.epilogue == kDenseGateGrad && b_mn && !ad) return launch_tiles<kDenseGateGrad, true, 1, false, BN>(g, ta, tiles, s);
  return ATENIA_ERR_UNSUPPORTED;
}

}  // namespace

int launch_dense_tiles(const DenseGemm& g, int columns, int split, cudaStream_t s) {
  if (split < 1 || split > 8 || split == 5 || split == 7 || (columns != 128 && columns != 256)) return ATENIA_ERR_SHAPE;
  TileArgs ta{};
  int rc = dense_error_word(&ta.err);
  if (rc) return rc;
  const int n_out = g.epilogue == kDenseSwiGLU ? columns / 2 : columns;
  int64_t tiles = 0;
  for (int i = 0; i < g.problems; ++i) {
    const DenseProblem& p = g.p[i];
    tiles += (int64_t)((p.M + BM - 1) / BM) * ((p.N + n_out - 1) / n_out);
    if (tiles * split > kDenseMostTiles) return ATENIA_ERR_SHAPE;
    if (p.kb < split) return ATENIA_ERR_SHAPE;
    ta.tile_end[i] = (int)tiles;
  }
  if (tiles == 0) return ATENIA_OK;
  ta.problems = g.problems;
  ta.a_rows = g.a_rows;
  ta.b_early = g.b_early;
  ta.a_early = g.a_early && g.b_early;
  ta.next_early = g.next_early;
  ta.split = split;
  ta.v_bytes = reduced_row_bytes(g);
  // (a ring of two stages at least)
  if (columns == 256 && ta.v_bytes + 2 * (g.a_rows * BK * 2 + TileSize<256>::kBBytes) > TileSize<256>::kRing) return launch_dense_tiles(g, 128, split, s);
  count_launch();
  count_tcgen05_launch();
  return columns == 256 ? launch_tiles_of<256>(g, ta, (int)tiles, s) : launch_tiles_of<128>(g, ta, (int)tiles, s);
}

int launch_dense_gemm(const DenseGemm& g, int num_sms, cudaStream_t s) {
  if (dense_rows_serve(g)) return launch_dense_rows(g, num_sms, s);
  DenseSize sizes[kMaxDenseProblems];
  for (int i = 0; i < g.problems; ++i) sizes[i] = {g.p[i].M, g.p[i].N, g.p[i].kb};
  const DensePlan plan =
      dense_plan(sizes, g.problems, g.a_rows, g.epilogue == kDenseSwiGLU, g.epilogue == kDenseGateGrad, g.a_rows == BM,
                 g.adapters ? g.adapters->n : 0, num_sms);
  if (plan.pairs) return launch_dense_pairs(g, plan.split, plan.tail_split, num_sms, s);
  return launch_dense_tiles(g, plan.columns, plan.split, s);
}

}  // namespace atenia
