// Dense products on CTA pairs (tcgen05 cta_group::2): tiles of 256 rows x 256 columns, for calls of many rows.
//
// Two CTAs on the two SMs of a TPC stage 128 A rows and half of the 256 B rows each (kDenseSwiGLU: rank 0 the gate rows of 128
// features, rank 1 their up rows) and the leader issues M256 x N256 x K16 MMAs over both CTAs' shared memory, so that a byte
// brought to an SM is used for twice the products of a single CTA's tile (whose MMAs wait for shared memory: 128 x 256 of one CTA
// reads and writes 192 bytes a cycle at full rate, a pair 128).  Persistent: one CTA per SM, two accumulators in tensor memory, so that the
// epilogue of a tile runs under the MMAs of the next.
//   k-block : 64; a stage is 16 KiB of A and 16 KiB of B per CTA, six stages (kDenseGateGrad five)
//   order   : bands of kBand row tiles, column tile by column tile, so that the 74 tiles at work at one time share few operand rows in L2
//   split   : where the tiles are too few, or the last wave's are, the pairs of a cluster (two, three or four) share a tile: consecutive k
//             ranges, added through distributed shared memory in rank order.  (The last wave is a launch of its own then: 5000 tokens of
//             2048 x 5632 have two whole waves of tiles and twelve tiles in the second product.)
//   epilogue: eight warps; a lane holds a row, so the results go through shared memory to TMA, which writes whole lines (32 bytes a
//             lane were 32 lines an access, and a tile's 5400 cycles of them hid only behind a reduction of 700 and more)
//
// Adapters as in dense_gemm.cu: behind the k-blocks of a tile come the steps of the adapters that its rows have, with the lanes
// of other rows disabled.  What an adapter costs is its MMAs over all 256 rows and their masks (about 600 cycles a tile and adapter at
// rank 32 of gate and up).  What bounds the rest: the power cap (5000 tokens of 2048 x 5632: 223 us cold, 1.55 PFLOP/s; 270 in a loop, at the
// rate that the library's product sustains), and whole waves of tiles for some thousand rows.
//
// No TMA multicast is used: every CTA fetches its own tiles (cp.async.bulk.tensor ... cta_group::2 only routes the completion to
// the leader's mbarrier).  Barriers: full[s] lives in the leader and collects the bytes of both CTAs; empty[s] and acc_full[b] exist
// in both CTAs and are signalled by tcgen05.commit with a CTA mask; acc_empty[b] lives in the leader and is arrived on by the
// epilogue warps of both CTAs.
#include <type_traits>

#include "dense_gemm.cuh"

namespace atenia {
namespace {
using namespace tc;

constexpr int kPairM = 256, kPairN = 256;
constexpr int kPairStages = 6;  // at most
constexpr int kOperandBytes = BM * BK * 2;  // 16 KiB of A, and of B
constexpr int kPairStageBytes = 2 * kOperandBytes;
constexpr int kEpiWarps = 8;
constexpr int kPairThreads = 64 + 32 * kEpiWarps;
constexpr int kPairTmemCols = 512;
// Behind the ring each epilogue warp has a piece of shared memory for what it hands to TMA: 32 rows of 64 columns, or of 32 of each of
// the three results of kDenseGateGrad (whose ring is a stage shorter for it).
template <int EPI>
struct PairSize {
  static constexpr int kResults = EPI == kDenseGateGrad ? 3 : 1;
  static constexpr int kCols = EPI == kDenseGateGrad ? 32 : 64;
  static constexpr int kWarpBytes = kResults * kCols * 2 * 32;
  static constexpr int kStages = EPI == kDenseGateGrad ? 5 : 6;
  static constexpr int kSmem = kStages * kPairStageBytes + kEpiWarps * kWarpBytes + 1024;  // (and 1.4 KiB of barriers and lists)
  static_assert(kSmem <= 225 * 1024 && BM * (kPairN + 4) * 4 <= kStages * kPairStageBytes, "");
};
constexpr int kBand = 8;

struct __align__(8) PairBars {
  uint64_t full[kPairStages];
  uint64_t empty[kPairStages];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t listed[2];    // the lists of a tile's adapters, and the MMA issuer done with them
  uint64_t unlisted[2];
  uint32_t tmem_base;
  int abort_flag;
};
struct PairArgs {
  int problems, first, tiles, split, b_early, a_early, next_early;  // tiles first .. tiles - 1
  int tile_end[kMaxDenseProblems];
  DeviceError* err;
};
struct NoAdapters {};
template <int NP>
struct Problems {
  DenseProblem p[NP];
};
struct PairResults {
  CUtensorMap out[3];  // of the problems, or dg, du, h
};

constexpr uint32_t kPairIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(kPairM >> 4) << 24);

__device__ __forceinline__ uint32_t at_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// The following run in a converged warp; one lane (always the same) issues the instruction.
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n\t}"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// The four MMAs of one k-block; `a_step`, `b_step`: descriptor distance of K = 16.
template <uint64_t A_STEP, uint64_t B_STEP>
__device__ __forceinline__ void mma_kblock(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred e, p, t;\n\t"
      ".reg .b64 a, b;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.eq.b32 t, 0, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "add.s64 a, %1, %5;\n\tadd.s64 b, %2, %6;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, t;\n\t"
      "add.s64 a, a, %5;\n\tadd.s64 b, b, %6;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, t;\n\t"
      "add.s64 a, a, %5;\n\tadd.s64 b, b, %6;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, t;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "n"(A_STEP), "n"(B_STEP)
      : "memory");
}
// (see tc_mma_bf16_lanes_one)
__device__ __forceinline__ void mma_lanes(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, int steps,
                                          const uint32_t (&off)[8]) {
  asm volatile(
      "{\n\t.reg .pred e, t, p;\n\t"
      ".reg .b64 a, b;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.eq.b32 t, 0, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%4, %5, %6, %7, %8, %9, %10, %11}, t;\n\t"
      "setp.gt.and.s32 p, %12, 1, e;\n\tadd.s64 a, %1, 2;\n\tadd.s64 b, %2, 2;\n\t"
      "@p tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, {%4, %5, %6, %7, %8, %9, %10, %11}, t;\n\t"
      "setp.gt.and.s32 p, %12, 2, e;\n\tadd.s64 a, %1, 4;\n\tadd.s64 b, %2, 4;\n\t"
      "@p tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, {%4, %5, %6, %7, %8, %9, %10, %11}, t;\n\t"
      "setp.gt.and.s32 p, %12, 3, e;\n\tadd.s64 a, %1, 6;\n\tadd.s64 b, %2, 6;\n\t"
      "@p tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, {%4, %5, %6, %7, %8, %9, %10, %11}, t;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(off[0]), "r"(off[1]), "r"(off[2]), "r"(off[3]), "r"(off[4]),
        "r"(off[5]), "r"(off[6]), "r"(off[7]), "r"(steps)
      : "memory");
}
__device__ __forceinline__ void commit_both(uint32_t bar, uint32_t lead) {
  const uint16_t mask = (uint16_t)(3u << lead);
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}"
      ::"r"(bar), "h"(mask)
      : "memory");
}

__device__ __forceinline__ void store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// 16 bytes of row `row` at 16-byte piece `c` of a box of rows of ROW_BYTES (64 or 128) under the swizzle of that width
template <int ROW_BYTES>
__device__ __forceinline__ void stage16(uint32_t box, int row, int c, const uint4& v) {
  const uint32_t at = box + row * ROW_BYTES + ((c ^ (ROW_BYTES == 128 ? row & 7 : (row >> 1) & 3)) << 4);
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

struct Tile {
  int which, m0, n0;
};
template <int EPI, int NP>
__device__ __forceinline__ Tile tile_of(const Problems<NP>& ps, const PairArgs& pa, int t) {
  Tile o;
  o.which = 0;
  if constexpr (NP > 1) {
    while (o.which + 1 < pa.problems && t >= pa.tile_end[o.which]) ++o.which;
    if (o.which > 0) t -= pa.tile_end[o.which - 1];
  }
  constexpr int N_OUT = EPI == kDenseSwiGLU ? kPairN / 2 : kPairN;
  const int m_tiles = (ps.p[o.which].M + kPairM - 1) / kPairM, n_tiles = (ps.p[o.which].N + N_OUT - 1) / N_OUT;
  const int band = t / (kBand * n_tiles), in_band = t - band * kBand * n_tiles;
  const int height = min(kBand, m_tiles - band * kBand);
  const int nt = in_band / height;
  o.m0 = (band * kBand + in_band - nt * height) * kPairM;
  o.n0 = nt * N_OUT;
  return o;
}

// The adapters of a tile come in rounds: one or two stages with the tile's reduced rows, then stages of B, as many adapters in each as
// fit, until the ring is full.
template <int EPI>
struct AdapterRounds : AdapterChunks<EPI> {
  static constexpr int kRows = EPI == kDenseSwiGLU ? 64 : 128;  // a CTA's half of the B rows of a chunk
  int v_bytes, v_slots, b_bytes, group, b_stages;
  __device__ __forceinline__ explicit AdapterRounds(const DenseAdapters& ad) : AdapterChunks<EPI>(ad) {
    v_bytes = BM * 2 * this->widest;
    v_slots = kPairStageBytes / v_bytes;
    b_bytes = kRows * 2 * this->widest;
    group = kPairStageBytes / (b_bytes * this->chunks);  // (four chunks of 64 columns are a stage)
    b_stages = kPairStages - (this->chunks > v_slots ? 2 : 1);
  }
};
// The adapters of two tiles, found by the producer between its loads (in ascending order; of a cut reduction every split-th)
struct PairLists {
  uint16_t adapter[2][kPairM];
  int count[2];
};

template <int EPI, bool B_MN, int NP, bool AD>
__global__ void __launch_bounds__(kPairThreads, 1)
dense_pair_kernel(const __grid_constant__ Problems<NP> ps, const __grid_constant__ PairArgs pa, const __grid_constant__ PairResults res,
                  const __grid_constant__ std::conditional_t<AD, DenseAdapters, NoAdapters> ad) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ PairBars bars;
  __shared__ std::conditional_t<AD, PairLists, NoAdapters> lists;
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  float* part = reinterpret_cast<float*>(smem_raw + (ring - smem_u32(smem_raw)));
  volatile int* abort_flag = &bars.abort_flag;
  const int warp = uniform_warp();
  const int lane = threadIdx.x & 31;
  const uint32_t in_cluster = cluster_rank();
  const uint32_t rank = in_cluster & 1, lead = in_cluster & ~1u;  // of the pair
  const bool leader = rank == 0;
  // split 1: a pair walks the tiles; else the `split` pairs of a cluster share one tile's reduction
  const int split = pa.split;
  const int pair = pa.first + (split > 1 ? (int)(blockIdx.x >> 1) / split : (int)(blockIdx.x >> 1));
  const int num_pairs = split > 1 ? pa.tiles : (int)(gridDim.x >> 1);
  const int piece = split > 1 ? (int)(in_cluster >> 1) : 0;
  constexpr int N_OUT = EPI == kDenseSwiGLU ? kPairN / 2 : kPairN;
  constexpr int kStages = PairSize<EPI>::kStages;
  constexpr bool A_MN = NP > 1;

  auto kb_begin = [&](const DenseProblem& p) { return (int)((int64_t)p.kb * piece / split); };
  auto kb_end = [&](const DenseProblem& p) { return (int)((int64_t)p.kb * (piece + 1) / split); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&bars.full[s]), 1);
      mbar_init(smem_u32(&bars.empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&bars.acc_full[b]), 1);
      mbar_init(smem_u32(&bars.acc_empty[b]), 2 * kEpiWarps);
      mbar_init(smem_u32(&bars.listed[b]), 1);
      mbar_init(smem_u32(&bars.unlisted[b]), 1);
    }
    bars.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_base)),
                 "r"(kPairTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_barrier();  // barriers of both CTAs are initialised before anyone signals them
  tc_fence_after();
  const uint32_t tmem = bars.tmem_base;

  if (warp == 0) {
    // ================= TMA producer (both CTAs) =================
    int stage = 0;
    uint32_t phase = 0, armed = 0;
    bool ok = true;
    auto load_b = [&](const DenseProblem& p, const Tile& t, int kb, uint32_t dst, uint32_t bar) {
      const int seg = EPI != kDenseSwiGLU && kb >= p.kb0;
      const int k = (kb - (seg ? p.kb0 : 0)) * BK;
      if constexpr (EPI == kDenseSwiGLU) {
        load_2d(dst, &p.b[rank], bar, k, t.n0);
        load_2d(dst + 8192, &p.b[rank], bar, k, t.n0 + 64);
      } else {
        const int n = t.n0 + (int)rank * 128;
        load_2d(dst, &p.b[seg], bar, B_MN ? n : k, B_MN ? k : n);
        load_2d(dst + 8192, &p.b[seg], bar, B_MN ? n + 64 : k, B_MN ? k : n + 64);
      }
    };
    auto load_a = [&](const DenseProblem& p, const Tile& t, int kb, uint32_t dst, uint32_t bar) {
      const int seg = EPI != kDenseSwiGLU && kb >= p.kb0;
      const int k = (kb - (seg ? p.kb0 : 0)) * BK;
      const int m = t.m0 + (int)rank * BM;
      load_2d(dst, &p.a[seg], bar, A_MN ? m : k, A_MN ? k : m);
      if constexpr (A_MN) load_2d(dst + 8192, &p.a[seg], bar, m + 64, k);
    };
    auto free_stage = [&]() {
      if (!mbar_wait(smem_u32(&bars.empty[stage]), phase ^ 1u, abort_flag)) {
        if (lane == 0) report_error(pa.err, ATENIA_ERR_DEVICE_TIMEOUT, 2700 + stage);
        *abort_flag = 1;
        ok = false;
      }
      ok = __all_sync(0xffffffffu, ok);
      return ok;
    };
    auto next_stage = [&]() {
      armed |= 1u << stage;
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1u;
      }
    };
    int ahead = 0;
    if (pa.b_early && pair < pa.tiles) {
      const Tile t = tile_of<EPI, NP>(ps, pa, pair);
      const DenseProblem& p = ps.p[NP > 1 ? t.which : 0];
      const int kb0 = kb_begin(p);
      ahead = min(kb_end(p) - kb0, kStages);
      for (int i = 0; i < ahead; ++i) {
        const uint32_t bar = at_rank(smem_u32(&bars.full[i]), lead), dst = ring + i * kPairStageBytes;
        if (leader) mbar_expect_tx_one(smem_u32(&bars.full[i]), 2 * kPairStageBytes);
        load_b(p, t, kb0 + i, dst + kOperandBytes, bar);
        if (pa.a_early) load_a(p, t, kb0 + i, dst, bar);
      }
    }
    if (!pa.a_early) {
      chain_wait();
      if (pa.next_early) chain_next();
    }
    const std::conditional_t<AD, AdapterRounds<EPI>, NoAdapters> r(ad);
    int it = 0;
    for (int i = pair; ok && i < pa.tiles; i += num_pairs, ++it) {
      const Tile t = tile_of<EPI, NP>(ps, pa, i);
      const DenseProblem& p = ps.p[NP > 1 ? t.which : 0];
      int32_t id[8], last = -1;
      int found = 0, index = 0;
      auto find_next = [&]() {
        if constexpr (AD) {
          last = next_adapter(id, last);
          if (last == kNoAdapter) return;
          if (index++ % split != piece) return;
          if (lane == 0) lists.adapter[it & 1][found] = (uint16_t)last;
          ++found;
        }
      };
      if constexpr (AD) {
        load_ids(id, ad.ids, t.m0, p.M - t.m0, ad.n, lane);
        // (the leader's issuer is done with the list of the tile before last; the other CTA's list is the producer's own)
        if (leader && !mbar_wait(smem_u32(&bars.unlisted[it & 1]), ((it >> 1) & 1) ^ 1u, abort_flag)) {
          if (lane == 0) report_error(pa.err, ATENIA_ERR_DEVICE_TIMEOUT, 2710 + (it & 1));
          *abort_flag = 1;
          ok = false;
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      for (int kb = kb_begin(p), end = kb_end(p); kb < end; ++kb) {
        const uint32_t full = smem_u32(&bars.full[stage]), bar = at_rank(full, lead), dst = ring + stage * kPairStageBytes;
        if (ahead > 0) {  // (the first tile's first blocks)
          --ahead;
          if (!pa.a_early) load_a(p, t, kb, dst, bar);
        } else {
          if (!free_stage()) break;
          if (leader) mbar_expect_tx_one(full, 2 * kPairStageBytes);
          load_b(p, t, kb, dst + kOperandBytes, bar);
          load_a(p, t, kb, dst, bar);
        }
        next_stage();
        if (AD && last != kNoAdapter && kb > kb_begin(p)) find_next();
      }
      if constexpr (AD) {
        while (ok && last != kNoAdapter) find_next();
        __syncwarp();
        if (leader && lane == 0) {
          lists.count[it & 1] = found;
          mbar_arrive(smem_u32(&bars.listed[it & 1]));
        }
        chain_wait();  // v is the kernel before's
        for (int done = 0; ok && done < found * ad.parts;) {
          const int of = done < found ? 0 : 1, to = (of + 1) * found;  // (which part of the reduced rows, for all adapters)
          // the tile's reduced rows, for the stages of B that follow
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (half * r.v_slots >= r.chunks || !ok) break;
            if (!free_stage()) break;
            const uint32_t full = smem_u32(&bars.full[stage]), bar = at_rank(full, lead), dst = ring + stage * kPairStageBytes;
            int columns = 0;
#pragma unroll
            for (int c = 0; c < kMaxChunks; ++c)
              if (c < r.chunks && c >= half * r.v_slots && c < (half + 1) * r.v_slots) columns += r.width[c];
            if (leader) mbar_expect_tx_one(full, 2 * columns * BM * 2);
#pragma unroll
            for (int c = 0; c < kMaxChunks; ++c)
              if (c < r.chunks && c >= half * r.v_slots && c < (half + 1) * r.v_slots)
                load_3d(dst + (c - half * r.v_slots) * r.v_bytes, &ad.seg[r.second[c]].v, bar, r.column[c], t.m0 + (int)rank * BM, of);
            next_stage();
          }
          for (int b = 0; ok && b < r.b_stages && done < to; ++b) {
            if (!free_stage()) break;
            const int here = min(to - done, r.group);
            const uint32_t full = smem_u32(&bars.full[stage]), bar = at_rank(full, lead);
            uint32_t dst = ring + stage * kPairStageBytes;
            if (leader) mbar_expect_tx_one(full, 2 * here * r.columns * r.kRows * 2);
            const int n = t.n0 + (int)rank * (N_OUT / 2);
            for (int q = 0; q < here; ++q) {
              const int a = lists.adapter[it & 1][done - of * found + q];
#pragma unroll
              for (int c = 0; c < kMaxChunks; ++c) {
                if (c >= r.chunks) break;
                const CUtensorMap* map = &ad.seg[r.second[c]].b;
                load_3d(dst, map, bar, r.column[c], n, a);
                if constexpr (EPI != kDenseSwiGLU) load_3d(dst + 128 * r.width[c], map, bar, r.column[c], n + 64, a);
                dst += r.b_bytes;
              }
            }
            done += here;
            next_stage();
          }
        }
      }
    }
    chain_wait();
    chain_next();  // (every load is on its way: what follows may be launched)
    if (*abort_flag && leader && lane == 0) {
      // let the copies already issued (both CTAs') land before the pair's shared memory is released
      for (int s = 0; s < kStages; ++s) {
        if (!(armed & (1u << s))) continue;
        const uint32_t par = s < stage ? phase : phase ^ 1u;
        for (int i = 0; i < (1 << 16) && !mbar_try_wait(smem_u32(&bars.full[s]), par); ++i) {}
      }
    }
  } else if (warp == 1) {
    // ================= MMA issuer (leader CTA only) =================
    if (leader) {
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;
      bool ok = true;
      const std::conditional_t<AD, AdapterRounds<EPI>, NoAdapters> r(ad);
      auto filled = [&]() {
        if (!mbar_wait(smem_u32(&bars.full[stage]), phase, abort_flag)) {
          if (lane == 0) report_error(pa.err, ATENIA_ERR_DEVICE_TIMEOUT, 2800 + stage);
          *abort_flag = 1;
          ok = false;
        }
        ok = __all_sync(0xffffffffu, ok);
        if (ok) tc_fence_after();
        return ok;
      };
      auto step_stage = [&]() {
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      };
      auto used = [&]() {
        commit_both(smem_u32(&bars.empty[stage]), lead);
        step_stage();
      };
      constexpr uint32_t idesc = kPairIdesc | (uint32_t(A_MN) << 15) | (uint32_t(B_MN) << 16) | (uint32_t(kPairN >> 3) << 17);
      for (int i = pair; ok && i < pa.tiles; i += num_pairs, ++it) {
        const Tile t = tile_of<EPI, NP>(ps, pa, i);
        const DenseProblem& p = ps.p[NP > 1 ? t.which : 0];
        int32_t id[8];
        if constexpr (AD) load_ids(id, ad.ids, t.m0, p.M - t.m0, ad.n, lane);
        const int acc = it & 1;
        if (!mbar_wait(smem_u32(&bars.acc_empty[acc]), ((it >> 1) & 1) ^ 1u, abort_flag)) {
          if (lane == 0) report_error(pa.err, ATENIA_ERR_DEVICE_TIMEOUT, 2900 + acc);
          *abort_flag = 1;
          ok = false;
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * kPairN;
        const int begin = kb_begin(p), end = kb_end(p);
        for (int kb = begin; kb < end; ++kb) {
          if (!filled()) break;
          const uint32_t sa = ring + stage * kPairStageBytes;
          mma_kblock<kOperandStep<A_MN>, kOperandStep<B_MN>>(d, operand_desc<A_MN>(sa), operand_desc<B_MN>(sa + kOperandBytes), idesc,
                                                             kb > begin ? 1u : 0u);
          used();
        }
        if constexpr (AD) {
          if (ok && !mbar_wait(smem_u32(&bars.listed[it & 1]), (it >> 1) & 1, abort_flag)) {
            if (lane == 0) report_error(pa.err, ATENIA_ERR_DEVICE_TIMEOUT, 2910 + (it & 1));
            *abort_flag = 1;
            ok = false;
          }
          ok = __all_sync(0xffffffffu, ok);
          const int found = ok ? lists.count[it & 1] : 0;
          for (int done = 0; ok && done < found * ad.parts;) {
            const int of = done < found ? 0 : 1, to = (of + 1) * found;
            const int v_stage = stage, v_next = stage + 1 == kStages ? 0 : stage + 1;
            const bool two = r.chunks > r.v_slots;
            if (!filled()) break;
            step_stage();  // (given back behind the MMAs that read it)
            if (two) {
              if (!filled()) break;
              step_stage();
            }
            uint64_t dv[kMaxChunks];
#pragma unroll
            for (int c = 0; c < kMaxChunks; ++c) {
              const bool over = c >= r.v_slots;
              dv[c] = make_smem_desc_width(ring + (over ? v_next : v_stage) * kPairStageBytes + (over ? c - r.v_slots : c) * r.v_bytes, r.width[c]);
            }
            for (int b = 0; ok && b < r.b_stages && done < to; ++b) {
              if (!filled()) break;
              const int here = min(to - done, r.group);
              uint32_t at = ring + stage * kPairStageBytes;
              for (int q = 0; q < here; ++q) {
                uint32_t off[8];
                lanes_off(off, id, (int32_t)lists.adapter[it & 1][done - of * found + q]);
#pragma unroll
                for (int c = 0; c < kMaxChunks; ++c) {
                  if (c >= r.chunks) break;
                  constexpr uint32_t idesc_ad = kPairIdesc | (uint32_t(N_OUT >> 3) << 17);
                  const uint64_t db = make_smem_desc_width(at, r.width[c]);
                  mma_lanes(d + (r.second[c] ? N_OUT : 0), dv[c], db, idesc_ad, r.steps[c], off);
                  at += r.b_bytes;
                }
              }
              done += here;
              used();
            }
            if (!ok) break;
            commit_both(smem_u32(&bars.empty[v_stage]), lead);
            if (two) commit_both(smem_u32(&bars.empty[v_next]), lead);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bars.unlisted[it & 1]));
        }
        if (ok) commit_both(smem_u32(&bars.acc_full[acc]), lead);
      }
    }
  } else {
    // ================= epilogue (warps 2..9 of both CTAs) =================
    chain_wait();
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const int row_in = (int)rank * BM + quarter * 32 + lane;
    const uint32_t box = ring + kStages * kPairStageBytes + (warp - 2) * PairSize<EPI>::kWarpBytes;
    int it = 0;
    for (int i = pair; i < pa.tiles; i += num_pairs, ++it) {
      const Tile t = tile_of<EPI, NP>(ps, pa, i);
      const DenseProblem& p = ps.p[NP > 1 ? t.which : 0];
      const int acc = it & 1;
      const int row = t.m0 + row_in;
      const int n = t.n0 + half * (N_OUT / 2);
      const int cols = min(N_OUT / 2, p.N - n);
      Saved<EPI, 16> kept, next;
      if (split == 1) kept.load(p, row, n, row < p.M && cols > 0);
      const bool ready = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.acc_full[acc]), (it >> 1) & 1, abort_flag));
      if (!ready) {
        if (lane == 0) report_error(pa.err, ATENIA_ERR_DEVICE_TIMEOUT, 3000 + acc);
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const uint32_t taddr = tmem + (uint32_t(quarter * 32) << 16) + acc * kPairN + half * (N_OUT / 2);
      if (split > 1) {  // (one tile: the sums go to the ring, which nothing uses any more)
        float* mine = part + (quarter * 32 + lane) * kSumsPitch<kPairN> + half * 128;
        const uint32_t from = tmem + (uint32_t(quarter * 32) << 16) + half * 128;
#pragma unroll 2
        for (int c = 0; c < 128; c += 16) {
          uint32_t v[16];
          tc_ld16(from + c, v);
          tc_ld_wait();
#pragma unroll
          for (int j = 0; j < 4; ++j)
            reinterpret_cast<uint4*>(mine + c)[j] = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
        break;
      }
      constexpr int kCols = PairSize<EPI>::kCols, kResults = PairSize<EPI>::kResults;
      const bool any = t.m0 + (int)rank * BM + quarter * 32 < p.M;
#pragma unroll 1
      for (int c0 = 0; c0 < cols; c0 += kCols) {
        if (lane == 0) store_wait_read();  // (the piece's last store)
        __syncwarp();
#pragma unroll
        for (int c = 0; c < kCols; c += 16) {
          next.load(p, row, n + c0 + c + 16, row < p.M && c0 + c + 16 < cols);
          uint32_t v[16], v1[16];
          tc_ld16(taddr + c0 + c, v);
          if constexpr (EPI == kDenseSwiGLU) tc_ld16(taddr + N_OUT + c0 + c, v1);
          tc_ld_wait();
          float f[16], f1[16], o[16], du[16], h[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            f[j] = __uint_as_float(v[j]);
            f1[j] = EPI == kDenseSwiGLU ? __uint_as_float(v1[j]) : 0.f;
          }
          dense_values<EPI, 16>(p, row, n + c0 + c, row < p.M && c0 + c < cols, f, f1, kept, o, du, h);
          kept = next;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            stage16<kCols * 2>(box, lane, c / 8 + q, pack8(o + 8 * q));
            if constexpr (EPI == kDenseGateGrad) {
              stage16<kCols * 2>(box + kCols * 64, lane, c / 8 + q, pack8(du + 8 * q));
              stage16<kCols * 2>(box + 2 * kCols * 64, lane, c / 8 + q, pack8(h + 8 * q));
            }
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0 && any) {
#pragma unroll
          for (int r = 0; r < kResults; ++r)
            store_2d(&res.out[kResults > 1 ? r : t.which], box + r * kCols * 64, n + c0, row - lane);
          store_commit();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_remote(at_rank(smem_u32(&bars.acc_empty[acc]), lead));
    }
    if (lane == 0) store_wait();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (split > 1) {
    cluster_barrier();
    if (!*abort_flag) {
      const Tile t = tile_of<EPI, NP>(ps, pa, pair);
      const DenseProblem& p = ps.p[NP > 1 ? t.which : 0];
      const int m0 = t.m0 + (int)rank * BM;
      const int rows = max(0, min(BM, p.M - m0)), cols = min(N_OUT, p.N - t.n0);
      if (split == 2) add_parts<EPI, kPairN, 2, 2>(p, m0, t.n0, rows, cols, smem_u32(part), piece, rank);
      else if (split == 3) add_parts<EPI, kPairN, 3, 2>(p, m0, t.n0, rows, cols, smem_u32(part), piece, rank);
      else add_parts<EPI, kPairN, 4, 2>(p, m0, t.n0, rows, cols, smem_u32(part), piece, rank);
    }
    __syncthreads();
  }
  cluster_barrier();  // no CTA leaves while its peers may still signal or read it
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kPairTmemCols) : "memory");
  }
}

template <int EPI, bool B_MN, int NP, bool AD>
int launch_pairs(const DenseGemm& g, PairArgs pa, int num_sms, cudaStream_t s) {
  auto kernel = dense_pair_kernel<EPI, B_MN, NP, AD>;
  static FirstUse ready[kMaxDevices];
  if (const int rc = allow_shared_memory(ready, kernel, PairSize<EPI>::kSmem)) return rc;
  Problems<NP> ps;
  for (int i = 0; i < NP; ++i) ps.p[i] = g.p[i];
  std::conditional_t<AD, DenseAdapters, NoAdapters> ad{};
  if constexpr (AD) ad = *g.adapters;
  const int tiles = pa.tiles - pa.first;
  const int pairs = pa.split > 1 ? tiles * pa.split : num_sms / 2 < tiles ? num_sms / 2 : tiles;
  pa.next_early = g.next_early && 2 * pairs < num_sms;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2 * pa.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * pairs);
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = PairSize<EPI>::kSmem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = g.chained ? 2 : 1;
  PairResults res{};
  auto map = [](CUtensorMap* m, const __nv_bfloat16* out, const DenseProblem& p) {
    constexpr uint32_t cols = PairSize<EPI>::kCols;
    return encode_tmap_bf16(m, out, {(uint64_t)p.N, (uint64_t)p.M, 0}, {cols, 32, 1}, 2 * cols);
  };
  int rc = ATENIA_OK;
  for (int i = 0; i < NP && !rc; ++i) rc = map(&res.out[i], g.p[i].out, g.p[i]);
  if (EPI == kDenseGateGrad && !rc) rc = map(&res.out[1], g.p[0].out_du, g.p[0]);
  if (EPI == kDenseGateGrad && !rc) rc = map(&res.out[2], g.p[0].out_h, g.p[0]);
  if (rc) return rc;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, ps, pa, res, ad);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return (int)e;
}

int launch_range(const DenseGemm& g, const PairArgs& pa, int num_sms, cudaStream_t s) {
  count_launch();
  count_tcgen05_launch();
  const bool ad = g.adapters != nullptr;
  const bool b_mn = g.p[0].b_mn;
  if (g.problems > 1)
    return g.epilogue == kDensePlain && b_mn && !ad ? launch_pairs<kDensePlain, true, kMaxDenseProblems, false>(g, pa, num_sms, s) : ATENIA_ERR_UNSUPPORTED;
  if (ad && b_mn) return ATENIA_ERR_UNSUPPORTED;
  if (g.epilogue == kDenseSwiGLU && !b_mn)
    return ad ? launch_pairs<kDenseSwiGLU, false, 1, true>(g, pa, num_sms, s) : launch_pairs<kDenseSwiGLU, false, 1, false>(g, pa, num_sms, s);
  if (g.epilogue == kDensePlain)
    return ad     ? launch_pairs<kDensePlain, false, 1, true>(g, pa, num_sms, s)
           : b_mn ? launch_pairs<kDensePlain, true, 1, false>(g, pa, num_sms, s)
                  : launch_pairs<kDensePlain, false, 1, false>(g, pa, num_sms, s);
  if (g.epilogue == kDenseGateGrad && b_mn && !ad) return launch_pairs<kDenseGateGrad, true, 1, false>(g, pa, num_sms, s);
  return ATENIA_ERR_UNSUPPORTED;
}

}  // namespace

int launch_dense_pairs(const DenseGemm& g, int split, int tail_split, int num_sms, cudaStream_t s) {
  if (split < 1 || split > 4 || tail_split < 1 || tail_split > 4) return ATENIA_ERR_SHAPE;
  PairArgs pa{};
  int rc = dense_error_word(&pa.err);
  if (rc) return rc;
  const int n_out = g.epilogue == kDenseSwiGLU ? kPairN / 2 : kPairN;
  int64_t tiles = 0;
  for (int i = 0; i < g.problems; ++i) {
    const DenseProblem& p = g.p[i];
    tiles += (int64_t)((p.M + kPairM - 1) / kPairM) * ((p.N + n_out - 1) / n_out);
    if (tiles * split > kDenseMostTiles || p.kb < split || p.kb < tail_split) return ATENIA_ERR_SHAPE;
    pa.tile_end[i] = (int)tiles;
  }
  if (tiles == 0) return ATENIA_OK;
  if (g.a_rows != BM) return ATENIA_ERR_SHAPE;
  pa.problems = g.problems;
  pa.tiles = (int)tiles;
  pa.split = split;
  pa.b_early = g.b_early;
  pa.a_early = g.a_early && g.b_early;
  const int waves = (int)tiles / (num_sms / 2);
  if (split > 1 || tail_split == 1 || waves == 0 || waves * (num_sms / 2) == tiles) return launch_range(g, pa, num_sms, s);
  // the tiles of whole waves, then the rest with their reductions cut.  The second launch's operands are the first's, so they were there
  // when the first let it start; its epilogues wait for the first, so what comes behind it waits for both.
  pa.tiles = waves * (num_sms / 2);
  if ((rc = launch_range(g, pa, num_sms, s))) return rc;
  DenseGemm tail = g;
  tail.chained = true;
  pa.first = pa.tiles;
  pa.tiles = (int)tiles;
  pa.split = tail_split;
  pa.b_early = pa.a_early = true;
  return launch_range(tail, pa, num_sms, s);
}

}  // namespace atenia
