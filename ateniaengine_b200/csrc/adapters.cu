// First half of the low-rank adapters: v[t, :] = scale[a] * (A_a x[t, :]) with a = ids[t], in one or two bf16 parts (adapter_parts; the
// second product's operand; the sums, over CTAs too, are f32).
//
// A tile is 128 token rows; its distinct adapters, in the order of their first rows, are taken up to 128 rank rows at a time (of gate
// and up together where they fit) as the N side of one MMA, and a row keeps the columns of its own adapter.  Rows of other adapters are
// computed and dropped: each A is read once a tile, and a tensor core has the products to spare (128 rows, rank 16 of 4096 inputs: 2 GFLOP
// for 128 adapters instead of 17 MFLOP).  CTAs side by side take passes of adapters, and a cluster of up to 8 cuts the reduction and adds in
// rank order (reduce_plan).  What bounds it is latency: of 6.3 us inside the kernel (1100 rows, rank 64 of 2048 inputs, a pass, four
// k-blocks a CTA) the list of adapters takes 1.0, the first load 0.8, the MMAs behind the loads 0.9, the two barriers of the cluster
// 1.0 each and the sums 0.7.
#include "dense_choice.cuh"
#include "dense_gemm.cuh"

namespace atenia {
namespace {
using namespace tc;

constexpr int kRankRows = 128;      // rank rows of a tile at most
constexpr int kRedStages = 6;       // at most
constexpr int kRedThreads = 192;
constexpr int kRedTmemCols = 128;
constexpr int kRedRingBytes = 100 * 1024;
constexpr int kRedPitch = kAdapterMaxRank + 4;  // floats (see kSumsPitch)
constexpr int kRedPartBytes = BM * kRedPitch * 4;  // f32 sums [row][rank row]
static_assert(kRedPartBytes <= kRedRingBytes, "");

struct __align__(8) RedBars {
  uint64_t full[kRedStages];
  uint64_t empty[kRedStages];
  uint64_t acc_full;
  uint32_t tmem_base;
  int abort_flag;
};

// What a CTA works on: the rank rows of one projection, or those of both side by side
struct RedPart {
  int first, count, rank0, cols;  // projections first .. first + count - 1; rank rows of the first and of all
};

// This rank's share of the tile's sums, four rank rows a thread, added in rank order.  The threads of all ranks take neighbouring pieces,
// since a pass's rows, those of one or two adapters, are neighbours more often than not.
template <int S>
__device__ __forceinline__ void add_rows(const AdapterReduce& ar, const RedPart& rp, int m0, int rows, uint32_t part,
                                         const float (*scales)[BM], const int16_t* slot, int begin_slot, int end_slot, int rank) {
  const int quads = rp.cols / 4, total = rows * quads;
  for (int i = rank * kRedThreads + (int)threadIdx.x; i < total; i += S * kRedThreads) {
    const int t = i / quads, j = 4 * (i - t * quads);
    if (slot[t] < begin_slot || slot[t] >= end_slot) continue;
    const AdapterReduce::Projection& p = ar.p[rp.first + (j >= rp.rank0)];
    const int at = j >= rp.rank0 ? j - rp.rank0 : j;
    const float scale = scales[j >= rp.rank0][t];
    float4 v[S];
#pragma unroll
    for (int q = 0; q < S; ++q) v[q] = ld_cluster_f32x4(part + (t * kRedPitch + j) * 4, q);
    float4 sum = v[0];
#pragma unroll
    for (int q = 1; q < S; ++q) sum.x += v[q].x, sum.y += v[q].y, sum.z += v[q].z, sum.w += v[q].w;
    sum.x *= scale, sum.y *= scale, sum.z *= scale, sum.w *= scale;
    __nv_bfloat16* to = p.v + (int64_t)(m0 + t) * p.rank + at;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(sum.x, sum.y), pack_bf16x2(sum.z, sum.w));
    if (ar.parts > 1)
      *reinterpret_cast<uint2*>(to + (int64_t)ar.M * p.rank) = make_uint2(pack_bf16x2(left_of_bf16(sum.x), left_of_bf16(sum.y)),
                                                                          pack_bf16x2(left_of_bf16(sum.z), left_of_bf16(sum.w)));
  }
}

__global__ void __launch_bounds__(kRedThreads)
adapter_reduce_kernel(const __grid_constant__ AdapterReduce ar, int split, int lanes, int together, int stages, DeviceError* err) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ RedBars bars;
  __shared__ TileList list;
  __shared__ int16_t slot[BM];  // of a row's adapter in the list, -1 where it has none
  __shared__ float scales[2][BM];  // ... and its scales
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  float* part = reinterpret_cast<float*>(smem_raw + (ring - smem_u32(smem_raw)));
  volatile int* abort_flag = &bars.abort_flag;
  const int warp = uniform_warp();
  const int lane = threadIdx.x & 31;
  const int rank = split > 1 ? (int)cluster_rank() : 0;
  const int m_tiles = (ar.M + BM - 1) / BM;
  int unit = blockIdx.x / split;
  const int first_pass = unit % lanes;
  unit /= lanes;
  const int m0 = (unit % m_tiles) * BM;
  const int rows = min(BM, ar.M - m0);
  RedPart rp;
  rp.first = together ? 0 : unit / m_tiles;
  rp.count = together ? ar.projections : 1;
  rp.rank0 = ar.p[rp.first].rank;
  rp.cols = rp.count > 1 ? rp.rank0 + ar.p[1].rank : rp.rank0;
  const int per_pass = kRankRows / rp.cols;

  const int kb_begin = (int)((int64_t)ar.kb * rank / split), kb_end = (int)((int64_t)ar.kb * (rank + 1) / split);
  const int a_bytes = ar.a_rows * BK * 2;
  const int stage_bytes = a_bytes + kRankRows * BK * 2;
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
                 "r"(kRedTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  chain_wait();
  chain_next();  // what follows reads nothing of this kernel's before its own wait
  if (warp >= 2) {
    const int w = warp - 2, r = 32 * w + lane;
    list_adapters(list, ar.ids, m0, rows, ar.n, w, lane);
    asm volatile("bar.sync 1, 128;" ::: "memory");
    int at = -1;
    const int32_t mine = list.id[r];
    if (mine != kNoAdapter)
      for (int i = 0; i < list.count; ++i) at = list.adapter[i] == mine ? i : at;
    slot[r] = (int16_t)at;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem_base;
  const int count = list.count;

  int stage = 0;
  uint32_t phase = 0, armed = 0, acc_phase = 0;
  bool ok = true;
  for (int pass = first_pass; pass * per_pass < count; pass += lanes) {  // (alike in all CTAs of the cluster)
    const int begin = pass * per_pass, here = min(per_pass, count - begin);
    if (warp == 0) {
      fence_proxy_async();  // (the ring held the last pass's sums)
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        if (!mbar_wait(smem_u32(&bars.empty[stage]), phase ^ 1u, abort_flag)) {
          if (lane == 0) report_error(err, ATENIA_ERR_DEVICE_TIMEOUT, 2400 + stage);
          *abort_flag = 1;
          ok = false;
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t bar = smem_u32(&bars.full[stage]), dst = ring + stage * stage_bytes;
        mbar_expect_tx_one(bar, a_bytes + here * rp.cols * BK * 2);
        tma_load_2d_one(dst, &ar.x, bar, kb * BK, m0);
        for (int i = 0; i < here; ++i) {
          const uint32_t to = dst + a_bytes + i * rp.cols * BK * 2;
          tma_load_3d_one(to, &ar.p[rp.first].a, bar, kb * BK, 0, list.adapter[begin + i]);
          if (rp.count > 1) tma_load_3d_one(to + rp.rank0 * BK * 2, &ar.p[1].a, bar, kb * BK, 0, list.adapter[begin + i]);
        }
        armed |= 1u << stage;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (*abort_flag && lane == 0) {
        for (int s = 0; s < stages; ++s) {
          if (!(armed & (1u << s))) continue;
          const uint32_t par = s < stage ? phase : phase ^ 1u;
          for (int i = 0; i < (1 << 16) && !mbar_try_wait(smem_u32(&bars.full[s]), par); ++i) {}
        }
      }
    } else if (warp == 1) {
      const int n_mma = (here * rp.cols + 15) / 16 * 16;
      const uint32_t idesc =
          (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(128 >> 4) << 24) | (uint32_t(n_mma >> 3) << 17);
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        if (!mbar_wait(smem_u32(&bars.full[stage]), phase, abort_flag)) {
          if (lane == 0) report_error(err, ATENIA_ERR_DEVICE_TIMEOUT, 2500 + stage);
          *abort_flag = 1;
          ok = false;
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t sa = ring + stage * stage_bytes;
        const uint64_t da = make_smem_desc(sa), db = make_smem_desc(sa + a_bytes);
#pragma unroll
        for (int k = 0; k < BK / UMMA_K; ++k) tc_mma_bf16_one(tmem, da + 2 * k, db + 2 * k, idesc, kb > kb_begin || k > 0);
        tc_commit_one(smem_u32(&bars.empty[stage]));
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) tc_commit_one(smem_u32(&bars.acc_full));
    } else {
      const int quarter = warp & 3;
      const int row = quarter * 32 + lane;
      if (pass == first_pass && slot[row] >= 0)  // (behind the pass's loads; what follows waits for them)
        for (int i = 0; i < rp.count; ++i) scales[i][row] = ar.p[rp.first + i].scale[list.id[row]];
      const bool ready = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.acc_full), acc_phase, abort_flag));
      if (!ready) {
        if (lane == 0) report_error(err, ATENIA_ERR_DEVICE_TIMEOUT, 2600);
        *abort_flag = 1;
      } else if (quarter * 32 < rows) {
        tc_fence_after();
        const uint32_t taddr = tmem + (uint32_t(quarter * 32) << 16);
        const int mine = slot[row] - begin;
        for (int i = 0; i < here; ++i) {
          if (!__any_sync(0xffffffffu, mine == i)) continue;
#pragma unroll 1
          for (int j = 0; j < rp.cols; j += 32) {
            uint32_t v[4][8];
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (j + 8 * q < rp.cols) tc_ld8(taddr + i * rp.cols + j + 8 * q, v[q]);
            tc_ld_wait();
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (mine == i && j + 8 * q < rp.cols) {
                uint4* dst = reinterpret_cast<uint4*>(part + row * kRedPitch + j + 8 * q);
                dst[0] = make_uint4(v[q][0], v[q][1], v[q][2], v[q][3]);
                dst[1] = make_uint4(v[q][4], v[q][5], v[q][6], v[q][7]);
              }
          }
        }
        tc_fence_before();
      }
    }
    acc_phase ^= 1u;
    __syncthreads();
    if (split > 1) cluster_barrier();
    if (!*abort_flag) {
      const uint32_t sums = smem_u32(part);
      if (split == 1) add_rows<1>(ar, rp, m0, rows, sums, scales, slot, begin, begin + here, rank);
      else if (split == 2) add_rows<2>(ar, rp, m0, rows, sums, scales, slot, begin, begin + here, rank);
      else if (split == 4) add_rows<4>(ar, rp, m0, rows, sums, scales, slot, begin, begin + here, rank);
      else add_rows<8>(ar, rp, m0, rows, sums, scales, slot, begin, begin + here, rank);
    }
    __syncthreads();
    if (split > 1) cluster_barrier();  // no CTA goes on, or leaves, while another reads its sums
    tc_fence_after();
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kRedTmemCols) : "memory");
  }
}

}  // namespace

int launch_adapter_reduce(const AdapterReduce& r, int num_sms, cudaStream_t s) {
  const int m_tiles = (r.M + BM - 1) / BM;
  if (m_tiles == 0 || r.projections == 0) return ATENIA_OK;
  if (r.few) return launch_adapter_gemv(r, s);
  DeviceError* err = nullptr;
  int rc = dense_error_word(&err);
  if (rc) return rc;
  const bool together = r.projections > 1 && r.p[0].rank + r.p[1].rank <= kRankRows;
  int widest = 0;
  for (int i = 0; i < r.projections; ++i) widest = together ? widest + r.p[i].rank : (r.p[i].rank > widest ? r.p[i].rank : widest);
  const int64_t tiles = (int64_t)m_tiles * (together ? 1 : r.projections);
  if (tiles > (1 << 24)) return ATENIA_ERR_SHAPE;
  const ReducePlan plan = reduce_plan(r.M, tiles, r.kb, r.n, kRankRows / widest, num_sms);
  const int split = plan.split, lanes = plan.lanes;
  const int64_t units = tiles * lanes;
  const int stage_bytes = r.a_rows * BK * 2 + kRankRows * BK * 2;
  int stages = kRedRingBytes / stage_bytes;
  if (stages > kRedStages) stages = kRedStages;
  static FirstUse ready[kMaxDevices];
  if (const int rc = allow_shared_memory(ready, adapter_reduce_kernel, kRedRingBytes + 1024)) return rc;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(units * split));
  cfg.blockDim = dim3(kRedThreads);
  cfg.dynamicSmemBytes = kRedRingBytes + 1024;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = r.chained ? 2 : 1;
  count_launch();
  count_tcgen05_launch();
  const cudaError_t e = cudaLaunchKernelEx(&cfg, adapter_reduce_kernel, r, split, lanes, (int)together, stages, err);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return (int)e;
}

}  // namespace atenia
