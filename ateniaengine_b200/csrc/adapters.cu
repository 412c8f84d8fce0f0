// First half of the low-rank adapters: v[t, :] = scale[a] * (A_a x[t, :]) with a = ids[t], rounded to bf16 (the second product's
// operand; the sums, over CTAs too, are f32).
//
// A tile is 128 token rows; its distinct adapters, in ascending order of their ids, are taken up to 128 rank rows at a time as the
// N side of one MMA, and a row keeps the columns of its own adapter.  Rows of other adapters are computed and dropped: a
// decode batch in which every row has its own adapter reads each A once, which is what bounds it, and a tensor core has the
// products to spare (64 rows, rank 16: 1 GFLOP instead of 8 MFLOP per 4096 inputs).  A cluster of up to 8 CTAs cuts the reduction
// and adds in rank order.
#include "dense_gemm.cuh"

namespace atenia {
namespace {
using namespace tc;

constexpr int kRankRows = 128;      // rank rows of a tile at most
constexpr int kMaxList = kRankRows / 8;
constexpr int kRedStages = 6;       // at most
constexpr int kRedThreads = 192;
constexpr int kRedTmemCols = 128;
constexpr int kRedRingBytes = 100 * 1024;
constexpr int kRedPitch = kAdapterMaxRank + 4;  // floats (see kPartPitch)
constexpr int kRedPartBytes = BM * kRedPitch * 4;  // f32 sums [row][rank row]
static_assert(kRedPartBytes <= kRedRingBytes, "");

struct __align__(8) RedBars {
  uint64_t full[kRedStages];
  uint64_t empty[kRedStages];
  uint64_t acc_full;
  uint32_t tmem_base;
  int abort_flag;
};

// This rank's share of the tile's sums, four rank rows a thread, added in rank order.
template <int S>
__device__ __forceinline__ void add_rows(const AdapterReduce& ar, int proj, int m0, int rows, uint32_t part, const int32_t* row_id,
                                         int rank) {
  const int r = ar.p[proj].rank, quads = r / 4, total = rows * quads;
  const int begin = total * rank / S, end = total * (rank + 1) / S;
  for (int i = begin + (int)threadIdx.x; i < end; i += kRedThreads) {
    const int t = i / quads, j = 4 * (i - t * quads);
    const int32_t a = row_id[t];
    if (a == kNoAdapter) continue;
    const float scale = ar.p[proj].scale[a];
    float4 v[S];
#pragma unroll
    for (int q = 0; q < S; ++q) v[q] = ld_cluster_f32x4(part + (t * kRedPitch + j) * 4, q);
    float4 sum = v[0];
#pragma unroll
    for (int q = 1; q < S; ++q) sum.x += v[q].x, sum.y += v[q].y, sum.z += v[q].z, sum.w += v[q].w;
    *reinterpret_cast<uint2*>(ar.p[proj].v + (int64_t)(m0 + t) * r + j) =
        make_uint2(pack_bf16x2(sum.x * scale, sum.y * scale), pack_bf16x2(sum.z * scale, sum.w * scale));
  }
}

__global__ void __launch_bounds__(kRedThreads)
adapter_reduce_kernel(const __grid_constant__ AdapterReduce ar, int split, int passes, int stages, DeviceError* err) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ RedBars bars;
  __shared__ int32_t list[kMaxList];
  __shared__ int32_t row_id[BM];  // the row's adapter where this pass has it, else kNoAdapter
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  float* part = reinterpret_cast<float*>(smem_raw + (ring - smem_u32(smem_raw)));
  volatile int* abort_flag = &bars.abort_flag;
  const int warp = uniform_warp();
  const int lane = threadIdx.x & 31;
  const int rank = split > 1 ? (int)cluster_rank() : 0;
  const int m_tiles = (ar.M + BM - 1) / BM;
  int unit = blockIdx.x / split;
  const int pass = unit % passes;
  unit /= passes;
  const int m0 = (unit % m_tiles) * BM;
  const int proj = unit / m_tiles;
  const int r = ar.p[proj].rank;
  const int rows = min(BM, ar.M - m0);
  const int per_pass = kRankRows / r;

  // (the ids are the caller's)
  chain_wait();
  chain_next();  // what follows reads nothing of this kernel's before its own wait
  int32_t id[4];
  load_ids(id, ar.ids, m0, rows, ar.n, lane);
  int count = 0, first = kNoAdapter, last = kNoAdapter;
  {
    int32_t a = -1;
    for (int i = 0; i < (pass + 1) * per_pass && (a = next_adapter(id, a)) != kNoAdapter; ++i) {
      if (i < pass * per_pass) continue;
      if (count == 0) first = a;
      last = a;
      if (threadIdx.x == 0) list[count] = a;
      ++count;
    }
  }
  if (count == 0) return;  // (the whole cluster: it shares tile and pass)

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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem_base;

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0, armed = 0;
    bool ok = true;
    for (int kb = kb_begin; kb < kb_end; ++kb) {
      if (!mbar_wait(smem_u32(&bars.empty[stage]), phase ^ 1u, abort_flag)) {
        if (lane == 0) report_error(err, ATENIA_ERR_DEVICE_TIMEOUT, 2400 + stage);
        *abort_flag = 1;
        ok = false;
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint32_t bar = smem_u32(&bars.full[stage]), dst = ring + stage * stage_bytes;
      mbar_expect_tx_one(bar, a_bytes + count * r * BK * 2);
      tma_load_2d_one(dst, &ar.x, bar, kb * BK, m0);
      for (int i = 0; i < count; ++i)
        tma_load_3d_one(dst + a_bytes + i * r * BK * 2, &ar.p[proj].a, bar, kb * BK, 0, list[i]);
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
    const int n_mma = (count * r + 15) / 16 * 16;
    const uint32_t idesc =
        (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(128 >> 4) << 24) | (uint32_t(n_mma >> 3) << 17);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
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
    const int32_t all = quarter == 0 ? id[0] : quarter == 1 ? id[1] : quarter == 2 ? id[2] : id[3];
    const int32_t mine = all >= first && all <= last ? all : kNoAdapter;  // (ascending ids: the pass has all between)
    row_id[row] = mine;
    const bool ready = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.acc_full), 0, abort_flag));
    if (!ready) {
      if (lane == 0) report_error(err, ATENIA_ERR_DEVICE_TIMEOUT, 2600);
      *abort_flag = 1;
    } else if (quarter * 32 < rows) {
      tc_fence_after();
      const uint32_t taddr = tmem + (uint32_t(quarter * 32) << 16);
      for (int i = 0; i < count; ++i) {
        if (!__any_sync(0xffffffffu, mine == list[i])) continue;
#pragma unroll 1
        for (int j = 0; j < r; j += 8) {
          uint32_t v[8];
          tc_ld8(taddr + i * r + j, v);
          tc_ld_wait();
          if (mine == list[i]) {
            uint4* dst = reinterpret_cast<uint4*>(part + row * kRedPitch + j);
            dst[0] = make_uint4(v[0], v[1], v[2], v[3]);
            dst[1] = make_uint4(v[4], v[5], v[6], v[7]);
          }
        }
      }
      tc_fence_before();
    }
  }

  __syncthreads();
  if (split > 1) cluster_barrier();
  if (!*abort_flag) {
    if (split == 1) add_rows<1>(ar, proj, m0, rows, smem_u32(part), row_id, rank);
    else if (split == 2) add_rows<2>(ar, proj, m0, rows, smem_u32(part), row_id, rank);
    else if (split == 4) add_rows<4>(ar, proj, m0, rows, smem_u32(part), row_id, rank);
    else add_rows<8>(ar, proj, m0, rows, smem_u32(part), row_id, rank);
  }
  __syncthreads();
  if (split > 1) cluster_barrier();  // no CTA leaves while another reads its sums
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
  // a tile has no more distinct adapters than rows
  const int most = r.n < BM ? (r.M < r.n ? r.M : r.n) : (r.M < BM ? r.M : BM);
  int passes = 1;
  for (int i = 0; i < r.projections; ++i) {
    const int per_pass = kRankRows / r.p[i].rank;
    const int need = (most + per_pass - 1) / per_pass;
    if (need > passes) passes = need;
  }
  const int64_t units = (int64_t)m_tiles * passes * r.projections;
  if (units > (1 << 26)) return ATENIA_ERR_SHAPE;
  int split = 1;
  while (split < 8 && units * split < 2 * num_sms && r.kb >= 4 * split) split *= 2;
  const int stage_bytes = r.a_rows * BK * 2 + kRankRows * BK * 2;
  int stages = kRedRingBytes / stage_bytes;
  if (stages > kRedStages) stages = kRedStages;
  static bool attr_set[kMaxDevices] = {};
  if (first_use_on_current_device(attr_set)) {
    ATENIA_CUDA_TRY(cudaFuncSetAttribute(adapter_reduce_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRedRingBytes + 1024));
  }
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, adapter_reduce_kernel, r, split, passes, stages, err);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return (int)e;
}

}  // namespace atenia
