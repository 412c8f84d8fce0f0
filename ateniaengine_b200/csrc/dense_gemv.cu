// Dense products of one or two rows on the CUDA cores, and the first half of the adapters of a decode batch.
//
// A tile of the tensor-core kernels costs its pipeline (tensor memory, barriers, a ring to fill, a cluster to add in) before its
// first and after its last byte; for a handful of rows the weights' bytes are all there is, and here a warp asks for them straight
// away: two weight rows (kDenseSwiGLU: gate and up of one feature), 16 bytes a lane, four loads of each on their way.
// A block's eight warps are row pairs times pieces of the reduction (1, 2, 4, 8: the launch's choice, so that every SM has warps
// enough); pieces are added in order.  Sums are f32; products are those of the bf16 values.
//
// B200, calls one after another on weights out of L2, block of one / two tokens, these kernels and dense_gemm.cu's, us: 512 x 1408
// 4.3 / 5.6 and 8.0, 2048 x 2816 9.6 / 12.1 and 14.2, 4096 x 14336 60 / 66 and 61 (its bytes at the copy rate: 54.5); four tokens lose
// everywhere (11 .. 130), the conversions and the token rows' reads then cost more than the weights.  Eight loads of each row on their
// way: 6.4, 12.0, 57; two blocks an SM.
//
// Adapters: the lanes of a row add v[t, j] B[a, n, j] to their partial sums.  A token reads its own adapter only.
#include <type_traits>

#include "dense_gemm.cuh"

namespace atenia {
namespace {
using namespace tc;

constexpr int kVecWarps = 8;
constexpr int kVecThreads = 32 * kVecWarps;
constexpr int kAhead = 4;        // 16-byte loads of each row on their way
constexpr int kVecBlocks = 3;    // blocks an SM holds (96 KiB of weights on their way)

struct VecArgs {
  const __nv_bfloat16* x;       // [T, K]
  const __nv_bfloat16* w0;      // kDenseSwiGLU: gate, else [N, K]
  const __nv_bfloat16* w1;      // kDenseSwiGLU: up
  __nv_bfloat16* out;           // [T, N]
  float* gate;
  float* up;
  int N, K, pieces;
  bool early;                   // the weights are not the kernel before's
};
struct VecAdapters {
  const __nv_bfloat16* v[2];  // [T, rank]
  const __nv_bfloat16* b[2];  // [n, N, rank]
  int rank[2];
  const int32_t* ids;
  int n;
};
struct NoVecAdapters {};

__device__ __forceinline__ uint4 load16(const __nv_bfloat16* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint4 load16_once(const __nv_bfloat16* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ float dot8(const uint4& a, const uint4& b, float acc) {
  const uint32_t* p = &a.x;
  const uint32_t* q = &b.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    acc = __fmaf_rn(bf16lo(p[i]), bf16lo(q[i]), acc);
    acc = __fmaf_rn(bf16hi(p[i]), bf16hi(q[i]), acc);
  }
  return acc;
}

template <int EPI, int NT, bool AD>
__global__ void __launch_bounds__(kVecThreads, kVecBlocks)
dense_gemv_kernel(const __grid_constant__ VecArgs va, const __grid_constant__ std::conditional_t<AD, VecAdapters, NoVecAdapters> ad) {
  __shared__ float part[kVecWarps][2 * NT];
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  const int piece = warp % va.pieces;
  const int pair = blockIdx.x * (kVecWarps / va.pieces) + warp / va.pieces;
  const int pairs = EPI == kDenseSwiGLU ? va.N : va.N / 2;
  const bool live = pair < pairs;
  const int64_t row = EPI == kDenseSwiGLU ? pair : 2 * (int64_t)pair;
  const __nv_bfloat16* w0 = va.w0 + row * va.K;
  const __nv_bfloat16* w1 = EPI == kDenseSwiGLU ? va.w1 + row * va.K : w0 + va.K;
  const int vecs = va.K / 8;
  const int begin = (int)((int64_t)vecs * piece / va.pieces), end = (int)((int64_t)vecs * (piece + 1) / va.pieces);
  uint4 a[kAhead], b[kAhead];
  const uint4 zero = make_uint4(0, 0, 0, 0);
  auto fetch = [&](int v0) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int v = v0 + 32 * i + lane;
      const bool in = live && v < end;
      a[i] = in ? load16_once(w0 + 8 * (int64_t)v) : zero;
      b[i] = in ? load16_once(w1 + 8 * (int64_t)v) : zero;
    }
  };
  if (va.early) fetch(begin);
  chain_wait();
  if (!va.early) fetch(begin);
  float acc[2][NT] = {};
  for (int v0 = begin; v0 < end; v0 += 32 * kAhead) {
    if (v0 > begin) fetch(v0);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const __nv_bfloat16* xt = va.x + (int64_t)t * va.K;
      uint4 x[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int v = v0 + 32 * i + lane;
        x[i] = v < end ? load16(xt + 8 * (int64_t)v) : zero;
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        acc[0][t] = dot8(a[i], x[i], acc[0][t]);
        acc[1][t] = dot8(b[i], x[i], acc[1][t]);
      }
    }
  }
  if constexpr (AD) {
    if (live && piece == 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int id = ad.ids[t];
        if (id < 0 || id >= ad.n) continue;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int seg = EPI == kDenseSwiGLU ? q : 0;
          const int r = ad.rank[seg];
          const int64_t n = EPI == kDenseSwiGLU ? row : row + q;
          const __nv_bfloat16* bp = ad.b[seg] + ((int64_t)id * va.N + n) * r;
          const __nv_bfloat16* vp = ad.v[seg] + (int64_t)t * r;
          for (int j = lane; j < r; j += 32) acc[q][t] = __fmaf_rn(__bfloat162float(vp[j]), __bfloat162float(bp[j]), acc[q][t]);
        }
      }
    }
  }
  chain_next();
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[q][t] += __shfl_xor_sync(0xffffffffu, acc[q][t], o);
    }
  if (va.pieces > 1) {
    if (lane == 0) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int t = 0; t < NT; ++t) part[warp][q * NT + t] = acc[q][t];
    }
    __syncthreads();
    if (piece == 0) {
      for (int i = 1; i < va.pieces; ++i)
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[q][t] += part[warp + i][q * NT + t];
    }
  }
  if (live && piece == 0 && lane == 0) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int64_t at = (int64_t)t * va.N + row;
      if constexpr (EPI == kDenseSwiGLU) {
        va.out[at] = __float2bfloat16(silu_mul(acc[0][t], acc[1][t]));
        if (va.gate) {
          const int64_t kept = (row / 4 * NT + t) * 4 + row % 4;  // (in quads: [N / 4][T][4])
          va.gate[kept] = acc[0][t];
          va.up[kept] = acc[1][t];
        }
      } else {
        *reinterpret_cast<uint32_t*>(va.out + at) = pack_bf16x2(acc[0][t], acc[1][t]);
      }
    }
  }
}

// v[t, j .. j + 3] of one token: the block's warps take pieces of the reduction.  Tokens that share an adapter read it again from L2.
constexpr int kRankGroup = 4;
struct VecReduce {
  struct Projection {
    const __nv_bfloat16* a;  // [n, rank, K]
    const float* scale;
    __nv_bfloat16* v;
    int rank;
  } p[2];
  const __nv_bfloat16* x;
  const int32_t* ids;
  int K, n;
};
__global__ void __launch_bounds__(kVecThreads) adapter_gemv_kernel(const __grid_constant__ VecReduce vr) {
  __shared__ float part[kVecWarps][kRankGroup];
  chain_wait();
  chain_next();  // what follows reads nothing of this kernel's before its own wait
  const VecReduce::Projection& p = vr.p[blockIdx.z];
  const int t = blockIdx.y, j0 = blockIdx.x * kRankGroup;
  const int id = vr.ids[t];
  if (j0 >= p.rank || id < 0 || id >= vr.n) return;
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  const int vecs = vr.K / 8;
  const __nv_bfloat16* a = p.a + ((int64_t)id * p.rank + j0) * vr.K;
  const __nv_bfloat16* x = vr.x + (int64_t)t * vr.K;
  float acc[kRankGroup] = {};
#pragma unroll 2
  for (int v = threadIdx.x; v < vecs; v += kVecThreads) {
    const uint4 xv = load16(x + 8 * (int64_t)v);
    uint4 w[kRankGroup];
#pragma unroll
    for (int j = 0; j < kRankGroup; ++j) w[j] = load16(a + (int64_t)j * vr.K + 8 * (int64_t)v);
#pragma unroll
    for (int j = 0; j < kRankGroup; ++j) acc[j] = dot8(w[j], xv, acc[j]);
  }
#pragma unroll
  for (int j = 0; j < kRankGroup; ++j) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
    if (lane == 0) part[warp][j] = acc[j];
  }
  __syncthreads();
  if (threadIdx.x < kRankGroup) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kVecWarps; ++i) sum += part[i][threadIdx.x];
    p.v[(int64_t)t * p.rank + j0 + threadIdx.x] = __float2bfloat16(sum * p.scale[id]);
  }
}

template <int EPI, int NT, bool AD>
int launch_vec(const DenseGemm& g, const VecArgs& va, int blocks, cudaStream_t s) {
  std::conditional_t<AD, VecAdapters, NoVecAdapters> ad{};
  if constexpr (AD) {
    for (int i = 0; i < 2; ++i) {
      ad.v[i] = g.adapters->seg[i].v_ptr;
      ad.b[i] = g.adapters->seg[i].b_ptr;
      ad.rank[i] = g.adapters->seg[i].rank;
    }
    ad.ids = g.adapters->ids;
    ad.n = g.adapters->n;
  }
  return launch_chained(g.chained, dense_gemv_kernel<EPI, NT, AD>, dim3(blocks), dim3(kVecThreads), 0, s, va, ad);
}
template <int EPI, bool AD>
int launch_vec_tokens(const DenseGemm& g, const VecArgs& va, int blocks, cudaStream_t s) {
  if (g.p[0].M == 1) return launch_vec<EPI, 1, AD>(g, va, blocks, s);
  return launch_vec<EPI, 2, AD>(g, va, blocks, s);
}

}  // namespace

bool dense_gemv_serves(const DenseGemm& g) {
  const DenseProblem& p = g.p[0];
  return g.problems == 1 && !p.b_mn && (g.epilogue == kDensePlain || g.epilogue == kDenseSwiGLU) && dense_gemv_rows(p.M, p.N, p.K);
}

int launch_dense_gemv(const DenseGemm& g, int num_sms, cudaStream_t s) {
  const DenseProblem& p = g.p[0];
  VecArgs va{};
  va.x = p.a_ptr;
  va.w0 = p.b_ptr[0];
  va.w1 = p.b_ptr[1];
  va.out = p.out;
  va.gate = p.gate;
  va.up = p.up;
  va.N = p.N;
  va.K = p.K;
  va.early = g.b_early;
  const int pairs = g.epilogue == kDenseSwiGLU ? p.N : p.N / 2;
  // pieces until the SMs have 16 warps each, of a vector per lane at least
  va.pieces = 1;
  while (va.pieces < kVecWarps && (int64_t)pairs * va.pieces < 16 * (int64_t)num_sms && p.K >= 512 * va.pieces) va.pieces *= 2;
  const int per_block = kVecWarps / va.pieces;
  const int blocks = (pairs + per_block - 1) / per_block;
  count_launch();
  const bool ad = g.adapters != nullptr;
  if (g.epilogue == kDenseSwiGLU)
    return ad ? launch_vec_tokens<kDenseSwiGLU, true>(g, va, blocks, s) : launch_vec_tokens<kDenseSwiGLU, false>(g, va, blocks, s);
  return ad ? launch_vec_tokens<kDensePlain, true>(g, va, blocks, s) : launch_vec_tokens<kDensePlain, false>(g, va, blocks, s);
}

int launch_adapter_gemv(const AdapterReduce& r, cudaStream_t s) {
  VecReduce vr{};
  int rank = 0;
  for (int i = 0; i < r.projections; ++i) {
    vr.p[i].a = r.p[i].a_ptr;
    vr.p[i].scale = r.p[i].scale;
    vr.p[i].v = r.p[i].v;
    vr.p[i].rank = r.p[i].rank;
    if (r.p[i].rank > rank) rank = r.p[i].rank;
  }
  vr.x = r.x_ptr;
  vr.ids = r.ids;
  vr.K = r.K;
  vr.n = r.n;
  count_launch();
  return launch_chained(r.chained, adapter_gemv_kernel, dim3(rank / kRankGroup, r.M, r.projections), dim3(kVecThreads), 0, s, vr);
}

}  // namespace atenia
