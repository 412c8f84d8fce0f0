// Dense products of up to 16 rows, and the first half of the adapters of a decode batch.
//
// A tile of the tcgen05 kernels costs its pipeline (tensor memory, barriers, a ring to fill, a cluster to add in) before its first and
// after its last byte; for a handful of rows the weights' bytes are all there is, and here a warp asks for them straight away into
// the registers that multiply them: 16 weight rows (kDenseSwiGLU: gate and up of eight features) as the m16 side of mma.sync
// m16n8k16, the token rows as its n side, 8 or 16 of them.  Lanes take 32 bytes of a row each, 64 of k a step: that orders k inside a
// step differently from the instruction's operands, for weights and tokens alike, which a sum does not mind.  Two or three steps are on
// their way (RowsShape).  A block's eight warps are row groups times pieces of the reduction (rows_plan), which are added in order.
// h of a block of up to eight tokens comes in two parts, its rounding to bf16 and what that left, as twice the tokens of the second
// product: their columns would be empty, and the result is as exact as its own rounding (its error is 1.42 times that otherwise).
// B200, weights out of L2, us, this kernel / dense_gemm.cu's: block of 1 token, 512 x 1408 4.5 / 7.5, 2048 x 2816 10.4 / 14.3, 2048 x 5632
// 16.4 / 19.6; of 16, 5.3 / 8.1, 12.5 / 14.8; one product 4096 x 4096 8.2 / 11.1 (1 token), 8.5 / 11.9 (8).  The bytes of a block
// of 2048 x 2816 take 5.4 us at the copy rate: what is left is the two launches and their first loads.
//
// Adapters: a warp adds its piece of the rank columns, v[t, j] B[a, n, j] for the tokens and rows that its lanes hold.  A token reads its
// own adapter only.
#include <type_traits>

#include "dense_choice.cuh"
#include "dense_gemm.cuh"

namespace atenia {
namespace {
using namespace tc;

constexpr int kVecWarps = 8;
constexpr int kVecThreads = 32 * kVecWarps;
constexpr int kStep = 64;  // k of a step: 32 bytes a lane
// Steps on their way and blocks an SM holds: more of a warp, or more warps for gate and up of a large matrix, where these fill the last
// wave about as well.  B200, blocks of one token, all products with three steps and two blocks / gate and up with two and three, us: 512 x
// 1408 4.5 / 5.1, 2048 x 5632 19.3 / 16.4, 1024 x 16384 31.8 / 26.9, 4096 x 14336 63.5 / 60.8, 4096 x 8192 (filled to 0.87 and 0.77) 36.0 /
// 38.3.  One product with three steps and two blocks / two and three, four tokens: 4096 x 8192 14.1 / 17.4, 5120 x 5120 13.0 / 13.1.
template <bool LARGE>
struct RowsShape {
  static constexpr int kAhead = LARGE ? 2 : 3;
  static constexpr int kBlocks = LARGE ? 3 : 2;
};
constexpr int64_t kLargeElements = (int64_t)1 << 24;

struct VecArgs {
  const __nv_bfloat16* x;   // [T, K]
  const __nv_bfloat16* w0;  // kDenseSwiGLU: gate, else [N, K]
  const __nv_bfloat16* w1;  // kDenseSwiGLU: up
  __nv_bfloat16* out;       // [T, N]
  float* gate;
  float* up;
  int T, N, K, pieces;
  bool early;               // the weights are not the kernel before's
  bool x_rest, out_rest;    // behind x, and behind out, comes what rounding them left
};
struct VecAdapters {
  const __nv_bfloat16* v[2];  // [parts, T, rank]
  const __nv_bfloat16* b[2];  // [n, N, rank]
  int rank[2];
  const int32_t* ids;
  int n, parts;
};
struct NoVecAdapters {};

__device__ __forceinline__ uint4 load16(const __nv_bfloat16* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
// 32 bytes a lane: four lanes have a whole line of a row (16 bytes of eight rows are eight half lines, and the lines are what L1 counts)
struct Words {
  uint32_t w[8];
};
__device__ __forceinline__ Words load32_once(const __nv_bfloat16* p) {
  Words v;
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
               : "l"(p));
  return v;
}
__device__ __forceinline__ Words load32(const __nv_bfloat16* p) {
  Words v;
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
               : "l"(p)
               : "memory");
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
__device__ __forceinline__ void mma_rows(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT: tiles of eight tokens (x in two parts: the first half of them the tokens, the other half what their rounding left).  Lane 4 g + i
// holds 32 bytes (piece i of a step) of weight rows g and g + 8 and of tokens g, g + 8, and sums of those rows for tokens 2 i and 2 i + 1
// of a tile.
template <int EPI, int NT, bool AD, bool LARGE>
__global__ void __launch_bounds__(kVecThreads, RowsShape<LARGE>::kBlocks)
dense_rows_kernel(const __grid_constant__ VecArgs va, const __grid_constant__ std::conditional_t<AD, VecAdapters, NoVecAdapters> ad) {
  __shared__ __align__(16) float part[kVecWarps][NT][32][4];
  constexpr int kAhead = RowsShape<LARGE>::kAhead;
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  const int g = lane >> 2, i4 = lane & 3;
  const int piece = warp % va.pieces;
  const int group = blockIdx.x * (kVecWarps / va.pieces) + warp / va.pieces;
  constexpr int kGroupRows = EPI == kDenseSwiGLU ? 8 : 16;  // result columns of a group
  const int n0 = group * kGroupRows + g, n1 = EPI == kDenseSwiGLU ? n0 : n0 + 8;
  const bool live = group * kGroupRows < va.N;  // (N is a multiple of 16)
  const __nv_bfloat16* w0 = va.w0 + (int64_t)n0 * va.K + 16 * i4;
  const __nv_bfloat16* w1 = (EPI == kDenseSwiGLU ? va.w1 : va.w0) + (int64_t)n1 * va.K + 16 * i4;
  const int steps = (va.K + kStep - 1) / kStep;
  const int begin = (int)((int64_t)steps * piece / va.pieces), end = live ? (int)((int64_t)steps * (piece + 1) / va.pieces) : begin;
  Words a[kAhead], b[kAhead];
  const Words zero = {};
  auto fetch = [&](int s0) {
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      const bool in = s0 + s < end && kStep * (s0 + s) + 16 * i4 < va.K;
      a[s] = in ? load32_once(w0 + kStep * (int64_t)(s0 + s)) : zero;
      b[s] = in ? load32_once(w1 + kStep * (int64_t)(s0 + s)) : zero;
    }
  };
  if (va.early) fetch(begin);
  chain_wait();
  if (!va.early) fetch(begin);
  float c[NT][4] = {};
  const __nv_bfloat16* x[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int column = 8 * t + g;
    const bool rest = va.x_rest && column >= 4 * NT;
    x[t] = va.x + ((int64_t)min(rest ? column - 4 * NT : column, va.T - 1) + (rest ? va.T : 0)) * va.K + 16 * i4;
  }
  for (int s0 = begin; s0 < end; s0 += kAhead) {
    if (s0 > begin) fetch(s0);
    Words xv[NT][kAhead];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        const bool in = s0 + s < end && kStep * (s0 + s) + 16 * i4 < va.K;
        xv[t][s] = in ? load32(x[t] + kStep * (int64_t)(s0 + s)) : zero;
      }
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int q = 0; q < 8; q += 2)
          mma_rows(c[t], a[s].w[q], b[s].w[q], a[s].w[q + 1], b[s].w[q + 1], xv[t][s].w[q], xv[t][s].w[q + 1]);
  }
  if (va.x_rest) {  // both parts of a token's x
#pragma unroll
    for (int q = 0; q < 4; ++q) c[0][q] += NT == 1 ? __shfl_xor_sync(0xffffffffu, c[0][q], 2) : c[NT - 1][q];
  }
  if constexpr (AD) {
    if (live) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int token = 8 * t + 2 * i4 + q;
          const int id = token < va.T ? ad.ids[token] : -1;
          if (id < 0 || id >= ad.n) continue;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int seg = EPI == kDenseSwiGLU ? h : 0;
            const int r = ad.rank[seg];
            const __nv_bfloat16* bp = ad.b[seg] + ((int64_t)id * va.N + (h ? n1 : n0)) * r;
            const __nv_bfloat16* vp = ad.v[seg] + (int64_t)token * r;
            for (int j = 8 * piece; j < r; j += 8 * va.pieces) {
              const uint4 bv = load16(bp + j);
              c[t][2 * h + q] = dot8(load16(vp + j), bv, c[t][2 * h + q]);
              if (ad.parts > 1) c[t][2 * h + q] = dot8(load16(vp + (int64_t)va.T * r + j), bv, c[t][2 * h + q]);
            }
          }
        }
    }
  }
  chain_next();
  if (va.pieces > 1) {
#pragma unroll
    for (int t = 0; t < NT; ++t) *reinterpret_cast<float4*>(part[warp][t][lane]) = make_float4(c[t][0], c[t][1], c[t][2], c[t][3]);
    __syncthreads();
    if (piece > 0) return;
    for (int i = 1; i < va.pieces; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float4 v = *reinterpret_cast<const float4*>(part[warp + i][t][lane]);
        c[t][0] += v.x, c[t][1] += v.y, c[t][2] += v.z, c[t][3] += v.w;
      }
  }
  if (!live) return;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int token = 8 * t + 2 * i4 + q;
      if (token >= va.T) continue;
      __nv_bfloat16* out = va.out + (int64_t)token * va.N;
      if constexpr (EPI == kDenseSwiGLU) {
        const float o = silu_mul(c[t][q], c[t][2 + q]);
        out[n0] = __float2bfloat16(o);
        if (va.out_rest) out[(int64_t)va.T * va.N + n0] = __float2bfloat16(left_of_bf16(o));
        if (va.gate) {
          const int64_t kept = ((int64_t)(n0 / 4) * va.T + token) * 4 + n0 % 4;  // (in quads: [N / 4][T][4])
          va.gate[kept] = c[t][q];
          va.up[kept] = c[t][2 + q];
        }
      } else {
        out[n0] = __float2bfloat16(c[t][q]);
        out[n1] = __float2bfloat16(c[t][2 + q]);
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
  int T, K, n, parts;
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
    sum *= p.scale[id];
    __nv_bfloat16* to = p.v + (int64_t)t * p.rank + j0 + threadIdx.x;
    *to = __float2bfloat16(sum);
    if (vr.parts > 1) to[(int64_t)vr.T * p.rank] = __float2bfloat16(left_of_bf16(sum));
  }
}

template <int EPI, int NT, bool AD, bool LARGE>
int launch_rows(const DenseGemm& g, const VecArgs& va, int blocks, cudaStream_t s) {
  std::conditional_t<AD, VecAdapters, NoVecAdapters> ad{};
  if constexpr (AD) {
    for (int i = 0; i < 2; ++i) {
      ad.v[i] = g.adapters->seg[i].v_ptr;
      ad.b[i] = g.adapters->seg[i].b_ptr;
      ad.rank[i] = g.adapters->seg[i].rank;
    }
    ad.ids = g.adapters->ids;
    ad.n = g.adapters->n;
    ad.parts = g.adapters->parts;
  }
  return launch_chained(g.chained, dense_rows_kernel<EPI, NT, AD, LARGE>, dim3(blocks), dim3(kVecThreads), 0, s, va, ad);
}
template <int EPI, bool AD>
int launch_rows_tokens(const DenseGemm& g, const VecArgs& va, bool large, int blocks, cudaStream_t s) {
  // two tiles of eight: more than eight tokens, or more than four in two parts
  if (va.T > 8 || (va.x_rest && va.T > 4)) return launch_rows<EPI, 2, AD, false>(g, va, blocks, s);
  if constexpr (EPI == kDenseSwiGLU)
    if (large) return launch_rows<EPI, 1, AD, true>(g, va, blocks, s);
  return launch_rows<EPI, 1, AD, false>(g, va, blocks, s);
}

}  // namespace

bool dense_rows_serve(const DenseGemm& g) {
  const DenseProblem& p = g.p[0];
  return g.problems == 1 && !p.b_mn && (g.epilogue == kDensePlain || g.epilogue == kDenseSwiGLU) &&
         dense_rows(p.M, p.N, p.K, g.epilogue == kDenseSwiGLU, p.a_ptr, p.b_ptr[0], p.b_ptr[1]);
}

int launch_dense_rows(const DenseGemm& g, int num_sms, cudaStream_t s) {
  const DenseProblem& p = g.p[0];
  VecArgs va{};
  va.x = p.a_ptr;
  va.w0 = p.b_ptr[0];
  va.w1 = p.b_ptr[1];
  va.out = p.out;
  va.gate = p.gate;
  va.up = p.up;
  va.T = p.M;
  va.N = p.N;
  va.K = p.K;
  va.early = g.b_early;
  va.x_rest = p.a_rest;
  va.out_rest = p.out_rest;
  const int groups = g.epilogue == kDenseSwiGLU ? p.N / 8 : p.N / 16;
  const int steps = (p.K + kStep - 1) / kStep;
  const RowsPlan few = rows_plan(groups, steps, kVecWarps, RowsShape<false>::kBlocks * num_sms);
  const RowsPlan many = rows_plan(groups, steps, kVecWarps, RowsShape<true>::kBlocks * num_sms);
  const bool large = g.epilogue == kDenseSwiGLU && (int64_t)2 * p.N * p.K > kLargeElements && p.M <= 8 && many.used >= 0.92 * few.used;
  const RowsPlan& plan = large ? many : few;
  const int blocks = plan.blocks;
  va.pieces = plan.pieces;
  count_launch();
  const bool ad = g.adapters != nullptr;
  if (g.epilogue == kDenseSwiGLU)
    return ad ? launch_rows_tokens<kDenseSwiGLU, true>(g, va, large, blocks, s) : launch_rows_tokens<kDenseSwiGLU, false>(g, va, large, blocks, s);
  return ad ? launch_rows_tokens<kDensePlain, true>(g, va, large, blocks, s) : launch_rows_tokens<kDensePlain, false>(g, va, large, blocks, s);
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
  vr.T = r.M;
  vr.K = r.K;
  vr.parts = r.parts;
  vr.n = r.n;
  count_launch();
  return launch_chained(r.chained, adapter_gemv_kernel, dim3(rank / kRankGroup, r.M, r.projections), dim3(kVecThreads), 0, s, vr);
}

}  // namespace atenia
