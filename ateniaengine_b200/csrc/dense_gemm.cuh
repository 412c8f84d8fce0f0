// Products of the dense feed-forward block and of the low-rank adapters: what the kernels (dense_gemm.cu,
// dense_pair.cu, dense_rows.cu, adapters.cu) and the entry points (gated_ffn.cu) share.
//
// Every product is D[m, n] = sum_k A[m, k] B[n, k] with D row-major.  An operand lies in memory either with k contiguous
// ("K-major": activations times weights as the models store them) or with its own rows contiguous ("MN-major": the transposed
// reads of the backward pass, where the reduction runs over the rows of a row-major matrix).  Both come through TMA into
// 128-byte-swizzled tiles and the MMA reads either, so nothing is transposed in memory.
#pragma once
#include "dense_choice.cuh"
#include "tc_common.cuh"

namespace atenia {

// What the forward pass keeps for the backward one (g and u, f32) is laid out in quads, [N / 4][M][4]: a lane of tensor memory holds a
// row of D, so a warp that takes four features of 32 tokens reads or writes 512 bytes in a row, where the rows of a plain [M, N]
// would be 32 lines an access.
enum DenseEpilogue {
  kDensePlain = 0,     // out[m, n] = D
  kDenseSwiGLU = 1,    // B = gate and up rows of the same features: out[m, f] = silu(g) u, optionally g and u in quads
  kDenseGateGrad = 2,  // D = dh: dg, du and h from the saved g and u
};

struct DenseProblem {
  CUtensorMap a[2], b[2];  // kDenseSwiGLU: b[0] gate, b[1] up.  Else the k-blocks from kb0 on come through a[1] and b[1]
  int M, N, kb, kb0;       // N: columns of `out`; kb: k-blocks of 64 in all
  bool b_mn;               // MN-major operands: B, or (several problems in a launch) A and B
  __nv_bfloat16* out;      // [M, N]
  float* gate;             // kDenseSwiGLU: g and u to be saved, or null; kDenseGateGrad: the saved ones
  float* up;
  const __nv_bfloat16* a_ptr;     // the same operands for the kernels that read them plainly (dense_rows.cu)
  const __nv_bfloat16* b_ptr[2];
  int K;
  bool a_rest, out_rest;          // dense_rows.cu, up to kRestMost rows: A, or `out`, is followed by what its rounding to bf16 left
  __nv_bfloat16* out_du;   // kDenseGateGrad: du and h [M, N] (dg is `out`)
  __nv_bfloat16* out_h;
};

// One projection's adapters beside the product: D[m, :] += B_a v[m, :] for a = ids[m].  (kDenseSwiGLU: segment 0 acts on the
// gate columns, segment 1 on the up columns; a segment of rank 0 adds nothing.)
struct AdapterSegment {
  CUtensorMap v;  // [parts, M, rank] bf16, box {width, rows, 1}, swizzle of the box's width
  CUtensorMap b;  // [n, N, rank] bf16, box {width, 64, 1}, likewise
  int rank, width;  // adapter_width(rank)
  const __nv_bfloat16* v_ptr;
  const __nv_bfloat16* b_ptr;
};
// Rank columns of a box.  TMA takes as long for a row of 32 bytes as for one of 128 (about 4 cycles): boxes are as wide as the rank lets
// them (columns past it are filled with zeros and left out of the MMAs).
inline int adapter_width(int rank) { return rank > 32 ? 64 : rank > 16 ? 32 : 16; }
// The reduced rows are rounded to bf16, the second product's operand.  Where the adapters may make a good part of a sum (its terms are
// `rank` beside `in`), that rounding would show in the result beside its own; then what the first rounding left is a second operand,
// multiplied by the same B.  Root mean square of the error, block of 256 x 2048 with rank 128 on all three projections, one part / two:
// 0.0025 / 0.0023 (0.0017 is the rounding of the result, 0.0017 that of h).
inline int adapter_parts(int rank, int64_t in) { return (int64_t)32 * rank > in ? 2 : 1; }
struct DenseAdapters {
  AdapterSegment seg[2];
  const int32_t* ids;  // [M]; an id outside [0, n) means none
  int n, parts;
};

constexpr int kMaxDenseProblems = 3;
struct DenseGemm {
  DenseProblem p[kMaxDenseProblems];
  int problems;
  int epilogue;
  const DenseAdapters* adapters;  // or null (host pointer, copied at the launch)
  int a_rows;                    // rows of A a stage holds: of a K-major A's box (dense_a_rows), else 128
  bool chained;                  // see launch_chained
  bool b_early;                  // B is not written by the kernel before: its first tiles are requested before the wait
  bool a_early;                  // neither is A: only the adapters' v, and the stores, wait
  bool next_early;               // what follows reads nothing of this product's: it may start on SMs that this one leaves
                                 // free (a launch of pairs on all of them does not let it: 4096 tokens, 2048 x 5632 420 / 425 us)
};
int launch_dense_gemm(const DenseGemm& g, int num_sms, cudaStream_t s);   // chooses between them
int launch_dense_tiles(const DenseGemm& g, int columns, int split, cudaStream_t s);  // dense_gemm.cu
int launch_dense_pairs(const DenseGemm& g, int split, int tail_split, int num_sms, cudaStream_t s);  // dense_pair.cu
int launch_dense_rows(const DenseGemm& g, int num_sms, cudaStream_t s);   // dense_rows.cu, where it serves the product
bool dense_rows_serve(const DenseGemm& g);
// Up to 8 rows of a matrix of at most 2^25 elements and up to 16 of one of at most 2^23; one row of any.  Operands on 32-byte
// boundaries, which the kernel's loads want (any row of a matrix is on one if the first is).  B200, block of 16 tokens, this kernel /
// dense_gemm.cu's, us: 512 x 1408 5.3 / 8.1, 2048 x 2816 12.5 / 14.8, 2048 x 5632 22.4 / 20.5; of eight 5.0 / 7.8, 11.4 / 14.5, 18.8 /
// 20.1, 4096 x 14336 65.7 / 61.8; of one 60.1 / 61.0.
constexpr int kRowsMost = 16, kRestMost = 8;
inline bool dense_rows(int64_t M, int64_t N, int64_t K, bool two, const void* x, const void* w0, const void* w1) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w0) | (two ? reinterpret_cast<uintptr_t>(w1) : 0);
  return (at & 31) == 0 && M <= kRowsMost && (M == 1 || N * K <= (M <= 8 ? (int64_t)1 << 25 : (int64_t)1 << 23));
}

// Rows of a K-major A box: all of a small batch, so that a call of few tokens moves few token rows.
inline int dense_a_rows(int64_t rows) { return rows >= 128 ? 128 : (int)((rows + 7) / 8 * 8); }

// v[t, :] = scale[a] * (A_a x[t, :]), a = ids[t], for up to two projections of the same rows
struct AdapterReduce {
  struct Projection {
    CUtensorMap a;  // [n, rank, K] bf16, box {64, rank, 1}, 128-byte swizzle
    const float* scale;  // [n]
    __nv_bfloat16* v;    // [parts, M, rank]
    int rank;
    const __nv_bfloat16* a_ptr;
  } p[2];
  int projections;
  CUtensorMap x;  // [M, K], box {64, a_rows}
  const __nv_bfloat16* x_ptr;
  const int32_t* ids;
  int M, K, kb, n, a_rows, parts;
  bool few;  // adapter_gemv_rows: the maps are not encoded
  bool chained;
};
int launch_adapter_reduce(const AdapterReduce& r, int num_sms, cudaStream_t s);
int launch_adapter_gemv(const AdapterReduce& r, cudaStream_t s);  // dense_rows.cu, for few tokens
// It reads an adapter once per token: up to this many tokens, and elements of A over all of them.  B200, adapter_linear of 4096 x 4096
// with this kernel / adapters.cu's, us: 20 tokens, rank 16, 4 adapters 12.5 / 14.3, 128 adapters 13.8 / 18.9; 64 tokens, rank 64 18.2 /
// 19.3 and 25.0 / 27.7; 128 tokens, rank 16 18.4 / 19.7 and 29.4 / 32.0; 128 tokens, rank 64, above the limit 25.6 / 23.2 and 39.1 / 41.8.
inline bool adapter_gemv_rows(int64_t M, int64_t rank, int64_t K) { return M <= 128 && M * rank * K <= (int64_t)16 << 20; }
constexpr int kAdapterMaxRank = 128;

// Where kernels of these files record a wait that gave up: one word per device, read by atenia_ffn_check.
int dense_error_word(DeviceError** out);

// bf16 map of up to three dimensions (innermost first, contiguous); dims[2] = 0: two
int encode_tmap_bf16(CUtensorMap* out, const void* base, const uint64_t (&dims)[3], const uint32_t (&box)[3], int swizzle_bytes);

// ---- device side -------------------------------------------------------------------------------
#ifdef __CUDACC__
namespace tc {
// Descriptor of an MN-major operand under the 128-byte swizzle: atoms of 64 elements x 8 k; the next 8 k 1024 bytes on
// (stride offset), the next 64 elements 8192 bytes on (leading offset; a box of 64 k x 64 elements).
__device__ __forceinline__ uint64_t make_smem_desc_mn(uint32_t smem_addr) {
  uint64_t d = static_cast<uint64_t>((smem_addr >> 4) & 0x3FFF);
  d |= static_cast<uint64_t>(8192 >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
// K-major operand of `width` (16, 32, 64) columns a row under the swizzle of that width; eight-row groups follow one another.
__device__ __forceinline__ uint64_t make_smem_desc_width(uint32_t smem_addr, int width) {
  uint64_t d = static_cast<uint64_t>((smem_addr >> 4) & 0x3FFF);
  d |= static_cast<uint64_t>(1) << 16;
  d |= static_cast<uint64_t>(width) << 32;  // 8 rows x 2 width bytes >> 4
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(width == 64 ? 2 : width == 32 ? 4 : 6) << 61;
  return d;
}
// The chunks (boxes of up to `width` rank columns) that one adapter of a product comes in: segment 0's, then segment 1's; at most
// four.  Loops over them are unrolled, so that what they read stays in registers.
constexpr int kMaxChunks = 4;
template <int EPI>
struct AdapterChunks {
  int chunks, widest;  // widest: the wider segment's width, which sets the distance of chunks in shared memory
  int width[kMaxChunks], column[kMaxChunks], steps[kMaxChunks];  // steps: K = 16 steps that hold rank columns
  bool second[kMaxChunks];                                       // of segment 1
  int columns;                                                   // of all chunks
  __device__ __forceinline__ explicit AdapterChunks(const DenseAdapters& ad) {
    const int w0 = ad.seg[0].rank > 0 ? ad.seg[0].width : 0;
    const int w1 = EPI == kDenseSwiGLU && ad.seg[1].rank > 0 ? ad.seg[1].width : 0;
    const int n0 = w0 ? (ad.seg[0].rank + w0 - 1) / w0 : 0, n1 = w1 ? (ad.seg[1].rank + w1 - 1) / w1 : 0;
    chunks = n0 + n1;
    widest = max(w0, w1);
    columns = 0;
#pragma unroll
    for (int c = 0; c < kMaxChunks; ++c) {
      second[c] = c >= n0;
      width[c] = second[c] ? w1 : w0;
      column[c] = (second[c] ? c - n0 : c) * width[c];
      steps[c] = c < chunks ? (min(width[c], (second[c] ? ad.seg[1].rank : ad.seg[0].rank) - column[c]) + 15) / 16 : 0;
      columns += c < chunks ? width[c] : 0;
    }
  }
};
template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t smem_addr) {
  return MN ? make_smem_desc_mn(smem_addr) : make_smem_desc(smem_addr);
}
// K = 16 further inside the tile: 32 bytes of the swizzle row, or 16 rows of 128 bytes
template <bool MN>
constexpr uint64_t kOperandStep = MN ? (2048 >> 4) : (32 >> 4);

__device__ __forceinline__ void tma_load_3d_one(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n\t}"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// One to four accumulating MMAs (K = 16 each, 32 bytes apart inside the rows) that leave the lanes whose bit is set in `off` as they are.
// In one block: the masks go to the registers of the instruction once.
__device__ __forceinline__ void tc_mma_bf16_lanes_one(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, int steps,
                                                      const uint32_t (&off)[4]) {
  asm volatile(
      "{\n\t.reg .pred e, t, p;\n\t"
      ".reg .b64 a, b;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.eq.b32 t, 0, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%4, %5, %6, %7}, t;\n\t"
      "setp.gt.and.s32 p, %8, 1, e;\n\tadd.s64 a, %1, 2;\n\tadd.s64 b, %2, 2;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, {%4, %5, %6, %7}, t;\n\t"
      "setp.gt.and.s32 p, %8, 2, e;\n\tadd.s64 a, %1, 4;\n\tadd.s64 b, %2, 4;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, {%4, %5, %6, %7}, t;\n\t"
      "setp.gt.and.s32 p, %8, 3, e;\n\tadd.s64 a, %1, 6;\n\tadd.s64 b, %2, 6;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, {%4, %5, %6, %7}, t;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(off[0]), "r"(off[1]), "r"(off[2]), "r"(off[3]), "r"(steps)
      : "memory");
}
__device__ __forceinline__ void tc_ld8(uint32_t taddr, uint32_t (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(taddr));
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Four floats at this offset of the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\t"
      "mapa.shared::cluster.u32 a, %4, %5;\n\t"
      "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(addr), "r"(rank));
  return v;
}

__device__ __forceinline__ float4 ld_shared_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

constexpr int kNoAdapter = 0x7fffffff;
// The ids of 32 * W token rows from `row0` on, W per lane; kNoAdapter where a row is past the end or has none.
template <int W>
__device__ __forceinline__ void load_ids(int32_t (&id)[W], const int32_t* __restrict__ ids, int64_t row0, int rows, int n, int lane) {
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int r = 32 * w + lane;
    const int32_t v = r < rows ? ids[row0 + r] : -1;
    id[w] = v >= 0 && v < n ? v : kNoAdapter;
  }
}
// The smallest id above `last` that some row has, kNoAdapter if there is none: the adapters of a tile in ascending order, found
// alike by every warp that walks them.
template <int W>
__device__ __forceinline__ int32_t next_adapter(const int32_t (&id)[W], int32_t last) {
  int32_t m = kNoAdapter;
#pragma unroll
  for (int w = 0; w < W; ++w) m = id[w] > last && id[w] < m ? id[w] : m;
  return __reduce_min_sync(0xffffffffu, m);
}
// Bit set: the row does not have adapter `a`.
template <int W>
__device__ __forceinline__ void lanes_off(uint32_t (&off)[W], const int32_t (&id)[W], int32_t a) {
#pragma unroll
  for (int w = 0; w < W; ++w) off[w] = __ballot_sync(0xffffffffu, id[w] != a);
}

// The distinct adapters of a tile's rows in the order of their first rows, by the 128 threads of four warps (thread r: row r).
struct __align__(16) TileList {
  int32_t id[BM];     // of the rows, kNoAdapter where a row has none
  int32_t adapter[BM];
  int32_t count;
  int32_t in_warp[4];
};
__device__ __forceinline__ void list_adapters(TileList& l, const int32_t* __restrict__ ids, int64_t row0, int rows, int n, int w, int lane) {
  const int r = 32 * w + lane;
  const int32_t raw = r < rows ? ids[row0 + r] : -1;
  const int32_t id = raw >= 0 && raw < n ? raw : kNoAdapter;
  l.id[r] = id;
  asm volatile("bar.sync 1, 128;" ::: "memory");
  const uint32_t same = __match_any_sync(0xffffffffu, id);  // (every lane: not behind the test)
  bool first = id != kNoAdapter && (same & ((1u << lane) - 1)) == 0;
  if (w > 0) first = first && l.id[32 * w - 1] != id;
  if (__any_sync(0xffffffffu, first)) {  // (in a prompt most warps' rows only go on with the last one's adapter)
    const int4* before = reinterpret_cast<const int4*>(l.id);
#pragma unroll 4
    for (int q = 0; q < 8 * w; ++q) {
      const int4 v = before[q];
      first = first && v.x != id && v.y != id && v.z != id && v.w != id;
    }
  }
  const uint32_t b = __ballot_sync(0xffffffffu, first);
  if (lane == 0) l.in_warp[w] = __popc(b);
  asm volatile("bar.sync 1, 128;" ::: "memory");
  int at = __popc(b & ((1u << lane) - 1)), total = 0;
  for (int q = 0; q < 4; ++q) {
    if (q < w) at += l.in_warp[q];
    total += l.in_warp[q];
  }
  if (first) l.adapter[at] = id;
  if (r == 0) l.count = total;
}

// dg, du and h of one element
__device__ __forceinline__ void gate_grad(float dh, float g, float u, float& dg, float& du, float& h) {
  const float s = __fdividef(1.0f, 1.0f + __expf(-g));
  dg = dh * u * (s * (1.0f + g * (1.0f - s)));
  du = dh * (g * s);
  h = silu_mul(g, u);
}
// Four features of a token in the quads of the saved projections
__device__ __forceinline__ float4* quad(float* base, const DenseProblem& p, int row, int col) {
  return reinterpret_cast<float4*>(base) + (int64_t)(col >> 2) * p.M + row;
}
// What rounding `v` to bf16 leaves (nothing of an infinity)
__device__ __forceinline__ float left_of_bf16(float v) {
  const float r = v - __bfloat162float(__float2bfloat16(v));
  return fabsf(r) <= fabsf(v) ? r : 0.f;
}
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
// The saved projections of N columns of a row (kDenseGateGrad): asked for before the sums are there, or the epilogue waits for each.
template <int EPI, int N>
struct Saved {
  float4 g[EPI == kDenseGateGrad ? N / 4 : 1], u[EPI == kDenseGateGrad ? N / 4 : 1];
  __device__ __forceinline__ void load(const DenseProblem& p, int row, int col, bool in) {
    if constexpr (EPI == kDenseGateGrad) {
#pragma unroll
      for (int j = 0; j < N / 4; ++j) {
        g[j] = in ? *quad(p.gate, p, row, col + 4 * j) : make_float4(0.f, 0.f, 0.f, 0.f);
        u[j] = in ? *quad(p.up, p, row, col + 4 * j) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
  }
};
// The values that N neighbouring columns of one row become (acc1: the up columns of kDenseSwiGLU): o, and du and h of kDenseGateGrad.
// `in`: the row exists, the saved projections may be written.
template <int EPI, int N>
__device__ __forceinline__ void dense_values(const DenseProblem& p, int row, int col, bool in, const float (&acc)[N], const float (&acc1)[N],
                                             const Saved<EPI, N>& kept, float (&o)[N], float (&du)[N], float (&h)[N]) {
  if constexpr (EPI == kDensePlain) {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = acc[j];
  } else if constexpr (EPI == kDenseSwiGLU) {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = silu_mul(acc[j], acc1[j]);
    if (p.gate && in) {
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        *quad(p.gate, p, row, col + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
        *quad(p.up, p, row, col + j) = make_float4(acc1[j], acc1[j + 1], acc1[j + 2], acc1[j + 3]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      gate_grad(acc[4 * j], kept.g[j].x, kept.u[j].x, o[4 * j], du[4 * j], h[4 * j]);
      gate_grad(acc[4 * j + 1], kept.g[j].y, kept.u[j].y, o[4 * j + 1], du[4 * j + 1], h[4 * j + 1]);
      gate_grad(acc[4 * j + 2], kept.g[j].z, kept.u[j].z, o[4 * j + 2], du[4 * j + 2], h[4 * j + 2]);
      gate_grad(acc[4 * j + 3], kept.g[j].w, kept.u[j].w, o[4 * j + 3], du[4 * j + 3], h[4 * j + 3]);
    }
  }
}
// ... stored from the lane that holds the row; N = 16 or 4
template <int EPI, int N>
__device__ __forceinline__ void dense_emit(const DenseProblem& p, int row, int col, const float (&acc)[N], const float (&acc1)[N],
                                           const Saved<EPI, N>& kept) {
  float o[N], du[N], h[N];
  dense_values<EPI, N>(p, row, col, true, acc, acc1, kept, o, du, h);
  auto store = [&](__nv_bfloat16* base, const float (&v)[N]) {
    __nv_bfloat16* dst = base + (int64_t)row * p.N + col;
    if constexpr (N == 16) {
      reinterpret_cast<uint4*>(dst)[0] = pack8(v);
      reinterpret_cast<uint4*>(dst)[1] = pack8(v + 8);
    } else {
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    }
  };
  store(p.out, o);
  if constexpr (EPI == kDenseGateGrad) {
    store(p.out_du, du);
    store(p.out_h, h);
  }
}
// Sums of a tile in shared memory, [row][column]: floats of a row, so that eight lanes' 16-byte accesses fall into different banks
template <int COLUMNS>
constexpr int kSumsPitch = COLUMNS + 4;
// Share `share` of S of a tile whose sums lie in the shared memory of S CTAs (ranks first, first + STEP, ...): four columns of a row
// at a time, added in rank order.  A warp covers one row, or eight rows of four quads where the saved projections are written too.
// (All S loads of an element are on their way at once; more elements a thread cost the registers that the second CTA of an SM needs:
// four of them 2048 x 2816, 128 tokens 23.2 -> 29.5 us.)
template <int EPI, int BN, int S, int STEP>
__device__ __forceinline__ void add_parts(const DenseProblem& p, int m0, int n0, int rows, int cols, uint32_t part, int share, int first) {
  constexpr int N_OUT = EPI == kDenseSwiGLU ? BN / 2 : BN;
  constexpr int kHalves = EPI == kDenseSwiGLU ? 2 : 1;
  const bool by_quads = EPI == kDenseGateGrad || (EPI == kDenseSwiGLU && p.gate != nullptr);
  const int quads = cols / 4;
  const int row_groups = (rows + 7) / 8;
  const int total = by_quads ? row_groups * ((quads + 3) / 4) * 32 : rows * quads;
  const int begin = total * share / S, end = total * (share + 1) / S;
#pragma unroll 1
  for (int i = begin + (int)threadIdx.x; i < end; i += (int)blockDim.x) {
    int row, col;
    if (by_quads) {
      const int w = i >> 5, l = i & 31, g = w / row_groups;
      row = (w - g * row_groups) * 8 + (l & 7);
      col = 4 * (4 * g + (l >> 3));
      if (row >= rows || col >= cols) continue;
    } else {
      row = i / quads;
      col = 4 * (i - row * quads);
    }
    const uint32_t from = part + (row * kSumsPitch<BN> + col) * 4;
    Saved<EPI, 4> kept;
    kept.load(p, m0 + row, n0 + col, true);
    float4 v[kHalves][S];
#pragma unroll
    for (int q = 0; q < S; ++q)
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
        v[h][q] = q == share ? ld_shared_f32x4(from + h * N_OUT * 4) : ld_cluster_f32x4(from + h * N_OUT * 4, first + STEP * q);
    float acc[2][4] = {};
#pragma unroll
    for (int q = 0; q < S; ++q)
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        acc[h][0] += v[h][q].x, acc[h][1] += v[h][q].y;
        acc[h][2] += v[h][q].z, acc[h][3] += v[h][q].w;
      }
    dense_emit<EPI, 4>(p, m0 + row, n0 + col, acc[0], acc[1], kept);
  }
}
}  // namespace tc
#endif

}  // namespace atenia
