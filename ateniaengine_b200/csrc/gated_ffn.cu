// Entry points of the dense gated feed-forward block, its backward pass and the low-rank adapters, and their host side.
//
//   forward   g = x Wg^T, u = x Wu^T, h = silu(g) u (one kernel); y = h Wd^T
//   backward  dh = dy Wd, from it with the saved g and u: dg, du and h again (one kernel);
//             dx = dg Wg + du Wu (one reduction of 2 d_ff); dWg = dg^T x, dWu = du^T x, dWd = dy^T h (one launch)
//   adapters  v = scale A x of the rows' own adapters, then their B v inside the projection's kernel
//
// The calls keep no state: the caller passes the workspace, so that two calls, streams or captured graphs share nothing but
// what the caller lets them share.  g and u are saved in f32 (8 bytes per token and feature): rounded to bf16 they would
// add as much to the gradients' error as the two roundings that the operands of the second products need anyway.
#include <mutex>

#include "dense_gemm.cuh"
#include "error_word.cuh"

namespace atenia {

namespace {

static __device__ DeviceError g_dense_error;
static __device__ DeviceError g_taken_error;  // by a check
std::mutex g_mu, g_check_mu[kMaxDevices];
DeviceError* g_error_addr[kMaxDevices] = {};
int g_sms[kMaxDevices] = {};

int num_sms_of_current_device(int* out) {
  int dev = -1;
  ATENIA_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return ATENIA_ERR_UNSUPPORTED;
  std::lock_guard<std::mutex> lk(g_mu);
  if (!g_sms[dev]) ATENIA_CUDA_TRY(cudaDeviceGetAttribute(&g_sms[dev], cudaDevAttrMultiProcessorCount, dev));
  *out = g_sms[dev];
  return ATENIA_OK;
}

constexpr int64_t kMaxRows = 1 << 24, kMaxWidth = 1 << 20;
constexpr int kMaxAdapters = ATENIA_ADAPTER_MAX_COUNT;

uint64_t align256(uint64_t v) { return (v + 255) / 256 * 256; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
struct Range {
  const void* p;  // (null: none)
  uint64_t bytes;
};
bool overlap(const Range& a, const Range& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
  return a.p && b.p && x < y + b.bytes && y < x + a.bytes;
}
// Does an output lie over an input or over another output?
template <int O, int I>
bool overlap_any(const Range (&outs)[O], const Range (&ins)[I]) {
  for (int i = 0; i < O; ++i) {
    for (const Range& in : ins)
      if (overlap(outs[i], in)) return true;
    for (int j = 0; j < i; ++j)
      if (overlap(outs[i], outs[j])) return true;
  }
  return false;
}
int kblocks(int64_t k) { return (int)((k + tc::BK - 1) / tc::BK); }

// [rows, cols] row-major in boxes of `box_rows` rows x 64 columns
int matrix_map(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int box_rows) {
  return encode_tmap_bf16(m, base, {(uint64_t)cols, (uint64_t)rows, 0}, {64, (uint32_t)box_rows, 1}, 128);
}

// Does dense_rows.cu serve the product?  Its kernel reads through plain pointers and needs no maps.
bool reads_plainly(const DenseProblem& p, const void* a, const void* b0, const void* b1) {
  return dense_rows(p.M, p.N, p.K, b1 != nullptr, a, b0, b1);
}

// A [M, K] and B [N, K] of a product without transposed operands: their maps and plain pointers
int set_operands(DenseProblem* p, const void* a, const void* b0, const void* b1, int a_rows) {
  p->a_ptr = static_cast<const __nv_bfloat16*>(a);
  p->b_ptr[0] = static_cast<const __nv_bfloat16*>(b0);
  p->b_ptr[1] = static_cast<const __nv_bfloat16*>(b1);
  p->kb = p->kb0 = kblocks(p->K);
  if (reads_plainly(*p, a, b0, b1)) return ATENIA_OK;
  int rc = matrix_map(&p->a[0], a, p->M, p->K, a_rows);
  if (!rc) rc = matrix_map(&p->b[0], b0, p->N, p->K, 64);
  if (!rc && b1) rc = matrix_map(&p->b[1], b1, p->N, p->K, 64);
  return rc;
}

// h of a call's tokens; of a few it may come in two parts (dense_rows.cu)
uint64_t h_bytes(int64_t T, int64_t d_ff) { return align256((uint64_t)T * d_ff * (T <= kRestMost ? 4 : 2)); }

bool rank_ok(int r) { return r >= 8 && r <= kAdapterMaxRank && r % 8 == 0; }
int check_adapter(const AteniaLowRank& a) {
  if (!rank_ok(a.rank)) return ATENIA_ERR_SHAPE;
  if (!a.a || !a.b || !a.scale) return ATENIA_ERR_NULL;
  if (!aligned16(a.a) || !aligned16(a.b) || !aligned4(a.scale)) return ATENIA_ERR_SHAPE;
  return ATENIA_OK;
}
// What a projection's adapters are read from
struct AdapterRanges {
  Range a, b, scale;
  AdapterRanges(const AteniaLowRank* s, int64_t in, int64_t out, int n) : a{}, b{}, scale{} {
    if (!s || s->rank == 0) return;
    a = {s->a, (uint64_t)n * s->rank * in * 2};
    b = {s->b, (uint64_t)n * s->rank * out * 2};
    scale = {s->scale, (uint64_t)n * 4};
  }
};
// (room for two parts: the calls that ask for the size do not all know the width that decides)
uint64_t reduced_bytes(int64_t T, int rank) { return rank > 0 ? align256((uint64_t)T * rank * 4) : 0; }

// One projection's adapters: the first half's projection and the second half's segment, with v at `v`.
int encode_adapter(const AteniaLowRank& a, int64_t T, int64_t in, int64_t out, int n, int a_rows, int parts, bool few_reduce,
                   bool plain, void* v, AdapterReduce::Projection* red, AdapterSegment* seg) {
  const uint64_t r = (uint64_t)a.rank;
  int rc = few_reduce ? ATENIA_OK : encode_tmap_bf16(&red->a, a.a, {(uint64_t)in, r, (uint64_t)n}, {64, (uint32_t)r, 1}, 128);
  const uint32_t width = (uint32_t)adapter_width(a.rank);
  seg->width = (int)width;
  if (!rc && !plain) rc = encode_tmap_bf16(&seg->v, v, {r, (uint64_t)T, (uint64_t)parts}, {width, (uint32_t)a_rows, 1}, 2 * width);
  if (!rc && !plain) rc = encode_tmap_bf16(&seg->b, a.b, {r, (uint64_t)out, (uint64_t)n}, {width, 64, 1}, 2 * width);
  red->scale = a.scale;
  red->v = static_cast<__nv_bfloat16*>(v);
  red->rank = seg->rank = a.rank;
  red->a_ptr = static_cast<const __nv_bfloat16*>(a.a);
  seg->v_ptr = red->v;
  seg->b_ptr = static_cast<const __nv_bfloat16*>(a.b);
  return rc;
}

// The reduced rows of up to two projections of the same input, and what the product (which may read `plain`ly) needs of them.
struct AdapterPlan {
  AdapterReduce red{};
  DenseAdapters add{};
};
int plan_adapters(AdapterPlan* p, const AteniaLowRank* const (&sets)[2], const int32_t* ids, int n, const void* x, int64_t T,
                  int64_t in, int64_t out, bool plain, uint8_t** ws, bool chained) {
  const int a_rows = dense_a_rows(T);
  p->red.ids = p->add.ids = ids;
  p->red.n = p->add.n = n;
  p->red.M = (int)T;
  p->red.K = (int)in;
  p->red.kb = kblocks(in);
  p->red.x_ptr = static_cast<const __nv_bfloat16*>(x);
  p->red.a_rows = a_rows;
  p->red.chained = chained;
  int rank = 0;
  for (const AteniaLowRank* a : sets) rank = a && a->rank > rank ? a->rank : rank;
  p->red.few = adapter_gemv_rows(T, rank, in);
  p->red.parts = p->add.parts = adapter_parts(rank, in);
  int rc = p->red.few ? ATENIA_OK : matrix_map(&p->red.x, x, T, in, a_rows);
  for (int i = 0; i < 2 && !rc; ++i) {
    if (!sets[i] || sets[i]->rank == 0) continue;
    rc = encode_adapter(*sets[i], T, in, out, n, a_rows, p->red.parts, p->red.few, plain, *ws, &p->red.p[p->red.projections], &p->add.seg[i]);
    p->red.projections += 1;
    *ws += reduced_bytes(T, sets[i]->rank);
  }
  return rc;
}

int check_sizes(int64_t T, int64_t d, int64_t f) {
  if (T < 0 || T > kMaxRows || d < 16 || f < 16 || d > kMaxWidth || f > kMaxWidth || d % 16 || f % 16) return ATENIA_ERR_SHAPE;
  return ATENIA_OK;
}

int check_ffn_adapters(const AteniaFfnAdapters* ad) {
  if (!ad->ids) return ATENIA_ERR_NULL;
  if (ad->n < 1 || ad->n > kMaxAdapters || !aligned4(ad->ids)) return ATENIA_ERR_SHAPE;
  const AteniaLowRank* sets[3] = {&ad->gate, &ad->up, &ad->down};
  for (const AteniaLowRank* a : sets) {
    if (a->rank == 0) continue;
    int rc = check_adapter(*a);
    if (rc) return rc;
  }
  return ATENIA_OK;
}

}  // namespace

int dense_error_word(DeviceError** out) {
  int dev = -1;
  ATENIA_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return ATENIA_ERR_UNSUPPORTED;
  std::lock_guard<std::mutex> lk(g_mu);
  if (!g_error_addr[dev]) {
    void* p = nullptr;
    ATENIA_CUDA_TRY(cudaGetSymbolAddress(&p, g_dense_error));
    if (!p) return ATENIA_ERR_DRIVER;
    g_error_addr[dev] = static_cast<DeviceError*>(p);
  }
  *out = g_error_addr[dev];
  return ATENIA_OK;
}

}  // namespace atenia

extern "C" {

uint64_t atenia_gated_ffn_workspace_bytes(int T, int d_model, int d_ff, const AteniaFfnAdapters* adapters, int backward) {
  using namespace atenia;
  if (check_sizes(T, d_model, d_ff)) return 0;
  const uint64_t rows = align256((uint64_t)T * d_ff * 2);
  if (backward) return 3 * rows;  // dg, du, h
  uint64_t n = h_bytes(T, d_ff);
  if (adapters)
    for (const AteniaLowRank* a : {&adapters->gate, &adapters->up, &adapters->down}) {
      if (a->rank != 0 && !rank_ok(a->rank)) return 0;
      n += reduced_bytes(T, a->rank);
    }
  return n;
}

uint64_t atenia_adapter_linear_workspace_bytes(int T, int rank) {
  return T < 0 || T > atenia::kMaxRows || !atenia::rank_ok(rank) ? 0 : atenia::reduced_bytes(T, rank);
}

int atenia_gated_ffn_forward(const void* x, const void* w_gate, const void* w_up, const void* w_down, int T, int d_model, int d_ff,
                             const AteniaFfnAdapters* adapters, void* y, float* saved_gate, float* saved_up, void* workspace,
                             uint64_t workspace_bytes, void* stream) {
  using namespace atenia;
  int rc = check_sizes(T, d_model, d_ff);
  if (rc) return rc;
  if (!w_gate || !w_up || !w_down || !saved_gate != !saved_up) return ATENIA_ERR_NULL;
  if (adapters && (rc = check_ffn_adapters(adapters))) return rc;
  if (T == 0) return ATENIA_OK;
  if (!x || !y || !workspace) return ATENIA_ERR_NULL;
  for (const void* p : {x, w_gate, w_up, w_down, (const void*)y, (const void*)saved_gate, (const void*)saved_up, (const void*)workspace})
    if (!aligned16(p)) return ATENIA_ERR_SHAPE;
  const uint64_t need = atenia_gated_ffn_workspace_bytes(T, d_model, d_ff, adapters, 0);
  if (workspace_bytes < need) return ATENIA_ERR_CAPACITY;
  {
    const uint64_t row = (uint64_t)T * d_model * 2, weight = (uint64_t)d_model * d_ff * 2, kept = (uint64_t)T * d_ff * 4;
    const int n = adapters ? adapters->n : 0;
    const AdapterRanges gate(adapters ? &adapters->gate : nullptr, d_model, d_ff, n), up(adapters ? &adapters->up : nullptr, d_model, d_ff, n),
        down(adapters ? &adapters->down : nullptr, d_ff, d_model, n);
    const Range outs[4] = {{y, row}, {saved_gate, kept}, {saved_up, kept}, {workspace, need}};
    const Range ins[13] = {{w_gate, weight}, {w_up, weight}, {w_down, weight}, gate.a, gate.b, gate.scale, up.a, up.b, up.scale,
                           down.a, down.b, down.scale, {adapters ? adapters->ids : nullptr, (uint64_t)T * 4}};
    if (overlap_any(outs, ins)) return ATENIA_ERR_SHAPE;
    for (int i = 1; i < 4; ++i)  // (y may be x: the products that write it read h)
      if (overlap(outs[i], {x, row})) return ATENIA_ERR_SHAPE;
  }
  int sms = 0;
  if ((rc = num_sms_of_current_device(&sms))) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  __nv_bfloat16* h = reinterpret_cast<__nv_bfloat16*>(ws);
  ws += h_bytes(T, d_ff);
  const int64_t d = d_model, F = d_ff;

  AdapterPlan first, second;
  const bool ad1 = adapters && (adapters->gate.rank || adapters->up.rank), ad2 = adapters && adapters->down.rank;
  DenseGemm g1{};
  g1.problems = 1;
  g1.epilogue = kDenseSwiGLU;
  g1.chained = true;
  g1.a_rows = dense_a_rows(T);
  DenseProblem& p1 = g1.p[0];
  p1.M = T;
  p1.N = d_ff;
  p1.K = d_model;
  p1.out = h;
  p1.gate = saved_gate;
  p1.up = saved_up;
  rc = set_operands(&p1, x, w_gate, w_up, g1.a_rows);
  DenseGemm g2{};
  g2.problems = 1;
  g2.epilogue = kDensePlain;
  g2.a_rows = g1.a_rows;
  g2.chained = g2.b_early = true;
  DenseProblem& p2 = g2.p[0];
  p2.M = T;
  p2.N = d_model;
  p2.K = d_ff;
  p2.out = static_cast<__nv_bfloat16*>(y);
  if (!rc) rc = set_operands(&p2, h, w_down, nullptr, g2.a_rows);
  p1.out_rest = p2.a_rest = T <= kRestMost && reads_plainly(p1, x, w_gate, w_up) && reads_plainly(p2, h, w_down, nullptr);
  if (!rc && ad1) {
    rc = plan_adapters(&first, {&adapters->gate, &adapters->up}, adapters->ids, adapters->n, x, T, d, F, reads_plainly(p1, x, w_gate, w_up), &ws, true);
    g1.adapters = &first.add;
    g1.b_early = g1.a_early = true;  // (only the adapters' rows are the kernel before's)
  }
  if (!rc && ad2) {
    rc = plan_adapters(&second, {&adapters->down, nullptr}, adapters->ids, adapters->n, h, T, F, d, reads_plainly(p2, h, w_down, nullptr), &ws, true);
    g2.adapters = &second.add;
    // (h too: the kernel before is the reduction, whose CTAs let this one start when the one that wrote h had completed)
    g2.a_early = true;
  }
  if (!rc && ad1) rc = launch_adapter_reduce(first.red, sms, s);
  if (!rc) rc = launch_dense_gemm(g1, sms, s);
  if (!rc && ad2) rc = launch_adapter_reduce(second.red, sms, s);
  if (!rc) rc = launch_dense_gemm(g2, sms, s);
  return rc;
}

int atenia_gated_ffn_backward(const void* dy, const void* x, const void* w_gate, const void* w_up, const void* w_down,
                              const float* saved_gate, const float* saved_up, int T, int d_model, int d_ff, void* dx, void* dw_gate,
                              void* dw_up, void* dw_down, void* workspace, uint64_t workspace_bytes, void* stream) {
  using namespace atenia;
  int rc = check_sizes(T, d_model, d_ff);
  if (rc) return rc;
  if (!w_gate || !w_up || !w_down || !dw_gate || !dw_up || !dw_down) return ATENIA_ERR_NULL;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t d = d_model, F = d_ff;
  if (T == 0) {  // sums over no token
    for (void* p : {dw_gate, dw_up, dw_down}) ATENIA_CUDA_TRY(cudaMemsetAsync(p, 0, (size_t)(d * F * 2), s));
    return ATENIA_OK;
  }
  if (!dy || !x || !dx || !saved_gate || !saved_up || !workspace) return ATENIA_ERR_NULL;
  for (const void* p : {dy, x, w_gate, w_up, w_down, (const void*)saved_gate, (const void*)saved_up, (const void*)dx, (const void*)dw_gate,
                        (const void*)dw_up, (const void*)dw_down, (const void*)workspace})
    if (!aligned16(p)) return ATENIA_ERR_SHAPE;
  const uint64_t need = atenia_gated_ffn_workspace_bytes(T, d_model, d_ff, nullptr, 1);
  if (workspace_bytes < need) return ATENIA_ERR_CAPACITY;
  {
    const uint64_t row = (uint64_t)T * d * 2, weight = (uint64_t)d * F * 2, kept = (uint64_t)T * F * 4;
    const Range outs[5] = {{dx, row}, {dw_gate, weight}, {dw_up, weight}, {dw_down, weight}, {workspace, need}};
    const Range ins[7] = {{dy, row}, {x, row}, {w_gate, weight}, {w_up, weight}, {w_down, weight}, {saved_gate, kept}, {saved_up, kept}};
    if (overlap_any(outs, ins)) return ATENIA_ERR_SHAPE;
  }
  int sms = 0;
  if ((rc = num_sms_of_current_device(&sms))) return rc;
  const uint64_t rows = align256((uint64_t)T * F * 2);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  __nv_bfloat16* dg = reinterpret_cast<__nv_bfloat16*>(ws);
  __nv_bfloat16* du = reinterpret_cast<__nv_bfloat16*>(ws + rows);
  __nv_bfloat16* h = reinterpret_cast<__nv_bfloat16*>(ws + 2 * rows);

  DenseGemm g1{};  // dh = dy Wd: the reduction runs over the rows of Wd [d, F]
  g1.problems = 1;
  g1.epilogue = kDenseGateGrad;
  g1.a_rows = dense_a_rows(T);
  g1.chained = true;
  DenseProblem& p1 = g1.p[0];
  p1.M = T;
  p1.N = d_ff;
  p1.b_mn = true;
  p1.kb = p1.kb0 = kblocks(d);
  p1.out = dg;
  p1.out_du = du;
  p1.out_h = h;
  p1.gate = const_cast<float*>(saved_gate);
  p1.up = const_cast<float*>(saved_up);
  rc = matrix_map(&p1.a[0], dy, T, d, g1.a_rows);
  if (!rc) rc = matrix_map(&p1.b[0], w_down, d, F, 64);

  DenseGemm g2{};  // dx = dg Wg + du Wu
  g2.problems = 1;
  g2.epilogue = kDensePlain;
  g2.a_rows = g1.a_rows;
  g2.chained = g2.b_early = true;
  g2.next_early = true;  // (backward pass of 64 tokens, 512 x 1408 17.8 -> 17.0 us, of 1021, 2048 x 5632 132.4 -> 129.4)
  DenseProblem& p2 = g2.p[0];
  p2.M = T;
  p2.N = d_model;
  p2.b_mn = true;
  p2.kb0 = kblocks(F);
  p2.kb = 2 * p2.kb0;
  p2.out = static_cast<__nv_bfloat16*>(dx);
  if (!rc) rc = matrix_map(&p2.a[0], dg, T, F, g2.a_rows);
  if (!rc) rc = matrix_map(&p2.a[1], du, T, F, g2.a_rows);
  if (!rc) rc = matrix_map(&p2.b[0], w_gate, F, d, 64);
  if (!rc) rc = matrix_map(&p2.b[1], w_up, F, d, 64);

  DenseGemm g3{};  // the weights' gradients: reductions over the tokens
  g3.problems = 3;
  g3.epilogue = kDensePlain;
  g3.a_rows = tc::BM;
  g3.chained = g3.b_early = g3.a_early = true;  // (its operands are older than the kernel before it, which waited for them)
  const void* lhs[3] = {dg, du, dy};
  const void* rhs[3] = {x, x, h};
  void* out[3] = {dw_gate, dw_up, dw_down};
  for (int i = 0; i < 3; ++i) {
    DenseProblem& p = g3.p[i];
    p.M = i < 2 ? d_ff : d_model;
    p.N = i < 2 ? d_model : d_ff;
    p.b_mn = true;
    p.kb = p.kb0 = kblocks(T);
    p.out = static_cast<__nv_bfloat16*>(out[i]);
    if (!rc) rc = matrix_map(&p.a[0], lhs[i], T, p.M, 64);
    if (!rc) rc = matrix_map(&p.b[0], rhs[i], T, p.N, 64);
  }
  if (!rc) rc = launch_dense_gemm(g1, sms, s);
  if (!rc) rc = launch_dense_gemm(g2, sms, s);
  if (!rc) rc = launch_dense_gemm(g3, sms, s);
  return rc;
}

int atenia_adapter_linear(const void* x, const void* weight, int T, int d_in, int d_out, const AteniaLowRank* adapter,
                          const int32_t* ids, int n, void* y, void* workspace, uint64_t workspace_bytes, void* stream) {
  using namespace atenia;
  int rc = check_sizes(T, d_in, d_out);
  if (rc) return rc;
  if (!weight || !adapter) return ATENIA_ERR_NULL;
  if (n < 1 || n > kMaxAdapters) return ATENIA_ERR_SHAPE;
  if ((rc = check_adapter(*adapter))) return rc;
  if (T == 0) return ATENIA_OK;
  if (!x || !ids || !y || !workspace) return ATENIA_ERR_NULL;
  for (const void* p : {x, weight, (const void*)y, (const void*)workspace})
    if (!aligned16(p)) return ATENIA_ERR_SHAPE;
  if (!aligned4(ids)) return ATENIA_ERR_SHAPE;
  const uint64_t need = atenia_adapter_linear_workspace_bytes(T, adapter->rank);
  if (workspace_bytes < need) return ATENIA_ERR_CAPACITY;
  {
    const AdapterRanges ad(adapter, d_in, d_out, n);
    const Range outs[2] = {{y, (uint64_t)T * d_out * 2}, {workspace, need}};
    const Range ins[6] = {{x, (uint64_t)T * d_in * 2}, {weight, (uint64_t)d_in * d_out * 2}, ad.a, ad.b, ad.scale, {ids, (uint64_t)T * 4}};
    if (overlap_any(outs, ins)) return ATENIA_ERR_SHAPE;
  }
  int sms = 0;
  if ((rc = num_sms_of_current_device(&sms))) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  AdapterPlan plan;
  DenseGemm g{};
  g.problems = 1;
  g.epilogue = kDensePlain;
  g.a_rows = dense_a_rows(T);
  g.adapters = &plan.add;
  g.chained = g.b_early = g.a_early = true;
  DenseProblem& p = g.p[0];
  p.M = T;
  p.N = d_out;
  p.K = d_in;
  p.out = static_cast<__nv_bfloat16*>(y);
  rc = plan_adapters(&plan, {adapter, nullptr}, ids, n, x, T, d_in, d_out, reads_plainly(p, x, weight, nullptr), &ws, true);
  if (!rc) rc = set_operands(&p, x, weight, nullptr, g.a_rows);
  if (!rc) rc = launch_adapter_reduce(plan.red, sms, s);
  if (!rc) rc = launch_dense_gemm(g, sms, s);
  return rc;
}

int atenia_ffn_check(void* stream) {
  using namespace atenia;
  DeviceError* word = nullptr;
  int rc = dense_error_word(&word);
  if (rc) return rc;
  int dev = -1;
  void* taken = nullptr;
  ATENIA_CUDA_TRY(cudaGetDevice(&dev));
  ATENIA_CUDA_TRY(cudaGetSymbolAddress(&taken, g_taken_error));
  DeviceError e{};
  rc = take_device_error(word, static_cast<DeviceError*>(taken), g_check_mu[dev], static_cast<cudaStream_t>(stream), &e);
  return rc ? rc : e.code;
}

}  // extern "C"
