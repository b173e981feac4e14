// qmm.cu -- the linear operator (nsq_linear) and the mixture-of-experts layer
// (nsq_moe_ffn, nsq_moe_layer): preparation kernel, launch planning, checks.
#include <cudaTypedefs.h>

#include <mutex>

#include "qmm.cuh"

namespace nsq {

int launch_qmm_q4k(int layout, const QmmParams& p, const CUtensorMap* maps, int grid, size_t smem, cudaStream_t st);
int launch_qmm_q5k(int layout, const QmmParams& p, const CUtensorMap* maps, int grid, size_t smem, cudaStream_t st);
int launch_qmm_q6k(int layout, const QmmParams& p, const CUtensorMap* maps, int grid, size_t smem, cudaStream_t st);
int launch_qmm_q40(int layout, const QmmParams& p, const CUtensorMap* maps, int grid, size_t smem, cudaStream_t st);
int launch_qmm_q80(int layout, const QmmParams& p, const CUtensorMap* maps, int grid, size_t smem, cudaStream_t st);
int check_weights(const void* w, int type, int layout, int64_t K);
int device_check(int* num_sms);
int run_gemm_epi(const uint8_t* w, int type, int layout, const void* x, const float* bias, int act, const void* residual,
                 void* y, int64_t M, int64_t N, int64_t K, cudaStream_t st, int num_sms);

constexpr int kPrepThreads = 32 * kQmmWarps;
constexpr int kRouteTok = 8;  // tokens of one CTA's logits
constexpr int kQmmMaxCtas = 320;  // of a product: two per SM
constexpr int kOwnRecords = 8;   // records that a CTA of nsq_linear's product makes itself
constexpr size_t kTicketBytes = (size_t)kQmmMaxCtas * kQmmWarps * 4;

// Activation records of rows x nsb units, one warp each.
template <typename T>
__device__ __forceinline__ void make_records(const T* __restrict__ x, int64_t rows, int64_t K, int nsb, int order,
                                             uint8_t* __restrict__ recs, int64_t block) {
  const int64_t job = block * kQmmWarps + (threadIdx.x >> 5);
  if (job >= rows * nsb) return;
  const int64_t row = job / nsb;
  const int sb = (int)(job - row * nsb);
  qmm_make_record(x + row * K + 256 * sb, (int)min((int64_t)256, K - 256 * sb), order, recs + job * kQmmRec,
                  threadIdx.x & 31);
}

template <typename T>
__global__ void __launch_bounds__(kPrepThreads) qmm_prep_kernel(const T* __restrict__ x, int64_t rows, int64_t K,
                                                                int nsb, int order, uint8_t* __restrict__ recs,
                                                                int32_t* __restrict__ tickets) {
  qmm_dep_wait();
  qmm_dep_launch();
  for (int i = blockIdx.x * kPrepThreads + threadIdx.x; i < (int)(kTicketBytes / 4); i += gridDim.x * kPrepThreads) tickets[i] = 0;
  make_records(x, rows, K, nsb, order, recs, blockIdx.x);
}

__device__ __forceinline__ float4 load4(const float* p, bool wide) {
  return wide ? *reinterpret_cast<const float4*>(p) : make_float4(p[0], p[1], p[2], p[3]);
}

// First kernel of a mixture-of-experts call: the first nlog CTAs compute the
// router's logits (one expert, eight tokens each), the others the activation
// records; they also zero the counters of the products.  With given picks the first CTA
// lists them by expert.  Two experts' logits may lie arbitrarily close, and a
// pick that flips changes the output by whole experts: products of f32 are
// exact in f64, and the sums are f64.
__global__ void __launch_bounds__(kPrepThreads) moe_logits_kernel(const __grid_constant__ QmmParams p,
                                                                  const float* __restrict__ x,
                                                                  const float* __restrict__ router, int64_t K, int order,
                                                                  uint8_t* __restrict__ recs, double* __restrict__ logits,
                                                                  int nlog) {
  extern __shared__ __align__(16) int32_t route_mem[];
  __shared__ double part[kQmmWarps][kRouteTok];
  qmm_dep_wait();
  qmm_dep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((int)blockIdx.x >= nlog) {
    make_records(x, p.M, K, p.nsb, order, recs, blockIdx.x - nlog);
    const int64_t counters = (int64_t)p.M * p.top_k * ((p.n + 255) / 256);
    for (int64_t i = (int64_t)(blockIdx.x - nlog) * kPrepThreads + threadIdx.x; i < counters;
         i += (int64_t)(gridDim.x - nlog) * kPrepThreads)
      p.done[i] = 0;
    for (int i = (blockIdx.x - nlog) * kPrepThreads + threadIdx.x; i < (int)(2 * kTicketBytes / 4);
         i += (gridDim.x - nlog) * kPrepThreads)
      p.tickets[i] = 0;
    return;
  }
  if (!router) {
    qmm_build_lists(p, route_mem);
    return;
  }
  const int e = blockIdx.x % p.E, m0 = (int)blockIdx.x / p.E * kRouteTok;
  const int mc = min(kRouteTok, p.M - m0);
  const float* w = router + (int64_t)e * K;
  const bool wide = ((reinterpret_cast<uintptr_t>(router) | reinterpret_cast<uintptr_t>(x)) & 15) == 0;  // K % 32 == 0
  double acc[kRouteTok] = {};
  // four 16-byte loads of the row are in flight
  for (int64_t k0 = 4 * threadIdx.x; k0 < K; k0 += 4 * 4 * kPrepThreads) {
    float4 a[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t k = k0 + 4 * kPrepThreads * q;
      a[q] = k < K ? load4(w + k, wide) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll
    for (int t = 0; t < kRouteTok; ++t) {
      if (t < mc) {
        float4 b[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t k = k0 + 4 * kPrepThreads * q;
          b[q] = k < K ? load4(x + (int64_t)(m0 + t) * K + k, wide) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
          acc[t] = fma((double)a[q].x, (double)b[q].x,
                       fma((double)a[q].y, (double)b[q].y,
                           fma((double)a[q].z, (double)b[q].z, fma((double)a[q].w, (double)b[q].w, acc[t]))));
      }
    }
  }
#pragma unroll
  for (int t = 0; t < kRouteTok; ++t) {
    if (t < mc) {
      double v = acc[t];
#pragma unroll
      for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) part[warp][t] = v;
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < mc) {
    double v = 0.0;
    for (int i = 0; i < kQmmWarps; ++i) v += part[i][threadIdx.x];
    logits[(int64_t)(m0 + threadIdx.x) * p.E + e] = v;
  }
}

// One CTA picks the experts from the logits and lists the picks by expert.
__global__ void __launch_bounds__(512) moe_lists_kernel(const __grid_constant__ QmmParams p) {
  extern __shared__ __align__(16) int32_t route_mem[];
  qmm_dep_wait();
  qmm_dep_launch();
  qmm_build_lists(p, route_mem);
}

template <typename... Params, typename... Args>
static int launch_pdl(void (*kern)(Params...), int64_t grid, int threads, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  note_launch();
  return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? NSQ_OK : NSQ_ERR_CUDA;
}

template <typename T>
static int launch_prep(const T* x, int64_t rows, int64_t K, int order, uint8_t* recs, int32_t* tickets, cudaStream_t st) {
  const int nsb = (int)((K + 255) / 256);
  return launch_pdl(qmm_prep_kernel<T>, (rows * nsb + kQmmWarps - 1) / kQmmWarps, kPrepThreads, 0, st, x, rows, K, nsb,
                    order, recs, tickets);
}

static int launch_route(const QmmParams& p, const float* x, const float* router, int64_t K, int order, uint8_t* recs,
                        double* logits, cudaStream_t st) {
  const size_t lists = ((size_t)3 * p.M * p.top_k + p.E) * 4;  // at most 14 KB
  const int nlog = router ? p.E * ((p.M + kRouteTok - 1) / kRouteTok) : 1;
  const int64_t rec_ctas = ((int64_t)p.M * p.nsb + kQmmWarps - 1) / kQmmWarps;
  const int rc = launch_pdl(moe_logits_kernel, nlog + rec_ctas, kPrepThreads, router ? 0 : lists, st, p, x, router, K,
                            order, recs, logits, nlog);
  if (rc || !router) return rc;
  return launch_pdl(moe_lists_kernel, 1, 512, lists, st, p);
}

struct QmmShape {
  int CB, PA, PG, MT;
};
template <int TYPE>
static constexpr QmmShape shape_t(int TS) {
  return {QmmFmt<TYPE>::CB, QmmFmt<TYPE>::PA, QmmFmt<TYPE>::PG, qmm_tiles<TYPE>(TS)};
}
static QmmShape qmm_shape(int type, int TS) {
  switch (type) {
    case NSQ_TYPE_Q4_K: return shape_t<NSQ_TYPE_Q4_K>(TS);
    case NSQ_TYPE_Q5_K: return shape_t<NSQ_TYPE_Q5_K>(TS);
    case NSQ_TYPE_Q6_K: return shape_t<NSQ_TYPE_Q6_K>(TS);
    case NSQ_TYPE_Q4_0: return shape_t<NSQ_TYPE_Q4_0>(TS);
    default: return shape_t<NSQ_TYPE_Q8_0>(TS);
  }
}

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static std::once_flag once;
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// Rows of weights as [rows x rb / 2] 16-bit elements, boxes of box_rows x pitch bytes.
static bool encode_rows(CUtensorMap* map, const uint8_t* w, int64_t rows, int64_t rb, int box_rows, int pitch) {
  auto enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[2] = {(cuuint64_t)(rb / 2), (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)rb};
  cuuint32_t box[2] = {(cuuint32_t)(pitch / 2), (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<uint8_t*>(w), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Plans and launches one product.  groups: the most groups there can be.
struct QmmPlan {
  size_t smem;
  int64_t grid;
};
static int plan_qmm(QmmParams& p, int type, int64_t groups, int num_sms, QmmPlan* plan) {
  const QmmShape f = qmm_shape(type, p.TS);
  const int64_t most_units = p.mode == kQmmDown ? groups * p.nsb : p.nsb;
  const int64_t slots = 2 * (int64_t)num_sms < kQmmMaxCtas ? 2 * (int64_t)num_sms : kQmmMaxCtas;
  const int P = p.mode == kQmmLinear ? 0 : p.M * p.top_k;
  const size_t fixed = kQmmCtl + (P ? qmm_lists_bytes(P, p.E, p.TS) : 0);
  const size_t ys = (size_t)kQmmWarps * p.YC * 16 * f.MT * 4;
  const int pitch = p.rb % 16 == 0 ? f.PA : f.PG;
  // Columns of K per CTA (KW), the rest of the 8 warps being row tiles, and
  // whether tasks are divided: the choice with the least time by a simple
  // model.  A CTA's time is its steps x (the bytes of its rows, and a third of
  // those of the records that its row tiles share, which come from L2), and
  // about three steps to put divided tasks together; each doubling of KW costs
  // 5% for the sums of its columns (1 token, two experts of [14336 x 4096]:
  // KW = 1 61 us, KW = 8 with an eighth fewer steps 69 us).
  double best = 0;
  size_t smem = 0;
  int64_t grid = 0;
  for (int KW = 1; KW <= kQmmWarps; KW *= 2) {
    if (KW > 1 && KW / 2 >= most_units) break;
    QmmParams t = p;
    t.KW = KW;
    t.RW = kQmmWarps / KW;
    const size_t slot = qmm_slot_bytes(t.RW * f.MT, pitch, p.TS);
    // two buffers of partial sums let a task's be joined while the next runs
    t.PB = KW > 1 && fixed + 2 * ys + 2 * KW * slot <= (size_t)kQmmSmemHalf ? 2 : 1;
    t.stages = kQmmMaxStages;
    while (t.stages > 2 && fixed + t.PB * ys + t.stages * KW * slot > (size_t)kQmmSmemHalf) --t.stages;
    const size_t need = fixed + t.PB * ys + t.stages * KW * slot;
    if (need > (size_t)kQmmSmemMax) continue;
    if (KW > 1 && KW / 2 < tune(kTuneQmmKW, 0)) smem = 0;  // fewer columns than asked for: only where more do not fit
    const int64_t here = need > (size_t)kQmmSmemHalf ? slots / 2 : slots;  // CTAs at a time
    const int64_t rows = (int64_t)(p.mode == kQmmUp ? 8 : 16) * f.MT * t.RW;
    // (an expert's share of the picks usually is one group)
    const int64_t tasks = (p.n + rows - 1) / rows * (p.mode == kQmmUp ? (groups < p.E ? groups : p.E) : 1);
    const int64_t units = p.mode == kQmmDown ? (groups < p.E ? groups : p.E) * p.nsb : p.nsb;
    const int64_t st = (units + KW - 1) / KW;
    const int columns = KW == 1 ? 0 : KW == 2 ? 1 : KW == 4 ? 2 : 3;
    const double bytes = KW * (16.0 * f.MT * t.RW * pitch + 0.3 * (p.TS < 4 ? p.TS : 0.5 * p.TS) * kQmmRec) / here;
    for (int whole = 1; whole >= 0; --whole) {
      const int only = tune(kTuneQmmSplit, -1);
      if (only >= 0 && whole == (only > 0)) continue;
      const int64_t steps = whole ? (tasks + here - 1) / here * st : (tasks * st + here - 1) / here + 3;
      const double time = steps * bytes * (1.0 + 0.05 * columns);
      if (smem == 0 || time < best) {
        best = time;
        smem = need;
        p.KW = t.KW;
        p.RW = t.RW;
        p.PB = t.PB;
        p.stages = t.stages;
        p.whole = whole;
        grid = here;
        if (whole && p.mode != kQmmUp && tasks < grid) grid = tasks;
        if (!whole && p.mode != kQmmUp && tasks * st < grid) grid = tasks * st;
      }
    }
  }
  if (smem == 0) return NSQ_ERR_SHAPE;
  *plan = QmmPlan{smem, grid};
  return NSQ_OK;
}

static int launch_qmm(QmmParams& p, const QmmPlan& plan, int type, int layout, cudaStream_t st) {
  const QmmShape f = qmm_shape(type, p.TS);
  const size_t smem = plan.smem;
  const int64_t grid = plan.grid;
  // TMA boxes where every row starts 16-byte aligned (experts and tensors then do too)
  alignas(64) CUtensorMap maps[2] = {};
  const int64_t rows = p.wbytes / p.rb;
  p.rows_aligned = p.rb % 16 == 0;
  if (p.rows_aligned) {
    if (rows > 0x7FFFFFFF) return NSQ_ERR_SHAPE;
    const int box_rows = f.MT * (p.mode == kQmmUp ? 8 : 16);
    if (!encode_rows(&maps[0], p.w0, rows, p.rb, box_rows, f.PA)) return NSQ_ERR_CUDA;
    if (p.mode == kQmmUp && !encode_rows(&maps[1], p.w1, rows, p.rb, box_rows, f.PA)) return NSQ_ERR_CUDA;
  }
  switch (type) {
    case NSQ_TYPE_Q4_K: return launch_qmm_q4k(layout, p, maps, (int)grid, smem, st);
    case NSQ_TYPE_Q5_K: return launch_qmm_q5k(layout, p, maps, (int)grid, smem, st);
    case NSQ_TYPE_Q6_K: return launch_qmm_q6k(layout, p, maps, (int)grid, smem, st);
    case NSQ_TYPE_Q4_0: return launch_qmm_q40(layout, p, maps, (int)grid, smem, st);
    case NSQ_TYPE_Q8_0: return launch_qmm_q80(layout, p, maps, (int)grid, smem, st);
    default: return NSQ_ERR_TYPE;
  }
}

static int run_qmm(QmmParams p, int type, int layout, int64_t groups, cudaStream_t st, int num_sms) {
  QmmPlan plan{};
  const int rc = plan_qmm(p, type, groups, num_sms, &plan);
  return rc ? rc : launch_qmm(p, plan, type, layout, st);
}

static int64_t units_of(int64_t K) { return (K + 255) / 256; }
// Workspace of divided tasks: two parts of up to 8 row tiles per CTA, tickets.
static size_t parts_bytes(int64_t tokens, int64_t TS) {
  return (size_t)kQmmMaxCtas * 2 * kQmmWarps * (TS > 8 ? 16 : 32) * tokens * 4;
}
// Whether two ranges of memory share a byte (NULL shares none).
static bool overlap(const void* a, size_t an, const void* b, size_t bn) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x && y && x < y + bn && y < x + an;
}
static bool act_ok(int act) { return act >= NSQ_ACT_NONE && act <= NSQ_ACT_RELU; }

// Workspace of a mixture-of-experts call, in this order.
struct MoeSpace {
  size_t logits, recs_x, h, recs_h, groups, plist, pwts, ptok, ngroups, done, tickets, parts, total;
};
// Tokens of a group: 16, or 8 where an expert has 4 or fewer on average.
static int64_t moe_group(int64_t E, int64_t M, int64_t top_k) {
  const int64_t cap = M * top_k <= 4 * E ? 8 : kQmmMaxTok;
  return M < cap ? M : cap;
}
static MoeSpace moe_space(int64_t E, int64_t D, int64_t F, int64_t M, int64_t top_k) {
  MoeSpace s{};
  const int64_t P = M * top_k;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~size_t(255);
    return here;
  };
  s.logits = take((size_t)(M * E) * 8);
  s.recs_x = take((size_t)(M * units_of(D)) * kQmmRec);
  s.h = take((size_t)(P * F) * 4);
  s.recs_h = take((size_t)(P * units_of(F)) * kQmmRec);
  s.groups = take((size_t)P * sizeof(QmmGroup));
  s.plist = take((size_t)P * 4);
  s.pwts = take((size_t)P * 4);
  s.ptok = take((size_t)P * 4);
  s.ngroups = take(4);
  s.done = take((size_t)(P * units_of(F)) * 4);
  s.tickets = take(2 * kTicketBytes);  // of both products
  // never less than a smaller call's: one of few tokens or picks may have
  // groups of 8, whose row tiles are twice as high as those of 9 to 16
  const int64_t of8 = 4 * E > 8 ? 4 * E : 8;  // tokens that have, with one pick
  const size_t parts = parts_bytes(M, moe_group(E, M, top_k)), parts8 = parts_bytes(M < of8 ? M : of8, 8);
  s.parts = take(parts > parts8 ? parts : parts8);
  s.total = at;
  return s;
}

static int check_moe(const nsq_moe* moe, int64_t M, int64_t top_k) {
  if (!moe) return NSQ_ERR_NULL;
  if (moe->n_expert < 1 || moe->n_expert > NSQ_MOE_MAX_EXPERTS || moe->n_embd < 1 || moe->n_ff < 1) return NSQ_ERR_SHAPE;
  if (moe->n_embd > (1 << 20) || moe->n_ff > (1 << 20)) return NSQ_ERR_SHAPE;
  if (M < 1 || M > NSQ_MOE_MAX_TOKENS || top_k < 1 || top_k > NSQ_MOE_MAX_TOP_K || top_k > moe->n_expert)
    return NSQ_ERR_SHAPE;
  if (!act_ok(moe->act)) return NSQ_ERR_TYPE;
  int rc;
  if ((rc = check_weights(moe->w_gate, moe->type_in, moe->layout_in, moe->n_embd))) return rc;
  if ((rc = check_weights(moe->w_up, moe->type_in, moe->layout_in, moe->n_embd))) return rc;
  return check_weights(moe->w_down, moe->type_down, moe->layout_down, moe->n_ff);
}

// Both entry points: the router's part is left out when w_router is NULL.
static int run_moe(const nsq_moe* moe, const float* w_router, int score, const float* sel_bias, float scale,
                   const float* x, const float* residual, float* y, int32_t* ids, float* weights, int64_t M,
                   int64_t top_k, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_moe(moe, M, top_k);
  if (rc) return rc;
  if (!x || !y || !ids || !weights) return NSQ_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(residual) |
       reinterpret_cast<uintptr_t>(ids) | reinterpret_cast<uintptr_t>(weights) |
       reinterpret_cast<uintptr_t>(w_router) | reinterpret_cast<uintptr_t>(sel_bias)) & 3)
    return NSQ_ERR_ALIGN;
  const int64_t E = moe->n_expert, D = moe->n_embd, F = moe->n_ff;
  const MoeSpace s = moe_space(E, D, F, M, top_k);
  if (!workspace || workspace_bytes < s.total) return NSQ_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return NSQ_ERR_ALIGN;
  // What the call writes (y, the workspace, the router's picks) lies apart from
  // what it reads and from one another; but y may lie on x, which the first
  // kernel alone reads, and on residual, element on element.
  const size_t xb = (size_t)(M * D) * 4, pb = (size_t)(M * top_k) * 4;
  struct Range {
    const void* at;
    size_t bytes;
  };
  const Range ws_r{workspace, s.total}, y_r{y, xb}, ids_r{ids, pb}, wts_r{weights, pb}, x_r{x, xb}, res_r{residual, xb};
  const Range only_read[] = {
      {w_router, (size_t)(E * D) * 4},
      {sel_bias, (size_t)E * 4},
      {moe->w_gate, (size_t)(E * F * (D / nsq_block_weights(moe->type_in)) * nsq_block_bytes(moe->type_in))},
      {moe->w_up, (size_t)(E * F * (D / nsq_block_weights(moe->type_in)) * nsq_block_bytes(moe->type_in))},
      {moe->w_down, (size_t)(E * D * (F / nsq_block_weights(moe->type_down)) * nsq_block_bytes(moe->type_down))}};
  auto meet = [](const Range& a, const Range& b) { return overlap(a.at, a.bytes, b.at, b.bytes); };
  for (const Range& r : only_read) {
    if (meet(r, ws_r) || meet(r, y_r) || (w_router && (meet(r, ids_r) || meet(r, wts_r)))) return NSQ_ERR_SHAPE;
  }
  for (const Range& r : {x_r, res_r}) {
    if (meet(r, ws_r) || (w_router && (meet(r, ids_r) || meet(r, wts_r)))) return NSQ_ERR_SHAPE;
  }
  if ((residual != y && meet(res_r, y_r)) || meet(ids_r, wts_r) || meet(y_r, ids_r) || meet(y_r, wts_r) ||
      meet(ws_r, y_r) || meet(ws_r, ids_r) || meet(ws_r, wts_r))
    return NSQ_ERR_SHAPE;
  int num_sms = 0;
  if ((rc = device_check(&num_sms))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  double* logits = reinterpret_cast<double*>(ws + s.logits);
  QmmParams p{};
  p.M = (int)M;
  p.top_k = (int)top_k;
  p.TS = (int)moe_group(E, M, top_k);
  p.parts = reinterpret_cast<float*>(ws + s.parts);
  p.tickets = reinterpret_cast<int32_t*>(ws + s.tickets);
  p.E = (int)E;
  p.score = w_router ? score : -1;
  p.logits = logits;
  p.sel_bias = sel_bias;
  p.scale = scale;
  p.ids = ids;
  p.wts = weights;
  p.groups = reinterpret_cast<QmmGroup*>(ws + s.groups);
  p.plist = reinterpret_cast<int32_t*>(ws + s.plist);
  p.pwts = reinterpret_cast<float*>(ws + s.pwts);
  p.ptok = reinterpret_cast<int32_t*>(ws + s.ptok);
  p.ngroups = reinterpret_cast<int32_t*>(ws + s.ngroups);
  p.act = moe->act;
  p.dtype = NSQ_OUT_F32;
  p.h = reinterpret_cast<float*>(ws + s.h);
  p.recs_h = ws + s.recs_h;
  p.done = reinterpret_cast<int32_t*>(ws + s.done);
  p.order_h = qmm_order(moe->type_down, moe->layout_down);
  const int64_t P = M * top_k;

  p.mode = kQmmUp;
  p.YC = p.TS;
  p.n = F;
  p.K = D;
  p.nsb = (int)units_of(D);
  p.nblk = (int)(D / 32);
  p.rb = D / nsq_block_weights(moe->type_in) * nsq_block_bytes(moe->type_in);
  p.w0 = static_cast<const uint8_t*>(moe->w_gate);
  p.w1 = static_cast<const uint8_t*>(moe->w_up);
  p.wbytes = E * F * p.rb;
  p.recs = ws + s.recs_x;
  if ((rc = launch_route(p, x, w_router, D, qmm_order(moe->type_in, moe->layout_in), ws + s.recs_x, logits, st)))
    return rc;
  if ((rc = run_qmm(p, moe->type_in, moe->layout_in, P, st, num_sms))) return rc;

  p.mode = kQmmDown;
  p.tickets += kTicketBytes / 4;
  p.YC = p.M;
  p.n = D;
  p.K = F;
  p.nsb = (int)units_of(F);
  p.nblk = (int)(F / 32);
  p.rb = F / nsq_block_weights(moe->type_down) * nsq_block_bytes(moe->type_down);
  p.w0 = static_cast<const uint8_t*>(moe->w_down);
  p.w1 = nullptr;
  p.wbytes = E * D * p.rb;
  p.recs = ws + s.recs_h;
  p.residual = residual;
  p.y = y;
  return run_qmm(p, moe->type_down, moe->layout_down, P, st, num_sms);
}

}  // namespace nsq

using namespace nsq;

extern "C" {

static size_t linear_records(int64_t M, int64_t K) { return ((size_t)(M * units_of(K)) * kQmmRec + 255) & ~size_t(255); }

size_t nsq_linear_workspace_size(int64_t M, int64_t K) {
  if (M < 1 || M > NSQ_GEMV_MAX_M || K < 1) return 0;
  // never less than a smaller call's: 8 tokens have row tiles twice as high as 9 to 15
  const size_t parts = parts_bytes(M, M), of8 = parts_bytes(M < 8 ? M : 8, 8);
  return linear_records(M, K) + kTicketBytes + (parts > of8 ? parts : of8);
}

int nsq_linear(const void* w, int ggml_type, int q6k_layout, const void* x, const float* bias, int act,
               const void* residual, void* y, int dtype, int64_t M, int64_t N, int64_t K, void* workspace,
               size_t workspace_bytes, void* stream) {
  int rc = check_weights(w, ggml_type, q6k_layout, K);
  if (rc) return rc;
  if (!act_ok(act) || (dtype != NSQ_OUT_F32 && dtype != NSQ_OUT_BF16)) return NSQ_ERR_TYPE;
  if (M < 1 || M > (int64_t)1 << 24 || N < 1 || N > (int64_t)1 << 24 || K > (int64_t)1 << 24) return NSQ_ERR_SHAPE;
  const bool prompt = M > NSQ_GEMV_MAX_M;
  if (prompt && (dtype != NSQ_OUT_BF16 || K % 256)) return NSQ_ERR_SHAPE;
  if (!x || !y) return NSQ_ERR_NULL;
  const uintptr_t mask = dtype == NSQ_OUT_F32 ? 3 : 1;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(residual)) & mask)
    return NSQ_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(bias) & 3) return NSQ_ERR_ALIGN;
  const size_t es = dtype == NSQ_OUT_F32 ? 4 : 2, xb = (size_t)(M * K) * es, yb = (size_t)(M * N) * es;
  const bool y_on_x = overlap(x, xb, y, yb);
  const size_t w_bytes = (size_t)(N * (K / nsq_block_weights(ggml_type)) * nsq_block_bytes(ggml_type));
  const bool y_on_others = (residual != y && overlap(residual, yb, y, yb)) || overlap(bias, (size_t)N * 4, y, yb) ||
                           overlap(w, w_bytes, y, yb);
  if (prompt) {
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) return NSQ_ERR_ALIGN;
    if (y_on_x || y_on_others) return NSQ_ERR_SHAPE;
    int sms = 0;
    if ((rc = device_check(&sms))) return rc;
    return run_gemm_epi(static_cast<const uint8_t*>(w), ggml_type, q6k_layout, x, bias, act, residual, y, M, N, K,
                        static_cast<cudaStream_t>(stream), sms);
  }
  if (!workspace || workspace_bytes < nsq_linear_workspace_size(M, K)) return NSQ_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return NSQ_ERR_ALIGN;
  const size_t wb = nsq_linear_workspace_size(M, K);
  if (y_on_others || overlap(workspace, wb, x, xb) || overlap(workspace, wb, y, yb) ||
      overlap(workspace, wb, residual, yb) || overlap(workspace, wb, bias, (size_t)N * 4) ||
      overlap(workspace, wb, w, w_bytes))
    return NSQ_ERR_SHAPE;
  int num_sms = 0;
  if ((rc = device_check(&num_sms))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* recs = static_cast<uint8_t*>(workspace);
  const int order = qmm_order(ggml_type, q6k_layout);
  QmmParams p{};
  p.tickets = reinterpret_cast<int32_t*>(recs + linear_records(M, K));
  p.parts = reinterpret_cast<float*>(recs + linear_records(M, K) + kTicketBytes);
  p.mode = kQmmLinear;
  p.M = p.TS = p.YC = (int)M;
  p.top_k = 1;
  p.act = act;
  p.dtype = dtype;
  p.n = N;
  p.K = K;
  p.nsb = (int)units_of(K);
  p.nblk = (int)(K / 32);
  p.rb = K / nsq_block_weights(ggml_type) * nsq_block_bytes(ggml_type);
  p.w0 = static_cast<const uint8_t*>(w);
  p.wbytes = N * p.rb;
  p.recs = recs;
  p.bias = bias;
  p.residual = residual;
  p.y = y;
  QmmPlan plan{};
  if ((rc = plan_qmm(p, ggml_type, 1, num_sms, &plan))) return rc;
  // One record per warp at most: every CTA makes them itself, which takes less
  // than a kernel before it (1 token, Q8_0 1152 x 896: 5.5 against 6.7 us, and
  // 2.4 us less on the host; two per warp, Q4_K 4096 x 4096: 8.1 against 7.8).
  // Divided tasks need that kernel for their tickets, and an output over x
  // needs every record made before it.
  const size_t own = (size_t)p.nsb * qmm_recs_bytes(p.TS);
  if (p.whole && !y_on_x && M * p.nsb <= kOwnRecords &&
      plan.smem + own <= (size_t)(plan.smem <= (size_t)kQmmSmemHalf ? kQmmSmemHalf : kQmmSmemMax)) {
    p.x = x;
    p.order = order;
    plan.smem += own;
  } else {
    rc = dtype == NSQ_OUT_F32
             ? launch_prep(static_cast<const float*>(x), M, K, order, recs, p.tickets, st)
             : launch_prep(static_cast<const __nv_bfloat16*>(x), M, K, order, recs, p.tickets, st);
    if (rc) return rc;
  }
  return launch_qmm(p, plan, ggml_type, q6k_layout, st);
}

size_t nsq_moe_workspace_size(const nsq_moe* moe, int64_t M, int64_t top_k) {
  if (!moe || moe->n_expert < 1 || moe->n_embd < 1 || moe->n_ff < 1 || M < 1 || M > NSQ_MOE_MAX_TOKENS || top_k < 1 ||
      top_k > NSQ_MOE_MAX_TOP_K)
    return 0;
  return moe_space(moe->n_expert, moe->n_embd, moe->n_ff, M, top_k).total;
}

int nsq_moe_ffn(const nsq_moe* moe, const float* x, const int32_t* ids, const float* weights, const float* residual,
                float* y, int64_t M, int64_t top_k, void* workspace, size_t workspace_bytes, void* stream) {
  return run_moe(moe, nullptr, 0, nullptr, 1.0f, x, residual, y, const_cast<int32_t*>(ids), const_cast<float*>(weights),
                 M, top_k, workspace, workspace_bytes, stream);
}

int nsq_moe_layer(const nsq_moe* moe, const float* w_router, int score, const float* sel_bias, float scale,
                  const float* x, const float* residual, float* y, int32_t* ids, float* weights, int64_t M,
                  int64_t top_k, void* workspace, size_t workspace_bytes, void* stream) {
  if (!w_router) return NSQ_ERR_NULL;
  if (score < NSQ_SCORE_SOFTMAX || score > NSQ_SCORE_SIGMOID_NORM) return NSQ_ERR_TYPE;
  return run_moe(moe, w_router, score, sel_bias, scale, x, residual, y, ids, weights, M, top_k, workspace,
                 workspace_bytes, stream);
}

}  // extern "C"
