// qmm.cuh -- products of a few tokens with GGUF-quantised weights, exact to
// about 3e-7 (f32 outputs), for the linear operator and the two products of
// a mixture-of-experts layer.
//
//   out[t, n] = sum_k x[t, k] * W[n, k]         t: up to 16 tokens of a group
//
// Mathematics.  x' = x / s is split into two fp16 numbers hi + lo (22 bits);
// s is one power of two per (token, 256 of K), so that |x'| < 2^15.  mma.sync
// m16n8k16 (fp16 in, f32 out) takes 16 weight rows as A and 4 tokens as B, the
// hi and lo part of a token being two neighbouring columns; every product is
// exact and the sums are f32.  A holds small integers, two per register:
//   Q4_K, Q5_K  q masked out of its word is the fp16 subnormal q * 2^-24 (or
//               q * 2^-20 four bits higher); times sc * 2^10 (2^6) it is
//               q * sc * 2^-14, exact (q * sc <= 1953).  The mins enter once
//               per 256 weights as a second MMA over the sums of 16
//               activations:  d * sum(q sc x) - dmin * sum(m T)
//   Q6_K        (q - 32) * sc does not fit 11 bits: q - 32 as (1024 + q) -
//               1056, one MMA per 16-weight scale group, scaled in f32
//   Q4_0, Q8_0  q - 8 and the int8 likewise, the scale of 32 in f32
// A must be normal numbers: the tensor cores align the products by their
// exponent fields, so a subnormal A (as the masked q itself) costs up to ten
// bits of the sum (1e-5 instead of 3e-7).
//
// What bounds it: HBM for the weights; the unpacking takes about 1.8 issue
// slots per weight (Q4_K), half of an SM's issue rate at HBM speed, so the
// matrix instructions leave room for 4 tokens at the price of one.
//
// Layout.  A CTA is 8 consumer warps = RW row tiles of 16 MT weight rows x KW
// columns, and one producer warp.  A task is a tile of 16 MT RW rows; its
// units of 256 weights of K are dealt to the columns in turn.  A column has
// its own ring of shared-memory slots (the weight bytes of its RW tiles and
// the activation records of the unit) behind full / empty mbarriers, filled by
// TMA: one 2-D box of rows where rows start 16-byte aligned, else one bulk
// copy per row.  The partial sums of the KW columns meet in shared memory,
// those of a K split over a cluster through distributed shared memory, always
// in the same order.  Every wait is bounded.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "nsq_common.cuh"

namespace nsq {

// ---------------------------------------------------------------------------
// Prepared activations: one record per (row, 256 of K).
//   [0, 512)      hi parts: 16-byte unit 4i + c = the operands of MMA steps
//                 2i, 2i+1 of lane c of each quad
//   [512, 1024)   lo parts, unit index ^ 4 (hi and lo of a token are read by
//                 neighbouring lanes: the other half of the banks)
//   [1024, 1088)  T / 32, T = the sums of 16 consecutive x', as hi and lo:
//                 per lane c the four groups 2c, 2c+1, 2c+8, 2c+9
//   [1088, 1092)  s
// Which k a place holds goes by the format of the weights (QmmOrder).
constexpr int kQmmRec = 1104;
constexpr int kQmmWarps = 8;
constexpr int kQmmThreads = 32 * (kQmmWarps + 1);  // and the producer warp
constexpr int kQmmMaxStages = 4;
constexpr int kQmmCtl = 1024;  // barriers and counters at the start of the shared memory
constexpr int kQmmMaxTok = 16;  // tokens of a group
constexpr int kQmmSmemMax = 227 * 1024 - 1024;   // dynamic shared memory of a CTA alone on its SM
constexpr int kQmmSmemHalf = 113 * 1024 - 1024;  // of one of two CTAs

enum QmmOrder : int { kOrdK45 = 0, kOrd32 = 1, kOrdQ6 = 2 };

__host__ __device__ constexpr int qmm_order(int type, int layout) {
  return type == NSQ_TYPE_Q4_K || type == NSQ_TYPE_Q5_K ? kOrdK45
         : type == NSQ_TYPE_Q6_K && layout == NSQ_Q6K_GGML ? kOrdQ6
                                                           : kOrd32;
}
// First k of the two runs of four that unit (i, c) of a record holds.
__device__ __forceinline__ void qmm_runs(int order, int i, int c, int& k0, int& k1) {
  if (order == kOrdK45) {
    k0 = 64 * c + 4 * i;
    k1 = k0 + 32;
  } else if (order == kOrd32) {
    k0 = 32 * i + 4 * c;
    k1 = k0 + 16;
  } else {
    k0 = 128 * (i >> 2) + 64 * (i & 1) + 16 * ((i >> 1) & 1) + 4 * c;
    k1 = k0 + 32;
  }
}

__device__ __forceinline__ uint32_t qmm_h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 qmm_u2h(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ uint32_t qmm_mul2(uint32_t a, __half2 b) { return qmm_h2u(__hmul2(qmm_u2h(a), b)); }

// hi and lo of two values as fp16 pairs.
__device__ __forceinline__ void qmm_split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  hi = qmm_h2u(h);
  lo = qmm_h2u(__floats2half2_rn(a - f.x, b - f.y));
}

// One warp turns 256 values (those at and after `valid` count as 0) into a record.
template <typename T>
__device__ __forceinline__ void qmm_make_record(const T* __restrict__ src, int valid, int order, uint8_t* rec,
                                                int lane) {
  const int i = lane >> 2, c = lane & 3;
  int k[2];
  qmm_runs(order, i, c, k[0], k[1]);
  float v[8];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if constexpr (sizeof(T) == 4) {
      const bool wide = ((reinterpret_cast<uintptr_t>(src) & 15) == 0) && k[r] + 4 <= valid;
      if (wide) {
        const float4 f = *reinterpret_cast<const float4*>(src + k[r]);
        v[4 * r] = f.x; v[4 * r + 1] = f.y; v[4 * r + 2] = f.z; v[4 * r + 3] = f.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * r + e] = k[r] + e < valid ? (float)src[k[r] + e] : 0.0f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * r + e] = k[r] + e < valid ? __bfloat162float(src[k[r] + e]) : 0.0f;
    }
  }
  uint32_t mx = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) mx = max(mx, __float_as_uint(v[e]) & 0x7FFFFFFFu);
  mx = __reduce_max_sync(0xffffffffu, mx);
  // exponent field E of the largest: s = 2^(E - 127 - 14), so x' < 2^15.
  // Below 2^-112 the scale stays (1/s must be finite): such values lose bits
  // at 2^-136.  Infinities and NaN pass through and spoil this token alone.
  const int E = min(max((int)(mx >> 23), 15), 254);
  const float s = __uint_as_float((uint32_t)(E - 14) << 23);
  const float inv = __uint_as_float((uint32_t)(268 - E) << 23);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= inv;
  // the pairs of the MMA operands are values (0, 2) and (1, 3) of a run
  uint4 hi, lo;
  qmm_split2(v[0], v[2], hi.x, lo.x);
  qmm_split2(v[1], v[3], hi.y, lo.y);
  qmm_split2(v[4], v[6], hi.z, lo.z);
  qmm_split2(v[5], v[7], hi.w, lo.w);
  *reinterpret_cast<uint4*>(rec + 16 * lane) = hi;
  *reinterpret_cast<uint4*>(rec + 512 + 16 * (lane ^ 4)) = lo;
  // sums of 16: four lanes hold a group's runs (those of equal i, or of
  // equal c for the K45 order)
  const int m0 = order == kOrdK45 ? 4 : 1, m1 = 2 * m0;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float t = (v[4 * r] + v[4 * r + 1]) + (v[4 * r + 2] + v[4 * r + 3]);
    t += __shfl_xor_sync(0xffffffffu, t, m0);
    t += __shfl_xor_sync(0xffffffffu, t, m1);
    if ((lane & (m0 | m1)) == 0) {
      t *= 0.03125f;
      const int g = k[r] >> 4;
      const int at = ((g & 7) >> 1) * 4 + (g & 1) + (g >= 8 ? 2 : 0);
      const __half h = __float2half_rn(t);
      *reinterpret_cast<__half*>(rec + 1024 + 2 * at) = h;
      *reinterpret_cast<__half*>(rec + 1056 + 2 * at) = __float2half_rn(t - __half2float(h));
    }
  }
  if (lane == 0) *reinterpret_cast<float*>(rec + 1088) = s;
}

// ---------------------------------------------------------------------------
struct QmmGroup {
  int expert, start, count, pad;  // tokens plist[start .. start + count)
};

enum QmmMode : int { kQmmLinear = 0, kQmmUp = 1, kQmmDown = 2 };

struct QmmParams {
  int mode, RW, KW, stages, split;
  int TS;        // token slots of a unit (the largest group)
  int YC;        // columns of the partial sums: TS, or M for kQmmDown
  int M, top_k;  // tokens; picks per token
  int act, dtype;
  int nsb;       // units of a weight row: ceil(K / 256)
  int nblk;      // K / 32
  int rows_aligned;  // every row starts 16-byte aligned: TMA boxes
  int PB;            // buffers of partial sums (0: outputs straight from registers)
  int64_t n, K, rb;          // rows of one expert, K, bytes of a row
  const uint8_t* w0;         // weights (kQmmUp: gate)
  const uint8_t* w1;         // kQmmUp: up
  int64_t wbytes;            // bytes of all experts' rows
  const uint8_t* recs;       // activation records [row][nsb]
  // kQmmLinear
  const float* bias;
  // kQmmLinear, kQmmDown
  const void* residual;
  void* y;
  // kQmmUp, kQmmDown
  float* h;                  // [M * top_k][n] (written by kQmmUp)
  int E, score;              // experts; -1: ids and wts are given, else they are outputs
  const double* logits;      // [M][E]
  const float* sel_bias;
  float scale;
  int32_t* ids;
  float* wts;
  QmmGroup* groups;          // lists of the picks by expert, written by kQmmUp
  int32_t* plist;
  float* pwts;
  int32_t* ngroups;
};

__device__ __forceinline__ void qmm_dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void qmm_dep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ void qmm_tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar, uint64_t pol) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, "
      "%3}], [%4], %5;" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar)), "l"(pol)
      : "memory");
}
__device__ __forceinline__ void qmm_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

__device__ __forceinline__ void qmm_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float qmm_act(float v, int act) {
  switch (act) {
    case NSQ_ACT_SILU: return v / (1.0f + expf(-v));
    case NSQ_ACT_GELU: return 0.5f * v * erfcf(-0.70710678118654752f * v);
    case NSQ_ACT_GELU_TANH: {
      // 0.5 (1 + tanh u) = 1 / (1 + e^(-2u))
      const float u = 1.5957691216057308f * (v + 0.044715f * v * v * v);
      return v / (1.0f + expf(-u));
    }
    case NSQ_ACT_RELU: return v < 0.0f ? 0.0f : v;
    default: return v;
  }
}

// ---------------------------------------------------------------------------
// Per format: bytes of a unit of one row (CB), row tiles per warp (MT) and the
// pitches of a slot's rows: with 16-byte aligned rows (PA, the TMA box) and
// without (PG: the copies then carry up to 14 bytes before and 15 after the
// unit).  The pitches put the reads of 8 rows x 4 lanes on distinct banks.
// Two row tiles share their B operands and bookkeeping; the wider formats
// have one, for the depth of the ring.
template <int TYPE> struct QmmFmt;
template <> struct QmmFmt<NSQ_TYPE_Q4_K> { static constexpr int CB = 144, PA = 144, PG = 144, MT = 2; };
template <> struct QmmFmt<NSQ_TYPE_Q5_K> { static constexpr int CB = 176, PA = 176, PG = 176, MT = 2; };
template <> struct QmmFmt<NSQ_TYPE_Q6_K> { static constexpr int CB = 210, PA = 240, PG = 240, MT = 1; };
template <> struct QmmFmt<NSQ_TYPE_Q4_0> { static constexpr int CB = 144, PA = 144, PG = 176, MT = 2; };
template <> struct QmmFmt<NSQ_TYPE_Q8_0> { static constexpr int CB = 272, PA = 272, PG = 304, MT = 1; };

// All shared memory is addressed as an offset from this array, so that loads
// stay shared-memory loads with immediate offsets.  TMA boxes land on 128-byte
// boundaries: slots are multiples of 128 bytes from its start.  Static shared
// memory would come before it and leave it only 16-byte aligned, whatever is
// declared here, so the kernel has none: the barriers take the first bytes.
extern __shared__ __align__(128) uint8_t qmm_smem[];
template <typename T>
__device__ __forceinline__ T qmm_lds(uint32_t off) {
  return *reinterpret_cast<const T*>(qmm_smem + off);
}

// Where this lane reads the B operands of NT n-tiles: its token and part in
// each (a record of zeros for absent tokens).
template <int NT>
struct QmmB {
  uint32_t even[NT], odd[NT];  // units 4i + c of even and odd i, less 64 i
  uint32_t t[NT];              // the T sums
  __device__ __forceinline__ QmmB(uint32_t recs, uint32_t zeros, int count, int lr, int c) {
    const int tok = lr >> 1, flip = (lr & 1) * 64;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const uint32_t r = 4 * j + tok < count ? recs + (4 * j + tok) * kQmmRec : zeros;
      even[j] = r + (flip << 3) + 16 * c + flip;  // lo parts at + 512, units ^ 4
      odd[j] = r + (flip << 3) + 16 * c - flip;
      t[j] = r + 1024 + (flip >> 1) + 8 * c;
    }
  }
  __device__ __forceinline__ uint4 steps(int j, int i) const {
    return qmm_lds<uint4>(((i & 1) ? odd[j] : even[j]) + 64 * i);
  }
};

// A weight row whose first byte lies at an even offset: words at even
// offsets as two aligned words and a funnel shift.
struct QmmRow {
  uint32_t at, a0, a2, s0, s2;
  __device__ __forceinline__ explicit QmmRow(uint32_t off)
      : at(off), a0(off & ~3u), a2((off + 2) & ~3u), s0((off & 2) * 8), s2(((off + 2) & 2) * 8) {}
  template <int OFF>
  __device__ __forceinline__ uint32_t word(uint32_t more) const {  // more: a multiple of 4
    if constexpr (OFF % 4 == 0) {
      return __funnelshift_r(qmm_lds<uint32_t>(a0 + more + OFF), qmm_lds<uint32_t>(a0 + more + OFF + 4), s0);
    } else {
      return __funnelshift_r(qmm_lds<uint32_t>(a2 + more + OFF - 2), qmm_lds<uint32_t>(a2 + more + OFF + 2), s2);
    }
  }
  __device__ __forceinline__ uint32_t u16(int off) const { return qmm_lds<uint16_t>(at + off); }
  __device__ __forceinline__ uint32_t u8(int off) const { return qmm_lds<uint8_t>(at + off); }
};
// Calls f(integral_constant 0), ..., f(N - 1), so that offsets are constants.
template <int N, int I = 0, typename Fn>
__device__ __forceinline__ void qmm_for(Fn&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    qmm_for<N, I + 1>(f);
  }
}

// Byte b (a runtime number) of w as two equal fp16: 1024 + byte.
__device__ __forceinline__ __half2 qmm_dup1024(uint32_t w, int b) {
  return qmm_u2h(__byte_perm(w, 0x64646464u, 0x4040u | (uint32_t)(b | (b << 8))));
}

// Two fp16 1024 + v (or 1024 + 16 v) less their offset, exactly.
__device__ __forceinline__ uint32_t qmm_off(uint32_t v, float off) {
  return qmm_h2u(__hadd2(qmm_u2h(v), __float2half2_rn(off)));
}
__device__ __forceinline__ uint32_t qmm_off16(uint32_t v, float off) {
  return qmm_h2u(__hfma2(qmm_u2h(v), __float2half2_rn(0.0625f), __float2half2_rn(off)));
}

// One unit's products u[tile][j][row half], without the token scale s.  o: the
// shared-memory offsets of this lane's weight rows lane / 4 and lane / 4 + 8
// of each row tile; c = lane % 4; nv: valid 32-weight blocks (Q4_0, Q8_0).
template <int TYPE, int LAYOUT, int MT, int NT>
__device__ __forceinline__ void qmm_unit(const uint32_t (&o)[MT][2], int c, const QmmB<NT>& B, int nv,
                                         float (&u)[MT][NT][2]) {
  if constexpr (TYPE == NSQ_TYPE_Q4_K || TYPE == NSQ_TYPE_Q5_K) {
    __half2 sa[MT][2], sb[MT][2];  // scales of sub-blocks 2c and 2c+1, times 2^10 and 2^6
    const __half2 k1024 = __float2half2_rn(1024.0f), k64 = __float2half2_rn(64.0f);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      uint32_t ma[2], mb[2];
      float dm[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint4 h = qmm_lds<uint4>(o[t][r]);
        dm[r] = h2f((uint16_t)(h.x >> 16)) * -32.0f;
        // 6-bit scales of sub-blocks 2c, 2c+1: bytes of y (c < 2), or of w and y's upper bits
        const uint32_t s = c < 2 ? h.y & 0x3F3F3F3Fu : (h.w & 0x0F0F0F0Fu) | ((h.y >> 2) & 0x30303030u);
        const uint32_t m_lo = h.z & 0x3F3F3F3Fu, m_hi = ((h.w >> 4) & 0x0F0F0F0Fu) | ((h.z >> 2) & 0x30303030u);
        sa[t][r] = __hmul2(__hsub2(qmm_dup1024(s, (2 * c) & 3), k1024), k1024);
        sb[t][r] = __hmul2(__hsub2(qmm_dup1024(s, (2 * c + 1) & 3), k1024), k64);
        ma[r] = qmm_h2u(__hsub2(qmm_dup1024(m_lo, c), k1024));
        mb[r] = qmm_h2u(__hsub2(qmm_dup1024(m_hi, c), k1024));
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint2 b = qmm_lds<uint2>(B.t[j]);
        float am[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // the mins against T
        qmm_mma(am, ma[0], ma[1], mb[0], mb[1], b.x, b.y);
        u[t][j][0] = dm[0] * (am[0] + am[1]);
        u[t][j][1] = dm[1] * (am[2] + am[3]);
      }
    }
    constexpr int QS = TYPE == NSQ_TYPE_Q4_K ? 16 : 48;
    [[maybe_unused]] uint2 hn[MT][2];
    if constexpr (TYPE == NSQ_TYPE_Q5_K && LAYOUT == NSQ_Q6K_NODESTOR) {
      // bit l of word 2c (2c+1) of qh is the fifth bit of weight l of sub-block 2c (2c+1)
#pragma unroll
      for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int r = 0; r < 2; ++r) hn[t][r] = qmm_lds<uint2>(o[t][r] + 16 + 8 * c);
      }
    }
    float acc[MT][NT][4];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[t][j][0] = acc[t][j][1] = acc[t][j][2] = acc[t][j][3] = 0.0f;
    }
#pragma unroll
    for (int i4 = 0; i4 < 2; ++i4) {
      uint4 q[MT][2];
      [[maybe_unused]] uint4 hg[MT][2];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          q[t][r] = qmm_lds<uint4>(o[t][r] + QS + 32 * c + 16 * i4);
          // ggml: bit 2c (2c+1) of byte l is the fifth bit of weight l of sub-block 2c (2c+1)
          if constexpr (TYPE == NSQ_TYPE_Q5_K && LAYOUT == NSQ_Q6K_GGML) hg[t][r] = qmm_lds<uint4>(o[t][r] + 16 + 16 * i4);
        }
      }
#pragma unroll
      for (int ii = 0; ii < 4; ++ii) {
        const int i = 4 * i4 + ii;
        uint4 b[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) b[j] = B.steps(j, i);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          uint32_t a[2][4];  // [row]: sub-block 2c (values 0,2 | 1,3), sub-block 2c+1 (the same)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t w = ii == 0 ? q[t][r].x : ii == 1 ? q[t][r].y : ii == 2 ? q[t][r].z : q[t][r].w;
            const uint32_t w8 = w >> 8;
            uint32_t v0 = w & 0x000F000Fu, v1 = w8 & 0x000F000Fu, v2 = w & 0x00F000F0u, v3 = w8 & 0x00F000F0u;
            if constexpr (TYPE == NSQ_TYPE_Q5_K && LAYOUT == NSQ_Q6K_GGML) {
              const uint32_t g =
                  (ii == 0 ? hg[t][r].x : ii == 1 ? hg[t][r].y : ii == 2 ? hg[t][r].z : hg[t][r].w) >> (2 * c);
              v0 |= (g << 4) & 0x00100010u;
              v1 |= (g >> 4) & 0x00100010u;
              v2 |= (g << 7) & 0x01000100u;
              v3 |= (g >> 1) & 0x01000100u;
            } else if constexpr (TYPE == NSQ_TYPE_Q5_K) {
              const uint32_t g = (hn[t][r].x >> (4 * i)) & 15u, f = (hn[t][r].y >> (4 * i)) & 15u;
              v0 |= (g * 0x00040010u) & 0x00100010u;  // bits 0, 2 -> 4, 20
              v1 |= (g * 0x00020008u) & 0x00100010u;  // bits 1, 3 -> 4, 20
              v2 |= (f * 0x00400100u) & 0x01000100u;
              v3 |= (f * 0x00200080u) & 0x01000100u;
            }
            a[r][0] = qmm_mul2(v0, sa[t][r]);
            a[r][1] = qmm_mul2(v1, sa[t][r]);
            a[r][2] = qmm_mul2(v2, sb[t][r]);
            a[r][3] = qmm_mul2(v3, sb[t][r]);
          }
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            qmm_mma(acc[t][j], a[0][0], a[1][0], a[0][1], a[1][1], b[j].x, b[j].y);
            qmm_mma(acc[t][j], a[0][2], a[1][2], a[0][3], a[1][3], b[j].z, b[j].w);
          }
        }
      }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float d = h2f((uint16_t)qmm_lds<uint16_t>(o[t][r])) * 16384.0f;
#pragma unroll
        for (int j = 0; j < NT; ++j) u[t][j][r] += d * (acc[t][j][2 * r] + acc[t][j][2 * r + 1]);
      }
    }
  } else if constexpr (TYPE == NSQ_TYPE_Q4_0 || TYPE == NSQ_TYPE_Q8_0) {
    constexpr int BB = TYPE == NSQ_TYPE_Q4_0 ? 18 : 34;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int j = 0; j < NT; ++j) u[t][j][0] = u[t][j][1] = 0.0f;
    }
    qmm_for<8>([&](auto I) {
      constexpr int i = decltype(I)::value;
      uint4 b[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) b[j] = B.steps(j, i);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        uint32_t a[2][4];
        float d[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const QmmRow row(o[t][r]);
          d[r] = i < nv ? h2f((uint16_t)row.u16(BB * i)) : 0.0f;
          const uint32_t w = row.template word<BB * i + 2>(4 * c);
          if constexpr (TYPE == NSQ_TYPE_Q4_0) {
            // 1024 + q and 1024 + 16 q
            const uint32_t w8 = w >> 8;
            a[r][0] = qmm_off((w & 0x000F000Fu) | 0x64006400u, -1032.0f);
            a[r][1] = qmm_off((w8 & 0x000F000Fu) | 0x64006400u, -1032.0f);
            a[r][2] = qmm_off16((w & 0x00F000F0u) | 0x64006400u, -72.0f);
            a[r][3] = qmm_off16((w8 & 0x00F000F0u) | 0x64006400u, -72.0f);
          } else {
            const uint32_t x = w ^ 0x80808080u, y = row.template word<BB * i + 18>(4 * c) ^ 0x80808080u;
            a[r][0] = qmm_off(__byte_perm(x, 0x64646464u, 0x4240), -1152.0f);
            a[r][1] = qmm_off(__byte_perm(x, 0x64646464u, 0x4341), -1152.0f);
            a[r][2] = qmm_off(__byte_perm(y, 0x64646464u, 0x4240), -1152.0f);
            a[r][3] = qmm_off(__byte_perm(y, 0x64646464u, 0x4341), -1152.0f);
          }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          qmm_mma(acc, a[0][0], a[1][0], a[0][1], a[1][1], b[j].x, b[j].y);
          qmm_mma(acc, a[0][2], a[1][2], a[0][3], a[1][3], b[j].z, b[j].w);
          u[t][j][0] += d[0] * (acc[0] + acc[1]);
          u[t][j][1] += d[1] * (acc[2] + acc[3]);
        }
      }
    });
  } else {  // Q6_K
    static_assert(MT == 1, "one row tile");
    const QmmRow rows[2] = {QmmRow(o[0][0]), QmmRow(o[0][1])};
    auto& v = u[0];
#pragma unroll
    for (int j = 0; j < NT; ++j) v[j][0] = v[j][1] = 0.0f;
    float d[2];
    uint32_t sw[2][4];  // the 16 scale bytes, + 128
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      d[r] = h2f((uint16_t)rows[r].u16(208));
      if constexpr (LAYOUT == NSQ_Q6K_NODESTOR) d[r] *= 0.015625f;  // scale (b - 128) / 64
      qmm_for<4>([&](auto I) {
        constexpr int i = decltype(I)::value;
        sw[r][i] = rows[r].template word<192 + 4 * i>(0);
        if constexpr (LAYOUT == NSQ_Q6K_GGML) sw[r][i] ^= 0x80808080u;
      });
    }
    // scale byte g of row r as f32
    auto scale = [&](int r, int g) {
      return __uint_as_float(__byte_perm(sw[r][g >> 2], 0x4B000000u, 0x7440u | (uint32_t)(g & 3))) - 8388736.0f;
    };
    auto group = [&](int j, const uint32_t (&a)[2][2], uint32_t b0, uint32_t b1, float s0, float s1) {
      float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      qmm_mma(acc, a[0][0], a[1][0], a[0][1], a[1][1], b0, b1);
      v[j][0] += s0 * (acc[0] + acc[1]);
      v[j][1] += s1 * (acc[2] + acc[3]);
    };
    constexpr uint32_t kL = 0x000F000Fu, kH = 0x00F000F0u, kB = 0x64006400u;
    if constexpr (LAYOUT == NSQ_Q6K_GGML) {
      qmm_for<4>([&](auto P) {  // (half n, 16-group of its runs of 32)
        constexpr int pp = decltype(P)::value, n = pp >> 1, g = pp & 1;
        uint32_t a[4][2][2];  // [run t][row][values 0,2 | 1,3]
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t A = rows[r].template word<64 * n + 16 * g>(4 * c);
          const uint32_t Bw = rows[r].template word<64 * n + 32 + 16 * g>(4 * c);
          const uint32_t H = rows[r].template word<128 + 32 * n + 16 * g>(4 * c);
          const uint32_t A8 = A >> 8, B8 = Bw >> 8, Hl4 = H << 4, Hl2 = H << 2, Hr4 = H >> 4, Hr6 = H >> 6;
          a[0][r][0] = qmm_off((A & kL) | ((Hl4 & 0x00300030u) | kB), -1056.0f);
          a[0][r][1] = qmm_off((A8 & kL) | ((Hr4 & 0x00300030u) | kB), -1056.0f);
          a[1][r][0] = qmm_off((Bw & kL) | ((Hl2 & 0x00300030u) | kB), -1056.0f);
          a[1][r][1] = qmm_off((B8 & kL) | ((Hr6 & 0x00300030u) | kB), -1056.0f);
          a[2][r][0] = qmm_off((A & kH) | ((Hl4 & 0x03000300u) | kB), -1536.0f);  // 16 (q - 32)
          a[2][r][1] = qmm_off((A8 & kH) | ((Hr4 & 0x03000300u) | kB), -1536.0f);
          a[3][r][0] = qmm_off((Bw & kH) | ((Hl2 & 0x03000300u) | kB), -1536.0f);
          a[3][r][1] = qmm_off((B8 & kH) | ((Hr6 & 0x03000300u) | kB), -1536.0f);
        }
        float s[4][2];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
          for (int r = 0; r < 2; ++r) s[t][r] = scale(r, 8 * n + g + 2 * t) * (t < 2 ? 1.0f : 0.0625f);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 b0 = B.steps(j, 2 * pp), b1 = B.steps(j, 2 * pp + 1);
          group(j, a[0], b0.x, b0.y, s[0][0], s[0][1]);
          group(j, a[1], b0.z, b0.w, s[1][0], s[1][1]);
          group(j, a[2], b1.x, b1.y, s[2][0], s[2][1]);
          group(j, a[3], b1.z, b1.w, s[3][0], s[3][1]);
        }
      });
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t a[2][2][2];  // [group 2i, 2i+1][row][values 0,2 | 1,3]
        float s[2][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int g = 2 * i + t;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            // values 4c .. 4c+3 of the group: ql bytes 8g + 2c, + 1; qh byte 4g + c
            const uint32_t lo = __byte_perm(rows[r].u16(8 * g + 2 * c), 0, 0x4140);
            const uint32_t hb = rows[r].u8(128 + 4 * g + c);
            // bits 0-1, 4-5 and 2-3, 6-7 of hb
            a[t][r][0] = qmm_off((lo & kL) | (((hb * 0x00010010u) & 0x00300030u) | kB), -1056.0f);
            a[t][r][1] = qmm_off(((lo >> 4) & kL) | (((hb * 0x00004004u) & 0x00300030u) | kB), -1056.0f);
            s[t][r] = scale(r, g);
          }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 b = B.steps(j, i);
          group(j, a[0], b.x, b.y, s[0][0], s[0][1]);
          group(j, a[1], b.z, b.w, s[1][0], s[1][1]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      v[j][0] *= d[0];
      v[j][1] *= d[1];
    }
  }
}

// ---------------------------------------------------------------------------
// Lists of the picks by expert (kQmmUp and kQmmDown).  Every CTA of kQmmUp
// builds them for itself from the logits or the given ids, in shared memory:
// that costs about a microsecond and saves a launch; CTA 0 writes them out.
struct QmmLists {
  QmmGroup* groups;
  int32_t* plist;  // picks sorted by (expert, pick)
  float* pwts;     // their weights
  int32_t* ptok;   // their tokens
  int ngroups;
};

__device__ __forceinline__ uint64_t qmm_key(double v) {  // ordered as v; NaN below everything, 0 is taken
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  return v != v ? 1ull : (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}

// One warp picks token m's experts: ids and weights of top_k picks.
__device__ __forceinline__ void qmm_route(const QmmParams& p, int m, int lane, int32_t* ids, float* wts) {
  constexpr int EP = NSQ_MOE_MAX_EXPERTS / 32;
  const double* l = p.logits + (int64_t)m * p.E;
  const bool sig = p.score == NSQ_SCORE_SIGMOID_NORM;
  const bool by_score = sig || p.sel_bias;  // else the order of the logits is that of the scores
  double mx = -INFINITY, sum = 0.0;
  if (!sig) {
    for (int e = lane; e < p.E; e += 32) mx = fmax(mx, l[e]);
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (p.score == NSQ_SCORE_SOFTMAX || by_score) {
      for (int e = lane; e < p.E; e += 32) sum += exp(l[e] - mx);
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
  }
  auto score = [&](double v) { return sig ? 1.0 / (1.0 + exp(-v)) : sum > 0.0 ? exp(v - mx) / sum : exp(v - mx); };
  uint64_t key[EP];
#pragma unroll
  for (int i = 0; i < EP; ++i) {
    const int e = lane + 32 * i;
    key[i] = 0;
    if (e < p.E) {
      const double v = l[e];
      key[i] = qmm_key(by_score ? score(v) + (p.sel_bias ? (double)p.sel_bias[e] : 0.0) : v);
    }
  }
  double total = 0.0, mine = 0.0;  // lane j keeps pick j's score
  int mine_id = 0;
  for (int j = 0; j < p.top_k; ++j) {
    uint64_t best = 0;
    int at = 0x7FFFFFFF;
#pragma unroll
    for (int i = 0; i < EP; ++i) {
      if (key[i] > best) {
        best = key[i];
        at = lane + 32 * i;
      }
    }
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
    const bool me = (uint32_t)(best >> 32) == hi && (uint32_t)best == lo;
    const int id = (int)__reduce_min_sync(0xffffffffu, (uint32_t)(me ? at : 0x7FFFFFFF));
#pragma unroll
    for (int i = 0; i < EP; ++i) {
      if (lane + 32 * i == id) key[i] = 0;
    }
    const double s = score(l[id]);
    total += s;
    if (lane == j) {
      mine = s;
      mine_id = id;
    }
  }
  if (lane < p.top_k) {
    ids[lane] = mine_id;
    wts[lane] = (float)((p.score == NSQ_SCORE_SOFTMAX ? mine : mine / total) * (double)p.scale);
  }
}

// scratch: 2 * P ints
__device__ __forceinline__ QmmLists qmm_build_lists(const QmmParams& p, uint8_t* mem, int32_t* scratch, int* s_n) {
  const int P = p.M * p.top_k;
  QmmLists L;
  L.groups = reinterpret_cast<QmmGroup*>(mem);
  L.plist = reinterpret_cast<int32_t*>(L.groups + P);
  L.pwts = reinterpret_cast<float*>(L.plist + P);
  L.ptok = reinterpret_cast<int32_t*>(L.pwts + P);
  int32_t* ids = scratch;
  float* wts = reinterpret_cast<float*>(scratch + P);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool first = blockIdx.x == 0;
  if (p.score >= 0) {
    for (int m = warp; m < p.M; m += kQmmWarps + 1) {
      qmm_route(p, m, lane, ids + m * p.top_k, wts + m * p.top_k);
      __syncwarp();
      if (first && lane < p.top_k) {
        p.ids[m * p.top_k + lane] = ids[m * p.top_k + lane];
        p.wts[m * p.top_k + lane] = wts[m * p.top_k + lane];
      }
    }
  } else {
    // an expert given twice by a token counts once, with the sum of its
    // weights: so a group holds a token once
    for (int q = threadIdx.x; q < P; q += kQmmThreads) {
      const int base = q - q % p.top_k, e = p.ids[q];
      bool keep = e >= 0 && e < p.E;
      float w = 0.0f;
      for (int r = base; r < base + p.top_k; ++r) {
        if (p.ids[r] == e) {
          if (r < q) keep = false;
          w += p.wts[r];
        }
      }
      ids[q] = keep ? e : -1;
      wts[q] = w;
    }
  }
  __syncthreads();
  // place of a pick: the number of valid picks that come before it
  for (int q = threadIdx.x; q < P; q += kQmmThreads) {
    const int e = ids[q];
    if (e < 0) continue;
    int pos = 0, rank = 0, same = 0;
    for (int r = 0; r < P; ++r) {
      const int o = ids[r];
      pos += o >= 0 && (o < e || (o == e && r < q));
      rank += o == e && r < q;
      same += o == e;
    }
    L.plist[pos] = q;
    L.pwts[pos] = wts[q];
    L.ptok[pos] = q / p.top_k;
    // groups of this expert start at every TS-th of its picks; their number
    // so far is filled in below
    L.groups[pos].expert = e;
    L.groups[pos].count = rank % p.TS == 0 ? min(p.TS, same - rank) : 0;
  }
  if (threadIdx.x == 0) *s_n = 0;
  __syncthreads();
  if (warp == 0) {
    int valid = 0;
    for (int q = lane; q < P; q += 32) valid += ids[q] >= 0;
    valid = __reduce_add_sync(0xffffffffu, valid);
    int n = 0;
    for (int b = 0; b < valid; b += 32) {  // in place: a group never moves up
      const int q = b + lane;
      const QmmGroup g = q < valid ? L.groups[q] : QmmGroup{0, 0, 0, 0};
      const uint32_t starts = __ballot_sync(0xffffffffu, g.count > 0);
      const int at = n + __popc(starts & ((1u << lane) - 1));
      if (g.count > 0) L.groups[at] = QmmGroup{g.expert, q, g.count, 0};
      n += __popc(starts);
      __syncwarp();
    }
    if (lane == 0) *s_n = n;
  }
  __syncthreads();
  L.ngroups = *s_n;
  if (first) {
    for (int q = threadIdx.x; q < P; q += kQmmThreads) {
      if (q < L.ngroups) p.groups[q] = L.groups[q];
      p.plist[q] = L.plist[q];
      p.pwts[q] = L.pwts[q];
    }
    if (threadIdx.x == 0) *p.ngroups = L.ngroups;
  }
  return L;
}

__device__ __forceinline__ QmmLists qmm_load_lists(const QmmParams& p, uint8_t* mem) {
  const int P = p.M * p.top_k;
  QmmLists L;
  L.groups = reinterpret_cast<QmmGroup*>(mem);
  L.plist = reinterpret_cast<int32_t*>(L.groups + P);
  L.pwts = reinterpret_cast<float*>(L.plist + P);
  L.ptok = reinterpret_cast<int32_t*>(L.pwts + P);
  L.ngroups = *p.ngroups;
  for (int q = threadIdx.x; q < P; q += kQmmThreads) {
    if (q < L.ngroups) L.groups[q] = p.groups[q];
    const int pick = p.plist[q];
    L.plist[q] = pick;
    L.ptok[q] = (int)((uint32_t)pick / (uint32_t)p.top_k);
    L.pwts[q] = p.pwts[q];
  }
  __syncthreads();
  return L;
}

__device__ __forceinline__ uint32_t qmm_cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void qmm_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float qmm_ld_cluster(const float* p, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

// Bytes of a slot: RW tiles of rows at this pitch, then TS records.
__host__ __device__ inline uint32_t qmm_slot_bytes(int row_tiles, int pitch, int TS) {
  return (uint32_t)(row_tiles * 16 * pitch + (TS * kQmmRec + 127) / 128 * 128);
}
inline size_t qmm_lists_bytes(int P) { return (size_t)P * (sizeof(QmmGroup) + 12); }

// Bias, activation and residual (kQmmLinear), or the residual alone
// (kQmmDown), for one finished sum.
__device__ __forceinline__ void qmm_store(const QmmParams& p, int col, int row, float v) {
  const int64_t at = (int64_t)col * p.n + row;
  if (p.mode == kQmmLinear) {
    if (p.bias) v += p.bias[row];
    v = qmm_act(v, p.act);
  }
  if (p.dtype == NSQ_OUT_F32) {
    if (p.residual) v += static_cast<const float*>(p.residual)[at];
    static_cast<float*>(p.y)[at] = v;
  } else {
    if (p.residual) v += __bfloat162float(static_cast<const __nv_bfloat16*>(p.residual)[at]);
    static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v);
  }
}

// Where a column stands: its task (tile, and the group for kQmmUp), its unit
// (u, of group g and column sb of K).
struct QmmCursor {
  int tile, g, sb, u;
};

template <int TYPE, int LAYOUT, int NT, int MODE>
__global__ void __launch_bounds__(kQmmThreads, 2)
    qmm_kernel(const __grid_constant__ QmmParams p, const __grid_constant__ CUtensorMap map0,
               const __grid_constant__ CUtensorMap map1) {
  using F = QmmFmt<TYPE>;
  constexpr int BB = Fmt<TYPE>::BB;
  constexpr int MT = F::MT;
  constexpr int WR = 16 * MT;                       // weight rows of a warp
  constexpr int OR = MODE == kQmmUp ? WR / 2 : WR;  // output rows of a warp
  uint8_t* const smem = qmm_smem;
  auto* const full = reinterpret_cast<uint64_t(*)[kQmmMaxStages]>(smem);           // [column][slot]
  auto* const empty = reinterpret_cast<uint64_t(*)[kQmmMaxStages]>(smem + 256);
  auto* const ready = reinterpret_cast<uint64_t(*)[2]>(smem + 512);                // [row tiles][buffer]
  auto* const taken = reinterpret_cast<uint64_t(*)[2]>(smem + 640);
  int* const s_n = reinterpret_cast<int*>(smem + 768);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int KW = p.KW, RW = p.RW, S = p.stages, TS = p.TS, YC = p.YC;
  const int pitch = p.rows_aligned ? F::PA : F::PG;
  const uint32_t slot_bytes = qmm_slot_bytes(RW * MT, pitch, TS);
  const uint32_t recs_at = RW * WR * pitch;          // of a slot
  const uint32_t ring_bytes = S * KW * slot_bytes;
  // partial sums [buffer][warp][YC][WR]; a split product keeps them in the
  // ring, which is idle by then, except kQmmDown's, which grow unit by unit
  const bool in_ring = MODE != kQmmDown && p.split > 1;
  float* const ys = reinterpret_cast<float*>(smem + kQmmCtl + (in_ring ? 0 : ring_bytes));
  const int ys_warp = YC * WR, ys_buf = kQmmWarps * ys_warp;
  const uint32_t zeros = kQmmCtl + ring_bytes + (in_ring ? 0 : p.PB * ys_buf * 4);  // a record of zeros
  const int rank = p.split > 1 ? (int)qmm_cluster_rank() : 0;
  const int cta = blockIdx.x / p.split, nctas = gridDim.x / p.split;
  const int tile_rows = OR * RW;
  const int tiles = (int)((p.n + tile_rows - 1) / tile_rows);

  {
    // the boxes' destination: a misaligned one would fault (the address is
    // hidden from the compiler, which takes the declared alignment for granted)
    uint32_t start = smem_u32(smem);
    asm volatile("" : "+r"(start));
    if (start & 127) {
      report_status(NSQ_ERR_ALIGN);
      return;
    }
  }
  for (int i = threadIdx.x; i < kQmmRec / 4; i += kQmmThreads) reinterpret_cast<uint32_t*>(smem + zeros)[i] = 0u;
  if (threadIdx.x == 0) {
    for (int i = 0; i < KW; ++i) {
      for (int k = 0; k < S; ++k) {
        mbar_init(&full[i][k], 1);
        mbar_init(&empty[i][k], RW);
      }
    }
    for (int i = 0; i < RW; ++i) {
      for (int k = 0; k < 2; ++k) {
        mbar_init(&ready[i][k], KW);
        mbar_init(&taken[i][k], 1);
      }
    }
    fence_mbar_init();
  }
  QmmLists L{};
  if constexpr (MODE == kQmmLinear) {
    L.ngroups = 1;
    __syncthreads();
  } else {
    qmm_dep_wait();
    qmm_dep_launch();
    uint8_t* lists_mem = smem + zeros + kQmmRec;
    if constexpr (MODE == kQmmUp) {
      L = qmm_build_lists(p, lists_mem, reinterpret_cast<int32_t*>(smem + kQmmCtl), s_n);
      fence_proxy_async_smem();  // the ring held the lists' scratch
      __syncthreads();
    } else {
      L = qmm_load_lists(p, lists_mem);
    }
  }
  const int units = MODE == kQmmDown ? L.ngroups * p.nsb : p.nsb;
  const int u0 = p.split > 1 ? (int)((int64_t)units * rank / p.split) : 0;
  const int u1 = p.split > 1 ? (int)((int64_t)units * (rank + 1) / p.split) : units;

  // cursors: column kw takes units u0 + kw, u0 + kw + KW, ... of every task
  const int up_dg = MODE == kQmmUp ? nctas / tiles : 0, up_dt = MODE == kQmmUp ? nctas - up_dg * tiles : nctas;
  auto first_task = [&](QmmCursor& c) {
    c.tile = cta;
    c.g = 0;
    if constexpr (MODE == kQmmUp) {
      c.g = cta / tiles;
      c.tile = cta - c.g * tiles;
    }
  };
  auto first_unit = [&](QmmCursor& c, int kw) {
    c.u = c.sb = u0 + kw;
    if constexpr (MODE == kQmmDown) {
      c.g = c.u / p.nsb;
      c.sb = c.u - c.g * p.nsb;
    }
  };
  auto live = [&](const QmmCursor& c) { return MODE == kQmmUp ? c.g < L.ngroups : c.tile < tiles; };
  auto next_unit = [&](QmmCursor& c) {
    c.u += KW;
    c.sb += KW;
    if constexpr (MODE == kQmmDown) {
      while (c.sb >= p.nsb) {
        c.sb -= p.nsb;
        ++c.g;
      }
    }
  };
  auto next_task = [&](QmmCursor& c) {
    c.tile += up_dt;
    if constexpr (MODE == kQmmUp) {
      c.g += up_dg;
      if (c.tile >= tiles) {
        c.tile -= tiles;
        ++c.g;
      }
    }
  };

  bool ok = true;
  if (warp == kQmmWarps) {
    // ---- producer.  With TMA boxes lane (kw, t0) serves column kw: its t0-th
    // lane issues the box and every lane its share of the records.  Without,
    // the whole warp copies the rows of one column after the other.
    const uint64_t pol = l2_policy_evict_first();
    const uint32_t base = smem_u32(smem);  // slots are offsets from it
    auto box = [&](const QmmCursor& c, uint32_t slot, uint64_t* bar) {
      const int row0 = (MODE == kQmmLinear ? 0 : L.groups[c.g].expert) * (int)p.n + c.tile * tile_rows;
      const int x = ((c.sb * F::CB) & ~15) / 2;  // 16-bit elements
      if constexpr (MODE == kQmmUp) {
        qmm_tma_2d(slot, &map0, x, row0, bar, pol);
        qmm_tma_2d(slot + RW * (WR / 2) * pitch, &map1, x, row0, bar, pol);
      } else {
        qmm_tma_2d(slot, &map0, x, row0, bar, pol);
      }
    };
    auto group_count = [&](const QmmCursor& c) { return MODE == kQmmLinear ? p.M : L.groups[c.g].count; };
    auto record = [&](const QmmCursor& c, int t) {
      int row = t;
      if constexpr (MODE == kQmmUp) row = L.ptok[L.groups[c.g].start + t];
      if constexpr (MODE == kQmmDown) row = L.plist[L.groups[c.g].start + t];
      return p.recs + ((int64_t)row * p.nsb + c.sb) * kQmmRec;
    };
    if (p.rows_aligned) {
      const int kw = lane & (KW - 1), t0 = lane / KW, dt = 32 / KW;
      const uint32_t w_bytes = RW * WR * pitch;
      QmmCursor c;
      first_task(c);
      first_unit(c, kw);
      int n = 0;  // units of this column so far
      if constexpr (MODE == kQmmLinear) {
        // the weights do not depend on the kernels before: the first boxes go
        // out ahead of the dependency wait
        QmmCursor w = c;
        for (int k = 0; k < S && t0 == 0 && live(w); ++k) {
          while (live(w) && w.u >= u1) {
            next_task(w);
            first_unit(w, kw);
            if (w.u >= u1) break;  // a column without units
          }
          if (!live(w) || w.u >= u1) break;
          qmm_expect_tx(&full[kw][k], w_bytes);
          box(w, base + kQmmCtl + (k * KW + kw) * slot_bytes, &full[kw][k]);
          next_unit(w);
        }
        __syncwarp();
        qmm_dep_wait();
        qmm_dep_launch();
      }
      int stage = 0;
      uint32_t phase = 0;
      for (; ok && live(c); next_task(c)) {
        for (first_unit(c, kw); c.u < u1; next_unit(c)) {
          uint64_t* bar = &full[kw][stage];
          if (n >= S && !mbar_wait_bounded(&empty[kw][stage], phase ^ 1)) {
            ok = false;
            break;
          }
          const uint32_t slot = kQmmCtl + (stage * KW + kw) * slot_bytes;
          const int count = group_count(c);
          if (t0 == 0) {
            const bool early = MODE == kQmmLinear && n < S;
            mbar_arrive_expect_tx(bar, (early ? 0 : w_bytes) + count * kQmmRec);
            if (!early) box(c, base + slot, bar);
          }
          for (int t = t0; t < count; t += dt) bulk_g2s(smem + slot + recs_at + t * kQmmRec, record(c, t), kQmmRec, bar);
          ++n;
          if (++stage == S) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    } else {
      if constexpr (MODE == kQmmLinear) {
        qmm_dep_wait();
        qmm_dep_launch();
      }
      // all columns step by step; a column's slot and phase go by its own count of units
      int n[kQmmWarps];
#pragma unroll
      for (int k = 0; k < kQmmWarps; ++k) n[k] = 0;
      QmmCursor c;
      first_task(c);
      for (; ok && live(c); next_task(c)) {
        for (int s0 = 0; ok && u0 + s0 < u1; s0 += KW) {
#pragma unroll
          for (int kw = 0; kw < kQmmWarps; ++kw) {
            const int u = u0 + s0 + kw;
            if (kw >= KW || u >= u1 || !ok) continue;
            QmmCursor d = c;
            d.u = d.sb = u;
            if constexpr (MODE == kQmmDown) {
              d.g = u / p.nsb;
              d.sb = u - d.g * p.nsb;
            }
            const int stage = n[kw] % S, turn = n[kw] / S;
            ++n[kw];
            uint64_t* bar = &full[kw][stage];
            if (turn > 0 && !mbar_wait_bounded(&empty[kw][stage], (turn & 1) ^ 1)) {
              ok = false;
              continue;
            }
            fence_proxy_async_smem();  // a tensor's last bytes are stored by hand
            const uint32_t slot = kQmmCtl + (stage * KW + kw) * slot_bytes;
            const int64_t row0 = (MODE == kQmmLinear ? 0 : (int64_t)L.groups[d.g].expert * p.n) + d.tile * tile_rows;
            const int valid = (int)min((int64_t)tile_rows, p.n - (int64_t)d.tile * tile_rows);
            int need = F::CB;
            if constexpr (Fmt<TYPE>::QK == 32) need = min(8, p.nblk - 8 * d.sb) * BB;
            const int64_t cap = p.wbytes & ~(int64_t)15;
            auto span = [&](int r, const uint8_t*& w, int64_t& a, int64_t& e, int64_t& end) {
              int rr = r;
              w = p.w0;
              if constexpr (MODE == kQmmUp) {
                if (r >= RW * (WR / 2)) {
                  rr -= RW * (WR / 2);
                  w = p.w1;
                }
              }
              if (rr >= valid) return false;
              const int64_t at = (row0 + rr) * p.rb + (int64_t)d.sb * F::CB;
              a = at & ~(int64_t)15;
              end = at + need;
              e = (end + 15) & ~(int64_t)15;
              if (e > cap) e = cap > a ? cap : a;
              return true;
            };
            const int count = group_count(d);
            uint32_t bytes = lane < count ? kQmmRec : 0;
            for (int r = lane; r < RW * WR; r += 32) {
              const uint8_t* w;
              int64_t a, e, end;
              if (!span(r, w, a, e, end)) continue;
              bytes += (uint32_t)(e - a);
              for (int64_t i = e; i < end; ++i) smem[slot + r * pitch + (i - a)] = w[i];  // past the last whole 16 bytes
            }
            bytes = __reduce_add_sync(0xffffffffu, bytes);
            __syncwarp();
            if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
            __syncwarp();
            for (int r = lane; r < RW * WR; r += 32) {
              const uint8_t* w;
              int64_t a, e, end;
              if (span(r, w, a, e, end) && e > a) bulk_g2s(smem + slot + r * pitch, w + a, (uint32_t)(e - a), bar);
            }
            if (lane < count) bulk_g2s(smem + slot + recs_at + lane * kQmmRec, record(d, lane), kQmmRec, bar);
          }
        }
      }
    }
  } else {
    // ---- consumers
    if constexpr (MODE == kQmmLinear) qmm_dep_wait();  // residual and outputs
    const int kw = warp & (KW - 1), rw = warp / KW;
    const int lr = lane >> 2, lc = lane & 3;
    const bool split = p.split > 1;
    float tot[MT][NT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int j = 0; j < NT; ++j) tot[t][j][0] = tot[t][j][1] = 0.0f;
    }
    // rows of this lane in a slot: row half h of tile t
    auto slot_row = [&](int t, int h) {
      if constexpr (MODE == kQmmUp) {
        return MT == 2 ? (t * RW + rw) * 16 + 8 * h + lr : (h * RW + rw) * 8 + lr;
      } else {
        return rw * WR + 16 * t + 8 * h + lr;
      }
    };
    int stage = 0, seq = 0;
    uint32_t phase = 0;
    QmmCursor c;
    first_task(c);
    for (; ok && live(c); next_task(c), ++seq) {
      const int buf = p.PB == 2 ? seq & 1 : 0, turn = p.PB == 2 ? seq >> 1 : seq;
      float* my_ys = ys + buf * ys_buf + warp * ys_warp;
      const bool own_ys = p.PB > 0 && !split;
      if constexpr (MODE == kQmmDown) {
        if (own_ys && turn > 0 && !mbar_wait_bounded(&taken[rw][buf], (turn & 1) ^ 1)) {
          ok = false;
          break;
        }
        __syncwarp();
        for (int i = lane; i < ys_warp; i += 32) my_ys[i] = 0.0f;
        __syncwarp();
      }
      for (first_unit(c, kw); c.u < u1; next_unit(c)) {
        if (!mbar_wait_bounded(&full[kw][stage], phase)) {
          ok = false;
          break;
        }
        __syncwarp();
        const int count = MODE == kQmmLinear ? p.M : L.groups[c.g].count;
        const uint32_t slot = kQmmCtl + (stage * KW + kw) * slot_bytes;
        uint32_t o[MT][2];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = slot_row(t, h);
            uint32_t mis = 0;
            if constexpr (F::CB % 16 != 0 || Fmt<TYPE>::QK == 32) {
              mis = (uint32_t)(c.sb * F::CB) & 15;
              if (!p.rows_aligned) {
                const int rr = MODE == kQmmUp && r >= RW * (WR / 2) ? r - RW * (WR / 2) : r;
                const int64_t row = (MODE == kQmmLinear ? 0 : (int64_t)L.groups[c.g].expert * p.n) + c.tile * tile_rows + rr;
                mis = (uint32_t)(row * p.rb + (int64_t)c.sb * F::CB) & 15;
              }
            }
            o[t][h] = slot + r * pitch + mis;
          }
        }
        float uv[MT][NT][2];
        const int nv = min(8, p.nblk - 8 * c.sb);
        // as many n-tiles as the group has tokens
        auto unit = [&](auto N) {
          constexpr int nt = decltype(N)::value;
          const QmmB<nt> B(slot + recs_at, zeros, count, lr, lc);
          float v[MT][nt][2];
          qmm_unit<TYPE, LAYOUT, MT, nt>(o, lc, B, nv, v);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
#pragma unroll
            for (int j = 0; j < nt; ++j) {
              uv[t][j][0] = v[t][j][0];
              uv[t][j][1] = v[t][j][1];
            }
          }
        };
        if (NT == 1 || count <= 4) {
          unit(std::integral_constant<int, 1>{});
        } else if (NT == 2 || count <= 8) {
          unit(std::integral_constant<int, NT < 2 ? NT : 2>{});
        } else {
          unit(std::integral_constant<int, NT>{});
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int tk = 4 * j + lc;
          if (tk < count) {
            float s = qmm_lds<float>(slot + recs_at + tk * kQmmRec + 1088);
            if constexpr (MODE == kQmmDown) {
              const int pick = L.groups[c.g].start + tk;
              const float w = L.pwts[pick];
              float* q = my_ys + L.ptok[pick] * WR + lr;
#pragma unroll
              for (int t = 0; t < MT; ++t) {
                q[16 * t] += w * (s * uv[t][j][0]);
                q[16 * t + 8] += w * (s * uv[t][j][1]);
              }
            } else {
#pragma unroll
              for (int t = 0; t < MT; ++t) {
                tot[t][j][0] += s * uv[t][j][0];
                tot[t][j][1] += s * uv[t][j][1];
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[kw][stage]);
        if (++stage == S) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok || split) break;  // a split product has one task; its sums are joined below
      const int row0 = c.tile * tile_rows + rw * OR;
      if (p.PB == 0) {
        // ---- KW == 1: outputs straight from the registers
        const int cnt = MODE == kQmmLinear ? p.M : L.groups[c.g].count;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int tk = 4 * j + lc;
#pragma unroll
          for (int t = 0; t < MT; ++t) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if constexpr (MODE == kQmmUp) {
                // gate and up of an output row: row halves of one tile, or two tiles
                if ((MT == 2 ? t : h) == 0 && tk < cnt) {
                  const int row = row0 + (MT == 2 ? 8 * h : 0) + lr;
                  const float up = MT == 2 ? tot[MT - 1][j][h] : tot[0][j][1];
                  if (row < p.n) p.h[(int64_t)L.plist[L.groups[c.g].start + tk] * p.n + row] = qmm_act(tot[t][j][h], p.act) * up;
                }
              } else if constexpr (MODE == kQmmLinear) {
                const int row = row0 + 16 * t + 8 * h + lr;
                if (tk < cnt && row < p.n) qmm_store(p, tk, row, tot[t][j][h]);
              }
            }
          }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
          for (int j = 0; j < NT; ++j) tot[t][j][0] = tot[t][j][1] = 0.0f;
        }
        continue;
      }
      // ---- join the KW columns' sums: every warp leaves its own, one of them adds
      if constexpr (MODE != kQmmDown) {
        if (turn > 0 && !mbar_wait_bounded(&taken[rw][buf], (turn & 1) ^ 1)) {
          ok = false;
          break;
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            if (4 * j + lc < YC) {
              float* q = my_ys + (4 * j + lc) * WR + 16 * t + lr;
              q[0] = tot[t][j][0];
              q[8] = tot[t][j][1];
            }
            tot[t][j][0] = tot[t][j][1] = 0.0f;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ready[rw][buf]);
      if (kw == (seq & (KW - 1))) {
        if (!mbar_wait_bounded(&ready[rw][buf], turn & 1)) {
          ok = false;
          break;
        }
        __syncwarp();
        const float* y0 = ys + buf * ys_buf + rw * KW * ys_warp;
        auto sum_kw = [&](int col, int r) {
          float v = y0[col * WR + r];
          for (int k = 1; k < KW; ++k) v += y0[k * ys_warp + col * WR + r];
          return v;
        };
        const int cnt = MODE == kQmmUp ? L.groups[c.g].count : p.M;
        for (int i = lane; i < OR * cnt; i += 32) {
          const int col = i / OR, r = i % OR;
          if (row0 + r < p.n) {
            if constexpr (MODE == kQmmUp) {
              const float gate = sum_kw(col, r), up = sum_kw(col, r + OR);
              p.h[(int64_t)L.plist[L.groups[c.g].start + col] * p.n + row0 + r] = qmm_act(gate, p.act) * up;
            } else {
              qmm_store(p, col, row0 + r, sum_kw(col, r));
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&taken[rw][buf]);
      }
    }
    if constexpr (MODE == kQmmLinear) {
      if (split) {
        // every warp of the CTA is done with the ring
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kQmmWarps) : "memory");
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            if (4 * j + lc < YC) {
              float* q = ys + warp * ys_warp + (4 * j + lc) * WR + 16 * t + lr;
              q[0] = tot[t][j][0];
              q[8] = tot[t][j][1];
            }
          }
        }
      }
    }
  }
  if constexpr (MODE != kQmmUp) {
    if (p.split > 1) {
      // ---- a K split over the cluster: each rank adds its columns' sums into
      // those of its first column, rank 0 adds the ranks' in order
      __syncthreads();
      const int outs = RW * WR * p.M;
      auto place = [&](int i, int& col, int& r) -> float* {
        col = i / (RW * WR);
        r = i - col * (RW * WR);
        return ys + (r / WR) * KW * ys_warp + col * WR + r % WR;
      };
      for (int i = threadIdx.x; i < outs; i += kQmmThreads) {
        int col, r;
        float* q = place(i, col, r);
        float v = q[0];
        for (int k = 1; k < KW; ++k) v += q[k * ys_warp];
        q[0] = v;
      }
      qmm_cluster_sync();
      if (rank == 0) {
        for (int i = threadIdx.x; i < outs; i += kQmmThreads) {
          int col, r;
          const float* q = place(i, col, r);
          float v = q[0];
          for (int k = 1; k < p.split; ++k) v += qmm_ld_cluster(q, (uint32_t)k);
          const int row = cta * tile_rows + r;
          if (row < p.n) qmm_store(p, col, row, v);
        }
      }
      qmm_cluster_sync();  // the leader has read every rank's sums
    }
  }
}

}  // namespace nsq
