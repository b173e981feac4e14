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
// Layout.  A CTA is 8 warps = RW row tiles of 16 weight rows x KW columns of
// 256 weights ("units").  Per step every warp computes one unit; raw weight
// bytes and the prepared activation records of the step arrive by cp.async in
// a ring of shared-memory stages.  Partial sums of the KW warps meet in
// shared memory, those of a K split over a cluster through distributed
// shared memory, always in the same order.
#pragma once

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
constexpr int kQmmThreads = 32 * kQmmWarps;
constexpr int kQmmMaxTok = 16;  // tokens of a group
constexpr int kQmmSmemMax = 227 * 1024 - 64;   // dynamic shared memory of a CTA alone on its SM
constexpr int kQmmSmemHalf = 113 * 1024 - 64;  // of one of two CTAs

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

__device__ __forceinline__ void qmm_cp16(uint32_t dst, const void* src, int bytes, uint64_t pol) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes),
               "l"(pol)
               : "memory");
}
__device__ __forceinline__ void qmm_cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void qmm_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// The oldest of the `stages` - 1 groups in flight has landed.
__device__ __forceinline__ void qmm_wait(int stages) {
  if (stages == 2) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else if (stages == 3) {
    asm volatile("cp.async.wait_group 1;" ::: "memory");
  } else {
    asm volatile("cp.async.wait_group 2;" ::: "memory");
  }
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
// Per format: bytes and weights of a unit of one row, its copies of 16 bytes
// and the pitch of its shared-memory row.  Rows of Q4_0, Q8_0 and Q6_K start
// at any even address, so their copies carry up to 14 bytes before the unit.
// The pitches put the reads of 8 rows x 4 lanes on distinct banks.
template <int TYPE> struct QmmFmt;
template <> struct QmmFmt<NSQ_TYPE_Q4_K> { static constexpr int CB = 144, NCH = 9, PITCH = 144; static constexpr bool aligned = true; };
template <> struct QmmFmt<NSQ_TYPE_Q5_K> { static constexpr int CB = 176, NCH = 11, PITCH = 176; static constexpr bool aligned = true; };
template <> struct QmmFmt<NSQ_TYPE_Q6_K> { static constexpr int CB = 210, NCH = 14, PITCH = 240; static constexpr bool aligned = false; };
template <> struct QmmFmt<NSQ_TYPE_Q4_0> { static constexpr int CB = 144, NCH = 10, PITCH = 176; static constexpr bool aligned = false; };
template <> struct QmmFmt<NSQ_TYPE_Q8_0> { static constexpr int CB = 272, NCH = 18, PITCH = 304; static constexpr bool aligned = false; };

// B operands of MMA steps 2i and 2i+1 for n-tile j (0 for absent tokens).
struct QmmB {
  const uint8_t* rec;  // this lane's token and part of n-tile 0
  int c, flip, count, tok;
  __device__ __forceinline__ uint4 steps(int j, int i) const {
    uint4 b = make_uint4(0, 0, 0, 0);
    if (4 * j + tok < count)
      b = *reinterpret_cast<const uint4*>(rec + 4 * j * kQmmRec + ((((4 * i + c) ^ flip)) << 4));
    return b;
  }
};

// 32-bit word at an even shared-memory address.
__device__ __forceinline__ uint32_t qmm_ld2(const uint8_t* p) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  const uint32_t* b = reinterpret_cast<const uint32_t*>(a & ~uintptr_t(3));
  return __funnelshift_r(b[0], b[1], (uint32_t)(a & 3) * 8);
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

// Adds one unit's products to u[j][row half] (without the token scale s).
// r0, r1: this lane's weight rows lane / 4 and lane / 4 + 8; T: the lane's
// token sums of n-tile 0; nv: valid 32-weight blocks (Q4_0, Q8_0).
template <int TYPE, int LAYOUT, int NT>
__device__ __forceinline__ void qmm_unit(const uint8_t* r0, const uint8_t* r1, const QmmB& B, int nv, float (&u)[NT][2]) {
  const int c = B.c;
  const uint8_t* rows[2] = {r0, r1};

  if constexpr (TYPE == NSQ_TYPE_Q4_K || TYPE == NSQ_TYPE_Q5_K) {
    __half2 sa[2], sb[2];  // scales of sub-blocks 2c and 2c+1, times 2^10 and 2^6
    uint32_t ma[2], mb[2];
    float d[2], dm[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint4 h = *reinterpret_cast<const uint4*>(rows[r]);
      d[r] = h2f((uint16_t)(h.x & 0xFFFF));
      dm[r] = h2f((uint16_t)(h.x >> 16));
      const uint32_t s_lo = h.y & 0x3F3F3F3Fu, m_lo = h.z & 0x3F3F3F3Fu;
      const uint32_t s_hi = (h.w & 0x0F0F0F0Fu) | ((h.y >> 2) & 0x30303030u);
      const uint32_t m_hi = ((h.w >> 4) & 0x0F0F0F0Fu) | ((h.z >> 2) & 0x30303030u);
      const uint32_t s = c < 2 ? s_lo : s_hi;
      const __half2 k1024 = __float2half2_rn(1024.0f), k64 = __float2half2_rn(64.0f);
      sa[r] = __hmul2(__hsub2(qmm_dup1024(s, (2 * c) & 3), k1024), k1024);
      sb[r] = __hmul2(__hsub2(qmm_dup1024(s, (2 * c + 1) & 3), k1024), k64);
      ma[r] = qmm_h2u(__hsub2(qmm_dup1024(m_lo, c), k1024));
      mb[r] = qmm_h2u(__hsub2(qmm_dup1024(m_hi, c), k1024));
    }
    constexpr int QS = TYPE == NSQ_TYPE_Q4_K ? 16 : 48;
    uint32_t q[2][8];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint4 lo = *reinterpret_cast<const uint4*>(rows[r] + QS + 32 * c);
      const uint4 hi = *reinterpret_cast<const uint4*>(rows[r] + QS + 32 * c + 16);
      q[r][0] = lo.x; q[r][1] = lo.y; q[r][2] = lo.z; q[r][3] = lo.w;
      q[r][4] = hi.x; q[r][5] = hi.y; q[r][6] = hi.z; q[r][7] = hi.w;
    }
    [[maybe_unused]] uint32_t qh[2][8];
    if constexpr (TYPE == NSQ_TYPE_Q5_K && LAYOUT == NSQ_Q6K_GGML) {
      // bit 2c (2c+1) of byte l is the fifth bit of weight l of sub-block 2c (2c+1)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint4 lo = *reinterpret_cast<const uint4*>(rows[r] + 16);
        const uint4 hi = *reinterpret_cast<const uint4*>(rows[r] + 32);
        qh[r][0] = lo.x >> (2 * c); qh[r][1] = lo.y >> (2 * c); qh[r][2] = lo.z >> (2 * c); qh[r][3] = lo.w >> (2 * c);
        qh[r][4] = hi.x >> (2 * c); qh[r][5] = hi.y >> (2 * c); qh[r][6] = hi.z >> (2 * c); qh[r][7] = hi.w >> (2 * c);
      }
    } else if constexpr (TYPE == NSQ_TYPE_Q5_K) {
      // NodeStor: bit l of word 2c (2c+1) of qh
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint2 v = *reinterpret_cast<const uint2*>(rows[r] + 16 + 8 * c);
        qh[r][0] = v.x;
        qh[r][1] = v.y;
      }
    }
    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t a[2][4];  // [row]: sub-block 2c (values 0,2 | 1,3), sub-block 2c+1 (the same)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t w = q[r][i], w8 = w >> 8;
        uint32_t v0 = w & 0x000F000Fu, v1 = w8 & 0x000F000Fu, v2 = w & 0x00F000F0u, v3 = w8 & 0x00F000F0u;
        if constexpr (TYPE == NSQ_TYPE_Q5_K && LAYOUT == NSQ_Q6K_GGML) {
          const uint32_t g = qh[r][i];
          v0 |= (g << 4) & 0x00100010u;
          v1 |= (g >> 4) & 0x00100010u;
          v2 |= (g << 7) & 0x01000100u;
          v3 |= (g >> 1) & 0x01000100u;
        } else if constexpr (TYPE == NSQ_TYPE_Q5_K) {
          const uint32_t g = (qh[r][0] >> (4 * i)) & 15u, f = (qh[r][1] >> (4 * i)) & 15u;
          v0 |= (g * 0x00040010u) & 0x00100010u;  // bits 0, 2 -> 4, 20
          v1 |= (g * 0x00020008u) & 0x00100010u;  // bits 1, 3 -> 4, 20
          v2 |= (f * 0x00400100u) & 0x01000100u;
          v3 |= (f * 0x00200080u) & 0x01000100u;
        }
        a[r][0] = qmm_mul2(v0, sa[r]);
        a[r][1] = qmm_mul2(v1, sa[r]);
        a[r][2] = qmm_mul2(v2, sb[r]);
        a[r][3] = qmm_mul2(v3, sb[r]);
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if (j == 0 || 4 * j < B.count) {
          const uint4 b = B.steps(j, i);
          qmm_mma(acc[j], a[0][0], a[1][0], a[0][1], a[1][1], b.x, b.y);
          qmm_mma(acc[j], a[0][2], a[1][2], a[0][3], a[1][3], b.z, b.w);
        }
      }
    }
    float am[NT][4];  // the mins against T
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      am[j][0] = am[j][1] = am[j][2] = am[j][3] = 0.0f;
      if (j == 0 || 4 * j < B.count) {
        uint2 t = make_uint2(0, 0);
        // rec points at the part's operands (0 or 512): hi T at 1024, lo T at 1056
        if (4 * j + B.tok < B.count)
          t = *reinterpret_cast<const uint2*>(B.rec + 4 * j * kQmmRec + (B.flip ? 1056 - 512 : 1024) + 8 * c);
        qmm_mma(am[j], ma[0], ma[1], mb[0], mb[1], t.x, t.y);
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
        u[j][r] = (d[r] * 16384.0f) * (acc[j][2 * r] + acc[j][2 * r + 1]) -
                  (dm[r] * 32.0f) * (am[j][2 * r] + am[j][2 * r + 1]);
    }
  } else if constexpr (TYPE == NSQ_TYPE_Q4_0 || TYPE == NSQ_TYPE_Q8_0) {
    constexpr int BB = TYPE == NSQ_TYPE_Q4_0 ? 18 : 34;
#pragma unroll
    for (int j = 0; j < NT; ++j) u[j][0] = u[j][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t a[2][4];
      float d[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint8_t* blk = rows[r] + BB * i;
        d[r] = i < nv ? h2f((uint16_t)ld_u16(blk)) : 0.0f;
        const uint32_t w = qmm_ld2(blk + 2 + 4 * c);
        if constexpr (TYPE == NSQ_TYPE_Q4_0) {
          // 1024 + q and 1024 + 16 q
          const uint32_t w8 = w >> 8;
          a[r][0] = qmm_off((w & 0x000F000Fu) | 0x64006400u, -1032.0f);
          a[r][1] = qmm_off((w8 & 0x000F000Fu) | 0x64006400u, -1032.0f);
          a[r][2] = qmm_off16((w & 0x00F000F0u) | 0x64006400u, -72.0f);
          a[r][3] = qmm_off16((w8 & 0x00F000F0u) | 0x64006400u, -72.0f);
        } else {
          const uint32_t x = w ^ 0x80808080u, y = qmm_ld2(blk + 18 + 4 * c) ^ 0x80808080u;
          a[r][0] = qmm_off(__byte_perm(x, 0x64646464u, 0x4240), -1152.0f);
          a[r][1] = qmm_off(__byte_perm(x, 0x64646464u, 0x4341), -1152.0f);
          a[r][2] = qmm_off(__byte_perm(y, 0x64646464u, 0x4240), -1152.0f);
          a[r][3] = qmm_off(__byte_perm(y, 0x64646464u, 0x4341), -1152.0f);
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if (j == 0 || 4 * j < B.count) {
          const uint4 b = B.steps(j, i);
          float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          qmm_mma(acc, a[0][0], a[1][0], a[0][1], a[1][1], b.x, b.y);
          qmm_mma(acc, a[0][2], a[1][2], a[0][3], a[1][3], b.z, b.w);
          u[j][0] += d[0] * (acc[0] + acc[1]);
          u[j][1] += d[1] * (acc[2] + acc[3]);
        }
      }
    }
  } else {  // Q6_K
#pragma unroll
    for (int j = 0; j < NT; ++j) u[j][0] = u[j][1] = 0.0f;
    float d[2];
    uint32_t sw[2][4];  // the 16 scale bytes, + 128
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      d[r] = h2f((uint16_t)ld_u16(rows[r] + 208));
      if constexpr (LAYOUT == NSQ_Q6K_NODESTOR) d[r] *= 0.015625f;  // scale (b - 128) / 64
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sw[r][i] = qmm_ld2(rows[r] + 192 + 4 * i);
        if constexpr (LAYOUT == NSQ_Q6K_GGML) sw[r][i] ^= 0x80808080u;
      }
    }
    // scale byte g of row r as f32
    auto scale = [&](int r, int g) {
      return __uint_as_float(__byte_perm(sw[r][g >> 2], 0x4B000000u, 0x7440u | (uint32_t)(g & 3))) - 8388736.0f;
    };
    auto group = [&](int j, const uint32_t (&a)[2][2], uint32_t b0, uint32_t b1, float s0, float s1) {
      float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      qmm_mma(acc, a[0][0], a[1][0], a[0][1], a[1][1], b0, b1);
      u[j][0] += s0 * (acc[0] + acc[1]);
      u[j][1] += s1 * (acc[2] + acc[3]);
    };
    if constexpr (LAYOUT == NSQ_Q6K_GGML) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {  // (half n, 16-group of its runs of 32)
        const int n = p >> 1, g = p & 1;
        uint32_t a[4][2][2];  // [run t][row][values 0,2 | 1,3]
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t A = qmm_ld2(rows[r] + 64 * n + 16 * g + 4 * c);
          const uint32_t Bw = qmm_ld2(rows[r] + 64 * n + 32 + 16 * g + 4 * c);
          const uint32_t H = qmm_ld2(rows[r] + 128 + 32 * n + 16 * g + 4 * c);
          const uint32_t A8 = A >> 8, B8 = Bw >> 8, Hl4 = H << 4, Hl2 = H << 2, Hr4 = H >> 4, Hr6 = H >> 6;
          constexpr uint32_t kL = 0x000F000Fu, kH = 0x00F000F0u, kB = 0x64006400u;
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
          if (j == 0 || 4 * j < B.count) {
            const uint4 b0 = B.steps(j, 2 * p), b1 = B.steps(j, 2 * p + 1);
            group(j, a[0], b0.x, b0.y, s[0][0], s[0][1]);
            group(j, a[1], b0.z, b0.w, s[1][0], s[1][1]);
            group(j, a[2], b1.x, b1.y, s[2][0], s[2][1]);
            group(j, a[3], b1.z, b1.w, s[3][0], s[3][1]);
          }
        }
      }
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
            const uint32_t lo = __byte_perm(ld_u16(rows[r] + 8 * g + 2 * c), 0, 0x4140);
            const uint32_t hb = ld_u8(rows[r] + 128 + 4 * g + c);
            // bits 0-1, 4-5 and 2-3, 6-7 of hb
            a[t][r][0] = qmm_off((lo & 0x000F000Fu) | (((hb * 0x00010010u) & 0x00300030u) | 0x64006400u), -1056.0f);
            a[t][r][1] = qmm_off(((lo >> 4) & 0x000F000Fu) | (((hb * 0x00004004u) & 0x00300030u) | 0x64006400u), -1056.0f);
            s[t][r] = scale(r, g);
          }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if (j == 0 || 4 * j < B.count) {
            const uint4 b = B.steps(j, i);
            group(j, a[0], b.x, b.y, s[0][0], s[0][1]);
            group(j, a[1], b.z, b.w, s[1][0], s[1][1]);
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      u[j][0] *= d[0];
      u[j][1] *= d[1];
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
  int32_t* ids = scratch;
  float* wts = reinterpret_cast<float*>(scratch + P);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool first = blockIdx.x == 0;
  if (p.score >= 0) {
    for (int m = warp; m < p.M; m += kQmmWarps) {
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
  L.ngroups = *p.ngroups;
  for (int q = threadIdx.x; q < P; q += kQmmThreads) {
    if (q < L.ngroups) L.groups[q] = p.groups[q];
    L.plist[q] = p.plist[q];
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

// Bytes of shared memory.
__host__ __device__ inline size_t qmm_stage_bytes(int pitch, int KW, int TS) {
  return (size_t)kQmmWarps * 16 * pitch + (size_t)KW * TS * kQmmRec;
}
inline size_t qmm_lists_bytes(int P) { return (size_t)P * (sizeof(QmmGroup) + 8); }

// One task is one row tile (of one group for kQmmUp, of all groups for
// kQmmDown); its units are (group, 256 of K).  A cluster of `split` CTAs
// shares a task's units.
template <int TYPE, int LAYOUT, int NT>
__global__ void __launch_bounds__(kQmmThreads, 2) qmm_kernel(const QmmParams p) {
  using F = QmmFmt<TYPE>;
  constexpr int BB = Fmt<TYPE>::BB;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int s_n;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int KW = p.KW, RW = p.RW, S = p.stages, TS = p.TS, YC = p.YC;
  const int kw = warp % KW, rw = warp / KW;
  const size_t stage_bytes = qmm_stage_bytes(F::PITCH, KW, TS);
  float* ys = reinterpret_cast<float*>(smem + S * stage_bytes);  // [warp][YC][16]
  float* red = ys + (size_t)kQmmWarps * YC * 16;                 // [YC][16 RW], for a split K
  uint8_t* lists_mem = reinterpret_cast<uint8_t*>(red + (p.split > 1 ? YC * 16 * RW : 0));
  const int rank = p.split > 1 ? (int)qmm_cluster_rank() : 0;
  const int cta = blockIdx.x / p.split, nctas = gridDim.x / p.split;
  const uint64_t pol = l2_policy_evict_first();
  const int tile_rows = p.mode == kQmmUp ? 8 * RW : 16 * RW;
  const int tiles = (int)((p.n + tile_rows - 1) / tile_rows);

  QmmLists L{};
  if (p.mode == kQmmUp) {
    qmm_dep_wait();
    qmm_dep_launch();
    L = qmm_build_lists(p, lists_mem, reinterpret_cast<int32_t*>(smem), &s_n);
  } else if (p.mode == kQmmDown) {
    qmm_dep_wait();
    qmm_dep_launch();
    L = qmm_load_lists(p, lists_mem);
  } else {
    L.ngroups = 1;
  }
  const int tasks = p.mode == kQmmUp ? tiles * L.ngroups : tiles;
  const int units = p.mode == kQmmDown ? L.ngroups * p.nsb : p.nsb;
  const int u0 = (int)((int64_t)units * rank / p.split), u1 = (int)((int64_t)units * (rank + 1) / p.split);
  const int steps = max(1, (units / p.split + (units % p.split ? 1 : 0) + KW - 1) / KW);

  auto group_of = [&](int task, int u, int& sb) {  // group of a task's unit
    if (p.mode == kQmmDown) {
      const int g = u / p.nsb;
      sb = u - g * p.nsb;
      return g;
    }
    sb = u;
    return p.mode == kQmmUp ? task / tiles : 0;
  };
  auto row_base = [&](int task) { return (int64_t)(p.mode == kQmmUp ? task % tiles : task) * tile_rows; };
  // first byte of the unit in weight row r of this warp (r < 16)
  auto unit_ptr = [&](int expert, int64_t base, int r, int sb) {
    const uint8_t* w = p.w0;
    int64_t row;
    if (p.mode == kQmmUp) {
      row = base + rw * 8 + (r & 7);
      if (r >= 8) w = p.w1;
    } else {
      row = base + rw * 16 + r;
    }
    if (row >= p.n) row = p.n - 1;  // rows past the end repeat the last one; their sums are not written
    return w + ((int64_t)expert * p.n + row) * p.rb + (int64_t)sb * F::CB;
  };
  auto issue_w = [&](int task, int step, int stage) {
    const int u = u0 + step * KW + kw;
    if (task >= tasks || u >= u1) return;
    int sb;
    const int g = group_of(task, u, sb);
    const int expert = p.mode == kQmmLinear ? 0 : L.groups[g].expert;
    const int64_t base = row_base(task);
    const uint32_t dst = smem_u32(smem + stage * stage_bytes + (size_t)warp * 16 * F::PITCH);
#pragma unroll
    for (int i = 0; i < (16 * F::NCH + 31) / 32; ++i) {
      const int idx = lane + 32 * i;
      const int r = idx / F::NCH, ch = idx % F::NCH;
      if (r < 16) {
        const uint8_t* src = unit_ptr(expert, base, r, sb);
        if constexpr (F::aligned) {
          qmm_cp16(dst + r * F::PITCH + 16 * ch, src + 16 * ch, 16, pol);
        } else {
          const int mis = (int)(reinterpret_cast<uintptr_t>(src) & 15);
          int need = F::CB;
          if constexpr (Fmt<TYPE>::QK == 32) need = min(8, p.nblk - 8 * sb) * BB;
          if (16 * ch < mis + need) {
            const uint8_t* a = src - mis + 16 * ch;
            const uint8_t* end = (p.mode == kQmmUp && r >= 8 ? p.w1 : p.w0) + p.wbytes;
            qmm_cp16(dst + r * F::PITCH + 16 * ch, a, (int)min((int64_t)16, (int64_t)(end - a)), pol);
          }
        }
      }
    }
  };
  auto issue_b = [&](int task, int step, int stage) {
    const int u = u0 + step * KW + kw;
    if (task >= tasks || u >= u1) return;
    int sb;
    const int g = group_of(task, u, sb);
    const int count = p.mode == kQmmLinear ? p.M : L.groups[g].count;
    const int start = p.mode == kQmmLinear ? 0 : L.groups[g].start;
    const uint32_t dst =
        smem_u32(smem + stage * stage_bytes + (size_t)kQmmWarps * 16 * F::PITCH + (size_t)kw * TS * kQmmRec);
    constexpr int RC = kQmmRec / 16;
    for (int idx = rw * 32 + lane; idx < count * RC; idx += RW * 32) {
      const int t = idx / RC, ch = idx - t * RC;
      int row = t;
      if (p.mode != kQmmLinear) {
        row = L.plist[start + t];
        if (p.mode == kQmmUp) row /= p.top_k;
      }
      qmm_cp16(dst + t * kQmmRec + 16 * ch, p.recs + ((int64_t)row * p.nsb + sb) * kQmmRec + 16 * ch);
    }
  };

  // producer cursor
  int ptask = cta, pstep = 0;
  auto advance = [&](int& task, int& step) {
    if (++step == steps) {
      step = 0;
      task += nctas;
    }
  };
  for (int s = 0; s < S - 1; ++s) {
    issue_w(ptask, pstep, s);
    advance(ptask, pstep);
  }
  if (p.mode == kQmmLinear) {
    // the weights do not depend on the kernels before; the records do
    qmm_dep_wait();
    qmm_dep_launch();
  }
  {
    int t = cta, st = 0;
    for (int s = 0; s < S - 1; ++s) {
      issue_b(t, st, s);
      qmm_commit();
      advance(t, st);
    }
  }

  float tot[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j) tot[j][0] = tot[j][1] = 0.0f;
  float* my_ys = ys + (size_t)warp * YC * 16;
  const int lr = lane >> 2, lc = lane & 3;
  int stage = 0;
  for (int task = cta, step = 0; task < tasks;) {
    qmm_wait(S);
    __syncthreads();
    {
      const int ps = stage == 0 ? S - 1 : stage - 1;
      issue_w(ptask, pstep, ps);
      issue_b(ptask, pstep, ps);
      qmm_commit();
      advance(ptask, pstep);
    }
    if (p.mode == kQmmDown && step == 0) {
      for (int i = lane; i < YC * 16; i += 32) my_ys[i] = 0.0f;
      __syncwarp();
    }
    const int u = u0 + step * KW + kw;
    if (u < u1) {
      int sb;
      const int g = group_of(task, u, sb);
      const int count = p.mode == kQmmLinear ? p.M : L.groups[g].count;
      const uint8_t* wst = smem + stage * stage_bytes + (size_t)warp * 16 * F::PITCH;
      const uint8_t* bst = smem + stage * stage_bytes + (size_t)kQmmWarps * 16 * F::PITCH + (size_t)kw * TS * kQmmRec;
      const uint8_t* r0 = wst + lr * F::PITCH;
      const uint8_t* r1 = r0 + 8 * F::PITCH;
      if constexpr (!F::aligned) {
        const int expert = p.mode == kQmmLinear ? 0 : L.groups[g].expert;
        const int64_t base = row_base(task);
        r0 += reinterpret_cast<uintptr_t>(unit_ptr(expert, base, lr, sb)) & 15;
        r1 += reinterpret_cast<uintptr_t>(unit_ptr(expert, base, lr + 8, sb)) & 15;
      }
      QmmB B;
      B.c = lc;
      B.flip = (lr & 1) * 4;
      B.tok = lr >> 1;
      B.count = count;
      B.rec = bst + B.tok * kQmmRec + (lr & 1) * 512;
      float uv[NT][2];
      qmm_unit<TYPE, LAYOUT, NT>(r0, r1, B, min(8, p.nblk - 8 * sb), uv);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int t = 4 * j + lc;
        if (t < count) {
          const float s = *reinterpret_cast<const float*>(bst + t * kQmmRec + 1088);
          if (p.mode == kQmmDown) {
            const int pick = L.groups[g].start + t;
            const float w = L.pwts[pick];
            float* q = my_ys + (L.plist[pick] / p.top_k) * 16 + lr;
            q[0] += w * (s * uv[j][0]);
            q[8] += w * (s * uv[j][1]);
          } else {
            tot[j][0] += s * uv[j][0];
            tot[j][1] += s * uv[j][1];
          }
        }
      }
      __syncwarp();
    }
    if (step == steps - 1) {
      // ---- the task's sums
      if (p.mode != kQmmDown) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if (4 * j + lc < YC) {
            my_ys[(4 * j + lc) * 16 + lr] = tot[j][0];
            my_ys[(4 * j + lc) * 16 + lr + 8] = tot[j][1];
          }
          tot[j][0] = tot[j][1] = 0.0f;
        }
      }
      __syncthreads();
      const int64_t base = row_base(task);
      auto sum_kw = [&](int col, int r) {  // over the KW warps of row r (0 .. 16 RW - 1)
        const float* q = ys + ((size_t)(r >> 4) * KW * YC + col) * 16 + (r & 15);
        float v = q[0];
        for (int k = 1; k < KW; ++k) v += q[(size_t)k * YC * 16];
        return v;
      };
      if (p.mode == kQmmUp) {
        const int g = task / tiles, count = L.groups[g].count, start = L.groups[g].start;
        for (int i = threadIdx.x; i < tile_rows * count; i += kQmmThreads) {
          const int col = i / tile_rows, r = i - col * tile_rows;
          const int64_t row = base + r;
          if (row < p.n) {
            const int q = (r >> 3) * 16 + (r & 7);
            const float gate = sum_kw(col, q), up = sum_kw(col, q + 8);
            p.h[(int64_t)L.plist[start + col] * p.n + row] = qmm_act(gate, p.act) * up;
          }
        }
      } else {
        const int cols = p.M;
        if (p.split > 1) {
          for (int i = threadIdx.x; i < tile_rows * cols; i += kQmmThreads) red[i] = sum_kw(i / tile_rows, i % tile_rows);
          qmm_cluster_sync();
        }
        if (rank == 0) {
          for (int i = threadIdx.x; i < tile_rows * cols; i += kQmmThreads) {
            const int col = i / tile_rows, r = i - col * tile_rows;
            const int64_t row = base + r;
            if (row < p.n) {
              float v;
              if (p.split > 1) {
                v = red[i];
                for (int k = 1; k < p.split; ++k) v += qmm_ld_cluster(red + i, (uint32_t)k);
              } else {
                v = sum_kw(col, r);
              }
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
          }
        }
        if (p.split > 1) qmm_cluster_sync();  // the leader has read every rank's sums
      }
    }
    advance(task, step);
    if (++stage == S) stage = 0;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

}  // namespace nsq
