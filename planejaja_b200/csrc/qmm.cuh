// qmm.cuh -- products of a few tokens with GGUF-quantised weights, exact to
// about 3e-7 (f32 outputs), for the linear operator and the two products of
// a mixture-of-experts layer.
//
//   out[t, n] = sum_k x[t, k] * W[n, k]         t: up to 16 tokens of a group
//
// Mathematics.  x = s X with integers |X| < 2^23 and one scale s per (token,
// 256 of K); X is three signed bytes ("limbs", X = sum 256^l X_l, each
// -128..127).  The formats' integers meet the limbs in mma.sync m16n8k32 / k16
// (u8 x s8, exact s32 sums): 16 weight rows as A and eight columns as B,
// which are two tokens of four limbs (the fourth a copy, not used) or, from
// five tokens on, one limb of eight tokens (six such tiles for 9 to 16 tokens,
// over weights unpacked once: 14336 x 4096 Q4_K, 16 tokens 31 us; by eights 33).  The integer scale of a group
// multiplies its sum in s32 too, so the first rounding comes after 256 weights:
//   Q4_K, Q5_K  sum sc_j (sum q X_l): |sum| < 2^29;  d times it in f32.  The
//               mins enter through the limb sums T of 16 activations (at most
//               2048, exact in fp16):  - dmin * sum m T  by one fp16 MMA
//   Q6_K        the same with 16-weight groups; q - 32 through T
//   Q4_0, Q8_0  one f32 scale per 32 weights; q - 8 through T
// With max the largest of its 256 an activation v is off by at most max / 2^22:
// 1 / s and s are each off by 2^-24 of themselves (2 |v| / 2^24), the product
// v / s, below 2^23, by a quarter and its rounding to X by a half of a step s =
// max / 8355710 (1.51 max / 2^24); small v lose little more than the half step,
// max / 2^24.  (max below 2^-63: s is a power of two, the half step at most
// max / 2^22, and below 2^-120 it is 2^-142.)  So values far below an outlier
// of their 256 keep fewer bits than f32 has.  A limb's f32 value is off by
// 2^-24 of the limb's sum: norm errors of a product are about 2e-7.
//
// Measured on B200: the byte MMA (4096 products), the fp16 MMA (2048), take 8
// cycles of a scheduler each; logic, permutes, IMAD and fp16x2 take 2.  A
// first form with fp16 operands (x as hi + lo, two columns a token, q * sc in
// fp16) needs a multiply or subtract per pair of weights beside the mask; this
// one masks four weights at a time.  Counted for Q4_K and one n-tile of tokens,
// 290 against about 170 cycles per 16 x 256 weights.
//
// What bounds it.  Up to 4 tokens HBM and the start and end of a kernel: two
// experts' [14336 x 4096] Q4_K in 61 us are 3.2 TB/s with 10 us of routing and
// starts; Q5_K [28672 x 8192], 3 tokens, 47 us = 3.4 TB/s, its fifth bits' logic.
// From five tokens on instructions: with groups of up to 8 tokens (three
// n-tiles) 400 per 16 x 256 weights, loads and bookkeeping included, at 0.6 a
// cycle and scheduler; 16 tokens over 8 experts 301 us = 3.0 TB/s.
//
// Layout.  A CTA is 8 warps = RW row tiles of 16 MT weight rows x KW columns.
// A task is a tile of 16 MT RW rows; its units of 256 weights of K are dealt
// to the columns in turn.  A column has its own ring of shared-memory slots
// (the weight bytes of its RW tiles and the activation records of the unit)
// behind full mbarriers.  Every warp refills its own rows as soon as it has
// used them: one 2-D TMA box where rows start 16-byte aligned, else 16-byte
// asynchronous copies; the column's warps refill the records in turn.  (A
// producer warp would cost a ninth warp's registers, 96 instead of 128 a
// thread, and ties the columns together.)  The partial sums of the KW columns
// meet in shared memory.  The CTAs share all tasks' steps evenly (a CTA may
// hold parts of two tasks; with a task's steps never divided 16 tokens over 8
// experts take 575 us instead of 301), and a divided task's parts meet in the
// workspace, where the last to arrive adds them up in the CTAs' order.  No CTA
// waits for another; every other wait is bounded.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "nsq_common.cuh"

namespace nsq {

// ---------------------------------------------------------------------------
// Prepared activations: one record per (row, 256 of K).
//   [0, 768)    three limbs of 256 bytes: 16-byte unit 4i + c = the operands
//               of lane c of each quad in turn i; units of the middle limb are
//               exchanged (^ 4), so that neighbouring limbs of a token, which
//               neighbouring lanes read, lie in different banks
//   [768, 864)  T, the sums of 16 consecutive X_l, as fp16: per limb and lane
//               c the groups 2c, 2c+1, 2c+8, 2c+9
//   [864, 868)  s (NaN when a value is not finite)
// Which k a place holds goes by the format of the weights (QmmOrder).  In
// shared memory records lie 960 bytes apart: neighbouring tokens then are in
// different banks too.
constexpr int kQmmRec = 880;
constexpr int kQmmRecPitch = 960;
constexpr int kQmmRecT = 768;
constexpr int kQmmRecS = 864;
constexpr int kQmmWarps = 8;
constexpr int kQmmThreads = 32 * kQmmWarps;
constexpr int kQmmMaxStages = 4;
constexpr int kQmmCtl = 1024;  // barriers and counters at the start of the shared memory
constexpr int kQmmMaxTok = 16;  // tokens of a group
constexpr int kQmmSmemMax = 227 * 1024 - 1024;  // dynamic shared memory of a CTA alone on its SM
constexpr int kQmmSmemHalf = 113 * 1024;         // of one of two CTAs (a CTA takes 1 KB more for itself)

enum QmmOrder : int { kOrdK45 = 0, kOrd32 = 1, kOrdQ6 = 2, kOrdQ6N = 3 };

__host__ __device__ constexpr int qmm_order(int type, int layout) {
  return type == NSQ_TYPE_Q4_K || type == NSQ_TYPE_Q5_K ? kOrdK45
         : type == NSQ_TYPE_Q6_K                        ? (layout == NSQ_Q6K_GGML ? kOrdQ6 : kOrdQ6N)
                                                        : kOrd32;
}
// First k of the two runs of four in half h (8 bytes per limb) of unit (i, c).
__device__ __forceinline__ void qmm_runs(int order, int i, int c, int h, int& k0, int& k1) {
  if (order == kOrdK45) {  // sub-block 2i + h, weights 8c .. 8c + 7
    k0 = 64 * i + 32 * h + 8 * c;
    k1 = k0 + 4;
  } else if (order == kOrd32) {  // block 2i + h, weights 4c .. and 16 + 4c ..
    k0 = 32 * (2 * i + h) + 4 * c;
    k1 = k0 + 16;
  } else if (order == kOrdQ6) {  // half i / 2, 16-group i % 2 of its runs of 32 number 2h, 2h + 1
    k0 = 128 * (i >> 1) + 64 * h + 16 * (i & 1) + 4 * c;
    k1 = k0 + 32;
  } else {  // groups 4i + 2h, 4i + 2h + 1
    k0 = 16 * (4 * i + 2 * h) + 4 * c;
    k1 = k0 + 16;
  }
}

__device__ __forceinline__ uint32_t qmm_h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 qmm_u2h(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// One warp turns 256 values (those at and after `valid` count as 0) into a
// record.  FRESH: values that other CTAs of this kernel wrote, read from L2.
template <typename T, bool FRESH = false>
__device__ __forceinline__ void qmm_make_record(const T* src, int valid, int order, uint8_t* rec, int lane) {
  const int i = lane >> 3, c = (lane >> 1) & 3, h = lane & 1;
  int k[2];
  qmm_runs(order, i, c, h, k[0], k[1]);
  float v[8];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if constexpr (sizeof(T) == 4) {
      const bool wide = ((reinterpret_cast<uintptr_t>(src) & 15) == 0) && k[r] + 4 <= valid;
      if (wide) {
        const float4* q = reinterpret_cast<const float4*>(src + k[r]);
        const float4 f = FRESH ? __ldcg(q) : *q;
        v[4 * r] = f.x; v[4 * r + 1] = f.y; v[4 * r + 2] = f.z; v[4 * r + 3] = f.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[4 * r + e] = k[r] + e < valid ? (FRESH ? __ldcg(src + k[r] + e) : src[k[r] + e]) : 0.0f;
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
  // the largest value becomes kTop, one below the largest X = 127 (256^2 + 256
  // + 1): its product with the rounded 1 / s may be half above.
  // Values below 2^-63 get a power of two instead (s may be subnormal, and
  // exact; 1 / s may not overflow, so they are scaled twice), with |X| < 2^22;
  // below 2^-120 it stays and values lose bits at 2^-141.
  constexpr float kTop = 8355710.0f;
  const int E = (int)(mx >> 23);
  float s, pre, inv;
  if (E >= 64) {
    const float m = __uint_as_float(mx);
    pre = 1.0f;
    inv = kTop / m;
    s = m / kTop;
  } else {
    const int F = max(E, 7);  // s = 2^(F - 148)
    pre = 18446744073709551616.0f;  // 2^64
    inv = __uint_as_float((uint32_t)(127 + 148 - 64 - F) << 23);
    s = F >= 22 ? __uint_as_float((uint32_t)(F - 21) << 23) : __uint_as_float(1u << (F + 1));
  }
  if (mx >= 0x7F800000u) s = __uint_as_float(0x7FC00000u);  // infinity or NaN: this token alone is spoilt
  int sum[2][3];
  uint32_t limb[2][3];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    uint32_t y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int X = __float2int_rn((v[4 * r + e] * pre) * inv);
      y[e] = ((uint32_t)X + 0x00008080u) ^ 0x00008080u;  // bytes 0, 1, 2 are the limbs
    }
    // transpose: byte l of the four words
    const uint32_t a = __byte_perm(y[0], y[1], 0x5140), b = __byte_perm(y[2], y[3], 0x5140);
    limb[r][0] = __byte_perm(a, b, 0x5410);
    limb[r][1] = __byte_perm(a, b, 0x7632);
    limb[r][2] = __byte_perm(__byte_perm(y[0], y[1], 0x0062), __byte_perm(y[2], y[3], 0x0062), 0x5410);
#pragma unroll
    for (int l = 0; l < 3; ++l) sum[r][l] = dp4a_ss(limb[r][l], 0x01010101u, 0);
  }
#pragma unroll
  for (int l = 0; l < 3; ++l)
    *reinterpret_cast<uint2*>(rec + 256 * l + 16 * ((4 * i + c) ^ (4 * (l & 1))) + 8 * h) =
        make_uint2(limb[0][l], limb[1][l]);
  // T: in the K45 order the lane's 8 values and its neighbour's (c ^ 1) are a
  // group; else each run is a quarter of one, over c
#pragma unroll
  for (int l = 0; l < 3; ++l) {
    int t0 = order == kOrdK45 ? sum[0][l] + sum[1][l] : sum[0][l], t1 = sum[1][l];
    t0 += __shfl_xor_sync(0xffffffffu, t0, 2);
    t1 += __shfl_xor_sync(0xffffffffu, t1, 2);
    if (order != kOrdK45) {
      t0 += __shfl_xor_sync(0xffffffffu, t0, 4);
      t1 += __shfl_xor_sync(0xffffffffu, t1, 4);
    }
    auto put = [&](int g, int t) {
      *reinterpret_cast<__half*>(rec + kQmmRecT + 32 * l + ((g & 7) >> 1) * 8 + ((g & 1) + (g >= 8 ? 2 : 0)) * 2) =
          __int2half_rn(t);
    };
    if (order == kOrdK45) {
      if ((c & 1) == 0) put(k[0] >> 4, t0);
    } else if (c == 0) {
      put(k[0] >> 4, t0);
      put(k[1] >> 4, t1);
    }
  }
  if (lane == 0) *reinterpret_cast<float*>(rec + kQmmRecS) = s;
}

// ---------------------------------------------------------------------------
struct QmmGroup {
  int expert, start, count, pad;  // tokens plist[start .. start + count)
};

enum QmmMode : int { kQmmLinear = 0, kQmmUp = 1, kQmmDown = 2 };

struct QmmParams {
  int mode, RW, KW, stages;
  int TS;        // token slots of a unit (the largest group)
  int YC;        // columns of the partial sums: TS, or M for kQmmDown
  int M, top_k;  // tokens; picks per token
  int act, dtype;
  int nsb;       // units of a weight row: ceil(K / 256)
  int nblk;      // K / 32
  int rows_aligned;  // every row starts 16-byte aligned: TMA boxes
  int PB;            // buffers of partial sums
  int whole;         // tasks are not divided
  float* parts;      // sums of divided tasks, [CTA][2][row tile][YC][WR]
  int32_t* tickets;  // steps of them that are done, [CTA][row tile], zeroed by the kernel before
  int64_t n, K, rb;          // rows of one expert, K, bytes of a row
  const uint8_t* w0;         // weights (kQmmUp: gate)
  const uint8_t* w1;         // kQmmUp: up
  int64_t wbytes;            // bytes of all experts' rows
  const uint8_t* recs;       // activation records [row][nsb]
  // kQmmLinear
  const void* x;             // [M][K]: every CTA makes all records itself, there are few (else NULL: see recs)
  int order;                 // of their values
  const float* bias;
  // kQmmLinear, kQmmDown
  const void* residual;
  void* y;
  // kQmmUp, kQmmDown
  float* h;                  // [M * top_k][n] (written by kQmmUp)
  uint8_t* recs_h;           // its records for kQmmDown, made by kQmmUp's last finisher of each 256 rows,
  int32_t* done;             // counted here, [group][256 rows], zeroed by the routing kernel
  int order_h;
  int E, score;              // experts; -1: ids and wts are given, else they are outputs
  const double* logits;      // [M][E]
  const float* sel_bias;
  float scale;
  int32_t* ids;
  float* wts;
  QmmGroup* groups;          // lists of the picks by expert, written by kQmmUp
  int32_t* plist;
  float* pwts;
  int32_t* ptok;
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

// 16 bytes to shared memory; those past the first `bytes` are zeros and not read.
__device__ __forceinline__ void qmm_cp_async(uint32_t dst, const uint8_t* src, int bytes, uint64_t pol) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes), "l"(pol)
               : "memory");
}
// One arrival when all copies of this thread so far have landed.
__device__ __forceinline__ void qmm_cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// fp16 MMA (mins against T), accumulating from zero.
__device__ __forceinline__ void qmm_mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, "
      "%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// Byte MMAs from the constant `init`: weights u8 (or s8) x limbs s8, 32 and 16 of K.
template <bool SIGNED>
__device__ __forceinline__ void qmm_mma_k32(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1, int init) {
  if constexpr (SIGNED) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, "
        "%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(init));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, "
        "%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(init));
  }
}
__device__ __forceinline__ void qmm_mma_k16(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%7, %7, %7, %7};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(b0), "r"(0));
}

static __device__ __noinline__ float qmm_act(float v, int act) {
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
// Two row tiles share a unit's bookkeeping; the wider formats have one, for
// the depth of the ring.
template <int TYPE> struct QmmFmt;
template <> struct QmmFmt<NSQ_TYPE_Q4_K> { static constexpr int CB = 144, PA = 160, PG = 160, MT = 2; };
template <> struct QmmFmt<NSQ_TYPE_Q5_K> { static constexpr int CB = 176, PA = 176, PG = 176, MT = 2; };
template <> struct QmmFmt<NSQ_TYPE_Q6_K> { static constexpr int CB = 210, PA = 240, PG = 240, MT = 1; };
template <> struct QmmFmt<NSQ_TYPE_Q4_0> { static constexpr int CB = 144, PA = 144, PG = 176, MT = 2; };
template <> struct QmmFmt<NSQ_TYPE_Q8_0> { static constexpr int CB = 272, PA = 272, PG = 304, MT = 1; };

// Row tiles of a warp for groups of up to TS tokens: one beyond 4 tokens for
// the 32-weight formats and beyond 8 for all.  Two of them share a unit's
// bookkeeping, some 100 of 470 instructions (16 tokens, 8 experts of
// [14336 x 4096] Q4_K and Q6_K: 342 -> 313 us).
template <int TYPE>
__host__ __device__ constexpr int qmm_tiles(int TS) {
  return TS > 8 || (TS > 4 && Fmt<TYPE>::QK == 32) ? 1 : QmmFmt<TYPE>::MT;
}

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

// Where this lane (column n = lane / 4) reads the B operands of n-tile j.
//   LIMBS == false: tile j holds tokens first + 2j and first + 2j + 1, column n
//                   limb n % 4 of token first + 2j + n / 4 (limb 3: limb 0
//                   again, its sums are not used)
//   LIMBS == true:  tile j holds limb j % 3 of token first + 8 (j / 3) + n
// Columns of absent tokens hold what was there; their sums are not used.
template <bool LIMBS>
struct QmmB {
  uint32_t base[2];  // units 4i + c of even and odd i (less 64 i), of the limb with its units in order
  uint32_t t;        // the sums T
  float k256;        // what the second limb of a pair of columns counts
  __device__ __forceinline__ QmmB(uint32_t recs, int first, int n, int c) {
    if constexpr (LIMBS) {
      const uint32_t r = recs + (first + n) * kQmmRecPitch;
      base[0] = base[1] = r + 16 * c;
      t = r + kQmmRecT + 8 * c;
    } else {
      const int limb = (n & 3) == 3 ? 0 : n & 3, flip = (limb & 1) * 64;
      const uint32_t r = recs + (first + (n >> 2)) * kQmmRecPitch;
      base[0] = r + 256 * limb + 16 * c + flip;
      base[1] = r + 256 * limb + 16 * c - flip;
      t = r + kQmmRecT + 32 * limb + 8 * c;
    }
    k256 = c & 1 ? 0.0f : 256.0f;
  }
  __device__ __forceinline__ uint4 unit(int j, int i) const {
    // the middle limb's units are exchanged
    if constexpr (LIMBS)
      return qmm_lds<uint4>(base[0] + j / 3 * 8 * kQmmRecPitch + 256 * (j % 3) + (j % 3 == 1 ? 64 * (i ^ 1) : 64 * i));
    return qmm_lds<uint4>(base[i & 1] + 2 * kQmmRecPitch * j + 64 * i);
  }
  __device__ __forceinline__ uint2 sums(int j) const {
    return qmm_lds<uint2>(t + (LIMBS ? j / 3 * 8 * kQmmRecPitch + 32 * (j % 3) : 2 * kQmmRecPitch * j));
  }
};
// Values of a lane per row half: one of a token's two limb pairs per tile, or
// (LIMBS, three tiles) two whole tokens, 2c and 2c + 1.
template <int NI, bool LIMBS>
constexpr int kQmmVals = LIMBS ? 2 * NI / 3 : NI;
// u += k * (the tiles' sums f as values)
template <int NI, bool LIMBS>
__device__ __forceinline__ void qmm_add(float (&u)[kQmmVals<NI, LIMBS>][2], const float (&k)[2], const float (&f)[NI][4],
                                        float k256) {
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if constexpr (LIMBS) {
#pragma unroll
      for (int q = 0; q < kQmmVals<NI, LIMBS>; ++q) {
        const int e = 2 * r + (q & 1), j = 3 * (q >> 1);
        u[q][r] = fmaf(k[r], fmaf(65536.0f, f[j + 2][e], fmaf(256.0f, f[j + 1][e], f[j][e])), u[q][r]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NI; ++j) u[j][r] = fmaf(k[r], fmaf(k256, f[j][2 * r + 1], f[j][2 * r]), u[j][r]);
    }
  }
}

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

// Byte b (a constant) of w as an unsigned or signed int.
__device__ __forceinline__ int qmm_u8(uint32_t w, int b) { return (int)__byte_perm(w, 0, 0x4440u | (uint32_t)b); }
template <int b>
__device__ __forceinline__ int qmm_s8(uint32_t w) {
  int v;  // a selector's top bit repeats the byte's sign
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(v) : "r"(w), "n"(0x8880 + 0x1111 * b));
  return v;
}
// One row tile's products of a unit for NI n-tiles: the values u (see QmmB)
// per row half, without the token scale.  o: the shared-memory offsets of this
// lane's weight rows lane / 4 and lane / 4 + 8; c = lane % 4; nv: valid
// 32-weight blocks (Q4_0, Q8_0).
template <int TYPE, int LAYOUT, int NI, bool LIMBS>
__device__ __forceinline__ void qmm_unit(const uint32_t (&o)[2], int c, const QmmB<LIMBS>& B, int nv,
                                         float (&u)[kQmmVals<NI, LIMBS>][2]) {
#pragma unroll
  for (int q = 0; q < kQmmVals<NI, LIMBS>; ++q) u[q][0] = u[q][1] = 0.0f;
  // u += k * (A against the sums T)
  auto against_t = [&](uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const float (&k)[2]) {
    float am[NI][4];
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const uint2 b = B.sums(j);
      qmm_mma_f16(am[j], a0, a1, a2, a3, b.x, b.y);
    }
    qmm_add<NI, LIMBS>(u, k, am, B.k256);
  };
  if constexpr (TYPE == NSQ_TYPE_Q4_K || TYPE == NSQ_TYPE_Q5_K) {
    const __half2 k1024 = __float2half2_rn(1024.0f);
    uint32_t sc[2][2];  // [row]: scales of sub-blocks 0..3 and 4..7
    float d[2];
    {
      uint32_t ma[2], mb[2];
      float dm[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint4 h = qmm_lds<uint4>(o[r]);
        d[r] = h2f((uint16_t)(h.x & 0xFFFF)) * (TYPE == NSQ_TYPE_Q4_K ? 0.0625f : 1.0f);
        dm[r] = -h2f((uint16_t)(h.x >> 16));
        sc[r][0] = h.y & 0x3F3F3F3Fu;
        sc[r][1] = (h.w & 0x0F0F0F0Fu) | ((h.y >> 2) & 0x30303030u);
        const uint32_t m_lo = h.z & 0x3F3F3F3Fu, m_hi = ((h.w >> 4) & 0x0F0F0F0Fu) | ((h.z >> 2) & 0x30303030u);
        ma[r] = qmm_h2u(__hsub2(qmm_dup1024(m_lo, c), k1024));  // T's groups 2c, 2c+1 are sub-block c
        mb[r] = qmm_h2u(__hsub2(qmm_dup1024(m_hi, c), k1024));
      }
      against_t(ma[0], ma[1], mb[0], mb[1], dm);
    }
    constexpr int QS = TYPE == NSQ_TYPE_Q4_K ? 16 : 48;
    [[maybe_unused]] uint2 hg[2];
    if constexpr (TYPE == NSQ_TYPE_Q5_K && LAYOUT == NSQ_Q6K_GGML) {
      // bit j of byte l is the fifth bit of weight l of sub-block j
#pragma unroll
      for (int r = 0; r < 2; ++r) hg[r] = qmm_lds<uint2>(o[r] + 16 + 8 * c);
    }
    int sum[NI][4];
#pragma unroll
    for (int j = 0; j < NI; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[j][e] = 0;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // sub-blocks 2i, 2i + 1; weights 8c .. 8c + 7 of each
      uint32_t a[2][2], b[2][2];   // [row][word]
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint2 w = qmm_lds<uint2>(o[r] + QS + 32 * i + 8 * c);
        if constexpr (TYPE == NSQ_TYPE_Q4_K) {
          a[r][0] = w.x & 0x0F0F0F0Fu;
          a[r][1] = w.y & 0x0F0F0F0Fu;
          b[r][0] = w.x & 0xF0F0F0F0u;
          b[r][1] = w.y & 0xF0F0F0F0u;
        } else {
          uint32_t e0, e1, f0, f1;  // the fifth bits at 0x10 of each byte
          if constexpr (LAYOUT == NSQ_Q6K_GGML) {
            auto at4 = [](uint32_t v, int bit) { return (bit <= 4 ? v << (4 - bit) : v >> (bit - 4)) & 0x10101010u; };
            e0 = at4(hg[r].x, 2 * i);
            e1 = at4(hg[r].y, 2 * i);
            f0 = at4(hg[r].x, 2 * i + 1);
            f1 = at4(hg[r].y, 2 * i + 1);
          } else {
            // NodeStor: bit l of word j of qh
            const uint32_t ge = qmm_lds<uint8_t>(o[r] + 16 + 8 * i + c), gf = qmm_lds<uint8_t>(o[r] + 20 + 8 * i + c);
            e0 = ((ge & 15u) * 0x02040810u) & 0x10101010u;
            e1 = ((ge >> 4) * 0x02040810u) & 0x10101010u;
            f0 = ((gf & 15u) * 0x02040810u) & 0x10101010u;
            f1 = ((gf >> 4) * 0x02040810u) & 0x10101010u;
          }
          a[r][0] = (w.x & 0x0F0F0F0Fu) | e0;
          a[r][1] = (w.y & 0x0F0F0F0Fu) | e1;
          b[r][0] = ((w.x >> 4) & 0x0F0F0F0Fu) | f0;
          b[r][1] = ((w.y >> 4) & 0x0F0F0F0Fu) | f1;
        }
      }
      int se[2], so[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        se[r] = qmm_u8(sc[r][i >> 1], (2 * i) & 3) * (TYPE == NSQ_TYPE_Q4_K ? 16 : 1);  // (odd sub-blocks count 16 times)
        so[r] = qmm_u8(sc[r][i >> 1], (2 * i + 1) & 3);
      }
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const uint4 x = B.unit(j, i);
        int acc[4];
        qmm_mma_k32<false>(acc, a[0][0], a[1][0], a[0][1], a[1][1], x.x, x.y, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[j][e] += acc[e] * se[e >> 1];
        qmm_mma_k32<false>(acc, b[0][0], b[1][0], b[0][1], b[1][1], x.z, x.w, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[j][e] += acc[e] * so[e >> 1];
      }
    }
    float f[NI][4];
#pragma unroll
    for (int j = 0; j < NI; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[j][e] = (float)sum[j][e];
    }
    qmm_add<NI, LIMBS>(u, d, f, B.k256);
  } else if constexpr (TYPE == NSQ_TYPE_Q4_0 || TYPE == NSQ_TYPE_Q8_0) {
    constexpr int BB = TYPE == NSQ_TYPE_Q4_0 ? 18 : 34;
    // the sums start at the bits of 1.5 * 2^23: as f32 they are that plus the
    // sum (below 2^20), without a conversion
    constexpr int kMagic = 0x4B400000;
    constexpr float kMagicF = 12582912.0f;
    const QmmRow rows[2] = {QmmRow(o[0]), QmmRow(o[1])};
    if constexpr (TYPE == NSQ_TYPE_Q4_0) {
      uint32_t ta[2][2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t d = c + 4 * q < nv ? rows[r].u16(BB * (c + 4 * q)) : 0u;
          ta[r][q] = d | (d << 16);
        }
      }
      const float k[2] = {-8.0f, -8.0f};
      against_t(ta[0][0], ta[1][0], ta[0][1], ta[1][1], k);
    }
    qmm_for<8>([&](auto I) {
      constexpr int i = decltype(I)::value;
      uint32_t a[2][2];
      float d[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        d[r] = i < nv ? h2f((uint16_t)rows[r].u16(BB * i)) : 0.0f;
        const uint32_t w = rows[r].template word<BB * i + 2>(4 * c);
        if constexpr (TYPE == NSQ_TYPE_Q4_0) {
          a[r][0] = w & 0x0F0F0F0Fu;
          a[r][1] = (w >> 4) & 0x0F0F0F0Fu;
        } else {
          a[r][0] = w;
          a[r][1] = rows[r].template word<BB * i + 18>(4 * c);
        }
      }
      float f[NI][4];
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const uint4 x = B.unit(j, i >> 1);
        int acc[4];
        qmm_mma_k32<TYPE == NSQ_TYPE_Q8_0>(acc, a[0][0], a[1][0], a[0][1], a[1][1], (i & 1) ? x.z : x.x, (i & 1) ? x.w : x.y,
                                           kMagic);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[j][e] = __int_as_float(acc[e]) - kMagicF;
      }
      qmm_add<NI, LIMBS>(u, d, f, B.k256);
    });
  } else {  // Q6_K
    const QmmRow rows[2] = {QmmRow(o[0]), QmmRow(o[1])};
    float d[2];
    uint32_t sw[2][4];  // the 16 scale bytes, signed
    uint32_t ta[2][2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      d[r] = h2f((uint16_t)rows[r].u16(208));
      if constexpr (LAYOUT == NSQ_Q6K_NODESTOR) d[r] *= 0.015625f;  // scale (b - 128) / 64
      qmm_for<4>([&](auto I) {
        constexpr int i = decltype(I)::value;
        sw[r][i] = rows[r].template word<192 + 4 * i>(0);
        if constexpr (LAYOUT == NSQ_Q6K_NODESTOR) sw[r][i] ^= 0x80808080u;
      });
      // scales 2c, 2c+1 and 2c+8, 2c+9 in fp16
      const uint32_t sel = 0x4040u | (uint32_t)((2 * c) & 3) | (uint32_t)(((2 * c + 1) & 3) << 8);
      const __half2 off = __float2half2_rn(1152.0f);
      ta[r][0] = qmm_h2u(__hsub2(qmm_u2h(__byte_perm((c < 2 ? sw[r][0] : sw[r][1]) ^ 0x80808080u, 0x64646464u, sel)), off));
      ta[r][1] = qmm_h2u(__hsub2(qmm_u2h(__byte_perm((c < 2 ? sw[r][2] : sw[r][3]) ^ 0x80808080u, 0x64646464u, sel)), off));
    }
    int sum[NI][4];
    const float k[2] = {-32.0f * d[0], -32.0f * d[1]};
    against_t(ta[0][0], ta[1][0], ta[0][1], ta[1][1], k);
#pragma unroll
    for (int j = 0; j < NI; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[j][e] = 0;
    }
    qmm_for<4>([&](auto P) {
      constexpr int i = decltype(P)::value;
      uint32_t a[4][2];  // [16-group of this turn][row]: four 6-bit values
      int s[4][2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if constexpr (LAYOUT == NSQ_Q6K_GGML) {
          // half n, 16-group g of its runs of 32
          constexpr int n = i >> 1, g = i & 1;
          const uint32_t A = rows[r].template word<64 * n + 16 * g>(4 * c);
          const uint32_t Bw = rows[r].template word<64 * n + 32 + 16 * g>(4 * c);
          const uint32_t H = rows[r].template word<128 + 32 * n + 16 * g>(4 * c);
          a[0][r] = (A & 0x0F0F0F0Fu) | ((H << 4) & 0x30303030u);
          a[1][r] = (Bw & 0x0F0F0F0Fu) | ((H << 2) & 0x30303030u);
          a[2][r] = ((A >> 4) & 0x0F0F0F0Fu) | (H & 0x30303030u);
          a[3][r] = ((Bw >> 4) & 0x0F0F0F0Fu) | ((H >> 2) & 0x30303030u);
          // scales 8n + g + 2t
          s[0][r] = qmm_s8<g>(sw[r][2 * n]);
          s[1][r] = qmm_s8<g + 2>(sw[r][2 * n]);
          s[2][r] = qmm_s8<g>(sw[r][2 * n + 1]);
          s[3][r] = qmm_s8<g + 2>(sw[r][2 * n + 1]);
        } else {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            // values 4c .. 4c+3 of group 4i + t: ql bytes 8g + 2c, + 1; qh byte 4g + c
            const int g = 4 * i + t;
            const uint32_t lo = __byte_perm(rows[r].u16(8 * g + 2 * c), 0, 0x1100);
            const uint32_t hb = rows[r].u8(128 + 4 * g + c) * 0x01010101u;
            const uint32_t hh = ((hb << 4) & 0x30u) | ((hb << 2) & 0x3000u) | (hb & 0x300000u) | ((hb >> 2) & 0x30000000u);
            a[t][r] = (lo & 0x000F000Fu) | ((lo >> 4) & 0x0F000F00u) | hh;
          }
          s[0][r] = qmm_s8<0>(sw[r][i]);
          s[1][r] = qmm_s8<1>(sw[r][i]);
          s[2][r] = qmm_s8<2>(sw[r][i]);
          s[3][r] = qmm_s8<3>(sw[r][i]);
        }
      }
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const uint4 x = B.unit(j, i);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          int acc[4];
          qmm_mma_k16(acc, a[t][0], a[t][1], xs[t]);
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[j][e] += acc[e] * s[t][e >> 1];
        }
      }
    });
    float f[NI][4];
#pragma unroll
    for (int j = 0; j < NI; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[j][e] = (float)sum[j][e];
    }
    qmm_add<NI, LIMBS>(u, d, f, B.k256);
  }
}

// ---------------------------------------------------------------------------
// Lists of the picks by expert (kQmmUp and kQmmDown), built by the routing
// kernel and copied into every CTA's shared memory.
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
// EP: experts of a lane.
template <int EP>
__device__ __forceinline__ void qmm_route(const QmmParams& p, int m, int lane, int32_t* ids, float* wts) {
  const double* l = p.logits + (int64_t)m * p.E;
  const bool sig = p.score == NSQ_SCORE_SIGMOID_NORM;
  const bool by_score = sig || p.sel_bias;  // else the order of the logits is that of the scores
  double v[EP];  // logits, then scores where the order needs them, of experts lane, lane + 32, ...
  double mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < EP; ++i) {
    v[i] = 0.0;
    if (lane + 32 * i < p.E) {
      v[i] = l[lane + 32 * i];
      mx = fmax(mx, v[i]);
    }
  }
  double sum = 1.0;
  if (!sig) {
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (p.score == NSQ_SCORE_SOFTMAX || by_score) {
      sum = 0.0;
#pragma unroll 1
      for (int e = lane; e < p.E; e += 32) sum += exp(l[e] - mx);
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
  }
  auto score = [&](double x) { return sig ? 1.0 / (1.0 + exp(-x)) : exp(x - mx) / sum; };
  uint64_t key[EP];
#pragma unroll
  for (int i = 0; i < EP; ++i) {
    key[i] = 0;
    if (32 * i < p.E) {
      const int e = lane + 32 * i;
      if (by_score) v[i] = score(v[i]);
      if (e < p.E) key[i] = qmm_key(by_score && p.sel_bias ? v[i] + (double)p.sel_bias[e] : v[i]);
    }
  }
  double mine = 0.0;  // lane j keeps pick j's score (or logit)
  int mine_id = 0;
#pragma unroll 1
  for (int j = 0; j < p.top_k; ++j) {
    uint64_t best = 0;
    double at_best = 0.0;
    int at = 0x7FFFFFFF;
#pragma unroll
    for (int i = 0; i < EP; ++i) {
      if (key[i] > best) {
        best = key[i];
        at = lane + 32 * i;
        at_best = v[i];
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
    const double got = __shfl_sync(0xffffffffu, at_best, id & 31);
    if (lane == j) {
      mine = got;
      mine_id = id;
    }
  }
  const double s = by_score ? mine : score(mine);
  double total = lane < p.top_k ? s : 0.0;
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane < p.top_k) {
    ids[lane] = mine_id;
    wts[lane] = (float)((p.score == NSQ_SCORE_SOFTMAX ? s : s / total) * (double)p.scale);
  }
}

// One CTA builds the lists.  mem: 3 P + E ints of shared memory.
__device__ __forceinline__ void qmm_build_lists(const QmmParams& p, int32_t* mem) {
  const int P = p.M * p.top_k;
  int32_t* ids = mem;
  float* wts = reinterpret_cast<float*>(mem + P);
  int32_t* ranks = mem + 2 * P;
  int32_t* first = mem + 3 * P;  // [E] picks of an expert so far, then its first place
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (p.score >= 0) {
    for (int m = warp; m < p.M; m += warps) {
      int32_t* to = ids + m * p.top_k;
      float* tw = wts + m * p.top_k;
      if (p.E <= 32) {
        qmm_route<1>(p, m, lane, to, tw);
      } else if (p.E <= 128) {
        qmm_route<4>(p, m, lane, to, tw);
      } else {
        qmm_route<NSQ_MOE_MAX_EXPERTS / 32>(p, m, lane, to, tw);
      }
      __syncwarp();
      if (lane < p.top_k) {
        p.ids[m * p.top_k + lane] = ids[m * p.top_k + lane];
        p.wts[m * p.top_k + lane] = wts[m * p.top_k + lane];
      }
    }
  } else {
    // an expert given twice by a token counts once, with the sum of its
    // weights: so a group holds a token once
    for (int q = threadIdx.x; q < P; q += blockDim.x) {
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
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) first[e] = 0;
  __syncthreads();
  if (warp != 0) return;
  // one warp, 32 picks at a time: a pick's rank among its expert's picks
  for (int b = 0; b < P; b += 32) {
    const int q = b + lane, e = q < P ? ids[q] : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    int base = 0;
    if (e >= 0) base = first[e];
    __syncwarp();
    if (q < P) ranks[q] = base + __popc(same & ((1u << lane) - 1));
    if (e >= 0 && lane == __ffs(same) - 1) first[e] = base + __popc(same);
    __syncwarp();
  }
  // picks and groups of the experts before each: groups start at every TS-th
  // pick of an expert
  int picks = 0, groups = 0;
  for (int b = 0; b < p.E; b += 32) {
    const int e = b + lane, n = e < p.E ? first[e] : 0, m = (n + p.TS - 1) / p.TS;
    int np = n, ng = m;  // inclusive sums over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, np, o), g = __shfl_up_sync(0xffffffffu, ng, o);
      if (lane >= o) {
        np += a;
        ng += g;
      }
    }
    if (e < p.E) {
      first[e] = picks + np - n;
      for (int i = 0; i < m; ++i)
        p.groups[groups + ng - m + i] = QmmGroup{e, picks + np - n + i * p.TS, min(p.TS, n - i * p.TS), 0};
    }
    picks += __shfl_sync(0xffffffffu, np, 31);
    groups += __shfl_sync(0xffffffffu, ng, 31);
  }
  __syncwarp();
  for (int q = lane; q < P; q += 32) {
    if (ids[q] < 0) continue;
    const int pos = first[ids[q]] + ranks[q];
    p.plist[pos] = q;
    p.pwts[pos] = wts[q];
    p.ptok[pos] = q / p.top_k;
  }
  if (lane == 0) *p.ngroups = groups;
}

// The most groups of P picks: a partly filled one per expert, the others full.
__host__ __device__ inline int qmm_most_groups(int P, int E, int TS) { return min(P, min(P, E) + P / TS); }

__device__ __forceinline__ QmmLists qmm_load_lists(const QmmParams& p, uint8_t* mem) {
  const int P = p.M * p.top_k;
  QmmLists L;
  L.groups = reinterpret_cast<QmmGroup*>(mem);
  const int most = qmm_most_groups(P, p.E, p.TS);
  L.plist = reinterpret_cast<int32_t*>(L.groups + most);
  L.pwts = reinterpret_cast<float*>(L.plist + P);
  L.ptok = reinterpret_cast<int32_t*>(L.pwts + P);
  // from L2: kQmmDown reads them while the kernel before it still runs
  L.ngroups = __ldcg(p.ngroups);
  for (int q = threadIdx.x; q < P; q += kQmmThreads) {  // entries past the lists' ends are not used
    if (q < most) reinterpret_cast<int4*>(L.groups)[q] = __ldcg(reinterpret_cast<const int4*>(p.groups) + q);
    L.plist[q] = __ldcg(p.plist + q);
    L.ptok[q] = __ldcg(p.ptok + q);
    L.pwts[q] = __ldcg(p.pwts + q);
  }
  return L;
}

// Bytes of a slot: RW tiles of rows at this pitch, then TS records.
__host__ __device__ inline uint32_t qmm_recs_bytes(int TS) {
  // whole n-tiles of tokens: absent ones are read too
  const int tokens = TS <= 2 ? 2 : TS <= 4 ? 4 : TS <= 8 ? 8 : 16;
  return (uint32_t)((tokens * kQmmRecPitch + 127) / 128 * 128);
}
__host__ __device__ inline uint32_t qmm_slot_bytes(int row_tiles, int pitch, int TS) {
  return (uint32_t)(row_tiles * 16 * pitch) + qmm_recs_bytes(TS);
}
inline size_t qmm_lists_bytes(int P, int E, int TS) {
  return (size_t)qmm_most_groups(P, E, TS) * sizeof(QmmGroup) + (size_t)P * 12;
}

// Bias, activation and residual (kQmmLinear), or the residual alone
// (kQmmDown), for one finished sum.
__device__ __forceinline__ int qmm_add_acq_rel(int32_t* p, int v) {
  int old;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
  return old;
}
struct QmmAdd {
  float bias, residual;
};
__device__ __forceinline__ QmmAdd qmm_adds(const QmmParams& p, int col, int row) {
  QmmAdd a{0.0f, 0.0f};
  const int64_t at = (int64_t)col * p.n + row;
  if (p.mode == kQmmLinear && p.bias) a.bias = p.bias[row];
  if (p.residual)
    a.residual = p.dtype == NSQ_OUT_F32 ? static_cast<const float*>(p.residual)[at]
                                        : __bfloat162float(static_cast<const __nv_bfloat16*>(p.residual)[at]);
  return a;
}
static __device__ __noinline__ void qmm_store(const QmmParams& p, int col, int row, float v, QmmAdd a) {
  const int64_t at = (int64_t)col * p.n + row;
  if (p.mode == kQmmLinear) v = qmm_act(v + a.bias, p.act);
  v += a.residual;
  if (p.dtype == NSQ_OUT_F32) {
    static_cast<float*>(p.y)[at] = v;
  } else {
    static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v);
  }
}

// One or four (aligned) floats; FRESH: written by another CTA of this kernel.
template <bool FRESH = false, int V>
__device__ __forceinline__ void qmm_load(float (&v)[V], const float* from) {
  if constexpr (V == 4) {
    const float4* q = reinterpret_cast<const float4*>(from);
    const float4 f = FRESH ? __ldcg(q) : *q;
    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
  } else {
    v[0] = FRESH ? __ldcg(from) : *from;
  }
}

// Where a column stands: its task (tile, and the group for kQmmUp), the step
// in it, its unit (u, of group g and column sb of K), and the steps that the
// CTA has left.
struct QmmCursor {
  int tile, g, s, u, sb, left;
};

// TC: the most tokens of a group (2, 4, 8 or 16).
//
// A task is one tile of output rows (of one group for kQmmUp); its units
// (group and 256 of K) are dealt to the KW columns in turn, KW a step.  The
// grid's CTAs share the steps of all tasks evenly, in order, so a CTA may
// begin and end inside a task; p.whole keeps tasks whole.  A row tile's part
// of a divided task goes to the workspace, and the last part to arrive adds
// them up in the order of the CTAs.
template <int TYPE, int LAYOUT, int TC, int MODE>
__global__ void __launch_bounds__(kQmmThreads, 2)
    qmm_kernel(const __grid_constant__ QmmParams p, const __grid_constant__ CUtensorMap map0,
               const __grid_constant__ CUtensorMap map1) {
  using F = QmmFmt<TYPE>;
  constexpr int BB = Fmt<TYPE>::BB;
  constexpr int MT = qmm_tiles<TYPE>(TC);
  constexpr int NQ = TC == 2 ? 1 : TC <= 8 ? 2 : 4;  // values of a lane per row half
  constexpr int WR = 16 * MT;                       // weight rows of a warp
  constexpr int OR = MODE == kQmmUp ? WR / 2 : WR;  // output rows of a warp
  uint8_t* const smem = qmm_smem;
  auto* const full = reinterpret_cast<uint64_t(*)[kQmmMaxStages]>(smem);  // [column][slot]
  auto* const used = reinterpret_cast<uint64_t(*)[kQmmMaxStages]>(smem + 256);
  auto* const ready = reinterpret_cast<uint64_t(*)[2]>(smem + 512);  // [row tile][buffer]
  auto* const taken = reinterpret_cast<uint64_t(*)[2]>(smem + 640);
  int* const rows_done = reinterpret_cast<int*>(smem + 768);  // [task % 8] row tiles that stored h
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int KW = p.KW, RW = p.RW, S = p.stages, TS = p.TS, YC = p.YC;
  const int kw = warp & (KW - 1), rw = warp / KW;
  const int lr = lane >> 2, lc = lane & 3;
  const int pitch = p.rows_aligned ? F::PA : F::PG;
  const uint32_t slot_bytes = qmm_slot_bytes(RW * MT, pitch, TS);
  const uint32_t recs_at = RW * WR * pitch;  // of a slot
  const uint32_t ring_bytes = S * KW * slot_bytes;
  // partial sums [buffer][warp][YC][WR]
  float* const ys = reinterpret_cast<float*>(smem + kQmmCtl + ring_bytes);
  const int ys_warp = YC * WR, ys_buf = kQmmWarps * ys_warp;
  // records of all units, where the CTA makes them itself
  const bool own_recs = MODE == kQmmLinear && p.x != nullptr;
  const uint32_t own_at = kQmmCtl + ring_bytes + p.PB * ys_buf * 4;
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
  if (threadIdx.x == 0) {
    if (p.rows_aligned) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map0)) : "memory");
      if constexpr (MODE == kQmmUp) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map1)) : "memory");
    }
    for (int i = 0; i < KW; ++i) {
      for (int k = 0; k < S; ++k) {
        // rows of every warp (one arrival per warp, or per lane), records (one warp: with the rows)
        mbar_init(&full[i][k], (p.rows_aligned ? RW : 32 * RW) + (RW > 1 && !own_recs));
        mbar_init(&used[i][k], RW);
      }
    }
    for (int i = 0; i < RW; ++i) {
      for (int k = 0; k < 2; ++k) {
        mbar_init(&ready[i][k], KW);
        mbar_init(&taken[i][k], 1);
      }
    }
    for (int i = 0; i < 8; ++i) rows_done[i] = 0;
    fence_mbar_init();
  }
  QmmLists L{};
  if constexpr (MODE == kQmmLinear) {
    L.ngroups = 1;
  } else {
    if constexpr (MODE == kQmmUp) {
      qmm_dep_wait();
      qmm_dep_launch();
    }
    // kQmmDown does not wait here: the lists' kernel was complete before any
    // CTA of kQmmUp let this kernel start
    L = qmm_load_lists(p, smem + kQmmCtl + ring_bytes + p.PB * ys_buf * 4);
  }
  __syncthreads();

  // ---- this CTA's steps [a, b) of all tasks
  const int units = MODE == kQmmDown ? L.ngroups * p.nsb : p.nsb;
  const int st = max(1, (units + KW - 1) / KW);  // steps of a task
  const int64_t tasks = MODE == kQmmUp ? (int64_t)tiles * L.ngroups : tiles;
  const int64_t T = tasks * st;
  // no more CTAs than steps, so that each of the G has a part of a divided task
  const int64_t G = min((int64_t)gridDim.x, max(T, (int64_t)1)), me = min((int64_t)blockIdx.x, G);
  const int64_t a = p.whole ? tasks * me / G * st : T * me / G;
  const int64_t b = blockIdx.x >= G ? a : p.whole ? tasks * (me + 1) / G * st : T * (me + 1) / G;
  auto set_unit = [&](QmmCursor& c) {
    c.u = c.sb = c.s * KW + kw;
    if constexpr (MODE == kQmmDown) {
      c.g = c.u / p.nsb;
      c.sb = c.u - c.g * p.nsb;
    }
  };
  auto next_task = [&](QmmCursor& c) {
    c.s = 0;
    if constexpr (MODE == kQmmDown) {
      c.g = kw / p.nsb;
      c.u = kw;
      c.sb = kw - c.g * p.nsb;
    } else {
      c.u = c.sb = kw;
    }
    ++c.tile;
    if constexpr (MODE == kQmmUp) {
      if (c.tile == tiles) {
        c.tile = 0;
        ++c.g;
      }
    }
  };
  auto next_step = [&](QmmCursor& c) {  // within a task
    ++c.s;
    c.u += KW;
    c.sb += KW;
    if constexpr (MODE == kQmmDown) {
      while (c.sb >= p.nsb) {
        c.sb -= p.nsb;
        ++c.g;
      }
    }
  };
  QmmCursor c;
  {
    const int64_t task = a / st;
    c.s = (int)(a - task * st);
    c.left = (int)(b - a);
    c.g = MODE == kQmmUp ? (int)(task / tiles) : 0;
    c.tile = (int)(task - (int64_t)c.g * tiles);
    set_unit(c);
  }
  auto expert_of = [&](const QmmCursor& q) { return MODE == kQmmLinear ? 0 : L.groups[q.g].expert; };
  auto count_of = [&](const QmmCursor& q) { return MODE == kQmmLinear ? p.M : L.groups[q.g].count; };

  // ---- refills.  The producing cursor runs S units ahead; a column without a
  // unit in a step skips it.
  QmmCursor pc = c;
  auto settle = [&] {  // to the next step with a unit
    while (pc.left > 0 && pc.u >= units) {
      --pc.left;
      if (pc.s + 1 == st) {
        next_task(pc);
      } else {
        next_step(pc);
      }
    }
  };
  auto advance = [&] {
    --pc.left;
    if (pc.s + 1 == st) {
      next_task(pc);
    } else {
      next_step(pc);
    }
    settle();
  };
  settle();
  const uint64_t pol = l2_policy_evict_first();
  const uint32_t my_rows = rw * WR * pitch;  // of a slot
  // this warp's weight rows of unit pc into a slot (kQmmUp: gate rows, then up
  // rows); more: bytes that follow on the same barrier phase
  auto fill_rows = [&](int stage, uint32_t more) {
    uint64_t* bar = &full[kw][stage];
    const uint32_t slot = kQmmCtl + (stage * KW + kw) * slot_bytes + my_rows;
    const int first = pc.tile * tile_rows + rw * OR;  // of the expert's rows
    if (p.rows_aligned) {
      if (lane == 0) {
        const int row0 = expert_of(pc) * (int)p.n + first;
        const int x = ((pc.sb * F::CB) & ~15) / 2;  // 16-bit elements
        const uint32_t dst = smem_u32(smem) + slot;
        mbar_arrive_expect_tx(bar, WR * pitch + more);
        qmm_tma_2d(dst, &map0, x, row0, bar, pol);
        if constexpr (MODE == kQmmUp) qmm_tma_2d(dst + (WR / 2) * pitch, &map1, x, row0, bar, pol);
      }
    } else {
      // four lanes per row copy 16 bytes each at a time: one bulk copy per row
      // takes 650 to 1300 cycles a unit to issue
      int need = F::CB;
      if constexpr (Fmt<TYPE>::QK == 32) need = min(8, p.nblk - 8 * pc.sb) * BB;
      if (more != 0 && lane == 0) qmm_expect_tx(bar, more);
      __syncwarp();
      const int64_t row0 = (int64_t)expert_of(pc) * p.n + first;
#pragma unroll 1
      for (int r = lane >> 2; r < WR; r += 8) {
        const int rr = MODE == kQmmUp && r >= WR / 2 ? r - WR / 2 : r;
        const uint8_t* w = MODE == kQmmUp && r >= WR / 2 ? p.w1 : p.w0;
        const int64_t at = (row0 + rr) * p.rb + (int64_t)pc.sb * F::CB, a16 = at & ~(int64_t)15;
        const int64_t left = p.wbytes - a16;  // of the tensor
        const int chunks = first + rr < p.n ? (int)((at + need - a16 + 15) >> 4) : 0;
        const uint32_t dst = smem_u32(smem) + slot + r * pitch;
#pragma unroll
        for (int k = 0; k < (F::PG / 16 + 3) / 4; ++k) {
          const int j = (lane & 3) + 4 * k;
          if (j < chunks) qmm_cp_async(dst + 16 * j, w + a16 + 16 * j, (int)min((int64_t)16, left - 16 * j), pol);
        }
      }
      qmm_cp_async_arrive(bar);
    }
  };
  auto fill_records = [&](int stage) {
    uint64_t* bar = &full[kw][stage];
    uint8_t* dst = smem + kQmmCtl + (stage * KW + kw) * slot_bytes + recs_at;
    const int count = count_of(pc);
    if (RW > 1 && lane == 0) mbar_arrive_expect_tx(bar, count * kQmmRec);
    __syncwarp();
    if (lane < count) {
      int row = lane;
      if constexpr (MODE == kQmmUp) row = L.ptok[L.groups[pc.g].start + lane];
      if constexpr (MODE == kQmmDown) row = L.plist[L.groups[pc.g].start + lane];
      bulk_g2s(dst + lane * kQmmRecPitch, p.recs + ((int64_t)row * p.nsb + pc.sb) * kQmmRec, kQmmRec, bar);
    }
  };
  // The column's warps refill the records of its units in turn: it takes a warp
  // about 500 cycles (always the same one: the others wait 750 cycles a unit).
  int rec_unit = kw;  // units of the column whose records were refilled, from kw on
  auto my_turn = [&] { return rw == (rec_unit++ & (RW - 1)); };
  if (own_recs) {
    qmm_dep_wait();
    qmm_dep_launch();
    for (int k = 0; k < S && pc.left > 0; ++k) {
      fill_rows(k, 0);
      advance();
    }
    for (int j = warp; j < p.M * p.nsb; j += kQmmWarps) {
      const int row = j / p.nsb, sb = j - row * p.nsb, valid = (int)min((int64_t)256, p.K - 256 * sb);
      uint8_t* rec = smem + own_at + sb * qmm_recs_bytes(TS) + row * kQmmRecPitch;
      const int64_t at = row * p.K + 256 * sb;
      if (p.dtype == NSQ_OUT_F32) {
        qmm_make_record(static_cast<const float*>(p.x) + at, valid, p.order, rec, lane);
      } else {
        qmm_make_record(static_cast<const __nv_bfloat16*>(p.x) + at, valid, p.order, rec, lane);
      }
    }
    __syncthreads();
  } else if constexpr (MODE != kQmmUp) {
    // the weights do not depend on the kernel before; records, residual and
    // outputs do
    const QmmCursor start = pc;
    for (int k = 0; k < S && pc.left > 0; ++k) {
      fill_rows(k, RW == 1 ? count_of(pc) * kQmmRec : 0);
      advance();
    }
    __syncwarp();
    qmm_dep_wait();
    qmm_dep_launch();
    pc = start;
    for (int k = 0; k < S && pc.left > 0; ++k) {
      if (my_turn()) fill_records(k);
      advance();
    }
  } else {
    for (int k = 0; k < S && pc.left > 0; ++k) {
      fill_rows(k, RW == 1 ? count_of(pc) * kQmmRec : 0);
      if (my_turn()) fill_records(k);
      advance();
    }
  }

  bool ok = true;
  float tot[MT][NQ][2];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
#pragma unroll
    for (int j = 0; j < NQ; ++j) tot[t][j][0] = tot[t][j][1] = 0.0f;
  }
  // calls f(token, row of the warp, sum) for the sums of a task of `count`
  // tokens and clears them: with up to 4 tokens the two lanes that share a
  // token add their limbs and take a row half each, else a lane has whole ones
  auto each_sum = [&](int count, auto&& f) {
    const int half = lc & 1;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        if (TC > 4 && count > 4) {
          const int tk = 8 * (q >> 1) + 2 * lc + (q & 1);
          f(tk, 16 * t + lr, tot[t][q][0]);
          f(tk, 16 * t + lr + 8, tot[t][q][1]);
        } else if (q < 2) {
          const float give = half ? tot[t][q][0] : tot[t][q][1];
          const float v = (half ? tot[t][q][1] : tot[t][q][0]) + __shfl_xor_sync(0xffffffffu, give, 1);
          f(2 * q + (lc >> 1), 16 * t + lr + 8 * half, v);
        }
        tot[t][q][0] = tot[t][q][1] = 0.0f;
      }
    }
  };
  int stage = 0, seq = 0;
  // kQmmUp: the sums of this row tile became h.  The CTA's last row tile of
  // the task reports the task's rows; whoever completes 256 rows of h makes
  // their records.  (A report per row tile would fence 8 times as often.)
  auto report_rows = [&](int g, int row, int rows, int turns) {
    __syncwarp();
    rows = min(rows, (int)p.n - row);
    if (rows <= 0) return;
    const int sb = row >> 8, valid = min(256, (int)p.n - 256 * sb), nsb = ((int)p.n + 255) >> 8;
    int last = 0;
    if (lane == 0) {
      bool mine = true;
      if (turns > 1) {  // row tiles of this CTA
        __threadfence_block();
        int* count = rows_done + (seq & 7);  // warps of a CTA are at most S < 8 tasks apart
        mine = atomicAdd(count, 1) == turns - 1;
        if (mine) *count = 0;
        __threadfence_block();
      }
      if (mine) last = qmm_add_acq_rel(p.done + (int64_t)g * nsb + sb, rows) + rows == valid;
    }
    if (!__shfl_sync(0xffffffffu, last, 0)) return;
    __syncwarp();  // what lane 0 acquired is the other lanes' too (a shuffle orders no memory)
    const int count = L.groups[g].count, start = L.groups[g].start;
    for (int t = 0; t < count; ++t) {
      const int64_t pick = L.plist[start + t];
      qmm_make_record<float, true>(p.h + pick * p.n + 256 * sb, valid, p.order_h, p.recs_h + (pick * nsb + sb) * kQmmRec, lane);
    }
  };
  uint32_t phase = 0;
  int owed = -1;  // slot whose records are still to be refilled for pc
  for (; ok && c.left > 0; ++seq) {
    // ---- one task, or this CTA's part of it
    const int buf = p.PB == 2 ? seq & 1 : 0, turn = p.PB == 2 ? seq >> 1 : seq;
    const int s_first = c.s, n_steps = min(st - c.s, c.left);
    const int tile = c.tile, task_g = c.g;
    float* my_ys = ys + buf * ys_buf + warp * ys_warp;
    auto claim_ys = [&] {  // the buffer's last sums have been joined
      if (KW > 1 && turn > 0 && !mbar_wait_bounded(&taken[rw][buf], (turn & 1) ^ 1)) ok = false;
      __syncwarp();
    };
    if constexpr (MODE == kQmmDown) {
      claim_ys();
      for (int i = lane; i < ys_warp; i += 32) my_ys[i] = 0.0f;
      __syncwarp();
    }
    // kQmmDown: the sums of a group so far go to its tokens' places, weighted
    // (once per group: once per unit took 40 of its 370 instructions)
    [[maybe_unused]] int acc_g = -1;
    auto spread = [&](int g) {
      if (g < 0) return;
      const int count = L.groups[g].count, start = L.groups[g].start;
      each_sum(count, [&](int tk, int r, float v) {
        if (tk < count) my_ys[L.ptok[start + tk] * WR + r] += L.pwts[start + tk] * v;
      });
      __syncwarp();
    };
    [[maybe_unused]] int task_count = 0;
    if constexpr (MODE != kQmmDown) task_count = count_of(c);
    for (int i = 0; i < n_steps && ok; ++i) {
      if (c.u < units) {
        if (owed >= 0) {
          // the records of the slot used last: free when all RW warps are done
          if (my_turn()) {
            if (!mbar_wait_bounded(&used[kw][owed], owed > stage ? phase ^ 1 : phase)) {
              ok = false;
              break;
            }
            __syncwarp();
            fill_records(owed);
          }
          owed = -1;
          advance();
        }
        if (!mbar_wait_bounded(&full[kw][stage], phase)) {
          ok = false;
          break;
        }
        __syncwarp();
        if constexpr (MODE == kQmmDown) {
          if (c.g != acc_g) {
            spread(acc_g);
            acc_g = c.g;
          }
        }
        const int count = MODE == kQmmDown ? count_of(c) : task_count;
        const uint32_t slot = kQmmCtl + (stage * KW + kw) * slot_bytes;
        const uint32_t recs = own_recs ? own_at + c.sb * qmm_recs_bytes(TS) : slot + recs_at;
        const int nv = min(8, p.nblk - 8 * c.sb);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          uint32_t o[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = MODE == kQmmUp && MT == 1 ? 8 * h + lr : 16 * t + 8 * h + lr;  // of this warp's rows
            uint32_t mis = 0;
            if constexpr (F::CB % 16 != 0 || Fmt<TYPE>::QK == 32) {
              mis = (uint32_t)(c.sb * F::CB) & 15;
              if (!p.rows_aligned) {
                const int rr = MODE == kQmmUp && r >= WR / 2 ? r - WR / 2 : r;
                const uint32_t row = (uint32_t)expert_of(c) * (uint32_t)p.n + (uint32_t)(tile * tile_rows + rw * OR + rr);
                mis = (row * (uint32_t)p.rb + (uint32_t)(c.sb * F::CB)) & 15;
              }
            }
            o[h] = slot + my_rows + r * pitch + mis;
          }
          auto unit = [&](auto N, auto Limbs) {
            constexpr int ni = decltype(N)::value;
            constexpr bool limbs = decltype(Limbs)::value;
            constexpr int nq = kQmmVals<ni, limbs>;
            const QmmB<limbs> B(recs, 0, lr, lc);
            float v[nq][2];
            qmm_unit<TYPE, LAYOUT, ni, limbs>(o, lc, B, nv, v);
#pragma unroll
            for (int q = 0; q < nq; ++q) {
              const int tk = limbs ? 8 * (q >> 1) + 2 * lc + (q & 1) : 2 * q + (lc >> 1);
              float s = tk < count ? qmm_lds<float>(recs + tk * kQmmRecPitch + kQmmRecS) : 0.0f;
              if (!limbs && (lc & 1)) s *= 65536.0f;  // limb 2 of the token
              const float y0 = s * v[q][0], y1 = s * v[q][1];
              tot[t][q][0] += y0;
              tot[t][q][1] += y1;
            }
          };
          using std::integral_constant;
          using std::false_type;
          using std::true_type;
          if (TC == 2 || count <= 2) {
            unit(integral_constant<int, 1>{}, false_type{});
          } else if (TC == 4 || count <= 4) {
            if constexpr (TC > 2) unit(integral_constant<int, 2>{}, false_type{});
          } else if (TC == 8 || count <= 8) {
            if constexpr (TC > 4) unit(integral_constant<int, 3>{}, true_type{});
          } else if constexpr (TC > 8) {
            unit(integral_constant<int, 6>{}, true_type{});
          }
        }
        __syncwarp();
        if (RW > 1 && !own_recs && lane == 0) mbar_arrive(&used[kw][stage]);
        if (pc.left > 0) {
          if (own_recs) {
            fill_rows(stage, 0);
            advance();
          } else if (RW == 1) {
            fill_rows(stage, count_of(pc) * kQmmRec);
            fill_records(stage);
            advance();
          } else {
            fill_rows(stage, 0);
            owed = stage;
          }
        }
        if (++stage == S) {
          stage = 0;
          phase ^= 1;
        }
      }
      next_step(c);
    }
    if (!ok) break;
    if constexpr (MODE == kQmmDown) spread(acc_g);
    c.left -= n_steps;
    c.s = s_first + n_steps;  // (columns without a unit in the last step count it too)
    const bool ends = c.s == st;
    if (ends) next_task(c);
    // ---- the sums: every column leaves its own; one of them adds them up
    const int cnt = MODE == kQmmUp ? task_count : p.M;
    if constexpr (MODE != kQmmDown) {
      claim_ys();
      each_sum(cnt, [&](int tk, int r, float v) {
        if (tk < cnt) my_ys[tk * WR + r] = v;
      });
    }
    __syncwarp();
    if (KW > 1) {
      if (lane == 0) mbar_arrive(&ready[rw][buf]);
      if (kw != (seq & (KW - 1))) continue;
      if (!mbar_wait_bounded(&ready[rw][buf], turn & 1)) {
        ok = false;
        break;
      }
      __syncwarp();
    }
    const float* y0 = ys + buf * ys_buf + rw * KW * ys_warp;
    // V places [token][row ..] at once: four, or one where that takes the warp
    // two turns at most (a lane makes its outputs one after the other: a token
    // alone loses 1.5 us by four; 7 tokens win 5 us by it)
    const bool wide = OR * cnt > 64;
    auto joined = [&](auto& v, int at) {
      constexpr int V = sizeof(v) / 4;
      qmm_load(v, y0 + at);
      for (int k = 1; k < KW; ++k) {
        float f[V];
        qmm_load(f, y0 + k * ys_warp + at);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += f[e];
      }
    };
    const int row0 = tile * tile_rows + rw * OR;
    // writes the outputs of this row tile, sum(v, at) being the sums of V places
    auto emit_by = [&](auto width, auto&& sum) {
      constexpr int V = decltype(width)::value;
      for (int i = lane; i < OR / V * cnt; i += 32) {
        const int col = i / (OR / V), r = i % (OR / V) * V;
        if (row0 + r >= p.n) continue;
        float v[V];
        sum(v, col * WR + r);
        if constexpr (MODE == kQmmUp) {
          float up[V];
          sum(up, col * WR + r + OR);
          float* h = p.h + (int64_t)L.plist[L.groups[task_g].start + col] * p.n + row0 + r;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            if (row0 + r + e < p.n) h[e] = qmm_act(v[e], p.act) * up[e];
          }
        } else {
          QmmAdd add[V] = {};
#pragma unroll
          for (int e = 0; e < V; ++e) {
            if (row0 + r + e < p.n) add[e] = qmm_adds(p, col, row0 + r + e);
          }
#pragma unroll
          for (int e = 0; e < V; ++e) {
            if (row0 + r + e < p.n) qmm_store(p, col, row0 + r + e, v[e], add[e]);
          }
        }
      }
    };
    auto emit = [&](auto&& sum) {
      if (wide) {
        emit_by(std::integral_constant<int, 4>{}, sum);
      } else {
        emit_by(std::integral_constant<int, 1>{}, sum);
      }
    };
    // the buffer is free as soon as it was read: the reports below take 1 to 2 us
    auto release_ys = [&] {
      __syncwarp();
      if (KW > 1 && lane == 0) mbar_arrive(&taken[rw][buf]);
    };
    if (s_first == 0 && ends) {
      emit(joined);
      release_ys();
      if constexpr (MODE == kQmmUp) report_rows(task_g, tile * tile_rows, tile_rows, RW);
    } else {
      // ---- a part of a divided task
      const int64_t f0 = MODE == kQmmUp ? ((int64_t)task_g * tiles + tile) * st : (int64_t)tile * st;
      const int c_lo = (int)(((f0 + 1) * G - 1) / T), c_hi = (int)(((f0 + st) * G - 1) / T);
      auto part_of = [&](int cta) {
        return p.parts + ((int64_t)(cta * 2 + (cta == c_lo ? 1 : 0)) * kQmmWarps + rw) * ys_warp;
      };
      float* mine = part_of((int)blockIdx.x);
      for (int i = 4 * lane; i < WR * cnt; i += 128) {
        float v[4];
        joined(v, i);
        *reinterpret_cast<float4*>(mine + i) = make_float4(v[0], v[1], v[2], v[3]);
      }
      release_ys();
      int last = 0;
      if (lane == 0) last = qmm_add_acq_rel(p.tickets + c_lo * kQmmWarps + rw, n_steps) + n_steps == st;
      if (__shfl_sync(0xffffffffu, last, 0)) {
        __syncwarp();  // (as in report_rows)
        // eight parts' loads at a time: one after the other their latencies
        // were 50 us of 32 tokens' and 64 experts' 207
        emit([&](auto& v, int at) {
          constexpr int V = sizeof(v) / 4;
#pragma unroll
          for (int e = 0; e < V; ++e) v[e] = 0.0f;
          for (int q = c_lo; q <= c_hi; q += 8) {
            float f[8][V] = {};
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              if (q + k <= c_hi) qmm_load<true>(f[k], part_of(q + k) + at);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
#pragma unroll
              for (int e = 0; e < V; ++e) v[e] += f[k][e];
            }
          }
        });
        if constexpr (MODE == kQmmUp) report_rows(task_g, row0, OR, 1);
      }
    }
  }
}

}  // namespace nsq
