// quant.cuh — the NVFP4 block quantisers: sixteen values -> one e4m3 scale and
// eight bytes of e2m1 codes.  Shared by the activation quantiser, the dual
// GEMM's NVFP4 output and the block norm's.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

namespace nvfp4dg {

// One 16-element block -> NVFP4: returns the e4m3 scale byte
// e4m3(amax / 6) (round to nearest even, saturating at 448) and sets w0/w1
// to the eight bytes of e2m1 codes of q = RN(v / scale) rounded to the e2m1
// grid (nearest, ties to the even code, saturating at 6, sign kept), all-zero
// codes when the scale is 0.  The forms below (the compare form for 16-bit
// values, encode_rcp16) give the same codes, so the fused NVFP4 output
// equals quantising the fp16 result, whichever form each side uses.
//
// No division: the e2m1 code of q only depends on how q compares with the
// grid midpoints t in {0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5}, and
// RN(v / s) < t  <=>  v < t * s  (and = <=> =) for every fp32 v and e4m3
// scale s.  t * s has at most 7 significant bits, so it is exact; and with
// s = b 2^e, 1 <= b < 2, t = a 2^f, 1 <= a < 2, the fp32 neighbours of
// t * s lie more than s * ulp(t) / 2 away from it (their spacing is at least
// 2^(e+f-23) > b 2^(e+f-24)), so no v other than t * s has a quotient that
// rounds onto t.  Ties at 0.25, 1.25, 2.5, 5 go down (strict >), those at
// 0.75, 1.75, 3.5 up (>=, written as > the float just below).  With an
// IEEE division per element instead, the NVFP4-output epilogue took 18.5
// instead of 15.2 us on the 256 x 4096 x 7168 problem.
__device__ __forceinline__ uint8_t quant_block16(const float* v, uint32_t& w0,
                                                 uint32_t& w1) {
  float amax = 0.f;
#pragma unroll
  for (int q = 0; q < 16; ++q) amax = fmaxf(amax, fabsf(v[q]));
  const __nv_fp8_storage_t sb =
      __nv_cvt_float_to_fp8(amax / 6.0f, __NV_SATFINITE, __NV_E4M3);
  const float sd =
      __half2float(__half(__nv_cvt_fp8_to_halfraw(sb, __NV_E4M3)));
  w0 = 0;
  w1 = 0;
  if (sd > 0.f) {
    auto below = [](float x) { return __uint_as_float(__float_as_uint(x) - 1u); };
    const float t0 = 0.25f * sd, t1 = below(0.75f * sd), t2 = 1.25f * sd,
                t3 = below(1.75f * sd), t4 = 2.5f * sd, t5 = below(3.5f * sd),
                t6 = 5.0f * sd;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      // the number of midpoints below |v| (t0 < t1 < ... < t6), by a
      // three-level binary search
      const float a = fabsf(v[i]);
      const bool b2 = a > t3;
      const bool b1 = a > (b2 ? t5 : t1);
      const bool b0 = a > (b2 ? (b1 ? t6 : t4) : (b1 ? t2 : t0));
      const uint32_t m = (b2 ? 4u : 0u) | (b1 ? 2u : 0u) | (b0 ? 1u : 0u);
      const uint32_t code = m | ((__float_as_uint(v[i]) >> 28) & 8u);
      if (i < 8)
        w0 |= code << (4 * i);
      else
        w1 |= code << (4 * (i - 8));
    }
  }
  return static_cast<uint8_t>(sb);
}

// The same block quantiser for 16-bit elements (fp16 or bf16), held as
// eight packed pairs (element 2i in the low half of p[i]), two elements per
// instruction.  Every midpoint product t * s (at most 7 significant bits,
// between 2^-11 and 2240) is exact in fp16 and in bf16, and for a 16-bit v,
// v >= T <=> v > the 16-bit value below T; so comparing 16-bit keys with
// packed 2-wide compares gives exactly the codes of the fp32 form above.
// The NVFP4-output epilogue uses this compare form (which keeps the GEMM
// kernels' register allocation as it is); the activation quantiser uses
// quant_block16_x2 below, which gives the same codes with fewer
// instructions and hands blocks holding a NaN to this form.
template <typename H2>
struct Half2Ops;
template <>
struct Half2Ops<__half2> {
  static __device__ __forceinline__ uint32_t bits(float x) {  // x exact
    return __half_as_ushort(__float2half_rn(x));
  }
  static __device__ __forceinline__ float lo(uint32_t u) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(u)));
  }
  static __device__ __forceinline__ float hi(uint32_t u) { return lo(u >> 16); }
  static constexpr uint32_t kInfKey = 0x7C00u;  // |v| bits of +inf
};
template <>
struct Half2Ops<__nv_bfloat162> {
  static __device__ __forceinline__ uint32_t bits(float x) {  // x exact
    return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  }
  static __device__ __forceinline__ float lo(uint32_t u) {
    return __uint_as_float(u << 16);
  }
  static __device__ __forceinline__ float hi(uint32_t u) {
    return __uint_as_float(u & 0xFFFF0000u);
  }
  static constexpr uint32_t kInfKey = 0x7F80u;
};

template <typename H2>
__device__ __forceinline__ H2 as_h2(uint32_t u) {
  return *reinterpret_cast<const H2*>(&u);
}

template <typename H2>
__device__ __forceinline__ uint8_t quant_block16_x2_cmp(const uint32_t (&p)[8],
                                                        uint32_t& w0,
                                                        uint32_t& w1) {
  using Ops = Half2Ops<H2>;
  uint32_t a[8];  // |v| pairs: the keys
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = p[i] & 0x7FFF7FFFu;
  H2 m2 = as_h2<H2>(a[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m2 = __hmax2(m2, as_h2<H2>(a[i]));
  uint32_t mu;
  *reinterpret_cast<H2*>(&mu) = m2;
  const float amax = fmaxf(Ops::lo(mu), Ops::hi(mu));
  const __nv_fp8_storage_t sb =
      __nv_cvt_float_to_fp8(amax / 6.0f, __NV_SATFINITE, __NV_E4M3);
  const float sd =
      __half2float(__half(__nv_cvt_fp8_to_halfraw(sb, __NV_E4M3)));
  w0 = 0;
  w1 = 0;
  if (sd > 0.f) {
    auto rep2 = [](uint32_t b) { return b | (b << 16); };
    const uint32_t t0 = rep2(Ops::bits(0.25f * sd)),
                   t1 = rep2(Ops::bits(0.75f * sd) - 1u),
                   t2 = rep2(Ops::bits(1.25f * sd)),
                   t3 = rep2(Ops::bits(1.75f * sd) - 1u),
                   t4 = rep2(Ops::bits(2.5f * sd)),
                   t5 = rep2(Ops::bits(3.5f * sd) - 1u),
                   t6 = rep2(Ops::bits(5.0f * sd));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const H2 k = as_h2<H2>(a[i]);
      const uint32_t b2 = __hgt2_mask(k, as_h2<H2>(t3));
      const uint32_t b1 = __hgt2_mask(k, as_h2<H2>((t5 & b2) | (t1 & ~b2)));
      const uint32_t th = (t6 & b1) | (t4 & ~b1), tl = (t2 & b1) | (t0 & ~b1);
      const uint32_t b0 = __hgt2_mask(k, as_h2<H2>((th & b2) | (tl & ~b2)));
      const uint32_t code = (b2 & 0x00040004u) | (b1 & 0x00020002u) |
                            (b0 & 0x00010001u) |
                            ((p[i] >> 12) & 0x00080008u);  // the sign bits
      const uint32_t byte = (code & 0xFu) | ((code >> 12) & 0xF0u);
      if (i < 4)
        w0 |= byte << (8 * i);
      else
        w1 |= byte << (8 * (i - 4));
    }
  }
  return static_cast<uint8_t>(sb);
}

// Eight values x (fp32 bit patterns, x[0] first) -> four bytes of e2m1
// codes (element 2i in the low nibble of byte i) of q = x * rh + RN(x * rl),
// rounded once (packed fma), by the hardware conversion (round to nearest
// even, saturating at 6, sign kept).
__device__ __forceinline__ uint32_t e2m1_scaled8(const uint32_t (&x)[8],
                                                 float rh, float rl) {
  uint32_t r;
  asm("{\n\t"
      ".reg .b64 V, P, RH, RL;\n\t"
      ".reg .b32 q0, q1, q2, q3, q4, q5, q6, q7;\n\t"
      ".reg .b8 c0, c1, c2, c3;\n\t"
      "mov.b64 RH, {%9, %9};\n\t"
      "mov.b64 RL, {%10, %10};\n\t"
      "mov.b64 V, {%1, %2};\n\t"
      "mul.rn.f32x2 P, V, RL;\n\t"
      "fma.rn.f32x2 V, V, RH, P;\n\t"
      "mov.b64 {q0, q1}, V;\n\t"
      "mov.b64 V, {%3, %4};\n\t"
      "mul.rn.f32x2 P, V, RL;\n\t"
      "fma.rn.f32x2 V, V, RH, P;\n\t"
      "mov.b64 {q2, q3}, V;\n\t"
      "mov.b64 V, {%5, %6};\n\t"
      "mul.rn.f32x2 P, V, RL;\n\t"
      "fma.rn.f32x2 V, V, RH, P;\n\t"
      "mov.b64 {q4, q5}, V;\n\t"
      "mov.b64 V, {%7, %8};\n\t"
      "mul.rn.f32x2 P, V, RL;\n\t"
      "fma.rn.f32x2 V, V, RH, P;\n\t"
      "mov.b64 {q6, q7}, V;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c0, q1, q0;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c1, q3, q2;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c2, q5, q4;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c3, q7, q6;\n\t"
      "mov.b32 %0, {c0, c1, c2, c3};\n\t"
      "}"
      : "=r"(r)
      : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]),
        "r"(x[6]), "r"(x[7]), "f"(rh), "f"(rl));
  return r;
}

// One block's scale byte e4m3(amax / 6) and the e2m1 codes of its sixteen
// values x (fp32 bit patterns) under it, with v / s replaced by
// v * rh + RN(v * rl), rounded once, where rh = 1/s rounded toward zero and
// rl = RN((1 - s * rh) * rh) >= 0 (the residual 1 - s * rh is exact in one
// fma), and q rounded to e2m1 by the hardware conversion.  rh + rl is 1/s
// to about 2^-46 relative, so q is v / s to about 2^-45 relative:
//  * v / s exactly on a midpoint t (v = t * s) lands exactly on t and takes
//    the same tie rule;
//  * otherwise v / s lies at least ~2^-29 relative away from every fp32
//    rounding boundary t +- ulp(t) / 2 (v = (t +- ulp(t) / 2) * s would need
//    25 significant bits), so RN(q) and RN(v / s) fall on the same side of
//    t, or are both t.
// rl >= 0 keeps the sign of -0 (x * rl = -0); values whose quotient
// overflows saturate at 6 either way.  For 16-bit v, tests/test_oracle.py
// simulates this arithmetic for every finite value under every positive
// e4m3 s on the CPU, and a GPU test runs all of those pairs through the
// kernel; fp32 v are tested on and around every midpoint and boundary.
// (A single rounded reciprocal, q = RN(v * RN(1/s)), is not enough: ties
// at 1.25, 2.5 and 5 under scales of mantissa 1.875 round the wrong way.)
// (rh, rl) depend on the scale byte alone, so the kernel reads them from a
// 128-entry table in shared memory (rcp_pair fills it); a zero scale has
// (0, 0) and its codes are cleared by a select.
__device__ __forceinline__ float2 rcp_pair(uint32_t sb) {
  const float sd =
      __half2float(__half(__nv_cvt_fp8_to_halfraw(sb, __NV_E4M3)));
  if (!(sd > 0.f)) return make_float2(0.f, 0.f);
  const float rh = __frcp_rz(sd);
  return make_float2(rh, __fmul_rn(__fmaf_rn(-sd, rh, 1.0f), rh));
}
__device__ __forceinline__ uint8_t encode_rcp16(float amax,
                                                const uint32_t (&x)[16],
                                                uint32_t& w0, uint32_t& w1,
                                                const float2* rtab) {
  const __nv_fp8_storage_t sb =
      __nv_cvt_float_to_fp8(amax / 6.0f, __NV_SATFINITE, __NV_E4M3);
  const float2 r = rtab[sb & 0x7F];  // amax >= 0: the sign bit is clear
  const uint32_t(&xa)[8] = *reinterpret_cast<const uint32_t(*)[8]>(x);
  const uint32_t(&xb)[8] = *reinterpret_cast<const uint32_t(*)[8]>(x + 8);
  const uint32_t a = e2m1_scaled8(xa, r.x, r.y);
  const uint32_t b = e2m1_scaled8(xb, r.x, r.y);
  w0 = sb != 0 ? a : 0u;
  w1 = sb != 0 ? b : 0u;
  return static_cast<uint8_t>(sb);
}
// The same with (rh, rl) computed for the block: fp32 rows, for which the
// table lookup measured slower (25.8 against 25.2 us on 4096 x 7168).
__device__ __forceinline__ uint8_t encode_rcp16_direct(float amax,
                                                       const uint32_t (&x)[16],
                                                       uint32_t& w0,
                                                       uint32_t& w1) {
  const __nv_fp8_storage_t sb =
      __nv_cvt_float_to_fp8(amax / 6.0f, __NV_SATFINITE, __NV_E4M3);
  const float2 r = rcp_pair(sb);
  const uint32_t(&xa)[8] = *reinterpret_cast<const uint32_t(*)[8]>(x);
  const uint32_t(&xb)[8] = *reinterpret_cast<const uint32_t(*)[8]>(x + 8);
  w0 = 0;
  w1 = 0;
  if (sb != 0) {
    w0 = e2m1_scaled8(xa, r.x, r.y);
    w1 = e2m1_scaled8(xb, r.x, r.y);
  }
  return static_cast<uint8_t>(sb);
}

// The activation quantiser's 16-bit block form: amax as the largest |v| key
// (16-bit keys order like |v|), then encode_rcp16.  A block holding a NaN
// (key above +inf's) goes to the compare form.
template <typename H2>
__device__ __forceinline__ uint8_t quant_block16_x2(const uint32_t (&p)[8],
                                                    uint32_t& w0,
                                                    uint32_t& w1,
                                                    const float2* rtab) {
  using Ops = Half2Ops<H2>;
  uint32_t km = p[0] & 0x7FFF7FFFu;
#pragma unroll
  for (int i = 1; i < 8; ++i) km = __vmaxu2(km, p[i] & 0x7FFF7FFFu);
  const uint32_t key = max(km & 0xFFFFu, km >> 16);
  if (key > Ops::kInfKey) return quant_block16_x2_cmp<H2>(p, w0, w1);
  uint32_t x[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[2 * i] = __float_as_uint(Ops::lo(p[i]));
    x[2 * i + 1] = __float_as_uint(Ops::hi(p[i]));
  }
  return encode_rcp16(Ops::lo(key), x, w0, w1, rtab);
}

// The activation quantiser's fp32 block form: amax as the largest |v| bit
// pattern, then encode_rcp16_direct; a block holding a NaN goes to
// quant_block16.
__device__ __forceinline__ uint8_t quant_block16_rcp(const float (&v)[16],
                                                     uint32_t& w0,
                                                     uint32_t& w1) {
  uint32_t x[16];
  uint32_t km = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    x[i] = __float_as_uint(v[i]);
    km = max(km, x[i] & 0x7FFFFFFFu);
  }
  if (km > 0x7F800000u) return quant_block16(v, w0, w1);
  return encode_rcp16_direct(__uint_as_float(km), x, w0, w1);
}

}  // namespace nvfp4dg
