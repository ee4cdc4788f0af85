// Arithmetic of the 16-bit feed-forward operators (activations, their slopes,
// the 8-bit groups of activation checkpoints) and their memory-bound kernels.
#pragma once

#include <math_constants.h>

#include "common.cuh"

namespace dsv4 {

// ---- shared memory ----
__device__ __forceinline__ void st_shared_v4(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ void st_shared_u16(uint32_t a, uint32_t v) {
  asm volatile("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tst.shared.b16 [%0], h;\n\t}" ::"r"(a),
               "r"(v)
               : "memory");
}
__device__ __forceinline__ uint32_t ld_shared_u16(uint32_t a) {
  uint32_t v;
  asm volatile("{\n\t.reg .b16 h;\n\tld.shared.b16 h, [%1];\n\tcvt.u32.u16 %0, h;\n\t}"
               : "=r"(v)
               : "r"(a)
               : "memory");
  return v;
}

// 32 lanes x 32 consecutive fp32 columns of TMEM, waited on at once.
__device__ __forceinline__ void tmem_ld_f32x32(uint32_t taddr, float (&f)[32]) {
  int32_t v[32];
  tmem_ld_x32_wait(taddr, v);
#pragma unroll
  for (int j = 0; j < 32; ++j) f[j] = __int_as_float(v[j]);
}

__device__ __forceinline__ void tmem_ld_f32x16(uint32_t taddr, float (&f)[16]) {
  int32_t v[16];
  tmem_ld_x16(taddr, v);
  tmem_ld_wait_regs(v);
#pragma unroll
  for (int j = 0; j < 16; ++j) f[j] = __int_as_float(v[j]);
}

// ---- 16-bit values ----
template <bool BF16>
__device__ __forceinline__ uint32_t pack_16(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  }
  return r;
}

template <bool BF16>
__device__ __forceinline__ float unpack_16(uint32_t w, int hi) {
  if constexpr (BF16) {
    return __uint_as_float(hi ? (w & 0xffff0000u) : (w << 16));
  } else {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(hi ? w >> 16 : w)));
  }
}

template <bool BF16>
__device__ __forceinline__ float ld_16(const void* p, int64_t i) {
  return unpack_16<BF16>(static_cast<const uint16_t*>(p)[i], 0);
}

template <bool BF16>
__device__ __forceinline__ void pack_row(const float (&v)[32], uint32_t (&w)[16]) {
#pragma unroll
  for (int j = 0; j < 16; ++j) w[j] = pack_16<BF16>(v[2 * j], v[2 * j + 1]);
}

// ---- activations: value and slope ----
// Fast fp32: values within 2^-18 of |z| + 1 and, where they are small
// differences, within 2^-14 of themselves (results are rounded to 2^-8 or 2^-11
// of themselves); powers of two and reciprocals that underflow are 0.  gelu_tanh
// is z sigmoid(2a) with a = sqrt(2/pi) (z + 0.044715 z^3), since (1 + tanh a) / 2
// = sigmoid(2a).
enum Act : int { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4 };

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float rcp_approx(float a) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
  return r;
}

constexpr float kLog2E = 1.4426950408889634f;

// 1 / (1 + exp(-z))
__device__ __forceinline__ float sigmoid_fast(float z) {
  return rcp_approx(1.f + exp2_approx(-kLog2E * z));
}

constexpr float kGeluC = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluK = 0.044715f;

// The normal distribution's function and density times sqrt(2 pi), for gelu:
// the tail Phi(-x) = t (a1 + t (a2 + ...)) exp(-x^2 / 2), t = 1 / (1 + p x), x >=
// 0.  Coefficients and p fitted to Phi(-x) exp(x^2 / 2) on [0, 13.5] for the
// least largest error of the tail relative to itself, errors next to 0 weighted
// up to 32 times as high: off by at most 4.5e-7 absolute and, with the fp32
// exponent's rounding, 2^-15 of itself down to x = 12.5 (an error bounded
// absolutely alone passes half a bf16 step of the value from x = 5.5 on).  One
// exponential serves the value and the slope.
__device__ __forceinline__ float normal_cdf(float z, float& density) {
  const float t = rcp_approx(1.f + 0.2982272751f * fabsf(z));
  density = exp2_approx(z * z * (-0.5f * kLog2E));
  float q = -0.08083245341f * t + 0.2319667356f;
  q = q * t - 0.03341316405f;
  q = q * t + 0.1514508873f;
  q = q * t + 0.1113202308f;
  q = q * t + 0.1195077637f;
  q *= t * density;
  return z < 0.f ? q : 1.f - q;
}

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == kActRelu) return z <= 0.f ? 0.f : z;
  if constexpr (ACT == kActSilu) return z * sigmoid_fast(z);
  if constexpr (ACT == kActGelu) {
    float density;
    return z * normal_cdf(z, density);
  }
  if constexpr (ACT == kActGeluTanh)
    return z * sigmoid_fast(kGeluC * (z + kGeluK * z * z * z));
  return z;
}

template <int ACT>
__device__ __forceinline__ void act_both(float z, float& a, float& slope) {
  if constexpr (ACT == kActRelu) {
    a = z <= 0.f ? 0.f : z;
    slope = z <= 0.f ? 0.f : 1.f;
  } else if constexpr (ACT == kActSilu) {
    const float s = sigmoid_fast(z);
    a = z * s;
    slope = s * (1.f + z * (1.f - s));
  } else if constexpr (ACT == kActGelu) {
    float density;
    const float phi = normal_cdf(z, density);
    a = z * phi;
    slope = phi + z * 0.39894228040143268f * density;
  } else if constexpr (ACT == kActGeluTanh) {
    // past |z| = 100 the sigmoid is 0 or 1 and its slope 0: z is held there so
    // that infinity * 0 does not arise
    const float c = fminf(fmaxf(z, -100.f), 100.f);
    const float s = sigmoid_fast(kGeluC * (z + kGeluK * z * z * z));
    a = z * s;
    slope = s + s * (1.f - s) * kGeluC * (c + 3.f * kGeluK * c * c * c);
  } else {
    a = z;
    slope = 1.f;
  }
}

template <typename F>
__device__ __forceinline__ void act_dispatch(int act, F&& f) {
  switch (act) {
    case kActRelu: f(std::integral_constant<int, kActRelu>{}); break;
    case kActSilu: f(std::integral_constant<int, kActSilu>{}); break;
    case kActGelu: f(std::integral_constant<int, kActGelu>{}); break;
    case kActGeluTanh: f(std::integral_constant<int, kActGeluTanh>{}); break;
    default: f(std::integral_constant<int, kActNone>{}); break;
  }
}

__device__ __forceinline__ void act_row(int act, float (&v)[32]) {
  act_dispatch(act, [&](auto kind) {
    constexpr int K = decltype(kind)::value;
    if constexpr (K != kActNone) {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = act_value<K>(v[j]);
    }
  });
}

// min(g, limit) and clamp(u, -limit, limit), NaN kept (torch.clamp)
__device__ __forceinline__ float clamp_top(float g, float limit) { return g > limit ? limit : g; }
__device__ __forceinline__ float clamp_both(float u, float limit) {
  return u > limit ? limit : (u < -limit ? -limit : u);
}

template <int ACT>
__device__ __forceinline__ void gated_backward(float limit, float dh, float g, float u, float& dg,
                                               float& du, float& h) {
  const float gc = clamp_top(g, limit), uc = clamp_both(u, limit);
  float a, s;
  act_both<ACT>(gc, a, s);
  dg = g > limit ? 0.f : dh * uc * s;  // NaN passes: it has to show in the gradient
  du = fabsf(u) > limit ? 0.f : dh * a;
  h = a * uc;
}

// 16 columns of a row
template <bool BF16>
__device__ __forceinline__ void gated_backward_row(int act, float limit, const float (&dh)[16],
                                                   const float (&g)[16], const float (&u)[16],
                                                   uint32_t (&wg)[8], uint32_t (&wu)[8],
                                                   uint32_t (&wh)[8]) {
  act_dispatch(act, [&](auto kind) {
    constexpr int K = decltype(kind)::value;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float dg[2], du[2], h[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        gated_backward<K>(limit, dh[2 * j + i], g[2 * j + i], u[2 * j + i], dg[i], du[i], h[i]);
      wg[j] = pack_16<BF16>(dg[0], dg[1]);
      wu[j] = pack_16<BF16>(du[0], du[1]);
      wh[j] = pack_16<BF16>(h[0], h[1]);
    }
  });
}

// ---- 8-bit groups ----
// 32 values of a row share a scale: code = 127 v / amax rounded to the nearest
// whole number (ties to even) of the exact quotient, value = code * (amax / 127).
// 32 keeps a channel's outliers from costing its neighbours more than half a
// step of their own group, at 1.125 bytes per value.  A group that holds an
// infinity or a NaN has scale NaN (all of it decodes to NaN); one whose
// largest magnitude is below 2^-100 holds zeros.
constexpr int kGroup = 32;
constexpr float kTinyGroup = 7.8886090522101181e-31f;  // 2^-100


// Whole steps up to amax.  The scale is rounded toward zero: that many steps
// never pass amax, so the largest finite value stays finite.
constexpr float kSteps8 = 127.f;

__device__ __forceinline__ float group_step(uint32_t amax_bits, float steps) {
  const float amax = __uint_as_float(amax_bits);
  if (amax_bits >= 0x7f800000u) return CUDART_NAN_F;
  if (amax < kTinyGroup) return 0.f;
  // the product is within two units of the last place of the quotient, and the
  // remainder of a neighbour is exact: the largest with none below zero
  float y = amax * (1.f / steps);
  if (__fmaf_rn(-y, steps, amax) < 0.f) y = __uint_as_float(__float_as_uint(y) - 1);
  if (__fmaf_rn(-y, steps, amax) < 0.f) y = __uint_as_float(__float_as_uint(y) - 1);
  const float up = __uint_as_float(__float_as_uint(y) + 1);
  if (__fmaf_rn(-up, steps, amax) >= 0.f) y = up;
  return y;
}

// steps / amax to about 2^-22; 0 for a group that holds zeros or decodes to NaN
__device__ __forceinline__ float group_inverse(uint32_t amax_bits, float steps) {
  const float amax = __uint_as_float(amax_bits);
  if (amax_bits >= 0x7f800000u || amax < kTinyGroup) return 0.f;
  return amax > 1.8446744e19f ? (steps * 5.4210109e-20f) * rcp_approx(amax * 5.4210109e-20f)
                              : steps * rcp_approx(amax);  // 2^64, 2^-64
}

// Correctly rounded 127 v / amax for 16-bit v: p = 127 v is exact, the first
// estimate is off by a few units of the last place, and one step with the
// exact remainder p - q amax mends that.  A tie (k + 1/2) comes out as itself.
__device__ __forceinline__ float group_quotient(float v, float amax) {
  const float shrink = amax > 1.8446744e19f ? 5.4210109e-20f : 1.f;
  const float a = amax * shrink, r = rcp_approx(a), p = v * (127.f * shrink), q = p * r;
  return __fmaf_rn(__fmaf_rn(-q, a, p), r, q);
}

// 16-bit values.  A tie 254 v = (2k + 1) amax needs k = 63 unless amax's
// significand is a multiple of 127: then |v| = amax / 2 and the code is 64, the
// even neighbour, away from zero.  No other quotient of 16-bit values lies
// within 2^-19 (relative) of a half.  So v * inverse * (1 + 2^-21), off by at
// most 2^-22 more, rounds every value of such a group as the exact quotient.
// Groups with the special significand (1 in 128) take the exact one.
constexpr float kTieBias = 1.f + 1.f / 2097152.f;

__device__ __forceinline__ bool group_special(uint32_t amax_bits) {
  return (((amax_bits >> 13) & 0x3ffu) + 1024u) % 127u == 0;
}

// fp32 values: within 6e-5 of a half the sign of 127 v - (f + 1/2) amax
// decides, taken exactly (both products as rounded part + remainder).
__device__ __noinline__ int quantize_code_near(float v, float q, float amax) {
  const float f = floorf(fabsf(q));
  if (fabsf(fabsf(q) - f - 0.5f) >= 6e-5f) return __float2int_rn(q);
  const float shrink = amax > 1.8446744e19f ? 5.4210109e-20f : 1.f;
  const float x = fabsf(v) * shrink, a = amax * shrink, c = f + 0.5f;
  const float p = 127.f * x, pl = __fmaf_rn(127.f, x, -p);
  const float t = c * a, tl = __fmaf_rn(c, a, -t);
  const float d = (p - t) + (pl - tl);
  const int fi = static_cast<int>(f);
  const int r = d > 0.f ? fi + 1 : d < 0.f ? fi : fi + (fi & 1);
  return q < 0.f ? -r : r;
}

// Adding 1.5 * 2^23 rounds to the nearest whole number (ties to even) and leaves
// it in the low bits, so a code is one fused multiply-add of value and inverse.
constexpr float kWhole = 12582912.f;

// Four such sums -> four code bytes.
__device__ __forceinline__ uint32_t pack_codes(float a, float b, float c, float d) {
  const uint32_t lo = prmt(__float_as_uint(a), __float_as_uint(b), 0x0040u);
  const uint32_t hi = prmt(__float_as_uint(c), __float_as_uint(d), 0x0040u);
  return prmt(lo, hi, 0x5410u);
}

// 4 codes of fp32 values
__device__ __forceinline__ uint32_t quantize4_f32(const float (&v)[4], float inverse, float amax) {
  float q[4], near = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    q[i] = v[i] * inverse;
    near = fmaxf(near, fabsf(q[i] - rintf(q[i])));
  }
  if (near > 0.4999f) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w |= (static_cast<uint32_t>(quantize_code_near(v[i], q[i], amax)) & 0xffu) << (8 * i);
    return w;
  }
  return pack_codes(q[0] + kWhole, q[1] + kWhole, q[2] + kWhole, q[3] + kWhole);
}

// What the backward pass needs of a value before its activation is kept as
// groups too, in 8 bits or in 16: a thread's own 32 fp32 sums -> codes and the
// scale.  (A sum next to the border of two codes is itself only known to its
// last bits.)  16 bits hold a value to 2^-15 of the group's largest, where bf16
// may be off by 2^-8 of every value: gradients are then as exact as their own
// rounding, at 2.125 bytes a value.
__device__ __forceinline__ uint32_t group_top(const float (&v)[32]) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  return top;
}

__device__ __forceinline__ float keep_group8(const float (&v)[32], uint32_t (&codes)[8]) {
  const uint32_t top = group_top(v);
  const float inv = group_inverse(top, kSteps8);
  if (inv == 0.f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) codes[j] = 0;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      codes[j] = pack_codes(__fmaf_rn(v[4 * j], inv, kWhole), __fmaf_rn(v[4 * j + 1], inv, kWhole),
                            __fmaf_rn(v[4 * j + 2], inv, kWhole), __fmaf_rn(v[4 * j + 3], inv, kWhole));
  }
  return group_step(top, kSteps8);
}

// 16 bits: a sign and 15 bits of magnitude that count up with the value, in
// steps of the group's largest value / kSteps.  From kEdge steps on the code is
// the whole number of steps; below that the leading bits of a float, kBits
// digits behind the leading one (at code 2^14 both are kEdge steps, and both go
// on by one step).  So a value is held to half a step (2^-15 of the largest) and,
// where that is more, to 2^-(kBits + 1) of itself: 2^-10 for bf16 tensors, 2^-11
// for fp16, at least as well as in the tensor's own type.  No value loses its
// digits to larger neighbours, however many there are.  (Down to 2^-36 of the
// largest, 2^-19 for fp16, which trades range for a digit; below that to 2^-45
// and 2^-29 of it.)
//
// Equal steps, with a test for a value that stands out of its group, cost less
// but fail beside two such values: their own squares raise the mean they are
// compared with.  Here against that: 2048 x 2048 -> 7168, z kept, gelu 59.7 us
// (59.0), its activation backward 23.8 (22.2); gated 4096 x 1024 -> 2 x 2048 45
// (40), its backward pass 43.8 (40.3); gated 4096 x 7168 -> 2 x 2048 174 (172).
template <bool BF16>
struct Kept16 {
  static constexpr int kBits = BF16 ? 9 : 10;
  static constexpr int kEdge = 1 << kBits;
  static constexpr int kShift = 23 - kBits;
  // the largest is code 32766: one is left to count it up
  static constexpr float kSteps = 32766 - 16384 + kEdge;
  static constexpr float kLinear = 8388608.f + (16384 - kEdge);  // 2^23 and the code of no steps
  // kEdge times the power of two has the bits 2^14 << kShift
  static constexpr float kToFine = BF16 ? 0x1p-104f * (1.f + 0x1p-10f) : 0x1p-121f * (1.f + 0x1p-11f);
  static constexpr float kFromFine = BF16 ? 0x1p104f : 0x1p121f;
};

// The value of the code in the lower or upper (`hi`) half of w; scale > 0.
template <bool BF16>
__device__ __forceinline__ float kept16_value(uint32_t w, int hi, float scale) {
  using K = Kept16<BF16>;
  const uint32_t p = prmt(w & 0x7fff7fffu, 0x4b000000u, hi ? 0x7432u : 0x7410u);  // 2^23 + magnitude
  const float linear = __uint_as_float(p) - K::kLinear;
  const float fine = __uint_as_float(p << K::kShift) * K::kFromFine;
  const float v = scale * (linear >= K::kEdge ? linear : fine);
  return __uint_as_float(__float_as_uint(v) | ((hi ? w : w << 16) & 0x80000000u));
}

// Magnitude code (its low 15 bits) of |t| steps.  Below the edge the float's
// digits are cut, not rounded: kToFine stands half a step above its power of
// two, so that the error stays within 2^-(kBits + 1) to either side.
template <bool BF16>
__device__ __forceinline__ uint32_t kept16_magnitude(float t) {
  using K = Kept16<BF16>;
  uint32_t m;
  asm("{\n\t.reg .pred p;\n\t.reg .f32 a;\n\t"
      "abs.f32 a, %1;\n\t"
      "setp.ge.f32 p, a, %2;\n\t"
      "mul.f32 %0, %1, %3;\n\t"
      "shr.u32 %0, %0, %4;\n\t"
      "@p add.f32 %0, a, %5;\n\t}"
      : "=&r"(m)
      : "f"(t), "f"(static_cast<float>(K::kEdge)), "f"(K::kToFine), "n"(K::kShift), "f"(K::kLinear));
  return m;
}

// Codes of two values: their magnitudes' and their signs.
__device__ __forceinline__ uint32_t kept16_signs(uint32_t m, float v0, float v1) {
  const uint32_t signs = prmt(__float_as_uint(v0), __float_as_uint(v1), 0x7632u);
  return (m & 0x7fff7fffu) | (signs & 0x80008000u);
}

template <bool BF16>
__device__ __forceinline__ uint32_t kept16_codes(float v0, float v1, float inv) {
  const uint32_t m0 = kept16_magnitude<BF16>(v0 * inv), m1 = kept16_magnitude<BF16>(v1 * inv);
  return kept16_signs(prmt(m0, m1, 0x5410u), v0, v1);
}

// max(|a|, |b|, |c|); NaN if one is
__device__ __forceinline__ float max_abs_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A group that holds an infinity or a NaN: fp16 multiples of a power of two,
// which lose only that value, marked by a negative scale.
__device__ __forceinline__ float keep_not_finite(const float (&v)[32], float limit, bool keep_sign,
                                                 uint32_t (&codes)[16]) {
  uint32_t top = 0;  // of the finite values
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const uint32_t b = __float_as_uint(v[j]) & 0x7fffffffu;
    if (b < 0x7f800000u) top = max(top, b);
  }
  // the largest lands in [2^14, 2^15); scales from 2^-114 to 2^113
  const uint32_t e = max(top >> 23, 27u) - 14u;
  const float unit = __uint_as_float(e << 23), inv = __uint_as_float((254u - e) << 23);
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    uint32_t w = pack_16<false>(v[2 * j] * inv, v[2 * j + 1] * inv);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x = v[2 * j + i];
      const uint32_t one = i ? 0x10000u : 1u;  // magnitudes count up away from zero
      if (keep_sign && (w & (0x7fffu * one)) == 0 && x != 0.f) w += one;
      const bool over = fabsf(x) > limit, kept = fabsf(unit * unpack_16<false>(w, i)) > limit;
      if (over && !kept) w += one;
      if (!over && kept) w -= one;
    }
    codes[j] = w;
  }
  return -unit;
}

// With a clamp limit the code stays on the value's side of it: the backward
// pass asks |z| <= limit of the kept value, and one kept over the border would
// lose or gain its whole gradient.  Values read back count up with the code, so
// codes are held below and above the border between two of them.  For relu a
// value other than zero keeps its sign the same way.  That is one step instead
// of half a step next to the border.
template <bool BF16>
__device__ __forceinline__ float keep_group16(const float (&v)[32], float limit, bool keep_sign,
                                              uint32_t (&codes)[16]) {
  using K = Kept16<BF16>;
  float most = fabsf(v[0]);
#pragma unroll
  for (int j = 0; j < 16; ++j) most = max_abs_nan(most, v[2 * j], v[2 * j + 1]);
  if (!(most < CUDART_INF_F)) return keep_not_finite(v, limit, keep_sign, codes);
  const uint32_t top = __float_as_uint(fmaxf(most, kTinyGroup));
  const float inv = group_inverse(top, K::kSteps), scale = group_step(top, K::kSteps);
  // (no kept value is off by 2^-8 of itself: further below the limit there is no side to keep)
  if (most * (1.f + 0x1p-8f) <= limit && !keep_sign) {
#pragma unroll
    for (int j = 0; j < 16; ++j) codes[j] = kept16_codes<BF16>(v[2 * j], v[2 * j + 1], inv);
    return scale;
  }
  // the last code that is read back within the limit (32767 where all are)
  int last = kept16_magnitude<BF16>(fminf(limit * inv, K::kSteps + 1.f)) & 0x7fffu;
  if (last < 32767 && kept16_value<BF16>(last + 1, 0, scale) <= limit) ++last;
  if (kept16_value<BF16>(last, 0, scale) > limit) --last;
  if (kept16_value<BF16>(last, 0, scale) > limit) --last;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    int m[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x = fabsf(v[2 * j + i]);
      m[i] = kept16_magnitude<BF16>(x * inv) & 0x7fffu;
      m[i] = x > limit ? max(m[i], last + 1) : min(m[i], last);
      if (keep_sign && m[i] == 0 && x != 0.f) m[i] = 1;
    }
    codes[j] = kept16_signs(prmt(m[0], m[1], 0x5410u), v[2 * j], v[2 * j + 1]);
  }
  return scale;
}

// N 16-bit codes of a group (scale < 0: fp16 multiples) -> values
template <bool BF16, int N>
__device__ __forceinline__ void kept16_values(const uint32_t (&w)[N / 2], float scale, float (&v)[N]) {
  if (scale < 0.f) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = -scale * unpack_16<false>(w[j >> 1], j & 1);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = kept16_value<BF16>(w[j >> 1], j & 1, scale);
  }
}

__device__ __forceinline__ float code8_value(uint32_t w, int byte) {
  return __uint_as_float(prmt(w ^ 0x80808080u, 0x4b000000u, 0x7440u + byte)) - 8388736.f;
}

// No pointer of the kernels below is __restrict__: under programmatic dependent
// launch a kernel's blocks may be resident while the kernel before it still
// writes what they will read, and a load from memory declared read-only may
// take the non-coherent path, which the wait at entry says nothing about.

// ---- 8 consecutive 16-bit values from any even address ----
// A matrix's first byte and the one behind its last.
struct Extent {
  uint64_t lo, hi;
};

__device__ __forceinline__ Extent extent_of(const uint16_t* p, int64_t rows, int64_t ld, int64_t k) {
  const uint64_t lo = reinterpret_cast<uint64_t>(p);
  return {lo, lo + 2 * static_cast<uint64_t>((rows - 1) * ld + k)};
}

// The two aligned 16-byte pieces around 8 values.
struct Window {
  uint4 a, b;
};

__device__ __forceinline__ Window load_window(const uint16_t* p, int left, const Extent& e) {
  const uint64_t at = reinterpret_cast<uint64_t>(p) & ~15ull;
  Window w;
  if (left >= 8 && at >= e.lo && at + 32 <= e.hi) {
    w.a = *reinterpret_cast<const uint4*>(at);
    w.b = *reinterpret_cast<const uint4*>(at + 16);
  } else {  // at the matrix's ends: the 8 values themselves, put where the shift finds them
    uint32_t v[8] = {};
    const int off = static_cast<int>(reinterpret_cast<uint64_t>(p) & 15) >> 1;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int j = i - off;
      if (j >= 0 && j < 8 && j < left) v[i >> 1] |= static_cast<uint32_t>(p[j]) << (16 * (i & 1));
    }
    w.a = make_uint4(v[0], v[1], v[2], v[3]);
    w.b = make_uint4(v[4], v[5], v[6], v[7]);
  }
  return w;
}

// 16 bytes of the window from byte `off` (even, below 16)
__device__ __forceinline__ uint4 shift_window(const Window& w, int off) {
  const uint32_t v[8] = {w.a.x, w.a.y, w.a.z, w.a.w, w.b.x, w.b.y, w.b.z, w.b.w};
  uint32_t t[6], u[5];
#pragma unroll
  for (int i = 0; i < 6; ++i) t[i] = off & 8 ? v[i + 2] : v[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) u[i] = off & 4 ? t[i + 1] : t[i];
  const int bits = off & 2 ? 16 : 0;
  return make_uint4(__funnelshift_r(u[0], u[1], bits), __funnelshift_r(u[1], u[2], bits),
                    __funnelshift_r(u[2], u[3], bits), __funnelshift_r(u[3], u[4], bits));
}

// 8 consecutive 16-bit values of a row, packed; those past `cols` read as 0.
__device__ __forceinline__ uint4 load_words8(const void* base, int64_t at, int64_t col, int64_t cols,
                                             bool vec) {
  const uint16_t* p = static_cast<const uint16_t*>(base) + at;
  if (vec && col + 8 <= cols) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4] = {};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (col + j < cols) w[j >> 1] |= static_cast<uint32_t>(p[j]) << (16 * (j & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int DT>
__device__ __forceinline__ void store_piece8(void* base, int64_t at, int64_t col, int64_t cols,
                                             bool vec, const float (&v)[8]) {
  if constexpr (DT == DSV4_F32) {
    float* p = static_cast<float*>(base) + at;
    if (vec && col + 8 <= cols) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < cols) p[j] = v[j];
    }
  } else {
    constexpr bool BF16 = DT == DSV4_BF16;
    uint16_t* p = static_cast<uint16_t*>(base) + at;
    const uint32_t w[4] = {pack_16<BF16>(v[0], v[1]), pack_16<BF16>(v[2], v[3]),
                           pack_16<BF16>(v[4], v[5]), pack_16<BF16>(v[6], v[7])};
    if (vec && col + 8 <= cols) {
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < cols) p[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
    }
  }
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// ---- activation checkpoint: rows -> 8-bit groups ----
// A block takes 32 rows x 256 columns.  A lane owns 8 columns (a quarter of a
// group, 16 bytes of a 16-bit row), so a warp reads 512 contiguous bytes of a
// row and writes 256 of codes; it keeps its four rows' loads in flight
// together.  The four lanes of a group work out one row's scale each and share
// it.  Scales lie [group][row]; they pass through shared memory so that a warp
// writes one group's 32 rows together.  Codes rows are padded to the group
// with zeros.  Bound by issue slots next to memory: 16-bit rows stay packed
// through the maximum (two values an instruction) and a code costs one
// multiply-add.  8192 x 7168 bf16: 32 us (5.8 TB/s), back again 31 us.
// 16-bit rows that are not 16-byte aligned come as windows of two pieces and
// go as pieces put together from two lanes (8192 x 7166: 46 and 58 us; value by
// value 53 and 155).
template <int DT, bool VEC>
__global__ void __launch_bounds__(256, DT == DSV4_F32 || !VEC ? 4 : 6)
    checkpoint_kernel(const void* x, int64_t ld, int64_t m, int64_t k,
                      int64_t k32, uint32_t col_blocks, int8_t* codes,
                      float* scales) {
  pdl_entry();
  constexpr bool F32 = DT == DSV4_F32;
  constexpr int kWords = F32 ? 8 : 4;
  __shared__ float s_scale[8][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t row_block = blockIdx.x / col_blocks, col_block = blockIdx.x - row_block * col_blocks;
  const int64_t row0 = static_cast<int64_t>(row_block) * 32 + warp;
  const int64_t col = static_cast<int64_t>(col_block) * 256 + lane * 8;
  const uint32_t* const p =
      reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(x) + (row0 * ld + col) * (F32 ? 4 : 2));
  const int64_t step = 8 * ld * (F32 ? 4 : 2);
  uint32_t raw[4][kWords];
  if (!VEC && !F32 && col < k) {
    const uint16_t* const first = static_cast<const uint16_t*>(x);
    const Extent e = extent_of(first, m, ld, k);
    const int left = k - col < 8 ? static_cast<int>(k - col) : 8;
    Window w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i].a = w[i].b = make_uint4(0, 0, 0, 0);
      if (row0 + 8 * i < m) w[i] = load_window(first + (row0 + 8 * i) * ld + col, left, e);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = shift_window(w[i], static_cast<int>(reinterpret_cast<uint64_t>(first + (row0 + 8 * i) * ld + col) & 15));
      raw[i][0] = v.x, raw[i][1] = v.y, raw[i][2] = v.z, raw[i][3] = v.w;
    }
  } else if (VEC && col + 8 <= k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* q = reinterpret_cast<const uint8_t*>(p) + i * step;
#pragma unroll
      for (int h = 0; h < kWords; h += 4) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row0 + 8 * i < m) v = *reinterpret_cast<const uint4*>(q + 4 * h);
        raw[i][h] = v.x, raw[i][h + 1] = v.y, raw[i][h + 2] = v.z, raw[i][h + 3] = v.w;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* q = reinterpret_cast<const uint8_t*>(p) + i * step;
#pragma unroll
      for (int j = 0; j < kWords; ++j) raw[i][j] = 0;
      if (row0 + 8 * i >= m) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (col + j >= k) continue;
        if constexpr (F32) {
          raw[i][j] = reinterpret_cast<const uint32_t*>(q)[j];
        } else {
          raw[i][j >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(q)[j]) << (16 * (j & 1));
        }
      }
    }
  }
  // the bits of |largest value|: as whole numbers they order like the values,
  // infinities and NaN above all
  uint32_t top[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (F32) {
      uint32_t t = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) t = max(t, raw[i][j] & 0x7fffffffu);
      t = max(t, __shfl_xor_sync(0xffffffffu, t, 1));
      top[i] = max(t, __shfl_xor_sync(0xffffffffu, t, 2));
    } else {
      uint32_t t = raw[i][0] & 0x7fff7fffu;
#pragma unroll
      for (int j = 1; j < 4; ++j) t = max_u16x2(t, raw[i][j] & 0x7fff7fffu);
      t = max_u16x2(t, __shfl_xor_sync(0xffffffffu, t, 1));
      t = max_u16x2(t, __shfl_xor_sync(0xffffffffu, t, 2));
      t = max(t & 0xffffu, t >> 16);
      top[i] = __float_as_uint(unpack_16<DT == DSV4_BF16>(t, 0));
    }
  }
  const int sub = lane & 3;
  const uint32_t mine = sub == 0 ? top[0] : sub == 1 ? top[1] : sub == 2 ? top[2] : top[3];
  s_scale[lane >> 2][warp + 8 * sub] = group_step(mine, kSteps8);
  float own = group_inverse(mine, kSteps8);
  if (!F32) own = group_special(mine) ? -own : own * kTieBias;
  int8_t* const c = codes + row0 * k32 + col;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float inv = __shfl_sync(0xffffffffu, own, (lane & 28) + i);
    uint32_t w[2] = {0, 0};
    if constexpr (F32) {
      if (inv != 0.f) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(raw[i][4 * h + j]);
          w[h] = quantize4_f32(v, inv, __uint_as_float(top[i]));
        }
      }
    } else {
      float q[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) q[j] = unpack_16<DT == DSV4_BF16>(raw[i][j >> 1], j & 1);
      if (inv > 0.f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = __fmaf_rn(q[j], inv, kWhole);
      } else if (inv < 0.f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = group_quotient(q[j], __uint_as_float(top[i])) + kWhole;
      } else {  // zeros, or a group that holds an infinity or a NaN
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = kWhole;
      }
      w[0] = pack_codes(q[0], q[1], q[2], q[3]);
      w[1] = pack_codes(q[4], q[5], q[6], q[7]);
    }
    if (row0 + 8 * i < m && col < k32)
      *reinterpret_cast<uint2*>(c + i * 8 * k32) = make_uint2(w[0], w[1]);
  }
  __syncthreads();
  const int64_t group = static_cast<int64_t>(col_block) * 8 + warp, row = row0 - warp + lane;
  if (group * kGroup < k32 && row < m) scales[group * m + row] = s_scale[warp][lane];
}

// 8 values of each lane, side by side from an even address on that is not
// 16-byte aligned: a lane stores the aligned piece that begins in the lane
// before it; what no piece covers goes value by value.  All lanes take part.
__device__ __forceinline__ void store_shifted8(uint16_t* p, const uint32_t (&w)[4], int lane, int64_t col,
                                               int64_t cols) {
  const int off = static_cast<int>(reinterpret_cast<uint64_t>(p) & 15);  // the same in all lanes
  const int head = (16 - off) >> 1;  // values before the next aligned address
  Window two;
  two.b = make_uint4(w[0], w[1], w[2], w[3]);
  two.a = make_uint4(__shfl_up_sync(0xffffffffu, w[0], 1), __shfl_up_sync(0xffffffffu, w[1], 1),
                     __shfl_up_sync(0xffffffffu, w[2], 1), __shfl_up_sync(0xffffffffu, w[3], 1));
  const bool whole = lane > 0 && col + head <= cols, next = lane < 31 && col + 8 + head <= cols;
  if (whole) *reinterpret_cast<uint4*>(p + head - 8) = shift_window(two, 16 - off);
  if (!whole || !next) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j < cols && (j < head ? !whole : !next)) p[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
  }
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(256, VEC ? 8 : 5)
    restore_kernel(const int8_t* codes, const float* scales, int64_t m,
                   int64_t k, int64_t k32, uint32_t col_blocks, void* out, int64_t ldo) {
  pdl_entry();
  __shared__ float s_scale[8][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t row_block = blockIdx.x / col_blocks, col_block = blockIdx.x - row_block * col_blocks;
  const int64_t row0 = static_cast<int64_t>(row_block) * 32;
  const int64_t col = static_cast<int64_t>(col_block) * 256 + lane * 8;
  uint2 c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = row0 + warp + 8 * i;
    c[i] = make_uint2(0, 0);
    if (row < m && col < k32) c[i] = *reinterpret_cast<const uint2*>(codes + row * k32 + col);
  }
  const int64_t group = static_cast<int64_t>(col_block) * 8 + warp, srow = row0 + lane;
  s_scale[warp][lane] = group * kGroup < k32 && srow < m ? scales[group * m + srow] : 0.f;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = row0 + warp + 8 * i;
    const float s = s_scale[lane >> 2][warp + 8 * i];
    const uint32_t w[2] = {c[i].x, c[i].y};
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = s * code8_value(w[j >> 2], j & 3);
    uint16_t* const at = static_cast<uint16_t*>(out) + row * ldo + col;
    if (DT != DSV4_F32 && !VEC && (reinterpret_cast<uint64_t>(at) & 15) != 0) {
      constexpr bool BF16 = DT == DSV4_BF16;
      const uint32_t q[4] = {pack_16<BF16>(v[0], v[1]), pack_16<BF16>(v[2], v[3]),
                             pack_16<BF16>(v[4], v[5]), pack_16<BF16>(v[6], v[7])};
      if (row < m) store_shifted8(at, q, lane, col, k);
    } else if (row < m && col < k) {
      store_piece8<DT>(out, row * ldo + col, col, k, VEC || DT != DSV4_F32, v);
    }
  }
}

// ---- backward of activation and bias ----
// dz = dy act'(z), and the column sums of dz over a slab of rows (the bias
// gradient's partial sums, added by column_sum_kernel in slab order: the same
// result every time).  One pass over dy and z.  Without an activation only
// the sums are formed (dz = dy).  A lane owns 8 columns, a block 256; warps
// take every eighth row of the slab.  Bound by its arithmetic next to memory:
// 2048 x 7168 bf16 and its bias gradient take 23 us for gelu (the next row's
// loads in flight save 9) and 18 for relu.
struct ActBackward {
  const void* dy;
  int64_t lddy;
  int vec_dy;
  const void* zq;  // kept z: codes [m][n32] of zbits and scales [n32 / 32][m]
  int zbits;
  const float* zs;
  int64_t n32;
  void* dz;       // null: sums only
  int64_t lddz;
  int vec_dz;
  float* partial;  // [slabs][n] or null
  int64_t m, n, slab_rows;
  int act;
};

template <bool BF16>
__global__ void __launch_bounds__(256, 4) act_backward_kernel(const ActBackward p) {
  pdl_entry();
  constexpr int DT = BF16 ? DSV4_BF16 : DSV4_F16;
  __shared__ float s_sum[8][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 256 + lane * 8;
  const int64_t begin = static_cast<int64_t>(blockIdx.y) * p.slab_rows;
  const int64_t end = begin + p.slab_rows < p.m ? begin + p.slab_rows : p.m;
  float sum[8] = {};
  if (col < p.n) {
    act_dispatch(p.act, [&](auto kind) {
      constexpr int K = decltype(kind)::value;
      const float* const zs = p.zs + col / kGroup * p.m;
      // the next row's loads are in flight while a row is worked on
      const auto fetch = [&](int64_t row, uint4& d, uint4& c, float& s) {
        d = load_words8(p.dy, row * p.lddy + col, col, p.n, p.vec_dy);
        if constexpr (K != kActNone) {
          s = zs[row];
          if (p.zbits == 8) {
            const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(p.zq) + row * p.n32 + col);
            c.x = q.x, c.y = q.y;
          } else {
            c = *reinterpret_cast<const uint4*>(static_cast<const int16_t*>(p.zq) + row * p.n32 + col);
          }
        }
      };
      uint4 nd = {}, nc = {};
      float ns = 0.f;
      if (begin + warp < end) fetch(begin + warp, nd, nc, ns);
#pragma unroll 1
      for (int64_t row = begin + warp; row < end; row += 8) {
        const uint32_t dw[4] = {nd.x, nd.y, nd.z, nd.w}, c[4] = {nc.x, nc.y, nc.z, nc.w};
        const float s = ns;
        if (row + 8 < end) fetch(row + 8, nd, nc, ns);
        float d[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = unpack_16<BF16>(dw[j >> 1], j & 1);
        if constexpr (K != kActNone) {
          float z[8];
          if (p.zbits == 8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) z[j] = s * code8_value(c[j >> 2], j & 3);
          } else {
            kept16_values<BF16>(c, s, z);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float a, slope;
            act_both<K>(z[j], a, slope);
            d[j] *= slope;  // (past the last column dy is 0, and the sum is not stored)
          }
          store_piece8<DT>(p.dz, row * p.lddz + col, col, p.n, p.vec_dz, d);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += d[j];
      }
    });
  }
  if (!p.partial) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) s_sum[warp][lane * 8 + j] = sum[j];
  __syncthreads();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c < p.n) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += s_sum[w][threadIdx.x];
    p.partial[blockIdx.y * p.n + c] = t;
  }
}

// A block: 32 columns; its 8 warps take every eighth slab, then add up.
template <bool BF16>
__global__ void __launch_bounds__(256)
    column_sum_kernel(const float* partial, int64_t slabs, int64_t n,
                      void* out) {
  pdl_entry();
  __shared__ float s_sum[8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float t = 0.f;
  if (c < n) {
#pragma unroll 4
    for (int64_t s = warp; s < slabs; s += 8) t += partial[s * n + c];
  }
  s_sum[warp][lane] = t;
  __syncthreads();
  if (warp != 0 || c >= n) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) t += s_sum[w][lane];
  static_cast<uint16_t*>(out)[c] = static_cast<uint16_t>(pack_16<BF16>(t, 0.f) & 0xffffu);
}

// ---- rows of any strides -> rows that TMA can read (16-byte aligned) ----
// 32 x 32 tiles through shared memory: reads follow the smaller stride.
__global__ void __launch_bounds__(256)
    pack_rows_kernel(const uint16_t* in, int64_t s0, int64_t s1, int64_t rows,
                     int64_t cols, uint32_t col_blocks, uint16_t* out, int64_t ldo) {
  pdl_entry();
  __shared__ uint16_t tile[32][33];
  const int a = threadIdx.x & 31, b = threadIdx.x >> 5;
  const uint32_t row_block = blockIdx.x / col_blocks, col_block = blockIdx.x - row_block * col_blocks;
  const int64_t r0 = static_cast<int64_t>(row_block) * 32, c0 = static_cast<int64_t>(col_block) * 32;
  const bool by_rows = s1 <= s0 || s0 == 0;
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const int r = by_rows ? b + i : a, c = by_rows ? a : b + i;
    if (r0 + r < rows && c0 + c < cols) tile[r][c] = in[(r0 + r) * s0 + (c0 + c) * s1];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    if (r0 + b + i < rows && c0 + a < cols) out[(r0 + b + i) * ldo + c0 + a] = tile[b + i][a];
}

// Rows of contiguous values, from any even address to 16-byte aligned ones:
// windows of two pieces, shifted (8192 x 7167: 39 us; through the tiles 110).
__global__ void __launch_bounds__(256)
    pack_windows_kernel(const uint16_t* in, int64_t ld, int64_t rows, int64_t cols,
                        uint32_t col_blocks, uint16_t* out, int64_t ldo) {
  pdl_entry();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t row_block = blockIdx.x / col_blocks, col_block = blockIdx.x - row_block * col_blocks;
  const int64_t row0 = static_cast<int64_t>(row_block) * 32 + warp;
  const int64_t col = static_cast<int64_t>(col_block) * 256 + lane * 8;
  if (col >= cols) return;
  const int left = cols - col < 8 ? static_cast<int>(cols - col) : 8;
  const Extent e = extent_of(in, rows, ld, cols);
  Window w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i].a = w[i].b = make_uint4(0, 0, 0, 0);
    if (row0 + 8 * i < rows) w[i] = load_window(in + (row0 + 8 * i) * ld + col, left, e);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = row0 + 8 * i;
    if (row >= rows) break;
    const uint4 v = shift_window(w[i], static_cast<int>(reinterpret_cast<uint64_t>(in + row * ld + col) & 15));
    uint16_t* const q = out + row * ldo + col;
    if (left == 8) {
      *reinterpret_cast<uint4*>(q) = v;
    } else {
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < left) q[j] = static_cast<uint16_t>(u[j >> 1] >> (16 * (j & 1)));
    }
  }
}

}  // namespace dsv4
