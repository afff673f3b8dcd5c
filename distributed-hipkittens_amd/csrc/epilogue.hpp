// Epilogue of the dense FP8 products: act(z + bias) + residual, fp32, of the four
// consecutive columns that a lane holds, rounded once when the caller stores them.
//
//   silu(z) = z / (1 + e^-z),  gelu(z) = z Phi(z),
//   gelu_tanh(z) = z (1 + tanh u) / 2 = z / (1 + e^-2u),  u = sqrt(2/pi) (z + 0.044715 z^3)
//
// with the hardware exp2 and reciprocal (an ulp each); the reciprocal is 0 from 2^126 on, which makes SiLU 0 below
// z = -87.3, where it is -1e-36 (1 / (1 + 2^x) as the square of 2^(-x/2) there keeps the normal numbers and cost
// 8192x14336x512 28 us of 109 as a select, 6 behind a branch that no ordinary value takes).  Phi through its
// tail: with
// t = min(|z|, 20) and s = 1 / (1 + 0.31 t),
//   Q(t) = Phi(-t) = e^(-t^2/2) P(s),   gelu(z) = max(z, 0) - t Q(t)
// where P, of degree 8 without a constant term, is fitted to Phi(-t) e^(t^2/2) in relative error,
// 2.1e-7 at most over 0 <= t <= 21 (least squares reweighted towards the largest error), so that small
// negative results keep their bits, too.  15 instructions and two of the transcendental unit's,
// where erff takes about 40.  Past 20, Q is 0 in fp32.
#pragma once

#include "common.hpp"

namespace hkmoe {

enum class Act : int32_t { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3, kGeluTanh = 4 };

struct EpilogueArgs {
  const void* bias;      // [N] or null
  const void* residual;  // [M, N] in C's type, or null; may be C
  Act act;
  int32_t bias_f32;
};

// 1 / (1 + 2^x)
__device__ __forceinline__ float inv_1_exp2(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x)); }

__device__ __forceinline__ float gelu_erf(float z) {
  const float t = fminf(fabsf(z), 20.0f);  // a NaN's 20 does no harm: the first term keeps it
  const float s = __builtin_amdgcn_rcpf(__builtin_fmaf(0.31f, t, 1.0f));
  float p = 0.035773511f;
  p = __builtin_fmaf(p, s, -0.14138612f);
  p = __builtin_fmaf(p, s, 0.15481046f);
  p = __builtin_fmaf(p, s, -0.014781747f);
  p = __builtin_fmaf(p, s, 0.11010987f);
  p = __builtin_fmaf(p, s, 0.10775089f);
  p = __builtin_fmaf(p, s, 0.12406693f);
  p = __builtin_fmaf(p, s, 0.12365626f);
  const float e = __builtin_amdgcn_exp2f(t * t * -0.72134752f) * s;  // log2(e) / 2
  return __builtin_fmaf(-t, p * e, z < 0.0f ? 0.0f : z);
}

__device__ __forceinline__ f32x4 activate(f32x4 z, Act act) {
  // `act` is the same for the whole launch: scalar branches
  if (act == Act::kRelu) {
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = z[i] < 0.0f ? 0.0f : z[i];  // a NaN stays
  } else if (act == Act::kSilu) {
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = z[i] * inv_1_exp2(z[i] * -1.44269504f);
  } else if (act == Act::kGelu) {
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = gelu_erf(z[i]);
  } else if (act == Act::kGeluTanh) {
    // 2 u log2(e) = z (2.302208 + 0.1029432 z^2)
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = z[i] * inv_1_exp2(z[i] * __builtin_fmaf(z[i] * z[i], -0.10294324f, -2.3022082f));
  }
  return z;
}

// Four values as they are stored.
__device__ __forceinline__ f32x4 as_f32x4(f32x4 v) { return v; }
__device__ __forceinline__ f32x4 as_f32x4(uint2 u) {
  return f32x4{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
               __uint_as_float(u.y & 0xffff0000u)};
}
__device__ __forceinline__ f32x4 load4(const void* p, int64_t i, bool f32) {
  if (f32) return *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
  return as_f32x4(*reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i));
}

// Bias of columns col .. col + 3 (zeros without one).
__device__ __forceinline__ f32x4 epilogue_bias(const EpilogueArgs& e, int col) {
  return e.bias != nullptr ? load4(e.bias, col, e.bias_f32) : f32x4{0.f, 0.f, 0.f, 0.f};
}

// ---------------------------------------------------------------------------
// Products to fp32's own precision, for fp32 C.  The FP8 matrix instructions line up the
// products of eight neighbouring K to the largest of them and drop what is below 2^-16 of
// it or so: a sum of random operands is off by 1.5e-5 of its size, whatever K is (both
// v_mfma_f32_16x16x128_f8f6f4 and v_mfma_f32_16x16x32_fp8_fp8; the sums themselves are fp32).  bf16
// C does not see that; fp32 C would lose eight bits.  There the operands are widened to bf16,
// which holds every e4m3 value, and multiplied by v_mfma_f32_16x16x32_bf16 (1e-7 off), at half the
// matrix rate.  MX: the conversion multiplies by the block's power of two (exact between 2^-133
// and 2^128), so that the instruction needs no scales.
// ---------------------------------------------------------------------------
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

// 2^(byte - 127) of byte I of a word of e8m0 exponents.  255, e8m0's NaN, becomes an infinite scale, of which the
// conversion reads the exponent field: it gives NaN for every element, zeros too, as the scaled MFMA does.
template <int I>
__device__ __forceinline__ float e8m0_scale(int word) {
  const uint32_t e = (static_cast<uint32_t>(word) >> (8 * I)) & 0xffu;
  return __uint_as_float(e == 0 ? 0x00400000u : e << 23);
}

// Eight e4m3 values (w0's bytes, then w1's) times scale.
__device__ __forceinline__ bf16x8_t widen8(int w0, int w1, float scale) {
  union {
    bf16x2_t p[4];
    bf16x8_t v;
  } u;
  u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false);
  u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true);
  u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false);
  u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true);
  return u.v;
}

// A lane's 32 K bytes of an operand row, times scale: bytes 8s .. 8s + 7 in v[s].
struct WideFrag {
  bf16x8_t v[4];
};
__device__ __forceinline__ WideFrag widen(const i32x8& f, float scale) {
  WideFrag w;
#pragma unroll
  for (int s = 0; s < 4; ++s) w.v[s] = widen8(f[2 * s], f[2 * s + 1], scale);
  return w;
}

}  // namespace hkmoe
