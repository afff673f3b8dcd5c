// Residual addition, root-mean-square norm and e4m3 quantisation in one pass.
//
//   r = rnd(x + residual)                (kept in x's type: the new residual stream)
//   m = mean_j r_j^2,  rstd = fl32(1 / sqrt(m + eps)), at most the largest fp32 value
//   n_j = fl32(fl32(r_j rstd) w_j)       (q, and rnd(n) as bf16 where asked for)
//
// and n quantised as quant_group_kernel, quant_mx_kernel and quant_tensor_kernel
// would (same scales, same bytes).  The norm reads the rounded r, so that a
// caller which keeps only the stream sees the same norm.  The sum of squares and
// rstd are taken in 64 bits: the sum is then exact to far below an fp32 rounding
// step, so rstd, every n and with them every byte are those of the formula,
// whatever the order of the sum (an fp32 sum in another order moves one e4m3 byte
// in ~10^5).  A row costs one 64-bit FMA per value, which HBM hides.
//
// Bound by HBM: per value it reads x and the residual and writes the residual, one
// byte and, where asked for, the bf16 norm.  One workgroup per row, the row in
// registers between the sum and the quantisation (8 values a chunk, 16-byte
// loads), so each value is read once.  8192x7168 bf16 with a residual, groups and the bf16
// norm: 118 us, 4.5 TB/s (a copy of 4 GiB: 4.7); 139 at first after a pause of a second, where a
// copy keeps its time.
#pragma once

#include "common.hpp"
#include "moe_kernels.hpp"

namespace hkmoe {

enum class NormScale { kGroup, kMx, kStatic, kAmax };

struct NormParams {
  const void* x;
  const void* residual;  // may be null
  const void* weight;    // [cols]
  void* residual_out;    // null without a residual
  uint16_t* norm_out;    // bf16, may be null
  uint8_t* q;
  void* s;            // group: fp32, mx: e8m0; static: unused; amax: fp32 [1], the second launch's
  const float* scale;  // static
  float* rstd;         // amax: [rows]
  float* amax;         // amax: one per workgroup
  int64_t rows;
  int32_t cols;
  int32_t w_f32;
  double eps;
};

constexpr int kNormChunk = 8;          // values per thread and step
constexpr int kNormMaxThreads = 1024;
constexpr int kNormAmaxGroups = 1024;  // workgroups of the per-tensor form's first launch

struct F8v {
  float v[8];
};

__device__ __forceinline__ F8v unpack_bf16x8(uint4 u) {
  F8v f;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f.v[2 * i] = __uint_as_float(w[i] << 16);
    f.v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  return f;
}
__device__ __forceinline__ uint4 pack_bf16x8(const F8v& f) {
  return uint4{pack_bf16x2(f.v[0], f.v[1]), pack_bf16x2(f.v[2], f.v[3]), pack_bf16x2(f.v[4], f.v[5]),
               pack_bf16x2(f.v[6], f.v[7])};
}

template <bool F32>
__device__ __forceinline__ F8v load8(const void* p, int64_t i) {
  if constexpr (F32) {
    const f32x4* s = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
    const f32x4 a = s[0], b = s[1];
    return F8v{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
  } else {
    return unpack_bf16x8(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i));
  }
}
template <bool F32>
__device__ __forceinline__ void store8(void* p, int64_t i, const F8v& f) {
  if constexpr (F32) {
    f32x4* d = reinterpret_cast<f32x4*>(static_cast<float*>(p) + i);
    d[0] = f32x4{f.v[0], f.v[1], f.v[2], f.v[3]};
    d[1] = f32x4{f.v[4], f.v[5], f.v[6], f.v[7]};
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = pack_bf16x8(f);
  }
}

__device__ __forceinline__ f32x4 lo4(const F8v& f) { return f32x4{f.v[0], f.v[1], f.v[2], f.v[3]}; }
__device__ __forceinline__ f32x4 hi4(const F8v& f) { return f32x4{f.v[4], f.v[5], f.v[6], f.v[7]}; }
__device__ __forceinline__ float max_abs8(const F8v& f) { return fmaxf(max_abs4(lo4(f)), max_abs4(hi4(f))); }

// The sum over a workgroup, the same on every thread.  `red` holds one double per
// wave and is free for reuse after the caller's next barrier.
__device__ __forceinline__ double group_sum(double v, double* red) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, kWave);
  const int waves = blockDim.x / kWave;
  if (waves == 1) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
  for (int w = 0; w < waves; ++w) v += red[w];
  return v;
}

// Eight values n of columns j.. quantised with one scale: 8 bytes.  |n| may exceed
// 448 sc only where the caller gave the scale: there the values are cut to 512 sc
// first, which saturates to the same bytes and keeps quot_e4m3 inside its range.
template <bool CUT>
__device__ __forceinline__ uint2 quant8(F8v n, float sc, const QuotScale& qs) {
  if constexpr (CUT) {
    const float top = 512.0f * sc;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (fabsf(n.v[i]) > top) n.v[i] = __builtin_copysignf(top, n.v[i]);
  }
  return uint2{quant4(lo4(n), sc, qs), quant4(hi4(n), sc, qs)};
}

// One row per workgroup (kAmax: rows blockIdx.x, + gridDim.x, ...), CH chunks of 8
// values per thread.  cols % 128 == 0 for groups, % 32 for MX, else % 8, so the 16 (4) lanes
// that share a scale are active together.
template <bool F32, NormScale SC, int CH>
__global__ __launch_bounds__(kNormMaxThreads) void rms_norm_quant_kernel(NormParams p) {
  __shared__ double red[2][kNormMaxThreads / kWave];
  __shared__ float redm[kNormMaxThreads / kWave];
  const int cols = p.cols;
  float amax = 0.0f;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    const int64_t base = row * cols;
    F8v r[CH];
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int j = (c * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * kNormChunk;
      if (j < cols) r[c] = load8<F32>(p.x, base + j);
    }
    if (p.residual != nullptr) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int j = (c * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * kNormChunk;
        if (j < cols) {
          const F8v o = load8<F32>(p.residual, base + j);
#pragma unroll
          for (int i = 0; i < 8; ++i) r[c].v[i] += o.v[i];
          if constexpr (F32) {
            store8<true>(p.residual_out, base + j, r[c]);
          } else {
            const uint4 u = pack_bf16x8(r[c]);
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.residual_out) + base + j) = u;
            r[c] = unpack_bf16x8(u);
          }
        }
      }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int j = (c * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * kNormChunk;
      if (j < cols) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = __builtin_fma(static_cast<double>(r[c].v[i]), static_cast<double>(r[c].v[i]), sum);
      }
    }
    sum = group_sum(sum, red[turn]);
    // past fp32 (rows of zeros with eps below 2^-256) the largest one, so that zeros stay zeros
    const float inv = static_cast<float>(1.0 / sqrt(sum / static_cast<double>(cols) + p.eps)), most = 0x1.fffffep127f;
    const float rstd = inv > most ? most : inv;
    if constexpr (SC == NormScale::kAmax) {
      if (threadIdx.x == 0) p.rstd[row] = rstd;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int j = (c * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * kNormChunk;
      const bool live = j < cols;
      F8v n = {};
      if (live) {
        const F8v w = p.w_f32 ? load8<true>(p.weight, j) : load8<false>(p.weight, j);
#pragma unroll
        for (int i = 0; i < 8; ++i) n.v[i] = r[c].v[i] * rstd * w.v[i];
        if (p.norm_out != nullptr) store8<false>(p.norm_out, base + j, n);
      }
      const float m = max_abs8(n);
      if constexpr (SC == NormScale::kGroup) {
        const float sc = scale_from_amax(row16_max(m));
        const QuotScale qs = quot_scale(sc);
        if (live) {
          *reinterpret_cast<uint2*>(p.q + base + j) = quant8<false>(n, sc, qs);
          if ((threadIdx.x & 15) == 0) static_cast<float*>(p.s)[(base + j) / kGroup] = sc;
        }
      } else if constexpr (SC == NormScale::kMx) {
        float b = fmaxf(m, __shfl_xor(m, 1, kWave));
        b = fmaxf(b, __shfl_xor(b, 2, kWave));
        const uint32_t e = min((__float_as_uint(b) >> 23) & 0xffu, 254u);
        const int sh = 127 - static_cast<int>(e);
        if (live) {
          float t[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) t[i] = __builtin_amdgcn_ldexpf(n.v[i], sh);
          *reinterpret_cast<uint2*>(p.q + base + j) =
              uint2{pack_e4m3x4(t[0], t[1], t[2], t[3]), pack_e4m3x4(t[4], t[5], t[6], t[7])};
          if ((threadIdx.x & 3) == 0) static_cast<uint8_t*>(p.s)[(base + j) / 32] = static_cast<uint8_t>(e);
        }
      } else if constexpr (SC == NormScale::kStatic) {
        // 448 sc may be past fp32: there n and sc are taken 2^-24 as large (what that loses of n is far
        // below the smallest e4m3 value), so that an infinite n is cut as any other
        const float by = *p.scale > 0x1p100f ? 0x1p-24f : 1.0f, sc = *p.scale * by;
#pragma unroll
        for (int i = 0; i < 8; ++i) n.v[i] *= by;
        if (live) *reinterpret_cast<uint2*>(p.q + base + j) = quant8<true>(n, sc, quot_scale(sc));
      } else {
        amax = fmaxf(amax, m);
      }
    }
  }
  if constexpr (SC == NormScale::kAmax) {
    amax = wave_max(amax);
    if ((threadIdx.x & 63) == 0) redm[threadIdx.x >> 6] = amax;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (unsigned w = 1; w < blockDim.x / kWave; ++w) amax = fmaxf(amax, redm[w]);
      p.amax[blockIdx.x] = amax;
    }
  }
}

// Second launch of the per-tensor form: n again from the stream (r: the residual's
// output, or x without one) and rstd, the scale from the first launch's maxima.
template <bool F32>
__global__ __launch_bounds__(256) void norm_quant_tensor_kernel(const void* __restrict__ r, const void* __restrict__ weight,
                                                                int w_f32, const float* __restrict__ rstd,
                                                                const float* __restrict__ amax, int amax_count,
                                                                int64_t rows, int cols, uint8_t* __restrict__ q,
                                                                float* __restrict__ s) {
  __shared__ float red[4];
  float m = 0.0f;
  for (int i = threadIdx.x; i < amax_count; i += 256) m = fmaxf(m, amax[i]);
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  const float sc = scale_from_amax(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
  const QuotScale qs = quot_scale(sc);
  if (blockIdx.x == 0 && threadIdx.x == 0) s[0] = sc;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float rs = rstd[row];
    for (int j = threadIdx.x * kNormChunk; j < cols; j += 256 * kNormChunk) {
      const F8v v = load8<F32>(r, row * cols + j);
      const F8v w = w_f32 ? load8<true>(weight, j) : load8<false>(weight, j);
      F8v n;
#pragma unroll
      for (int i = 0; i < 8; ++i) n.v[i] = v.v[i] * rs * w.v[i];
      *reinterpret_cast<uint2*>(q + row * cols + j) = quant8<false>(n, sc, qs);
    }
  }
}

}  // namespace hkmoe
