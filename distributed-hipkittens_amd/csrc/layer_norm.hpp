// Layer norm with the residual's addition, and its gradient.
//
//   r = rnd(x + residual)                     (kept in x's type: the new residual stream)
//   m = mean_j r_j,  v = mean_j (r_j - m)^2,  rstd = fl32(1 / sqrt(v + eps))
//   n_j = fl32((r_j - m) rstd),               y_j = rnd(n_j w_j + b_j)
//
//   g_j = dy_j w_j,  dx_j = rnd(rstd (g_j - mean g - n_j mean(g n)) + dr_j)
//   dw_j = sum_rows dy_j n_j,  db_j = sum_rows dy_j
//
// Forward: one pass, the row in registers between its sums and its output.  The two
// sums are taken in 64 bits of r_j - r_0 (r_0 near the row's values where those are
// far from zero), so v keeps its bits whatever the mean is; m is kept as two fp32
// terms, because one would cost r - m as many bits as |m| is larger than its spread.
// Backward: the row's two sums in fp32, and in the same pass every thread's own
// columns of dw and db over the workgroup's rows, in registers; one partial per
// workgroup goes to the workspace and a second launch adds them in order, in 64 bits.  While rows
// are few, a launch costs more than their bytes: there dw and db, which need no sums over a row
// (n comes from the forward pass's stats), get workgroups of their own beside the rows'.
// Nothing is added atomically: the same call gives the same bits.
#pragma once

#include "norm_quant.hpp"

namespace hkmoe {

constexpr int kLnParts = 256;                                       // workgroups of the gradient, see layer_norm_parts
constexpr int kLnRowThreads = 256;                                  // of a workgroup that has several rows
constexpr int kLnMaxCols = 2 * kNormMaxThreads * kNormChunk;        // 16384
// Threads of a workgroup, at most.  Past 8192 columns a thread of 1024 has two chunks of a row (four each on 512
// threads, with half the loads in flight, 2048x8200 bf16: 33 us forward and 50 backward against 26 and 37).
constexpr int ln_threads(int lanes) { return lanes != 0 ? kLnRowThreads : kNormMaxThreads; }

struct LayerNormParams {
  const void* x;
  const void* residual;  // may be null
  const void* weight;    // [cols]
  const void* bias;      // [cols], may be null
  void* y;
  void* residual_out;  // null without a residual
  f32x4* stats;        // [rows]: m's two terms, rstd, 0
  int64_t rows;
  int32_t cols;
  int32_t w_f32;
  double eps;
};

struct LayerNormGradParams {
  const void* dy;
  const void* r;       // the stream that the norm read
  const void* weight;  // [cols]
  const void* dr;      // may be null
  const f32x4* stats;
  void* dx;
  float* part;  // [gridDim.x][2][cols] (not COLS)
  void* dw;
  void* db;  // may be null
  int64_t rows;
  int32_t cols;
  int32_t w_f32;
  int32_t col_groups;  // COLS: workgroups of 64 columns, in front of the rows'
};

// Threads of a row: LANES lanes of a wave (one wave's rows need no barrier), or with
// LANES 0 the whole workgroup.  A workgroup's rows: ln_rows, row slot ln_slot.
template <int LANES>
__device__ __forceinline__ int ln_rows() { return LANES == 0 ? 1 : kLnRowThreads / LANES; }
template <int LANES>
__device__ __forceinline__ int ln_slot() { return LANES == 0 ? 0 : static_cast<int>(threadIdx.x) / LANES; }
template <int LANES>
__device__ __forceinline__ int ln_col(int c) {
  const int w = LANES == 0 ? static_cast<int>(blockDim.x) : LANES, l = LANES == 0 ? static_cast<int>(threadIdx.x) : static_cast<int>(threadIdx.x) % LANES;
  return (c * w + l) * kNormChunk;
}

// Sums of the 16 lanes of a DPP row, the same on each (quad pairs, quad swap, half-row and row
// mirrors), without the LDS crossbar of a shuffle.
template <int CTRL, typename T>
__device__ __forceinline__ T dpp_swap(T v) {
  if constexpr (sizeof(T) == 8) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = static_cast<uint32_t>(u), hi = static_cast<uint32_t>(u >> 32);
    const uint32_t l = __builtin_amdgcn_update_dpp(lo, lo, CTRL, 0xf, 0xf, false), h = __builtin_amdgcn_update_dpp(hi, hi, CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(T, (static_cast<uint64_t>(h) << 32) | l);
  } else {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(u, u, CTRL, 0xf, 0xf, false));
  }
}
template <typename T>
__device__ __forceinline__ T dpp_row_sum(T v) {
  v += dpp_swap<0xB1>(v);
  v += dpp_swap<0x4E>(v);
  v += dpp_swap<0x141>(v);
  return v + dpp_swap<0x140>(v);
}
template <typename T>
__device__ __forceinline__ T lane_value(T v, int lane) {
  if constexpr (sizeof(T) == 8) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(u), lane), hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(u >> 32), lane);
    return __builtin_bit_cast(T, (static_cast<uint64_t>(hi) << 32) | lo);
  } else {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(uint32_t, v), lane));
  }
}

// Two sums over a row's threads, the same on each of them.  `red` (LANES 0) holds two
// values per wave and is free again after the caller's next barrier.
template <int LANES, typename T>
__device__ __forceinline__ void row_sums(T& a, T& b, T (*red)[2]) {
  a = dpp_row_sum(a);
  b = dpp_row_sum(b);
  if constexpr (LANES == 32) {
    a += __shfl_xor(a, 16, kWave);
    b += __shfl_xor(b, 16, kWave);
  } else if constexpr (LANES != 16) {  // whole waves: the DPP rows' sums through scalar registers
    a = (lane_value(a, 0) + lane_value(a, 16)) + (lane_value(a, 32) + lane_value(a, 48));
    b = (lane_value(b, 0) + lane_value(b, 16)) + (lane_value(b, 32) + lane_value(b, 48));
  }
  if constexpr (LANES == 0) {
    const int waves = blockDim.x / kWave, l = threadIdx.x & 15;  // at most 16
    if ((threadIdx.x & 63) == 0) {
      red[threadIdx.x >> 6][0] = a;
      red[threadIdx.x >> 6][1] = b;
    }
    __syncthreads();
    a = l < waves ? red[l][0] : T(0);
    b = l < waves ? red[l][1] : T(0);
    a = dpp_row_sum(a);
    b = dpp_row_sum(b);
  }
}

// 1 / sqrt(v): the hardware's estimate (about 2^-24 off) and one Newton step, 2^-46.  v at least 2^-260,
// below which the caller's fp32 result is at its largest value anyway.
__device__ __forceinline__ double inv_sqrt(double v) {
  v = v < 0x1p-260 ? 0x1p-260 : v;  // a NaN stays
  const double y = __builtin_amdgcn_rsq(v);
  return y * __builtin_fma(-0.5 * v * y, y, 1.5);
}

// Eight values as they are stored, so that rows loaded ahead cost half the registers in bf16.
template <bool F32>
struct Raw8 {
  uint4 u;
  __device__ __forceinline__ void load(const void* p, int64_t i) { u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i); }
  __device__ __forceinline__ F8v get() const { return unpack_bf16x8(u); }
};
template <>
struct Raw8<true> {
  F8v u;
  __device__ __forceinline__ void load(const void* p, int64_t i) { u = load8<true>(p, i); }
  __device__ __forceinline__ F8v get() const { return u; }
};

// Rows blockIdx.x * rows per workgroup, + gridDim.x * that, ...; the next row's loads go out before
// the sums of this one are waited for.
template <bool F32, int CH, int LANES>
__global__ __launch_bounds__(ln_threads(LANES)) void layer_norm_kernel(LayerNormParams p) {
  __shared__ double red[2][LANES == 0 ? kNormMaxThreads / kWave : 1][2];
  const int cols = p.cols;
  const int64_t step = static_cast<int64_t>(gridDim.x) * ln_rows<LANES>();
  int64_t row = static_cast<int64_t>(blockIdx.x) * ln_rows<LANES>() + ln_slot<LANES>();
  const double inv_n = 1.0 / static_cast<double>(cols);
  Raw8<F32> x[CH], o[CH];
  float first = 0.0f;
  auto load = [&](int64_t at) __attribute__((always_inline)) {
    if (at < p.rows) {
      const int64_t base = at * cols;
      first = F32 ? static_cast<const float*>(p.x)[base] : bf16_bits_to_f32(static_cast<const uint16_t*>(p.x)[base]);
      if (p.residual != nullptr)
        first += F32 ? static_cast<const float*>(p.residual)[base]
                     : bf16_bits_to_f32(static_cast<const uint16_t*>(p.residual)[base]);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int j = ln_col<LANES>(c);
        if (j < cols) {
          x[c].load(p.x, base + j);
          if (p.residual != nullptr) o[c].load(p.residual, base + j);
        }
      }
    }
  };
  load(row);
  int turn = 0;
  // LANES 0: the whole workgroup has one row, so the barriers are met together
  for (; row < p.rows; row += step, turn ^= 1) {
    const int64_t base = row * cols;
    const float near = first;
    F8v r[CH];
    double s1 = 0.0, s2 = 0.0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (ln_col<LANES>(c) < cols) {
        r[c] = x[c].get();
        if (p.residual != nullptr) {
          const F8v a = o[c].get();
#pragma unroll
          for (int i = 0; i < 8; ++i) r[c].v[i] += a.v[i];
          if constexpr (!F32) r[c] = unpack_bf16x8(pack_bf16x8(r[c]));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const double d = static_cast<double>(r[c].v[i]) - static_cast<double>(near);
          s1 += d;
          s2 = __builtin_fma(d, d, s2);
        }
      }
    }
    load(row + step);
    // residual_out may be x or residual: every thread has read what it will overwrite, and `first`,
    // which all of them read, is overwritten after the barrier below (or by the same wave)
    row_sums<LANES>(s1, s2, red[turn]);
    if (p.residual != nullptr) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int j = ln_col<LANES>(c);
        if (j < cols) store8<F32>(p.residual_out, base + j, r[c]);
      }
    }
    const double d1 = s1 * inv_n, mean = d1 + static_cast<double>(near), var = s2 * inv_n - d1 * d1;
    const float mh = static_cast<float>(mean), ml = static_cast<float>(mean - static_cast<double>(mh));
    // past fp32 (constant rows with eps below 2^-256) the largest one, so that zeros stay zeros
    const float inv = static_cast<float>(inv_sqrt((var > 0.0 ? var : var * 0.0) + p.eps)), most = 0x1.fffffep127f;
    const float rstd = inv > most ? most : inv;
    if ((LANES == 0 ? threadIdx.x : threadIdx.x % LANES) == 0) p.stats[row] = f32x4{mh, ml, rstd, 0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int j = ln_col<LANES>(c);
      if (j < cols) {
        const F8v w = p.w_f32 ? load8<true>(p.weight, j) : load8<false>(p.weight, j);
        F8v b = {};
        if (p.bias != nullptr) b = p.w_f32 ? load8<true>(p.bias, j) : load8<false>(p.bias, j);
        F8v n;
#pragma unroll
        for (int i = 0; i < 8; ++i) n.v[i] = __builtin_fmaf(((r[c].v[i] - mh) - ml) * rstd, w.v[i], b.v[i]);
        store8<F32>(p.y, base + j, n);
      }
    }
  }
}

// Value j of dw or db (which may be null) in its type.
__device__ __forceinline__ void put_sum(void* to, int j, float v, int w_f32) {
  if (to == nullptr) return;
  if (w_f32)
    static_cast<float*>(to)[j] = v;
  else
    static_cast<uint16_t*>(to)[j] = static_cast<uint16_t>(bf16_rne_bits(v));
}

// dw and db of columns 64 blockIdx.x .. + 63 over all rows: 8 lanes of 8 columns to a row, the lanes'
// sums and then the waves' added in order.
template <bool F32>
__device__ __forceinline__ void layer_norm_grad_cols(const LayerNormGradParams& p) {
  __shared__ float red[kNormMaxThreads / kWave][128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x / kWave;
  const int j = blockIdx.x * 64 + (lane & 7) * kNormChunk;
  F8v dw{}, db{};
  if (j < p.cols) {
#pragma unroll 4
    for (int64_t row = wave * 8 + (lane >> 3); row < p.rows; row += waves * 8) {
      const f32x4 st = p.stats[row];
      Raw8<F32> r, dy;
      r.load(p.r, row * p.cols + j);
      dy.load(p.dy, row * p.cols + j);
      const F8v x = r.get(), d = dy.get();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dw.v[i] = __builtin_fmaf(d.v[i], ((x.v[i] - st.x) - st.y) * st.z, dw.v[i]);
        db.v[i] += d.v[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int o = 8; o <= 32; o <<= 1) {
      dw.v[i] += __shfl_xor(dw.v[i], o, kWave);
      db.v[i] += __shfl_xor(db.v[i], o, kWave);
    }
  }
  if (lane < 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      red[wave][lane * 8 + i] = dw.v[i];
      red[wave][64 + lane * 8 + i] = db.v[i];
    }
  }
  __syncthreads();
  if (threadIdx.x < 128) {
    const int col = blockIdx.x * 64 + (threadIdx.x & 63);
    float s = 0.0f;
    for (int w = 0; w < waves; ++w) s += red[w][threadIdx.x];
    if (col < p.cols) put_sum(threadIdx.x < 64 ? p.dw : p.db, col, s, p.w_f32);
  }
}

// Rows blockIdx.x * rows per workgroup, + gridDim.x * that, ...; the next row is loaded
// before the sums of this one are waited for (kAhead).  COLS: dw and db in workgroups of their own.
template <bool F32, int CH, int LANES, bool COLS>
__global__ __launch_bounds__(ln_threads(LANES)) void layer_norm_grad_kernel(LayerNormGradParams p) {
  const int first = COLS ? p.col_groups : 0;
  if constexpr (COLS) {
    if (static_cast<int>(blockIdx.x) < first) return layer_norm_grad_cols<F32>(p);
  }
  __shared__ float red[2][LANES == 0 ? kNormMaxThreads / kWave : 1][2];
  // wide rows leave no registers for a row ahead, nor for keeping g and n, beside the sums of dw and db
  constexpr bool kAhead = LANES != 0 || CH == 1 || COLS;
  const int cols = p.cols;
  const int64_t step = static_cast<int64_t>(gridDim.x - first) * ln_rows<LANES>();
  int64_t row = static_cast<int64_t>(blockIdx.x - first) * ln_rows<LANES>() + ln_slot<LANES>();
  const float inv_n = 1.0f / static_cast<float>(cols);
  F8v dw[CH], db[CH];
  Raw8<F32> r[CH], dy[CH];
  f32x4 st{};
  auto load = [&](int64_t at) __attribute__((always_inline)) {
    if (at < p.rows) {
      st = p.stats[at];
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int j = ln_col<LANES>(c);
        if (j < cols) {
          r[c].load(p.r, at * cols + j);
          dy[c].load(p.dy, at * cols + j);
        }
      }
    }
  };
#pragma unroll
  for (int c = 0; c < CH; ++c) dw[c] = db[c] = F8v{};
  // g, n and the output gradient of a chunk
  auto terms = [&](int c, F8v& g, F8v& n, F8v& d) __attribute__((always_inline)) {
    const int j = ln_col<LANES>(c);
    const F8v w = p.w_f32 ? load8<true>(p.weight, j) : load8<false>(p.weight, j);
    const F8v x = r[c].get();
    d = dy[c].get();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      n.v[i] = ((x.v[i] - st.x) - st.y) * st.z;
      g.v[i] = d.v[i] * w.v[i];
    }
  };
  load(row);
  int turn = 0;
  // LANES 0: the whole workgroup has one row, so the barriers are met together
  for (; row < p.rows; row += step, turn ^= 1) {
    const int64_t base = row * cols;
    const float rstd = st.z;
    F8v g[CH], n[CH];
    Raw8<F32> dr[CH];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int j = ln_col<LANES>(c);
      if (j < cols) {
        if (kAhead && p.dr != nullptr) dr[c].load(p.dr, base + j);
        F8v d;
        terms(c, g[c], n[c], d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (!COLS) {
            dw[c].v[i] = __builtin_fmaf(d.v[i], n[c].v[i], dw[c].v[i]);
            db[c].v[i] += d.v[i];
          }
          s1 += g[c].v[i];
          s2 = __builtin_fmaf(g[c].v[i], n[c].v[i], s2);
        }
      }
    }
    if constexpr (kAhead) load(row + step);
    row_sums<LANES>(s1, s2, red[turn]);
    const float m1 = s1 * inv_n, m2 = s2 * inv_n;
    if constexpr (!kAhead) asm volatile("" : "+v"(st.x), "+v"(st.z));  // or the compiler keeps n after all
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int j = ln_col<LANES>(c);
      if (j < cols) {
        F8v d;
        if (!kAhead && p.dr != nullptr) dr[c].load(p.dr, base + j);
        if constexpr (!kAhead) terms(c, g[c], n[c], d);
        F8v add{};
        if (p.dr != nullptr) add = dr[c].get();
        F8v o;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          o.v[i] = __builtin_fmaf(__builtin_fmaf(-n[c].v[i], m2, g[c].v[i] - m1), rstd, add.v[i]);
        store8<F32>(p.dx, base + j, o);
      }
    }
    if constexpr (!kAhead) load(row + step);
  }
  if constexpr (COLS) return;
  float* part = p.part + static_cast<int64_t>(blockIdx.x) * 2 * cols;
  if constexpr (LANES == 0) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int j = ln_col<LANES>(c);
      if (j < cols) {
        store8<true>(part, j, dw[c]);
        store8<true>(part, cols + j, db[c]);
      }
    }
  } else {
    // the workgroup's row slots meet in LDS, 8 columns of a lane at a time
    __shared__ float meet[kLnRowThreads][9];
#pragma unroll
    for (int c = 0; c < 2 * CH; ++c) {
      const F8v& v = c < CH ? dw[c] : db[c - CH];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) meet[threadIdx.x][i] = v.v[i];
      __syncthreads();
      for (int u = threadIdx.x; u < LANES * 8; u += kLnRowThreads) {  // value u % 8 of lane u / 8
        const int l = u / 8, j = ((c % CH) * LANES + l) * kNormChunk + u % 8;
        float s = 0.0f;
        for (int q = 0; q < kLnRowThreads / LANES; ++q) s += meet[q * LANES + l][u % 8];
        if (j < cols) part[(c < CH ? 0 : cols) + j] = s;
      }
    }
  }
}

// The partials of `count` workgroups added in order, in 64 bits: 64 values per workgroup, each of
// its 16 waves a sixteenth of the partials (16 loads of a lane in flight: 256 partials in one round).
constexpr int kLnSumThreads = 1024;
__global__ __launch_bounds__(kLnSumThreads) void layer_norm_sum_kernel(const float* __restrict__ part, int count, int cols,
                                                                       void* dw, void* db, int w_f32) {
  constexpr int kWaves = kLnSumThreads / 64;
  __shared__ double red[kWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = blockIdx.x * 64 + lane;
  const int64_t width = 2 * static_cast<int64_t>(cols);
  double s = 0.0;
  if (i < width) {
    const int b0 = count * wave / kWaves, b1 = count * (wave + 1) / kWaves;
#pragma unroll 16
    for (int b = b0; b < b1; ++b) s += static_cast<double>(part[b * width + i]);
  }
  red[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || i >= width) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) s += red[w][lane];
  put_sum(i < cols ? dw : db, i < cols ? i : i - cols, static_cast<float>(s), w_f32);
}

}  // namespace hkmoe
