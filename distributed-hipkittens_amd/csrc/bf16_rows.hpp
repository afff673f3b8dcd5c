// bf16 products of few columns: the router's logits and the low-rank adapters.
//
//   logits[t, e] = sum_h x[t, h] w[e, h]                                (router)
//   out[t] = y[t] + c_l (x[t] A_l^T) B_l^T,  l = ids[t]                 (adapters)
//
// Both stream x once past a weight that the caches hold, so both are bound by HBM
// (or, for a few rows, by the latency of two launches).  The matrix instruction is
// v_mfma_f32_16x16x32_bf16: products of two bf16 values are exact in fp32 and sums
// are kept in fp32.  Lane l supplies row l % 16 of either operand and the 8 K values
// from 8 (l / 16) on, one 16-byte load straight from a row-major matrix; lane l of
// the result holds rows 4 (l / 16) + 0..3, column l % 16.
#pragma once

#include "common.hpp"

namespace hkmoe {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma_bf16_16x16x32(const bf16x8& a, const bf16x8& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ bf16x8 zero_bf16x8() { return __builtin_bit_cast(bf16x8, i32x4{0, 0, 0, 0}); }

constexpr int kRowsWaves = 4;   // waves per workgroup, one K step each in turn
constexpr int kRowsBlock = 64;  // rows per workgroup (4 MFMA row tiles)
constexpr int kRowsStep = 64;   // K per step: whole 128-byte lines

// acc[mt][nt] += rows of x (MT tiles of 16; xr: this lane's row in each, null: zeros)
// times rows of w (wr, likewise), over K steps step0, step0 + kRowsWaves, ... < steps.
template <int MT, int NT>
__device__ __forceinline__ void rows_product(const uint16_t* const (&xr)[MT], const uint16_t* const (&wr)[NT], int K,
                                             int step0, int steps, f32x4 (&acc)[MT][NT]) {
  const int k_lane = 8 * (lane_id() >> 4);
  for (int st = step0; st < steps; st += kRowsWaves) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = st * kRowsStep + 32 * h + k_lane;
      bf16x8 a[MT], b[NT];
#pragma unroll
      for (int i = 0; i < MT; ++i)
        a[i] = xr[i] != nullptr && k < K ? *reinterpret_cast<const bf16x8*>(xr[i] + k) : zero_bf16x8();
#pragma unroll
      for (int i = 0; i < NT; ++i)
        b[i] = wr[i] != nullptr && k < K ? *reinterpret_cast<const bf16x8*>(wr[i] + k) : zero_bf16x8();
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = mfma_bf16_16x16x32(a[i], b[j], acc[i][j]);
    }
  }
}

// Sums the waves' tiles in wave order and hands (row, column, value) of the
// [16 MT, 16 NT] result to `put`.  red: kRowsWaves * MT * NT * 256 floats of LDS.
template <int MT, int NT, typename Put>
__device__ __forceinline__ void rows_reduce(const f32x4 (&acc)[MT][NT], float* red, Put put) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int kTile = MT * NT * 256;
  __syncthreads();  // red is free: the last user's reads are done
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        red[wave * kTile + ((i * 16 + 4 * (lane >> 4) + r) * NT + j) * 16 + (lane & 15)] = acc[i][j][r];
  __syncthreads();
  for (int e = threadIdx.x; e < kTile; e += kRowsWaves * 64) {
    float v = red[e];
#pragma unroll
    for (int w = 1; w < kRowsWaves; ++w) v += red[w * kTile + e];
    put(e / (16 * NT), e % (16 * NT), v);
  }
}

// ---------------------------------------------------------------------------
// router
// ---------------------------------------------------------------------------
struct RouterParams {
  const uint16_t* x;  // [T, H]
  const uint16_t* w;  // [E, H]
  float* logits;      // [T, E]
  int64_t rows;
  int32_t experts, hidden;
};

template <int MT, int NT>
__global__ __launch_bounds__(kRowsWaves * 64) void router_kernel(RouterParams p) {
  __shared__ float red[kRowsWaves * MT * NT * 256];
  const int64_t row0 = blockIdx.x * static_cast<int64_t>(16 * MT);
  const int col0 = blockIdx.y * 16 * NT;
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  const uint16_t* xr[MT];
  const uint16_t* wr[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t t = row0 + 16 * i + (lane & 15);
    xr[i] = t < p.rows ? p.x + t * p.hidden : nullptr;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int e = col0 + 16 * j + (lane & 15);
    wr[j] = e < p.experts ? p.w + static_cast<int64_t>(e) * p.hidden : nullptr;
  }
  f32x4 acc[MT][NT] = {};
  rows_product<MT, NT>(xr, wr, p.hidden, wave, (p.hidden + kRowsStep - 1) / kRowsStep, acc);
  rows_reduce<MT, NT>(acc, red, [&](int r, int c, float v) {
    if (row0 + r < p.rows && col0 + c < p.experts) p.logits[(row0 + r) * p.experts + col0 + c] = v;
  });
}

// ---------------------------------------------------------------------------
// adapters
//
// Rows come in blocks of kRowsBlock in their own order, and a workgroup takes the
// rows of one adapter of one block: a segment of a prefill fills whole blocks, and
// the requests of a decode batch each find their workgroup, with no sorted order
// to build first.  Two launches: the narrow product v = x A_l^T (its K split over
// `splits` workgroups, each writing its own fp32 partial sums), then y + c_l v B_l^T.
// ---------------------------------------------------------------------------
struct LoraParams {
  const void* y;
  void* out;
  int64_t y_stride, out_stride;  // elements between rows
  const uint16_t* x;
  int64_t x_stride;
  const uint16_t* a;     // [L, R, H]
  const uint16_t* b;     // [L, N, R]
  const int32_t* ids;    // [T]; outside [0, L): no adapter
  const float* scaling;  // [L], may be null
  float* v;              // [splits][T][R]
  int64_t rows;
  int32_t adapters, hidden, n, rank, splits, cols_per_wg;
};

constexpr int kLoraRankTiles = 4;  // ranks per pass of the narrow product, in 16s
constexpr int kLoraMaxRank = 256;

// The j-th distinct adapter among the block's rows, in order of first appearance
// (none: -2), and a mask of its rows.  Every wave finds the same.
struct LoraGroup {
  int id;
  uint64_t rows;
};
__device__ __forceinline__ LoraGroup lora_group(int id, uint64_t live, int j) {
  LoraGroup g{-2, 0};
  while (live != 0) {
    const int first = __builtin_ctzll(live);
    g.id = __builtin_amdgcn_readlane(id, first);
    g.rows = __ballot(id == g.id) & live;
    if (j-- == 0) return g;
    live &= ~g.rows;
  }
  return LoraGroup{-2, 0};
}

// Row (0..63) of the k-th set bit of m, -1 past the last.
__device__ __forceinline__ int nth_row(uint64_t m, int k) {
  // lane l's rank among the set bits, turned round by a permute over the wave
  const int lane = lane_id();
  const int rank = __builtin_popcountll(m & ((1ull << lane) - 1));
  const bool set = (m >> lane) & 1;
  const int at = __builtin_amdgcn_ds_permute(4 * (set ? rank : 63), set ? lane : -1);
  // lane 63 receives -1 from unset lanes unless all 64 bits are set
  const int n = __builtin_popcountll(m);
  const int got = __builtin_amdgcn_ds_bpermute(4 * (k & 63), at);
  return k < n ? got : -1;
}

// This lane's adapter of row block `blk`: -1 for rows without one, -2 past the end.
__device__ __forceinline__ int lora_id(const LoraParams& p, int64_t blk) {
  const int64_t t = blk * kRowsBlock + lane_id();
  int id = -2;
  if (t < p.rows) {
    id = p.ids[t];
    if (id < 0 || id >= p.adapters) id = -1;
  }
  return id;
}

template <int MT, int NT>
__device__ __forceinline__ void lora_shrink_tile(const LoraParams& p, int64_t t0, const LoraGroup& g, int r0, int split,
                                                 float* red) {
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  const uint16_t* xr[MT];
  const uint16_t* wr[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int row = nth_row(g.rows, 16 * i + (lane & 15));
    xr[i] = row >= 0 ? p.x + (t0 + row) * p.x_stride : nullptr;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int r = r0 + 16 * j + (lane & 15);
    wr[j] = r < p.rank ? p.a + (static_cast<int64_t>(g.id) * p.rank + r) * p.hidden : nullptr;
  }
  // this workgroup's share of the K steps
  const int steps = (p.hidden + kRowsStep - 1) / kRowsStep;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * split / p.splits);
  const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / p.splits);
  f32x4 acc[MT][NT] = {};
  rows_product<MT, NT>(xr, wr, p.hidden, s0 + wave, s1, acc);
  float* v = p.v + static_cast<int64_t>(split) * p.rows * p.rank;
  rows_reduce<MT, NT>(acc, red, [&](int i, int c, float val) {
    const int row = nth_row(g.rows, i);
    if (row >= 0 && r0 + c < p.rank) v[(t0 + row) * p.rank + r0 + c] = val;
  });
}

// grid: (row blocks, adapters of a block taken at a time, splits)
__global__ __launch_bounds__(kRowsWaves * 64) void lora_shrink_kernel(LoraParams p) {
  __shared__ float red[kRowsWaves * 4 * kLoraRankTiles * 256];
  const int64_t blk = blockIdx.x;
  const int id = lora_id(p, blk);
  const uint64_t live = __ballot(id >= 0);
  for (int j = blockIdx.y;; j += gridDim.y) {
    const LoraGroup g = lora_group(id, live, j);
    if (g.id < 0) return;
    const int n = __builtin_popcountll(g.rows);
    for (int r0 = 0; r0 < p.rank; r0 += 16 * kLoraRankTiles) {
      if (n > 16)
        lora_shrink_tile<4, kLoraRankTiles>(p, blk * kRowsBlock, g, r0, blockIdx.z, red);
      else
        lora_shrink_tile<1, kLoraRankTiles>(p, blk * kRowsBlock, g, r0, blockIdx.z, red);
    }
  }
}

// The narrow product's terms in bf16: v = t0 + t1 (+ t2), each the rounding of what
// the terms before it leave, 2^-17 (2^-25) of |v| at most: a single bf16 term would
// be off by 2^-9, more than an fp32 output may lose and as much as a bf16 one rounds.
// B is bf16 already and every product is exact, so two terms give a bf16 output,
// three an fp32 one, the result of an fp32 v.  An infinite or NaN v keeps its value
// in t0 and leaves 0 in the others.
template <int TERMS>
__device__ __forceinline__ void split_bf16(float v, uint16_t (&t)[TERMS]) {
#pragma unroll
  for (int i = 0; i < TERMS; ++i) {
    t[i] = static_cast<uint16_t>(bf16_rne_bits(v));
    const float back = bf16_bits_to_f32(t[i]);
    v = __builtin_isfinite(back) ? v - back : 0.0f;
  }
}

// grid: (row blocks, adapters of a block taken at a time, column parts).  Group 0..
// are the adapters as above; the rows without one are a group of their own, copied.
// Each wave takes 64 columns at a time.  The operands are swapped (B rows first), and
// result row 4g + i of column tile jt is column 16g + 4jt + i: a lane then holds 16
// adjacent columns of one row.
template <bool F32, int TERMS>
__global__ __launch_bounds__(kRowsWaves * 64) void lora_expand_kernel(LoraParams p) {
  constexpr int kPad = 8;  // row pitch off a multiple of the banks' width
  __shared__ __align__(16) uint16_t vt[TERMS][kRowsBlock][64 + kPad];
  const int64_t blk = blockIdx.x, t0 = blk * kRowsBlock;
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  const int id = lora_id(p, blk);
  const bool copy = p.y != p.out;
  const uint64_t live = __ballot(copy ? id >= -1 : id >= 0);
  const int c_begin = blockIdx.z * p.cols_per_wg, c_end = min(c_begin + p.cols_per_wg, p.n);
  for (int j = blockIdx.y;; j += gridDim.y) {
    const LoraGroup g = lora_group(id, live, j);
    if (g.id == -2) return;
    const int n = __builtin_popcountll(g.rows);
    const int m_tiles = (n + 15) / 16;
    const float c = g.id >= 0 && p.scaling != nullptr ? p.scaling[g.id] : 1.0f;
    for (int mt = 0; mt < m_tiles; ++mt) {
      const int row = nth_row(g.rows, 16 * mt + (lane & 15));
      const int64_t t = t0 + row;
      for (int col0 = c_begin; col0 < c_end; col0 += kRowsWaves * 64) {
        const int n_wave = col0 + 64 * wave;
        const int n_lane = n_wave + 16 * (lane >> 4);
        f32x4 acc[4];
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) {
          acc[jt] = f32x4{0.f, 0.f, 0.f, 0.f};
          if (row >= 0 && n_lane + 4 * jt < c_end) {
            const int64_t at = t * p.y_stride + n_lane + 4 * jt;
            if constexpr (F32) {
              acc[jt] = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p.y) + at);
            } else {
              const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.y) + at);
              acc[jt] = f32x4{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u),
                              __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u)};
            }
          }
        }
        if (g.id >= 0) {
          for (int r0 = 0; r0 < p.rank; r0 += 64) {
            __syncthreads();
            // 16 rows x 64 ranks of v: the splits' sums, scaled, as bf16 terms
            for (int e = threadIdx.x; e < 16 * 64; e += kRowsWaves * 64) {
              const int i = e >> 6, r = r0 + (e & 63);
              const int vr = nth_row(g.rows, 16 * mt + i);
              float v = 0.0f;
              if (vr >= 0 && r < p.rank) {
                const float* src = p.v + (t0 + vr) * p.rank + r;
                for (int s = 0; s < p.splits; ++s) v += src[static_cast<int64_t>(s) * p.rows * p.rank];
                v *= c;
              }
              uint16_t t16[TERMS];
              split_bf16<TERMS>(v, t16);
#pragma unroll
              for (int q = 0; q < TERMS; ++q) vt[q][i][e & 63] = t16[q];
            }
            __syncthreads();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int k = 32 * h + 8 * (lane >> 4);
              if (r0 + 32 * h >= p.rank) break;
              bf16x8 f[TERMS];
#pragma unroll
              for (int q = 0; q < TERMS; ++q) f[q] = *reinterpret_cast<const bf16x8*>(&vt[q][lane & 15][k]);
#pragma unroll
              for (int jt = 0; jt < 4; ++jt) {
                const int m = lane & 15;
                const int col = n_wave + 16 * (m >> 2) + 4 * jt + (m & 3);
                bf16x8 bf = zero_bf16x8();
                if (col < c_end && r0 + k < p.rank)
                  bf = *reinterpret_cast<const bf16x8*>(p.b + (static_cast<int64_t>(g.id) * p.n + col) * p.rank + r0 + k);
#pragma unroll
                for (int q = TERMS - 1; q >= 0; --q) acc[jt] = mfma_bf16_16x16x32(bf, f[q], acc[jt]);
              }
            }
          }
        }
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) {
          if (row >= 0 && n_lane + 4 * jt < c_end) {
            const int64_t at = t * p.out_stride + n_lane + 4 * jt;
            if constexpr (F32)
              *reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + at) = acc[jt];
            else
              *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) =
                  uint2{pack_bf16x2(acc[jt][0], acc[jt][1]), pack_bf16x2(acc[jt][2], acc[jt][3])};
          }
        }
      }
    }
  }
}

}  // namespace hkmoe
