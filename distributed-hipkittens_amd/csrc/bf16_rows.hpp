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

#include "gemm_small.hpp"

namespace hkmoe {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma_bf16_16x16x32(const bf16x8& a, const bf16x8& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ bf16x8 zero_bf16x8() { return __builtin_bit_cast(bf16x8, i32x4{0, 0, 0, 0}); }

constexpr int kRowsBlock = 64;  // rows per workgroup at most (4 MFMA row tiles)
constexpr int kRowsStep = 64;   // K per step: whole 128-byte lines

// acc[mt][nt] += rows of x (MT tiles of 16; xr: this lane's row in each) times rows of
// w (wr, likewise), over K steps st, st + stride, ... < steps of 64.  Rows past the
// last may repeat a valid one: a result row depends on its own operand rows alone.
// The loads of up to DEPTH steps are issued before the first product, so that
// 2 DEPTH (MT + NT) of them are in flight per wave.
template <int MT, int NT, int DEPTH>
__device__ __forceinline__ void rows_product(const uint16_t* const (&xr)[MT], const uint16_t* const (&wr)[NT], int K,
                                             int st, int stride, int steps, f32x4 (&acc)[MT][NT]) {
  const int k_lane = 8 * (lane_id() >> 4);
  bf16x8 a[DEPTH][2][MT], b[DEPTH][2][NT];
  auto load = [&](int d, int k0) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = k0 + 32 * h + k_lane;
#pragma unroll
      for (int i = 0; i < MT; ++i) a[d][h][i] = *reinterpret_cast<const bf16x8*>(xr[i] + k);
#pragma unroll
      for (int i = 0; i < NT; ++i) b[d][h][i] = *reinterpret_cast<const bf16x8*>(wr[i] + k);
    }
  };
  auto mma = [&](int d) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = mfma_bf16_16x16x32(a[d][h][i], b[d][h][j], acc[i][j]);
  };
  const int full = min(steps, K / kRowsStep);  // steps without a ragged end
  for (; st + (DEPTH - 1) * stride < full; st += DEPTH * stride) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(d, (st + d * stride) * kRowsStep);
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) mma(d);
  }
  for (; st < full; st += stride) {
    load(0, st * kRowsStep);
    mma(0);
  }
  if (st < steps) {  // K's last step, K % 64 != 0
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = st * kRowsStep + 32 * h + k_lane;
#pragma unroll
      for (int i = 0; i < MT; ++i) a[0][h][i] = k < K ? *reinterpret_cast<const bf16x8*>(xr[i] + k) : zero_bf16x8();
#pragma unroll
      for (int i = 0; i < NT; ++i) b[0][h][i] = k < K ? *reinterpret_cast<const bf16x8*>(wr[i] + k) : zero_bf16x8();
    }
    mma(0);
  }
}

// Sums the waves' tiles in wave order and hands (row, column, value) of the
// [16 MT, 16 NT] result to `put`.  red: WAVES * MT * NT * 256 floats of LDS.
template <int MT, int NT, int WAVES, typename Put>
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
  for (int e = threadIdx.x; e < kTile; e += WAVES * 64) {
    float v = red[e];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += red[w * kTile + e];
    put(e / (16 * NT), e % (16 * NT), v);
  }
}

// ---------------------------------------------------------------------------
// Tiles of many rows: operands through LDS
//
// A load in operand order touches 16 rows of 64 bytes, and a CU gets a third of its
// rate from such loads (8192x7168 rows against 64 columns: 37 us straight into
// registers, of which 17 for the columns alone).  So the rows of both operands come in
// whole 128-byte lines by global->LDS DMA, K steps of 64 in a ring of STAGES, swizzled
// (chunk c of row r at slot c ^ swz(r)) so that the fragment reads spread over the banks.
// WM x WN waves, each with MT x NT tiles of 16x16 outputs.
// ---------------------------------------------------------------------------
template <int BM_, int BN_, int WM_, int WN_, int STAGES_>
struct Panel {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_;
  static constexpr int kWaves = WM * WN, MT = BM / 16 / WM, NT = BN / 16 / WN;
  static constexpr int kLoads = (BM + BN) / 8 / kWaves;  // DMA instructions per wave and step
  static constexpr int kStage = (BM + BN) * 2 * kRowsStep;
  static constexpr int kLds = STAGES * kStage;
  static_assert((BM + BN) % (8 * kWaves) == 0 && BM % (16 * WM) == 0 && BN % (16 * WN) == 0, "tile");
  static_assert(STAGES >= 2 && STAGES <= 4, "small_wait_stage covers at most 3 newer stages");
};

// acc += the tile over K steps s0 .. s1 - 1.  row_of(i): row i of the BM rows of x, then of
// the BN rows of w (16-byte aligned; rows past the last may repeat a valid one).  Every wave of the workgroup calls it; on return all
// are done with smem.
template <typename P, typename RowOf>
__device__ __forceinline__ void panel_product(uint8_t* smem, RowOf row_of, int K, int s0, int s1, f32x4 (&acc)[P::MT][P::NT]) {
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, lg = lane >> 4, wm = wave / P::WN, wn = wave % P::WN;
  const uint16_t* src[P::kLoads];
  int off[P::kLoads];  // K offset of this lane's chunk in a step
#pragma unroll
  for (int i = 0; i < P::kLoads; ++i) {
    const int r = 8 * (wave + P::kWaves * i) + (lane >> 3);
    off[i] = 8 * ((lane & 7) ^ swz(r));
    src[i] = row_of(r) + off[i];
  }
  const int n = s1 - s0;
  auto issue = [&](int i) __attribute__((always_inline)) {
    uint8_t* st = smem + (i % P::STAGES) * P::kStage;
    const int k0 = (s0 + i) * kRowsStep;
    const bool ragged = k0 + kRowsStep > K;
#pragma unroll
    for (int u = 0; u < P::kLoads; ++u) {
      const uint16_t* at = src[u] + k0;
      if (ragged && k0 + off[u] >= K) at = src[u] - off[u];  // past the row: any of its chunks, zeroed below
      __builtin_amdgcn_global_load_lds(reinterpret_cast<const __attribute__((address_space(1))) void*>(reinterpret_cast<uintptr_t>(at)),
                                       reinterpret_cast<HK_LDS void*>(reinterpret_cast<uintptr_t>(st + (wave + P::kWaves * u) * 1024)),
                                       16, 0, 0);
    }
  };
  const int pre = min(P::STAGES - 1, n);
  for (int i = 0; i < pre; ++i) issue(i);
  const int fx = swz(l16);
  for (int i = 0; i < n; ++i) {
    small_wait_stage<P::kLoads>(min(P::STAGES - 2, n - 1 - i));
    if (i + P::STAGES - 1 < n) issue(i + P::STAGES - 1);  // into the slot that every wave has read
    const uint8_t* st = smem + (i % P::STAGES) * P::kStage;
    bf16x8 a[2][P::MT], b[2][P::NT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int slot = ((4 * h + lg) ^ fx) * 16;
#pragma unroll
      for (int j = 0; j < P::MT; ++j) a[h][j] = *reinterpret_cast<const bf16x8*>(st + (16 * (wm * P::MT + j) + l16) * 128 + slot);
#pragma unroll
      for (int j = 0; j < P::NT; ++j) b[h][j] = *reinterpret_cast<const bf16x8*>(st + (P::BM + 16 * (wn * P::NT + j) + l16) * 128 + slot);
    }
    if ((s0 + i + 1) * kRowsStep > K) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if ((s0 + i) * kRowsStep + 32 * h + 8 * lg >= K) {
#pragma unroll
          for (int j = 0; j < P::MT; ++j) a[h][j] = zero_bf16x8();
#pragma unroll
          for (int j = 0; j < P::NT; ++j) b[h][j] = zero_bf16x8();
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < P::MT; ++j)
#pragma unroll
        for (int l = 0; l < P::NT; ++l) acc[j][l] = mfma_bf16_16x16x32(a[h][j], b[h][l], acc[j][l]);
  }
  __syncthreads();
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

// One workgroup per tile of [16 MT, 16 NT] logits, K split over its waves.
template <int MT, int NT, int WAVES, int DEPTH>
__global__ __launch_bounds__(WAVES * 64) void router_kernel(RouterParams p) {
  __shared__ float red[WAVES * MT * NT * 256];
  const int64_t row0 = blockIdx.x * static_cast<int64_t>(16 * MT);
  const int col0 = blockIdx.y * 16 * NT;
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  const uint16_t* xr[MT];
  const uint16_t* wr[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xr[i] = p.x + min(row0 + 16 * i + (lane & 15), p.rows - 1) * p.hidden;
#pragma unroll
  for (int j = 0; j < NT; ++j) wr[j] = p.w + static_cast<int64_t>(min(col0 + 16 * j + (lane & 15), p.experts - 1)) * p.hidden;
  f32x4 acc[MT][NT] = {};
  rows_product<MT, NT, DEPTH>(xr, wr, p.hidden, wave, WAVES, (p.hidden + kRowsStep - 1) / kRowsStep, acc);
  rows_reduce<MT, NT, WAVES>(acc, red, [&](int r, int c, float v) {
    if (row0 + r < p.rows && col0 + c < p.experts) p.logits[(row0 + r) * p.experts + col0 + c] = v;
  });
}

// Many rows: one workgroup per panel tile.  The column tiles of a row tile run side by
// side on one XCD (workgroups go round-robin over the 8), so x comes from HBM once.
template <typename P>
__global__ __launch_bounds__(P::kWaves * 64) void router_panel_kernel(RouterParams p, int row_tiles, int col_tiles) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int slot = blockIdx.x >> 3;
  const int rt = (slot / col_tiles) * 8 + (blockIdx.x & 7), ct = slot % col_tiles;
  if (rt >= row_tiles) return;
  const int64_t row0 = static_cast<int64_t>(rt) * P::BM;
  const int col0 = ct * P::BN;
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  f32x4 acc[P::MT][P::NT] = {};
  auto row_of = [&](int i) __attribute__((always_inline)) {
    return i < P::BM ? p.x + min(row0 + i, p.rows - 1) * p.hidden
                     : p.w + static_cast<int64_t>(min(col0 + i - P::BM, p.experts - 1)) * p.hidden;
  };
  panel_product<P>(smem, row_of, p.hidden, 0, (p.hidden + kRowsStep - 1) / kRowsStep, acc);
#pragma unroll
  for (int j = 0; j < P::MT; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t row = row0 + 16 * (wave / P::WN * P::MT + j) + 4 * (lane >> 4) + r;
#pragma unroll
      for (int l = 0; l < P::NT; ++l) {
        const int col = col0 + 16 * (wave % P::WN * P::NT + l) + (lane & 15);
        if (row < p.rows && col < p.experts) p.logits[row * p.experts + col] = acc[j][l][r];
      }
    }
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
  int32_t adapters, hidden, n, rank, splits, cols_per_wg;  // cols_per_wg: a multiple of 256
};

constexpr int kLoraWaves = 4;
constexpr int kLoraMaxRank = 256;

// The row block of a workgroup: each XCD (workgroups are dealt to them in turn) takes a run
// of blocks, so that the adapters of its segments stay in its L2.  The grid is a multiple
// of 8 wide; -1 past the last block.
__device__ __forceinline__ int64_t lora_block(const LoraParams& p) {
  const int64_t blocks = (p.rows + kRowsBlock - 1) / kRowsBlock;
  if (blocks <= 8) return blockIdx.x < blocks ? blockIdx.x : -1;
  const int64_t per = gridDim.x / 8, blk = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  return blk < blocks ? blk : -1;
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

// Calls `f(id, n)` for this part's adapters among the block's `live` rows, with their n
// rows listed in `list` (LDS), in order.  With a part per row a part owns the adapter whose
// first row is its own: one step, however many adapters there are; with fewer parts it
// owns every parts-th adapter, so that two adapters of a block are two workgroups'.
// Uniform over the workgroup: every wave holds the same ids.
template <typename F>
__device__ __forceinline__ void lora_groups(int id, uint64_t live, int part, int parts, int* list, F f) {
  const int lane = lane_id();
  const bool by_row = parts >= kRowsBlock;
  uint64_t todo = by_row ? live & (1ull << part) : live;
  int turn = by_row ? part : 0;
  while (todo != 0) {
    const int first = __builtin_ctzll(todo);
    const int gid = __builtin_amdgcn_readlane(id, first);
    const uint64_t rows = __ballot(id == gid) & live;
    todo &= ~rows;
    if ((rows & ((1ull << first) - 1)) != 0) continue;  // by row: not its first
    const bool mine = turn == part;
    if (!by_row) turn = turn + 1 == parts ? 0 : turn + 1;
    if (!mine) continue;
    __syncthreads();  // the list's last user is done
    if (threadIdx.x < 64 && (rows >> lane & 1)) list[__builtin_popcountll(rows & ((1ull << lane) - 1))] = lane;
    __syncthreads();
    f(gid, __builtin_popcountll(rows));
  }
}

// v[split] of up to 16 MT rows of adapter `id` and 16 NT ranks from r0.
template <int MT, int NT, int DEPTH>
__device__ __forceinline__ void lora_shrink_tile(const LoraParams& p, int64_t t0, int id, int n, const int* list, int r0,
                                                 float* red) {
  const int lane = lane_id(), wave = threadIdx.x >> 6, split = blockIdx.z;
  const uint16_t* xr[MT];
  const uint16_t* wr[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xr[i] = p.x + (t0 + list[min(16 * i + (lane & 15), n - 1)]) * p.x_stride;
#pragma unroll
  for (int j = 0; j < NT; ++j)
    wr[j] = p.a + (static_cast<int64_t>(id) * p.rank + min(r0 + 16 * j + (lane & 15), p.rank - 1)) * p.hidden;
  // this workgroup's share of the K steps
  const int steps = (p.hidden + kRowsStep - 1) / kRowsStep;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * split / p.splits);
  const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / p.splits);
  f32x4 acc[MT][NT] = {};
  rows_product<MT, NT, DEPTH>(xr, wr, p.hidden, s0 + wave, kLoraWaves, s1, acc);
  float* v = p.v + (split * p.rows + t0) * p.rank;
  rows_reduce<MT, NT, kLoraWaves>(acc, red, [&](int i, int c, float val) {
    if (i < n && r0 + c < p.rank) v[static_cast<int64_t>(list[i]) * p.rank + r0 + c] = val;
  });
}

// The same for more than 16 rows, P::BN ranks from r0.
template <typename P>
__device__ __forceinline__ void lora_shrink_panel(const LoraParams& p, int64_t t0, int id, int n, const int* list, int r0,
                                                  uint8_t* smem) {
  const int lane = lane_id(), wave = threadIdx.x >> 6, split = blockIdx.z;
  const int steps = (p.hidden + kRowsStep - 1) / kRowsStep;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * split / p.splits);
  const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / p.splits);
  f32x4 acc[P::MT][P::NT] = {};
  auto row_of = [&](int i) __attribute__((always_inline)) {
    return i < P::BM ? p.x + (t0 + list[min(i, n - 1)]) * p.x_stride
                     : p.a + (static_cast<int64_t>(id) * p.rank + min(r0 + i - P::BM, p.rank - 1)) * p.hidden;
  };
  panel_product<P>(smem, row_of, p.hidden, s0, s1, acc);
  float* v = p.v + (split * p.rows + t0) * p.rank;
#pragma unroll
  for (int j = 0; j < P::MT; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * (wave / P::WN * P::MT + j) + 4 * (lane >> 4) + r;
#pragma unroll
      for (int l = 0; l < P::NT; ++l) {
        const int c = r0 + 16 * (wave % P::WN * P::NT + l) + (lane & 15);
        if (i < n && c < p.rank) v[static_cast<int64_t>(list[i]) * p.rank + c] = acc[j][l][r];
      }
    }
}

// grid: (row blocks, parts of a block's adapters, splits).  16 NT ranks at a time.
template <int NT>
__global__ __launch_bounds__(kLoraWaves * 64) void lora_shrink_kernel(LoraParams p) {
  using P = Panel<kRowsBlock, NT == 4 ? 64 : 32, NT == 4 ? 2 : 4, NT == 4 ? 2 : 1, 4>;
  constexpr int kRed = kLoraWaves * NT * 1024;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[P::kLds > kRed ? P::kLds : kRed];
  float* red = reinterpret_cast<float*>(smem);
  __shared__ int list[kRowsBlock];
  const int64_t blk = lora_block(p);
  if (blk < 0) return;
  const int id = lora_id(p, blk);
  lora_groups(id, __ballot(id >= 0), blockIdx.y, gridDim.y, list, [&](int gid, int n) {
    for (int r0 = 0; r0 < p.rank; r0 += 16 * NT) {
      if (n > 16)
        lora_shrink_panel<P>(p, blk * kRowsBlock, gid, n, list, r0, smem);
      else
        lora_shrink_tile<1, NT, 4>(p, blk * kRowsBlock, gid, n, list, r0, red);
    }
  });
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

constexpr int kLoraPad = 8;  // LDS row pitch: off a multiple of the banks' width, 16-byte aligned
constexpr int lora_pitch(int rank) { return (rank + 31) / 32 * 32 + kLoraPad; }
constexpr int lora_lds_bytes(int rank, int terms) { return terms * kRowsBlock * lora_pitch(rank) * 2; }

// out of one adapter's rows, two tiles of 16 at a time.  The operands are swapped (B rows
// first), and result row 4g + i of column tile jt is column 16g + 4jt + i: a lane then
// holds 16 adjacent columns of one row, and a wave whole 128-byte lines of it (bf16).  y
// comes in while the products run and is added last.  ONE: the rank fits one step of 64,
// and B is read once for all the rows.
template <bool F32, int TERMS, bool ONE>
__device__ __forceinline__ void lora_expand_rows(const LoraParams& p, int64_t t0, int id, int n, const int* list,
                                                 const uint16_t* vt, int c_begin, int c_end) {
  const int lane = lane_id(), wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
  const int pitch = lora_pitch(p.rank);
  const uint16_t* bm = p.b + static_cast<int64_t>(id) * p.n * p.rank;
  for (int col0 = c_begin + 64 * wave; col0 < c_end; col0 += 64 * kLoraWaves) {
    const int n_lane = col0 + 16 * g;
    const bool live[2] = {n_lane < c_end, n_lane + 8 < c_end};  // c_end % 8 == 0
    const uint16_t* br[4];
#pragma unroll
    for (int jt = 0; jt < 4; ++jt)
      br[jt] = bm + static_cast<int64_t>(min(col0 + 16 * (m >> 2) + 4 * jt + (m & 3), c_end - 1)) * p.rank;
    bf16x8 b[2][4];
    auto load_b = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = k0 + 32 * h + 8 * g;
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) b[h][jt] = k < p.rank ? *reinterpret_cast<const bf16x8*>(br[jt] + k) : zero_bf16x8();
      }
    };
    if constexpr (ONE) load_b(0);
    for (int i0 = 0; i0 < n; i0 += 32) {
      int64_t row[2];
      uint4 y[2][F32 ? 4 : 2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        row[i] = t0 + list[min(i0 + 16 * i + m, n - 1)];
        if (i0 + 16 * i + m < n) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!live[h]) continue;
            if constexpr (F32) {
              const uint4* src = reinterpret_cast<const uint4*>(static_cast<const float*>(p.y) + row[i] * p.y_stride + n_lane + 8 * h);
              y[i][2 * h] = src[0];
              y[i][2 * h + 1] = src[1];
            } else {
              y[i][h] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.y) + row[i] * p.y_stride + n_lane + 8 * h);
            }
          }
        }
      }
      f32x4 acc[2][4] = {};
      for (int k0 = 0; k0 < (ONE ? 1 : p.rank); k0 += 64) {
        if constexpr (!ONE) load_b(k0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (k0 + 32 * h >= p.rank) break;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = TERMS - 1; q >= 0; --q) {
              const bf16x8 f = *reinterpret_cast<const bf16x8*>(vt + (q * kRowsBlock + i0 + 16 * i + m) * pitch + k0 + 32 * h + 8 * g);
#pragma unroll
              for (int jt = 0; jt < 4; ++jt) acc[i][jt] = mfma_bf16_16x16x32(b[h][jt], f, acc[i][jt]);
            }
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i0 + 16 * i + m < n) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!live[h]) continue;
            if constexpr (F32) {
              f32x4* dst = reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + row[i] * p.out_stride + n_lane + 8 * h);
              dst[0] = __builtin_bit_cast(f32x4, y[i][2 * h]) + acc[i][2 * h];
              dst[1] = __builtin_bit_cast(f32x4, y[i][2 * h + 1]) + acc[i][2 * h + 1];
            } else {
              const uint32_t w[4] = {y[i][h].x, y[i][h].y, y[i][h].z, y[i][h].w};
              uint32_t o[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                o[e] = pack_bf16x2(__uint_as_float(w[e] << 16) + acc[i][2 * h + e / 2][2 * (e & 1)],
                                   __uint_as_float(w[e] & 0xffff0000u) + acc[i][2 * h + e / 2][2 * (e & 1) + 1]);
              *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + row[i] * p.out_stride + n_lane + 8 * h) =
                  uint4{o[0], o[1], o[2], o[3]};
            }
          }
        }
      }
    }
  }
}

// grid: (row blocks, parts of a block's adapters, column parts).  The rows without an
// adapter are a group of their own, copied unless out is y.
template <bool F32, int TERMS>
__global__ __launch_bounds__(kLoraWaves * 64, 3) void lora_expand_kernel(LoraParams p) {
  extern __shared__ __align__(16) uint16_t vt[];  // [TERMS][kRowsBlock][pitch]
  __shared__ int list[kRowsBlock];
  const int64_t blk = lora_block(p), t0 = blk * kRowsBlock;
  if (blk < 0) return;
  const int id = lora_id(p, blk);
  const int c_begin = blockIdx.z * p.cols_per_wg, c_end = min(c_begin + p.cols_per_wg, p.n);
  lora_groups(id, __ballot(p.y != p.out ? id >= -1 : id >= 0), blockIdx.y, gridDim.y, list, [&](int gid, int n) {
    if (gid < 0) {
      constexpr int kPer = F32 ? 4 : 8;  // values of 16 bytes
      const int chunks = (c_end - c_begin) / kPer;
      for (int i = 0; i < n; ++i) {
        const int64_t t = t0 + list[i];
        for (int c = threadIdx.x; c < chunks; c += kLoraWaves * 64) {
          const int64_t at = c_begin + c * kPer;
          const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.y) + (t * p.y_stride + at) * (16 / kPer));
          *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + (t * p.out_stride + at) * (16 / kPer)) = *src;
        }
      }
      return;
    }
    // v of the rows, the splits summed in order and scaled, as bf16 terms; 0 past the rank
    const int pitch = lora_pitch(p.rank), quads = (pitch - kLoraPad) / 4;
    const float c = p.scaling != nullptr ? p.scaling[gid] : 1.0f;
    for (int e = threadIdx.x; e < n * quads; e += kLoraWaves * 64) {
      const int i = e / quads, r = 4 * (e - i * quads);
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (r < p.rank) {
        const float* src = p.v + (t0 + list[i]) * p.rank + r;
        for (int s = 0; s < p.splits; s += 8) {  // the loads of eight splits at once
          f32x4 part[8];
#pragma unroll
          for (int u = 0; u < 8; ++u)
            part[u] = s + u < p.splits ? *reinterpret_cast<const f32x4*>(src + (s + u) * p.rows * p.rank) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int u = 0; u < 8; ++u) v += part[u];
        }
        v *= c;
      }
      uint16_t t16[4][TERMS];
#pragma unroll
      for (int u = 0; u < 4; ++u) split_bf16<TERMS>(v[u], t16[u]);
#pragma unroll
      for (int q = 0; q < TERMS; ++q)
        *reinterpret_cast<uint2*>(vt + (q * kRowsBlock + i) * pitch + r) =
            uint2{t16[0][q] | static_cast<uint32_t>(t16[1][q]) << 16, t16[2][q] | static_cast<uint32_t>(t16[3][q]) << 16};
    }
    __syncthreads();
    if (p.rank <= 64)
      lora_expand_rows<F32, TERMS, true>(p, t0, gid, n, list, vt, c_begin, c_end);
    else
      lora_expand_rows<F32, TERMS, false>(p, t0, gid, n, list, vt, c_begin, c_end);
  });
}

}  // namespace hkmoe
