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

#include "gemm_skinny.hpp"
#include "gemm_small.hpp"

namespace hkmoe {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma_bf16_16x16x32(const bf16x8& a, const bf16x8& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ bf16x8 zero_bf16x8() { return __builtin_bit_cast(bf16x8, i32x4{0, 0, 0, 0}); }

constexpr int kRowsBlock = 64;  // adapters' rows per workgroup at most (4 MFMA row tiles)
constexpr int kRowsStep = 64;   // K per step: whole 128-byte lines

// acc[nt] += 16 rows of x (xr: this lane's) times NT tiles of 16 rows of w (wr: this lane's
// row in each), over K steps st, st + stride, ... < steps of 64.  Rows past the
// last may repeat a valid one: a result row depends on its own operand rows alone.
// The loads of up to DEPTH steps are issued before the first product, so that
// 2 DEPTH (1 + NT) of them are in flight per wave.
template <int NT, int DEPTH>
__device__ __forceinline__ void rows_product(const uint16_t* xr, const uint16_t* const (&wr)[NT], int K, int st, int stride,
                                             int steps, f32x4 (&acc)[NT]) {
  const int k_lane = 8 * (lane_id() >> 4);
  bf16x8 a[DEPTH][2], b[DEPTH][2][NT];
  auto load = [&](int d, int k0) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = k0 + 32 * h + k_lane;
      a[d][h] = *reinterpret_cast<const bf16x8*>(xr + k);
#pragma unroll
      for (int i = 0; i < NT; ++i) b[d][h][i] = *reinterpret_cast<const bf16x8*>(wr[i] + k);
    }
  };
  auto mma = [&](int d) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[j] = mfma_bf16_16x16x32(a[d][h], b[d][h][j], acc[j]);
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
      a[0][h] = k < K ? *reinterpret_cast<const bf16x8*>(xr + k) : zero_bf16x8();
#pragma unroll
      for (int i = 0; i < NT; ++i) b[0][h][i] = k < K ? *reinterpret_cast<const bf16x8*>(wr[i] + k) : zero_bf16x8();
    }
    mma(0);
  }
}

// Sums the waves' tiles in wave order and hands (row, column, value) of the
// [16, 16 NT] result to `put`.  red: WAVES * NT * 256 floats of LDS.
template <int NT, int WAVES, typename Put>
__device__ __forceinline__ void rows_reduce(const f32x4 (&acc)[NT], float* red, Put put) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int kTile = NT * 256;
  __syncthreads();  // red is free: the last user's reads are done
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) red[wave * kTile + ((4 * (lane >> 4) + r) * NT + j) * 16 + (lane & 15)] = acc[j][r];
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
// registers, 29 through LDS).  So the rows of both operands come in
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
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0 && BM % (16 * WM) == 0 && BN % (16 * WN) == 0, "tile");
  static_assert(STAGES >= 2 && (STAGES - 1) * kLoads <= 63, "ring depth, vmcnt range");
};

// vmcnt wait that leaves this wave's loads of the newest `newer` (at most MOST) stages in
// flight, L loads each, then a barrier: every wave's loads of the older ones are in LDS, and
// every wave's LDS reads are done.  The compiler's own s_waitcnt (simm16: vmcnt in bits 0-3
// and 14-15, lgkmcnt in 8-11), so that it knows the fragments read so far to be complete
// and adds no lgkmcnt(0) between the next step's reads and this step's products
// (8192x7168x256 from the Infinity Cache 46 us, with the reads ahead of the products 42).
template <int L, int MOST>
__device__ __forceinline__ void panel_wait(int newer) {
  if constexpr (MOST > 0) {
    if (newer < MOST) return panel_wait<L, MOST - 1>(newer);
  }
  constexpr int kVm = L * MOST;
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((kVm & 15) | (kVm >> 4) << 14 | 0x70);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// acc += the tile over K steps s0 .. s1 - 1.  x, w: bases that the whole workgroup shares;
// x_off(i), w_off(i): byte offset from them (below 2^32 - 2^22, a multiple of 16) of row i
// of the BM rows and of the BN columns; rows past the last may repeat a valid one.
// Step kt's products run beside the LDS reads of step kt + 1 (two register sets) and the DMA
// of the steps after it.  Every wave of the workgroup calls it; on return all are done with
// smem.
template <typename P, typename XOff, typename WOff>
__device__ __forceinline__ void panel_product(uint8_t* smem, const uint16_t* x, XOff x_off, const uint16_t* w, WOff w_off, int K,
                                              int s0, int s1, f32x4 (&acc)[P::MT][P::NT]) {
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, lg = lane >> 4, wm = wave / P::WN, wn = wave % P::WN;
  constexpr int kAhead = P::STAGES - 1, kXLoads = P::BM / 8 / P::kWaves;
  const i32x4 x_srd = make_srd(x, 0xffffffffu), w_srd = make_srd(w, 0xffffffffu);
  uint32_t off[P::kLoads];
  int chunk[P::kLoads];  // this lane's chunk of a step
#pragma unroll
  for (int u = 0; u < P::kLoads; ++u) {
    const int r = 8 * (wave + P::kWaves * u) + (lane >> 3);
    chunk[u] = (lane & 7) ^ swz(r);
    off[u] = (u < kXLoads ? x_off(r) : w_off(r - P::BM)) + 16 * chunk[u];
  }
  const int n = s1 - s0;
  // DMA of step i.  The last one of K % 64 != 0 takes the step's first chunk in the place of
  // those past the row; their products are cut below.
  auto issue = [&](int i, auto ragged) __attribute__((always_inline)) {
    uint8_t* st = smem + (i % P::STAGES) * P::kStage;
    const int k0 = (s0 + i) * kRowsStep;
#pragma unroll
    for (int u = 0; u < P::kLoads; ++u) {
      uint32_t at = off[u];
      if constexpr (decltype(ragged)::value) {
        if (k0 + 8 * chunk[u] >= K) at -= 16 * chunk[u];
      }
      load_lds_16B(u < kXLoads ? x_srd : w_srd, st + (wave + P::kWaves * u) * 1024, static_cast<int>(at), 2 * k0);
    }
  };
  const int fx = swz(l16);
  struct Frags {
    bf16x8 a[2][P::MT], b[2][P::NT];
  };
  auto read = [&](int i, Frags& f) __attribute__((always_inline)) {
    const uint8_t* st = smem + (i % P::STAGES) * P::kStage;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int slot = ((4 * h + lg) ^ fx) * 16;
#pragma unroll
      for (int j = 0; j < P::MT; ++j) f.a[h][j] = *reinterpret_cast<const bf16x8*>(st + (16 * (wm * P::MT + j) + l16) * 128 + slot);
#pragma unroll
      for (int j = 0; j < P::NT; ++j) f.b[h][j] = *reinterpret_cast<const bf16x8*>(st + (P::BM + 16 * (wn * P::NT + j) + l16) * 128 + slot);
    }
  };
  auto mma = [&](const Frags& f) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < P::MT; ++j)
#pragma unroll
        for (int l = 0; l < P::NT; ++l) acc[j][l] = mfma_bf16_16x16x32(f.a[h][j], f.b[h][l], acc[j][l]);
  };
  // K's last step, K % 64 != 0: both operands 0 past K
  auto cut = [&](int i, Frags& f) __attribute__((always_inline)) {
    if ((s0 + i + 1) * kRowsStep <= K) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if ((s0 + i) * kRowsStep + 32 * h + 8 * lg < K) continue;
#pragma unroll
      for (int j = 0; j < P::MT; ++j) f.a[h][j] = zero_bf16x8();
#pragma unroll
      for (int j = 0; j < P::NT; ++j) f.b[h][j] = zero_bf16x8();
    }
  };
  if (n > 0) {
    const int pre = min(kAhead, n);
    for (int i = 0; i < pre; ++i) issue(i, std::true_type{});
    panel_wait<P::kLoads, kAhead - 1>(pre - 1);
    Frags f0, f1;
    read(0, f0);
    // Step i: DMA of step i + kAhead into the slot of step i - 1 (its reads are complete at
    // step i - 1's barrier), step i + 1's fragments, step i's products.
    auto step_full = [&](int i, Frags& cur, Frags& next) __attribute__((always_inline)) {
      issue(i + kAhead, std::false_type{});
      panel_wait<P::kLoads, kAhead - 1>(kAhead - 1);
      read(i + 1, next);
      mma(cur);
      // one LDS read, one product, in turn: a wave issues a read only every 40 cycles or so,
      // and the products fit between
#pragma unroll
      for (int u = 0; u < 2 * (P::MT + P::NT); ++u) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    auto step = [&](int i, Frags& cur, Frags& next) __attribute__((always_inline)) {
      if (i + kAhead < n) issue(i + kAhead, std::true_type{});
      if (i + 1 < n) {
        panel_wait<P::kLoads, kAhead - 1>(min(kAhead - 1, n - 2 - i));
        read(i + 1, next);
      } else {
        cut(i, cur);
      }
      __builtin_amdgcn_sched_barrier(0);
      mma(cur);
      __builtin_amdgcn_sched_barrier(0);
    };
    int i = 0;
    for (; i + 2 + kAhead < n; i += 2) {  // the DMA of all but K's last step
      step_full(i, f0, f1);
      step_full(i + 1, f1, f0);
    }
    for (; i + 1 < n; i += 2) {
      step(i, f0, f1);
      step(i + 1, f1, f0);
    }
    if (i < n) step(i, f0, f1);
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

// Few rows or few tiles: one workgroup per tile of [16 MT, 16 NT] logits, K split over its NW
// waves, each streaming its steps through an LDS ring of its own, DEPTH steps deep (whole
// 128-byte lines, no barrier in the loop); the partial tiles are summed in wave order.  16x16
// tiles on 16 waves: 64x4096x128 5.9 us, on 8 with twice the depth 7.3, straight into
// registers 8.8.
template <int MT_, int NT_, int NW_, int DEPTH_>
struct Strip {
  static constexpr int MT = MT_, NT = NT_, NW = NW_, DEPTH = DEPTH_;
  static constexpr int kStep = (MT + NT) * 2048, kRing = NW * DEPTH * kStep, kLd = 16 * NT + 4;
  static constexpr int kPart = NW * 16 * MT * kLd * 4, kLds = kRing > kPart ? kRing : kPart;
  static constexpr int kLoads = 2 * (MT + NT);  // DMA instructions per step
  static_assert(1 <= MT && MT <= NT && NT <= 2, "tile");
  static_assert(DEPTH >= 2 && kLoads * (DEPTH - 1) <= 63 && kLds <= kSkMaxLds, "ring depth, vmcnt range");
};

template <typename S>
__global__ __launch_bounds__(S::NW * 64) void router_strip_kernel(RouterParams p) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int64_t row0 = blockIdx.x * static_cast<int64_t>(16 * S::MT);
  const int col0 = blockIdx.y * 16 * S::NT;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, lg = lane >> 4, ld_row = lane >> 3;
  const int K = p.hidden, steps = (K + kRowsStep - 1) / kRowsStep;
  const int mine = (steps - wave + S::NW - 1) / S::NW;  // this wave's steps (0: none)
  const i32x4 x_srd = make_srd(p.x + row0 * K, 0xffffffffu), w_srd = make_srd(p.w, 0xffffffffu);
  const int last = static_cast<int>(min(static_cast<int64_t>(16 * S::MT), p.rows - row0)) - 1;
  // instruction u fills ring rows 8u .. 8u + 7, of x and then of w; the lane fetches the
  // chunk that lands swizzled.  Rows past the last repeat it (never stored).
  uint32_t off[S::kLoads];
#pragma unroll
  for (int u = 0; u < S::kLoads; ++u) {
    const int r = 8 * u + ld_row;
    off[u] = static_cast<uint32_t>(u < 2 * S::MT ? min(r, last) : min(col0 + r - 16 * S::MT, p.experts - 1)) * (2 * static_cast<uint32_t>(K)) +
             16 * ((lane & 7) ^ swz(r));
  }
  uint8_t* ring = smem + wave * S::DEPTH * S::kStep;
  // Steps past the last one go through empty descriptors (no memory traffic), so the loads
  // in flight stay a constant count.  K's last step, K % 64 != 0, takes its first chunk in
  // the place of those past the row; their products are cut below.
  auto issue = [&](int i, int slot) __attribute__((always_inline)) {
    const bool in = i < mine;
    const int k0 = in ? (wave + S::NW * i) * kRowsStep : 0;
    i32x4 xs = x_srd, ws = w_srd;
    xs.z = in ? xs.z : 0;
    ws.z = in ? ws.z : 0;
#pragma unroll
    for (int u = 0; u < S::kLoads; ++u) {
      uint32_t at = off[u];
      if (k0 + kRowsStep > K) {
        const int chunk = (lane & 7) ^ swz(8 * u + ld_row);
        if (k0 + 8 * chunk >= K) at -= 16 * chunk;
      }
      load_lds_16B(u < 2 * S::MT ? xs : ws, ring + slot * S::kStep + u * 1024, static_cast<int>(at), 2 * k0);
    }
  };
  const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ring)) + l16 * 128;
  const uint32_t lo_off = (lg ^ swz(l16)) << 4, hi_off = ((lg + 4) ^ swz(l16)) << 4;
  f32x4 acc[S::MT][S::NT] = {};
#pragma unroll
  for (int u = 0; u < S::DEPTH; ++u) issue(u, u);
  int slot = 0;
  for (int i = 0; i < mine; ++i) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(S::kLoads * (S::DEPTH - 1)) : "memory");
    const uint32_t lo = base + slot * S::kStep + lo_off, hi = base + slot * S::kStep + hi_off;
    i32x8 a[S::MT], b[S::NT];
    if constexpr (S::MT == 1) sk_frag<0>(lo, hi, a[0]);
    else sk_frag2<0>(lo, hi, a[0], a[1]);
    if constexpr (S::NT == 1) sk_frag<S::MT * 2048>(lo, hi, b[0]);
    else sk_frag2<S::MT * 2048>(lo, hi, b[0], b[1]);
    issue(i + S::DEPTH, slot);  // this wave has read the slot
    __builtin_amdgcn_sched_barrier(0);
    const int k0 = (wave + S::NW * i) * kRowsStep;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool cut = k0 + 32 * h + 8 * lg >= K;
      bf16x8 ah[S::MT], bh[S::NT];
#pragma unroll
      for (int j = 0; j < S::MT; ++j) ah[j] = cut ? zero_bf16x8() : __builtin_bit_cast(bf16x8, h ? a[j].hi : a[j].lo);
#pragma unroll
      for (int j = 0; j < S::NT; ++j) bh[j] = cut ? zero_bf16x8() : __builtin_bit_cast(bf16x8, h ? b[j].hi : b[j].lo);
#pragma unroll
      for (int j = 0; j < S::MT; ++j)
#pragma unroll
        for (int l = 0; l < S::NT; ++l) acc[j][l] = mfma_bf16_16x16x32(ah[j], bh[l], acc[j][l]);
    }
    slot = slot == S::DEPTH - 1 ? 0 : slot + 1;
  }
  // every wave's DMA has landed before the partial tiles overwrite the rings
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int j = 0; j < S::MT; ++j)
#pragma unroll
    for (int l = 0; l < S::NT; ++l)
#pragma unroll
      for (int r = 0; r < 4; ++r) part[(wave * 16 * S::MT + 16 * j + 4 * lg + r) * S::kLd + 16 * l + l16] = acc[j][l][r];
  __syncthreads();
  for (int e = threadIdx.x; e < 256 * S::MT * S::NT; e += S::NW * 64) {
    const int r = e / (16 * S::NT), c = e % (16 * S::NT);
    float v = part[r * S::kLd + c];
#pragma unroll
    for (int w = 1; w < S::NW; ++w) v += part[(w * 16 * S::MT + r) * S::kLd + c];
    if (row0 + r < p.rows && col0 + c < p.experts) p.logits[(row0 + r) * p.experts + col0 + c] = v;
  }
}

// Many rows: one workgroup per panel tile.  The column tiles of a row tile run side by
// side on one XCD (workgroups go round-robin over the 8), so x comes from HBM once.
// 8192x7168x256: 52 us, 2.5 TB/s and 580 TFLOP/s, bound by what a CU takes in (24 KiB a step).
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
  const int last = static_cast<int>(min(static_cast<int64_t>(P::BM), p.rows - row0)) - 1;
  const uint32_t pitch = 2 * static_cast<uint32_t>(p.hidden);  // H <= 2^20: 64 rows, 1024 experts stay below 2^32
  panel_product<P>(
      smem, p.x + row0 * p.hidden, [&](int i) { return min(i, last) * pitch; }, p.w,
      [&](int i) { return min(col0 + i, p.experts - 1) * pitch; }, p.hidden, 0, (p.hidden + kRowsStep - 1) / kRowsStep, acc);
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
// rows of one adapter of one block: the requests of a decode batch each find their
// workgroup.  Large batches are sorted by adapter first (lora_plan_kernel), so that
// the blocks are of one adapter each.  Then two launches: the narrow product
// v = x A_l^T (its K split over `splits` workgroups, each writing its own fp32 partial
// sums), and y + c_l v B_l^T.
// 8192 rows, 7168 -> 64 -> 4096, bf16: 31 us (22 at a copy's rate) and 43 (28).
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
  const int32_t* perm;        // [T] rows by adapter, null: row blocks as they come
  const i32x4* items;         // (adapter or -1, first place in perm, rows)
  const int32_t* item_count;
};

constexpr int kLoraWaves = 4;
constexpr int kLoraMaxRank = 256;

// Workgroup `bid` of a grid that is a multiple of 8 wide, as a place among `count`: each XCD
// (workgroups are dealt to them in turn) takes a run of places, so that the adapters of its
// rows stay in its L2.  -1 past the last.
__device__ __forceinline__ int64_t xcd_run(int64_t bid, int64_t count) {
  const int64_t per = (count + 7) / 8, at = (bid & 7) * per + (bid >> 3);
  return (bid >> 3) < per && at < count ? at : -1;
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

// Calls `f(id, n, t0)` for each group of rows of one adapter that is this workgroup's: its n
// (at most 64) rows are t0 + list[0 .. n - 1] (list: LDS).  `bare`: the rows without an
// adapter are a group, too (id < 0).  With a plan the workgroup's group is an item of it.
// Without one it takes adapters of its row block, in order of their first rows: with a part
// (blockIdx.y) per row the one whose first row is the part's own, which is one step, however
// many adapters there are; with fewer parts every parts-th, so that two adapters of a block are
// two workgroups'.  Uniform over the workgroup: every wave holds the same ids.
template <typename F>
__device__ __forceinline__ void lora_groups(const LoraParams& p, bool bare, int* list, F f) {
  const int lane = lane_id();
  const bool planned = p.items != nullptr;
  int64_t at, t0 = 0;
  uint64_t live = 0, todo = 0;
  int id = 0, turn = 0;
  const int part = blockIdx.y, parts = gridDim.y;
  const bool by_row = parts >= kRowsBlock;
  if (planned) {
    at = xcd_run(blockIdx.x, *p.item_count);
    todo = 1;
  } else {
    const int64_t blocks = (p.rows + kRowsBlock - 1) / kRowsBlock;
    at = blocks <= 8 ? blockIdx.x : xcd_run(blockIdx.x, blocks);
  }
  if (at < 0) return;
  if (!planned) {
    t0 = at * kRowsBlock;
    id = lora_id(p, at);
    live = __ballot(id >= (bare ? -1 : 0));
    todo = by_row ? live & (1ull << part) : live;
    turn = by_row ? part : 0;
  }
  while (todo != 0) {
    int gid, n;
    if (planned) {
      const i32x4 item = p.items[at];
      gid = item.x;
      n = item.z;
      if (gid < 0 && !bare) return;
      if (static_cast<int>(threadIdx.x) < n) list[threadIdx.x] = p.perm[item.y + threadIdx.x];
      todo = 0;
    } else {
      const int first = __builtin_ctzll(todo);
      gid = __builtin_amdgcn_readlane(id, first);
      const uint64_t rows = __ballot(id == gid) & live;
      todo &= ~rows;
      if ((rows & ((1ull << first) - 1)) != 0) continue;  // by row: not its first
      const bool mine = turn == part;
      if (!by_row) turn = turn + 1 == parts ? 0 : turn + 1;
      if (!mine) continue;
      n = __builtin_popcountll(rows);
      __syncthreads();  // the list's last user is done
      if (threadIdx.x < 64 && (rows >> lane & 1)) list[__builtin_popcountll(rows & ((1ull << lane) - 1))] = lane;
    }
    __syncthreads();
    f(gid, n, t0);
  }
}

// The plan: rows sorted by adapter (stable, so that a row's group, and with it the order of its
// sums, is the same every time), in items of at most 64 rows.  Without it every block of a
// shuffled batch reads every adapter (1078 rows over 24 adapters, 5672 -> 72 -> 896: 143 us
// without, 36 with).  One workgroup; each of its 16 waves counts and places a run of rows, 64
// at a time: in a trace 6.7 us for 2048 rows shuffled over 64 adapters, 8.1 for 8192 in
// segments of 7, of which half are the launch and the ids' latency.  LDS: counts [16][bins],
// places [bins], item places [bins], 512 ids per wave; bins = adapters + 1 (the last: none).
constexpr int kPlanWaves = 16, kPlanBins = 1536, kPlanRows = 65536, kPlanFlight = 8;
constexpr int lora_plan_lds(int bins) { return ((kPlanWaves + 2) * bins + kPlanWaves * kPlanFlight * 64) * 4; }
static_assert(lora_plan_lds(kPlanBins) <= kSkMaxLds - 1024, "LDS budget");
constexpr int64_t lora_plan_items(int64_t rows, int64_t adapters) {  // at most
  return rows / kRowsBlock + (rows < adapters + 1 ? rows : adapters + 1);
}

__global__ __launch_bounds__(kPlanWaves * 64) void lora_plan_kernel(const int32_t* __restrict__ ids, int rows, int adapters,
                                                                    int32_t* __restrict__ perm, i32x4* __restrict__ items,
                                                                    int32_t* __restrict__ item_count) {
  extern __shared__ int counts[];
  __shared__ uint64_t sums[kPlanWaves];
  const int bins = adapters + 1, tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int* start = counts + kPlanWaves * bins;
  int* item_start = start + bins;
  int* mine = counts + wave * bins;
  for (int b = lane; b < bins; b += 64) mine[b] = 0;
  const int per = (rows + 64 * kPlanWaves - 1) / (64 * kPlanWaves) * 64, end = min(rows, (wave + 1) * per);
  // f(t, bin) for 64 rows at a time in order (bin -1 past the wave's last).  The ids of eight
  // times 64 rows are loaded at once, and once for both passes where a wave has no more; through
  // LDS, so that the loop over them stays one (unrolled, fetching its code took 3 us).
  int* bins8 = item_start + bins + wave * kPlanFlight * 64;
  auto load = [&](int t8) __attribute__((always_inline)) {
    int id[kPlanFlight];
#pragma unroll
    for (int u = 0; u < kPlanFlight; ++u) id[u] = ids[min(t8 + 64 * u + lane, rows - 1)];
#pragma unroll
    for (int u = 0; u < kPlanFlight; ++u)
      bins8[64 * u + lane] = t8 + 64 * u + lane >= end ? -1 : id[u] < 0 || id[u] >= adapters ? adapters : id[u];
  };
  load(wave * per);
  auto each = [&](auto f) __attribute__((always_inline)) {
    for (int t8 = wave * per; t8 < end; t8 += 64 * kPlanFlight) {
      if (per > 64 * kPlanFlight) load(t8);
#pragma unroll 1
      for (int u = 0; u < kPlanFlight && t8 + 64 * u < end; ++u) f(t8 + 64 * u + lane, bins8[64 * u + lane]);
    }
  };
  // the lanes with this lane's bin: all of them, or a bit of the bin at a time
  auto same_bin = [&](int bin) __attribute__((always_inline)) {
    uint64_t same = __ballot(bin >= 0);
    if (__ballot(bin == __builtin_amdgcn_readfirstlane(bin)) == ~0ull) return same;
    for (int k = 0; 1 << k < bins; ++k) {
      const uint64_t set = __ballot(bin >> k & 1);
      same &= bin >> k & 1 ? set : ~set;
    }
    return same;
  };
  each([&](int, int bin) {
    const uint64_t same = same_bin(bin);
    if (bin >= 0 && (same & ((1ull << lane) - 1)) == 0) mine[bin] += __builtin_popcountll(same);
  });
  __syncthreads();
  // two bins per thread: the waves' places within a bin, the bins' places and items
  static_assert(kPlanBins <= 2 * 64 * kPlanWaves, "bins per thread");
  uint64_t v[2] = {0, 0};  // rows, items << 32
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int b = 2 * tid + u;
    if (b < bins) {
      int n = 0, c[kPlanWaves];
#pragma unroll
      for (int w = 0; w < kPlanWaves; ++w) c[w] = counts[w * bins + b];
#pragma unroll
      for (int w = 0; w < kPlanWaves; ++w) {
        counts[w * bins + b] = n;
        n += c[w];
      }
      v[u] = static_cast<uint64_t>((n + kRowsBlock - 1) / kRowsBlock) << 32 | static_cast<uint32_t>(n);
    }
  }
  uint64_t incl = v[0] + v[1];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t up = __shfl_up(static_cast<unsigned long long>(incl), o, kWave);
    if (lane >= o) incl += up;
  }
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  uint64_t at = incl - v[0] - v[1], all = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    if (w < wave) at += sums[w];
    all += sums[w];
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int b = 2 * tid + u;
    if (b < bins) {
      start[b] = static_cast<int>(at);
      item_start[b] = static_cast<int>(at >> 32);
    }
    at += v[u];
  }
  __syncthreads();
  const int n_items = static_cast<int>(all >> 32);
  if (tid == 0) *item_count = n_items;
  for (int i = tid; i < n_items; i += 64 * kPlanWaves) {
    int b = 0, past = bins;  // the last bin whose first item is not past i
    while (past - b > 1) {
      const int mid = (b + past) >> 1;
      if (item_start[mid] <= i) b = mid; else past = mid;
    }
    const int first = start[b] + (i - item_start[b]) * kRowsBlock;
    items[i] = i32x4{b == adapters ? -1 : b, first, min(kRowsBlock, (b + 1 < bins ? start[b + 1] : rows) - first), 0};
  }
  each([&](int t, int bin) {
    const uint64_t same = same_bin(bin);
    if (bin >= 0) {
      const uint64_t before = same & ((1ull << lane) - 1);
      const int to = start[bin] + mine[bin] + __builtin_popcountll(before);
      perm[to] = t;
      if (before == 0) mine[bin] += __builtin_popcountll(same);
    }
  });
}

// v[split] of up to 16 rows of adapter `id` and 16 NT ranks from r0.
template <int NT, int DEPTH>
__device__ __forceinline__ void lora_shrink_tile(const LoraParams& p, int64_t t0, int id, int n, const int* list, int r0,
                                                 float* red) {
  const int lane = lane_id(), wave = threadIdx.x >> 6, split = blockIdx.z;
  const uint16_t* xr = p.x + (t0 + list[min(lane & 15, n - 1)]) * p.x_stride;
  const uint16_t* wr[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
    wr[j] = p.a + (static_cast<int64_t>(id) * p.rank + min(r0 + 16 * j + (lane & 15), p.rank - 1)) * p.hidden;
  // this workgroup's share of the K steps
  const int steps = (p.hidden + kRowsStep - 1) / kRowsStep;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * split / p.splits);
  const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / p.splits);
  f32x4 acc[NT] = {};
  rows_product<NT, DEPTH>(xr, wr, p.hidden, s0 + wave, kLoraWaves, s1, acc);
  float* v = p.v + (split * p.rows + t0) * p.rank;
  rows_reduce<NT, kLoraWaves>(acc, red, [&](int i, int c, float val) {
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
  // the host keeps 64 rows of x (with a plan: all) and the ranks of an adapter below 2^32 bytes
  panel_product<P>(
      smem, p.x + t0 * p.x_stride, [&](int i) { return list[min(i, n - 1)] * static_cast<uint32_t>(2 * p.x_stride); },
      p.a + static_cast<int64_t>(id) * p.rank * p.hidden,
      [&](int i) { return min(r0 + i, p.rank - 1) * static_cast<uint32_t>(2 * p.hidden); }, p.hidden, s0, s1, acc);
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

// grid: (row blocks, parts of a block's adapters, splits), or (items, 1, splits).  16 NT ranks
// at a time.
template <int NT>
__global__ __launch_bounds__(kLoraWaves * 64) void lora_shrink_kernel(LoraParams p) {
  using P = Panel<kRowsBlock, NT == 4 ? 64 : 32, NT == 4 ? 2 : 4, NT == 4 ? 2 : 1, 4>;
  constexpr int kRed = kLoraWaves * NT * 1024;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[P::kLds > kRed ? P::kLds : kRed];
  float* red = reinterpret_cast<float*>(smem);
  __shared__ int list[kRowsBlock];
  lora_groups(p, false, list, [&](int gid, int n, int64_t t0) {
    for (int r0 = 0; r0 < p.rank; r0 += 16 * NT) {
      if (n > 16)
        lora_shrink_panel<P>(p, t0, gid, n, list, r0, smem);
      else
        lora_shrink_tile<NT, 4>(p, t0, gid, n, list, r0, red);
    }
  });
}

// The narrow product's terms in bf16: v = t0 + t1 (+ t2), each the rounding of what
// the terms before it leave, 2^-17 (2^-25) of |v| at most: a single bf16 term would
// be off by 2^-8, more than an fp32 output may lose and as much as a bf16 one rounds.
// B is bf16 already and every product is exact, so two terms give a bf16 output,
// three an fp32 one, the result of an fp32 v.  An infinite or NaN v keeps its value
// in t0 and leaves 0 in the others, and one past bf16's largest value becomes infinite.
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

// A wave's 16 x 64 products on their way from operand order to rows, fp32.
constexpr int kLoraTilePitch = 68;
constexpr int lora_lds_bytes(int rank, int terms) {
  return terms * kRowsBlock * lora_pitch(rank) * 2 + kLoraWaves * 16 * kLoraTilePitch * 4;
}

// 16 bytes of y / out.  NT: more than the L2s hold, touched once: 8192x4096 bf16 read and
// written in these pieces 26 us, with plain accesses 38; straight from operand order, 16
// rows of 64 bytes an access, 43.
template <bool NT>
__device__ __forceinline__ uint4 lora_load(const void* p) {
  if constexpr (NT) return ld_nt16(p);
  return *static_cast<const uint4*>(p);
}
template <bool NT>
__device__ __forceinline__ void lora_store(void* p, uint4 v) {
  if constexpr (NT) st_nt16(p, v);
  else *static_cast<uint4*>(p) = v;
}

// out of one adapter's rows, two tiles of 16 at a time, a wave 64 columns.  With B as the
// first operand a lane holds 4 adjacent columns of one row; the wave turns the tile round in
// LDS, so that y and out are accessed in whole 128-byte lines (fp32: two), the fp32 sum
// rounded once.  ONE: the rank fits one step of 64, and B is read once for all the rows.
template <bool F32, int TERMS, bool NT, bool ONE>
__device__ __forceinline__ void lora_expand_rows(const LoraParams& p, int64_t t0, int id, int n, const int* list,
                                                 const uint16_t* vt, float* tiles, int c_begin, int c_end) {
  using T = std::conditional_t<F32, float, uint16_t>;
  constexpr int kPer = 16 / sizeof(T), kLanes = 64 / kPer;      // values per piece, pieces per row
  constexpr int kRows = 64 / kLanes, kPieces = 16 / kRows;      // rows per access, accesses per tile
  const int lane = lane_id(), wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
  const int pitch = lora_pitch(p.rank), yr = lane / kLanes, yc = (lane % kLanes) * kPer;
  const uint16_t* bm = p.b + static_cast<int64_t>(id) * p.n * p.rank;
  float* tile = tiles + wave * 16 * kLoraTilePitch;
  // every lane loads (past the last row or column a valid place again): a load under a
  // branch is waited for before the next one
  auto row_of = [&](int i0, int i, int u) __attribute__((always_inline)) {
    return t0 + list[min(i0 + 16 * i + kRows * u + yr, n - 1)];
  };
  auto load_y = [&](int col0, int i0, uint4 (&y)[2][kPieces]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int u = 0; u < kPieces; ++u)
        y[i][u] = lora_load<NT>(static_cast<const T*>(p.y) + row_of(i0, i, u) * p.y_stride + min(col0 + yc, c_end - kPer));
  };
  uint4 y[2][kPieces], y_next[2][kPieces];
  load_y(c_begin + 64 * wave, 0, y);
  for (int col0 = c_begin + 64 * wave; col0 < c_end; col0 += 64 * kLoraWaves) {
    const bool live = col0 + yc < c_end;  // c_end is a multiple of 8
    const uint16_t* br[4];
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) br[jt] = bm + static_cast<int64_t>(min(col0 + 16 * jt + m, c_end - 1)) * p.rank;
    bf16x8 b[2][4];
    auto load_b = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = min(k0 + 32 * h + 8 * g, p.rank - 8);  // past the rank v is 0
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) b[h][jt] = *reinterpret_cast<const bf16x8*>(br[jt] + k);
      }
    };
    if constexpr (ONE) load_b(0);
    for (int i0 = 0; i0 < n; i0 += 32) {
      // the next pair's y ahead of this one's stores, which a later load would wait for
      const bool more = i0 + 32 < n;
      load_y(more ? col0 : col0 + 64 * kLoraWaves, more ? i0 + 32 : 0, y_next);
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
        // the wave's own LDS accesses are done in order
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) *reinterpret_cast<f32x4*>(tile + m * kLoraTilePitch + 16 * jt + 4 * g) = acc[i][jt];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
          const f32x4* src = reinterpret_cast<const f32x4*>(tile + (kRows * u + yr) * kLoraTilePitch + yc);
          uint4 o;
          if constexpr (F32) {
            o = __builtin_bit_cast(uint4, __builtin_bit_cast(f32x4, y[i][u]) + src[0]);
          } else {
            const f32x4 lo = src[0], hi = src[1];
            auto add = [](uint32_t w, float c0, float c1) {
              return pack_bf16x2(__uint_as_float(w << 16) + c0, __uint_as_float(w & 0xffff0000u) + c1);
            };
            o = uint4{add(y[i][u].x, lo[0], lo[1]), add(y[i][u].y, lo[2], lo[3]), add(y[i][u].z, hi[0], hi[1]),
                      add(y[i][u].w, hi[2], hi[3])};
          }
          if (live && i0 + 16 * i + kRows * u + yr < n)
            lora_store<NT>(static_cast<T*>(p.out) + row_of(i0, i, u) * p.out_stride + col0 + yc, o);
        }
        __builtin_amdgcn_wave_barrier();
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int u = 0; u < kPieces; ++u) y[i][u] = y_next[i][u];
    }
  }
}

// out = y for the listed rows, eight 16-byte loads in flight per thread.
template <bool F32, bool NT>
__device__ __forceinline__ void lora_copy_rows(const LoraParams& p, int64_t t0, int n, const int* list, int c_begin, int c_end) {
  using T = std::conditional_t<F32, float, uint16_t>;
  constexpr int kPer = 16 / sizeof(T), kFlight = 8, kThreads = kLoraWaves * 64;
  const int chunks = (c_end - c_begin) / kPer, total = n * chunks;
  for (int e0 = threadIdx.x; e0 < total; e0 += kFlight * kThreads) {
    uint4 v[kFlight];
    auto at = [&](int e, int64_t stride) __attribute__((always_inline)) {
      const int i = e / chunks;
      return (t0 + list[i]) * stride + c_begin + (e - i * chunks) * kPer;
    };
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      v[u] = lora_load<NT>(static_cast<const T*>(p.y) + at(min(e0 + u * kThreads, total - 1), p.y_stride));
    }
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const int e = e0 + u * kThreads;
      if (e < total) lora_store<NT>(static_cast<T*>(p.out) + at(e, p.out_stride), v[u]);
    }
  }
}

// grid: (row blocks, parts of a block's adapters, column parts), or (items, 1, column parts).  The rows without an
// adapter are a group of their own, copied unless out is y.
template <bool F32, int TERMS, bool NT>
__global__ __launch_bounds__(kLoraWaves * 64, F32 ? 2 : 3) void lora_expand_kernel(LoraParams p) {
  extern __shared__ __align__(16) float tiles[];  // [waves][16][pitch], then v's terms
  uint16_t* vt = reinterpret_cast<uint16_t*>(tiles + kLoraWaves * 16 * kLoraTilePitch);  // [TERMS][kRowsBlock][pitch]
  __shared__ int list[kRowsBlock];
  const int c_begin = blockIdx.z * p.cols_per_wg, c_end = min(c_begin + p.cols_per_wg, p.n);
  lora_groups(p, p.y != p.out, list, [&](int gid, int n, int64_t t0) {
    if (gid < 0) {
      lora_copy_rows<F32, NT>(p, t0, n, list, c_begin, c_end);
      return;
    }
    // v of the rows, the splits summed in order and scaled, as bf16 terms; 0 past the rank
    const int pitch = lora_pitch(p.rank), quads = (pitch - kLoraPad) / 4;
    const float c = p.scaling != nullptr ? p.scaling[gid] : 1.0f;
    // kEach quads and kMany splits per thread with their loads in flight together (one quad at a
    // time: 8192 rows, 7168 -> 64 -> 4096, 83.4 us a call, so 81.9)
    auto stage = [&](auto each, auto many) __attribute__((always_inline)) {
      constexpr int kEach = decltype(each)::value, kMany = decltype(many)::value, kThreads = kLoraWaves * 64;
      const int total = n * quads;
      for (int e0 = threadIdx.x; e0 < total; e0 += kEach * kThreads) {
        f32x4 v[kEach] = {};
        const float* src[kEach];
        int at[kEach], r[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
          const int e = min(e0 + k * kThreads, total - 1);  // past the end the last one again
          at[k] = e / quads;
          r[k] = 4 * (e - at[k] * quads);
          src[k] = p.v + (t0 + list[at[k]]) * p.rank + min(r[k], p.rank - 4);
        }
        for (int s = 0; s < p.splits; s += kMany) {
          f32x4 part[kEach][kMany];
#pragma unroll
          for (int u = 0; u < kMany; ++u)
#pragma unroll
            for (int k = 0; k < kEach; ++k)
              part[k][u] = *reinterpret_cast<const f32x4*>(src[k] + min(s + u, p.splits - 1) * p.rows * p.rank);
#pragma unroll
          for (int u = 0; u < kMany; ++u)
#pragma unroll
            for (int k = 0; k < kEach; ++k)
              if (s + u < p.splits) v[k] += part[k][u];
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
          v[k] *= c;
          if (r[k] >= p.rank) v[k] = f32x4{0.f, 0.f, 0.f, 0.f};
          uint16_t t16[4][TERMS];
#pragma unroll
          for (int u = 0; u < 4; ++u) split_bf16<TERMS>(v[k][u], t16[u]);
#pragma unroll
          for (int q = 0; q < TERMS; ++q)
            *reinterpret_cast<uint2*>(vt + (q * kRowsBlock + at[k]) * pitch + r[k]) =
                uint2{t16[0][q] | static_cast<uint32_t>(t16[1][q]) << 16, t16[2][q] | static_cast<uint32_t>(t16[3][q]) << 16};
        }
      }
    };
    if (p.splits == 1) stage(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
    else if (p.splits <= 4) stage(std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
    else stage(std::integral_constant<int, 2>{}, std::integral_constant<int, 8>{});
    __syncthreads();
    if (p.rank <= 64)
      lora_expand_rows<F32, TERMS, NT, true>(p, t0, gid, n, list, vt, tiles, c_begin, c_end);
    else
      lora_expand_rows<F32, TERMS, NT, false>(p, t0, gid, n, list, vt, tiles, c_begin, c_end);
  });
}

// Few rows: one workgroup per row and 256 CPT columns, CPT columns per thread, plain fp32
// products (v needs no terms).  What bounds a handful of rows is the chain of memory accesses
// and the instructions between them, and here two accesses follow the row's id: v, B and y
// together, then the store.  Each row reads its adapter's B, from the L2s where rows share it.
constexpr int kLoraSmallRank = 64;  // CPT columns take ranks up to 64 / CPT
template <bool F32, int CPT>
__global__ __launch_bounds__(256) void lora_expand_small_kernel(LoraParams p) {
  using T = std::conditional_t<F32, float, uint16_t>;
  constexpr int kChunks = kLoraSmallRank / 8 / CPT;  // of 8 ranks
  __shared__ __align__(16) float vs[kLoraSmallRank];
  const int64_t t = blockIdx.x;
  const int c0 = blockIdx.y * 256 * CPT + threadIdx.x;
  const int id = p.ids[t];
  const T* yr = static_cast<const T*>(p.y) + t * p.y_stride;
  T* out = static_cast<T*>(p.out) + t * p.out_stride;
  T y[CPT];
#pragma unroll
  for (int c = 0; c < CPT; ++c) y[c] = yr[min(c0 + 256 * c, p.n - 1)];
  if (id < 0 || id >= p.adapters) {
#pragma unroll
    for (int c = 0; c < CPT; ++c)
      if (p.y != p.out && c0 + 256 * c < p.n) out[c0 + 256 * c] = y[c];
    return;
  }
  uint4 b[CPT][kChunks];
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    const uint16_t* br = p.b + (static_cast<int64_t>(id) * p.n + min(c0 + 256 * c, p.n - 1)) * p.rank;
#pragma unroll
    for (int k = 0; k < kChunks; ++k)
      if (8 * k < p.rank) b[c][k] = *reinterpret_cast<const uint4*>(br + 8 * k);
  }
  if (static_cast<int>(threadIdx.x) < p.rank) {
    const float* src = p.v + t * p.rank + threadIdx.x;
    float v = 0.0f;
    for (int s = 0; s < p.splits; s += 8) {
      float part[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) part[u] = src[min(s + u, p.splits - 1) * p.rows * p.rank];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (s + u < p.splits) v += part[u];
    }
    vs[threadIdx.x] = p.scaling != nullptr ? v * p.scaling[id] : v;
  }
  __syncthreads();
  float d[CPT] = {};
#pragma unroll
  for (int k = 0; k < kChunks; ++k) {
    if (8 * k < p.rank) {
#pragma unroll
      for (int c = 0; c < CPT; ++c) {
        const uint32_t w[4] = {b[c][k].x, b[c][k].y, b[c][k].z, b[c][k].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          d[c] = __builtin_fmaf(vs[8 * k + 2 * e], __uint_as_float(w[e] << 16), d[c]);
          d[c] = __builtin_fmaf(vs[8 * k + 2 * e + 1], __uint_as_float(w[e] & 0xffff0000u), d[c]);
        }
      }
    }
  }
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    if (c0 + 256 * c >= p.n) continue;
    if constexpr (F32) out[c0 + 256 * c] = y[c] + d[c];
    else out[c0 + 256 * c] = static_cast<uint16_t>(bf16_rne_bits(bf16_bits_to_f32(y[c]) + d[c]));
  }
}

}  // namespace hkmoe
