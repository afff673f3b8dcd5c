// Dense product of e4m3 operands to fp32's own precision, with an epilogue: C[M,N] =
// act((sa*sb) A[M,K] . B[N,K]^T + bias) + residual, fp32 C, per-tensor scales or MX exponents
// (epilogue.hpp says why the products run in bf16).  For more rows than the strips of
// gemm_skinny.hpp take.
//
// 128x128 output tiles and the LDS ring of gemm_small.hpp: e4m3 in LDS, widened in registers,
// so LDS carries half the bytes of a bf16 product.  8 waves of 64x32 outputs, two per SIMD:
// two 32x32 blocks, each eight v_mfma_f32_32x32x16_bf16 a K step, with six conversions per MFMA.
// Those fit behind 32x32x16 (7.9 ns per 16x16x32 of work, two waves per SIMD, against 6.9 without
// any) and not behind 16x16x32 (9.3 against 7.3).  The conversions of the next 16 K run beside
// the MFMAs of this one, the LDS reads of step kt+1 beside step kt.
// Where they fill the chip, 256x128 tiles (gemm_fp8_wide256): waves of 64x64, four conversions per MFMA and
// a third less from LDS.  us, 128x128 / 256x128 tiles, a residual, both at once in one run: 1777x4096x2048
// 41.5 / 37.4, 2048x4096x4096 67.8 / 61.7, 8192x4096x7168 426 / 385 (1.25 PFLOP/s; a bf16 library
// product 1.4), MX 478 / 410; with half the tiles of a round 1024x4096x4096 36.2 / 52.6.  The
// chip's power takes its part: 8192x4096x7168 on 128x128 tiles took 350 with operands of ones for 418.
// 4 waves of 64x64 outputs on 128x128 tiles and 16x16x32 MFMAs came to 1.05 PFLOP/s where this kernel had 1.09.
#pragma once

#include "gemm_small.hpp"

namespace hkmoe {

static_assert(kSmTile * kSmTile * 4 <= sm_lds_bytes(false), "the output tile is staged in the ring");

template <bool MX>
__global__ __launch_bounds__(kSmThreads, 2) void gemm_fp8_wide(SmallGemmParams p) {
  constexpr int kStg = sm_stage_bytes(MX);
  constexpr int kLoads = MX ? 5 : 4;  // vector-memory instructions per wave and step
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, l32 = lane & 31, g32 = lane >> 5;
  const int wm = wave >> 2, wn = wave & 3;  // the wave's 64 rows and 32 columns
  const int fx = swz(l32);

  // tile of this workgroup, as in gemm_small.hpp
  const int g = gridDim.x;
  const int vid = (g & 7) == 0 ? (blockIdx.x & 7) * (g >> 3) + (blockIdx.x >> 3) : blockIdx.x;
  const int blk = vid >> 5, sl = vid & 31;
  const int mt = (blk / p.nbn) * 4 + (sl & 3), nt = (blk % p.nbn) * 8 + (sl >> 2);
  if (mt >= p.m_tiles || nt >= p.n_tiles) return;
  const int m0 = mt * kSmTile, n0 = nt * kSmTile;
  const int k_steps = p.k / kBK;

  // DMA as in gemm_small.hpp: instruction i of wave w fills LDS rows 64i + 8w + lane/8 of an
  // operand tile, swizzled; A rows past M repeat row M-1 (never stored).  MX: waves 0, 1 fetch the
  // words of A's 64-row groups (one past the padded rows repeats the last), 2, 3 B's, 4-7 repeat them.
  const int ld_row = 8 * wave + (lane >> 3);
  const int ld_chunk = (lane & 7) ^ swz(ld_row);
  const i32x4 a_srd = make_srd(p.a, p.a_bytes);
  const i32x4 b_srd = make_srd(p.b, p.b_bytes);
  int a_voff[2], b_voff[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    a_voff[i] = buf_off(min(m0 + 64 * i + ld_row, p.m - 1), p.k, ld_chunk * 16);
    b_voff[i] = buf_off(n0 + 64 * i + ld_row, p.k, ld_chunk * 16);
  }
  const int ww = wave & 3;
  const i32x4 w_srd = make_srd(ww < 2 ? p.a_scale : p.b_scale, 0xffffffffu);
  const int w_voff = ((ww < 2 ? min(m0 + 64 * ww, p.m64 - 64) : n0 + 64 * (ww - 2)) + lane) * 4;
  const int w_step = (ww < 2 ? p.m64 : p.n) * 4;
  auto issue = [&](int kt) __attribute__((always_inline)) {
    uint8_t* st = smem + (kt % kSmStages) * kStg;
    if constexpr (MX) load_lds_4B(w_srd, st + kSmStageBytes + ww * 256, w_voff, buf_off(kt, w_step, 0));
#pragma unroll
    for (int i = 0; i < 2; ++i) load_lds_16B(a_srd, st + (64 * i + 8 * wave) * kBK, a_voff[i], kt * kBK);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      load_lds_16B(b_srd, st + kSmOperandBytes + (64 * i + 8 * wave) * kBK, b_voff[i], kt * kBK);
  };

  // Fragments of a step: a[2i + h] bytes 64h + 32g32 .. +31 of row 64wm + 32i + l32, b[h] of column
  // 32wn + l32; MX: block 2h + g32, whose exponents are bytes 2i + l32/16 (columns: 2(wn % 2) + l32/16)
  // of word 16(2h + g32) + l32 % 16 of the 64-row group.
  struct Step {
    i32x8 a[4], b[2];
    int wa[2], wb[2];
  };
  const int sh_a = 8 * (l32 >> 4), sh_b = sh_a + 16 * (wn & 1);
  auto read_a = [&](const uint8_t* st, int i, int h, Step& s) __attribute__((always_inline)) {
    s.a[2 * i + h] = read_frag(st, 64 * wm + 32 * i + l32, 2 * h + g32, fx);
  };
  auto read_b = [&](const uint8_t* st, int h, Step& s) __attribute__((always_inline)) {
    if constexpr (MX) {
      const int32_t* words = reinterpret_cast<const int32_t*>(st + kSmStageBytes) + 16 * (2 * h + g32) + (l32 & 15);
      s.wa[h] = words[wm * 64];
      s.wb[h] = words[kSmTile + (wn >> 1) * 64];
    }
    s.b[h] = read_frag(st + kSmOperandBytes, 32 * wn + l32, 2 * h + g32, fx);
  };
  auto read = [&](int kt, Step& s) __attribute__((always_inline)) {
    const uint8_t* st = smem + (kt % kSmStages) * kStg;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      read_b(st, h, s);
      read_a(st, 0, h, s);
      read_a(st, 1, h, s);
    }
  };
  // A step's fragments have landed by the wait in front of the next step's reads; without this the
  // compiler, which does not see that wait, waits for those reads as well.
  auto landed = [&](Step& s) __attribute__((always_inline)) {
    asm volatile("" : "+v"(s.a[0]), "+v"(s.a[1]), "+v"(s.a[2]), "+v"(s.a[3]), "+v"(s.b[0]), "+v"(s.b[1]));
    if constexpr (MX) asm volatile("" : "+v"(s.wa[0]), "+v"(s.wa[1]), "+v"(s.wb[0]), "+v"(s.wb[1]));
  };

  f32x16 acc[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  struct Ops {
    bf16x8_t b, a0, a1;
  };
  auto conv = [&](const Step& s, int t) __attribute__((always_inline)) -> Ops {
    const int h = t >> 2, q = t & 3;  // K bytes 8q .. 8q + 7 of half h's 32
    const float sb = MX ? e8m0_scale<0>(s.wb[h] >> sh_b) : 1.0f, s0 = MX ? e8m0_scale<0>(s.wa[h] >> sh_a) : 1.0f,
                s1 = MX ? e8m0_scale<2>(s.wa[h] >> sh_a) : 1.0f;
    return Ops{widen8(s.b[h][2 * q], s.b[h][2 * q + 1], sb), widen8(s.a[h][2 * q], s.a[h][2 * q + 1], s0),
               widen8(s.a[2 + h][2 * q], s.a[2 + h][2 * q + 1], s1)};
  };
  // K 16t .. 16t + 15 of step s (o: its operands; left: the next ones)
  auto mma_at = [&](const Step& s, int t, Ops& o) __attribute__((always_inline)) {
    const Ops n = t < 7 ? conv(s, t + 1) : o;
    acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(o.b, o.a0, acc[0], 0, 0, 0);
    acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(o.b, o.a1, acc[1], 0, 0, 0);
    o = n;
  };
  auto mma = [&](const Step& s) __attribute__((always_inline)) {
    Ops o = conv(s, 0);
#pragma unroll
    for (int t = 0; t < 8; ++t) mma_at(s, t, o);
  };

  // The schedule of gemm_small.hpp: step kt's MFMAs beside the reads of kt+1 and the DMA of kt+3.
  const int pre = min(kSmAhead, k_steps);
  for (int kt = 0; kt < pre; ++kt) issue(kt);
  small_wait_stage<kLoads>(pre - 1);
  Step s0, s1;
  read(0, s0);
  auto step = [&](int kt, Step& cur, Step& next) __attribute__((always_inline)) {
    if (kt + kSmAhead < k_steps) issue(kt + kSmAhead);
    small_wait_stage<kLoads>(min(kSmAhead - 1, k_steps - 1 - (kt + 1)));
    landed(cur);
    read(kt + 1, next);
    __builtin_amdgcn_sched_barrier(0);
    mma(cur);
    __builtin_amdgcn_sched_barrier(0);
  };
  // Steady state: a third of the reads in front of each of the first three quarters of the MFMAs (all in
  // front, they hold up the first MFMAs: 38.2 against 37.3 us for 1777x4096x2048).
  auto step_full = [&](int kt, Step& cur, Step& next) __attribute__((always_inline)) {
    issue(kt + kSmAhead);
    small_wait_stage<kLoads>(kSmAhead - 1);
    landed(cur);
    const uint8_t* st = smem + ((kt + 1) % kSmStages) * kStg;
    Ops o = conv(cur, 0);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      __builtin_amdgcn_sched_barrier(0);
      if (q == 0) read_b(st, 0, next), read_a(st, 0, 0, next);
      if (q == 1) read_a(st, 1, 0, next), read_b(st, 1, next);
      if (q == 2) read_a(st, 0, 1, next), read_a(st, 1, 1, next);
      __builtin_amdgcn_sched_barrier(0);
      mma_at(cur, 2 * q, o);
      mma_at(cur, 2 * q + 1, o);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  int kt = 0;
  for (; kt + 1 + kSmAhead < k_steps; kt += 2) {
    step_full(kt, s0, s1);
    step_full(kt + 1, s1, s0);
  }
  for (; kt + 2 < k_steps; kt += 2) {
    step(kt, s0, s1);
    step(kt + 1, s1, s0);
  }

  // The output goes through LDS and is stored as whole rows (thread: 16-byte chunks tid + 512u of the
  // tile's rows of 32), and so is the residual loaded, in front of the last products, into the
  // registers of the next fragments.  Rows past M repeat the last one and are not stored.
  constexpr int kChunks = kSmTile * 32 / kSmThreads;
  f32x4 res[kChunks];
  const bool has_res = p.epi.residual != nullptr;
  auto load_res = [&]() __attribute__((always_inline)) {
    if (!has_res) return;
#pragma unroll
    for (int u = 0; u < kChunks; ++u) {
      const int idx = tid + kSmThreads * u, r = min(m0 + (idx >> 5), p.m - 1), c = idx & 31;
      res[u] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(static_cast<const float*>(p.epi.residual) +
                                                                         static_cast<int64_t>(r) * p.n + n0 + c * 4));
    }
  };
  if (kt + 1 < k_steps) {
    step(kt, s0, s1);
    load_res();
    mma(s1);
  } else {
    load_res();
    mma(s0);
  }

  // lane: row 64wm + 32i + l32, columns 32wn + 8j + 4g32 .. +3 in registers 4j .. 4j+3 of acc[i]; chunk c of
  // LDS row r at c ^ (r % 32)
  const float tens = MX ? 1.0f : (p.a_scale ? p.a_scale[0] : 1.0f) * (p.b_scale ? p.b_scale[0] : 1.0f);
  __syncthreads();  // every wave is done with the ring
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f32x4 bias = epilogue_bias(p.epi, n0 + 32 * wn + 8 * j + 4 * g32);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 64 * wm + 32 * i + l32, c = 8 * wn + 2 * j + g32;
      const f32x4 v{acc[i][4 * j] * tens, acc[i][4 * j + 1] * tens, acc[i][4 * j + 2] * tens, acc[i][4 * j + 3] * tens};
      *reinterpret_cast<f32x4*>(smem + r * 512 + ((c ^ (r & 31)) << 4)) = activate(v + bias, p.epi.act);
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    const int idx = tid + kSmThreads * u, r = idx >> 5, c = idx & 31;
    f32x4 v = *reinterpret_cast<const f32x4*>(smem + r * 512 + ((c ^ (r & 31)) << 4));
    if (has_res) v = v + res[u];
    if (m0 + r < p.m)
      __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(static_cast<float*>(p.c) + static_cast<int64_t>(m0 + r) * p.n + n0 + c * 4));
  }
}

// ---------------------------------------------------------------------------
// The same on 256x128 tiles.  A wave's fragments of a whole step, twice, beside its 64 sums a lane would not fit
// its registers, so the two halves of a step take turns: one is read while the other's products run.
// Three ring stages; a step's slot is free for the step after the next two when every wave has read
// its second half, in the middle of the step.
// ---------------------------------------------------------------------------
constexpr int kWbRows = 256, kWbStages = 3;
constexpr int kWbOperandBytes = kWbRows * kBK + kSmOperandBytes;  // A, then B
constexpr int wb_stage_bytes(bool mx) { return kWbOperandBytes + (mx ? (kWbRows + kSmTile) * 4 : 0); }
constexpr int wb_lds_bytes(bool mx) { return kWbStages * wb_stage_bytes(mx); }  // 144 KiB (148.5)
static_assert(wb_lds_bytes(true) <= 160 * 1024 && kWbRows * kSmTile * 4 <= wb_lds_bytes(false), "LDS budget");

template <bool MX>
__global__ __launch_bounds__(kSmThreads, 2) void gemm_fp8_wide256(SmallGemmParams p) {
  constexpr int kStg = wb_stage_bytes(MX);
  constexpr int kLoads = MX ? 7 : 6;  // vector-memory instructions per wave and step
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, l32 = lane & 31, g32 = lane >> 5;
  const int wm = wave >> 1, wn = wave & 1;  // the wave's 64 rows and 64 columns
  const int fx = swz(l32);

  // tile of this workgroup, as in gemm_small.hpp
  const int g = gridDim.x;
  const int vid = (g & 7) == 0 ? (blockIdx.x & 7) * (g >> 3) + (blockIdx.x >> 3) : blockIdx.x;
  const int blk = vid >> 5, sl = vid & 31;
  const int mt = (blk / p.nbn) * 4 + (sl & 3), nt = (blk % p.nbn) * 8 + (sl >> 2);
  if (mt >= p.m_tiles || nt >= p.n_tiles) return;
  const int m0 = mt * kWbRows, n0 = nt * kSmTile;
  const int k_steps = p.k / kBK;

  // DMA as above; MX: waves 0-3 fetch the words of A's 64-row groups, 4 and 5 B's, 6 and 7 repeat B's
  const int ld_row = 8 * wave + (lane >> 3);
  const int ld_chunk = (lane & 7) ^ swz(ld_row);
  const i32x4 a_srd = make_srd(p.a, p.a_bytes);
  const i32x4 b_srd = make_srd(p.b, p.b_bytes);
  int a_voff[4], b_voff[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) a_voff[i] = buf_off(min(m0 + 64 * i + ld_row, p.m - 1), p.k, ld_chunk * 16);
#pragma unroll
  for (int i = 0; i < 2; ++i) b_voff[i] = buf_off(n0 + 64 * i + ld_row, p.k, ld_chunk * 16);
  const int ww = wave < 6 ? wave : wave - 2;
  const i32x4 w_srd = make_srd(ww < 4 ? p.a_scale : p.b_scale, 0xffffffffu);
  const int w_voff = ((ww < 4 ? min(m0 + 64 * ww, p.m64 - 64) : n0 + 64 * (ww - 4)) + lane) * 4;
  const int w_step = (ww < 4 ? p.m64 : p.n) * 4;
  auto stage = [&](int kt) __attribute__((always_inline)) -> uint8_t* { return smem + (kt % kWbStages) * kStg; };
  auto issue = [&](int kt) __attribute__((always_inline)) {
    uint8_t* st = stage(kt);
    if constexpr (MX) load_lds_4B(w_srd, st + kWbOperandBytes + ww * 256, w_voff, buf_off(kt, w_step, 0));
#pragma unroll
    for (int i = 0; i < 4; ++i) load_lds_16B(a_srd, st + (64 * i + 8 * wave) * kBK, a_voff[i], kt * kBK);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      load_lds_16B(b_srd, st + kWbRows * kBK + (64 * i + 8 * wave) * kBK, b_voff[i], kt * kBK);
  };

  // Fragments of half a step: bytes 64h + 32g32 .. +31 of rows 64wm + 32i + l32 and of columns 64wn + 32i +
  // l32; MX: block 2h + g32, exponents in bytes 2i + l32/16 of the groups' words 16(2h + g32) + l32 % 16.
  struct Half {
    i32x8 a[2], b[2];
    int wa, wb;
  };
  const int sh = 8 * (l32 >> 4);
  auto read = [&](const uint8_t* st, int h, Half& s) __attribute__((always_inline)) {
    if constexpr (MX) {
      const int32_t* words = reinterpret_cast<const int32_t*>(st + kWbOperandBytes) + 16 * (2 * h + g32) + (l32 & 15);
      s.wa = words[wm * 64];
      s.wb = words[kWbRows + wn * 64];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s.b[i] = read_frag(st + kWbRows * kBK, 64 * wn + 32 * i + l32, 2 * h + g32, fx);
      s.a[i] = read_frag(st, 64 * wm + 32 * i + l32, 2 * h + g32, fx);
    }
  };
  auto landed = [&](Half& s) __attribute__((always_inline)) {
    asm volatile("" : "+v"(s.a[0]), "+v"(s.a[1]), "+v"(s.b[0]), "+v"(s.b[1]));
    if constexpr (MX) asm volatile("" : "+v"(s.wa), "+v"(s.wb));
  };

  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i >> 1][i & 1][r] = 0.f;
  struct Ops {
    bf16x8_t a[2], b[2];
  };
  auto conv = [&](const Half& s, int q) __attribute__((always_inline)) -> Ops {  // K bytes 8q .. 8q + 7 of its 32
    const float a0 = MX ? e8m0_scale<0>(s.wa >> sh) : 1.0f, a1 = MX ? e8m0_scale<2>(s.wa >> sh) : 1.0f;
    const float b0 = MX ? e8m0_scale<0>(s.wb >> sh) : 1.0f, b1 = MX ? e8m0_scale<2>(s.wb >> sh) : 1.0f;
    Ops o;
    o.a[0] = widen8(s.a[0][2 * q], s.a[0][2 * q + 1], a0);
    o.b[0] = widen8(s.b[0][2 * q], s.b[0][2 * q + 1], b0);
    o.a[1] = widen8(s.a[1][2 * q], s.a[1][2 * q + 1], a1);
    o.b[1] = widen8(s.b[1][2 * q], s.b[1][2 * q + 1], b1);
    return o;
  };
  auto mma = [&](const Half& s) __attribute__((always_inline)) {
    Ops o = conv(s, 0);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const Ops n = q < 3 ? conv(s, q + 1) : o;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(o.b[j], o.a[i], acc[i][j], 0, 0, 0);
      o = n;
    }
  };

  // Step kt: its second half is read beside the first one's products; then, with the next stage landed
  // and this one read by every wave, its slot takes step kt + 3, and the next step's first half is read
  // beside the second one's products.
  const int pre = min(kWbStages, k_steps);
  for (int kt = 0; kt < pre; ++kt) issue(kt);
  small_wait_stage<kLoads>(pre - 1);
  Half h0, h1;
  read(stage(0), 0, h0);
  auto step = [&](int kt, auto&& beside) __attribute__((always_inline)) {
    landed(h0);
    read(stage(kt), 1, h1);
    __builtin_amdgcn_sched_barrier(0);
    mma(h0);
    __builtin_amdgcn_sched_barrier(0);
    small_wait_stage<kLoads>(min(kWbStages - 2, k_steps - 2 - kt));
    if (kt + kWbStages < k_steps) issue(kt + kWbStages);
    landed(h1);
    read(stage(kt + 1), 0, h0);
    beside();
    __builtin_amdgcn_sched_barrier(0);
    mma(h1);
    __builtin_amdgcn_sched_barrier(0);
  };
  int kt = 0;
  for (; kt + 2 < k_steps; ++kt) step(kt, [] {});

  // The output through LDS as whole rows, as above; the residual is loaded after the last wait for a stage.
  constexpr int kChunks = kWbRows * 32 / kSmThreads;
  f32x4 res[kChunks];
  const bool has_res = p.epi.residual != nullptr;
  auto load_res = [&]() __attribute__((always_inline)) {
    if (!has_res) return;
#pragma unroll
    for (int u = 0; u < kChunks; ++u) {
      const int idx = tid + kSmThreads * u, r = min(m0 + (idx >> 5), p.m - 1), c = idx & 31;
      res[u] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(static_cast<const float*>(p.epi.residual) +
                                                                         static_cast<int64_t>(r) * p.n + n0 + c * 4));
    }
  };
  if (k_steps > 1)
    step(kt, load_res);
  else
    load_res();
  read(stage(k_steps - 1), 1, h1);
  mma(h0);
  mma(h1);

  // lane: row 64wm + 32i + l32, columns 64wn + 32j + 8q + 4g32 .. +3 in registers 4q .. 4q+3 of acc[i][j]
  const float tens = MX ? 1.0f : (p.a_scale ? p.a_scale[0] : 1.0f) * (p.b_scale ? p.b_scale[0] : 1.0f);
  __syncthreads();  // every wave is done with the ring
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 bias = epilogue_bias(p.epi, n0 + 64 * wn + 32 * j + 8 * q + 4 * g32);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 64 * wm + 32 * i + l32, c = 16 * wn + 8 * j + 2 * q + g32;
        const f32x16& a = acc[i][j];
        const f32x4 v{a[4 * q] * tens, a[4 * q + 1] * tens, a[4 * q + 2] * tens, a[4 * q + 3] * tens};
        *reinterpret_cast<f32x4*>(smem + r * 512 + ((c ^ (r & 31)) << 4)) = activate(v + bias, p.epi.act);
      }
    }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    const int idx = tid + kSmThreads * u, r = idx >> 5, c = idx & 31;
    f32x4 v = *reinterpret_cast<const f32x4*>(smem + r * 512 + ((c ^ (r & 31)) << 4));
    if (has_res) v = v + res[u];
    if (m0 + r < p.m)
      __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(static_cast<float*>(p.c) + static_cast<int64_t>(m0 + r) * p.n + n0 + c * 4));
  }
}

}  // namespace hkmoe
