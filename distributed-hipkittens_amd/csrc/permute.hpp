// Tokens sorted by expert and back, with the gradients of both ways, and the gradient
// of the router's weights to its logits.
//
// A slot is a token's j-th expert, f = t k + j of T k; its expert is ids[f], and ids
// outside [0, E) have none here (padding, an expert on another device).  The order is a
// stable sort of the slots by expert with the slots of no expert behind the last:
//   perm[p] = f, inv[f] = p, offsets[e] = first place of expert e, offsets[E] = places in use
//   xp[p] = x[perm[p] / k], 0 for p >= offsets[E]
//   dx[t] = rnd(sum_j dxp[inv[t,j]])             over the slots in use
//   out[t] = rnd(sum_j w[t,j] y[inv[t,j]])       over the slots in use, j ascending
//   dy[p] = rnd(w[f] dout[f / k]), 0 behind the last;  dw[t,j] = sum_h dout[t,h] y[inv[t,j],h]
//   dl[t,e] = sum_{j: idx[t,j] = e} w_j (dw_j - sum_i w_i dw_i)
//
// All of it is bound by HBM (rows of H values, read once and written once), but for
// decode-sized batches, which are bound by launches.  The rows are moved a token at a time: the
// token's row is read once and written to its k places (or its k rows read and one
// written), whole 16-byte chunks, non-temporal where nothing reads them soon.
#pragma once

#include "layer_norm.hpp"

namespace hkmoe {

constexpr int kSortThreads = 256;
constexpr int kSortSlots = 1024;   // slots that a sorting workgroup takes at a time
constexpr int kSortBlocks = 256;   // sorting workgroups, at most
constexpr int kMoveThreads = 512;  // of a workgroup that moves a token's rows, at most

__device__ __forceinline__ int sort_key(int id, int experts) {
  return static_cast<unsigned>(id) < static_cast<unsigned>(experts) ? id : experts;
}

// A workgroup's slots: `span` of them (a multiple of kSortSlots, so that kSortBlocks
// workgroups are enough).  Their counts[block][E + 1].
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const int32_t* __restrict__ ids, int64_t slots,
                                                                  int64_t span, int experts,
                                                                  int32_t* __restrict__ counts) {
  __shared__ int hist[kMaxExperts + 1];
  for (int e = threadIdx.x; e <= experts; e += kSortThreads) hist[e] = 0;
  __syncthreads();
  const int64_t f0 = blockIdx.x * span, f1 = f0 + span < slots ? f0 + span : slots;
#pragma unroll 4
  for (int64_t f = f0 + threadIdx.x; f < f1; f += kSortThreads) atomicAdd(&hist[sort_key(ids[f], experts)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= experts; e += kSortThreads)
    counts[static_cast<int64_t>(blockIdx.x) * (experts + 1) + e] = hist[e];
}

// Exclusive scan of one value per thread over kSortThreads threads.
__device__ __forceinline__ int sort_scan(int v, int* wave_tot) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int n = __shfl_up(incl, o, 64);
    if (lane >= o) incl += n;
  }
  if (lane == 63) wave_tot[wave] = incl;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int w = 0; w < kSortThreads / 64; ++w)
    if (w < wave) before += wave_tot[w];
  return before + incl - v;
}

// Places of a workgroup's slots.  Every workgroup adds up the counts by itself (at most
// kSortBlocks x E ints from L2), which costs less than a launch that does it for all.  Then
// kSortSlots at a time: a wave takes 256 of them in order, 64 at a time; lanes of equal
// expert find each other by a ballot per bit of the expert.
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(const int32_t* __restrict__ ids, int64_t slots,
                                                                  int64_t span, int experts,
                                                                  const int32_t* __restrict__ counts, int blocks,
                                                                  int32_t* __restrict__ offsets,
                                                                  int32_t* __restrict__ perm, int32_t* __restrict__ inv) {
  constexpr int kWaves = kSortThreads / 64, kPer = (kMaxExperts + kSortThreads) / kSortThreads;  // experts a thread
  constexpr int kTurns = kSortSlots / kSortThreads;
  __shared__ int at[kWaves][kMaxExperts + 1];  // a wave's next place of each expert
  __shared__ int base[kMaxExperts + 1];        // the next place of each expert
  __shared__ int wave_tot[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = experts + 1;
  {
    // thread: experts tid * per .. + per - 1
    const int per = (n + kSortThreads - 1) / kSortThreads;
    int total[kPer], before[kPer], mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = tid * per + i;
      total[i] = before[i] = 0;
      if (i < per && e < n) {
        const int own = blockIdx.x;
#pragma unroll 32
        for (int b = 0; b < blocks; ++b) {
          const int c = counts[static_cast<int64_t>(b) * n + e];
          before[i] += b < own ? c : 0;
          total[i] += c;
        }
      }
      mine += total[i];
    }
    int first = sort_scan(mine, wave_tot);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = tid * per + i;
      if (i < per && e < n) {
        if (blockIdx.x == 0) offsets[e] = first;
        base[e] = first + before[i];
        first += total[i];
      }
    }
  }
  const int bits = 32 - __builtin_clz(static_cast<unsigned>(experts));  // of the largest key
  const int64_t s0 = blockIdx.x * span, s1 = s0 + span < slots ? s0 + span : slots;
  for (int64_t c0 = s0; c0 < s1; c0 += kSortSlots) {
    for (int e = tid; e < n; e += kSortThreads) {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) at[w][e] = 0;
    }
    __syncthreads();
    const int64_t f0 = c0 + wave * (kSortSlots / kWaves) + lane;
    int key[kTurns];
#pragma unroll
    for (int u = 0; u < kTurns; ++u) key[u] = f0 + u * 64 < s1 ? sort_key(ids[f0 + u * 64], experts) : -1;
#pragma unroll
    for (int u = 0; u < kTurns; ++u)
      if (key[u] >= 0) atomicAdd(&at[wave][key[u]], 1);
    __syncthreads();
    for (int e = tid; e < n; e += kSortThreads) {
      int next = base[e];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const int c = at[w][e];
        at[w][e] = next;
        next += c;
      }
      base[e] = next;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
      uint64_t same = __ballot(key[u] >= 0);
      for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot((key[u] >> b) & 1);
        same &= (key[u] >> b) & 1 ? set : ~set;
      }
      if (key[u] >= 0) {
        const int p = at[wave][key[u]] + __popcll(same & ((uint64_t{1} << lane) - 1));
        perm[p] = static_cast<int32_t>(f0 + u * 64);
        inv[f0 + u * 64] = p;
        // the last of the equal lanes moves the place on, after all of them have read it
        __builtin_amdgcn_wave_barrier();
        if ((same >> lane) == 1) at[wave][key[u]] = p + 1;
      }
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
  }
}

// Small batches in one launch.  Workgroup (t, part) takes `each` slots of token t: it compares every slot's
// expert with theirs, which gives their places, and copies the token's row there; the last workgroup
// writes the offsets.
// N: slots whose places one pass over the ids counts (1 where a workgroup has one: 64 tokens x 8, rows of
// 8 KiB 3.4 us in a graph, with 4 4.4).
constexpr int kSortAtOnce = 4;
template <int N>
__global__ __launch_bounds__(kSortThreads) void permute_small_kernel(const int32_t* __restrict__ ids, int slots, int experts,
                                                                     int top_k, int parts, const uint8_t* __restrict__ x,
                                                                     int64_t row_bytes, uint8_t* __restrict__ xp,
                                                                     int32_t* __restrict__ offsets,
                                                                     int32_t* __restrict__ perm, int32_t* __restrict__ inv) {
  __shared__ int red[kSortThreads / 64][N];
  const int tid = threadIdx.x;
  if (blockIdx.x == gridDim.x - 1) {
    constexpr int kPer = (kMaxExperts + kSortThreads) / kSortThreads;
    __shared__ int hist[kMaxExperts + 1];
    const int n = experts + 1, per = (n + kSortThreads - 1) / kSortThreads;
    for (int e = tid; e < n; e += kSortThreads) hist[e] = 0;
    __syncthreads();
#pragma unroll 4
    for (int f = tid; f < slots; f += kSortThreads) atomicAdd(&hist[sort_key(ids[f], experts)], 1);
    __syncthreads();
    int mine = 0;
    for (int i = 0; i < kPer; ++i)
      if (i < per && tid * per + i < n) mine += hist[tid * per + i];
    int first = sort_scan(mine, red[0]);
    for (int i = 0; i < kPer; ++i) {
      const int e = tid * per + i;
      if (i < per && e < n) {
        offsets[e] = first;
        first += hist[e];
      }
    }
    return;
  }
  const int t = blockIdx.x / parts, part = blockIdx.x % parts;
  const int each = (top_k + parts - 1) / parts, j1 = min(top_k, (part + 1) * each);
  const uint4* from = reinterpret_cast<const uint4*>(x + t * row_bytes);
  const int chunks = static_cast<int>(row_bytes >> 4);
  for (int j0 = part * each; j0 < j1; j0 += N) {
    const int f0 = t * top_k + j0;
    int key[N], before[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      key[u] = sort_key(ids[j0 + u < j1 ? f0 + u : f0], experts);
      before[u] = 0;
    }
#pragma unroll 4
    for (int g = tid; g < slots; g += kSortThreads) {
      const int k = sort_key(ids[g], experts);
#pragma unroll
      for (int u = 0; u < N; ++u) before[u] += k < key[u] + (g < f0 + u);  // k < key, or equal and earlier
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) before[u] += __shfl_xor(before[u], o, 64);
      if ((tid & 63) == 0) red[tid >> 6][u] = before[u];
    }
    __syncthreads();
    int p[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      p[u] = 0;
#pragma unroll
      for (int w = 0; w < kSortThreads / 64; ++w) p[u] += red[w][u];
      if (tid == u && j0 + u < j1) {
        perm[p[u]] = f0 + u;
        inv[f0 + u] = p[u];
      }
    }
    for (int c = tid; c < chunks; c += kSortThreads) {
      const uint4 v = from[c];
#pragma unroll
      for (int u = 0; u < N; ++u)
        if (j0 + u < j1) st_nt16(reinterpret_cast<uint4*>(xp + p[u] * row_bytes) + c, key[u] < experts ? v : uint4{0, 0, 0, 0});
    }
    __syncthreads();  // red is the next slots'
  }
}

// Places in use, and whether a place is one: `inv` comes from the caller, and a row outside
// the buffer is never touched.
__device__ __forceinline__ unsigned places_in_use(const int32_t* in_use, int64_t slots) {
  const int64_t n = *in_use;
  return static_cast<unsigned>(n < 0 ? 0 : n < slots ? n : slots);
}

// A token's row to its places.
__global__ __launch_bounds__(kMoveThreads) void permute_rows_kernel(const uint8_t* __restrict__ x, int64_t tokens,
                                                                    int64_t row_bytes,
                                                                    const int32_t* __restrict__ inv, int top_k,
                                                                    const int32_t* __restrict__ in_use,
                                                                    uint8_t* __restrict__ xp) {
  const int64_t slots = tokens * top_k;
  const unsigned live = places_in_use(in_use, slots);
  const int chunks = static_cast<int>(row_bytes >> 4);
  for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
    const int32_t* at = inv + t * top_k;
    const uint4* from = reinterpret_cast<const uint4*>(x + t * row_bytes);
    for (int c = threadIdx.x; c < chunks; c += blockDim.x) {
      const uint4 v = ld_nt16(from + c);
      for (int j = 0; j < top_k; ++j) {
        const unsigned p = at[j];
        st_nt16(reinterpret_cast<uint4*>(xp + p * row_bytes) + c, p < live ? v : uint4{0, 0, 0, 0});
      }
    }
  }
}

// Eight values as they are stored, loaded non-temporally; unpacked where they are used, or the
// loads of several rows would wait for each other.
template <bool F32>
struct Rows8 {
  uint4 u[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    if constexpr (F32) {
      u[0] = ld_nt16(static_cast<const float*>(p) + i);
      u[1] = ld_nt16(static_cast<const float*>(p) + i + 4);
    } else {
      u[0] = ld_nt16(static_cast<const uint16_t*>(p) + i);
    }
  }
  __device__ __forceinline__ F8v get() const {
    if constexpr (F32)
      return F8v{{__uint_as_float(u[0].x), __uint_as_float(u[0].y), __uint_as_float(u[0].z), __uint_as_float(u[0].w),
                  __uint_as_float(u[1].x), __uint_as_float(u[1].y), __uint_as_float(u[1].z), __uint_as_float(u[1].w)}};
    else
      return unpack_bf16x8(u[0]);
  }
};
template <bool F32>
__device__ __forceinline__ void store8_nt(void* p, int64_t i, const F8v& f) {
  if constexpr (F32) {
    float* d = static_cast<float*>(p) + i;
    st_nt16(d, uint4{__float_as_uint(f.v[0]), __float_as_uint(f.v[1]), __float_as_uint(f.v[2]), __float_as_uint(f.v[3])});
    st_nt16(d + 4, uint4{__float_as_uint(f.v[4]), __float_as_uint(f.v[5]), __float_as_uint(f.v[6]), __float_as_uint(f.v[7])});
  } else {
    st_nt16(static_cast<uint16_t*>(p) + i, pack_bf16x8(f));
  }
}

// out[t] = sum_j w_j y[inv[t,j]] over the slots in use, w null: 1.  The loads of up to
// eight slots go out together.
template <bool F32>
__global__ __launch_bounds__(kMoveThreads) void combine_rows_kernel(const void* __restrict__ y, const float* __restrict__ w,
                                                                    int64_t tokens,
                                                                    const int32_t* __restrict__ inv, int top_k,
                                                                    const int32_t* __restrict__ in_use, int hidden,
                                                                    void* __restrict__ out) {
  const int64_t slots = tokens * top_k;
  const unsigned live = places_in_use(in_use, slots);
  for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
    const int32_t* at = inv + t * top_k;
    const float* wt = w + t * top_k;
    for (int c = threadIdx.x * 8; c < hidden; c += blockDim.x * 8) {
      F8v acc{};
      for (int j0 = 0; j0 < top_k; j0 += 8) {
        Rows8<F32> v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          if (j0 + u < top_k && static_cast<unsigned>(at[j0 + u]) < live) v[u].load(y, static_cast<int64_t>(at[j0 + u]) * hidden + c);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          if (j0 + u < top_k && static_cast<unsigned>(at[j0 + u]) < live) {
            const float s = w != nullptr ? wt[j0 + u] : 1.0f;
            const F8v r = v[u].get();
#pragma unroll
            for (int i = 0; i < 8; ++i) acc.v[i] = __builtin_fmaf(s, r.v[i], acc.v[i]);
          }
        }
      }
      store8_nt<F32>(out, t * hidden + c, acc);
    }
  }
}

// dy and dw of a token's slots, four at a time.
template <bool F32>
__global__ __launch_bounds__(kMoveThreads) void combine_grad_kernel(const void* __restrict__ dout, const void* __restrict__ y,
                                                                    const float* __restrict__ w, int64_t tokens,
                                                                    const int32_t* __restrict__ inv, int top_k,
                                                                    const int32_t* __restrict__ in_use, int hidden,
                                                                    void* __restrict__ dy, float* __restrict__ dw) {
  constexpr int kAt = 4;
  __shared__ float red[kMaxTopK][kMoveThreads / 64];
  const int64_t slots = tokens * top_k;
  const unsigned live = places_in_use(in_use, slots);
  for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
    const int32_t* at = inv + t * top_k;
    const float* wt = w + t * top_k;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int j0 = 0; j0 < top_k; j0 += kAt) {
      float dot[kAt];
#pragma unroll
      for (int u = 0; u < kAt; ++u) dot[u] = 0.0f;
      for (int c = threadIdx.x * 8; c < hidden; c += blockDim.x * 8) {
        Rows8<F32> v[kAt];
        const F8v d = load8<F32>(dout, t * hidden + c);
#pragma unroll
        for (int u = 0; u < kAt; ++u) {
          if (j0 + u < top_k && static_cast<unsigned>(at[j0 + u]) < live) v[u].load(y, static_cast<int64_t>(at[j0 + u]) * hidden + c);
        }
#pragma unroll
        for (int u = 0; u < kAt; ++u) {
          if (j0 + u < top_k) {
            const bool in = static_cast<unsigned>(at[j0 + u]) < live;
            const float s = wt[j0 + u];
            F8v o{};
            if (in) {
              const F8v r = v[u].get();
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                dot[u] = __builtin_fmaf(d.v[i], r.v[i], dot[u]);
                o.v[i] = s * d.v[i];
              }
            }
            if (static_cast<unsigned>(at[j0 + u]) < slots) store8_nt<F32>(dy, static_cast<int64_t>(at[j0 + u]) * hidden + c, o);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kAt; ++u) {
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) dot[u] += __shfl_xor(dot[u], o, 64);
        if (lane == 0 && j0 + u < top_k) red[j0 + u][wave] = dot[u];
      }
    }
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < top_k) {
      float s = 0.0f;
      for (int q = 0; q < static_cast<int>(blockDim.x) / 64; ++q) s += red[threadIdx.x][q];
      dw[t * top_k + threadIdx.x] = s;
    }
    __syncthreads();  // red is the next token's
  }
}

// One wave per token; a lane's columns e, e + 64, ... are compared with the k chosen
// experts (the same one twice adds up).
__global__ __launch_bounds__(256) void route_grad_kernel(const float* __restrict__ dw, const float* __restrict__ w,
                                                         const int32_t* __restrict__ idx, int64_t tokens, int experts,
                                                         int top_k, float* __restrict__ dlogits) {
  const int lane = threadIdx.x & 63;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (t >= tokens) return;
  // lane j < k (k <= 32) holds slot j
  const bool has = lane < top_k;
  const float wj = has ? w[t * top_k + lane] : 0.0f, dj = has ? dw[t * top_k + lane] : 0.0f;
  const int ej = has ? idx[t * top_k + lane] : -1;
  float s = wj * dj;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
  const float v = wj * (dj - s);
  for (int e0 = 0; e0 < experts; e0 += 64) {
    float g = 0.0f;
    for (int j = 0; j < top_k; ++j) {
      const float vj = lane_value(v, j);
      if (lane_value(ej, j) == e0 + lane) g += vj;
    }
    if (e0 + lane < experts) dlogits[t * experts + e0 + lane] = g;
  }
}

}  // namespace hkmoe
