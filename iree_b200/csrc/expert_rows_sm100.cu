// Rows of tokens moved to their experts and back.
//
//   dispatch   slots (t, j) whose id names one of the experts [first, first + E) are sorted by expert, stable in (t, j):
//              offsets[e] = slots of experts before e, position[t, j] = the slot's row (-1: dropped), order[i] = t * slots + j
//              of row i (-1 behind the last), rows[position[t, j]] = x[t]
//   combine    out[t] = sum_j weight[t, j] rows[position[t, j]]; without weights the gradient of dispatch
//   backward   drows[position[t, j]] = weight[t, j] dout[t], dweight[t, j] = <dout[t], rows[position[t, j]]>
//
// All of it moves bytes: each row is read once and written once, in 16-byte pieces where addresses and widths allow
// (8-byte and single elements otherwise); sums are f32, in slot order, rounded once. No atomics decide an order.
//
// The sort counts. One CTA owns a run of tokens; what it has to know of the rest is how many slots go to each expert before
// its run and in all. Up to 8192 slots every CTA counts all of them itself, one launch; above that a first launch leaves one
// histogram per run and a second one sums them along the runs. Ranks inside a run come from warp votes.
//
// Every kernel here lets the next one on the stream start after its own wait, not before: a kernel further on that fetches weights
// ahead of its wait (matrix-vector products under dispatch overlap) then finds only this one unfinished, not what it waited for.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "sm100_ptx.cuh"

namespace b200 {

constexpr int kRouteThreads = 512;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteRun = kRouteThreads;  // slots of a run that are ranked at a time: one per thread

template <int V>
struct Piece;  // V two-byte elements
template <>
struct Piece<8> { using type = uint4; };
template <>
struct Piece<4> { using type = uint2; };
template <>
struct Piece<1> { using type = uint16_t; };

template <bool BF16>
__device__ __forceinline__ float to_float(uint16_t bits) {
  if (BF16) return __uint_as_float(static_cast<uint32_t>(bits) << 16);
  return __half2float(__ushort_as_half(bits));
}
template <bool BF16>
__device__ __forceinline__ uint16_t to_bits(float v) {
  if (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  return __half_as_ushort(__float2half_rn(v));
}
template <int V>
union PieceValues {
  typename Piece<V>::type piece;
  uint16_t e[V];
};

// ---- sort and move ------------------------------------------------------------------------------------------------------

__device__ __forceinline__ int local_expert(int id, int first, int experts) {
  const unsigned l = static_cast<unsigned>(id) - static_cast<unsigned>(first);
  return id >= first && l < static_cast<unsigned>(experts) ? static_cast<int>(l) : -1;
}

// A warp moves a strip of 32 * V * 8 elements of a token at a time, 4 KiB: half of that lost a third of the rate (8192 x 8 rows
// of 2048: 60 us, 82 with strips of 2 KiB), and twice the warps per SM no more than evened out.
template <int V>
__device__ void move_rows(const uint16_t* __restrict__ x, uint16_t* __restrict__ rows, const int32_t* __restrict__ where,
                          int tokens, int64_t t0, int slots, int d0, int d1, int64_t ldx, int64_t ldr) {
  using P = typename Piece<V>::type;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int width = (d1 - d0) / V;
  constexpr int U = 8;
  const int strips = (width + 32 * U - 1) / (32 * U);
  for (int w = warp; w < tokens * strips; w += kRouteWarps) {
    const int t = w / strips, s = w - t * strips;
    const P* src = reinterpret_cast<const P*>(x + (t0 + t) * ldx + d0);
    const int c0 = s * 32 * U + lane;
    P v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + 32 * u < width) v[u] = src[c0 + 32 * u];
    for (int j = 0; j < slots; ++j) {
      const int pos = where[t * slots + j];
      if (pos < 0) continue;
      P* dst = reinterpret_cast<P*>(rows + static_cast<int64_t>(pos) * ldr + d0);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + 32 * u < width) __stcs(dst + c0 + 32 * u, v[u]);
    }
  }
}

}  // namespace b200

using namespace b200;

// One histogram per run of `run` tokens: counts[run][expert].
extern "C" __global__ void __launch_bounds__(b200::kRouteThreads)
    b200_expert_count(const int32_t* ids, int32_t* counts, int tokens, int slots, int experts, int first, int run) {
  __shared__ int hist[kRouteMaxExperts];
  for (int e = threadIdx.x; e < experts; e += kRouteThreads) hist[e] = 0;
  grid_dependency_wait();
  grid_launch_dependents();
  __syncthreads();
  const int64_t lo = static_cast<int64_t>(blockIdx.x) * run * slots;
  const int64_t hi = min(lo + static_cast<int64_t>(run) * slots, static_cast<int64_t>(tokens) * slots);
  for (int64_t i = lo + threadIdx.x; i < hi; i += kRouteThreads) {
    const int e = local_expert(ids[i], first, experts);
    if (e >= 0) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += kRouteThreads) counts[static_cast<int64_t>(blockIdx.x) * experts + e] = hist[e];
}

// The runs' histograms become, in place, the slots of each expert in the runs before; totals[expert]: in all runs. A CTA owns
// 32 experts (a lane each), its 16 warps equal parts of the runs.
extern "C" __global__ void __launch_bounds__(b200::kRouteThreads)
    b200_expert_scan(int32_t* counts, int32_t* totals, int runs, int experts) {
  __shared__ int part_sum[kRouteWarps][32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, e = blockIdx.x * 32 + lane;
  const int per = (runs + kRouteWarps - 1) / kRouteWarps, lo = warp * per, hi = min(lo + per, runs);
  constexpr int kBatch = 10;  // loads in flight per thread: all of a part, at most 148 runs / 16 warps
  int sum = 0;
  for (int r0 = lo; r0 < hi; r0 += kBatch) {
    int c[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) c[i] = r0 + i < hi && e < experts ? counts[static_cast<int64_t>(r0 + i) * experts + e] : 0;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) sum += c[i];
  }
  part_sum[warp][lane] = sum;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kRouteWarps; ++w) {
    if (w < warp) before += part_sum[w][lane];
    all += part_sum[w][lane];
  }
  for (int r0 = lo; r0 < hi; r0 += kBatch) {
    int c[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) c[i] = r0 + i < hi && e < experts ? counts[static_cast<int64_t>(r0 + i) * experts + e] : 0;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (r0 + i < hi && e < experts) counts[static_cast<int64_t>(r0 + i) * experts + e] = before;
      before += c[i];
    }
  }
  if (warp == 0 && e < experts) totals[e] = all;
}

// Grid: runs of tokens x column parts. counts, totals: of b200_expert_scan, or NULL (every CTA counts all ids).
extern "C" __global__ void __launch_bounds__(b200::kRouteThreads)
    b200_expert_route(const int32_t* ids, const int32_t* counts, const int32_t* totals, const uint16_t* x, int32_t* offsets, int32_t* position,
                      int32_t* order, uint16_t* rows, int tokens, int slots, int experts, int first, int run, int width,
                      int ldx, int ldr, int part_width, int vec) {
  extern __shared__ int shared[];
  int* next = shared;                  // the run's next row of each expert
  int* base = next + experts;          // the same at the start of the piece that is ranked
  int* total = base + experts;         // slots per expert, then offsets
  int* where = total + experts + 1;    // rows of the slots of one piece of the run
  uint16_t* warp_count = reinterpret_cast<uint16_t*>(where + kRouteRun);  // [warp][expert], then slots of the warps before
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int e = tid; e < experts; e += kRouteThreads) next[e] = total[e] = 0;
  grid_dependency_wait();
  grid_launch_dependents();
  __syncthreads();
  const int64_t all = static_cast<int64_t>(tokens) * slots;
  const int64_t t_lo = static_cast<int64_t>(blockIdx.x) * run, t_hi = min(t_lo + run, static_cast<int64_t>(tokens));
  if (counts) {
    for (int e = tid; e < experts; e += kRouteThreads) {
      total[e] = totals[e];
      next[e] = counts[static_cast<int64_t>(blockIdx.x) * experts + e];
    }
  } else {
    constexpr int kBatch = 8;  // ids loaded at a time
    for (int64_t i0 = tid; i0 < all; i0 += kRouteThreads * kBatch) {
      int id[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) id[i] = i0 + i * kRouteThreads < all ? local_expert(ids[i0 + i * kRouteThreads], first, experts) : -1;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (id[i] >= 0) {
          atomicAdd(&total[id[i]], 1);
          if (i0 + i * kRouteThreads < t_lo * slots) atomicAdd(&next[id[i]], 1);
        }
      }
    }
  }
  __syncthreads();
  if (warp == 0) {  // exclusive sums over experts
    int sum = 0;
    for (int e0 = 0; e0 < experts; e0 += 32) {
      const int e = e0 + lane, own = e < experts ? total[e] : 0;
      int incl = own;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += v;
      }
      if (e < experts) {
        total[e] = sum + incl - own;
        next[e] += sum + incl - own;
      }
      sum += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) total[experts] = sum;
  }
  __syncthreads();
  const int kept = total[experts];
  const bool writes = blockIdx.y == 0;  // the CTAs of the first column part write the tables
  if (writes && blockIdx.x == 0)
    for (int e = tid; e <= experts; e += kRouteThreads) offsets[e] = total[e];
  if (writes)
    for (int64_t i = kept + static_cast<int64_t>(blockIdx.x) * kRouteThreads + tid; i < all;
         i += static_cast<int64_t>(gridDim.x) * kRouteThreads)
      order[i] = -1;
  const int d0 = blockIdx.y * part_width, d1 = width - d0 < part_width ? width : d0 + part_width;
  const int tokens_at_once = max(1, kRouteRun / slots);
  for (int64_t t0 = t_lo; t0 < t_hi; t0 += tokens_at_once) {
    const int nt = static_cast<int>(min(static_cast<int64_t>(tokens_at_once), t_hi - t0));
    const int n = nt * slots;
    for (int i = tid; i < kRouteWarps * experts; i += kRouteThreads) warp_count[i] = 0;
    __syncthreads();
    const int e = tid < n ? local_expert(ids[t0 * slots + tid], first, experts) : -1;
    const unsigned peers = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(peers & ((1u << lane) - 1u));
    if (e >= 0 && rank == 0) warp_count[warp * experts + e] = static_cast<uint16_t>(__popc(peers));
    __syncthreads();
    for (int x_e = tid; x_e < experts; x_e += kRouteThreads) {  // slots of the expert in the warps before each one
      int at = 0;
#pragma unroll
      for (int w = 0; w < kRouteWarps; ++w) {
        const int c = warp_count[w * experts + x_e];
        warp_count[w * experts + x_e] = static_cast<uint16_t>(at);
        at += c;
      }
      base[x_e] = next[x_e];
      next[x_e] += at;
    }
    __syncthreads();
    if (tid < n) {
      const int pos = e >= 0 ? base[e] + warp_count[warp * experts + e] + rank : -1;
      where[tid] = pos;
      if (writes) {
        position[t0 * slots + tid] = pos;
        if (pos >= 0) order[pos] = static_cast<int32_t>(t0 * slots + tid);
      }
    }
    __syncthreads();
    if (vec == 8) move_rows<8>(x, rows, where, nt, t0, slots, d0, d1, ldx, ldr);
    else if (vec == 4) move_rows<4>(x, rows, where, nt, t0, slots, d0, d1, ldx, ldr);
    else move_rows<1>(x, rows, where, nt, t0, slots, d0, d1, ldx, ldr);
    __syncthreads();  // `where` is written again
  }
}

namespace b200 {

// ---- back to tokens -------------------------------------------------------------------------------------------------------
constexpr int kCombineThreads = 256;
constexpr int kCombineWarps = kCombineThreads / 32;

// A warp owns a strip of 32 * V * U columns of one token and adds the slots' rows in order. J > 1: J slots' places first,
// then all their pieces (8-byte pieces need the more of them on their way: 4095 x 4 rows of 2044 in 15.7 us, 20.4 with J = 1,
// U = 2; 16-byte pieces lose the warps that the registers cost: 8192 x 2 rows of 4096 in 34.5 us against 40.4 with J = 2).
template <bool BF16, int V, int U, int J>
__device__ void combine_body(const uint16_t* __restrict__ rows, const float* __restrict__ weights,
                             const int32_t* __restrict__ position, uint16_t* __restrict__ out, int tokens, int slots,
                             int width, int64_t ldr, int64_t ldo, int row_count) {
  using P = typename Piece<V>::type;
  const int lane = threadIdx.x & 31;
  const int pieces = width / V, strips = (pieces + 32 * U - 1) / (32 * U);
  const unsigned w = blockIdx.x * kCombineWarps + (threadIdx.x >> 5);
  if (w >= static_cast<unsigned>(tokens) * strips) return;
  const int64_t t = w / static_cast<unsigned>(strips);
  const int c0 = static_cast<int>(w - t * strips) * 32 * U + lane;
  float acc[U][V];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < V; ++i) acc[u][i] = 0.f;
  if constexpr (J > 1) {
    for (int j0 = 0; j0 < slots; j0 += J) {
      int pos[J];
      float weight[J];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        pos[j] = j0 + j < slots ? position[t * slots + j0 + j] : -1;
        if (static_cast<unsigned>(pos[j]) >= static_cast<unsigned>(row_count)) pos[j] = -1;
        weight[j] = weights && j0 + j < slots ? weights[t * slots + j0 + j] : 1.f;
      }
      PieceValues<V> v[J][U];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const P* src = reinterpret_cast<const P*>(rows + pos[j] * ldr);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (pos[j] >= 0 && c0 + 32 * u < pieces) v[j][u].piece = src[c0 + 32 * u];
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (pos[j] >= 0) {
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (c0 + 32 * u < pieces) {
#pragma unroll
              for (int i = 0; i < V; ++i) acc[u][i] = fmaf(weight[j], to_float<BF16>(v[j][u].e[i]), acc[u][i]);
            }
        }
      }
    }
  } else {
#pragma unroll 4
    for (int j = 0; j < slots; ++j) {
      const int pos = position[t * slots + j];
      if (static_cast<unsigned>(pos) >= static_cast<unsigned>(row_count)) continue;
      const float weight = weights ? weights[t * slots + j] : 1.f;
      const P* src = reinterpret_cast<const P*>(rows + pos * ldr);
      PieceValues<V> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + 32 * u < pieces) v[u].piece = src[c0 + 32 * u];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + 32 * u < pieces) {
#pragma unroll
          for (int i = 0; i < V; ++i) acc[u][i] = fmaf(weight, to_float<BF16>(v[u].e[i]), acc[u][i]);
        }
    }
  }
  P* dst = reinterpret_cast<P*>(out + t * ldo);
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (c0 + 32 * u < pieces) {
      PieceValues<V> v;
#pragma unroll
      for (int i = 0; i < V; ++i) v.e[i] = to_bits<BF16>(acc[u][i]);
      dst[c0 + 32 * u] = v.piece;
    }
}

// A warp owns a slot: its row's dot product with dout[t], and the scaled copy of dout[t].
template <bool BF16, int V, int U>
__device__ void combine_backward_body(const uint16_t* __restrict__ dout, const uint16_t* __restrict__ rows,
                                      const float* __restrict__ weights, const int32_t* __restrict__ position,
                                      uint16_t* __restrict__ drows, float* __restrict__ dweights, int tokens, int slots,
                                      int width, int64_t ldo, int64_t ldr, int row_count) {
  using P = typename Piece<V>::type;
  const int lane = threadIdx.x & 31;
  const unsigned slot = blockIdx.x * kCombineWarps + (threadIdx.x >> 5);
  if (slot >= static_cast<unsigned>(tokens) * slots) return;
  const int pos = position[slot];
  float dot = 0.f;
  if (static_cast<unsigned>(pos) < static_cast<unsigned>(row_count)) {
    const float weight = weights[slot];
    const int pieces = width / V;
    const P* d = reinterpret_cast<const P*>(dout + static_cast<int64_t>(slot / static_cast<unsigned>(slots)) * ldo);
    const P* r = reinterpret_cast<const P*>(rows + pos * ldr);
    P* o = reinterpret_cast<P*>(drows + pos * ldr);
    for (int c0 = lane; c0 < pieces; c0 += 32 * U) {
      PieceValues<V> dv[U], rv[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + 32 * u < pieces) {
          dv[u].piece = d[c0 + 32 * u];
          rv[u].piece = r[c0 + 32 * u];
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + 32 * u < pieces) {
          PieceValues<V> ov;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float dd = to_float<BF16>(dv[u].e[i]);
            dot = fmaf(dd, to_float<BF16>(rv[u].e[i]), dot);
            ov.e[i] = to_bits<BF16>(weight * dd);
          }
          o[c0 + 32 * u] = ov.piece;
        }
    }
#pragma unroll
    for (int s = 16; s; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
  }
  if (lane == 0) dweights[slot] = dot;
}

}  // namespace b200

#define B200_EXPERT_COMBINE(SUFFIX, BF16)                                                                                  \
  extern "C" __global__ void __launch_bounds__(b200::kCombineThreads, 6)                                                   \
      b200_expert_combine_##SUFFIX(const uint16_t* rows, const float* weights, const int32_t* position, uint16_t* out,     \
                                   int tokens, int slots, int width, int ldr, int ldo, int row_count) {                    \
    grid_dependency_wait();                                                                                                \
    grid_launch_dependents();                                                                                              \
    combine_body<BF16, 8, 2, 1>(rows, weights, position, out, tokens, slots, width, ldr, ldo, row_count);                     \
  }                                                                                                                        \
  extern "C" __global__ void __launch_bounds__(b200::kCombineThreads)                                                      \
      b200_expert_combine_narrow_##SUFFIX(const uint16_t* rows, const float* weights, const int32_t* position,             \
                                          uint16_t* out, int tokens, int slots, int width, int ldr, int ldo,               \
                                          int row_count, int vec) {                                                        \
    grid_dependency_wait();                                                                                                \
    grid_launch_dependents();                                                                                              \
    if (vec == 4) combine_body<BF16, 4, 4, 2>(rows, weights, position, out, tokens, slots, width, ldr, ldo, row_count);       \
    else combine_body<BF16, 1, 2, 4>(rows, weights, position, out, tokens, slots, width, ldr, ldo, row_count);                \
  }                                                                                                                        \
  extern "C" __global__ void __launch_bounds__(b200::kCombineThreads, 6)                                                   \
      b200_expert_combine_backward_##SUFFIX(const uint16_t* dout, const uint16_t* rows, const float* weights,              \
                                            const int32_t* position, uint16_t* drows, float* dweights, int tokens,         \
                                            int slots, int width, int ldo, int ldr, int row_count, int vec) {              \
    grid_dependency_wait();                                                                                                \
    grid_launch_dependents();                                                                                              \
    if (vec == 8)                                                                                                          \
      combine_backward_body<BF16, 8, 2>(dout, rows, weights, position, drows, dweights, tokens, slots, width, ldo, ldr,    \
                                        row_count);                                                                        \
    else if (vec == 4)                                                                                                     \
      combine_backward_body<BF16, 4, 2>(dout, rows, weights, position, drows, dweights, tokens, slots, width, ldo, ldr,    \
                                        row_count);                                                                        \
    else                                                                                                                   \
      combine_backward_body<BF16, 1, 4>(dout, rows, weights, position, drows, dweights, tokens, slots, width, ldo, ldr,    \
                                        row_count);                                                                        \
  }
B200_EXPERT_COMBINE(f16, false)
B200_EXPERT_COMBINE(bf16, true)
#undef B200_EXPERT_COMBINE
