// Few-rows products with 4-bit weights and group scales: matrix-vector products (1..16 activation rows) and the experts'
// products of a decoding batch, where every expert sees a few rows. Weights are read once and bound the time.
//
//   w[n, k]   = (q[n, k] - z[n, k / group]) * s[n, k / group]     zeros given: q = 0..15 as stored
//   w[n, k]   = q[n, k] * s[n, k / group]                         no zeros: q is two's complement, -8..7
//   out[m, n] = round(sum_k a[m, k] * w[n, k])
//
// Arithmetic. Per block of 32 * GQ values of K (the part of a scale group that a 128-wide chunk holds):
//   v = sum_k a q' - z' sum_k a,   total += s v      all in f32; q' is the stored nibble (top bit flipped when it is signed,
//                                                    z' = 8 then), so only the result is rounded to 16 bits.
// A nibble becomes a 16-bit float by a shift and one logic operation for two weights: under the exponent of 64 (f16: its bits
// land in mantissa bits 4..7) or 128 (bf16: bits 0..3), and z' grows by that much; the part that cancels is at most 158 / 15 of
// the sum it leaves, 2^-20 of it in f32. (f16 subnormals, q 2^-24 as stored, would spare the shifts; but the tensor core
// aligns products by their exponent fields, and sums lost up to six more bits there.) The sums of a are one more row of ones
// in the matrix instruction, shared by all weight tiles of a warp.
//
// Work. The weight rows of all active experts (one, for a matrix-vector product) form one list; every CTA gets an equal
// part of it, to the row, so that all SMs read the same number of bytes (tiles of 16 rows alone would leave the last round
// half empty: 688 tiles on 148 SMs are 4.65 rounds). A CTA's warps are WK along K x WN along N, chosen by the CTA for the
// rows it holds; a warp walks units of 16 rows x 128 K through a private ring of cp.async stages (no barrier between
// warps), and the WK partial sums meet in shared memory at the end, in order: results do not depend on timing.
// Activations are staged in slices, the next one while the present one is used.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "sm100_ptx.cuh"
#include "w4a16_decode.cuh"

namespace b200 {

constexpr int kStreamThreads = 512;
constexpr int kStreamWarps = kStreamThreads / 32;
constexpr int kStreamRing = 5;                        // units in flight per warp (4) and the one in use: 64 KiB per SM in flight
constexpr int kStreamUnitBytes = 1024;                // 16 weight rows x 128 K
constexpr int kStreamActBytes = 66 * 1024;            // one activation slice: 8 NB rows x (4096 / NB) K, 64 bytes of padding per row
constexpr int kStreamBatchMax = 64;                   // batches described at a time
constexpr int kStreamMaxExperts = 1024;
constexpr int kStreamTableBytes = kStreamBatchMax * 32 + (kStreamMaxExperts + 1) * 4 + 256;
constexpr int kStreamSmemBytes = 2 * kStreamActBytes + kStreamWarps * kStreamRing * kStreamUnitBytes + kStreamTableBytes;
static_assert(kStreamSmemBytes <= 232448, "per-CTA shared memory limit");

struct StreamBatch {
  int64_t w_row;    // first weight row, over all experts
  int32_t n0;       // the same within the expert = first result column
  int32_t nrows;    // weight rows
  int32_t a_row;    // first activation row
  int32_t mrows;    // activation rows
  int32_t wk_log2;  // warps along K
  int32_t pad;
};
static_assert(sizeof(StreamBatch) == 32, "table size");

__device__ __forceinline__ void stream_copy_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void stream_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void stream_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t and_xor(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(a), "r"(b), "r"(c));  // (a & b) ^ c
  return r;
}
template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if (BF16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
template <bool BF16>
__device__ __forceinline__ float half_bits_to_float(uint32_t bits) {
  if (BF16) return __uint_as_float(bits << 16);
  return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}

struct StreamArgs {
  const uint16_t* a;
  const uint8_t* wq;
  const uint16_t* scales;
  const uint16_t* zeros;     // NULL: signed nibbles
  const int32_t* offsets;    // NULL: one expert that owns all rows
  uint16_t* out;
  int M, N, K, group, lda, ldo, experts;
};

// NB: blocks of 8 activation rows a pass covers; GQ: 32-wide K blocks per scale application (group % (32 GQ) == 0).
template <bool BF16, int NB, int GQ>
__device__ void stream_body(const StreamArgs& p) {
  // weight tiles per warp: what fits the registers, and the partial sums of 16 warps one activation buffer
  constexpr int TM = NB == 1 ? 4 : 3;
  constexpr int kSliceK = 4096 / NB;
  constexpr int kActPitch = kSliceK * 2 + 64;      // bytes; 64 mod 128: eight lanes of a 16-byte read hit all banks
  constexpr int kRedPitch = 20;                    // floats per activation row of a partial tile (16 + padding)
  constexpr int kBlocks = 4 / GQ;                  // scale applications per chunk
  static_assert(8 * NB * kActPitch <= kStreamActBytes, "activation slice");
  static_assert(kStreamWarps * TM * 8 * NB * kRedPitch * 4 <= kStreamActBytes, "partial sums");

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t smem = smem_u32(smem_raw);
  uint8_t* table_gen = smem_raw + 2 * kStreamActBytes + kStreamWarps * kStreamRing * kStreamUnitBytes;
  StreamBatch* batches = reinterpret_cast<StreamBatch*>(table_gen);
  int* seg_first = reinterpret_cast<int*>(table_gen + kStreamBatchMax * 32);  // passes before each expert
  int* shared_words = seg_first + kStreamMaxExperts + 1;                      // [0] batches in the table

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem + 2 * kStreamActBytes + warp * (kStreamRing * kStreamUnitBytes);
  const int chunks = (p.K + 127) >> 7;
  const int slices = (p.K + kSliceK - 1) / kSliceK;
  const bool acts_aligned = !((reinterpret_cast<uintptr_t>(p.a) | (static_cast<uintptr_t>(p.lda) * 2)) & 15);
  const int groups = p.K / p.group;
  const int64_t w_pitch = p.K >> 1;

  grid_launch_dependents();
  // Experts: how many passes (8 NB activation rows each) each one needs comes from the dispatch ahead.
  int passes = (p.M + 8 * NB - 1) / (8 * NB);
  if (p.offsets) {
    grid_dependency_wait();
    if (warp == 0) {
      int sum = 0;
      for (int e0 = 0; e0 < p.experts; e0 += 32) {
        const int e = e0 + lane;
        int need = 0;
        if (e < p.experts) {
          const int lo = min(max(p.offsets[e], 0), p.M), hi = min(max(p.offsets[e + 1], lo), p.M);
          need = (hi - lo + 8 * NB - 1) / (8 * NB);
        }
        int incl = need;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, incl, d);
          if (lane >= d) incl += v;
        }
        if (e < p.experts) seg_first[e] = sum + incl - need;
        sum += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) seg_first[p.experts] = sum;
    }
    __syncthreads();
    passes = seg_first[p.experts];
  }
  const int64_t total = static_cast<int64_t>(passes) * p.N;  // weight rows to be read, over all passes
  const int64_t share = (total + gridDim.x - 1) / gridDim.x;
  int64_t row = share * blockIdx.x;
  const int64_t row_end = min(row + share, total);
  bool waited = p.offsets != nullptr;
  const uint32_t mask = BF16 ? 0x000f000fu : 0x00f000f0u;
  const uint32_t under = BF16 ? (p.zeros ? 0x43004300u : 0x43084308u) : (p.zeros ? 0x54005400u : 0x54805480u);
  const uint32_t ones = BF16 ? 0x3f803f80u : 0x3c003c00u;
  const float z_base = BF16 ? 128.f : 64.f;

  while (row < row_end) {  // one turn for up to kStreamBatchMax batches: one, unless the operands are very uneven
    __syncthreads();
    if (tid == 0) {
      int count = 0;
      int e = 0;
      int64_t pass = row / p.N;
      if (p.offsets) {
        int lo = 0, hi = p.experts;  // last expert whose first pass is <= pass
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (seg_first[mid] <= pass) lo = mid;
          else hi = mid;
        }
        e = lo;
      }
      int64_t r = row;
      while (r < row_end && count < kStreamBatchMax) {
        const int n0 = static_cast<int>(r - pass * p.N);
        const int64_t left = min(row_end - r, static_cast<int64_t>(p.N - n0));
        int first = 0, have = p.M, nth = static_cast<int>(pass);
        if (p.offsets) {
          while (seg_first[e + 1] <= pass) ++e;
          first = min(max(p.offsets[e], 0), p.M);
          have = min(max(p.offsets[e + 1], first), p.M) - first;
          nth = static_cast<int>(pass) - seg_first[e];
        }
        // Warps along K: the split with the fewest units for the busiest warp; ties to more warps along K (more
        // tiles per warp share the activation fragments).
        const int64_t cap = 8 * TM * 16;
        const int64_t parts = (left + cap - 1) / cap;
        const int nrows = static_cast<int>((left + parts - 1) / parts);
        const int tiles = (nrows + 15) >> 4;
        int best = 1, best_units = 0x7fffffff;
        for (int l = 4; l >= 1; --l) {
          const int wn = kStreamWarps >> l, per = (tiles + wn - 1) / wn;
          if (per > TM) continue;
          int units = 0;
          for (int s = 0; s < slices; ++s) {
            const int in_slice = min(kSliceK / 128, chunks - s * (kSliceK / 128));
            units += per * ((in_slice + (1 << l) - 1) >> l);
          }
          if (units < best_units) {
            best_units = units;
            best = l;
          }
        }
        StreamBatch b;
        b.w_row = static_cast<int64_t>(e) * p.N + n0;
        b.n0 = n0;
        b.nrows = nrows;
        b.a_row = first + nth * 8 * NB;
        b.mrows = min(8 * NB, have - nth * 8 * NB);
        b.wk_log2 = best;
        b.pad = 0;
        batches[count++] = b;
        r += nrows;
        if (n0 + nrows == p.N) ++pass;
      }
      shared_words[0] = count;
    }
    __syncthreads();
    const int count = shared_words[0];
    {
      int64_t covered = 0;
      for (int i = 0; i < count; ++i) covered += batches[i].nrows;
      row += covered;
    }
    const int steps = count * slices;

    // ---- unit sequence of this warp: (step = batch x slice, chunk of the slice, tile) ---------------------------------
    int is_step = -1, is_chunk = 0, is_chunks = 0, is_tile = 0, is_tiles = 0, is_slot = 0, is_wk = 0, is_wn = 0;
    StreamBatch is_b;
    uint32_t q0 = 0, q1 = 0, q2 = 0, q3 = 0;  // scales (low half) and zeros (high half) of the units in flight, rows g
    uint32_t r0 = 0, r1 = 0, r2 = 0, r3 = 0;  // rows g + 8
    auto issue_step = [&]() {  // moves the issue cursor to the next step in which this warp has a unit
      while (++is_step < steps) {
        const int b = is_step / slices, s = is_step - b * slices;
        is_b = batches[b];
        const int wk_n = 1 << is_b.wk_log2, wn_n = kStreamWarps >> is_b.wk_log2;
        is_wk = warp & (wk_n - 1);
        is_wn = warp >> is_b.wk_log2;
        const int tiles = (is_b.nrows + 15) >> 4;
        is_tiles = (tiles - is_wn + wn_n - 1) / wn_n;
        const int first = s * (kSliceK / 128);
        is_chunk = first + is_wk;
        is_chunks = min(chunks, first + kSliceK / 128);
        is_tile = 0;
        if (is_tiles > 0 && is_chunk < is_chunks) return;
      }
    };
    auto issue_unit = [&]() {
      // the scales queue moves up by one unit
      q0 = q1;
      q1 = q2;
      q2 = q3;
      r0 = r1;
      r1 = r2;
      r2 = r3;
      if (is_step < steps) {
        const int tile_row = (is_wn + is_tile * (kStreamWarps >> is_b.wk_log2)) << 4;
        const int k0 = is_chunk << 7;
        const uint32_t dst = ring + is_slot * kStreamUnitBytes;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = g + 8 * i, j = t;
          // rows behind the CTA's part and K behind the end are left as they are: what they hold meets nothing that is kept
          if (tile_row + r < is_b.nrows && k0 + 32 * j < p.K)
            stream_copy_16(dst + r * 64 + ((j ^ ((r >> 1) & 3)) << 4),
                        p.wq + (is_b.w_row + tile_row + r) * w_pitch + ((k0 + 32 * j) >> 1));
        }
        const int kk = min(k0 + 32 * t, p.K - 32);
        const int64_t last = is_b.w_row + is_b.nrows - 1;
        const int64_t at0 = min(is_b.w_row + tile_row + g, last) * groups + kk / p.group;
        const int64_t at1 = min(is_b.w_row + tile_row + g + 8, last) * groups + kk / p.group;
        q3 = __ldg(p.scales + at0);
        r3 = __ldg(p.scales + at1);
        if (p.zeros) {
          q3 |= static_cast<uint32_t>(__ldg(p.zeros + at0)) << 16;
          r3 |= static_cast<uint32_t>(__ldg(p.zeros + at1)) << 16;
        }
        if (++is_slot == kStreamRing) is_slot = 0;
        if (++is_tile == is_tiles) {
          is_tile = 0;
          is_chunk += 1 << is_b.wk_log2;
          if (is_chunk >= is_chunks) issue_step();
        }
      }
      stream_commit();
    };
    auto stage_acts = [&](int step) {
      const int b = step / slices, s = step - b * slices;
      const int k0 = s * kSliceK, kn = min(kSliceK, p.K - k0);
      const int a_row = batches[b].a_row, mrows = batches[b].mrows;
      const uint32_t dst = smem + (step & 1) * kStreamActBytes;
      uint8_t* dst_gen = smem_raw + (step & 1) * kStreamActBytes;
      if (acts_aligned) {
        const int pieces = kn >> 3;  // 16-byte pieces per row
        for (int i = tid; i < mrows * pieces; i += kStreamThreads) {
          const int m = i / pieces, c = i - m * pieces;
          stream_copy_16(dst + m * kActPitch + c * 16, p.a + static_cast<int64_t>(a_row + m) * p.lda + k0 + c * 8);
        }
      } else {
        for (int i = tid; i < mrows * kn; i += kStreamThreads) {
          const int m = i / kn, c = i - m * kn;
          *reinterpret_cast<uint16_t*>(dst_gen + m * kActPitch + c * 2) =
              p.a[static_cast<int64_t>(a_row + m) * p.lda + k0 + c];
        }
      }
      stream_commit();
    };

    issue_step();
#pragma unroll
    for (int i = 0; i < kStreamRing - 1; ++i) issue_unit();
    if (!waited) {  // matrix-vector product: weights and scales may be fetched ahead, activations may not
      grid_dependency_wait();
      waited = true;
    }
    stage_acts(0);
    int since = 0;  // groups committed after the activations that the next step needs
    int slot = 0;
    float total_acc[TM][NB * 4];

    for (int step = 0; step < steps; ++step) {
      const int bi = step / slices, s = step - bi * slices;
      // this thread's pieces of the step's activations have landed ...
      if (since == 0) stream_wait<0>();
      else if (since == 1) stream_wait<1>();
      else if (since == 2) stream_wait<2>();
      else stream_wait<3>();
      __syncthreads();  // ... and everybody's; the buffer of the step before is free
      since = 0;
      if (step + 1 < steps) stage_acts(step + 1);
      const StreamBatch b = batches[bi];
      const int wk_n = 1 << b.wk_log2, wn_n = kStreamWarps >> b.wk_log2;
      const int wk = warp & (wk_n - 1), wn = warp >> b.wk_log2;
      const int tiles = (b.nrows + 15) >> 4, my_tiles = (tiles - wn + wn_n - 1) / wn_n;
      if (s == 0) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < NB * 4; ++j) total_acc[i][j] = 0.f;
      }
      const int first = s * (kSliceK / 128), last = min(chunks, first + kSliceK / 128);
      const uint32_t act_base = smem + (step & 1) * kStreamActBytes + g * kActPitch + t * 16;
      if (my_tiles > 0) {
        for (int c = first + wk; c < last; c += wk_n) {
          const int qn = min(4, (p.K - (c << 7)) >> 5);  // 32-wide blocks that the chunk holds
          // activation fragments of the chunk: (a0, a4), (a2, a6), (a1, a5), (a3, a7) of each lane's eight values
          uint32_t bf[NB][4][4];
          float sum[NB][kBlocks][2];
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const bool live = nb * 8 + g < b.mrows;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint4 v = make_uint4(0, 0, 0, 0);
              if (live && q < qn) v = lds128(act_base + nb * 8 * kActPitch + ((c - first) << 8) + (q << 6));
              bf[nb][q][0] = __byte_perm(v.x, v.z, 0x5410);
              bf[nb][q][1] = __byte_perm(v.y, v.w, 0x5410);
              bf[nb][q][2] = __byte_perm(v.x, v.z, 0x7632);
              bf[nb][q][3] = __byte_perm(v.y, v.w, 0x7632);
            }
#pragma unroll
            for (int blk = 0; blk < kBlocks; ++blk) {
              float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int h = 0; h < GQ; ++h) {
                const int q = blk * GQ + h;
                mma_16816<BF16>(d, ones, ones, ones, ones, bf[nb][q][0], bf[nb][q][1]);
                mma_16816<BF16>(d, ones, ones, ones, ones, bf[nb][q][2], bf[nb][q][3]);
              }
              sum[nb][blk][0] = d[0];
              sum[nb][blk][1] = d[1];
            }
          }
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            if (i < my_tiles) {
              stream_wait<kStreamRing - 2>();
              __syncwarp();
              const uint32_t w_base = ring + slot * kStreamUnitBytes + g * 64 + t * 4;
              const int sw = (g >> 1) & 3;
              const uint32_t sc0 = q0, sc1 = r0;
#pragma unroll
              for (int blk = 0; blk < kBlocks; ++blk) {
                if (blk * GQ < qn) {
                  float acc[NB][4];
#pragma unroll
                  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[nb][j] = 0.f;
#pragma unroll
                  for (int h = 0; h < GQ; ++h) {
                    const int q = blk * GQ + h;
                    const uint32_t w0 = lds32(w_base + ((q ^ sw) << 4)), w1 = lds32(w_base + ((q ^ sw) << 4) + 512);
                    // nibbles (0, 4), (2, 6) and (1, 5), (3, 7) of either row
                    const uint32_t a0 = and_xor(BF16 ? w0 : w0 << 4, mask, under), a1 = and_xor(BF16 ? w1 : w1 << 4, mask, under);
                    const uint32_t a2 = and_xor(w0 >> (BF16 ? 8 : 4), mask, under), a3 = and_xor(w1 >> (BF16 ? 8 : 4), mask, under);
                    const uint32_t c0 = and_xor(BF16 ? w0 >> 4 : w0, mask, under), c1 = and_xor(BF16 ? w1 >> 4 : w1, mask, under);
                    const uint32_t c2 = and_xor(w0 >> (BF16 ? 12 : 8), mask, under), c3 = and_xor(w1 >> (BF16 ? 12 : 8), mask, under);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                      mma_16816<BF16>(acc[nb], a0, a1, a2, a3, bf[nb][q][0], bf[nb][q][1]);
                      mma_16816<BF16>(acc[nb], c0, c1, c2, c3, bf[nb][q][2], bf[nb][q][3]);
                    }
                  }
                  // lane t of a quad loaded the scale of the chunk's 32-wide block t
                  const uint32_t e0 = GQ == 4 ? sc0 : __shfl_sync(0xffffffffu, sc0, (lane & 28) | (blk * GQ));
                  const uint32_t e1 = GQ == 4 ? sc1 : __shfl_sync(0xffffffffu, sc1, (lane & 28) | (blk * GQ));
                  const float s0 = half_bits_to_float<BF16>(e0 & 0xffffu);
                  const float s1 = half_bits_to_float<BF16>(e1 & 0xffffu);
                  const float z0 = z_base + (p.zeros ? half_bits_to_float<BF16>(e0 >> 16) : 8.f);
                  const float z1 = z_base + (p.zeros ? half_bits_to_float<BF16>(e1 >> 16) : 8.f);
#pragma unroll
                  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                      const float v = fmaf(j < 2 ? -z0 : -z1, sum[nb][blk][j & 1], acc[nb][j]);
                      total_acc[i][nb * 4 + j] = fmaf(j < 2 ? s0 : s1, v, total_acc[i][nb * 4 + j]);
                    }
                  }
                }
              }
              if (++slot == kStreamRing) slot = 0;
              __syncwarp();  // every lane has read the unit: its slot may be filled again
              issue_unit();
              ++since;
            }
          }
        }
      }
      if (s == slices - 1) {
        // the WK partial sums of each tile meet, in order of K, in the buffer of this step's activations
        __syncthreads();
        float* red = reinterpret_cast<float*>(smem_raw + (step & 1) * kStreamActBytes);
        constexpr int kTile = 8 * NB * kRedPitch;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          if (i < my_tiles) {
            float* dst = red + (wk * tiles + wn + i * wn_n) * kTile;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                dst[(nb * 8 + 2 * t + (j & 1)) * kRedPitch + g + (j >> 1) * 8] = total_acc[i][nb * 4 + j];
          }
        }
        __syncthreads();
        for (int i = tid; i < b.mrows * (tiles << 4); i += kStreamThreads) {
          const int m = i / (tiles << 4), n = i - m * (tiles << 4);
          if (n < b.nrows) {
            const float* src = red + (n >> 4) * kTile + m * kRedPitch + (n & 15);
            float v = 0.f;
            for (int w = 0; w < wk_n; ++w) v += src[w * tiles * kTile];
            uint16_t bits;
            if (BF16) bits = __bfloat16_as_ushort(__float2bfloat16_rn(v));
            else bits = __half_as_ushort(__float2half_rn(v));
            p.out[static_cast<int64_t>(b.a_row + m) * p.ldo + b.n0 + n] = bits;
          }
        }
      }
    }
    stream_wait<0>();
  }
  if (!waited) grid_dependency_wait();
}

template <bool BF16, int NB>
__device__ __forceinline__ void stream_by_group(const StreamArgs& p) {
  if (p.group % 128 == 0) stream_body<BF16, NB, 4>(p);
  else if (p.group % 64 == 0) stream_body<BF16, NB, 2>(p);
  else stream_body<BF16, NB, 1>(p);
}

}  // namespace b200

// Bindings: activations, weights, scales, zero points (NULL: signed weights), row offsets of the experts (NULL: one
// expert), result.
#define B200_W4A16_STREAM(NAME, BF16, NB)                                                                                 \
  extern "C" __global__ void __launch_bounds__(b200::kStreamThreads, 1)                                                   \
      NAME(const uint16_t* a, const uint8_t* wq, const uint16_t* scales, const uint16_t* zeros, const int32_t* offsets,   \
           uint16_t* out, int M, int N, int K, int group, int lda, int ldo, int experts) {                                \
    b200::StreamArgs p = {a, wq, scales, zeros, offsets, out, M, N, K, group, lda, ldo, experts};                         \
    b200::stream_by_group<BF16, NB>(p);                                                                                   \
  }
B200_W4A16_STREAM(b200_w4a16_stream_f16_r8, false, 1)
B200_W4A16_STREAM(b200_w4a16_stream_f16_r16, false, 2)
B200_W4A16_STREAM(b200_w4a16_stream_bf16_r8, true, 1)
B200_W4A16_STREAM(b200_w4a16_stream_bf16_r16, true, 2)
#undef B200_W4A16_STREAM
