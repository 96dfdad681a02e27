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
// land in mantissa bits 4..7) or 2^-8 (bf16: bits 0..3, so it reads 2^-15 (128 + q')), and z' grows by 64 or 128; the part that
// cancels is at most 158 / 15 of the sum it leaves, 2^-20 of it in f32. In bf16 everything up to the result is kept 2^-15 times
// its value, which costs nothing (sums of activations are formed that way, the result is multiplied once): activations reach
// f32's largest numbers, and 128 of them times 143 would pass it where the scaled sum is a number again. What that takes from
// the other end: sums below 2^-111 round in steps of 2^-149 of f32's subnormals, 2^-134 of the value. (f16 subnormals, q 2^-24 as
// stored, would spare the shifts; but the tensor core aligns products by their exponent fields, and sums lost up to six more bits
// there.) The accumulator starts at minus that offset times the sum of a.
//
// Work. The weight rows of all active experts (one, for a matrix-vector product) form one list; every CTA gets an equal
// part of it, to the row, so that all SMs read the same number of bytes (tiles of 16 rows alone would leave the last round
// half empty: 688 tiles on 148 SMs are 4.65 rounds). A batch is up to 512 rows of the part: its row pairs of tiles (32 rows)
// go to WN warp columns and K to WK warps of each, WN x WK <= 16. A warp walks units of 32 rows x 128 K through a private
// ring of cp.async stages (no barrier between warps, and none between batches), and the WK partial sums meet in shared
// memory, in order: results do not depend on timing. Activations are staged in slices of K, the next slice while the present
// one is used; staging orders them as the unpacked nibbles come (k, k + 4) and leaves the sums of each scale block beside them.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "sm100_ptx.cuh"
#include "w4a16_decode.cuh"
#include "w4a16_stream_list.h"

namespace b200 {

constexpr int kStreamWarps = 16;
constexpr int kStreamThreads = kStreamWarps * 32;
constexpr int kStreamRing = 2;                     // units in flight per warp: 64 KiB per SM
constexpr int kStreamUnitBytes = 2048;             // 32 weight rows x 128 K
constexpr int kStreamScaleBytes = 1024;            // scales and zero points of 32 rows x 8 scale blocks, two slots per warp
constexpr int kStreamActBytes = 54 * 1024;         // one activation slice; later the warps' partial sums
constexpr int kStreamSumBytes = 4096;              // the slice's sums
constexpr int kStreamMaxExperts = 1024;
constexpr int kStreamScaleOffset = kStreamWarps * kStreamRing * kStreamUnitBytes;
constexpr int kStreamActOffset = kStreamScaleOffset + kStreamWarps * 2 * kStreamScaleBytes;
constexpr int kStreamSumOffset = kStreamActOffset + 2 * kStreamActBytes;
constexpr int kStreamTableOffset = kStreamSumOffset + 2 * kStreamSumBytes;
constexpr int kStreamWalkOffset = kStreamTableOffset + 2 * (kStreamMaxExperts + 1) * 4;
constexpr int kStreamWalkBytes = 304;              // per warp
constexpr int kStreamSmemBytes = kStreamWalkOffset + kStreamWarps * kStreamWalkBytes;
static_assert(kStreamSmemBytes <= 232448, "per-CTA shared memory limit");
constexpr float kStreamBf16Unit = 1.f / 32768.f;   // what bf16 sums are held in

// a / b for 0 <= a < 2^16, 0 < b <= 2^10: (a + 1/2) / b is at least 1 / 2b from a whole number, far more than the error.
__device__ __forceinline__ int small_div(int a, int b) {
  return __float2int_rd((static_cast<float>(a) + 0.5f) * __frcp_rn(static_cast<float>(b)));
}

struct StreamBatch {
  int64_t w_row;  // first weight row, over all experts
  int n0;         // the same within the expert = first result column
  int nrows;      // weight rows
  int a_row;      // first activation row
  int mrows;      // activation rows
  int wn;         // warp columns = pairs of tiles
  int wk;         // warps along K of each
};

// A CTA's part of the list of weight rows, batch by batch.
struct StreamList {
  const int* pass_first;  // passes before each expert (experts only)
  const int* row_first;   // activation rows before each expert
  int64_t row, row_end;   // in the list
  int64_t pass;
  int N, M, experts, cols, n0, e;

  __device__ void begin(int64_t from, int64_t to) {
    row = from;
    row_end = to;
    pass = row < N ? 0 : (row >> 32 ? row / N : static_cast<uint32_t>(row) / static_cast<uint32_t>(N));
    n0 = static_cast<int>(row - pass * N);
    e = 0;
    if (pass_first) {
      int hi = experts;  // last expert whose first pass is <= pass
      while (hi - e > 1) {
        const int mid = (e + hi) >> 1;
        if (pass_first[mid] <= pass) e = mid;
        else hi = mid;
      }
    }
  }
  __device__ bool next(StreamBatch& b) {
    if (row >= row_end) return false;
    const int64_t left = min(row_end - row, static_cast<int64_t>(N - n0));
    int first = 0, have = M, nth = static_cast<int>(pass);
    if (pass_first) {
      while (pass_first[e + 1] <= pass) ++e;
      first = row_first[e];
      have = row_first[e + 1] - first;
      nth = static_cast<int>(pass) - pass_first[e];
    }
    // Pairs of tiles for the 16 warps: 1-5, 7, 8 or 13-16; other counts would leave over a fifth of the warps idle.
    constexpr uint32_t kPairs = 0x1e1beu;
    const int most = static_cast<int>(min(left + 31, static_cast<int64_t>(kStreamWarps * 32)) >> 5);
    const int pairs = 31 - __clz(kPairs & ((2u << most) - 1u));
    b.w_row = static_cast<int64_t>(e) * N + n0;
    b.n0 = n0;
    b.nrows = static_cast<int>(min(left, static_cast<int64_t>(pairs * 32)));
    b.a_row = first + nth * cols;
    b.mrows = min(cols, have - nth * cols);
    b.wn = pairs;
    b.wk = small_div(kStreamWarps, pairs);
    row += b.nrows;
    n0 += b.nrows;
    if (n0 == N) {
      n0 = 0;
      ++pass;
    }
    return true;
  }
};

// Where a warp stands in the list: where it issues copies, and where it computes. Kept in shared memory (a step in every
// few thousand cycles reads it), advanced by lane 0.
struct StreamWalk {
  StreamList issue, compute;
  StreamBatch issue_batch, batch[2];  // batch: the one in use and the next
};
static_assert(sizeof(StreamWalk) <= kStreamWalkBytes, "walk");

__device__ __forceinline__ void stream_copy_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void stream_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void stream_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint2 stream_lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t stream_lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
// d = a b + c, c being (c0, c1) in both rows.
template <bool BF16>
__device__ __forceinline__ void mma_16816_first(float (&d)[4], float c0, float c1, uint32_t a0, uint32_t a1, uint32_t a2,
                                                uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
  }
}
// Four 8 x 16-byte matrices: lane l gives the address of row l & 7 of matrix l >> 3 and receives 4 bytes of row l >> 2 of each.
__device__ __forceinline__ uint4 ldmatrix_x4(uint32_t addr) {
  uint4 v;
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr));
  return v;
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
    mma_m16n8k16(d, a0, a1, a2, a3, b0, b1);
  }
}
template <bool BF16>
__device__ __forceinline__ float half_bits_to_float(uint32_t bits) {
  if (BF16) return __uint_as_float(bits << 16);
  return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}

// An array's start, 256 bytes at most, on its way to L2, in whole 16-byte pieces inside the array.
__device__ __forceinline__ void prefetch_l2(const void* base, int64_t bytes) {
  const uintptr_t begin = (reinterpret_cast<uintptr_t>(base) + 15) & ~static_cast<uintptr_t>(15);
  const uintptr_t end = (reinterpret_cast<uintptr_t>(base) + min(bytes, static_cast<int64_t>(256))) & ~static_cast<uintptr_t>(15);
  if (begin < end)
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(begin), "r"(static_cast<uint32_t>(end - begin)) : "memory");
}

struct StreamArgs {
  const uint16_t* a;
  const uint8_t* wq;
  const uint16_t* scales;
  const uint16_t* zeros;     // NULL: signed nibbles
  const int32_t* offsets;    // NULL: one expert that owns all rows
  uint16_t* out;
  int M, N, K, group, lda, ldo, experts;
  int slice_chunks, slices;  // chunks of 128 K per activation slice, and slices
  int groups;                // K / group
  int weights_ahead;         // weights and scales may be read before the dispatch ahead is complete
};

// NB: blocks of 8 activation rows a pass covers; GQ: 32-wide K blocks per scale application (group % (32 GQ) == 0).
template <bool BF16, int NB, int GQ>
__device__ void stream_body(const StreamArgs& p) {
  constexpr int kRedPitch = 20;                    // floats per activation row of a partial tile (16 + padding)
  constexpr int kTile = 8 * NB * kRedPitch;
  constexpr int kBlocks = 4 / GQ;                  // scale blocks per chunk of 128 K
  constexpr int kCols = 8 * NB;
  static_assert(kStreamWarps * 2 * kTile * 4 <= kStreamActBytes, "partial sums");

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t smem = smem_u32(smem_raw);
  int* pass_first = reinterpret_cast<int*>(smem_raw + kStreamTableOffset);  // passes before each expert
  int* row_first = pass_first + kStreamMaxExperts + 1;                       // activation rows before each expert

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int chunks = (p.K + 127) >> 7;
  // A slice holds the rows of one pass: as much of K as fits the buffers, in whole chunks (stream_slice of the host).
  const int slice_chunks = p.slice_chunks, slices = p.slices;
  const int slice_k = slice_chunks << 7;
  const int act_pitch = slice_k * 2 + 64;          // bytes; 64 mod 128: eight lanes of a 16-byte read hit all banks
  const bool acts_aligned = !((reinterpret_cast<uintptr_t>(p.a) | (static_cast<uintptr_t>(p.lda) * 2)) & 15);
  const int groups = p.groups;
  // Eight scale blocks of a row are 16 bytes to copy, or have to be picked one by one.
  const bool scales_aligned = p.group == 32 * GQ && groups % 8 == 0 &&
                              !((reinterpret_cast<uintptr_t>(p.scales) | reinterpret_cast<uintptr_t>(p.zeros)) & 15);
  // block of 32 K -> scale group without a division: exact for (K / 32) (group / 32) < 2^32
  const uint32_t group_blocks = static_cast<uint32_t>(p.group) >> 5;
  const uint32_t magic = group_blocks > 1 ? 0xffffffffu / group_blocks + 1u : 0u;
  const int last_block = (p.K >> 5) - 1;
  const int64_t w_pitch = p.K >> 1;

  // The next kernel may start once this one has waited for those ahead: what it fetches before its own wait (weights, under
  // dispatch overlap) can then be in the hands of this kernel only.
  auto wait_for_dispatches_ahead = []() {
    grid_dependency_wait();
    grid_launch_dependents();
  };
  if (p.offsets) wait_for_dispatches_ahead();
  // Experts: how many passes (8 NB activation rows each) each one needs comes from the dispatch ahead.
  int64_t passes = (p.M + kCols - 1) / kCols;
  if (p.offsets) {
    if (warp == 0) {
      int sum = 0;
      for (int e0 = 0; e0 < p.experts; e0 += 32) {
        const int e = e0 + lane;
        int lo = 0, need = 0;
        if (e < p.experts) {
          lo = min(max(p.offsets[e], 0), p.M);
          need = (min(max(p.offsets[e + 1], lo), p.M) - lo + kCols - 1) / kCols;
        }
        int incl = need;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, incl, d);
          if (lane >= d) incl += v;
        }
        if (e < p.experts) {
          pass_first[e] = sum + incl - need;
          row_first[e] = lo;
        }
        sum += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) {
        pass_first[p.experts] = sum;
        row_first[p.experts] = min(max(p.offsets[p.experts], 0), p.M);
      }
    }
    __syncthreads();
    passes = pass_first[p.experts];
  }
  const int64_t total = passes * p.N;  // weight rows to be read, over all passes
  const int64_t share = list_share(total, gridDim.x);
  StreamWalk& walk = *reinterpret_cast<StreamWalk*>(smem_raw + kStreamWalkOffset + warp * kStreamWalkBytes);
  if (lane == 0) {
    StreamList list = {p.offsets ? pass_first : nullptr, row_first, 0, 0, 0, p.N, p.M, p.experts, kCols, 0, 0};
    list.begin(min(share * blockIdx.x, total), min(share * (blockIdx.x + 1), total));
    walk.issue = list;
    walk.compute = list;
  }
  __syncwarp();
  if (warp < 3 && lane == 0) {
    // First lines of the CTA's weights, scales and zero points to L2, one array per warp: a prefetch hands no value over, so
    // it need not wait for the dispatch ahead, and the three address translations pass side by side before the ring begins.
    const StreamList& list = walk.issue;
    if (list.row < list.row_end) {
      const int64_t first = static_cast<int64_t>(list.e) * p.N + list.n0;
      if (warp == 0) prefetch_l2(p.wq + first * w_pitch, w_pitch);
      else if (warp == 1) prefetch_l2(p.scales + first * groups, groups * 2);
      else if (p.zeros) prefetch_l2(p.zeros + first * groups, groups * 2);
    }
  }
  if (!p.offsets && !p.weights_ahead) wait_for_dispatches_ahead();
  const uint32_t mask = BF16 ? 0x000f000fu : 0x00f000f0u;
  const uint32_t under = BF16 ? (p.zeros ? 0x3b803b80u : 0x3b883b88u) : (p.zeros ? 0x54005400u : 0x54805480u);
  // what the unpacked nibbles stand above their values (bf16: in units of kStreamBf16Unit): of all of them, or without the zero
  // points
  const float above = (BF16 ? 128.f : 64.f) + (p.zeros ? 0.f : 8.f);

    // ---- unit sequence of this warp: (batch, slice, its run of the slice's chunks), ahead of its use -----------------------
    bool is_more = true;
    int is_slice = slices, is_chunk = 0, is_end = 0, is_super = -1;
    uint32_t is_slot = 0, is_scales = 0;  // ring slot, and which of the two scale slots is filled next
    int is_wk = 0, is_nwk = 1;
    const uint8_t* is_w = nullptr;        // this lane's 16 bytes of row g of the pair, K = 0
    int32_t is_off1 = 0, is_off2 = 0, is_off3 = 0;  // bytes from there to rows g + 8, g + 16, g + 24 (the last row for rows behind it)
    int64_t is_s = 0;                     // first scale of row `lane` of the pair
    auto issue_run = [&]() {  // the next run of chunks that this warp has
      while (is_more) {
        if (++is_slice >= slices) {
          is_slice = 0;
          __syncwarp();  // every lane has read the batch before
          bool one_more = false;
          if (lane == 0) one_more = walk.issue.next(walk.issue_batch);
          __syncwarp();
          is_more = __any_sync(0xffffffffu, one_more);
          if (!is_more) return;
          const StreamBatch& b = walk.issue_batch;
          const int wk = small_div(warp, b.wn), wn = warp - wk * b.wn;
          const int r0 = wn * 32, last = b.nrows - 1, step = static_cast<int>(w_pitch);
          is_w = p.wq + (b.w_row + min(r0 + g, last)) * w_pitch + t * 16;
          is_off1 = (min(r0 + g + 8, last) - min(r0 + g, last)) * step;
          is_off2 = (min(r0 + g + 16, last) - min(r0 + g, last)) * step;
          is_off3 = (min(r0 + g + 24, last) - min(r0 + g, last)) * step;
          is_s = (b.w_row + min(r0 + lane, last)) * groups;
          is_wk = wk;
          is_nwk = b.wk;
        }
        if (is_wk >= is_nwk) continue;
        const int first = is_slice * slice_chunks, n = min(chunks - first, slice_chunks), per = small_div(n + is_nwk - 1, is_nwk);
        is_chunk = first + is_wk * per;
        is_end = min(is_chunk + per, first + n);
        is_super = -1;
        if (is_chunk < is_end) return;
      }
    };
    const uint32_t ring = smem + warp * (kStreamRing * kStreamUnitBytes);
    const uint32_t scale_ring = smem + kStreamScaleOffset + warp * (2 * kStreamScaleBytes);
    const uint32_t ring_piece = ring + (lane >> 2) * 64 + ((t ^ ((g >> 1) & 3)) << 4);  // 64-byte rows, pieces swizzled by row / 2
    auto issue_unit = [&]() {
      if (is_more) {
        if (is_chunk * 4 + t <= last_block) {  // K behind the end: what the slot holds meets zeros
          const uint8_t* src = is_w + (static_cast<int64_t>(is_chunk) << 6);
          const uint32_t dst = ring_piece + is_slot;
          stream_copy_16(dst, src);
          stream_copy_16(dst + 512, src + is_off1);
          stream_copy_16(dst + 1024, src + is_off2);
          stream_copy_16(dst + 1536, src + is_off3);
        }
        is_slot = is_slot == (kStreamRing - 1) * kStreamUnitBytes ? 0 : is_slot + kStreamUnitBytes;
        if (is_chunk / (2 * GQ) != is_super) {  // the next eight scale blocks of this lane's row
          is_super = is_chunk / (2 * GQ);
          const uint32_t dst = scale_ring + is_scales + lane * 16;
          is_scales ^= kStreamScaleBytes;
          if (scales_aligned) {
            stream_copy_16(dst, p.scales + is_s + is_super * 8);
            if (p.zeros) stream_copy_16(dst + 512, p.zeros + is_s + is_super * 8);
          } else {
            uint32_t sw[4] = {0, 0, 0, 0}, zw[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint32_t block = (is_super * 8 + i) * GQ;
              if (block <= static_cast<uint32_t>(last_block)) {
                const int64_t at = is_s + (group_blocks > 1 ? __umulhi(block, magic) : block);
                sw[i >> 1] |= static_cast<uint32_t>(__ldg(p.scales + at)) << ((i & 1) * 16);
                if (p.zeros) zw[i >> 1] |= static_cast<uint32_t>(__ldg(p.zeros + at)) << ((i & 1) * 16);
              }
            }
            sts128(dst, make_uint4(sw[0], sw[1], sw[2], sw[3]));
            if (p.zeros) sts128(dst + 512, make_uint4(zw[0], zw[1], zw[2], zw[3]));
          }
        }
        if (++is_chunk >= is_end) issue_run();
      }
      stream_commit();
    };

    // ---- activations: copied as they are, then ordered and summed by the thread that copied them. Warps share out the rows,
    // and each row's 16-byte pieces (the slice's K, up to whole chunks) go to the lanes of its warps in order.
    auto stage_acts = [&](const StreamBatch& b, int s, int buffer) {
      const int k0 = s * slice_k, pieces = min(slice_k, p.K - k0) >> 3;
      const int parts = small_div(kStreamWarps, b.mrows), part = small_div(warp, b.mrows), m = warp - part * b.mrows;
      if (acts_aligned && part < parts) {
        const uint32_t dst = smem + kStreamActOffset + buffer * kStreamActBytes + m * act_pitch;
        const uint16_t* src = p.a + static_cast<int64_t>(b.a_row + m) * p.lda + k0;
        for (int c = part * 32 + lane; c < pieces; c += parts * 32) stream_copy_16(dst + c * 16, src + c * 8);
      }
      stream_commit();
    };
    auto order_acts = [&](const StreamBatch& b, int s, int buffer) {
      const int k0 = s * slice_k, pieces = min(slice_k, p.K - k0) >> 3;
      const int padded = (pieces + 15) & ~15;  // to whole chunks: zeros, which the last unit multiplies
      const int parts = small_div(kStreamWarps, b.mrows), part = small_div(warp, b.mrows), m = warp - part * b.mrows;
      if (part >= parts) return;
      const uint32_t act = smem + kStreamActOffset + buffer * kStreamActBytes + m * act_pitch;
      float* sums = reinterpret_cast<float*>(smem_raw + kStreamSumOffset + buffer * kStreamSumBytes) + m;
      const uint16_t* row = p.a + static_cast<int64_t>(b.a_row + m) * p.lda + k0;
      for (int c0 = part * 32; c0 < padded; c0 += parts * 32) {
        const int c = c0 + lane;  // 4 GQ neighbouring lanes hold one scale block
        uint4 v = make_uint4(0, 0, 0, 0);
        if (c < pieces) {
          if (acts_aligned) {
            v = lds128(act + c * 16);
          } else {
            const uint16_t* src = row + c * 8;
            v.x = src[0] | static_cast<uint32_t>(src[1]) << 16;
            v.y = src[2] | static_cast<uint32_t>(src[3]) << 16;
            v.z = src[4] | static_cast<uint32_t>(src[5]) << 16;
            v.w = src[6] | static_cast<uint32_t>(src[7]) << 16;
          }
        }
        const uint32_t words[4] = {v.x, v.y, v.z, v.w};
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float lo = half_bits_to_float<BF16>(words[j] & 0xffffu), hi = half_bits_to_float<BF16>(words[j] >> 16);
          if (BF16) sum = fmaf(kStreamBf16Unit, lo, fmaf(kStreamBf16Unit, hi, sum));
          else sum += lo + hi;
        }
#pragma unroll
        for (int d = 1; d < 4 * GQ; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (c < padded) {
          // (a0, a4), (a2, a6), (a1, a5), (a3, a7)
          sts128(act + c * 16, make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.y, v.w, 0x5410),
                                          __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x7632)));
          if ((lane & (4 * GQ - 1)) == 0) sums[c / (4 * GQ) * kCols] = sum;
        }
      }
    };

    issue_run();
#pragma unroll
    for (int i = 0; i < kStreamRing; ++i) issue_unit();
    if (!p.offsets && p.weights_ahead) wait_for_dispatches_ahead();  // weights and scales were fetched ahead, activations may not be
    int turn = 0;  // which of the two batches is in use
    auto next_batch = [&](int into) {
      __syncwarp();  // every lane has read what was there
      bool one_more = false;
      if (lane == 0) one_more = walk.compute.next(walk.batch[into]);
      __syncwarp();
      return __any_sync(0xffffffffu, one_more) != 0;
    };
    bool more = next_batch(0);
    if (more) stage_acts(walk.batch[0], 0, 0);
    int since = 0;  // groups committed after the activations that the next step needs
    int buffer = 0, s = 0;
    uint32_t slot = 0, scale_slot = kStreamScaleBytes;
    float total_acc[2][NB * 4];

    while (more) {  // one step: a slice of a batch
      const bool ends = s == slices - 1;
      const StreamBatch& b = walk.batch[turn];
      // this thread's pieces of the step's activations have landed
      if (since == 0) stream_wait<0>();
      else if (since == 1) stream_wait<1>();
      else stream_wait<2>();
      order_acts(b, s, buffer);
      __syncthreads();  // everybody's pieces are in order; the buffer of the step before is free
      since = 0;
      if (!ends) {
        stage_acts(b, s + 1, buffer ^ 1);
      } else {
        more = next_batch(turn ^ 1);
        if (more) stage_acts(walk.batch[turn ^ 1], 0, buffer ^ 1);
      }
      const int wk = small_div(warp, b.wn), wn = warp - wk * b.wn;
      if (s == 0) {
#pragma unroll
        for (int j = 0; j < NB * 4; ++j) total_acc[0][j] = total_acc[1][j] = 0.f;
      }
      if (wk < b.wk) {
        const int first = s * slice_chunks, n = min(chunks - first, slice_chunks), per = small_div(n + b.wk - 1, b.wk);
        const int end = min(first + (wk + 1) * per, first + n);
        // Columns behind the last activation row repeat rows that there are: what comes out of them is not stored.
        uint32_t act_c[NB], sum_c = smem + kStreamSumOffset + buffer * kStreamSumBytes + t * 8 + wk * per * kBlocks * (kCols * 4);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          act_c[nb] = smem + kStreamActOffset + buffer * kStreamActBytes + min(nb * 8 + g, b.mrows - 1) * act_pitch + t * 16 +
                      ((wk * per) << 8);
        const uint32_t sw = (lane >> 1) & 3;
        const uint32_t w_lane = ring + lane * 64;
        const uint32_t w_at[4] = {w_lane + (sw << 4), w_lane + ((1 ^ sw) << 4), w_lane + ((2 ^ sw) << 4), w_lane + ((3 ^ sw) << 4)};
        int super = -1;
        for (int c = first + wk * per; c < end; ++c) {
          stream_wait<kStreamRing - 1>();
          __syncwarp();
          if (c / (2 * GQ) != super) {
            super = c / (2 * GQ);
            scale_slot ^= kStreamScaleBytes;
          }
          // scales and zero points of rows g, g + 8, g + 16, g + 24: the chunk's blocks are 8 / GQ bytes of each row
          const uint32_t sc_at = scale_ring + scale_slot + g * 16 + (c % (2 * GQ)) * (8 / GQ);
          uint32_t sc[4][GQ == 1 ? 2 : 1], zp[4][GQ == 1 ? 2 : 1];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if constexpr (GQ == 1) {
              const uint2 v = stream_lds64(sc_at + r * 128);
              sc[r][0] = v.x;
              sc[r][1] = v.y;
              if (p.zeros) {
                const uint2 z = stream_lds64(sc_at + r * 128 + 512);
                zp[r][0] = z.x;
                zp[r][1] = z.y;
              }
            } else if constexpr (GQ == 2) {
              sc[r][0] = lds32(sc_at + r * 128);
              if (p.zeros) zp[r][0] = lds32(sc_at + r * 128 + 512);
            } else {
              sc[r][0] = stream_lds16(sc_at + r * 128);
              if (p.zeros) zp[r][0] = stream_lds16(sc_at + r * 128 + 512);
            }
          }
#pragma unroll
          for (int blk = 0; blk < kBlocks; ++blk) {
            float acc[2][NB][4];
            float2 sum[NB];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) sum[nb] = lds64f(sum_c + blk * (kCols * 4) + nb * 32);
#pragma unroll
            for (int h = 0; h < GQ; ++h) {
              const int q = blk * GQ + h;
              uint4 bf[NB];
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) bf[nb] = lds128(act_c[nb] + (q << 6));
              const uint4 w = ldmatrix_x4(w_at[q] + slot);  // rows g, g + 8, g + 16, g + 24
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t w0 = i ? w.z : w.x, w1 = i ? w.w : w.y;
                // nibbles (0, 4), (2, 6) and (1, 5), (3, 7) of either row
                const uint32_t a0 = lop3_and_xor(BF16 ? w0 : w0 << 4, mask, under), a1 = lop3_and_xor(BF16 ? w1 : w1 << 4, mask, under);
                const uint32_t a2 = lop3_and_xor(w0 >> (BF16 ? 8 : 4), mask, under), a3 = lop3_and_xor(w1 >> (BF16 ? 8 : 4), mask, under);
                const uint32_t c0 = lop3_and_xor(BF16 ? w0 >> 4 : w0, mask, under), c1 = lop3_and_xor(BF16 ? w1 >> 4 : w1, mask, under);
                const uint32_t c2 = lop3_and_xor(w0 >> (BF16 ? 12 : 8), mask, under), c3 = lop3_and_xor(w1 >> (BF16 ? 12 : 8), mask, under);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                  if (h == 0)
                    mma_16816_first<BF16>(acc[i][nb], -above * sum[nb].x, -above * sum[nb].y, a0, a1, a2, a3, bf[nb].x, bf[nb].y);
                  else
                    mma_16816<BF16>(acc[i][nb], a0, a1, a2, a3, bf[nb].x, bf[nb].y);
                  mma_16816<BF16>(acc[i][nb], c0, c1, c2, c3, bf[nb].z, bf[nb].w);
                }
              }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {  // rows g + 8 r: half r & 1 of tile r >> 1
              const float scale = half_bits_to_float<BF16>((sc[r][blk >> 1] >> ((blk & 1) * 16)) & 0xffffu);
              if (p.zeros) {
                const float z = half_bits_to_float<BF16>((zp[r][blk >> 1] >> ((blk & 1) * 16)) & 0xffffu);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                  acc[r >> 1][nb][2 * (r & 1)] = fmaf(-z, sum[nb].x, acc[r >> 1][nb][2 * (r & 1)]);
                  acc[r >> 1][nb][2 * (r & 1) + 1] = fmaf(-z, sum[nb].y, acc[r >> 1][nb][2 * (r & 1) + 1]);
                }
              }
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                  total_acc[r >> 1][nb * 4 + 2 * (r & 1) + j] =
                      fmaf(scale, acc[r >> 1][nb][2 * (r & 1) + j], total_acc[r >> 1][nb * 4 + 2 * (r & 1) + j]);
            }
          }
          slot = slot == (kStreamRing - 1) * kStreamUnitBytes ? 0 : slot + kStreamUnitBytes;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) act_c[nb] += 256;
          sum_c += kBlocks * (kCols * 4);
          __syncwarp();  // every lane has read the unit: its slot may be filled again
          issue_unit();
          ++since;
        }
      }
      if (ends) {
        // the WK partial sums of each tile meet, in order of K, where this step's activations were
        __syncthreads();
        float* red = reinterpret_cast<float*>(smem_raw + kStreamActOffset + buffer * kStreamActBytes);
        if (wk < b.wk) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float* dst = red + (wk * b.wn + wn) * 2 * kTile + i * kTile;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                dst[(nb * 8 + 2 * t + (j & 1)) * kRedPitch + g + (j >> 1) * 8] = total_acc[i][nb * 4 + j];
          }
        }
        __syncthreads();
        // a warp takes 32 columns of one activation row at a time
        for (int i = warp; i < b.mrows * b.wn; i += kStreamWarps) {
          const int m = small_div(i, b.wn), n = (i - m * b.wn) * 32 + lane;
          if (n < b.nrows) {
            const float* src = red + (n >> 4) * kTile + m * kRedPitch + (n & 15);
            float v = 0.f;
            for (int w = 0; w < b.wk; ++w) v += src[w * b.wn * 2 * kTile];
            uint16_t bits;
            if (BF16) bits = __bfloat16_as_ushort(__float2bfloat16_rn(v * (1.f / kStreamBf16Unit)));
            else bits = __half_as_ushort(__float2half_rn(v));
            p.out[static_cast<int64_t>(b.a_row + m) * p.ldo + b.n0 + n] = bits;
          }
        }
        turn ^= 1;
        s = 0;
      } else {
        ++s;
      }
      buffer ^= 1;
    }
    stream_wait<0>();
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
           uint16_t* out, int M, int N, int K, int group, int lda, int ldo, int experts, int slice_chunks, int slices,  \
           int groups, int weights_ahead) {                                                                                \
    b200::StreamArgs p = {a, wq, scales, zeros, offsets, out, M, N, K, group, lda, ldo, experts,                  \
                          slice_chunks, slices, groups, weights_ahead};                                                    \
    b200::stream_by_group<BF16, NB>(p);                                                                                   \
  }
B200_W4A16_STREAM(b200_w4a16_stream_f16_r8, false, 1)
B200_W4A16_STREAM(b200_w4a16_stream_f16_r16, false, 2)
B200_W4A16_STREAM(b200_w4a16_stream_bf16_r8, true, 1)
B200_W4A16_STREAM(b200_w4a16_stream_bf16_r16, true, 2)
#undef B200_W4A16_STREAM
