// The experts' products with 4-bit weights where experts have more than a few rows each: tcgen05 with the dequantised weights
// as the tensor-memory operand.
//
//   out[i, n] = round(sum_k a[i, k] w16[e, n, k]),  w16 = round16((q - z) s)   for rows offsets[e] <= i < offsets[e + 1]
//
// The one rounding that is not the result's: a weight enters the tensor core as f16 or bf16, off by half a step of its own value
// (with a fractional zero point q - z is rounded as well). Its error is random from weight to weight: together with the result's
// rounding it measures 1.3 times the result's alone (root mean square, relative: bf16 0.0022 for 0.0017, f16 0.00028 for 0.00021). Scaling group sums in f32 instead would need the accumulator back in
// registers for every group, four times the tensor time. Sums are f32 in tensor memory.
//
// Roles as in b200_w4a16_gemm_wt: warp 0 fetches activation tiles (TMA, 128-byte swizzle, boxes of 64 rows x 64 K), warp 3 raw
// weight tiles (128 rows x 128 K), warps 8 and up expand weights into tensor memory (a thread owns a weight row = a lane), one
// thread of warp 1 issues the matrix instructions two K blocks at a time, warps 4-7 bring the transposed accumulator back.
// What differs: tiles are (expert, 128 weight rows, up to 256 activation rows), listed from the device's row offsets by every
// CTA itself. An expert's rows are cut into equal parts of a multiple of 16 (260 rows are 2 x 144, not 256 + 16), and the
// instruction is only as wide as the part. Rows of the next expert that a box brings along fall into accumulator columns
// that are not read; a piece of 64 result rows that the expert does not fill, or whose last columns are a part of 16 bytes, is
// stored by the threads, others by TMA.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "sm100_ptx.cuh"
#include "w4a16_decode.cuh"

namespace b200 {

constexpr int kExWRows = 128;                                // weight rows per tile = tensor-memory lanes
constexpr int kExRawStageBytes = kExWRows * 64;              // 128 rows x 128 int4
constexpr int kExAStageColumns = 32;                         // 64 K as pairs of 16 bits
constexpr int kExOutRows = 64;
constexpr int kExOutStageBytes = kExOutRows * kExWRows * 2;
constexpr int kExMaxExperts = 1024;
constexpr int kExBarrierBytes = 512;
constexpr int kExTableBytes = 2 * (kExMaxExperts + 1) * 4 + 56;

// Two shapes. Tiles of 256 activation rows: the matrix instructions bound it, two groups of dequant warps keep up. Tiles of 64
// rows, for experts with few rows: expanding the weights bounds it, four groups, and the memory that activations do not need
// holds more raw weights on their way.
template <int AROWS>
struct Ex {
  static constexpr bool kSmall = AROWS == 64;
  static constexpr int kActStages = kSmall ? 8 : 4;
  static constexpr int kActStageBytes = AROWS * 128;
  static constexpr int kRawStages = kSmall ? 12 : 6;
  static constexpr int kPairStages = kSmall ? 6 : 4;         // pairs of K blocks (128 K) expanded in tensor memory
  static constexpr int kAStages = 2 * kPairStages;
  static constexpr int kGroups = kSmall ? 4 : 2;             // dequant groups of four warps
  static constexpr int kThreads = 256 + 128 * kGroups;
  static constexpr int kSmemBytes = 1024 + kActStages * kActStageBytes + kRawStages * kExRawStageBytes + 2 * kExOutStageBytes +
                                    kExBarrierBytes + kExTableBytes;
  static_assert(kSmemBytes <= 232448, "per-CTA shared memory limit");
  static_assert(AROWS + kAStages * kExAStageColumns <= 512, "tensor memory columns");
};

struct alignas(128) ExWorkspace {
  uint8_t map_a[128];    // 16-bit [rows, K], 128-byte swizzle, box 64 x 64
  uint8_t map_w[128];    // u8 [experts * N, K/2], 64-byte swizzle, box 64 x 128
  uint8_t map_out[128];  // 16-bit [rows, N], no swizzle, box 128 x 64
  uint32_t status[18];
  uint32_t note[14];     // what prepare() built the maps for
};
constexpr uint32_t kExNoteMagic = 0x45585034u;

__device__ __forceinline__ void ex_report(ExWorkspace* ws, uint32_t code, uint32_t info) {
  if (atomicCAS(&ws->status[0], 0u, code) == 0u) ws->status[1] = info;
}

struct ExTile {
  int e, n0, row0, rows;  // rows of the tile, at least one
};

// Walks the tiles of one CTA; every role has its own.
template <int AROWS>
struct ExWalk {
  const int* first;  // tiles before each expert
  const int* row;    // rows before each expert
  int e;
  __device__ ExTile at(int t) {
    while (first[e + 1] <= t) ++e;
    const int local = t - first[e], count = row[e + 1] - row[e];
    const int parts = (count + AROWS - 1) / AROWS;
    const int per = ((count + parts - 1) / parts + 15) & ~15;
    const int tn = local / parts, tm = local - tn * parts;
    ExTile x;
    x.e = e;
    x.n0 = tn * kExWRows;
    x.row0 = row[e] + tm * per;
    x.rows = min(per, count - tm * per);
    return x;
  }
};

// True in one thread of the warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

template <bool BF16>
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (BF16) asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (BF16) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ uint32_t twice(uint32_t bits) { return __byte_perm(bits, 0u, 0x1010u); }

// What takes the offset of a stored nibble and its zero point away in one operation, exactly, for a whole zero point: the
// nibbles arrive as 1024 + n and 64 + n (f16: low and high nibble of a byte) or 128 + n (bf16).
template <bool BF16>
__device__ __forceinline__ uint32_t offset_of(float z) {
  if (BF16) return twice(__bfloat16_as_ushort(__float2bfloat16_rn(128.f + z)));
  return as_u32(__floats2half2_rn(-1024.f - z, -64.f - z));
}

// Eight weights in memory order, (w0, w1), (w2, w3), ...: (stored nibble) - (offset) as exact small integers. `flip` turns
// two's complement into value + 8.
template <bool BF16, bool FLIP>
__device__ __forceinline__ void unpack8_minus(uint32_t v, uint32_t offset, uint32_t (&q)[4]) {
  if (BF16) {
    const uint32_t high = v >> 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t pair;  // byte j of v in the low half, of v >> 4 in the high half
      asm("prmt.b32 %0, %1, %2, %3;" : "=r"(pair) : "r"(v), "r"(high), "r"(0x4400u + 0x1111u * j));
      q[j] = sub2<true>(lop3_and_xor(pair, 0x000f000fu, FLIP ? 0x43084308u : 0x43004300u), offset);
    }
  } else {
    const __half2 mul = __halves2half2(__float2half_rn(1.f), __float2half_rn(0.0625f));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t rep;
      asm("prmt.b32 %0, %1, %1, %2;" : "=r"(rep) : "r"(v), "r"(0x1111u * j));  // byte j in every byte
      // low half: 1024 + n_lo; high half: 1024 + 16 n_hi
      q[j] = as_u32(__hfma2(as_half2(lop3_and_xor(rep, 0x00f0000fu, FLIP ? 0x64806408u : 0x64006400u)), mul, as_half2(offset)));
    }
  }
}

template <int AROWS, bool BF16, bool ZEROS>
__device__ void experts_body(const uint16_t* __restrict__ scales, const uint16_t* __restrict__ zeros,
                             const int32_t* __restrict__ offsets, uint16_t* __restrict__ out, const void* a, const void* wq,
                             ExWorkspace* __restrict__ ws, int rows, int N, int K, int group, int lda, int ldo, int experts) {
  using X = Ex<AROWS>;
  constexpr int kGroups = X::kGroups;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t raw_base = smem_base + X::kActStages * X::kActStageBytes;
  const uint32_t out_base = raw_base + X::kRawStages * kExRawStageBytes;
  const uint32_t bars = out_base + 2 * kExOutStageBytes;
  uint8_t* bars_gen = smem_gen + (bars - smem_base);
  int* tile_first = reinterpret_cast<int*>(bars_gen + kExBarrierBytes);
  int* row_first = tile_first + kExMaxExperts + 1;
  auto act_early = [&](int i) { return bars + 8u * i; };  // "the first block of a pair is done with activation stage i"
  auto raw_full = [&](int i) { return bars + 8u * (X::kActStages + i); };
  auto raw_empty = [&](int i) { return bars + 8u * (X::kActStages + X::kRawStages + i); };
  auto a_full = [&](int i) { return bars + 8u * (X::kActStages + 2 * X::kRawStages + i); };
  auto a_empty = [&](int i) { return bars + 8u * (X::kActStages + 2 * X::kRawStages + X::kPairStages + i); };
  constexpr int kNumRingBars = X::kActStages + 2 * X::kRawStages + 2 * X::kPairStages;
  const uint32_t d_full = bars + 8u * kNumRingBars, d_empty = bars + 8u * (kNumRingBars + 1);
  const uint32_t tmem_slot = bars + 8u * (kNumRingBars + 2);
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(bars_gen + 8 * (kNumRingBars + 2));
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(bars_gen + 8 * (kNumRingBars + 2) + 4);
  static_assert(8 * (kNumRingBars + 3) <= kExBarrierBytes, "barrier area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_n = (N + kExWRows - 1) / kExWRows;
  const int num_kb = ((K + 127) >> 7) << 1;  // whole pairs of K blocks; TMA fills K behind the end with zeros

  if (threadIdx.x == 0) {
    for (int i = 0; i < X::kActStages; ++i) mbar_init(act_early(i), 1);
    for (int i = 0; i < X::kRawStages; ++i) {
      mbar_init(raw_full(i), 1);
      mbar_init(raw_empty(i), 4);
    }
    for (int i = 0; i < X::kPairStages; ++i) {
      mbar_init(a_full(i), 5);  // the four warps of a dequant group + the activation tiles' expect_tx
      mbar_init(a_empty(i), 1);
    }
    mbar_init(d_full, 1);
    mbar_init(d_empty, 4);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  grid_dependency_wait();
  grid_launch_dependents();  // behind the wait: whoever starts now finds no other kernel unfinished
  if (warp == 1) {  // the tile list: rows and tiles before each expert
    // A workspace that was not prepared for these operands holds no maps, or others': nothing is copied through it.
    const auto low = [](const void* p) { return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)); };
    const auto high = [](const void* p) { return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) >> 32); };
    const uint32_t want[14] = {kExNoteMagic, BF16, static_cast<uint32_t>(rows), static_cast<uint32_t>(N), static_cast<uint32_t>(K),
                               static_cast<uint32_t>(lda), static_cast<uint32_t>(ldo), static_cast<uint32_t>(experts),
                               low(a), high(a), low(wq), high(wq), low(out), high(out)};
    bool same = true;
#pragma unroll
    for (int i = 0; i < 14; ++i) same = same && (lane != i || ws->note[i] == want[i]);
    const bool prepared = __all_sync(0xffffffffu, same);
    if (!prepared && lane == 0 && blockIdx.x == 0) ex_report(ws, kStatusBadArgument, 0);
    int sum = 0;
    for (int e0 = 0; e0 < experts; e0 += 32) {
      const int e = e0 + lane;
      int lo = 0, need = 0;
      if (e < experts) {
        lo = min(max(offsets[e], 0), rows);
        const int hi = min(max(offsets[e + 1], lo), rows);
        need = (hi - lo + AROWS - 1) / AROWS * tiles_n;
      }
      int incl = need;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += v;
      }
      if (e < experts) {
        tile_first[e] = sum + incl - need;
        row_first[e] = lo;
      }
      sum += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      tile_first[experts] = prepared ? sum : 0;
      row_first[experts] = min(max(offsets[experts], 0), rows);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot_ptr;
  const uint32_t tmem_a = tmem_base + AROWS;
  const int num_tiles = tile_first[experts];
  ExWalk<AROWS> walk = {tile_first, row_first, 0};

  // The single-thread roles: the whole warp walks the loop and one elected thread issues, so that the operands of copies and
  // matrix instructions are values which the compiler knows to be uniform and need no move each from a thread's registers
  // (per pair of K blocks the issuing thread alone took 840 cycles otherwise, against 1024 of the tensor pipe; it takes 330).
  const int tiles = __shfl_sync(0xffffffffu, num_tiles, 0);
  if (warp == 0) {
    // -------- TMA producer of the activation tiles ----------------------------------------------------
    const bool leader = elect_one();
    if (leader) tensormap_fence_acquire(ws->map_a);
    uint32_t it = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const ExTile x = walk.at(t);
      const int row0 = __shfl_sync(0xffffffffu, x.row0, 0), boxes = __shfl_sync(0xffffffffu, (x.rows + 63) >> 6, 0);
      const uint32_t bytes = 2 * boxes * 64 * 128;
      for (int kb = 0; kb < num_kb; kb += 2, it += 2) {
        const uint32_t pair = it >> 1, prev = pair - X::kActStages / 2;
        const uint32_t full = a_full(pair % X::kPairStages);
        const uint32_t dst0 = smem_base + (it % X::kActStages) * X::kActStageBytes;
        const uint32_t dst1 = smem_base + ((it + 1) % X::kActStages) * X::kActStageBytes;
        // The stages' previous tenants were the blocks of pair - stages / 2; their MMAs' completion is what that pair's "empty"
        // barrier reports. With four stages of 256 rows that lead would be less than a load takes: the issuer reports the
        // first block's MMAs on a barrier of its own, and each stage is filled again as soon as its block is done.
        bool waited = true;
        if (pair >= X::kActStages / 2) {
          const uint32_t prev_block = it - X::kActStages;
          if (X::kSmall) waited = __all_sync(0xffffffffu, mbar_wait(a_empty(prev % X::kPairStages), (prev / X::kPairStages) & 1, abort_flag));
          else waited = __all_sync(0xffffffffu, mbar_wait(act_early(prev_block % X::kActStages), (prev_block / X::kActStages) & 1, abort_flag));
        }
        if (waited) {
          if (leader) {
            mbar_arrive_expect_tx(full, bytes);
            tma_load_3d(dst0, ws->map_a, full, kb * 64, row0, 0);
            if (X::kSmall) tma_load_3d(dst1, ws->map_a, full, (kb + 1) * 64, row0, 0);
            if (boxes > 1) tma_load_3d(dst0 + 64 * 128, ws->map_a, full, kb * 64, row0 + 64, 0);
            if (boxes > 2) tma_load_3d(dst0 + 128 * 128, ws->map_a, full, kb * 64, row0 + 128, 0);
            if (boxes > 3) tma_load_3d(dst0 + 192 * 128, ws->map_a, full, kb * 64, row0 + 192, 0);
          }
          __syncwarp();
          if (!X::kSmall && pair >= X::kActStages / 2)
            waited = __all_sync(0xffffffffu, mbar_wait(a_empty(prev % X::kPairStages), (prev / X::kPairStages) & 1, abort_flag));
        }
        if (!waited) {
          if (leader) {
            ex_report(ws, kStatusTimeoutEmpty, it);
            *abort_flag = 1;
          }
          ok = false;
          break;
        }
        if (!X::kSmall && leader) {
          tma_load_3d(dst1, ws->map_a, full, (kb + 1) * 64, row0, 0);
          if (boxes > 1) tma_load_3d(dst1 + 64 * 128, ws->map_a, full, (kb + 1) * 64, row0 + 64, 0);
          if (boxes > 2) tma_load_3d(dst1 + 128 * 128, ws->map_a, full, (kb + 1) * 64, row0 + 128, 0);
          if (boxes > 3) tma_load_3d(dst1 + 192 * 128, ws->map_a, full, (kb + 1) * 64, row0 + 192, 0);
        }
        __syncwarp();
      }
    }
  } else if (warp == 3) {
    // -------- TMA producer of the raw weights: 128 K per stage ------------------------------------------
    const bool leader = elect_one();
    if (leader) tensormap_fence_acquire(ws->map_w);
    uint32_t raw_it = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const ExTile x = walk.at(t);
      const int w_row = __shfl_sync(0xffffffffu, x.e * N + x.n0, 0);
      for (int g = 0; g < (num_kb >> 1); ++g, ++raw_it) {
        const uint32_t rs = raw_it % X::kRawStages;
        if (!__all_sync(0xffffffffu, mbar_wait(raw_empty(rs), ((raw_it / X::kRawStages) & 1) ^ 1, abort_flag))) {
          if (leader) {
            ex_report(ws, kStatusTimeoutEmpty, 0x10000u | raw_it);
            *abort_flag = 1;
          }
          ok = false;
          break;
        }
        if (leader) {
          mbar_arrive_expect_tx(raw_full(rs), kExRawStageBytes);
          tma_load_3d(raw_base + rs * kExRawStageBytes, ws->map_w, raw_full(rs), g * 64, w_row, 0);
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    // -------- MMA issuer -----------------------------------------------------------------------------------
    const uint64_t desc0 = make_smem_desc(smem_base, 16, 1024);
    constexpr uint32_t kStageUnits = X::kActStageBytes >> 4;
    const bool leader = elect_one();
    const uint32_t d_tmem = __shfl_sync(0xffffffffu, tmem_base, 0), a_tmem = d_tmem + AROWS;
    uint32_t it = 0, local_tile = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++local_tile) {
      const ExTile x = walk.at(t);
      const uint32_t n = __shfl_sync(0xffffffffu, static_cast<uint32_t>(x.rows + 15) & ~15u, 0);
      const uint32_t idesc = make_instr_desc(1u, BF16 ? 1u : 0u, BF16 ? 1u : 0u, 0u, 0u, kExWRows, n);
      if (!__all_sync(0xffffffffu, mbar_wait(d_empty, (local_tile & 1) ^ 1, abort_flag))) {
        if (leader) {
          ex_report(ws, kStatusTimeoutTmemEmpty, local_tile);
          *abort_flag = 1;
        }
        break;
      }
      tc_fence_after_sync();
      for (int kb = 0; kb < num_kb; kb += 2, it += 2) {
        const uint32_t pair = it >> 1, ps = pair % X::kPairStages;
        if (!__all_sync(0xffffffffu, mbar_wait(a_full(ps), (pair / X::kPairStages) & 1, abort_flag))) {
          if (leader) {
            ex_report(ws, kStatusTimeoutDequant, it);
            *abort_flag = 1;
          }
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint64_t b0 = desc0 + (it % X::kActStages) * kStageUnits, b1 = desc0 + ((it + 1) % X::kActStages) * kStageUnits;
        const uint32_t a0 = a_tmem + (it % X::kAStages) * kExAStageColumns, a1 = a_tmem + ((it + 1) % X::kAStages) * kExAStageColumns;
        if (leader) {
          if (kb == 0) mma_f16_ts_first(d_tmem, a0, b0, idesc);
          else mma_f16_ts_more(d_tmem, a0, b0, idesc);
          mma_f16_ts_more(d_tmem, a0 + 8, b0 + 2, idesc);
          mma_f16_ts_more(d_tmem, a0 + 16, b0 + 4, idesc);
          mma_f16_ts_more(d_tmem, a0 + 24, b0 + 6, idesc);
          if (!X::kSmall) tc_commit(act_early(it % X::kActStages));
          mma_f16_ts_more(d_tmem, a1, b1, idesc);
          mma_f16_ts_more(d_tmem, a1 + 8, b1 + 2, idesc);
          mma_f16_ts_more(d_tmem, a1 + 16, b1 + 4, idesc);
          mma_f16_ts_more(d_tmem, a1 + 24, b1 + 6, idesc);
          tc_commit(a_empty(ps));
        }
        __syncwarp();
      }
      if (ok && leader) tc_commit(d_full);
      __syncwarp();
    }
  } else if (warp >= 4 && warp < 8) {
    // -------- epilogue: D[n, i] -> staged [i, n] pieces -> TMA stores, or the threads' own ---------------------
    const int qd = warp & 3, et = threadIdx.x - 128;
    const bool issuer = et == 0;
    if (issuer) tensormap_fence_acquire(ws->map_out);
    uint32_t local_tile = 0, piece_it = 0;
    for (int t = blockIdx.x; t < num_tiles; t += gridDim.x, ++local_tile) {
      const ExTile x = walk.at(t);
      if (!__all_sync(0xffffffffu, mbar_wait(d_full, local_tile & 1, abort_flag))) {
        if (lane == 0) {
          ex_report(ws, kStatusTimeoutTmemFull, local_tile);
          *abort_flag = 1;
        }
        break;
      }
      tc_fence_after_sync();
      const int pieces = (x.rows + kExOutRows - 1) / kExOutRows;
      for (int pc = 0; pc < pieces; ++pc) {
        uint32_t v0[32], v1[32];
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(qd * 32) << 16) + pc * kExOutRows;
        tmem_ld_32x32(taddr, v0);
        tmem_ld_32x32(taddr + 32, v1);
        tc_wait_ld();
        if (pc == pieces - 1) {  // the accumulator is in registers / already stored: the next tile's MMAs may start
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(d_empty);
        }
        const uint32_t stage = out_base + (piece_it & 1) * kExOutStageBytes;
        if (issuer) bulk_wait_group_read<1>();  // the store issued from this buffer two pieces ago has read it
        named_barrier_sync(1, 128);
        const uint32_t dst = stage + (qd * 32 + lane) * 2;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          uint16_t h0, h1;
          if (BF16) {
            h0 = __bfloat16_as_ushort(__float2bfloat16_rn(__uint_as_float(v0[j])));
            h1 = __bfloat16_as_ushort(__float2bfloat16_rn(__uint_as_float(v1[j])));
          } else {
            h0 = __half_as_ushort(__float2half_rn(__uint_as_float(v0[j])));
            h1 = __half_as_ushort(__float2half_rn(__uint_as_float(v1[j])));
          }
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst + j * (kExWRows * 2)), "h"(h0) : "memory");
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst + (j + 32) * (kExWRows * 2)), "h"(h1) : "memory");
        }
        fence_proxy_async_smem();
        named_barrier_sync(1, 128);
        const int left = min(x.rows - pc * kExOutRows, kExOutRows), y = x.row0 + pc * kExOutRows;
        // A TMA store writes whole 16-byte pieces: where N ends inside one, it would write behind N as well.
        if (left == kExOutRows && (N % 8 == 0 || x.n0 + kExWRows <= N)) {
          if (issuer) tma_store_2d(ws->map_out, stage, x.n0, y);
        } else {
          for (int i = et; i < left * (kExWRows / 8); i += 128) {
            const int r = i >> 4, c = (i & 15) * 8, n = x.n0 + c;
            const uint4 v = lds128(stage + r * (kExWRows * 2) + c * 2);
            uint16_t* o = out + static_cast<int64_t>(y + r) * ldo + n;
            if (n + 8 <= N) {
              *reinterpret_cast<uint4*>(o) = v;
            } else {
              const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (n + j < N) o[j] = static_cast<uint16_t>(words[j >> 1] >> ((j & 1) * 16));
            }
          }
        }
        if (issuer) bulk_commit_group();  // one group per piece, empty where the threads store
        ++piece_it;
      }
    }
    if (issuer) bulk_wait_group<0>();
  } else if (warp >= 8) {
    // -------- dequant: raw int4 (64-byte swizzled rows) -> 64 columns of this thread's TMEM lane, a pair of K blocks at a time --
    const int td = threadIdx.x - 256;
    const int r = td & 127;   // weight row of the tile = TMEM lane
    const uint32_t grp = td >> 7;  // pairs grp, grp + groups, ... of the CTA's sequence
    const int groups = K / group;
    // Scale groups that a pair (128 K) holds: 1, 2 or 4, aligned with it; or any (a group of 96), one per 32 K.
    const int per_pair = group % 128 == 0 ? 1 : group == 64 ? 2 : 4;
    const bool direct = group == 32 || group == 64;   // a pair's scales are neighbours in memory
    const bool vector = direct && groups % per_pair == 0 && !((reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(zeros)) &
                                                             (2 * per_pair - 1));
    // block of 32 K -> scale group without a division per pair: exact for (K / 32) (group / 32) < 2^32
    const uint32_t group_blocks = static_cast<uint32_t>(group) >> 5;
    const uint32_t magic = group_blocks > 1 ? 0xffffffffu / group_blocks + 1u : 0u;
    const uint32_t last_block = (static_cast<uint32_t>(K) >> 5) - 1u;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int pairs = num_kb >> 1;
    const uint32_t sw_raw = (r >> 1) & 3;
    uint32_t pair_base = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < num_tiles && ok; t += gridDim.x, pair_base += pairs) {
      const ExTile x = walk.at(t);
      // rows behind the expert's last one are expanded with its scales and never stored
      const int64_t srow = (static_cast<int64_t>(x.e) * N + min(x.n0 + r, N - 1)) * groups;
      const uint16_t* s_row = scales + srow;
      const uint16_t* z_row = ZEROS ? zeros + srow : nullptr;
      uint32_t next_s[4] = {0, 0, 0, 0}, next_z[4] = {0, 0, 0, 0};  // the group's next pair: loaded one turn ahead
      auto fetch = [&](int p) {
        if (vector) {
          if (per_pair == 4) {
            const uint2 s = *reinterpret_cast<const uint2*>(s_row + p * 4);
            next_s[0] = s.x & 0xffffu;
            next_s[1] = s.x >> 16;
            next_s[2] = s.y & 0xffffu;
            next_s[3] = s.y >> 16;
            if (ZEROS) {
              const uint2 z = *reinterpret_cast<const uint2*>(z_row + p * 4);
              next_z[0] = z.x & 0xffffu;
              next_z[1] = z.x >> 16;
              next_z[2] = z.y & 0xffffu;
              next_z[3] = z.y >> 16;
            }
          } else {
            const uint32_t s = *reinterpret_cast<const uint32_t*>(s_row + p * 2);
            next_s[0] = next_s[1] = s & 0xffffu;
            next_s[2] = next_s[3] = s >> 16;
            if (ZEROS) {
              const uint32_t z = *reinterpret_cast<const uint32_t*>(z_row + p * 2);
              next_z[0] = next_z[1] = z & 0xffffu;
              next_z[2] = next_z[3] = z >> 16;
            }
          }
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (c == 0 || per_pair == 4 || (per_pair == 2 && c == 2)) {
              // behind K: scale and zero point 0, as (0 - z) s of the last group may be an infinity
              const uint32_t block = static_cast<uint32_t>(p) * 4 + c;
              const uint32_t g = group_blocks > 1 ? __umulhi(block, magic) : block;
              const bool there = block <= last_block;
              next_s[c] = there ? s_row[g] : 0;
              if (ZEROS) next_z[c] = there ? z_row[g] : 0;
            } else {
              next_s[c] = next_s[c - 1];
              next_z[c] = next_z[c - 1];
            }
          }
        }
      };
      int p = (grp - pair_base) & (kGroups - 1);
      if (p < pairs) fetch(p);
      for (; p < pairs; p += kGroups) {
        const uint32_t pair = pair_base + p, ps = pair % X::kPairStages;
        const int rs = pair % X::kRawStages;
        uint32_t s2[4], off2[4], z2[4];
        bool whole = true;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          s2[c] = twice(next_s[c]);
          if (ZEROS) {
            const float z = BF16 ? __uint_as_float(next_z[c] << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(next_z[c])));
            whole = whole && z == rintf(z) && fabsf(z) <= 64.f;
            off2[c] = offset_of<BF16>(z);
            z2[c] = twice(next_z[c]);
          } else {
            off2[c] = offset_of<BF16>(8.f);
            z2[c] = 0;
          }
        }
        if (p + kGroups < pairs) fetch(p + kGroups);
        const bool fast = !ZEROS || __all_sync(0xffffffffu, whole);
        if (!__all_sync(0xffffffffu, mbar_wait(raw_full(rs), (pair / X::kRawStages) & 1, abort_flag))) {
          if (lane == 0) {
            ex_report(ws, kStatusTimeoutFull, 0x10000u | pair);
            *abort_flag = 1;
          }
          ok = false;
          break;
        }
        if (!__all_sync(0xffffffffu, mbar_wait(a_empty(ps), ((pair / X::kPairStages) & 1) ^ 1, abort_flag))) {
          if (lane == 0) {
            ex_report(ws, kStatusTimeoutEmpty, 0x20000u | pair);
            *abort_flag = 1;
          }
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t raw_row = raw_base + rs * kExRawStageBytes + r * 64;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t v[32];  // v[16 c + 4 i + j]: weights 32 c + 8 i + 2 j and the next one, one column of the stage
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int chunk = h * 2 + c;  // 16-byte chunk of the 64-byte raw row = 32 weights
            const uint4 w = lds128(raw_row + ((chunk ^ sw_raw) << 4));
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
            if (fast) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint32_t q[4];
                unpack8_minus<BF16, !ZEROS>(words[i], off2[chunk], q);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[16 * c + 4 * i + j] = mul2<BF16>(q[j], s2[chunk]);
              }
            } else {  // a zero point that is no small whole number: taken away in its own, rounding, step
              const uint32_t plain = offset_of<BF16>(0.f);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint32_t q[4];
                unpack8_minus<BF16, false>(words[i], plain, q);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[16 * c + 4 * i + j] = mul2<BF16>(sub2<BF16>(q[j], z2[chunk]), s2[chunk]);
              }
            }
          }
          tmem_st_32x32(tmem_a + lane_base + ((pair * 2 + h) % X::kAStages) * kExAStageColumns, v);
        }
        tc_wait_st();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(a_full(ps));
          mbar_arrive(raw_empty(rs));
        }
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {  // copies in flight land before the block's shared memory is given up
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) {
    }
  }
  if (warp == 2) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace b200

// Bindings: scales, zero points (NULL: signed weights), row offsets, result, activations, weights (both reached through the
// workspace's maps; named to be compared with its note), workspace.
#define B200_W4A16_EXPERTS(NAME, AROWS, BF16)                                                                              \
  extern "C" __global__ void __launch_bounds__(b200::Ex<AROWS>::kThreads, 1)                                               \
      NAME(const uint16_t* scales, const uint16_t* zeros, const int32_t* offsets, uint16_t* out, const void* a,            \
           const void* wq, void* ws, int rows, int N, int K, int group, int lda, int ldo, int experts) {                   \
    b200::ExWorkspace* w = reinterpret_cast<b200::ExWorkspace*>(ws);                                                       \
    if (zeros)                                                                                                             \
      b200::experts_body<AROWS, BF16, true>(scales, zeros, offsets, out, a, wq, w, rows, N, K, group, lda, ldo, experts);  \
    else                                                                                                                   \
      b200::experts_body<AROWS, BF16, false>(scales, zeros, offsets, out, a, wq, w, rows, N, K, group, lda, ldo, experts); \
  }
B200_W4A16_EXPERTS(b200_w4a16_experts_f16, 256, false)
B200_W4A16_EXPERTS(b200_w4a16_experts_bf16, 256, true)
B200_W4A16_EXPERTS(b200_w4a16_experts_r64_f16, 64, false)
B200_W4A16_EXPERTS(b200_w4a16_experts_r64_bf16, 64, true)
#undef B200_W4A16_EXPERTS
