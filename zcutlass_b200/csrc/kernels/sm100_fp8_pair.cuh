// 8-bit block-scaled product on CTA pairs (cta_group::2), 256 x 256 output
// tiles, persistent: the large products (prefill, training).
//
//   D[m, n] = sum_b sa(m, b) * sb(n, b) * (A_b B_b^T)[m, n]  (+ bias[n])
//
// Per block of 128 k the pair's leader issues 4 MMAs of 256 x 256 x 32 into one
// of two 256-column TMEM buffers; each CTA holds its 128 rows x 256 columns.
// Eight accumulation warps per CTA (two per TMEM quarter, 128 columns each)
// read the buffer and add it, scaled, into 128 32-bit accumulators per thread,
// while the MMAs of the next block fill the other buffer.
//
// What bounds it: power for long products (8192 x 28672 x 4096 takes 615 us on
// zeros; on random bits 770-800 in a burst and 884 sustained, at 990 W and 1.4
// GHz with the power cap active), else a buffer's turnaround. At full rate a
// block takes the tensor pipe 512 cycles (531 measured), TMEM reads and 32-bit
// fma 343 by themselves. A buffer's turnaround (MMAs, commit, read, arrival at the
// leader) must fit two blocks' time, so nothing slow may sit on it:
//  - the warp that issues MMAs walks its loop as a whole, with its state in
//    uniform registers and one lane issuing (per-lane descriptors alone halved
//    the MMA rate: the accumulation warps leave few issue slots);
//  - scales never pass through the accumulation warps' registers as loads in
//    flight (a wait loop holds them up until the load returns): two otherwise
//    idle warps, one per TMEM buffer, put each block's scales in shared memory
//    and complete the buffer's `tmem_full` barrier together with the commit.
//    The scales are handed back on a barrier of this CTA, `read`;
//  - the arrival at the leader's `tmem_empty` hands back TMEM alone, so it is
//    not a release of memory to the cluster.
//
// Measured (random bits, 20 in a row): 8192 x 9472 x 4096 254 us, 2500 TFLOP/s;
// with a scale per row of B 334 us, 1900 TFLOP/s.
//
// With 128 x 128 weight scales the factor is one product per thread and block.
// With a scale per row of B (kRows) TMEM is read as 16 x 8 fragments, in which
// a thread meets only 32 of the 128 columns: a quarter of the shared-memory
// reads that a row per thread would need. Such loads bring 16 of 32 lanes at a
// time; they bound this variant. Cycles per block, the accumulation alone: a row
// per thread with one scale 343, fragments 720 (565 with the scales in
// registers), a row per thread with scales from shared memory 764, part of the
// columns each way 748 to 804.
//
// Roles per CTA: warp 0 TMA producer, warp 1 TMEM allocation and, in the
// leader, MMA issue, warps 2-3 scales; warps 4-11 accumulate, then write the
// tile (registers -> swizzled shared memory -> TMA, or row by row where D is
// ragged or unaligned) while the next tile's first blocks run. 128 accumulators
// and the TMEM chunks need more than the 168 registers three warps per SM
// sub-partition get: the first warpgroup hands registers over
// (128 x 72 + 256 x 216 = 384 x 168).
#pragma once

#include "sm100_fp8_common.cuh"

namespace zcb {

struct Fp8PairParams {
  int m, n, num_kb;
  int tiles_m, tiles_n, total_tiles, group_m;
  const float* a_scale;
  int64_t a_scale_row, a_scale_blk;
  const float* b_scale;
  int64_t b_scale_row, b_scale_blk;
  void* d;
  int64_t ldd;
  int d_type;
  bool tma_d;
  const void* bias;
  uint32_t idesc;
  int* error_word;
};

namespace fp8_pair {

using fp8::kBlockK;
constexpr int kHalf = 128;    // rows of A and of B per CTA
constexpr int kBlock = 256;   // tile edge
constexpr int kThreads = 384;
constexpr int kAuxThreads = 128;
constexpr int kAccWarps = 8;
constexpr int kBufs = 2;
constexpr uint32_t kTmemCols = 512;

template <bool kRows>
struct Smem {
  static constexpr int kStages = kRows ? 4 : 5;
  static constexpr int kOperand = kHalf * kBlockK;  // 16 KiB
  static constexpr int kStageBytes = 2 * kOperand;
  static constexpr int kOutOff = kStages * kStageBytes;
  static constexpr int kOutWarp = 8192;  // per accumulation warp: four chunks of 32 rows x 64 bytes
  static constexpr int kSlotFloats = kHalf + (kRows ? kBlock : 8);  // row scales, column (block) scales
  static constexpr int kScaleOff = kOutOff + kAccWarps * kOutWarp;
  static constexpr int kBarOff = kScaleOff + kBufs * kSlotFloats * 4;  // the scales of each TMEM buffer's block
  static constexpr int kNumBars = 2 * kStages + 3 * kBufs + 1;
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;
  static constexpr int kDynamicBytes = kMiscOff + 8;
  static_assert(kDynamicBytes <= 232448, "shared memory budget exceeded");
};

enum : int {
  kErrProducerEmpty = (34 << 4) | 1,
  kErrMmaFull = (34 << 4) | 2,
  kErrMmaTmemEmpty = (34 << 4) | 3,
  kErrAccTmemFull = (34 << 4) | 4,
  kErrScaleRead = (34 << 4) | 5,
  kErrAlignment = (34 << 4) | 6,
};

// Tiles in groups of group_m tile rows, column by column, so that concurrent tiles share operands in L2.
__device__ __forceinline__ void raster(int tile, const Fp8PairParams& p, int& tm, int& tn) {
  const int per_group = p.group_m * p.tiles_n;
  const int g = tile / per_group;
  const int first = g * p.group_m;
  const int rows = p.tiles_m - first < p.group_m ? p.tiles_m - first : p.group_m;
  const int in = tile - g * per_group;
  tm = first + in % rows;
  tn = in / rows;
}

// Four chunks of 32 rows x 64 bytes, in the 64-byte swizzle that the stores to D expect, from a warp's
// accumulators (all 128 columns of a 16-bit type, 64 of a 32-bit one).
template <bool kRows, int kType>
__device__ __forceinline__ void fill(uint8_t* out, const float* acc, int lane) {
  constexpr bool kWide = kType == fp8::kF32;
  if constexpr (!kRows) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint4* row = reinterpret_cast<uint4*>(out + c * 2048 + lane * 64);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint4 word;
        if constexpr (kWide) {
          const float* f = acc + 16 * c + 4 * q;
          word = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        } else {
          const float* f = acc + 32 * c + 8 * q;
          word = make_uint4(fp8::pack_out(f[0], f[1], kType), fp8::pack_out(f[2], f[3], kType), fp8::pack_out(f[4], f[5], kType),
                            fp8::pack_out(f[6], f[7], kType));
        }
        row[q ^ ((lane >> 1) & 3)] = word;
      }
    }
  } else {
    // Value j of 32: rows 16 (j / 16) + 8 (j % 4 / 2) + lane / 4, columns 8 (j / 4 % 4) + 2 (lane % 4) and the next.
#pragma unroll
    for (int j = 0; j < (kWide ? 64 : 128); j += 2) {
      const int row = 16 * ((j >> 4) & 1) + 8 * ((j >> 1) & 1) + (lane >> 2);
      const int g = (j >> 2) & 3;
      if constexpr (kWide) {
        const int c = 2 * (j >> 5) + (g >> 1), unit = 2 * (g & 1) + ((lane & 3) >> 1);
        *reinterpret_cast<float2*>(out + c * 2048 + row * 64 + ((unit ^ ((row >> 1) & 3)) << 4) + (lane & 1) * 8) =
            make_float2(acc[j], acc[j + 1]);
      } else {
        *reinterpret_cast<uint32_t*>(out + (j >> 5) * 2048 + row * 64 + ((g ^ ((row >> 1) & 3)) << 4) + (lane & 3) * 4) =
            fp8::pack_out(acc[j], acc[j + 1], kType);
      }
    }
  }
}

// Stores the four chunks (kCols columns each) at column n of rows m..m + 31.
template <int kCols>
__device__ __forceinline__ void flush(const uint8_t* out, const CUtensorMap* map, int n, int m, int lane) {
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
#pragma unroll
    for (int c = 0; c < 4; ++c) tma_store_2d(map, out + c * 2048, n + c * kCols, m);
    bulk_commit_group();
  }
}

template <bool kRows>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                const __grid_constant__ CUtensorMap tmap_d, const Fp8PairParams p) {
  using L = Smem<kRows>;
  constexpr int kStages = L::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);  // used in the leader
  uint64_t* empty = full + kStages;
  uint64_t* tmem_full = empty + kStages;
  uint64_t* tmem_empty = tmem_full + kBufs;  // used in the leader
  uint64_t* read = tmem_empty + kBufs;  // this CTA's warps have read the buffer and its scales
  uint64_t* drain = read + kBufs;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);
  float* const slots = reinterpret_cast<float*>(smem + L::kScaleOff);

  if ((smem_addr(smem) & 1023u) != 0) {  // the swizzled tiles need it; every CTA has the same base
    if (threadIdx.x == 0 && p.error_word != nullptr) atomicCAS(p.error_word, 0, kErrAlignment);
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kBufs; ++b) {
      mbar_init(&tmem_full[b], 2);  // the commit and the scales
      mbar_init(&tmem_empty[b], 2 * kAccWarps);
      mbar_init(&read[b], kAccWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
    if (p.tma_d) tma_prefetch_desc(&tmap_d);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();
  const WaitCtx ctx{abort_flag, p.error_word};
  const int pair = blockIdx.x >> 1;
  const int npairs = gridDim.x >> 1;

  // Every warp of a warpgroup executes its reallocation; the sum is what the block was launched with.
  if (warp < kAuxThreads / 32) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      // ------------------------------------------------------------ producer (both CTAs)
      const bool one = fp8::elect_one();
      uint32_t s = 0, phase = 1, it = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < p.total_tiles; tile += npairs) {
        int tm, tn;
        raster(tile, p, tm, tn);
        const int m0 = tm * kBlock + static_cast<int>(rank) * kHalf;
        const int n0 = tn * kBlock + static_cast<int>(rank) * kHalf;
        for (int kb = 0; kb < p.num_kb; ++kb, ++it) {
          ok = __all_sync(0xffffffffu, fp8::wait(&empty[s], phase, ctx, kErrProducerEmpty));
          if (!ok) break;
          if (one) {
            const uint32_t full_leader = map_shared_rank(smem_addr(&full[s]), 0);
            if (leader) mbar_arrive_expect_tx(&full[s], 2 * L::kStageBytes);
            uint8_t* at = smem + s * L::kStageBytes;
            tma_load_2d_pair(at, &tmap_a, full_leader, kb * kBlockK, m0);
            tma_load_2d_pair(at + L::kOperand, &tmap_b, full_leader, kb * kBlockK, n0);
          }
          __syncwarp();
          if (++s == kStages) s = 0, phase ^= 1u;
        }
      }
      if (!ok && one) {  // unwind: loads already issued must land before the CTAs can exit
        if (leader) {
          const uint32_t first = it > static_cast<uint32_t>(kStages) ? it - kStages : 0u;
          for (uint32_t j = first; j < it; ++j) mbar_wait_quiet(&full[j % kStages], (j / kStages) & 1u, 200000000ull);
        } else {
          for (int i = 0; i < 1000; ++i) sleep_ns(1000);  // the follower cannot poll the leader's barrier
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer (leader only)
      if (leader) {
        const bool one = fp8::elect_one();
        uint32_t s = 0, phase = 0, buf = 0, buf_phase = 1;
        bool ok = true, issued = false;
        const uint64_t desc0 = smem_desc_sw128(smem_addr(smem), 16, 1024);
        for (int tile = pair; ok && tile < p.total_tiles; tile += npairs) {
          for (int kb = 0; kb < p.num_kb; ++kb) {
            ok = fp8::wait(&full[s], phase, ctx, kErrMmaFull);
            ok = ok && fp8::wait_read(&tmem_empty[buf], buf_phase, ctx, kErrMmaTmemEmpty);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after_sync();
            if (one) {
              const uint64_t a = desc0 + (s * L::kStageBytes >> 4);
#pragma unroll
              for (int kk = 0; kk < kBlockK / fp8::kMmaK; ++kk)
                fp8::mma_pair(tmem_base + buf * kBlock, a + (kk * fp8::kMmaK >> 4),
                              a + ((L::kOperand + kk * fp8::kMmaK) >> 4), p.idesc, kk != 0 ? 1u : 0u);
              umma_commit_pair_multicast(&tmem_full[buf], 0x3);
              umma_commit_pair_multicast(&empty[s], 0x3);
            }
            __syncwarp();
            issued = true;
            buf ^= 1u;
            buf_phase ^= buf == 0 ? 1u : 0u;
            if (++s == kStages) s = 0, phase ^= 1u;
          }
        }
        if (!ok && issued && one) {
          umma_commit_pair_multicast(drain, 0x1);
          mbar_wait_quiet(drain, 0, 200000000ull);
        }
      }
      __syncwarp();
    } else {
      // ------------------------------------------------------------ scales (both CTAs)
      // Warp 2 + b serves the blocks of TMEM buffer b: block i's scales go where block i - 2's were once every
      // warp of this CTA has read those. So the buffer's `tmem_full` phase of block i - 2 is complete, too.
      const uint32_t buf = static_cast<uint32_t>(warp - 2);
      uint32_t i = 0;  // blocks so far, both buffers'
      bool ok = true;
      for (int tile = pair; ok && tile < p.total_tiles; tile += npairs) {
        int tm, tn;
        raster(tile, p, tm, tn);
        const int64_t m0 = static_cast<int64_t>(tm) * kBlock + rank * kHalf;
        const int64_t n0 = static_cast<int64_t>(tn) * kBlock;
        for (int kb = 0; ok && kb < p.num_kb; ++kb, ++i) {
          if ((i & 1u) != buf) continue;
          const float* sa = p.a_scale + kb * p.a_scale_blk;
          const float* sb = p.b_scale + kb * p.b_scale_blk;
          float a[kHalf / 32], b[kRows ? kBlock / 32 : 1];
#pragma unroll
          for (int j = 0; j < kHalf / 32; ++j) {
            const int64_t row = m0 + j * 32 + lane;
            a[j] = row < p.m ? ld_written(sa + row * p.a_scale_row) : 0.0f;
          }
          if constexpr (kRows) {
#pragma unroll
            for (int j = 0; j < kBlock / 32; ++j) {
              const int64_t col = n0 + j * 32 + lane;
              b[j] = col < p.n ? ld_written(sb + col * p.b_scale_row) : 0.0f;
            }
          } else {
            b[0] = lane < 2 && n0 + lane * kHalf < p.n ? ld_written(sb + (n0 / kHalf + lane) * p.b_scale_row) : 0.0f;
          }
          if (i >= kBufs) ok = fp8::wait(&read[buf], ((i / kBufs) & 1u) ^ 1u, ctx, kErrScaleRead);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          float* slot = slots + buf * L::kSlotFloats;
#pragma unroll
          for (int j = 0; j < kHalf / 32; ++j) slot[j * 32 + lane] = a[j];
          if constexpr (kRows) {
#pragma unroll
            for (int j = 0; j < kBlock / 32; ++j) slot[kHalf + j * 32 + lane] = b[j];
          } else {
            if (lane < 2) slot[kHalf + lane] = b[0];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&tmem_full[buf]);
        }
      }
    }
  } else {
    // ------------------------------------------------------------ accumulation and output (both CTAs)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int quarter = warp & 3;
    const int w = warp - kAuxThreads / 32;
    const int half = w >> 2;  // columns half * 128 ..
    uint8_t* out = smem + L::kOutOff + w * L::kOutWarp;
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + half * kHalf;
    uint32_t i = 0;
    bool ok = true;
    for (int tile = pair; ok && tile < p.total_tiles; tile += npairs) {
      int tm, tn;
      raster(tile, p, tm, tn);
      const int m0 = tm * kBlock + static_cast<int>(rank) * kHalf + quarter * 32;  // the warp's first row
      const int n0 = tn * kBlock + half * kHalf;
      // One row per thread: values 0..127 are its columns. kRows: values 32 c + 16 h + 4 g + e are fragment
      // element e of column group 4 c + g of the 16 rows h.
      float acc[kHalf];
#pragma unroll
      for (int j = 0; j < kHalf; ++j) acc[j] = 0.0f;
#pragma unroll 1
      for (int kb = 0; kb < p.num_kb; ++kb, ++i) {
        const uint32_t buf = i % kBufs;
        const float* slot = slots + buf * L::kSlotFloats;
        ok = fp8::wait(&tmem_full[buf], (i / kBufs) & 1u, ctx, kErrAccTmemFull);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t t0 = taddr + buf * kBlock;
        const auto read_done = [&] {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) {
            fp8::arrive_read(map_shared_rank(smem_addr(&tmem_empty[buf]), 0));
            mbar_arrive(&read[buf]);
          }
        };
        if constexpr (!kRows) {
          fp8::add_columns(acc, t0, [&] { return slot[quarter * 32 + lane] * slot[kHalf + half]; }, read_done);
        } else {
          // 32 columns of 16 rows per load: v[0], v[1] the two halves of the rows in one column group, v[2], v[3]
          // in the next. Four loads are in flight at a time (one ahead: 1 % slower).
          uint32_t v[4][16];
          const auto load = [&](int g) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              fp8::tmem_ld_16x256b_x4(t0 + (static_cast<uint32_t>(h * 16) << 16) + g * 32, v[2 * (g & 1) + h]);
          };
          const auto landed = [&] {
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 4; ++j) fp8::after_wait(v[j]);
          };
          load(0);
          load(1);
          float sa[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) sa[j] = slot[quarter * 32 + j * 8 + (lane >> 2)];
          const float2* sb = reinterpret_cast<const float2*>(slot + kHalf + half * kHalf) + (lane & 3);
          float2 cs[2][4];  // column scales of two groups
          const auto add = [&](int g) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              fp8::add_fragments(acc + g * 32 + h * 16, v[2 * (g & 1) + h], cs[g & 1], sa[2 * h], sa[2 * h + 1]);
          };
          fp8::load_column_scales(cs[0], sb);
          fp8::load_column_scales(cs[1], sb + 16);
          landed();
          add(0);
          load(2);
          fp8::load_column_scales(cs[0], sb + 32);
          add(1);
          load(3);
          fp8::load_column_scales(cs[1], sb + 48);
          landed();
          read_done();
          add(2);
          add(3);
        }
      }
      if (!ok) break;
      if (n0 >= p.n || m0 >= p.m) continue;
      if (p.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < kHalf; ++j) {
          const int col = kRows ? 32 * (j >> 5) + 8 * ((j >> 2) & 3) + 2 * (lane & 3) + (j & 1) : j;
          if (n0 + col < p.n) acc[j] += fp8::load_out(p.bias, n0 + col, p.d_type);
        }
      }
      if (p.tma_d && n0 + kHalf <= p.n) {
        // Chunks of 32 rows x 64 bytes (32 values of 16 bits, 16 of 32), four at a time: one fence and one group
        // of stores for all (a fence per chunk made the output 3000 cycles per tile, as long as four k blocks).
        if (p.d_type == fp8::kF32) {
#pragma unroll
          for (int round = 0; round < 2; ++round) {
            if (lane == 0) bulk_wait_group_read<0>();
            __syncwarp();
            fill<kRows, fp8::kF32>(out, acc + round * 64, lane);
            flush<16>(out, &tmap_d, n0 + round * 64, m0, lane);
          }
        } else {
          if (lane == 0) bulk_wait_group_read<0>();
          __syncwarp();
          if (p.d_type == fp8::kBf16) fill<kRows, fp8::kBf16>(out, acc, lane);
          else fill<kRows, fp8::kF16>(out, acc, lane);
          flush<32>(out, &tmap_d, n0, m0, lane);
        }
      } else {
        // Ragged or unaligned: through shared memory as 32-bit values, then whole rows of 32 columns.
        if (lane == 0) bulk_wait_group_read<0>();
        float* stage = reinterpret_cast<float*>(out);
        const int rows = p.m - m0 < 32 ? p.m - m0 : 32;
#pragma unroll
        for (int c = 0; c < kHalf / 32; ++c) {
          const int nc = n0 + c * 32;
          if (nc >= p.n) break;
          __syncwarp();
          const float* v = acc + c * 32;
          if constexpr (!kRows) {
#pragma unroll
            for (int q = 0; q < 8; ++q)
              *reinterpret_cast<float4*>(stage + lane * 32 + 4 * (q ^ (lane & 7))) =
                  make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const int row = 16 * (j >> 4) + 8 * ((j >> 1) & 1) + (lane >> 2);
              const int unit = 2 * ((j >> 2) & 3) + ((lane & 3) >> 1);
              *reinterpret_cast<float2*>(stage + row * 32 + 4 * (unit ^ (row & 7)) + 2 * (lane & 1)) = make_float2(v[j], v[j + 1]);
            }
          }
          __syncwarp();
          if (nc + lane < p.n) {
            for (int r = 0; r < rows; ++r)
              fp8::store_out(p.d, static_cast<int64_t>(m0 + r) * p.ldd + nc + lane, p.d_type,
                             stage[r * 32 + 4 * ((lane >> 2) ^ (r & 7)) + (lane & 3)]);
          }
        }
        __syncwarp();
      }
    }
    if (lane == 0) bulk_wait_group<0>();
    __syncwarp();
  }

  tc_fence_before_sync();
  __syncwarp();
  cluster_sync_all();  // no CTA leaves while its peer may still touch its memory
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

}  // namespace fp8_pair
}  // namespace zcb
