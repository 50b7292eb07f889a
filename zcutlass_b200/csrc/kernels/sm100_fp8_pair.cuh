// 8-bit block-scaled product on CTA pairs (cta_group::2), 256 x 256 output
// tiles, persistent: the large products (prefill, training).
//
//   D[m, n] = sum_b sa(m, b) * sb(n, b) * (A_b B_b^T)[m, n]  (+ bias[n])
//
// Per block of 128 k the pair's leader issues 4 MMAs of 256 x 256 x 32 into one
// of two 256-column TMEM buffers; each CTA holds its 128 rows x 256 columns.
// Eight accumulation warps per CTA (two per TMEM quarter, 128 columns each)
// read the buffer and add it, scaled, into 128 32-bit accumulators per thread,
// while the MMAs of the next block fill the other buffer. At full rate a block
// takes the tensor pipe 512 cycles per SM, and the accumulation warps 128
// columns x 8 warps: 256 cycles of TMEM reads and 128 of packed fma issue.
// 128 accumulators, one TMEM chunk in use and one in flight need more than the
// 168 registers three warps per SM sub-partition get: the first warpgroup hands
// registers over (128 x 72 + 256 x 216 = 384 x 168).
//
// With 128 x 128 weight scales the factor is one product per thread and block;
// with a scale per row of B (kRows) the 128 column scales of a warpgroup go
// through shared memory, two slots in turn.
//
// Roles per CTA: warp 0 TMA producer (stages of two k blocks: 2 x 32 KiB), warp
// 1 TMEM allocation and, in the leader, MMA issue; warps 4-11 accumulate, then
// write the tile (registers -> swizzled shared memory -> TMA, or row by row
// where D is ragged or unaligned) while the next tile's first blocks run.
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
constexpr int kStages = 3;
constexpr int kSub = 2;       // k blocks per stage
constexpr int kBufs = 2;
constexpr int kAhead = 4;
constexpr uint32_t kTmemCols = 512;

struct Smem {
  static constexpr int kOperand = kHalf * kBlockK;  // 16 KiB
  static constexpr int kSubBytes = 2 * kOperand;
  static constexpr int kStageBytes = kSub * kSubBytes;
  static constexpr int kOutOff = kStages * kStageBytes;
  static constexpr int kOutWarp = 4096;  // per accumulation warp
  static constexpr int kScaleOff = kOutOff + kAccWarps * kOutWarp;  // [2 column halves][2 slots][128] floats
  static constexpr int kBarOff = kScaleOff + 2 * 2 * kHalf * 4;
  static constexpr int kNumBars = 2 * kStages + 2 * kBufs + 1;
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;
  static constexpr int kDynamicBytes = kMiscOff + 16 + 1024 - 128;  // room to align a 128-byte aligned base to 1024
  static_assert(kDynamicBytes <= 232448, "shared memory budget exceeded");
};

enum : int {
  kErrProducerEmpty = (34 << 4) | 1,
  kErrMmaFull = (34 << 4) | 2,
  kErrMmaTmemEmpty = (34 << 4) | 3,
  kErrAccTmemFull = (34 << 4) | 4,
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

template <bool kRows>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                const __grid_constant__ CUtensorMap tmap_d, const Fp8PairParams p) {
  using L = Smem;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);  // used in the leader
  uint64_t* empty = full + kStages;
  uint64_t* tmem_full = empty + kStages;
  uint64_t* tmem_empty = tmem_full + kBufs;  // used in the leader
  uint64_t* drain = tmem_empty + kBufs;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kBufs; ++b) {
      mbar_init(&tmem_full[b], 1);
      mbar_init(&tmem_empty[b], 2 * kAccWarps);
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
      if (lane == 0) {
        uint32_t it = 0;
        bool ok = true;
        for (int tile = pair; ok && tile < p.total_tiles; tile += npairs) {
          int tm, tn;
          raster(tile, p, tm, tn);
          const int m0 = tm * kBlock + static_cast<int>(rank) * kHalf;
          const int n0 = tn * kBlock + static_cast<int>(rank) * kHalf;
          for (int kb = 0; kb < p.num_kb; kb += kSub, ++it) {
            const uint32_t s = it % kStages;
            if (!mbar_wait(&empty[s], ((it / kStages) & 1u) ^ 1u, ctx, kErrProducerEmpty)) {
              ok = false;
              break;
            }
            const int subs = p.num_kb - kb < kSub ? p.num_kb - kb : kSub;
            const uint32_t full_leader = map_shared_rank(smem_addr(&full[s]), 0);
            if (leader) mbar_arrive_expect_tx(&full[s], 2 * subs * L::kSubBytes);
  #pragma unroll
            for (int sub = 0; sub < kSub; ++sub) {
              if (sub >= subs) break;
              uint8_t* at = smem + s * L::kStageBytes + sub * L::kSubBytes;
              tma_load_2d_pair(at, &tmap_a, full_leader, (kb + sub) * kBlockK, m0);
              tma_load_2d_pair(at + L::kOperand, &tmap_b, full_leader, (kb + sub) * kBlockK, n0);
            }
          }
        }
        if (!ok) {  // unwind: loads already issued must land before the CTAs can exit
          if (leader) {
            const uint32_t first = it > static_cast<uint32_t>(kStages) ? it - kStages : 0u;
            for (uint32_t j = first; j < it; ++j) mbar_wait_quiet(&full[j % kStages], (j / kStages) & 1u, 200000000ull);
          } else {
            for (int i = 0; i < 1000; ++i) sleep_ns(1000);  // the follower cannot poll the leader's barrier
          }
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer (leader only)
      if (leader && lane == 0) {
        uint32_t it = 0, i = 0;  // stages and k blocks so far
        bool ok = true, issued = false;
        for (int tile = pair; ok && tile < p.total_tiles; tile += npairs) {
          for (int kb = 0; ok && kb < p.num_kb; kb += kSub, ++it) {
            const uint32_t s = it % kStages;
            if (!mbar_wait(&full[s], (it / kStages) & 1u, ctx, kErrMmaFull)) {
              ok = false;
              break;
            }
            const int subs = p.num_kb - kb < kSub ? p.num_kb - kb : kSub;
            for (int sub = 0; sub < subs; ++sub, ++i) {
              const uint32_t buf = i % kBufs;
              if (!mbar_wait(&tmem_empty[buf], ((i / kBufs) & 1u) ^ 1u, ctx, kErrMmaTmemEmpty)) {
                ok = false;
                break;
              }
              tc_fence_after_sync();
              const uint32_t a = smem_addr(smem + s * L::kStageBytes + sub * L::kSubBytes);
  #pragma unroll
              for (int kk = 0; kk < kBlockK / fp8::kMmaK; ++kk)
                fp8::mma_pair(tmem_base + buf * kBlock, smem_desc_sw128(a + kk * fp8::kMmaK, 16, 1024),
                              smem_desc_sw128(a + L::kOperand + kk * fp8::kMmaK, 16, 1024), p.idesc, kk != 0 ? 1u : 0u);
              issued = true;
              umma_commit_pair_multicast(&tmem_full[buf], 0x3);
            }
            if (ok) umma_commit_pair_multicast(&empty[s], 0x3);
          }
        }
        if (!ok && issued) {
          umma_commit_pair_multicast(drain, 0x1);
          mbar_wait_quiet(drain, 0, 200000000ull);
        }
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ accumulation and output (both CTAs)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int quarter = warp & 3;
    const int w = warp - kAuxThreads / 32;
    const int half = w >> 2;                              // columns half * 128 ..
    const int t = threadIdx.x & (kHalf - 1);              // thread of the half's warpgroup
    float* scales = reinterpret_cast<float*>(smem + L::kScaleOff) + half * 2 * kHalf;
    uint8_t* out = smem + L::kOutOff + w * L::kOutWarp;
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + half * kHalf;
    uint32_t i = 0;
    uint32_t chunk = 0;
    bool ok = true;
    const float* sa = nullptr;
    const float* sb = nullptr;
    bool row_ok = false, col_ok = false;
    float a_next[kAhead], b_next[kAhead];
    auto fetch = [&](int kb, float& a, float& b) {
      const bool in = kb < p.num_kb;
      a = in && row_ok ? __ldg(sa + kb * p.a_scale_blk) : 0.0f;
      b = in && col_ok ? __ldg(sb + kb * p.b_scale_blk) : 0.0f;
    };
    auto start = [&](int tile) {  // the first scales of a tile
      if (tile >= p.total_tiles) return;
      int tm, tn;
      raster(tile, p, tm, tn);
      const int64_t row = static_cast<int64_t>(tm) * kBlock + rank * kHalf + quarter * 32 + lane;
      const int64_t n0 = static_cast<int64_t>(tn) * kBlock + half * kHalf;
      const int64_t b = kRows ? n0 + t : n0 / kHalf;
      row_ok = row < p.m;
      col_ok = kRows ? n0 + t < p.n : n0 < p.n;
      sa = p.a_scale + row * p.a_scale_row;
      sb = p.b_scale + b * p.b_scale_row;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) fetch(u, a_next[u], b_next[u]);
    };
    start(pair);
    for (int tile = pair; ok && tile < p.total_tiles; tile += npairs) {
      int tm, tn;
      raster(tile, p, tm, tn);
      const int m0 = tm * kBlock + static_cast<int>(rank) * kHalf + quarter * 32;  // the warp's first row
      const int n0 = tn * kBlock + half * kHalf;
      uint64_t acc[kHalf / 2];
#pragma unroll
      for (int j = 0; j < kHalf / 2; ++j) acc[j] = 0;
#pragma unroll 1
      for (int kb = 0; kb < p.num_kb; ++kb) {
        const uint32_t buf = i % kBufs;
        float* slot = scales + (i & 1u) * kHalf;  // blocks of successive tiles keep alternating
        const uint64_t mine = fp8::both(kRows ? a_next[0] : a_next[0] * b_next[0]);
        if constexpr (kRows) slot[t] = b_next[0];
#pragma unroll
        for (int u = 0; u + 1 < kAhead; ++u) a_next[u] = a_next[u + 1], b_next[u] = b_next[u + 1];
        fetch(kb + kAhead, a_next[kAhead - 1], b_next[kAhead - 1]);
        ok = mbar_wait(&tmem_full[buf], (i / kBufs) & 1u, ctx, kErrAccTmemFull);
        if constexpr (kRows) ok = half == 0 ? fp8::barrier_and<1, kHalf>(ok) : fp8::barrier_and<2, kHalf>(ok);
        else ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ++i;
        tc_fence_after_sync();
        uint32_t v[2][16];
        fp8::tmem_ld_x16(taddr + buf * kBlock, v[0]);
#pragma unroll
        for (int c = 0; c < kHalf / 16; ++c) {
          uint32_t(&r)[16] = v[c & 1];
          fp8::tmem_ld_wait_x16(r);
          if (c + 1 < kHalf / 16) {
            fp8::tmem_ld_x16(taddr + buf * kBlock + (c + 1) * 16, v[(c + 1) & 1]);
          } else {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_shared_rank(smem_addr(&tmem_empty[buf]), 0));
          }
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            uint64_t s0 = mine, s1 = mine;
            if constexpr (kRows) {
              const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(slot + c * 16 + j);
              s0 = fp8::mul2(s.x, mine);
              s1 = fp8::mul2(s.y, mine);
            }
            fp8::fma2(acc[c * 8 + j / 2], s0, fp8::pack2(r[j], r[j + 1]));
            fp8::fma2(acc[c * 8 + j / 2 + 1], s1, fp8::pack2(r[j + 2], r[j + 3]));
          }
        }
      }
      if (!ok) break;
      start(tile + npairs);  // on their way while this tile is written
      const bool wide = p.d_type == fp8::kF32;
      // Chunks of 64 bytes per row (32 values of 16 bits, 16 of 32) go out by TMA, double-buffered.
#pragma unroll
      for (int c = 0; c < kHalf / 32; ++c) {
        const int nc = n0 + c * 32;
        if (nc >= p.n || m0 >= p.m) break;
        float v[32];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float2 f = fp8::unpack2(acc[c * 16 + j]);
          v[2 * j] = f.x;
          v[2 * j + 1] = f.y;
        }
        if (p.bias != nullptr) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (nc + j < p.n) v[j] += fp8::load_out(p.bias, nc + j, p.d_type);
        }
        if (p.tma_d && nc + 32 <= p.n) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h == 1 && !wide) break;
            uint8_t* buf = out + (chunk & 1u) * 2048;
            if (lane == 0) bulk_wait_group_read<1>();
            __syncwarp();
            uint4* row = reinterpret_cast<uint4*>(buf + lane * 64);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint4 word;
              if (wide) {
                const float* f = v + h * 16 + 4 * q;
                word = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
              } else {
                const float* f = v + 8 * q;
                word = make_uint4(fp8::pack_out(f[0], f[1], p.d_type), fp8::pack_out(f[2], f[3], p.d_type),
                                  fp8::pack_out(f[4], f[5], p.d_type), fp8::pack_out(f[6], f[7], p.d_type));
              }
              row[q ^ ((lane >> 1) & 3)] = word;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmap_d, buf, nc + h * 16, m0);
              bulk_commit_group();
            }
            ++chunk;
          }
        } else {
          // Ragged or unaligned: through shared memory as 32-bit values, then whole rows of 32 columns.
          if (lane == 0) bulk_wait_group_read<0>();
          __syncwarp();
          float* stage = reinterpret_cast<float*>(out);
#pragma unroll
          for (int q = 0; q < 8; ++q)
            *reinterpret_cast<float4*>(stage + lane * 32 + 4 * (q ^ (lane & 7))) =
                make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
          __syncwarp();
          const int rows = p.m - m0 < 32 ? p.m - m0 : 32;
          if (nc + lane < p.n) {
            for (int r = 0; r < rows; ++r)
              fp8::store_out(p.d, static_cast<int64_t>(m0 + r) * p.ldd + nc + lane, p.d_type,
                             stage[r * 32 + 4 * ((lane >> 2) ^ (r & 7)) + (lane & 3)]);
          }
          __syncwarp();
        }
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
