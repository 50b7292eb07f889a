// 8-bit block-scaled product with one output tile per cluster of CTAs along K:
// few rows of A (decode) and products too small for the pair kernel's tiles.
//
//   D[m, n] = sum_b sa(m, b) * sb(n, b) * (A_b B_b^T)[m, n]  (+ bias[n])
//
// kSwap (M <= 64): B's rows (weights) fill the 128-row MMA dimension and TM =
// 16, 32 or 64 rows of A sit on MMA-N, so the tensor core reads no padding of
// 128 rows and the weights, which are the bytes, are streamed once. Else A's
// rows are on MMA-M and the tile is 128 x 128.
//
// Per block of 128 k, 4 MMAs fill one of four TMEM buffers; the four
// accumulation warps (a TMEM lane per thread) add it, scaled, to 32-bit
// accumulators in registers. As in the pair kernel, the MMA warp keeps its state
// in uniform registers, and two warps stage each block's scales in shared
// memory and complete the buffer's barrier together with the commit. With one
// weight scale per 128 rows of B the staged value is the whole factor.
// With a scale per row of B (kRows) it is a factor per thread (kSwap), or TMEM is
// read as 16 x 8 fragments, in which a thread meets 32 of 128 columns.
//
// Bound by bytes: a stage of the TMA ring holds KSUB = 2 blocks. The same bytes
// in stages of one block: 512 x 4096 x 4096 20.2 us against 16.9, 1 x 6144 x 4096
// 8.2 against 8.4 (3 splits); half the ring: 48 x 4096 x 14336 17.1-17.3 against
// 15.6 with either. The splits' 32-bit
// partial tiles are added in split order through distributed shared memory, so
// the result does not depend on timing.
#pragma once

#include "sm100_fp8_common.cuh"

namespace zcb {

struct Fp8TileParams {
  int m, n, num_kb, splits, tiles_m;
  const float* a_scale;
  int64_t a_scale_row, a_scale_blk;
  const float* b_scale;
  int64_t b_scale_row, b_scale_blk;
  void* d;
  int64_t ldd;
  int d_type;
  bool vec_d;  // four consecutive n of D may be stored at once
  const void* bias;
  uint32_t idesc;
  int* error_word;
};

namespace fp8_tile {

using fp8::kBlockK;
constexpr int kBlockN = 128;
constexpr int kThreads = 256;
constexpr int kAccThreads = 128;
constexpr int kMaxSplits = 8;
constexpr int kBufs = 4;   // TMEM buffers

template <bool kSwap, int TM, bool kRows, int STAGES, int KSUB>
struct Smem {
  static_assert(kSwap ? (TM == 16 || TM == 32 || TM == 64) : TM == 128, "");
  static constexpr int kMmaN = kSwap ? TM : kBlockN;
  static constexpr int kABytes = TM * kBlockK;
  static constexpr int kBBytes = kBlockN * kBlockK;
  static constexpr int kSub = kABytes + kBBytes;  // B first: both start on 1024 bytes
  static constexpr int kStageBytes = KSUB * kSub;
  static constexpr int kRedBytes = TM * kBlockN * 4;  // the partial tile [m][n], over the drained ring
  static constexpr int kRing = STAGES * kStageBytes > kRedBytes ? STAGES * kStageBytes : kRedBytes;
  static constexpr int kSlotFloats = TM + (kRows ? kBlockN : 0);
  static constexpr int kScaleOff = kRing;
  static constexpr int kBarOff = kScaleOff + kBufs * kSlotFloats * 4;  // the scales of each TMEM buffer's block
  static constexpr int kNumBars = 2 * STAGES + 2 * kBufs + 1;
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;
  static constexpr int kDynamicBytes = kMiscOff + 16 + 1024;
  static constexpr uint32_t kTmemCols = kBufs * kMmaN;
  static_assert(kSub % 1024 == 0 && kABytes % 1024 == 0 && kDynamicBytes <= 232448, "");
};

enum : int {
  kErrProducerEmpty = (33 << 4) | 1,
  kErrMmaFull = (33 << 4) | 2,
  kErrMmaTmemEmpty = (33 << 4) | 3,
  kErrAccTmemFull = (33 << 4) | 4,
  kErrScaleRead = (33 << 4) | 5,
};

// Partial tile element (m, 4 g): rows rotate their 16-byte units where a thread writes a whole row.
template <bool kSwap>
__device__ __forceinline__ int red_at(int m, int g) {
  return m * kBlockN + 4 * (kSwap ? g : g ^ (m & 7));
}

template <bool kSwap, int TM, bool kRows, int STAGES, int KSUB>
__global__ void __launch_bounds__(kThreads, kSwap ? 2 : 1)
    gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                const Fp8TileParams p) {
  using L = Smem<kSwap, TM, kRows, STAGES, KSUB>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* empty = full + STAGES;
  uint64_t* tmem_full = empty + STAGES;
  uint64_t* tmem_empty = tmem_full + kBufs;
  uint64_t* drain = tmem_empty + kBufs;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);
  float* const slots = reinterpret_cast<float*>(smem + L::kScaleOff);
  float* const red = reinterpret_cast<float*>(smem);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int split = static_cast<int>(blockIdx.x % p.splits);  // the cluster rank: clusters are `splits` wide
  const int tile = static_cast<int>(blockIdx.x / p.splits);
  const int m0 = (tile % p.tiles_m) * TM, n0 = (tile / p.tiles_m) * kBlockN;
  const int kb0 = static_cast<int>(static_cast<int64_t>(split) * p.num_kb / p.splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(split + 1) * p.num_kb / p.splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kBufs; ++b) {
      mbar_init(&tmem_full[b], 2);  // the commit and the scales
      mbar_init(&tmem_empty[b], kAccThreads / 32);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  // Weights of the first stages on their way to L2 while the kernel before (often the quantisation of A) is
  // still running. A hint: if that kernel writes them, the copies in L2 are what it writes.
  if (warp == 0 && lane == 0) {
    for (int kb = kb0; kb < kb1 && kb < kb0 + STAGES * KSUB; ++kb) fp8::tma_prefetch_2d(&tmap_b, kb * kBlockK, n0);
  }
  griddep_wait();
  griddep_launch_dependents();
  const WaitCtx ctx{abort_flag, p.error_word};

  if (warp == 0) {
    // The whole warp walks the loop (uniform registers), one lane issues. B is read once when one tile of
    // rows covers M; A by every CTA.
    const bool one = fp8::elect_one();
    const uint64_t b_policy = p.tiles_m == 1 ? l2_policy_evict_first() : l2_policy_evict_last();
    const uint64_t a_policy = l2_policy_evict_last();
    uint32_t s = 0, phase = 1, it = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; kb += KSUB, ++it) {
      ok = __all_sync(0xffffffffu, fp8::wait(&empty[s], phase, ctx, kErrProducerEmpty));
      if (!ok) break;
      const int subs = kb1 - kb < KSUB ? kb1 - kb : KSUB;
      if (one) {
        mbar_arrive_expect_tx(&full[s], subs * L::kSub);
        uint8_t* at = smem + s * L::kStageBytes;
#pragma unroll
        for (int sub = 0; sub < KSUB; ++sub) {
          if (sub >= subs) break;
          tma_load_2d_hint(at + sub * L::kSub, &tmap_b, &full[s], (kb + sub) * kBlockK, n0, b_policy);
          tma_load_2d_hint(at + sub * L::kSub + L::kBBytes, &tmap_a, &full[s], (kb + sub) * kBlockK, m0, a_policy);
        }
      }
      __syncwarp();
      if (++s == STAGES) s = 0, phase ^= 1u;
    }
    if (!ok && one) {  // loads already issued must land before the CTA can exit
      const uint32_t first = it > static_cast<uint32_t>(STAGES) ? it - STAGES : 0u;
      for (uint32_t j = first; j < it; ++j) mbar_wait_quiet(&full[j % STAGES], (j / STAGES) & 1u, 200000000ull);
    }
    __syncwarp();
  } else if (warp == 1) {
    const bool one = fp8::elect_one();
    uint32_t s = 0, phase = 0, buf = 0, buf_phase = 1;
    bool ok = true, issued = false;
    const uint64_t desc0 = smem_desc_sw128(smem_addr(smem), 16, 1024);
    for (int kb = kb0; ok && kb < kb1; kb += KSUB) {
      ok = __all_sync(0xffffffffu, fp8::wait(&full[s], phase, ctx, kErrMmaFull));
      if (!ok) break;
#pragma unroll
      for (int sub = 0; sub < KSUB; ++sub) {
        if (kb + sub >= kb1) break;
        ok = __all_sync(0xffffffffu, fp8::wait(&tmem_empty[buf], buf_phase, ctx, kErrMmaTmemEmpty));
        if (!ok) break;
        tc_fence_after_sync();
        if (one) {
          const uint64_t b = desc0 + ((s * L::kStageBytes + sub * L::kSub) >> 4);
          const uint64_t a = b + (L::kBBytes >> 4);
#pragma unroll
          for (int kk = 0; kk < kBlockK / fp8::kMmaK; ++kk) {
            const uint64_t step = kk * fp8::kMmaK >> 4;
            fp8::mma(tmem_base + buf * L::kMmaN, (kSwap ? b : a) + step, (kSwap ? a : b) + step, p.idesc, kk != 0 ? 1u : 0u);
          }
          umma_commit(&tmem_full[buf]);
          if (sub == KSUB - 1) umma_commit(&empty[s]);
        }
        __syncwarp();
        issued = true;
        if (++buf == kBufs) buf = 0, buf_phase ^= 1u;
      }
      if (++s == STAGES) s = 0, phase ^= 1u;
    }
    if (!ok && issued && one) {
      umma_commit(drain);
      mbar_wait_quiet(drain, 0, 200000000ull);
    }
    __syncwarp();
  } else if (warp < 4) {
    // Scales: warp 2 + q serves the blocks of parity q. Block i's go where block i - 4's were once every warp has
    // read those and the TMEM buffer, so the buffer's `tmem_full` phase of block i - 4 is complete, too.
    bool ok = true;
    for (int kb = kb0 + warp - 2; ok && kb < kb1; kb += 2) {
      const uint32_t i = static_cast<uint32_t>(kb - kb0), buf = i % kBufs;
      const float* sa = p.a_scale + kb * p.a_scale_blk;
      const float* sb = p.b_scale + kb * p.b_scale_blk;
      constexpr int kA = (TM + 31) / 32;
      float a[kA], b[kRows ? kBlockN / 32 : 1];
#pragma unroll
      for (int j = 0; j < kA; ++j) {
        const int r = j * 32 + lane;
        a[j] = r < TM && m0 + r < p.m ? ld_written(sa + (m0 + r) * p.a_scale_row) : 0.0f;
      }
      if constexpr (kRows) {
#pragma unroll
        for (int j = 0; j < kBlockN / 32; ++j) {
          const int r = n0 + j * 32 + lane;
          b[j] = r < p.n ? ld_written(sb + r * p.b_scale_row) : 0.0f;
        }
      } else {
        b[0] = ld_written(sb + (n0 / kBlockN) * p.b_scale_row);
      }
      if (i >= kBufs) ok = fp8::wait(&tmem_empty[buf], ((i / kBufs) & 1u) ^ 1u, ctx, kErrScaleRead);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      float* slot = slots + buf * L::kSlotFloats;
#pragma unroll
      for (int j = 0; j < kA; ++j)
        if (j * 32 + lane < TM) slot[j * 32 + lane] = kRows ? a[j] : a[j] * b[0];
      if constexpr (kRows) {
#pragma unroll
        for (int j = 0; j < kBlockN / 32; ++j) slot[TM + j * 32 + lane] = b[j];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&tmem_full[buf]);
    }
  } else {
    // ------------------------------------------------------------ accumulation
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;  // TMEM lane
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    constexpr bool kFragments = kRows && !kSwap;
    constexpr int kSteps = L::kMmaN / 16;
    float acc[L::kMmaN];
#pragma unroll
    for (int j = 0; j < L::kMmaN; ++j) acc[j] = 0.0f;
    bool ok = true;
    uint32_t buf = 0, phase = 0;
#pragma unroll 1
    for (int kb = kb0; kb < kb1; ++kb) {
      const float* slot = slots + buf * L::kSlotFloats;
      ok = __all_sync(0xffffffffu, fp8::wait(&tmem_full[buf], phase, ctx, kErrAccTmemFull));
      if (!ok) break;
      tc_fence_after_sync();
      const uint32_t t0 = taddr + buf * L::kMmaN;
      uint32_t v[2][16];
      auto load = [&](int c, uint32_t(&r)[16]) {
        if constexpr (kFragments) fp8::tmem_ld_16x256b_x4(t0 + ((static_cast<uint32_t>(c & 1) * 16) << 16) + (c >> 1) * 32, r);
        else fp8::tmem_ld_x16(t0 + c * 16, r);
      };
      load(0, v[0]);
      const float mine = kSwap ? (kRows ? slot[TM + row] : 1.0f) : (kFragments ? 1.0f : slot[row]);
      float lo_hi[4];
      float2 cs[2][4];  // column scales, loaded two steps ahead
      const float2* sb = reinterpret_cast<const float2*>(slot + TM) + (lane & 3);
      if constexpr (kFragments) {
        fp8::load_column_scales(cs[0], sb);
#pragma unroll
        for (int j = 0; j < 4; ++j) lo_hi[j] = slot[quarter * 32 + j * 8 + (lane >> 2)];
      }
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        uint32_t(&r)[16] = v[c & 1];
        if constexpr (kFragments) {
          if (c % 2 == 0 && c + 2 < kSteps) fp8::load_column_scales(cs[(c / 2 + 1) & 1], sb + (c / 2 + 1) * 16);
        }
        fp8::tmem_ld_wait_x16(r);
        if (c + 1 < kSteps) {
          load(c + 1, v[(c + 1) & 1]);
        } else {
          tc_fence_before_sync();
          if constexpr (!kSwap) {  // nothing of the slot is read after this (fragments: two steps ahead)
            __syncwarp();
            if (lane == 0) mbar_arrive(&tmem_empty[buf]);
          }
        }
        if constexpr (kFragments) {
          fp8::add_fragments(acc + (c >> 1) * 32 + (c & 1) * 16, r, cs[(c / 2) & 1], lo_hi[2 * (c & 1)], lo_hi[2 * (c & 1) + 1]);
        } else if constexpr (kSwap) {
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 s = *reinterpret_cast<const float4*>(slot + c * 16 + j);
            const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int q = 0; q < 4; ++q)
              acc[c * 16 + j + q] = fmaf(kRows ? f[q] * mine : f[q], __uint_as_float(r[j + q]), acc[c * 16 + j + q]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[c * 16 + j] = fmaf(mine, __uint_as_float(r[j]), acc[c * 16 + j]);
        }
      }
      if constexpr (kSwap) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&tmem_empty[buf]);
      }
      if (++buf == kBufs) buf = 0, phase ^= 1u;
    }
    if (ok) {  // the partial tile: every load has landed and every MMA has read it
      if constexpr (kSwap) {
#pragma unroll
        for (int j = 0; j < TM; ++j) red[j * kBlockN + row] = acc[j];
      } else if constexpr (kFragments) {
#pragma unroll
        for (int j = 0; j < kBlockN; j += 2) {
          const int m = quarter * 32 + 16 * ((j >> 4) & 1) + 8 * ((j >> 1) & 1) + (lane >> 2);
          const int g = 8 * (j >> 5) + 2 * ((j >> 2) & 3) + ((lane & 3) >> 1);
          *reinterpret_cast<float2*>(red + red_at<kSwap>(m, g) + 2 * (lane & 1)) = make_float2(acc[j], acc[j + 1]);
        }
      } else {
#pragma unroll
        for (int g = 0; g < kBlockN / 4; ++g)
          *reinterpret_cast<float4*>(red + red_at<kSwap>(row, g)) =
              make_float4(acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]);
      }
    }
  }

  // Every thread of every CTA of the cluster reaches both barriers, also on the abort path.
  tc_fence_before_sync();
  __syncwarp();
  if (p.splits > 1) cluster_sync_all();
  else __syncthreads();
  {
    // CTA r of the cluster adds the partial tiles of its 4-column groups: thread t takes group t % groups of
    // rows t / groups, t / groups + per, ...
    const uint32_t red_addr = smem_addr(red);
    constexpr int kGroups = kBlockN / 4;
    const int g0 = split * kGroups / p.splits, groups = (split + 1) * kGroups / p.splits - g0;
    const int rows = p.m - m0 < TM ? p.m - m0 : TM;
    const int per = kThreads / groups;
    const int first = static_cast<int>(threadIdx.x) / groups;
    const int g = g0 + static_cast<int>(threadIdx.x) % groups;
    const int n = n0 + 4 * g;
    float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < p.n) bias[j] = fp8::load_out(p.bias, n + j, p.d_type);
    }
    const bool whole = p.vec_d && n + 4 <= p.n;
    auto put = [&](int mi, const float4& f) {
      const float v[4] = {f.x + bias[0], f.y + bias[1], f.z + bias[2], f.w + bias[3]};
      const int64_t at = static_cast<int64_t>(m0 + mi) * p.ldd + n;
      if (whole) {
        if (p.d_type == fp8::kF32)
          *reinterpret_cast<float4*>(static_cast<float*>(p.d) + at) = make_float4(v[0], v[1], v[2], v[3]);
        else
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.d) + at) =
              make_uint2(fp8::pack_out(v[0], v[1], p.d_type), fp8::pack_out(v[2], v[3], p.d_type));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.n) fp8::store_out(p.d, at + j, p.d_type, v[j]);
      }
    };
    if (p.splits == 1) {
#pragma unroll 4
      for (int mi = first; mi < rows; mi += per) put(mi, *reinterpret_cast<const float4*>(red + red_at<kSwap>(mi, g)));
    } else if (first < per && n < p.n) {  // every load below feeds a store: none may be left in flight
#pragma unroll 2
      for (int mi = first; mi < rows; mi += per) {
        const uint32_t off = static_cast<uint32_t>(red_at<kSwap>(mi, g) * 4);
        float4 part[kMaxSplits];
#pragma unroll
        for (int s = 0; s < kMaxSplits; ++s)
          if (s < p.splits) part[s] = fp8::ld_dsmem_v4f(red_addr + off, static_cast<uint32_t>(s));
        float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int s = 0; s < kMaxSplits; ++s)
          if (s < p.splits) f.x += part[s].x, f.y += part[s].y, f.z += part[s].z, f.w += part[s].w;
        put(mi, f);
      }
    }
  }
  __syncwarp();
  // No CTA leaves while a peer may still read its partial tile. Each thread's reads are done, since it has
  // stored their sums, and nothing is handed over, so the arrival need not wait for the stores to D.
  if (p.splits > 1) fp8::cluster_sync_relaxed();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

}  // namespace fp8_tile
}  // namespace zcb
