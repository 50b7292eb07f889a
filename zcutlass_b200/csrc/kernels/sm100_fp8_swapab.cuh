// 8-bit block-scaled product for few rows of A (decode, short prompts): B's
// rows (weights) fill the 128-row MMA dimension, MP = 16, 32, 64 or 128 rows of
// A (tokens) sit on MMA-N, and K is split over the CTAs of a cluster.
//
//   D^T[n, m] = sum_b sb(n, b) * sa(m, b) * (B_b A_b^T)[n, m]
//
// Bound by HBM while M is small: the weights are streamed once. A stage of the
// TMA ring holds KSUB blocks of 128 k (16 KiB of weights each). A thread of the
// four accumulation warps owns one weight row (TMEM lane) and MP accumulators;
// the token scales of a block, times the tile's weight scale, are staged in
// shared memory by the same warps, two slots in turn. With a scale per row of B
// (kRows) the thread's own row scale is a factor of its own.
// The splits' 32-bit partial tiles are added in split order through distributed
// shared memory, so the result does not depend on timing.
#pragma once

#include "sm100_fp8_common.cuh"

namespace zcb {

struct Fp8SwapParams {
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

namespace fp8_swap {

using fp8::kBlockK;
constexpr int kBlockN = 128;  // rows of B per tile (MMA M)
constexpr int kThreads = 192;
constexpr int kAccThreads = 128;
constexpr int kMaxSplits = 8;
constexpr int kAhead = 4;  // blocks the scale loads run ahead

template <int MP, int STAGES, int KSUB>
struct Smem {
  static constexpr int kWSub = kBlockN * kBlockK;  // 16 KiB
  static constexpr int kXSub = MP * kBlockK;
  static constexpr int kSub = kWSub + kXSub;
  static constexpr int kStageBytes = KSUB * kSub;
  static constexpr int kRedBytes = MP * kBlockN * 4;  // partial tile [m][n], over the drained ring
  static constexpr int kRing = STAGES * kStageBytes > kRedBytes ? STAGES * kStageBytes : kRedBytes;
  static constexpr int kScaleOff = kRing;  // [2][MP] floats
  static constexpr int kBarOff = kScaleOff + 2 * MP * 4;
  static constexpr int kBufs = 4;  // TMEM buffers; with MP <= 64 two CTAs fit an SM's 512 columns
  static constexpr int kNumBars = 2 * STAGES + 2 * kBufs + 1;
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;
  static constexpr int kDynamicBytes = kMiscOff + 16 + 1024;
  static constexpr uint32_t kTmemCols = kBufs * MP < 32 ? 32 : kBufs * MP;
  static_assert(MP == 16 || MP == 32 || MP == 64 || MP == 128, "");
  static_assert(kXSub % 1024 == 0 && kDynamicBytes <= 232448, "");
};

enum : int {
  kErrProducerEmpty = (33 << 4) | 1,
  kErrMmaFull = (33 << 4) | 2,
  kErrMmaTmemEmpty = (33 << 4) | 3,
  kErrAccTmemFull = (33 << 4) | 4,
};

template <int MP, int STAGES, int KSUB, bool kRows>
__global__ void __launch_bounds__(kThreads, MP == 128 ? 1 : 2)
    gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                const Fp8SwapParams p) {
  using L = Smem<MP, STAGES, KSUB>;
  constexpr int kBufs = L::kBufs;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* empty = full + STAGES;
  uint64_t* tmem_full = empty + STAGES;
  uint64_t* tmem_empty = tmem_full + kBufs;
  uint64_t* drain = tmem_empty + kBufs;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int split = static_cast<int>(blockIdx.x % p.splits);  // the cluster rank: clusters are `splits` wide
  const int tile = static_cast<int>(blockIdx.x / p.splits);
  const int m0 = (tile % p.tiles_m) * MP, n0 = (tile / p.tiles_m) * kBlockN;
  const int kb0 = static_cast<int>(static_cast<int64_t>(split) * p.num_kb / p.splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(split + 1) * p.num_kb / p.splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kBufs; ++b) {
      mbar_init(&tmem_full[b], 1);
      mbar_init(&tmem_empty[b], kAccThreads / 32);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();
  const WaitCtx ctx{abort_flag, p.error_word};

  if (warp == 0) {
    if (lane == 0) {
      // Weights are read once when one tile of tokens covers M; the tokens by every CTA.
      const uint64_t w_policy = p.tiles_m == 1 ? l2_policy_evict_first() : l2_policy_evict_last();
      const uint64_t x_policy = l2_policy_evict_last();
      uint32_t it = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; kb += KSUB, ++it) {
        const uint32_t s = it % STAGES;
        if (!fp8::wait(&empty[s], ((it / STAGES) & 1u) ^ 1u, ctx, kErrProducerEmpty)) {
          ok = false;
          break;
        }
        const int subs = kb1 - kb < KSUB ? kb1 - kb : KSUB;
        mbar_arrive_expect_tx(&full[s], subs * L::kSub);
#pragma unroll
        for (int sub = 0; sub < KSUB; ++sub) {
          if (sub >= subs) break;
          uint8_t* w = smem + s * L::kStageBytes + sub * L::kSub;
          tma_load_2d_hint(w, &tmap_w, &full[s], (kb + sub) * kBlockK, n0, w_policy);
          tma_load_2d_hint(w + L::kWSub, &tmap_x, &full[s], (kb + sub) * kBlockK, m0, x_policy);
        }
      }
      if (!ok) {  // loads already issued must land before the CTA can exit
        const uint32_t first = it > static_cast<uint32_t>(STAGES) ? it - STAGES : 0u;
        for (uint32_t j = first; j < it; ++j) mbar_wait_quiet(&full[j % STAGES], (j / STAGES) & 1u, 200000000ull);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      bool ok = true, issued = false;
      uint32_t i = 0;
      for (int kb = kb0; ok && kb < kb1; ++kb, ++i) {
        const uint32_t it = i / KSUB, sub = i % KSUB, s = it % STAGES;
        const uint32_t buf = i % kBufs;
        if (!fp8::wait(&tmem_empty[buf], ((i / kBufs) & 1u) ^ 1u, ctx, kErrMmaTmemEmpty) ||
            (sub == 0 && !fp8::wait(&full[s], (it / STAGES) & 1u, ctx, kErrMmaFull))) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t w = smem_addr(smem + s * L::kStageBytes + sub * L::kSub);
#pragma unroll
        for (int kk = 0; kk < kBlockK / fp8::kMmaK; ++kk)
          fp8::mma(tmem_base + buf * MP, smem_desc_sw128(w + kk * fp8::kMmaK, 16, 1024),
                   smem_desc_sw128(w + L::kWSub + kk * fp8::kMmaK, 16, 1024), p.idesc, kk != 0 ? 1u : 0u);
        issued = true;
        umma_commit(&tmem_full[buf]);
        if (sub == KSUB - 1) umma_commit(&empty[s]);
      }
      if (!ok && issued) {
        umma_commit(drain);
        mbar_wait_quiet(drain, 0, 200000000ull);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ accumulation
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;        // TMEM lane = row of B in the tile
    const int t = threadIdx.x - (kThreads - kAccThreads);
    float* scales = reinterpret_cast<float*>(smem + L::kScaleOff);
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const bool token = t < MP && m0 + t < p.m;
    const bool row_ok = n0 + row < p.n;
    const float* sa = p.a_scale + static_cast<int64_t>(m0 + t) * p.a_scale_row;
    const float* sb = p.b_scale + (kRows ? static_cast<int64_t>(n0 + row) : static_cast<int64_t>(n0 / kBlockN)) * p.b_scale_row;
    // Scales of the next kAhead blocks, in registers (zero outside the matrices).
    float a_next[kAhead], b_next[kAhead];
    auto fetch = [&](int kb, float& a, float& b) {
      const bool in = kb < kb1;
      a = in && token ? __ldg(sa + kb * p.a_scale_blk) : 0.0f;
      b = in && (!kRows || row_ok) ? __ldg(sb + kb * p.b_scale_blk) : 0.0f;
    };
#pragma unroll
    for (int u = 0; u < kAhead; ++u) fetch(kb0 + u, a_next[u], b_next[u]);
    uint64_t acc[MP / 2];
#pragma unroll
    for (int j = 0; j < MP / 2; ++j) acc[j] = 0;
    bool ok = true;
    // Unrolled by the distance of the scale loads: each has a register of its own until it is used.
#pragma unroll 1
    for (int kb = kb0; ok && kb < kb1; kb += kAhead) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (kb + u >= kb1) break;
        const uint32_t i = static_cast<uint32_t>(kb + u - kb0);
        const uint32_t buf = i % kBufs;
        float* slot = scales + (i & 1u) * MP;
        if (t < MP) slot[t] = kRows ? a_next[u] : a_next[u] * b_next[u];
        const uint64_t mine = fp8::both(b_next[u]);
        fetch(kb + u + kAhead, a_next[u], b_next[u]);
        ok = fp8::wait(&tmem_full[buf], (i / kBufs) & 1u, ctx, kErrAccTmemFull);
        ok = fp8::barrier_and<1, kAccThreads>(ok);  // the slot is written; all four warps go on, or none
        if (!ok) break;
        tc_fence_after_sync();
        uint32_t v[2][16];
        fp8::tmem_ld_x16(taddr + buf * MP, v[0]);
#pragma unroll
        for (int c = 0; c < MP / 16; ++c) {
          uint32_t(&w)[16] = v[c & 1];
          fp8::tmem_ld_wait_x16(w);
          if (c + 1 < MP / 16) {
            fp8::tmem_ld_x16(taddr + buf * MP + (c + 1) * 16, v[(c + 1) & 1]);
          } else {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tmem_empty[buf]);
          }
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(slot + c * 16 + j);
            uint64_t s0 = s.x, s1 = s.y;
            if constexpr (kRows) {
              s0 = fp8::mul2(s0, mine);
              s1 = fp8::mul2(s1, mine);
            }
            fp8::fma2(acc[c * 8 + j / 2], s0, fp8::pack2(w[j], w[j + 1]));
            fp8::fma2(acc[c * 8 + j / 2 + 1], s1, fp8::pack2(w[j + 2], w[j + 3]));
          }
        }
      }
    }
    if (ok && p.splits == 1) {
      const int n = n0 + row;
      if (row_ok) {
        const float bias = p.bias != nullptr ? fp8::load_out(p.bias, n, p.d_type) : 0.0f;
#pragma unroll
        for (int j = 0; j < MP; ++j) {
          const float2 v = fp8::unpack2(acc[j / 2]);
          if (m0 + j < p.m)
            fp8::store_out(p.d, static_cast<int64_t>(m0 + j) * p.ldd + n, p.d_type, ((j & 1) ? v.y : v.x) + bias);
        }
      }
    } else if (ok) {
      float* red = reinterpret_cast<float*>(smem);  // every load has landed and every MMA has read it
#pragma unroll
      for (int j = 0; j < MP; ++j) {
        const float2 v = fp8::unpack2(acc[j / 2]);
        red[j * kBlockN + row] = (j & 1) ? v.y : v.x;
      }
    }
  }

  tc_fence_before_sync();
  __syncwarp();
  if (p.splits > 1) {
    // Every thread of every CTA reaches both cluster barriers, also on the abort path.
    cluster_sync_all();
    const uint32_t red_addr = smem_addr(smem);
    constexpr int kGroups = kBlockN / 4;  // 4 consecutive n
    const int g0 = split * kGroups / p.splits, groups = (split + 1) * kGroups / p.splits - g0;
    const int rows = p.m - m0 < MP ? p.m - m0 : MP;
    const int total = groups * rows;
#pragma unroll 1
    for (int i = threadIdx.x; i < total; i += kThreads) {
      const int mi = i / groups, g = g0 + i % groups;
      const uint32_t off = static_cast<uint32_t>((mi * kBlockN + 4 * g) * 4);
      float4 part[kMaxSplits];
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s)
        if (s < p.splits) part[s] = fp8::ld_dsmem_v4f(red_addr + off, static_cast<uint32_t>(s));
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s)
        if (s < p.splits) {
          v[0] += part[s].x;
          v[1] += part[s].y;
          v[2] += part[s].z;
          v[3] += part[s].w;
        }
      const int n = n0 + 4 * g;
      const int64_t at = static_cast<int64_t>(m0 + mi) * p.ldd + n;
      if (p.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.n) v[j] += fp8::load_out(p.bias, n + j, p.d_type);
      }
      if (p.vec_d && n + 4 <= p.n) {
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
    }
    __syncwarp();
    cluster_sync_all();
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

}  // namespace fp8_swap
}  // namespace zcb
