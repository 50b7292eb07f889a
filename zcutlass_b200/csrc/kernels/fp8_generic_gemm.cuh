// 8-bit block-scaled product for operands TMA cannot describe (row strides
// that are no multiple of 16 bytes, unaligned bases): any size and alignment.
//
//   D[m, n] = sum_b sa[m, b] * sb[n, b] * sum_{k in block b} A[m, k] * B[n, k]  (+ bias[n])
//
// 64 x 64 outputs per block of 256 threads, 4 x 4 per thread. A block of 128 k is staged in shared
// memory as bytes by predicated loads, summed in 32 bits, then scaled into the 32-bit accumulators. On the
// CUDA cores: 95 ms, 20 TFLOP/s, at 8192 x 28672 x 4096.
#pragma once

#include "sm100_ptx.cuh"

namespace zcb {

struct Fp8GemmParams {
  int64_t m, n, k, lda, ldb, ldd;
  const uint8_t* a;
  const uint8_t* b;
  void* d;
  const float* a_scale;  // element (row, block) at row * a_scale_row + block * a_scale_blk
  int64_t a_scale_row, a_scale_blk;
  const float* b_scale;  // element (row / b_scale_rows, block)
  int64_t b_scale_row, b_scale_blk;
  int b_scale_rows;  // 1 or 128
  const void* bias;  // type of D; null: none
  int* error_word;
};

namespace fp8_generic {

constexpr int kTile = 64;
constexpr int kBlockK = 128;
constexpr int kPitch = kBlockK + 4;
constexpr int kThreads = 256;

template <bool kE5m2>
__device__ __forceinline__ float2 two(uint32_t pair) {
  uint32_t h;
  const uint16_t p = static_cast<uint16_t>(pair);
  if constexpr (kE5m2) asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"(p));
  else asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(p));
  return Elem<half>::unpack(h);
}

template <typename Out, bool kA5, bool kB5>
__global__ void __launch_bounds__(kThreads) gemm_kernel(const Fp8GemmParams p) {
  __shared__ __align__(16) uint8_t as[kTile * kPitch];
  __shared__ __align__(16) uint8_t bs[kTile * kPitch];
  griddep_wait();
  griddep_launch_dependents();
  const int64_t tiles_n = (p.n + kTile - 1) / kTile;
  const int64_t m0 = (blockIdx.x / tiles_n) * kTile, n0 = (blockIdx.x % tiles_n) * kTile;
  const int tm = threadIdx.x >> 4, tn = threadIdx.x & 15;  // rows tm + 16 i, columns tn + 16 j
  float acc[4][4] = {};
  for (int64_t k0 = 0, kb = 0; k0 < p.k; k0 += kBlockK, ++kb) {
    for (int i = threadIdx.x; i < kTile * kBlockK; i += kThreads) {
      const int r = i / kBlockK, c = i % kBlockK;
      const bool in_k = k0 + c < p.k;
      as[r * kPitch + c] = in_k && m0 + r < p.m ? p.a[(m0 + r) * p.lda + k0 + c] : 0;
      bs[r * kPitch + c] = in_k && n0 + r < p.n ? p.b[(n0 + r) * p.ldb + k0 + c] : 0;
    }
    __syncthreads();
    float part[4][4] = {};
    for (int c = 0; c < kBlockK; c += 4) {
      float av[4][4], bv[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t wa = *reinterpret_cast<const uint32_t*>(as + (tm + 16 * i) * kPitch + c);
        const uint32_t wb = *reinterpret_cast<const uint32_t*>(bs + (tn + 16 * i) * kPitch + c);
        const float2 a0 = two<kA5>(wa & 0xffffu), a1 = two<kA5>(wa >> 16);
        const float2 b0 = two<kB5>(wb & 0xffffu), b1 = two<kB5>(wb >> 16);
        av[i][0] = a0.x, av[i][1] = a0.y, av[i][2] = a1.x, av[i][3] = a1.y;
        bv[i][0] = b0.x, bv[i][1] = b0.y, bv[i][2] = b1.x, bv[i][3] = b1.y;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) part[i][j] = fmaf(av[i][q], bv[j][q], part[i][j]);
    }
    float sa[4], sb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t m = m0 + tm + 16 * i, n = n0 + tn + 16 * i;
      sa[i] = m < p.m ? p.a_scale[m * p.a_scale_row + kb * p.a_scale_blk] : 0.0f;
      sb[i] = n < p.n ? p.b_scale[(n / p.b_scale_rows) * p.b_scale_row + kb * p.b_scale_blk] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[i] * sb[j], part[i][j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + tm + 16 * i, n = n0 + tn + 16 * j;
      if (m >= p.m || n >= p.n) continue;
      float v = acc[i][j];
      Out* d = static_cast<Out*>(p.d) + m * p.ldd + n;
      const Out* bias = static_cast<const Out*>(p.bias);
      if constexpr (sizeof(Out) == 4) {
        *d = bias != nullptr ? v + bias[n] : v;
      } else {
        if (bias != nullptr) v += Elem<Out>::to_float(bias[n]);
        *d = Elem<Out>::from_float(v);
      }
    }
}

}  // namespace fp8_generic
}  // namespace zcb
