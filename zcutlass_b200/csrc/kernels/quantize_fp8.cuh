// Quantisation of f32/f16/bf16 matrices to 8-bit floating point (e4m3, e5m2)
// with one power-of-two scale per group of 128.
//
//   group g (1 x 128 values of a row, 128 x 1 of a column, or a 128 x 128 block):
//     amax = max |x|            s = 2^ceil(log2(amax / max8)), at least 2^-126, 1 when amax = 0
//     q    = x / s rounded to nearest even, so |q| <= max8 = 1.75 * 2^top (top = 8 for e4m3, 15 for e5m2)
//   A group that holds an infinity or a NaN gets s = NaN and q = NaN, so the fault reaches every result
//   that uses the group instead of vanishing in a scale.
//
// Scales are powers of two so that x / s is exact in 32 bits: the only rounding is the one to 8 bits, and
// any implementation of the formula gives the same bits. Against s = amax / max8 this gives up at most
// one binade at the low end of the type, where e4m3 still has 2^-9 of the group's largest value's binade.
//
// Memory-bound: 4 or 2 bytes in and 1 (2 with the transpose) out per value. Measured against 6.5 TB/s of a
// plain copy: rows of 8192 x 4096 bf16 18.7 us (5.4 TB/s), columns 18.1 (5.6), both 28.5 (4.7: every value is
// scaled and converted twice), 128 x 128 blocks of 14336 x 4096 f32 47.2 (6.2).
#pragma once

#include "sm100_ptx.cuh"

namespace zcb {

struct QuantizeParams {
  const void* x;
  int64_t rows, cols, ldx;
  uint8_t* q;  // [rows, cols], row stride ldq; null: not written
  int64_t ldq;
  float* scale;  // element (r, g) at r * scale_row + g * scale_blk
  int64_t scale_row, scale_blk;
  uint8_t* qt;  // [cols, rows], row stride ldqt; null: not written
  int64_t ldqt;
  float* scale_t;  // element (c, g) at c * scale_t_row + g * scale_t_blk
  int64_t scale_t_row, scale_t_blk;
  float* col_sums;  // [ceil(rows / 128), cols] sums over each 128 rows; null: not written
};

namespace quant {

constexpr int kGroup = 128;
constexpr int kRowThreads = 256;
constexpr int kLaneVals = 16;                          // values per lane in the row kernel
constexpr int kWarpVals = 32 * kLaneVals;              // 512 columns (4 groups) of one row per warp
constexpr int kTileThreads = 256;

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else return Elem<T>::to_float(v);
}

// 8 consecutive values, the first `n` of them in range (the others become 0).
// `vec`: the address is 16-byte aligned whenever n >= 8.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t n, bool vec, float (&v)[8]) {
  if (n >= 8 && vec) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p);
      const float4 b = *reinterpret_cast<const float4*>(p + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = Elem<T>::unpack(w[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.0f;
  }
}

// |v| as an integer: ordered as the values are, with infinity and NaN above all.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct Scale {
  float s, inverse;
};

// The smallest power of two s with amax <= 1.75 * 2^kTop * s, and 1 / s.
template <int kTop>
__device__ __forceinline__ Scale scale_of(uint32_t amax) {
  if (amax >= 0x7f800000u) {
    const float nan = __uint_as_float(0x7fffffffu);
    return {nan, nan};
  }
  if (amax == 0) return {1.0f, 1.0f};
  int k = static_cast<int>(amax >> 23) - 127 - kTop + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  k = k < -126 ? -126 : k;
  return {__uint_as_float(static_cast<uint32_t>(k + 127) << 23), __uint_as_float(static_cast<uint32_t>(127 - k) << 23)};
}

template <int kTop>
__device__ __forceinline__ uint32_t cvt2(float lo, float hi) {
  uint16_t r;
  if constexpr (kTop == 8)
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

template <int kTop>
__device__ __forceinline__ uint32_t cvt4(const float* v, float inverse) {
  return cvt2<kTop>(v[0] * inverse, v[1] * inverse) | (cvt2<kTop>(v[2] * inverse, v[3] * inverse) << 16);
}

// The first `n` of 8 bytes to p (8-byte aligned whenever n >= 8 and vec).
__device__ __forceinline__ void store8(uint8_t* p, uint2 b, int64_t n, bool vec) {
  if (n >= 8 && vec) {
    *reinterpret_cast<uint2*>(p) = b;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = static_cast<uint8_t>((i < 4 ? b.x >> (8 * i) : b.y >> (8 * (i - 4))) & 0xffu);
  }
}

// Rows only: a lane holds 16 values (16 bytes to write; 8 values per lane and whole runs per access took 22.6
// us, a persistent grid with the next loads ahead 19.0), 8 lanes one group, a warp 512 columns of a row; the 8 warps of a
// block take 8 rows of the same columns, whose scales are neighbours in the [group][row] layout.
template <typename T, int kTop>
__global__ void __launch_bounds__(kRowThreads) rows_kernel(const QuantizeParams p, bool vec_in, bool vec_out) {
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t chunks = (p.cols + kWarpVals - 1) / kWarpVals;
  const int64_t blocks = ((p.rows + 7) / 8) * chunks;
  for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int64_t r = (b / chunks) * 8 + warp;
    const int64_t c = (b % chunks) * kWarpVals + lane * kLaneVals;
    const int64_t n = r < p.rows ? p.cols - c : 0;
    const T* src = static_cast<const T*>(p.x) + r * p.ldx + c;
    float v[2][8];
    load8(src, n, vec_in, v[0]);
    load8(src + 8, n - 8, vec_in, v[1]);
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, max(abs_bits(v[0][i]), abs_bits(v[1][i])));
#pragma unroll
    for (int o = 1; o < 8; o *= 2) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (n <= 0) continue;
    const Scale s = scale_of<kTop>(amax);
    const uint4 out = make_uint4(cvt4<kTop>(v[0], s.inverse), cvt4<kTop>(v[0] + 4, s.inverse),
                                 cvt4<kTop>(v[1], s.inverse), cvt4<kTop>(v[1] + 4, s.inverse));
    uint8_t* dst = p.q + r * p.ldq + c;
    if (n >= 16 && vec_out) {
      *reinterpret_cast<uint4*>(dst) = out;
    } else {
      store8(dst, make_uint2(out.x, out.y), n, false);
      store8(dst + 8, make_uint2(out.z, out.w), n - 8, false);
    }
    if ((lane & 7) == 0) p.scale[r * p.scale_row + (c / kGroup) * p.scale_blk] = s.s;
  }
}

// Eight values as they are loaded: 16-bit types stay packed, so that a thread's 64 values take 32 registers
// and three or four blocks fit an SM (two, with the values unpacked, kept too few loads in flight).
template <typename T>
struct Raw8 {
  static constexpr int kWords = 8 * sizeof(T) / 4;
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const T* p, int64_t n, bool vec) {
    if (n >= 8 && vec) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + i);
        w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = i < n ? __float_as_uint(p[i]) : 0u;
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = (2 * i < n ? h[2 * i] : 0u) | (2 * i + 1 < n ? static_cast<uint32_t>(h[2 * i + 1]) << 16 : 0u);
    }
  }
  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
    else {
      const float2 f = Elem<T>::unpack(w[j >> 1]);
      return (j & 1) ? f.y : f.x;
    }
  }
};

// The largest magnitudes of words: 32-bit values, or the two 16-bit values of a word each on its own. Both are
// ordered as their bits are, infinities and NaN on top.
template <typename T>
__device__ __forceinline__ uint32_t max_mag(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 4) return max(a, b);
  else return __vmaxu2(a, b);
}
template <typename T>
__device__ __forceinline__ uint32_t mag(uint32_t w) {
  return w & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu);
}
// A magnitude as the bits of a 32-bit value (16-bit types: the low half).
template <typename T>
__device__ __forceinline__ uint32_t mag_bits(uint32_t m) {
  if constexpr (sizeof(T) == 4) return m;
  else return __float_as_uint(Elem<T>::unpack(m).x);
}

// A 128 x 128 tile per block, read once: 16 threads cover a row (8 columns each) and hold 8 consecutive
// rows, so a thread's 8 x 8 values give 8 bytes of a row and 8 bytes of a column of the results. The
// transposed bytes go through shared memory to be written as whole 128-byte rows; their 16-byte units are
// permuted by the column's eighth, so that the 16 threads of a row (8 columns apart) meet different banks.
// kBlock: one scale for the tile; else one per row (kRows) and one per column (kCols) of it.
// Four blocks per SM leave 64 registers: both axes of 16-bit values spill 72 bytes per thread and are faster for it
// (8192 x 4096 bf16 28.5 us against 29.5 with three blocks); blocks with the transpose, at three, spill 12
// (26.1 us, 5.1 TB/s).
template <typename T, int kTop, bool kRows, bool kCols, bool kBlock>
__global__ void __launch_bounds__(kTileThreads, sizeof(T) == 4 ? 2 : (kBlock && kRows && kCols ? 3 : 4))
    tile_kernel(const QuantizeParams p, bool vec_in, bool vec_q, bool vec_qt) {
  constexpr int kWarps = kTileThreads / 32;
  constexpr bool kColStats = kCols && !kBlock;
  constexpr int kWords = Raw8<T>::kWords;
  __shared__ __align__(16) uint32_t col_amax[kColStats ? kWarps : 1][kGroup * sizeof(T) / 4];
  __shared__ __align__(16) float col_part[kColStats ? kWarps : 1][kGroup];
  __shared__ __align__(16) float col_inverse[kGroup];
  __shared__ __align__(16) uint8_t turned[kCols ? kGroup * kGroup : 16];
  __shared__ uint32_t warp_amax[kWarps];
  griddep_wait();
  griddep_launch_dependents();
  const int slot = threadIdx.x >> 4;         // 8 rows
  const int warp = threadIdx.x >> 5;
  const int c0 = (threadIdx.x & 15) * 8;     // 8 columns
  const int64_t tiles_c = (p.cols + kGroup - 1) / kGroup;
  const int64_t tr = blockIdx.x / tiles_c, tc = blockIdx.x - tr * tiles_c;
  const int64_t row0 = tr * kGroup + slot * 8, col0 = tc * kGroup + c0;
  const int64_t n = p.cols - col0;
  Raw8<T> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    v[i].load(static_cast<const T*>(p.x) + (row0 + i) * p.ldx + col0, row0 + i < p.rows ? n : 0, vec_in);

  Scale block_scale{1.0f, 1.0f};
  if constexpr (kBlock) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < kWords; ++j) m = max_mag<T>(m, mag<T>(v[i].w[j]));
    uint32_t amax = mag_bits<T>(m);
    if constexpr (sizeof(T) == 2) amax = max(amax, mag_bits<T>(m >> 16));
    amax = __reduce_max_sync(0xffffffffu, amax);
    if ((threadIdx.x & 31) == 0) warp_amax[warp] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) amax = max(amax, warp_amax[w]);
    block_scale = scale_of<kTop>(amax);
    if (threadIdx.x == 0) {
      if (kRows) p.scale[tr * p.scale_row + tc * p.scale_blk] = block_scale.s;
      if (kCols) p.scale_t[tc * p.scale_t_row + tr * p.scale_t_blk] = block_scale.s;
    }
  }
  if constexpr (kColStats) {
    // Column maxima over the thread's 8 rows, then over the warp's two slots.
    uint32_t m[kWords] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < kWords; ++j) m[j] = max_mag<T>(m[j], mag<T>(v[i].w[j]));
#pragma unroll
    for (int j = 0; j < kWords; ++j) m[j] = max_mag<T>(m[j], __shfl_xor_sync(0xffffffffu, m[j], 16));
    if ((threadIdx.x & 16) == 0) {
#pragma unroll
      for (int j = 0; j < kWords; j += 4)
        *reinterpret_cast<uint4*>(&col_amax[warp][(threadIdx.x & 15) * kWords + j]) = make_uint4(m[j], m[j + 1], m[j + 2], m[j + 3]);
    }
    if (p.col_sums != nullptr) {
      float sum[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[j] += v[i].get(j);
        sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 16);
      }
      if ((threadIdx.x & 16) == 0) {
        *reinterpret_cast<float4*>(&col_part[warp][c0]) = make_float4(sum[0], sum[1], sum[2], sum[3]);
        *reinterpret_cast<float4*>(&col_part[warp][c0 + 4]) = make_float4(sum[4], sum[5], sum[6], sum[7]);
      }
    }
    __syncthreads();
    if (threadIdx.x < kGroup) {
      uint32_t amax = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        uint32_t word = col_amax[w][threadIdx.x * sizeof(T) / 4];
        if constexpr (sizeof(T) == 2) word = (threadIdx.x & 1) ? word >> 16 : word & 0xffffu;
        amax = max(amax, word);
      }
      const Scale s = scale_of<kTop>(mag_bits<T>(amax));
      col_inverse[threadIdx.x] = s.inverse;
      const int64_t c = tc * kGroup + threadIdx.x;
      if (c < p.cols) {
        p.scale_t[c * p.scale_t_row + tr * p.scale_t_blk] = s.s;
        if (p.col_sums != nullptr) {
          float sum = 0.0f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) sum += col_part[w][threadIdx.x];
          p.col_sums[tr * p.cols + c] = sum;
        }
      }
    }
    __syncthreads();
  }
  if constexpr (kRows) {
    // Row maxima over 16 threads. Each exchange halves the rows a thread is responsible for (two rows share
    // a word with 16-bit types), so 8 rows take 5 or 8 shuffles instead of 32, and each scale is computed by
    // the threads that end up with its row.
    constexpr int kPer = sizeof(T) == 2 ? 2 : 1;  // rows per word
    constexpr int kHeld = 8 / kPer;
    constexpr int kKeep = kPer == 2 ? 4 : 2;      // the last exchange that halves
    const int lane = threadIdx.x & 31;
    Scale mine[kPer];
    if constexpr (!kBlock) {
      uint32_t m[kHeld];
#pragma unroll
      for (int h = 0; h < kHeld; ++h) {
        uint32_t row[kPer];
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          row[e] = 0;
#pragma unroll
          for (int j = 0; j < kWords; ++j) row[e] = max_mag<T>(row[e], mag<T>(v[h * kPer + e].w[j]));
        }
        if constexpr (kPer == 2) m[h] = __vmaxu2(__byte_perm(row[0], row[1], 0x5410), __byte_perm(row[0], row[1], 0x7632));
        else m[h] = row[0];
      }
#pragma unroll
      for (int o = 8, left = kHeld; o >= 1; o /= 2) {
        if (o >= kKeep) {
          left /= 2;
          const bool upper = (lane & o) != 0;
#pragma unroll
          for (int h = 0; h < kHeld / 2; ++h) {
            if (h >= left) break;
            const uint32_t keep = upper ? m[h + left] : m[h], give = upper ? m[h] : m[h + left];
            m[h] = max_mag<T>(keep, __shfl_xor_sync(0xffffffffu, give, o));
          }
        } else {
          m[0] = max_mag<T>(m[0], __shfl_xor_sync(0xffffffffu, m[0], o));
        }
      }
      const int first = (kPer == 2 ? ((lane & 12) >> 2) : ((lane & 14) >> 1)) * kPer;  // the thread's first row
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        mine[e] = scale_of<kTop>(mag_bits<T>(e == 0 ? m[0] & (kPer == 2 ? 0xffffu : 0xffffffffu) : m[0] >> 16));
        const int64_t r = row0 + first + e;
        if ((lane & (kKeep - 1)) == 0 && r < p.rows) p.scale[r * p.scale_row + tc * p.scale_blk] = mine[e].s;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float inv = block_scale.inverse;
      if constexpr (!kBlock) inv = __shfl_sync(0xffffffffu, mine[i % kPer].inverse, (lane & 16) | (i / kPer) * kKeep);
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = v[i].get(j);
      if (row0 + i < p.rows)
        store8(p.q + (row0 + i) * p.ldq + col0, make_uint2(cvt4<kTop>(f, inv), cvt4<kTop>(f + 4, inv)), n, vec_q);
    }
  }
  if constexpr (kCols) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float inv = kBlock ? block_scale.inverse : col_inverse[c0 + j];
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = v[i].get(j);
      *reinterpret_cast<uint2*>(turned + (c0 + j) * kGroup + (((slot >> 1) ^ (threadIdx.x & 7)) << 4) + (slot & 1) * 8) =
          make_uint2(cvt4<kTop>(f, inv), cvt4<kTop>(f + 4, inv));
    }
    __syncthreads();
    // 8 threads write one 128-byte row of the transposed tile, 32 rows at a time.
    const int unit = threadIdx.x & 7;
    const int64_t r = tr * kGroup + unit * 16;
    const int64_t left = p.rows - r;
#pragma unroll
    for (int k = 0; k < kGroup; k += kTileThreads / 8) {
      const int c = k + (threadIdx.x >> 3);
      if (tc * kGroup + c >= p.cols) continue;
      const uint4 b = *reinterpret_cast<const uint4*>(turned + c * kGroup + ((unit ^ ((c >> 3) & 7)) << 4));
      uint8_t* dst = p.qt + (tc * kGroup + c) * p.ldqt + r;
      if (left >= 16 && vec_qt) {
        *reinterpret_cast<uint4*>(dst) = b;
      } else {
        store8(dst, make_uint2(b.x, b.y), left, false);
        store8(dst + 8, make_uint2(b.z, b.w), left - 8, false);
      }
    }
  }
}

// out[c] = sum over blocks of part[b][c], in order: the result does not depend on timing.
template <typename T>
__global__ void __launch_bounds__(256) sum_kernel(const float* part, int64_t blocks, int64_t cols, T* out) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= cols) return;
  float sum = 0.0f;
#pragma unroll 8
  for (int64_t b = 0; b < blocks; ++b) sum += part[b * cols + c];
  if constexpr (sizeof(T) == 4) out[c] = sum;
  else out[c] = Elem<T>::from_float(sum);
}

}  // namespace quant
}  // namespace zcb
