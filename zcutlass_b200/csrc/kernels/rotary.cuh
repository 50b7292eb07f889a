// Rotary positions on the heads of q and k, from a [positions, rotary_dim] table of cosines (first half
// of a row) and sines (second half), held in 32 bits.
//
//   pair (x1, x2) of a head at angle t:  y1 = x1 cos t - x2 sin t,  y2 = x2 cos t + x1 sin t
//   half layout:        pair i = (x[i], x[i + rotary_dim / 2])
//   interleaved layout: pair i = (x[2 i], x[2 i + 1])
//   values rotary_dim .. head_dim - 1 of a head pass through.
// The rotation is orthogonal up to the factor the table's entries share, so the gradient is the same
// kernel with the sines negated. Computed in 32 bits, rounded once to the tensor's type.
//
// Memory-bound: each value is read and written once. A thread takes one vector position of the head and
// walks over heads, so its cosines and sines are loaded once for all of them. Measured on views of a packed qkv
// matrix, 32 + 8 heads of 128, bf16: 8192 tokens 31.3 us (5.5 TB/s of the copy's 6.5; one head at a time and 64-bit
// division took 32.5), 16 tokens 1.9 us.
#pragma once

#include "sm100_ptx.cuh"

namespace zcb {

struct RotaryTensor {
  const void* in;
  void* out;
  int64_t in_token, in_head, out_token, out_head;  // strides in elements
  int heads;
};

struct RotaryParams {
  RotaryTensor x[2];  // q and k (heads = 0: absent)
  const void* positions;
  bool positions64;
  int64_t tokens;
  const float* table;
  int64_t table_rows, table_ld;
  int head_dim, rotary_dim;
  bool inverse;
  bool small;       // thread indices fit 31 bits
  int head_lanes;   // threads that share a token's heads
  int items;        // vector positions per head
  int* error_word;
};

namespace rotary {

constexpr int kThreads = 256;
constexpr int kErrPosition = (32 << 4) | 1;

// V values of T moved as one access (16 bytes, or one value).
template <typename T, int V>
struct Pack {
  static_assert(V == 1 || V * sizeof(T) == 16, "");
  static constexpr int kWords = V == 1 ? 1 : 4;
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 1) {
      if constexpr (sizeof(T) == 4) w[0] = __float_as_uint(*p);
      else w[0] = __float_as_uint(Elem<T>::to_float(*p));
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V == 1) {
      if constexpr (sizeof(T) == 4) *p = __uint_as_float(w[0]);
      else *p = Elem<T>::from_float(__uint_as_float(w[0]));
    } else {
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __device__ __forceinline__ void get(float (&v)[V]) const {
    if constexpr (V == 1 || sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float2 f = Elem<T>::unpack(w[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&v)[V]) {
    if constexpr (V == 1 || sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) w[i] = Elem<T>::pack(v[2 * i], v[2 * i + 1]);
    }
  }
};

// Vector positions of a head: half layout, V pairs per item (two accesses of V values), then
// (head_dim - rotary_dim) / V items that pass through; interleaved layout, V / 2 pairs in one access
// (V = 1: the two values of a pair), then the same. V = 1 takes any stride, alignment and size.
// A thread takes kBatch heads at a time, all their loads before the first store (in place, the compiler may
// not move a load over a store).
template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int kBatch = 4;
  constexpr int kParts = kInterleaved && V > 1 ? 1 : 2;      // accesses per item
  constexpr int kPairs = kInterleaved ? (V == 1 ? 1 : V / 2) : V;
  const uint32_t per_token = static_cast<uint32_t>(p.items) * p.head_lanes;
  int64_t token;
  uint32_t rest;
  if (p.small) {  // 32-bit division
    const uint32_t idx = blockIdx.x * kThreads + threadIdx.x;
    const uint32_t t = idx / per_token;
    token = t, rest = idx - t * per_token;
  } else {
    const int64_t idx = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    token = idx / per_token, rest = static_cast<uint32_t>(idx - token * per_token);
  }
  if (token >= p.tokens) return;
  const int lane = static_cast<int>(rest / p.items);
  const int item = static_cast<int>(rest) - lane * p.items;
  const int half = p.rotary_dim / 2;
  const int rot_items = half / kPairs;
  const int64_t pos = p.positions64 ? static_cast<const int64_t*>(p.positions)[token]
                                    : static_cast<int64_t>(static_cast<const int32_t*>(p.positions)[token]);
  const bool known = pos >= 0 && pos < p.table_rows;  // below 0: padding; above: an error
  if (pos >= p.table_rows && rest == 0 && p.error_word != nullptr) atomicCAS(p.error_word, 0, kErrPosition);
  const bool rotated = item < rot_items;
  const bool turn = rotated && known;  // else the values are copied as they are
  // Offsets of the item's accesses in a head.
  const int at0 = !rotated ? p.rotary_dim + (item - rot_items) * V : kInterleaved ? (V == 1 ? 2 * item : V * item) : V * item;
  const int at1 = kInterleaved ? at0 + 1 : at0 + half;
  const int parts = rotated ? kParts : 1;
  float c[kPairs] = {}, s[kPairs] = {};
  if (turn) {
    const float* row = p.table + pos * p.table_ld + item * kPairs;
    if constexpr (kPairs % 4 == 0) {
#pragma unroll
      for (int i = 0; i < kPairs; i += 4) {
        const float4 a = ld_written(reinterpret_cast<const float4*>(row + i));
        const float4 b = ld_written(reinterpret_cast<const float4*>(row + half + i));
        c[i] = a.x, c[i + 1] = a.y, c[i + 2] = a.z, c[i + 3] = a.w;
        s[i] = b.x, s[i + 1] = b.y, s[i + 2] = b.z, s[i + 3] = b.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) c[i] = ld_written(row + i), s[i] = ld_written(row + half + i);
    }
    if (p.inverse) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) s[i] = -s[i];
    }
  }
  const int heads = p.x[0].heads + p.x[1].heads;
  const T* in0 = static_cast<const T*>(p.x[0].in) + token * p.x[0].in_token;
  const T* in1 = static_cast<const T*>(p.x[1].in) + token * p.x[1].in_token;
  T* out0 = static_cast<T*>(p.x[0].out) + token * p.x[0].out_token;
  T* out1 = static_cast<T*>(p.x[1].out) + token * p.x[1].out_token;
  for (int h0 = lane; h0 < heads; h0 += kBatch * p.head_lanes) {
    Pack<T, V> v[kBatch][kParts];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int h = h0 + b * p.head_lanes;
      if (h >= heads) break;
      const T* in = h < p.x[0].heads ? in0 + h * p.x[0].in_head : in1 + (h - p.x[0].heads) * p.x[1].in_head;
      v[b][0].load(in + at0);
      if (kParts == 2 && parts == 2) v[b][kParts - 1].load(in + at1);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int h = h0 + b * p.head_lanes;
      if (h >= heads) break;
      T* out = h < p.x[0].heads ? out0 + h * p.x[0].out_head : out1 + (h - p.x[0].heads) * p.x[1].out_head;
      if (turn) {
        float x[kParts][V], y[kParts][V];
#pragma unroll
        for (int q = 0; q < kParts; ++q) v[b][q].get(x[q]);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const float x1 = kParts == 1 ? x[0][2 * i] : x[0][i];
          const float x2 = kParts == 1 ? x[0][(2 * i + 1) % V] : x[kParts - 1][i];
          const float y1 = x1 * c[i] - x2 * s[i], y2 = x2 * c[i] + x1 * s[i];
          if constexpr (kParts == 1) y[0][2 * i] = y1, y[0][(2 * i + 1) % V] = y2;
          else y[0][i] = y1, y[kParts - 1][i] = y2;
        }
#pragma unroll
        for (int q = 0; q < kParts; ++q) v[b][q].set(y[q]);
      }
      v[b][0].store(out + at0);
      if (kParts == 2 && parts == 2) v[b][kParts - 1].store(out + at1);
    }
  }
}

}  // namespace rotary
}  // namespace zcb
