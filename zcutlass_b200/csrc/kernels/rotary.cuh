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
// walks over heads, so its cosines and sines are loaded once for all of them.
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
  int head_lanes;   // threads that share a token's heads
  int items;        // vector positions per head
  int* error_word;
};

namespace rotary {

constexpr int kThreads = 256;
constexpr int kErrPosition = (32 << 4) | 1;

template <typename T, int V>
struct Pack;  // V values of T moved as one access
template <typename T>
struct Pack<T, 8> {
  static_assert(sizeof(T) == 2, "");
  __device__ static void load(const T* p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Elem<T>::unpack(w[i]);
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
  __device__ static void store(T* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]),
                                              Elem<T>::pack(v[4], v[5]), Elem<T>::pack(v[6], v[7]));
  }
};
template <>
struct Pack<float, 4> {
  __device__ static void load(const float* p, float (&v)[4]) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
  }
  __device__ static void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <typename T>
struct Pack<T, 1> {
  __device__ static void load(const T* p, float (&v)[1]) {
    if constexpr (sizeof(T) == 4) v[0] = *p;
    else v[0] = Elem<T>::to_float(*p);
  }
  __device__ static void store(T* p, const float (&v)[1]) {
    if constexpr (sizeof(T) == 4) *p = v[0];
    else *p = Elem<T>::from_float(v[0]);
  }
};

// Vector positions of a head: half layout, V pairs per item (two accesses of V values), then
// (head_dim - rotary_dim) / V items that pass through; interleaved layout, V / 2 pairs in one access
// (V = 1: the two values of a pair), then the same. V = 1 takes any stride, alignment and size.
template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int per_token = p.items * p.head_lanes;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t token = idx / per_token;
  if (token >= p.tokens) return;
  const int rest = static_cast<int>(idx - token * per_token);
  const int item = rest % p.items;
  const int half = p.rotary_dim / 2;
  constexpr int kStep = kInterleaved ? (V == 1 ? 2 : V) : V;  // values per access step of one item
  constexpr int kPairs = kInterleaved ? (V == 1 ? 1 : V / 2) : V;
  const int rot_items = half / kPairs;
  const bool turn = item < rot_items;
  const int64_t pos = p.positions64 ? static_cast<const int64_t*>(p.positions)[token]
                                    : static_cast<int64_t>(static_cast<const int32_t*>(p.positions)[token]);
  const bool known = pos >= 0 && pos < p.table_rows;  // below 0: padding; above: an error
  if (pos >= p.table_rows && rest == 0 && p.error_word != nullptr) atomicCAS(p.error_word, 0, kErrPosition);
  float c[kPairs] = {}, s[kPairs] = {};  // a position outside the table leaves the heads as they are
  if (turn && known) {
    const float* row = p.table + pos * p.table_ld + item * kPairs;
    if constexpr (kPairs % 4 == 0) {
#pragma unroll
      for (int i = 0; i < kPairs; i += 4) {
        const float4 a = *reinterpret_cast<const float4*>(row + i);
        const float4 b = *reinterpret_cast<const float4*>(row + half + i);
        c[i] = a.x, c[i + 1] = a.y, c[i + 2] = a.z, c[i + 3] = a.w;
        s[i] = b.x, s[i + 1] = b.y, s[i + 2] = b.z, s[i + 3] = b.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) c[i] = row[i], s[i] = row[half + i];
    }
    if (p.inverse) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) s[i] = -s[i];
    }
  }
  const int lane = rest / p.items;
  const int heads = p.x[0].heads + p.x[1].heads;
#pragma unroll 4
  for (int h = lane; h < heads; h += p.head_lanes) {
    const bool second = h >= p.x[0].heads;
    const RotaryTensor& x = p.x[second ? 1 : 0];
    const int hh = second ? h - p.x[0].heads : h;
    const T* in = static_cast<const T*>(x.in) + token * x.in_token + hh * x.in_head;
    T* out = static_cast<T*>(x.out) + token * x.out_token + hh * x.out_head;
    if (!turn) {
      if (in == out) continue;  // in place: nothing to move
      const int at = p.rotary_dim + (item - rot_items) * V;
      float v[V];
      Pack<T, V>::load(in + at, v);
      Pack<T, V>::store(out + at, v);
    } else if constexpr (kInterleaved && V > 1) {
      const int at = item * kStep;
      float v[V], y[V];
      Pack<T, V>::load(in + at, v);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        y[2 * i] = known ? v[2 * i] * c[i] - v[2 * i + 1] * s[i] : v[2 * i];
        y[2 * i + 1] = known ? v[2 * i + 1] * c[i] + v[2 * i] * s[i] : v[2 * i + 1];
      }
      Pack<T, V>::store(out + at, y);
    } else {
      const int a1 = kInterleaved ? 2 * item : item * V;
      const int a2 = kInterleaved ? 2 * item + 1 : half + item * V;
      float v1[V], v2[V], y1[V], y2[V];
      Pack<T, V>::load(in + a1, v1);
      Pack<T, V>::load(in + a2, v2);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        y1[i] = known ? v1[i] * c[i] - v2[i] * s[i] : v1[i];
        y2[i] = known ? v2[i] * c[i] + v1[i] * s[i] : v2[i];
      }
      Pack<T, V>::store(out + a1, y1);
      Pack<T, V>::store(out + a2, y2);
    }
  }
}

}  // namespace rotary
}  // namespace zcb
