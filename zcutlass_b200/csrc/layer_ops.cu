// Kernel choice and launch of the operators declared in layer_ops.hpp.
// Compiled for sm_100a only.
#include "layer_ops.hpp"

#include <algorithm>
#include <climits>

#include "kernels/fp8_generic_gemm.cuh"
#include "kernels/quantize_fp8.cuh"
#include "kernels/rotary.cuh"
#include "launchers.hpp"

namespace zcb {
namespace {

bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// One launch with the library's programmatic stream serialization.
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), int64_t grid, int threads, cudaStream_t stream, A... args) {
  if (grid < 1 || grid > INT_MAX) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = programmatic_launch() ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  count_launches(1);
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T, int kTop>
cudaError_t quantize(const QuantizeParams& p, bool block, cudaStream_t stream, int sms) {
  using namespace quant;
  const bool vec_in = aligned(p.x, 16) && p.ldx * static_cast<int64_t>(sizeof(T)) % 16 == 0;
  if (!block && p.qt == nullptr) {
    const int64_t blocks = div_up(p.rows, 8) * div_up(p.cols, kWarpVals);
    const bool vec_out = aligned(p.q, 16) && p.ldq % 16 == 0;
    return launch(rows_kernel<T, kTop>, std::min<int64_t>(blocks, 64 * static_cast<int64_t>(sms)), kRowThreads, stream, p,
                  vec_in, vec_out);
  }
  const bool vec_q = aligned(p.q, 8) && p.ldq % 8 == 0;
  const bool vec_qt = aligned(p.qt, 16) && p.ldqt % 16 == 0;
  const int64_t tiles = div_up(p.rows, kGroup) * div_up(p.cols, kGroup);
  auto go = [&](auto kernel) { return launch(kernel, tiles, kTileThreads, stream, p, vec_in, vec_q, vec_qt); };
  if (block) {
    if (p.qt == nullptr) return go(tile_kernel<T, kTop, true, false, true>);
    if (p.q == nullptr) return go(tile_kernel<T, kTop, false, true, true>);
    return go(tile_kernel<T, kTop, true, true, true>);
  }
  return p.q == nullptr ? go(tile_kernel<T, kTop, false, true, false>) : go(tile_kernel<T, kTop, true, true, false>);
}

template <typename Out>
cudaError_t generic_fp8(const Fp8GemmParams& p, bool a5, bool b5, cudaStream_t stream) {
  using namespace fp8_generic;
  const int64_t tiles = div_up(p.m, kTile) * div_up(p.n, kTile);
  auto go = [&](auto kernel) { return launch(kernel, tiles, kThreads, stream, p); };
  if (a5) return b5 ? go(gemm_kernel<Out, true, true>) : go(gemm_kernel<Out, true, false>);
  return b5 ? go(gemm_kernel<Out, false, true>) : go(gemm_kernel<Out, false, false>);
}

template <typename T, int V>
cudaError_t rotary_v(RotaryParams p, bool interleaved, cudaStream_t stream, int sms) {
  using namespace rotary;
  const int per_item = interleaved ? std::max(V / 2, 1) : V;
  p.items = p.rotary_dim / 2 / per_item + (p.head_dim - p.rotary_dim) / V;
  const int heads = p.x[0].heads + p.x[1].heads;
  // Threads per token: one per item and head lane. A thread that walks over several heads reuses its
  // cosines and sines and keeps more loads in flight; but first every SM gets two blocks.
  p.head_lanes = heads;
  while (p.head_lanes > 1 && (heads + p.head_lanes - 1) / p.head_lanes < 5 &&
         p.tokens * p.items * p.head_lanes > 4ll * sms * kThreads)
    p.head_lanes = (p.head_lanes + 1) / 2;
  const int64_t blocks = div_up(p.tokens * p.items * p.head_lanes, kThreads);
  return interleaved ? launch(rotary_kernel<T, V, true>, blocks, kThreads, stream, p)
                     : launch(rotary_kernel<T, V, false>, blocks, kThreads, stream, p);
}

template <typename T>
cudaError_t rotary_t(const RotaryParams& p, bool interleaved, cudaStream_t stream, int sms) {
  constexpr int kVec = 16 / sizeof(T);
  bool vec = p.rotary_dim % (interleaved ? kVec : 2 * kVec) == 0 && p.head_dim % kVec == 0 && aligned(p.table, 16) &&
             p.table_ld % 4 == 0 && p.rotary_dim % 8 == 0;
  for (const RotaryTensor& t : p.x) {
    if (t.heads == 0) continue;
    vec = vec && aligned(t.in, 16) && aligned(t.out, 16) && t.in_token % kVec == 0 && t.in_head % kVec == 0 &&
          t.out_token % kVec == 0 && t.out_head % kVec == 0;
  }
  return vec ? rotary_v<T, kVec>(p, interleaved, stream, sms) : rotary_v<T, 1>(p, interleaved, stream, sms);
}

}  // namespace

cudaError_t launch_quantize_fp8(const zcutlass_quantize_desc& d, const void* x, void* q, float* scale, void* qt,
                                float* scale_t, float* col_sums) {
  const DeviceInfo* info = current_device_info();
  if (info == nullptr) return cudaErrorInvalidDevice;
  const QuantizeParams p{x, d.rows, d.cols, d.ldx, static_cast<uint8_t*>(q), d.ldq, scale, d.scale_row, d.scale_blk,
                         static_cast<uint8_t*>(qt), d.ldqt, scale_t, d.scale_t_row, d.scale_t_blk, col_sums};
  const bool block = d.block_rows == 128;
  const cudaStream_t stream = static_cast<cudaStream_t>(d.stream);
  auto go = [&](auto zero) {
    using T = decltype(zero);
    return d.q_type == ZCUTLASS_E4M3 ? quantize<T, 8>(p, block, stream, info->sm_count)
                                     : quantize<T, 15>(p, block, stream, info->sm_count);
  };
  if (d.x_type == ZCUTLASS_F16) return go(half{});
  if (d.x_type == ZCUTLASS_BF16) return go(__nv_bfloat16{});
  return go(float{});
}

cudaError_t launch_sum_rows(const float* part, int64_t rows, int64_t cols, void* out, int32_t out_type,
                            cudaStream_t stream) {
  const int64_t blocks = div_up(cols, 256);
  if (out_type == ZCUTLASS_F16)
    return launch(quant::sum_kernel<half>, blocks, 256, stream, part, rows, cols, static_cast<half*>(out));
  if (out_type == ZCUTLASS_BF16)
    return launch(quant::sum_kernel<__nv_bfloat16>, blocks, 256, stream, part, rows, cols,
                  static_cast<__nv_bfloat16*>(out));
  return launch(quant::sum_kernel<float>, blocks, 256, stream, part, rows, cols, static_cast<float*>(out));
}

cudaError_t launch_gemm_fp8(const zcutlass_fp8_gemm_desc& d, const void* a, const float* a_scale, const void* b,
                            const float* b_scale, void* out) {
  const DeviceInfo* info = current_device_info();
  if (info == nullptr) return cudaErrorInvalidDevice;
  const Fp8GemmParams p{d.m, d.n, d.k, d.lda, d.ldb, d.ldd, static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(b),
                        out, a_scale, d.a_scale_row, d.a_scale_blk, b_scale, d.b_scale_row, d.b_scale_blk,
                        d.b_scale_rows, d.bias, info->error_word};
  const bool a5 = d.a_type == ZCUTLASS_E5M2, b5 = d.b_type == ZCUTLASS_E5M2;
  const cudaStream_t stream = static_cast<cudaStream_t>(d.stream);
  if (d.d_type == ZCUTLASS_F16) return generic_fp8<half>(p, a5, b5, stream);
  if (d.d_type == ZCUTLASS_BF16) return generic_fp8<__nv_bfloat16>(p, a5, b5, stream);
  return generic_fp8<float>(p, a5, b5, stream);
}

cudaError_t launch_rotary(const zcutlass_rotary_desc& d, const void* q, void* q_out, const void* k, void* k_out,
                          const void* positions, const float* table) {
  const DeviceInfo* info = current_device_info();
  if (info == nullptr) return cudaErrorInvalidDevice;
  RotaryParams p{};
  p.x[0] = {q, q_out, d.q_token, d.q_head, d.q_out_token, d.q_out_head, d.q_heads};
  p.x[1] = {k, k_out, d.k_token, d.k_head, d.k_out_token, d.k_out_head, d.k_heads};
  p.positions = positions;
  p.positions64 = d.positions64 != 0;
  p.tokens = d.tokens;
  p.table = table;
  p.table_rows = d.table_rows;
  p.table_ld = d.table_ld;
  p.head_dim = d.head_dim;
  p.rotary_dim = d.rotary_dim;
  p.inverse = d.inverse != 0;
  p.error_word = info->error_word;
  const cudaStream_t stream = static_cast<cudaStream_t>(d.stream);
  const bool inter = d.interleaved != 0;
  if (d.dtype == ZCUTLASS_F16) return rotary_t<half>(p, inter, stream, info->sm_count);
  if (d.dtype == ZCUTLASS_BF16) return rotary_t<__nv_bfloat16>(p, inter, stream, info->sm_count);
  return rotary_t<float>(p, inter, stream, info->sm_count);
}

}  // namespace zcb
