// Kernel choice and launch of the operators declared in layer_ops.hpp.
// Compiled for sm_100a only.
#include "layer_ops.hpp"

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdlib>
#include <cstring>

#include "kernels/fp8_generic_gemm.cuh"
#include "kernels/quantize_fp8.cuh"
#include "kernels/rotary.cuh"
#include "kernels/sm100_fp8_pair.cuh"
#include "kernels/sm100_fp8_tile.cuh"
#include "launchers.hpp"
#include "tma_desc.hpp"

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

// ---------------------------------------------------------------- 8-bit product on tcgen05

// One launch of a kernel with dynamic shared memory (its limit is raised once per device) in clusters of
// `cluster` CTAs.
template <typename... P, typename... A>
cudaError_t launch_cluster(void (*kernel)(P...), std::atomic<uint64_t>& ready, const DeviceInfo& dev, int smem, int64_t grid,
                           int threads, int cluster, cudaStream_t stream, const A&... args) {
  if (grid < 1 || grid > INT_MAX) return cudaErrorInvalidValue;
  const uint64_t bit = uint64_t(1) << (dev.ordinal & 63);
  if ((ready.load(std::memory_order_acquire) & bit) == 0) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit, std::memory_order_acq_rel);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (programmatic_launch()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  count_launches(1);
  return e != cudaSuccess ? e : cudaGetLastError();
}

bool fp8_map(CUtensorMap* map, const uint8_t* base, int64_t rows, int64_t k, int64_t ld, int box_rows) {
  return make_tma_2d(map, base, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rows, k, ld, box_rows, fp8::kBlockK, TmaSwizzle::B128);
}

struct Fp8Types {
  bool a5, b5;
  int d;  // zcutlass_dtype
  int d_bytes() const { return d == ZCUTLASS_F32 ? 4 : 2; }
};

template <bool kSwap, int TM, int STAGES, int KSUB>
cudaError_t tile_fp8(const Fp8GemmParams& g, const Fp8Types& t, const DeviceInfo& dev, int splits, cudaStream_t stream) {
  CUtensorMap ta, tb;
  if (!fp8_map(&ta, g.a, g.m, g.k, g.lda, TM) || !fp8_map(&tb, g.b, g.n, g.k, g.ldb, fp8_tile::kBlockN))
    return cudaErrorInvalidValue;
  const int64_t tiles_m = div_up(g.m, TM);
  Fp8TileParams p{};
  p.m = static_cast<int>(g.m), p.n = static_cast<int>(g.n);
  p.num_kb = static_cast<int>(div_up(g.k, fp8::kBlockK));
  p.splits = splits;
  p.tiles_m = static_cast<int>(tiles_m);
  p.a_scale = g.a_scale, p.a_scale_row = g.a_scale_row, p.a_scale_blk = g.a_scale_blk;
  p.b_scale = g.b_scale, p.b_scale_row = g.b_scale_row, p.b_scale_blk = g.b_scale_blk;
  p.d = g.d, p.ldd = g.ldd, p.d_type = t.d;
  p.vec_d = g.ldd % 4 == 0 && aligned(g.d, 4 * t.d_bytes());
  p.bias = g.bias;
  p.idesc = kSwap ? fp8::idesc(fp8_tile::kBlockN, TM, t.b5, t.a5) : fp8::idesc(TM, fp8_tile::kBlockN, t.a5, t.b5);
  p.error_word = dev.error_word;
  const int64_t grid = tiles_m * div_up(g.n, fp8_tile::kBlockN) * splits;
  static std::atomic<uint64_t> ready[2];
  if (g.b_scale_rows == 1)
    return launch_cluster(fp8_tile::gemm_kernel<kSwap, TM, true, STAGES, KSUB>, ready[1], dev,
                          fp8_tile::Smem<kSwap, TM, true, STAGES, KSUB>::kDynamicBytes, grid, fp8_tile::kThreads, splits,
                          stream, ta, tb, p);
  return launch_cluster(fp8_tile::gemm_kernel<kSwap, TM, false, STAGES, KSUB>, ready[0], dev,
                        fp8_tile::Smem<kSwap, TM, false, STAGES, KSUB>::kDynamicBytes, grid, fp8_tile::kThreads, splits,
                        stream, ta, tb, p);
}

cudaError_t pair_fp8(const Fp8GemmParams& g, const Fp8Types& t, const DeviceInfo& dev, cudaStream_t stream) {
  CUtensorMap ta, tb, td{};
  if (!fp8_map(&ta, g.a, g.m, g.k, g.lda, fp8_pair::kHalf) || !fp8_map(&tb, g.b, g.n, g.k, g.ldb, fp8_pair::kHalf))
    return cudaErrorInvalidValue;
  Fp8PairParams p{};
  p.m = static_cast<int>(g.m), p.n = static_cast<int>(g.n);
  p.num_kb = static_cast<int>(div_up(g.k, fp8::kBlockK));
  p.tiles_m = static_cast<int>(div_up(g.m, fp8_pair::kBlock)), p.tiles_n = static_cast<int>(div_up(g.n, fp8_pair::kBlock));
  if (static_cast<int64_t>(p.tiles_m) * p.tiles_n > INT_MAX - 1024) return cudaErrorInvalidValue;
  p.total_tiles = p.tiles_m * p.tiles_n;
  p.group_m = std::min(p.tiles_m, 16);
  p.a_scale = g.a_scale, p.a_scale_row = g.a_scale_row, p.a_scale_blk = g.a_scale_blk;
  p.b_scale = g.b_scale, p.b_scale_row = g.b_scale_row, p.b_scale_blk = g.b_scale_blk;
  p.d = g.d, p.ldd = g.ldd, p.d_type = t.d;
  const CUtensorMapDataType type = t.d == ZCUTLASS_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : t.d == ZCUTLASS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  p.tma_d = aligned(g.d, 16) && g.ldd * t.d_bytes() % 16 == 0 &&
            make_tma_2d(&td, g.d, type, t.d_bytes(), g.m, g.n, g.ldd, 32, 64 / t.d_bytes(), TmaSwizzle::B64);
  p.bias = g.bias;
  p.idesc = fp8::idesc(fp8_pair::kBlock, fp8_pair::kBlock, t.a5, t.b5);
  p.error_word = dev.error_word;
  const int64_t grid = 2 * std::min<int64_t>(p.total_tiles, dev.sm_count / 2);
  static std::atomic<uint64_t> ready[2];
  if (g.b_scale_rows == 1)
    return launch_cluster(fp8_pair::gemm_kernel<true>, ready[1], dev, fp8_pair::Smem<true>::kDynamicBytes, grid,
                          fp8_pair::kThreads, 2, stream,
                          ta, tb, td, p);
  return launch_cluster(fp8_pair::gemm_kernel<false>, ready[0], dev, fp8_pair::Smem<false>::kDynamicBytes, grid,
                        fp8_pair::kThreads, 2, stream,
                        ta, tb, td, p);
}

// ZCUTLASS_FORCE_KERNEL=fp8_generic | fp8_tile<rows> | fp8_pair pins the kernel of the 8-bit product
// (tests); other values concern the 16-bit GEMM alone.
bool forced(const char* kernel) {
  const char* f = std::getenv("ZCUTLASS_FORCE_KERNEL");
  return f != nullptr && std::strcmp(f, kernel) == 0;
}
bool any_forced() {
  const char* f = std::getenv("ZCUTLASS_FORCE_KERNEL");
  return f != nullptr && std::strncmp(f, "fp8_", 4) == 0;
}

// Clusters of `size` CTAs of the 128 x 128 tile kernel (one CTA per SM) that run at once: clusters stay within
// a GPC, so 148 SMs hold 74, 45, 33, 26, 22, 15 and 15 of 2 to 8. Asked once per device and size.
int resident_clusters(const DeviceInfo& dev, int size) {
  if (size == 1) return dev.sm_count;
  static std::atomic<int> known[64][fp8_tile::kMaxSplits + 1];
  std::atomic<int>& slot = known[dev.ordinal & 63][size];
  int n = slot.load(std::memory_order_relaxed);
  if (n > 0) return n;
  auto kernel = fp8_tile::gemm_kernel<false, 128, false, 3, 2>;
  constexpr int kBytes = fp8_tile::Smem<false, 128, false, 3, 2>::kDynamicBytes;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(size), 1, 1);
  cfg.blockDim = dim3(fp8_tile::kThreads, 1, 1);
  cfg.dynamicSmemBytes = kBytes;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(size);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
    (void)cudaGetLastError();
    n = dev.sm_count / (2 * size);
  }
  slot.store(n, std::memory_order_relaxed);
  return n;
}

// CTAs along K per tile, each with at least two blocks, at most a cluster of 8. The swapped kernel, two CTAs
// of which fit an SM: the power of two that gives (nearly) every SM one, since more only add partial tiles to
// exchange, and clusters of other sizes leave SMs out: 16 x 4096 x 4096 (32 tiles) takes 8.3, 6.5 and 7.6 us
// with 2, 4 and 8 splits, 1 x 6144 x 4096 (48 tiles) 8.6, 8.4, 7.4, 8.5 and 12.1 with 2, 3, 4, 5 and 6. Where a
// short K ends below the next power of two, all that it gives (3, 5 or 6) while that is no more than about 60
// CTAs: 1 x 256 x 1536 (2 tiles) takes 3.5 us with 4 splits and 3.1 with 6, 1 x 1536 x 1280 (12 tiles) 3.8 with 4
// and 3.7 with 5, but 1 x 2048 x 1536 (16 tiles) 3.9 with 4 and 4.1 with 6, 1 x 1024 x 1792 4.0 with 4, 4.2 with 7.
// 32 and 64 rows get a ring that fills the SM where that is a CTA each (see tensor_fp8): then no more clusters than
// run at once (32 x 2048 x 4096, 16 tiles: 10.1 us with 8 splits, 15 of whose clusters fit, 6.0 with 4; 64 rows
// 12.4 and 7.2). ZCUTLASS_SPLITK=<s> fixes the count, as it does for the 16-bit split-K kernels.
// The other kernel, one CTA of which fills an SM: as many as run at once (200 x 1024 x 4096, 16 tiles: 13.3 us with 8
// splits in two waves).
int tile_splits(int64_t tiles, int64_t num_kb, const DeviceInfo& dev, bool swap, bool two_per_sm) {
  const char* v = std::getenv("ZCUTLASS_SPLITK");
  const int most = static_cast<int>(std::min<int64_t>(fp8_tile::kMaxSplits, num_kb / 2));
  int s = 1;
  if (v != nullptr && v[0] != '\0') {
    s = std::atoi(v);
  } else if (swap) {
    while (2 * s <= most && s * tiles < dev.sm_count * 6 / 7) s *= 2;
    if (2 * s > most && most < 7 && most * tiles <= dev.sm_count * 3 / 7) s = most;
    if (!two_per_sm) {
      while (s > 1 && s * tiles <= dev.sm_count * 7 / 8 && tiles > resident_clusters(dev, s)) s /= 2;
    }
  } else {
    for (s = most; s > 1 && tiles > resident_clusters(dev, s); --s) {}
  }
  return std::max(1, std::min(s, most));
}

cudaError_t tensor_fp8(const Fp8GemmParams& g, const Fp8Types& t, const DeviceInfo& dev, cudaStream_t stream) {
  const int64_t tiles_n = div_up(g.n, 128), kb = div_up(g.k, fp8::kBlockK), sms = dev.sm_count;
  const bool any = any_forced();
  const auto splits = [&](int tm) { return tile_splits(tiles_n * div_up(g.m, tm), kb, dev, tm < 128, tm == 16); };
  // Where there is no more than a CTA per SM, one with two blocks per stage and the SM's whole shared memory
  // streams faster than one made for two per SM (48 x 4096 x 14336: 15.6 against 17.1 us; with 224 CTAs,
  // 64 x 28672 x 4096, 30.8 against 23.2). 16 rows are served by the same ring both ways.
  const auto alone = [&](int s) { return tiles_n * s <= sms * 7 / 8; };
  if (any ? forced("fp8_tile16") : g.m <= 16) return tile_fp8<true, 16, 3, 2>(g, t, dev, splits(16), stream);
  if (any ? forced("fp8_tile32") : g.m <= 32) {
    const int s = splits(32);
    return alone(s) ? tile_fp8<true, 32, 4, 2>(g, t, dev, s, stream) : tile_fp8<true, 32, 5, 1>(g, t, dev, s, stream);
  }
  if (any ? forced("fp8_tile64") : g.m <= 64) {
    const int s = splits(64);
    return alone(s) ? tile_fp8<true, 64, 4, 2>(g, t, dev, s, stream) : tile_fp8<true, 64, 4, 1>(g, t, dev, s, stream);
  }
  // Above that, whichever takes fewer waves of tiles: a wave takes about as long with 128 x 128 tiles on
  // every SM as with 256 x 256 tiles on every pair (18.3 and 18.5 us at K = 4096), and one wave of the former
  // can be shortened by splitting K.
  const int64_t waves = div_up(tiles_n * div_up(g.m, 128), sms);
  const int64_t pair_waves = div_up(div_up(g.m, 256) * div_up(g.n, 256), sms / 2);
  if (any ? forced("fp8_pair") : waves > 1 && pair_waves <= waves) return pair_fp8(g, t, dev, stream);
  return tile_fp8<false, 128, 3, 2>(g, t, dev, splits(128), stream);
}

template <typename T, int V>
cudaError_t rotary_v(RotaryParams p, bool interleaved, cudaStream_t stream, int sms) {
  using namespace rotary;
  const int per_item = interleaved ? std::max(V / 2, 1) : V;
  p.items = p.rotary_dim / 2 / per_item + (p.head_dim - p.rotary_dim) / V;
  const int heads = p.x[0].heads + p.x[1].heads;
  // Threads per token: one per item and head lane. A thread that walks over several heads reuses its
  // cosines and sines and keeps more loads in flight; but first every SM gets four blocks.
  p.head_lanes = heads;
  while (p.head_lanes > 1 && div_up(heads, p.head_lanes) < 4 && p.tokens * p.items * p.head_lanes > 8ll * sms * kThreads)
    p.head_lanes = (p.head_lanes + 1) / 2;
  const int64_t threads = p.tokens * p.items * p.head_lanes;
  p.small = threads < INT_MAX - kThreads;
  const int64_t blocks = div_up(threads, kThreads);
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
  if (d.k > 0 && aligned(a, 16) && aligned(b, 16) && d.lda % 16 == 0 && d.ldb % 16 == 0 && !forced("fp8_generic"))
    return tensor_fp8(p, {a5, b5, d.d_type}, *info, stream);
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
  p.error_word = info->data_word;
  const cudaStream_t stream = static_cast<cudaStream_t>(d.stream);
  const bool inter = d.interleaved != 0;
  if (d.dtype == ZCUTLASS_F16) return rotary_t<half>(p, inter, stream, info->sm_count);
  if (d.dtype == ZCUTLASS_BF16) return rotary_t<__nv_bfloat16>(p, inter, stream, info->sm_count);
  return rotary_t<float>(p, inter, stream, info->sm_count);
}

}  // namespace zcb
