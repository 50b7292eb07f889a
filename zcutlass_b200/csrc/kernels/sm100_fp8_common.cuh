// Parts the 8-bit tcgen05 kernels share: the kind::f8f6f4 MMA, packed 32-bit
// arithmetic and the scale-and-add that moves one 128-k block's product from
// TMEM into register accumulators.
//
// A scale that changes every 128 k cannot stay inside the tensor core's running
// sum, and general 32-bit scales cannot be given to it. So each block's product
// (4 MMAs of k = 32) goes to a TMEM buffer of its own, and the accumulation
// acc += (sa * sb) * product runs in 32 bits on registers, one TMEM read and one
// packed fma per two values, while the MMAs of the next blocks fill the other
// buffers.
#pragma once

#include "fp8_generic_gemm.cuh"
#include "sm100_ptx.cuh"

namespace zcb {
namespace fp8 {

constexpr int kBlockK = 128;  // bytes: one swizzled shared-memory row, one scale
constexpr int kMmaK = 32;

// Instruction descriptor for kind::f8f6f4 with an f32 accumulator, K-major
// operands: bits 4-5 D format (1 = f32), 7-9 A and 10-12 B format (0 e4m3,
// 1 e5m2), 17-22 N>>3, 24-28 M>>4.
__host__ __device__ constexpr uint32_t idesc(int m, int n, bool a_e5m2, bool b_e5m2) {
  return (1u << 4) | ((a_e5m2 ? 1u : 0u) << 7) | ((b_e5m2 ? 1u : 0u) << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      " .reg .pred p;\n"
      " setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void mma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n"
      " .reg .pred p;\n"
      " setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// 16 rows x 8 columns of 32 bits per 4 registers: registers 4 g, 4 g + 1 hold columns 8 g + (lane % 4) * 2
// and the next of row lane / 4, registers 4 g + 2, 4 g + 3 the same of row lane / 4 + 8.
__device__ __forceinline__ void tmem_ld_16x256b_x4(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// Waits for the thread's TMEM loads; the registers pass through so that no use of them moves above the wait.
__device__ __forceinline__ void tmem_ld_wait_x16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// mbar_wait for waits that come once per k block: the timer that bounds it is first read after 64 tries,
// since the read itself takes longer than such a wait.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, const WaitCtx& ctx, int code) {
  const uint32_t addr = smem_addr(bar);
#pragma unroll 1
  for (int i = 0; i < 64; ++i)
    if (mbar_try_wait(addr, parity)) return true;
  return mbar_wait(bar, parity, ctx, code);
}

// True in one lane of the (converged) warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(r));
  return r != 0;
}

// Hands a TMEM buffer back to the CTA of the pair that issues the MMAs: an arrival on its mbarrier at
// `cluster_addr`, and the wait for such arrivals. tcgen05.fence before the one and after the other orders the
// TMEM accesses, so both may be relaxed, but their scope is the cluster. Nothing in memory may be handed over
// with them. (A release at cluster scope waits for every access in flight: 1810 us against 1233 when the
// arriving warps still fetched the scales themselves.)
__device__ __forceinline__ void arrive_read(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool try_wait_read(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n"
      " .reg .pred p;\n"
      " mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ bool wait_read(uint64_t* bar, uint32_t parity, const WaitCtx& ctx, int code) {
  const uint32_t addr = smem_addr(bar);
#pragma unroll 1
  for (int i = 0; i < 64; ++i)
    if (try_wait_read(addr, parity)) return true;
  // The bounded wait, then the wait at the scope that counts (the phase stays complete until it is used).
  return mbar_wait(bar, parity, ctx, code) && try_wait_read(addr, parity);
}

// Packed 32-bit arithmetic: two values per instruction. The accumulation with row scales needs a product and
// an fma per value; packed, it takes half the issue slots (4 % of the whole product at 8192 x 28672 x 4096).
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// Registers of a load that has been waited for: no use of them moves above this point.
template <int N>
__device__ __forceinline__ void after_wait(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}

// acc += scale() * (128 columns of this thread's TMEM lane at t0); `read_done` is called when the last column has
// been read. Two loads of 32 columns are in flight at a time: eight of 16, one ahead, held the buffer 3 % of a
// product longer.
template <typename Scale, typename ReadDone>
__device__ __forceinline__ void add_columns(float (&acc)[128], uint32_t t0, Scale scale, ReadDone read_done) {
  uint32_t a[32], b[32];
  tmem_ld_32x32b_x32(t0, a);
  tmem_ld_32x32b_x32(t0 + 32, b);
  const float s = scale();  // from shared memory while the loads are on their way
  tmem_ld_wait();
  after_wait(a);
  after_wait(b);
#pragma unroll
  for (int j = 0; j < 32; ++j) acc[j] = fmaf(s, __uint_as_float(a[j]), acc[j]);
  tmem_ld_32x32b_x32(t0 + 64, a);
#pragma unroll
  for (int j = 0; j < 32; ++j) acc[32 + j] = fmaf(s, __uint_as_float(b[j]), acc[32 + j]);
  tmem_ld_32x32b_x32(t0 + 96, b);
  tmem_ld_wait();
  after_wait(a);
  after_wait(b);
  read_done();
#pragma unroll
  for (int j = 0; j < 32; ++j) acc[64 + j] = fmaf(s, __uint_as_float(a[j]), acc[64 + j]);
#pragma unroll
  for (int j = 0; j < 32; ++j) acc[96 + j] = fmaf(s, __uint_as_float(b[j]), acc[96 + j]);
}

// The four pairs of column scales that a thread meets in 32 columns, from `sb` (its pair of the first group).
__device__ __forceinline__ void load_column_scales(float2 (&s)[4], const float2* sb) {
#pragma unroll
  for (int g = 0; g < 4; ++g) s[g] = sb[g * 4];
}

// acc += (s * scale) * r for one 16 x 32 step of fragments: column scales s, row scales lo and hi of the
// fragment's two rows.
__device__ __forceinline__ void add_fragments(float* acc, const uint32_t (&r)[16], const float2 (&s)[4], float lo, float hi) {
  const uint64_t lo2 = pack2(lo, lo), hi2 = pack2(hi, hi);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const uint64_t s2 = pack2(s[g].x, s[g].y);
    float* q = acc + 4 * g;
    const float2 a = unpack2(fma2(mul2(s2, lo2), pack2(__uint_as_float(r[4 * g]), __uint_as_float(r[4 * g + 1])), pack2(q[0], q[1])));
    const float2 b = unpack2(fma2(mul2(s2, hi2), pack2(__uint_as_float(r[4 * g + 2]), __uint_as_float(r[4 * g + 3])), pack2(q[2], q[3])));
    q[0] = a.x, q[1] = a.y, q[2] = b.x, q[3] = b.y;
  }
}

__device__ __forceinline__ void cluster_sync_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n"
               "barrier.cluster.wait.aligned;" ::: "memory");
}

// Brings a box to L2.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int32_t c0, int32_t c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1)
               : "memory");
}

// Four floats at a shared-memory offset of another CTA of the cluster.
__device__ __forceinline__ float4 ld_dsmem_v4f(uint32_t local_addr, uint32_t rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(map_shared_rank(local_addr, rank))
               : "memory");
  return v;
}

// Output element types by their zcutlass_dtype value.
enum : int { kF16 = 0, kBf16 = 1, kF32 = 2 };

__device__ __forceinline__ float load_out(const void* p, int64_t i, int type) {
  if (type == kF32) return static_cast<const float*>(p)[i];
  if (type == kBf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const half*>(p)[i]);
}
__device__ __forceinline__ void store_out(void* p, int64_t i, int type, float v) {
  if (type == kF32) static_cast<float*>(p)[i] = v;
  else if (type == kBf16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<half*>(p)[i] = __float2half_rn(v);
}
__device__ __forceinline__ uint32_t pack_out(float lo, float hi, int type) {
  return type == kBf16 ? Elem<__nv_bfloat16>::pack(lo, hi) : Elem<half>::pack(lo, hi);
}

}  // namespace fp8
}  // namespace zcb
