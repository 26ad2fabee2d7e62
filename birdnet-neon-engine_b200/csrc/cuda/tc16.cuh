// tcgen05 kind::f16 building blocks of the operators over sequences (inline PTX): fp16 or bf16 operands (both of a type; a
// kind::tf32 product too),
// fp32 accumulators in TMEM, A from shared memory or TMEM, K-major and MN-major shared-memory tiles, TMEM loads and
// stores. Host side: the descriptor encoder and 3-D maps of [rows][heads][width] tensors.
#pragma once
#include <cuda.h>
#include <stdint.h>

#include "seq.cuh"
#include "tc.cuh"

namespace bnn {

// instruction descriptor of kind::f16: type code t (0 fp16, 1 bf16), fp32 D, M 128, N n (a multiple of 16, <= 256);
// a_mn / b_mn: the operand's tile is MN-major
__host__ __device__ constexpr uint32_t idesc_16(int t, int n, int a_mn, int b_mn) {
  return (1u << 4) | ((uint32_t)t << 7) | ((uint32_t)t << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// the same for kind::tf32, both operands K-major: 32 bytes of a row are its 8 K elements
__host__ __device__ constexpr uint32_t idesc_tf32(int n) {
  return (1u << 4) | (2u << 7) | (2u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// descriptor of an MN-major tile: k rows of 64 elements (128 bytes, 128-byte swizzle), 8-row groups back to back, the
// next 64 elements of the M or N index `panel` bytes on
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr, uint32_t panel) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void mma16_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma32_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
// A from TMEM: lane = row, a 32-bit column = two consecutive K elements
__device__ __forceinline__ void mma16_ts(uint32_t d, uint32_t ta, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(ta), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}

#define BNN_O4(r, i) "=r"((r)[i]), "=r"((r)[(i) + 1]), "=r"((r)[(i) + 2]), "=r"((r)[(i) + 3])
#define BNN_I4(r, i) "r"((r)[i]), "r"((r)[(i) + 1]), "r"((r)[(i) + 2]), "r"((r)[(i) + 3])
#define BNN_P4(r, i) "+r"((r)[i]), "+r"((r)[(i) + 1]), "+r"((r)[(i) + 2]), "+r"((r)[(i) + 3])

// this thread's lane, 16 consecutive 32-bit columns
__device__ __forceinline__ void tmem_ld16(uint32_t t, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : BNN_O4(r, 0), BNN_O4(r, 4), BNN_O4(r, 8), BNN_O4(r, 12)
      : "r"(t));
}
__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(t),
      BNN_I4(r, 0), BNN_I4(r, 4), BNN_I4(r, 8), BNN_I4(r, 12)
      : "memory");
}
// waits for this thread's TMEM loads; the registers they fill are operands, so that no use of them moves above
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : BNN_P4(r, 0), BNN_P4(r, 4), BNN_P4(r, 8), BNN_P4(r, 12)::"memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[16], uint32_t (&q)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : BNN_P4(r, 0), BNN_P4(r, 4), BNN_P4(r, 8), BNN_P4(r, 12), BNN_P4(q, 0), BNN_P4(q, 4), BNN_P4(q, 8),
                 BNN_P4(q, 12)::"memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[8], uint32_t (&q)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : BNN_P4(r, 0), BNN_P4(r, 4), BNN_P4(q, 0), BNN_P4(q, 4)::"memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// this thread's shared-memory writes before it, to the TMA and tensor-core proxies
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

#undef BNN_O4
#undef BNN_I4
#undef BNN_P4

// an fp32 pair as two words of 16-bit pairs whose sum is the pair up to the square of the type's unit roundoff
// (T: 1 fp16, 2 bf16); fp16 only for values scaled into its range
template <int T>
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
  hi = pack2f<T>(a, b);
  const float2 h = unpack2<T>(hi);
  lo = pack2f<T>(a - h.x, b - h.y);
}

// three parts: all of an fp32 value's 24 bits (bf16)
template <int T>
__device__ __forceinline__ void split3(float a, float b, uint32_t &hi, uint32_t &lo, uint32_t &lo2) {
  hi = pack2f<T>(a, b);
  const float2 h = unpack2<T>(hi);
  const float ra = a - h.x, rb = b - h.y;
  lo = pack2f<T>(ra, rb);
  const float2 l = unpack2<T>(lo);
  lo2 = pack2f<T>(ra - l.x, rb - l.y);
}
// one lane of a converged warp, the same for every call
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// host: a 3-D map of a 16-bit tensor [rows][heads][width] (row stride rs elements, heads back to back), boxes of 64
// elements x 1 head x box_rows rows, 128-byte swizzle, zero fill out of bounds: a width that ends inside a box reads
// zero past it, never the next head; 0 or a cudaError_t
int encode_heads(CUtensorMap *m, const void *base, int bf16, int width, int heads, long long rows, long long rs,
                 int box_rows);
// host: a 2-D map of a 16-bit matrix [rows][width] (row stride rs elements), boxes of box_w x box_rows, swizzle sw bytes
int encode_rows16(CUtensorMap *m, const void *base, int bf16, int width, long long rows, long long rs, int box_w,
                  int box_rows, int sw);
// host: a 3-D map of [slots][rows][width] back to back, boxes of box_w x box_rows x 1 slot, swizzle 2 box_w bytes
// (8 wide: none)
int encode_slots16(CUtensorMap *m, const void *base, int bf16, int width, int rows, int slots, int box_w, int box_rows);

}  // namespace bnn
