// Element types of the operators over sequences of windows (BNN_T_F32 / F16 / BF16, include/bnneon_cuda.h): loads to
// fp32 and the one rounding back; launches that overlap the one before.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace bnn {

template <int T> struct Elem;
template <> struct Elem<0> {
  using type = float;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Elem<1> {
  using type = __half;
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <> struct Elem<2> {
  using type = __nv_bfloat16;
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <int T> using elem_t = typename Elem<T>::type;

// two consecutive 16-bit values of a word, as fp32, and back (low half first)
template <int T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (T == 1) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
  else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w));
}
template <int T>
__device__ __forceinline__ uint32_t pack2f(float a, float b) {
  if constexpr (T == 1) { const __half2 v = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&v); }
  else { const __nv_bfloat162 v = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t *>(&v); }
}

// 8 consecutive elements by 16-byte accesses on 16-byte aligned addresses; stores of one element too (V = 1)
template <int T, int V>
__device__ __forceinline__ void load_elems(const elem_t<T> *p, float (&v)[V]) {
  static_assert(V == 8, "8 elements");
  if constexpr (T == 0) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 w = *reinterpret_cast<const uint4 *>(p);
    const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y), c = unpack2<T>(w.z), d = unpack2<T>(w.w);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
  }
}
template <int T, int V>
__device__ __forceinline__ void store_elems(elem_t<T> *p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = Elem<T>::put(v[0]);
  } else if constexpr (T == 0) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack2f<T>(v[0], v[1]), pack2f<T>(v[2], v[3]), pack2f<T>(v[4], v[5]),
                                               pack2f<T>(v[6], v[7]));
  }
}

// Programmatic dependent launch: the next launch on the stream may start (once every CTA has come here, and as SMs have
// room), and where the other side waits for this whole launch and its writes
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// the launch before it has ended, its writes are visible
__device__ __forceinline__ void wait_launch_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// a launch that may start before the one before it has ended
template <typename... Args>
cudaError_t launch_early(void (*kernel)(Args...), dim3 grid, int threads, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = at;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, args...);
}

}  // namespace bnn
