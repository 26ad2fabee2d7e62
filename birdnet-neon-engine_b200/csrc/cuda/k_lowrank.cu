// A projection shared by all rows beside low-rank adapters, one of many for each row (bnn_lowrank):
//
//   y_r = W x_r + bias + s_a B_a (A_a x_r),   a = slot[r] (none where it is outside [0, slots))
//
// W [N][K], A [slots][rank][K], B [slots][N][rank]; sums in fp32.
#include <cuda_runtime.h>

#include "bnn_kernels.h"
#include "seq.cuh"
#include "tc.cuh"

namespace bnn {
namespace {

// s_a A_a x_r: a warp a (row, rank index), hid [rows][rank]
template <int T>
__global__ void __launch_bounds__(256) k_lowrank_down(int rows, int K, const elem_t<T> *x, long long ldx,
                                                      const int32_t *slot, int slots, int rank, const elem_t<T> *A,
                                                      const float *scale, float *hid) {
  const long long u = (long long)blockIdx.x * 8 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (u >= (long long)rows * rank) return;
  const long long r = u / rank;
  const int j = (int)(u % rank), s = slot[r];
  float sum = 0.f;
  if (s >= 0 && s < slots) {
    const elem_t<T> *w = A + ((long long)s * rank + j) * K;
    for (int k = lane * 8; k < K; k += 256) {
      float xv[8], wv[8];
      load_elems<T, 8>(x + r * ldx + k, xv);
      load_elems<T, 8>(w + k, wv);
#pragma unroll
      for (int e = 0; e < 8; e++) sum = fmaf(xv[e], wv[e], sum);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    sum *= scale ? scale[s] : 1.f;
  }
  if (lane == 0) hid[u] = sum;
}

// y: a 64 x 64 tile a CTA, 4 x 4 outputs a thread, K in steps of 16 through shared memory
template <int T, int OT>
__global__ void __launch_bounds__(256) k_lowrank_up(int rows, int N, int K, const elem_t<T> *x, long long ldx,
                                                    const elem_t<T> *W, long long ldw, const float *bias,
                                                    const int32_t *slot, int slots, int rank, const elem_t<T> *B,
                                                    const float *hid, elem_t<OT> *y, long long ldy) {
  __shared__ float xs[16][65], ws[16][65];
  const long long r0 = (long long)blockIdx.y * 64;
  const int n0 = blockIdx.x * 64, tr = threadIdx.x / 16, tn = threadIdx.x % 16;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += 16) {
    for (int e = threadIdx.x; e < 1024; e += 256) {
      const int m = e / 16, k = e % 16;
      xs[k][m] = r0 + m < rows && k0 + k < K ? Elem<T>::get(x[(r0 + m) * ldx + k0 + k]) : 0.f;
      ws[k][m] = n0 + m < N && k0 + k < K ? Elem<T>::get(W[(n0 + m) * ldw + k0 + k]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; k++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = fmaf(xs[k][tr + 16 * i], ws[k][tn + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; i++) {
    const long long r = r0 + tr + 16 * i;
    if (r >= rows) continue;
    const int s = slot ? slot[r] : -1;
    for (int j = 0; j < 4; j++) {
      const int n = n0 + tn + 16 * j;
      if (n >= N) continue;
      float v = acc[i][j] + (bias ? bias[n] : 0.f);
      if (s >= 0 && s < slots)
        for (int e = 0; e < rank; e++)
          v = fmaf(hid[r * rank + e], Elem<T>::get(B[((long long)s * N + n) * rank + e]), v);
      y[r * ldy + n] = Elem<OT>::put(v);
    }
  }
}

template <int T>
cudaError_t run_lowrank(const bnnk_lowrank_args &p, cudaStream_t st) {
  using E = elem_t<T>;
  if (p.slot)
    k_lowrank_down<T><<<(int)(((long long)p.rows * p.rank + 7) / 8), 256, 0, st>>>(
        p.rows, p.K, (const E *)p.x, p.ldx, p.slot, p.slots, p.rank, (const E *)p.a, p.scale, p.hid);
  const dim3 grid((p.N + 63) / 64, (p.rows + 63) / 64);
  if (p.otype == 0)
    k_lowrank_up<T, 0><<<grid, 256, 0, st>>>(p.rows, p.N, p.K, (const E *)p.x, p.ldx, (const E *)p.w, p.ldw, p.bias,
                                             p.slot, p.slots, p.rank, (const E *)p.b, p.hid, (float *)p.y, p.ldy);
  else
    k_lowrank_up<T, T><<<grid, 256, 0, st>>>(p.rows, p.N, p.K, (const E *)p.x, p.ldx, (const E *)p.w, p.ldw, p.bias,
                                             p.slot, p.slots, p.rank, (const E *)p.b, p.hid, (E *)p.y, p.ldy);
  return cudaGetLastError();
}

}  // namespace
}  // namespace bnn

using namespace bnn;

extern "C" int bnnk_lowrank(const bnnk_lowrank_args *p, bnn_stream_t st) {
  if (p->rows <= 0) return 0;
  return p->type == 1 ? run_lowrank<1>(*p, (cudaStream_t)st) : run_lowrank<2>(*p, (cudaStream_t)st);
}
