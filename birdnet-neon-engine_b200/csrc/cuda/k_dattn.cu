// Linear attention with a decay for each key / value head (bnn_dattn): per sequence and head
//
//   S_t = lambda S_{t-1} + live_t k_t^T v_t,   o_t = live_t scale q_t S_t
//
// S [dk][dv] fp32, q heads in groups of G that share one k/v head and its S.
#include <cuda_runtime.h>

#include "bnn_kernels.h"
#include "seq.cuh"
#include "tc.cuh"

namespace bnn {
namespace {

struct DattnArgs {
  int n, H, Hk, G, dk, dv;
  long long tokens;
  const int32_t *cu, *slot;
  const uint8_t *live;
  const void *q, *k, *v;
  long long qts, kts, vts;
  const float *s0;
  float *s1;
  void *o;
  long long ots;
  const float *pow;  // [Hk][kDattnPow]: lambda^0 .. lambda^128
  float scale;
};

// a sequence's tokens [t0, t1): cu offsets kept inside the buffers, or token i for sequence i where cu is NULL
__device__ __forceinline__ void seq_range(const DattnArgs &a, int i, long long &t0, long long &t1) {
  if (!a.cu) { t0 = i; t1 = i + 1; return; }
  t0 = min(max((long long)a.cu[i], 0ll), a.tokens);
  t1 = min(max((long long)a.cu[i + 1], t0), a.tokens);
}

// ------------------------------------------------------------------ the recurrent form
//
// One CTA per (32 columns of S, head, sequence): a thread holds a float4 of S in up to 4 rows (row 4 warp + lane / 8
// + 4 warps p), a warp's access is 4 rows of 128 consecutive bytes. Per token the update and, for each q head of the
// group, the partial sums over the thread's rows, joined over the warp's 4 row groups by shuffles and over the warps
// through shared memory, in a fixed order.
// Bound by memory for single tokens: S is read once and written once (at most 8 + 8 KB a CTA).
constexpr int kRecG = 8;  // q heads whose partial sums are in shared memory at once

template <int T>
__global__ void __launch_bounds__(256) k_dattn_rec(const DattnArgs a) {
  __shared__ float part[2][kRecG][8][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
  const int hk = blockIdx.y, i = blockIdx.x, cs = blockIdx.z * 32, c0 = cs + (lane % 8) * 4;
  const int dk = a.dk, dv = a.dv;
  const bool col = c0 < dv;
  const long long slot = a.slot ? a.slot[i] : i;
  float4 S[4];
  int row[4];
  const long long sbase = (slot * a.Hk + hk) * (long long)dk * dv + c0;
#pragma unroll
  for (int p = 0; p < 4; p++) {
    row[p] = 4 * (warp + warps * p) + lane / 8;
    const bool in = row[p] < dk && col;
    S[p] = in && a.s0 && slot >= 0 ? *reinterpret_cast<const float4 *>(a.s0 + sbase + (long long)row[p] * dv)
                                   : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  long long t0, t1;
  seq_range(a, i, t0, t1);
  const float lam = a.pow[hk * kDattnPow + 1];
  int buf = 0;
  for (long long t = t0; t < t1; t++) {
    const bool live = !a.live || a.live[t];
    elem_t<T> *o = (elem_t<T> *)a.o + t * a.ots + (long long)hk * a.G * dv;
    if (!live) {
#pragma unroll
      for (int p = 0; p < 4; p++) { S[p].x *= lam; S[p].y *= lam; S[p].z *= lam; S[p].w *= lam; }
      for (int g = warp; g < a.G; g += warps)
        if (cs + lane < dv) o[(long long)g * dv + cs + lane] = Elem<T>::put(0.f);
      continue;
    }
    const elem_t<T> *k = (const elem_t<T> *)a.k + t * a.kts + (long long)hk * dk;
    const elem_t<T> *v = (const elem_t<T> *)a.v + t * a.vts + (long long)hk * dv + c0;
    const elem_t<T> *q = (const elem_t<T> *)a.q + t * a.qts + (long long)hk * a.G * dk;
    float4 vv = make_float4(0.f, 0.f, 0.f, 0.f);
    if (col) {
      const uint2 w = *reinterpret_cast<const uint2 *>(v);
      const float2 x = unpack2<T>(w.x), y = unpack2<T>(w.y);
      vv = make_float4(x.x, x.y, y.x, y.y);
    }
#pragma unroll
    for (int p = 0; p < 4; p++) {
      const float kk = row[p] < dk ? Elem<T>::get(k[row[p]]) : 0.f;
      S[p].x = fmaf(kk, vv.x, lam * S[p].x);
      S[p].y = fmaf(kk, vv.y, lam * S[p].y);
      S[p].z = fmaf(kk, vv.z, lam * S[p].z);
      S[p].w = fmaf(kk, vv.w, lam * S[p].w);
    }
    for (int g0 = 0; g0 < a.G; g0 += kRecG) {
      const int ng = min(kRecG, a.G - g0);
      for (int g = 0; g < ng; g++) {
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int p = 0; p < 4; p++) {
          if (row[p] >= dk) continue;
          const float qq = Elem<T>::get(q[(long long)(g0 + g) * dk + row[p]]);
          s.x = fmaf(qq, S[p].x, s.x);
          s.y = fmaf(qq, S[p].y, s.y);
          s.z = fmaf(qq, S[p].z, s.z);
          s.w = fmaf(qq, S[p].w, s.w);
        }
#pragma unroll
        for (int m = 8; m < 32; m <<= 1) {
          s.x += __shfl_xor_sync(0xffffffffu, s.x, m);
          s.y += __shfl_xor_sync(0xffffffffu, s.y, m);
          s.z += __shfl_xor_sync(0xffffffffu, s.z, m);
          s.w += __shfl_xor_sync(0xffffffffu, s.w, m);
        }
        if (lane < 8) *reinterpret_cast<float4 *>(&part[buf][g][warp][lane * 4]) = s;
      }
      __syncthreads();  // the buffer of two calls ago is free: every thread has passed the barrier after reading it
      for (int g = warp; g < ng; g += warps) {
        float s = 0.f;
        for (int w = 0; w < warps; w++) s += part[buf][g][w][lane];
        const int c = cs + lane;
        if (c < dv) o[(long long)(g0 + g) * dv + c] = Elem<T>::put(a.scale * s);
      }
      buf ^= 1;
    }
  }
  if (a.s1 && slot >= 0 && col) {
#pragma unroll
    for (int p = 0; p < 4; p++)
      if (row[p] < dk) *reinterpret_cast<float4 *>(a.s1 + sbase + (long long)row[p] * dv) = S[p];
  }
}

}  // namespace
}  // namespace bnn

using namespace bnn;

extern "C" int bnnk_dattn(const bnnk_dattn_args *p, bnn_stream_t st) {
  if (p->n <= 0) return 0;
  DattnArgs a = {p->n, p->H, p->Hk, p->H / p->Hk, p->dk, p->dv, p->tokens, p->cu, p->slot, p->live, p->q, p->k, p->v,
                 p->qts, p->kts, p->vts, p->s0, p->s1, p->o, p->ots, p->pow, p->scale};
  const int warps = (p->dk + 15) / 16;
  const dim3 grid(p->n, p->Hk, (p->dv + 31) / 32);
  if (p->type == 1) k_dattn_rec<1><<<grid, 32 * warps, 0, (cudaStream_t)st>>>(a);
  else k_dattn_rec<2><<<grid, 32 * warps, 0, (cudaStream_t)st>>>(a);
  return cudaGetLastError();
}
