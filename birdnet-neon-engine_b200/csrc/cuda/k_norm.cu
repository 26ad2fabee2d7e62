// The norms before and after a block, fused with its gate and residual scale (bnn_norm_gate):
//
//   u = norm(f) wpost + bpost,  x' = x + alpha gamma act(g) u,  h = norm(x') wpre + bpre
//
// norm(v) = v / sqrt(mean v^2 + eps), or with the mean taken out first (layer). One pass: a row's f, g and x are read
// once into registers, both norms' statistics are fp32 sums over the registers (the mean before the squares, so that
// nothing cancels), h is formed from x' before x' is rounded for its store. A row whose live byte is 0 keeps x and
// gets h = 0 whatever its f and g hold (they are not read).
//
// Bound by memory: f, g, x in, x', h out.
#include <cuda_runtime.h>

#include "bnn_kernels.h"
#include "seq.cuh"
#include "tc.cuh"

namespace bnn {
namespace {

constexpr int kNormThreads = 256;

struct NormArgs {
  int rows, D;
  const void *x, *f, *g;
  long long xs, fs, gs;
  const float *wpost, *bpost, *gamma, *wpre, *bpre;
  const uint8_t *live;
  void *xo, *h;
  long long xos, hs;
  float eps, alpha;
  int layer, gate;
};

__device__ __forceinline__ float gate_of(int gate, float g) {
  if (gate == 0) return 1.f;
  const float s = __fdividef(1.f, 1.f + __expf(-g));
  return gate == 1 ? s : g * s;
}

// the sum of v over the W warps of a row (W a power of two; W > 1: through shared memory, every warp of the block at
// the same call), in an order that does not depend on timing
template <int W>
__device__ __forceinline__ float row_sum(float v, float *red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (W > 1) {
    const int warp = threadIdx.x / 32;
    __syncthreads();  // the sums of the call before have been read
    if (threadIdx.x % 32 == 0) red[warp] = v;
    __syncthreads();
    v = 0.f;
    const int w0 = warp / W * W;
#pragma unroll
    for (int w = 0; w < W; w++) v += red[w0 + w];
  }
  return v;
}

template <int V>
__device__ __forceinline__ void load_vec(const float *p, float (&v)[V]) { load_elems<0, V>(p, v); }

// W warps a row, each thread NV groups of V consecutive elements: D <= 32 W NV V
template <int XT, int FT, int V, int NV, int W>
__global__ void __launch_bounds__(kNormThreads) k_norm_gate(const NormArgs a) {
  __shared__ float red[kNormThreads / 32];
  constexpr int R = kNormThreads / (32 * W);
  const int lane = threadIdx.x % (32 * W), sub = threadIdx.x / (32 * W), D = a.D;
  const float inv = 1.f / (float)D;
  for (long long r0 = (long long)blockIdx.x * R; r0 < a.rows; r0 += (long long)gridDim.x * R) {
    const long long r = r0 + sub;
    const bool in = r < a.rows, live = in && (!a.live || a.live[r]);
    const elem_t<XT> *x = (const elem_t<XT> *)a.x + r * a.xs;
    float y[NV][V];
    if (a.f) {
      const elem_t<FT> *f = (const elem_t<FT> *)a.f + r * a.fs, *g = (const elem_t<FT> *)a.g + r * a.gs;
      float u[NV][V], gg[NV][V];
#pragma unroll
      for (int k = 0; k < NV; k++) {
        const int c = (k * 32 * W + lane) * V;
#pragma unroll
        for (int j = 0; j < V; j++) u[k][j] = 0.f, gg[k][j] = 0.f, y[k][j] = 0.f;
        if (c < D && in) {
          load_elems<XT, V>(x + c, y[k]);
          if (live) {
            load_elems<FT, V>(f + c, u[k]);
            if (a.gate) load_elems<FT, V>(g + c, gg[k]);
          }
        }
      }
      float mean = 0.f, ss = 0.f;
      if (a.layer) {
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
          for (int j = 0; j < V; j++) mean += u[k][j];
        mean = row_sum<W>(mean, red) * inv;
      }
#pragma unroll
      for (int k = 0; k < NV; k++) {
        if ((k * 32 * W + lane) * V >= D) continue;
#pragma unroll
        for (int j = 0; j < V; j++) ss += (u[k][j] - mean) * (u[k][j] - mean);
      }
      const float rs = rsqrtf(row_sum<W>(ss, red) * inv + a.eps);
#pragma unroll
      for (int k = 0; k < NV; k++) {
        const int c = (k * 32 * W + lane) * V;
        if (c < D && live) {
          float w[V];
          if (a.wpost) load_vec<V>(a.wpost + c, w);
#pragma unroll
          for (int j = 0; j < V; j++) u[k][j] = (u[k][j] - mean) * rs * (a.wpost ? w[j] : 1.f);
          if (a.bpost) {
            load_vec<V>(a.bpost + c, w);
#pragma unroll
            for (int j = 0; j < V; j++) u[k][j] += w[j];
          }
          if (a.gamma) load_vec<V>(a.gamma + c, w);
#pragma unroll
          for (int j = 0; j < V; j++)
            y[k][j] += a.alpha * (a.gamma ? w[j] : 1.f) * (gate_of(a.gate, gg[k][j]) * u[k][j]);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < NV; k++) {
        const int c = (k * 32 * W + lane) * V;
#pragma unroll
        for (int j = 0; j < V; j++) y[k][j] = 0.f;
        if (c < D && in) load_elems<XT, V>(x + c, y[k]);
      }
    }
    if (a.xo && in) {
      elem_t<XT> *xo = (elem_t<XT> *)a.xo + r * a.xos;
#pragma unroll
      for (int k = 0; k < NV; k++) {
        const int c = (k * 32 * W + lane) * V;
        if (c < D) store_elems<XT, V>(xo + c, y[k]);
      }
    }
    if (!a.h) continue;
    float mean = 0.f, ss = 0.f;
    if (a.layer) {
#pragma unroll
      for (int k = 0; k < NV; k++)
#pragma unroll
        for (int j = 0; j < V; j++) mean += y[k][j];
      mean = row_sum<W>(mean, red) * inv;
    }
#pragma unroll
    for (int k = 0; k < NV; k++) {
      if ((k * 32 * W + lane) * V >= D) continue;
#pragma unroll
      for (int j = 0; j < V; j++) ss += (y[k][j] - mean) * (y[k][j] - mean);
    }
    const float rs = rsqrtf(row_sum<W>(ss, red) * inv + a.eps);
    if (!in) continue;
    elem_t<FT> *h = (elem_t<FT> *)a.h + r * a.hs;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const int c = (k * 32 * W + lane) * V;
      if (c >= D) continue;
      float w[V], b[V], o[V];
      if (a.wpre) load_vec<V>(a.wpre + c, w);
      if (a.bpre) load_vec<V>(a.bpre + c, b);
#pragma unroll
      for (int j = 0; j < V; j++) {
        o[j] = (y[k][j] - mean) * rs * (a.wpre ? w[j] : 1.f);
        if (a.bpre) o[j] += b[j];
        if (!live) o[j] = 0.f;
      }
      store_elems<FT, V>(h + c, o);
    }
  }
}

// Rows wider than the registers of a block hold: one block a row, each element formed again from f, g and x for every
// sum (the rows stay in L1 / L2), stored in the last pass, which reads an element's inputs before it writes there.
template <int XT, int FT>
__global__ void __launch_bounds__(kNormThreads) k_norm_gate_wide(const NormArgs a) {
  __shared__ float red[kNormThreads / 32];
  const int D = a.D;
  const float inv = 1.f / (float)D;
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const bool live = !a.live || a.live[r], upd = live && a.f;
    const elem_t<XT> *x = (const elem_t<XT> *)a.x + r * a.xs;
    const elem_t<FT> *f = (const elem_t<FT> *)a.f + r * a.fs, *g = (const elem_t<FT> *)a.g + r * a.gs;
    float fm = 0.f, frs = 0.f;
    if (upd) {
      float s = 0.f;
      if (a.layer) {
        for (int c = threadIdx.x; c < D; c += kNormThreads) s += Elem<FT>::get(f[c]);
        fm = row_sum<kNormThreads / 32>(s, red) * inv;
      }
      s = 0.f;
      for (int c = threadIdx.x; c < D; c += kNormThreads) {
        const float v = Elem<FT>::get(f[c]) - fm;
        s += v * v;
      }
      frs = rsqrtf(row_sum<kNormThreads / 32>(s, red) * inv + a.eps);
    }
    auto y_at = [&](int c) {
      float y = Elem<XT>::get(x[c]);
      if (upd) {
        float u = (Elem<FT>::get(f[c]) - fm) * frs * (a.wpost ? a.wpost[c] : 1.f);
        if (a.bpost) u += a.bpost[c];
        y += a.alpha * (a.gamma ? a.gamma[c] : 1.f) * (gate_of(a.gate, a.gate ? Elem<FT>::get(g[c]) : 0.f) * u);
      }
      return y;
    };
    float mean = 0.f, rs = 0.f;
    if (a.h && live) {
      float s = 0.f;
      if (a.layer) {
        for (int c = threadIdx.x; c < D; c += kNormThreads) s += y_at(c);
        mean = row_sum<kNormThreads / 32>(s, red) * inv;
      }
      s = 0.f;
      for (int c = threadIdx.x; c < D; c += kNormThreads) {
        const float v = y_at(c) - mean;
        s += v * v;
      }
      rs = rsqrtf(row_sum<kNormThreads / 32>(s, red) * inv + a.eps);
    }
    for (int c = threadIdx.x; c < D; c += kNormThreads) {
      const float y = y_at(c);
      if (a.xo) ((elem_t<XT> *)a.xo)[r * a.xos + c] = Elem<XT>::put(y);
      if (a.h) {
        float o = (y - mean) * rs * (a.wpre ? a.wpre[c] : 1.f);
        if (a.bpre) o += a.bpre[c];
        ((elem_t<FT> *)a.h)[r * a.hs + c] = Elem<FT>::put(live ? o : 0.f);
      }
    }
  }
}

template <int XT, int FT, int V, int NV, int W>
cudaError_t launch_w(const NormArgs &a, cudaStream_t st) {
  constexpr int R = kNormThreads / (32 * W);
  const long long blocks = (a.rows + (long long)R - 1) / R, most = 8LL * num_sms();
  k_norm_gate<XT, FT, V, NV, W><<<(int)(blocks < most ? blocks : most), kNormThreads, 0, st>>>(a);
  return cudaGetLastError();
}

template <int XT, int FT>
cudaError_t launch_norm(const NormArgs &a, bool vec, cudaStream_t st) {
  const int units = vec ? a.D / 8 : a.D;
  // few rows: a row over as many warps as give each thread one group; many: as few warps as hold the row
  const bool few = a.rows < 8 * num_sms();
  if (vec) {
    if (few || units > 256) {
      if (units <= 32) return launch_w<XT, FT, 8, 1, 1>(a, st);
      if (units <= 128) return launch_w<XT, FT, 8, 1, 4>(a, st);
      if (units <= 256) return launch_w<XT, FT, 8, 1, 8>(a, st);
      if (units <= 1024) return launch_w<XT, FT, 8, 4, 8>(a, st);
    } else {
      if (units <= 32) return launch_w<XT, FT, 8, 1, 1>(a, st);
      if (units <= 128) return launch_w<XT, FT, 8, 4, 1>(a, st);
      return launch_w<XT, FT, 8, 8, 1>(a, st);
    }
  } else {
    if (units <= 256) return launch_w<XT, FT, 1, 8, 1>(a, st);
    if (units <= 1024) return few ? launch_w<XT, FT, 1, 4, 8>(a, st) : launch_w<XT, FT, 1, 32, 1>(a, st);
    if (units <= 2048) return launch_w<XT, FT, 1, 8, 8>(a, st);
  }
  const long long most = 8LL * num_sms();
  k_norm_gate_wide<XT, FT><<<(int)(a.rows < most ? a.rows : most), kNormThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace bnn

using namespace bnn;

extern "C" int bnnk_norm_gate(const bnnk_norm_gate_args *p, bnn_stream_t st) {
  if (p->rows <= 0) return 0;
  NormArgs a = {p->rows, p->D, p->x, p->f, p->g, p->xs, p->fs, p->gs, p->wpost, p->bpost, p->gamma, p->wpre, p->bpre,
                p->live, p->xo, p->h, p->xos, p->hs, p->eps, p->alpha, p->layer, p->f ? p->gate : 0};
  // 8 elements an access: whole groups, and every row and vector on 16 bytes
  const uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.f | (uintptr_t)a.g | (uintptr_t)a.xo | (uintptr_t)a.h |
                       (uintptr_t)a.wpost | (uintptr_t)a.bpost | (uintptr_t)a.gamma | (uintptr_t)a.wpre |
                       (uintptr_t)a.bpre;
  const bool vec = a.D % 8 == 0 && !(at & 15) &&
                   !((a.xs | (a.f ? a.fs : 0) | (a.f && a.gate ? a.gs : 0) | (a.xo ? a.xos : 0) | (a.h ? a.hs : 0)) & 7);
  const cudaStream_t s = (cudaStream_t)st;
  if (p->xtype == 0 && p->type == 0) return launch_norm<0, 0>(a, vec, s);
  if (p->xtype == 0 && p->type == 1) return launch_norm<0, 1>(a, vec, s);
  if (p->xtype == 0 && p->type == 2) return launch_norm<0, 2>(a, vec, s);
  if (p->xtype == 1 && p->type == 1) return launch_norm<1, 1>(a, vec, s);
  if (p->xtype == 2 && p->type == 2) return launch_norm<2, 2>(a, vec, s);
  return cudaErrorInvalidValue;
}
