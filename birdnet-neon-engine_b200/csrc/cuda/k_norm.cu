// The norms before and after a block, fused with its gate and residual scale (bnn_norm_gate):
//
//   u = norm(f) wpost + bpost,  x' = x + alpha gamma act(g) u,  h = norm(x') wpre + bpre
//
// norm(v) = v / sqrt(mean v^2 + eps), or with the mean taken out first (layer). One pass: a row's f, g and x are read
// once into registers, both norms' statistics are fp32 sums over the registers (the mean before the squares, so that
// nothing cancels), h is formed from x' before x' is rounded for its store. A row whose live byte is 0 keeps x and
// gets h = 0 whatever its f and g hold (they are not read).
//
// Bound by memory: f, g, x in, x', h out. 28800 rows of 1536 (x fp32, the rest bf16, 619 MB): 119 us, 5.2 TB/s. A row
// over the warps of a block keeps a thread's share small (75 registers, 94 with biases); a warp a row took 242 us (250
// registers, few rows in flight), the same without the next row's loads ahead of this row's sums 141 us, without the vectors
// in registers 149 us. 24 warps an SM stay: with 16 and 32, 256 wide 43.3 -> 47.3 and 52.5 us (60000 rows), 1024 77.8 -> 89.3
// and 94.9 (28800), 1536 118 -> 168 and 148, 2048 90 -> 103 and 111 (16384), 4096 117 -> 111 and 122 (10000), cold caches.
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
  int shift;  // k_norm_gate<.., kShift>: the first row's start past a 16-byte boundary of f, in elements
};

// act(g). The fast exponential is off by about |g| 2^-23 of its value: fp32 activations have expf, since a g of theirs is
// exact to |g| 2^-25; of 16-bit ones g's own rounding moves it by |g| 2^-12 and more. 9000 x 1536 of fp32 take 54 us with
// either; with expf for 16-bit ones too, 28800 x 1536 of bf16 took 129 us in place of 118 (cold caches).
template <int FT>
__device__ __forceinline__ float gate_of(int gate, float g) {
  if (gate == 0) return 1.f;
  const float s = __fdividef(1.f, 1.f + (FT == 0 ? expf(-g) : __expf(-g)));
  return gate == 1 ? s : g * s;
}

// the sum of v over the block's warps, in an order that does not depend on timing. calls: the block's calls so far; two
// rows of 8 in turn, so that every warp has read a call's values (before it arrives at the next) when they are replaced
__device__ __forceinline__ float block_sum(float v, float (*red)[8], int &calls) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = blockDim.x / 32;
  if (warps > 1) {
    const int buf = calls++ & 1;
    if (threadIdx.x % 32 == 0) red[buf][threadIdx.x / 32] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < warps; w++) v += red[buf][w];
  }
  return v;
}

// V consecutive elements as they lie in memory
template <int T, int V>
struct Raw {
  static constexpr int words = V == 1 ? 1 : V * (T == 0 ? 4 : 2) / 4;
  uint32_t w[words];
  __device__ __forceinline__ void load(const elem_t<T> *p) {
    if constexpr (V == 1) {
      w[0] = T == 0 ? *reinterpret_cast<const uint32_t *>(p) : *reinterpret_cast<const uint16_t *>(p);
    } else {
#pragma unroll
      for (int i = 0; i < words; i += 4) {
        const uint4 v = reinterpret_cast<const uint4 *>(p)[i / 4];
        w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
      }
    }
  }
  // the elements j of the group's in the mask
  __device__ __forceinline__ void load_some(const elem_t<T> *p, unsigned mask) {
#pragma unroll
    for (int j = 0; j < V; j++)
      if ((mask >> j) & 1) {
        if constexpr (T == 0) w[j] = __float_as_uint(p[j]);
        else w[j / 2] |= (uint32_t)reinterpret_cast<const uint16_t *>(p)[j] << 16 * (j & 1);
      }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < words; i++) w[i] = 0;
  }
  __device__ __forceinline__ float at(int j) const {
    if constexpr (T == 0) return __uint_as_float(w[j]);
    else {
      const float2 f = unpack2<T>(w[j / 2]);
      return j & 1 ? f.y : f.x;
    }
  }
};

// the elements in the mask of a group of 8
template <int T, int V>
__device__ __forceinline__ void store_some(elem_t<T> *p, const float (&v)[V], unsigned mask) {
#pragma unroll
  for (int j = 0; j < V; j++)
    if ((mask >> j) & 1) p[j] = Elem<T>::put(v[j]);
}

// A block a row, each thread NV groups of V consecutive columns (D <= blockDim NV V), the same for all its rows: the
// vectors' values for them are read once and stay in registers (alpha gamma wpost as one). B: with bpost and bpre.
// kShift (V 8): rows that start anywhere, all tensors' at the same distance past 16 bytes; the groups lie on the 16-byte
// boundaries, the first and the last one partly outside the row: their loads take the neighbours' elements too, which are
// left out of the sums, their stores go element by element. A block's rows are 8 apart or a multiple, so the distance is
// one for all of them.
template <int XT, int FT, int V, int NV, bool B, bool kShift>
__global__ void __launch_bounds__(256) k_norm_gate(const NormArgs a) {
  __shared__ float red[2][8];
  int calls = 0;
  const int D = a.D;
  const float inv = 1.f / (float)D;
  const int shift = kShift ? (int)((a.shift + blockIdx.x * (a.xs & 7)) & 7) : 0;
  auto column = [&](int k) { return (k * (int)blockDim.x + (int)threadIdx.x) * V - shift; };
  unsigned some[NV];  // the group's elements inside the row
#pragma unroll
  for (int k = 0; k < NV; k++) {
    some[k] = 0;
#pragma unroll
    for (int j = 0; j < V; j++) some[k] |= (column(k) + j >= 0 && column(k) + j < D ? 1u : 0u) << j;
  }
  constexpr unsigned kAll = (1u << V) - 1;
  auto inside = [&](int k, int j) { return !kShift || ((some[k] >> j) & 1); };
  wait_launch_before();
  launch_dependents();
  float cu[NV][V], bu[NV][B ? V : 1], ch[NV][V], bh[NV][B ? V : 1];
#pragma unroll
  for (int k = 0; k < NV; k++)
#pragma unroll
    for (int j = 0; j < V; j++) {
      const int c = column(k) + j;
      const bool in = c >= 0 && c < D;
      const float gm = a.alpha * (a.gamma && in ? a.gamma[c] : 1.f);
      cu[k][j] = in ? gm * (a.wpost ? a.wpost[c] : 1.f) : 0.f;
      ch[k][j] = a.wpre && in ? a.wpre[c] : 1.f;
      if constexpr (B) {
        bu[k][j] = a.bpost && in ? gm * a.bpost[c] : 0.f;
        bh[k][j] = a.bpre && in ? a.bpre[c] : 0.f;
      }
    }
  Raw<XT, V> rx[NV], nx[NV];
  Raw<FT, V> rf[NV], rg[NV], nf[NV], ng[NV];
  // a row's values; a dead row's f and g are not read
  auto load = [&](long long r, bool live, Raw<XT, V> (&vx)[NV], Raw<FT, V> (&vf)[NV], Raw<FT, V> (&vg)[NV]) {
    const elem_t<XT> *x = (const elem_t<XT> *)a.x + r * a.xs;
    const elem_t<FT> *f = (const elem_t<FT> *)a.f + r * a.fs, *g = (const elem_t<FT> *)a.g + r * a.gs;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const int c = column(k);
      vx[k].zero();
      vf[k].zero();
      vg[k].zero();
      // past the row's ends another row's elements, read and left out; past the first and the last row's nothing
      if (kShift && ((c < 0 && r == 0) || (c + V > D && r == a.rows - 1))) {
        vx[k].load_some(x + c, some[k]);
        if (a.f && live) {
          vf[k].load_some(f + c, some[k]);
          if (a.gate) vg[k].load_some(g + c, some[k]);
        }
      } else if (c < D) {
        vx[k].load(x + c);
        if (a.f && live) {
          vf[k].load(f + c);
          if (a.gate) vg[k].load(g + c);
        }
      }
    }
  };
  bool live = blockIdx.x < a.rows && (!a.live || a.live[blockIdx.x]), next_live = false;
  if (blockIdx.x < a.rows) load(blockIdx.x, live, rx, rf, rg);
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const bool upd = a.f && live;
    // the block's next row, on its way while this one's sums wait for its warps
    const long long rn = r + gridDim.x;
    if (rn < a.rows) {
      next_live = !a.live || a.live[rn];
      load(rn, next_live, nx, nf, ng);
    }
    float y[NV][V];
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
      for (int j = 0; j < V; j++) y[k][j] = rx[k].at(j);
    // v is zero past the row's end, and stays out of the squares there
    auto in_row = [&](int k) { return column(k) < D; };
    if (upd) {
      float mean = 0.f, ss = 0.f;
      if (a.layer) {
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
          for (int j = 0; j < V; j++) mean += inside(k, j) ? rf[k].at(j) : 0.f;
        mean = block_sum(mean, red, calls) * inv;
      }
#pragma unroll
      for (int k = 0; k < NV; k++)
        if (in_row(k))
#pragma unroll
          for (int j = 0; j < V; j++) ss += inside(k, j) ? (rf[k].at(j) - mean) * (rf[k].at(j) - mean) : 0.f;
      const float rs = rsqrtf(block_sum(ss, red, calls) * inv + a.eps);
#pragma unroll
      for (int k = 0; k < NV; k++)
#pragma unroll
        for (int j = 0; j < V; j++) {
          float u = (rf[k].at(j) - mean) * rs * cu[k][j];
          if constexpr (B) u += bu[k][j];
          y[k][j] += gate_of<FT>(a.gate, rg[k].at(j)) * u;
        }
    }
    if (a.xo) {
      elem_t<XT> *xo = (elem_t<XT> *)a.xo + r * a.xos;
#pragma unroll
      for (int k = 0; k < NV; k++)
        if (in_row(k)) {
          if (!kShift || some[k] == kAll) store_elems<XT, V>(xo + column(k), y[k]);
          else if constexpr (kShift) store_some<XT, V>(xo + column(k), y[k], some[k]);
        }
    }
    if (a.h) {
      float mean = 0.f, ss = 0.f;
      if (a.layer) {
#pragma unroll
        for (int k = 0; k < NV; k++)
          if (in_row(k))
#pragma unroll
            for (int j = 0; j < V; j++) mean += inside(k, j) ? y[k][j] : 0.f;
        mean = block_sum(mean, red, calls) * inv;
      }
#pragma unroll
      for (int k = 0; k < NV; k++)
        if (in_row(k))
#pragma unroll
          for (int j = 0; j < V; j++) ss += inside(k, j) ? (y[k][j] - mean) * (y[k][j] - mean) : 0.f;
      const float rs = rsqrtf(block_sum(ss, red, calls) * inv + a.eps);
      elem_t<FT> *h = (elem_t<FT> *)a.h + r * a.hs;
#pragma unroll
      for (int k = 0; k < NV; k++) {
        if (!in_row(k)) continue;
        float o[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
          o[j] = (y[k][j] - mean) * rs * ch[k][j];
          if constexpr (B) o[j] += bh[k][j];
          if (!live) o[j] = 0.f;
        }
        if (!kShift || some[k] == kAll) store_elems<FT, V>(h + column(k), o);
        else if constexpr (kShift) store_some<FT, V>(h + column(k), o, some[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < NV; k++) { rx[k] = nx[k]; rf[k] = nf[k]; rg[k] = ng[k]; }
    live = next_live;
  }
}

// Rows wider than the registers of a block hold: one block a row, each element formed again from f, g and x for every
// sum (the rows stay in L1 / L2), stored in the last pass, which reads an element's inputs before it writes there.
template <int XT, int FT>
__global__ void __launch_bounds__(kNormThreads) k_norm_gate_wide(const NormArgs a) {
  __shared__ float red[2][8];
  int calls = 0;
  const int D = a.D;
  const float inv = 1.f / (float)D;
  wait_launch_before();
  launch_dependents();
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const bool live = !a.live || a.live[r], upd = live && a.f;
    const elem_t<XT> *x = (const elem_t<XT> *)a.x + r * a.xs;
    const elem_t<FT> *f = (const elem_t<FT> *)a.f + r * a.fs, *g = (const elem_t<FT> *)a.g + r * a.gs;
    float fm = 0.f, frs = 0.f;
    if (upd) {
      float s = 0.f;
      if (a.layer) {
        for (int c = threadIdx.x; c < D; c += kNormThreads) s += Elem<FT>::get(f[c]);
        fm = block_sum(s, red, calls) * inv;
      }
      s = 0.f;
      for (int c = threadIdx.x; c < D; c += kNormThreads) {
        const float v = Elem<FT>::get(f[c]) - fm;
        s += v * v;
      }
      frs = rsqrtf(block_sum(s, red, calls) * inv + a.eps);
    }
    auto y_at = [&](int c) {
      float y = Elem<XT>::get(x[c]);
      if (upd) {
        float u = (Elem<FT>::get(f[c]) - fm) * frs * (a.wpost ? a.wpost[c] : 1.f);
        if (a.bpost) u += a.bpost[c];
        y += a.alpha * (a.gamma ? a.gamma[c] : 1.f) * (gate_of<FT>(a.gate, a.gate ? Elem<FT>::get(g[c]) : 0.f) * u);
      }
      return y;
    };
    float mean = 0.f, rs = 0.f;
    if (a.h && live) {
      float s = 0.f;
      if (a.layer) {
        for (int c = threadIdx.x; c < D; c += kNormThreads) s += y_at(c);
        mean = block_sum(s, red, calls) * inv;
      }
      s = 0.f;
      for (int c = threadIdx.x; c < D; c += kNormThreads) {
        const float v = y_at(c) - mean;
        s += v * v;
      }
      rs = rsqrtf(block_sum(s, red, calls) * inv + a.eps);
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

template <int XT, int FT, int V, int NV, bool kShift = false>
cudaError_t launch_rows(const NormArgs &a, cudaStream_t st) {
  const int warps = (a.D + (kShift ? 7 : 0) + 32 * V * NV - 1) / (32 * V * NV);
  const long long most = (long long)num_sms() * (24 / warps) & (kShift ? ~7ll : ~0ll);
  const int blocks = (int)(a.rows < most ? a.rows : most);
  auto kernel = a.bpost || a.bpre ? k_norm_gate<XT, FT, V, NV, true, kShift> : k_norm_gate<XT, FT, V, NV, false, kShift>;
  // An early start hides a small call's latency (one row 8.5 -> 8.1 us). A full grid of blocks that stay would settle
  // unevenly in what the launch before leaves free (3000 x 1021, one element an access: 24.6 -> 29.4 us)
  if (blocks < num_sms()) return launch_early(kernel, dim3(blocks), 32 * warps, 0, st, a);
  kernel<<<blocks, 32 * warps, 0, st>>>(a);
  return cudaGetLastError();
}

template <int XT, int FT>
cudaError_t launch_norm(const NormArgs &a, bool vec, bool shifted, cudaStream_t st) {
  // Up to 2048 wide a thread has one group of 8 elements, up to 8192 four: 255 registers there and up to 350 bytes of them
  // spilled, and still ahead of the form without (fp32 residual, bf16, RMS, us with four groups / wide form: 16320 rows of
  // 2056 152 / 299, 8192 of 4096 100 / 283, 4096 of 8192 115 / 317, 300 of 4096 18.5 / 27.0; all fp32, layer norm, biases: 8192
  // of 4096 228 / 394). Past that, and for rows off 16 bytes past 2048, the wide form: 4092 of 8200 320 us, 1677 of 20000 408,
  // 8184 of 4100 293. Off 16 bytes with few rows, one element an access (500 rows, this form / wide: fp16, layer norm, 1021
  // wide 14.2 / 16.4, 1500 24.6 / 19.6, 2001 24.6 / 22.5; bf16, RMS, 1500 14.3 / 16.4, 2001 15.1 / 18.4; 20000 rows of 100, fp16
  // 22.5 / 129). Rows of any start, wide and many enough, by groups of 8 on the 16-byte boundaries:
  // 20000 rows, fp16, layer norm, us with groups of 8 between ends one by one / one element an access: 100 wide 20.6 / 18.7,
  // 193 22.5 / 34.9, 1533 150 / 281, 2001 152 / 379; 1021 wide, 1 row 5.5 / 3.9, 592 rows 8.8 / 8.2, 1184 12.3 / 13.9, 3000
  // 22.5 / 28.3 (1024 wide on 16 bytes: 16.5)
  if (shifted && a.D >= 192 && a.D <= 2041 && a.rows > 4 * num_sms()) return launch_rows<XT, FT, 8, 1, true>(a, st);
  if (vec) {
    if (a.D <= 2048) return launch_rows<XT, FT, 8, 1>(a, st);
    if (a.D <= 8192) return launch_rows<XT, FT, 8, 4>(a, st);
  } else {
    if (a.D <= 1024) return launch_rows<XT, FT, 1, 4>(a, st);
    if (a.D <= 2048) return launch_rows<XT, FT, 1, 8>(a, st);
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
  // rows of any start and width, all tensors' at the same elements of 8: the same with the ends one by one
  bool shifted = !vec;
  a.shift = -1;
  auto same = [&](const void *p, long long stride, int type) {
    if (!p) return;
    const int size = type == 0 ? 4 : 2, off = (int)((uintptr_t)p / size & 7);
    if ((uintptr_t)p % size || (stride & 7) != (a.xs & 7) || (a.shift >= 0 && off != a.shift)) shifted = false;
    a.shift = off;
  };
  same(a.x, a.xs, p->xtype);
  same(a.f, a.fs, p->type);
  if (a.f && a.gate) same(a.g, a.gs, p->type);
  same(a.xo, a.xos, p->xtype);
  same(a.h, a.hs, p->type);
  const cudaStream_t s = (cudaStream_t)st;
  if (p->xtype == 0 && p->type == 0) return launch_norm<0, 0>(a, vec, shifted, s);
  if (p->xtype == 0 && p->type == 1) return launch_norm<0, 1>(a, vec, shifted, s);
  if (p->xtype == 0 && p->type == 2) return launch_norm<0, 2>(a, vec, shifted, s);
  if (p->xtype == 1 && p->type == 1) return launch_norm<1, 1>(a, vec, shifted, s);
  if (p->xtype == 2 && p->type == 2) return launch_norm<2, 2>(a, vec, shifted, s);
  return cudaErrorInvalidValue;
}
