// Linear attention with a decay for each key / value head (bnn_dattn): per sequence and head
//
//   S_t = lambda S_{t-1} + live_t k_t^T v_t,   o_t = live_t scale q_t S_t
//
// S [dk][dv] fp32, q heads in groups of G that share one k/v head and its S.
#include <cuda.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "bnn_kernels.h"
#include "seq.cuh"
#include "smem_attr.cuh"
#include "sync.cuh"
#include "tc16.cuh"

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
  int over;  // not 0: the recurrent form has the sequences of up to so many tokens, the chunk form the others
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
// Bound by memory for single tokens: S is read once and written once (at most 8 + 8 KB a CTA). 300 sequences of 16 heads of
// 64 x 64 (160 MB): 30 us, 5.3 TB/s; one sequence: 3 us, two waits for memory.
constexpr int kRecG = 8;  // q heads whose partial sums are in shared memory at once

template <int T>
__global__ void __launch_bounds__(256) k_dattn_rec(const DattnArgs a) {
  __shared__ float part[2][kRecG][8][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
  const int hk = blockIdx.y, i = blockIdx.x, cs = blockIdx.z * 32, c0 = cs + (lane % 8) * 4;
  const int dk = a.dk, dv = a.dv;
  const bool col = c0 < dv;
  wait_launch_before();
  launch_dependents();
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
  if (a.over && t1 - t0 > a.over) return;
  const float lam = a.pow[hk * kDattnPow + 1];
  int buf = 0;
  for (long long t = t0; t < t1; t++) {
    const elem_t<T> *k = (const elem_t<T> *)a.k + t * a.kts + (long long)hk * dk;
    const elem_t<T> *v = (const elem_t<T> *)a.v + t * a.vts + (long long)hk * dv + c0;
    const elem_t<T> *q = (const elem_t<T> *)a.q + t * a.qts + (long long)hk * a.G * dk;
    elem_t<T> *o = (elem_t<T> *)a.o + t * a.ots + (long long)hk * a.G * dv;
    // all of the token's loads before the first use, a dead token's too: one wait for memory, with that for S
    const bool live = !a.live || a.live[t];
    const uint2 vw = col ? *reinterpret_cast<const uint2 *>(v) : make_uint2(0, 0);
    elem_t<T> kw[4], qw[4];
#pragma unroll
    for (int p = 0; p < 4; p++) {
      const int r = min(row[p], dk - 1);
      kw[p] = k[r];
      qw[p] = q[r];
    }
    if (!live) {
#pragma unroll
      for (int p = 0; p < 4; p++) { S[p].x *= lam; S[p].y *= lam; S[p].z *= lam; S[p].w *= lam; }
      for (int g = warp; g < a.G; g += warps)
        if (cs + lane < dv) o[(long long)g * dv + cs + lane] = Elem<T>::put(0.f);
      continue;
    }
    const float2 v0 = unpack2<T>(vw.x), v1 = unpack2<T>(vw.y);
    const float4 vv = make_float4(v0.x, v0.y, v1.x, v1.y);
#pragma unroll
    for (int p = 0; p < 4; p++) {
      const float kk = row[p] < dk ? Elem<T>::get(kw[p]) : 0.f;
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
          const float qq = Elem<T>::get(g0 + g == 0 ? qw[p] : q[(long long)(g0 + g) * dk + row[p]]);
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


// ------------------------------------------------------------------ the chunk form
//
// 128 tokens at a time, i, j in the chunk, S the state before it, n its tokens (lambda^x from a table):
//   o_i = scale (lambda^(i+1) q_i S + sum_{j <= i} lambda^(i-j) (q_i . k_j) v_j)
//   S'  = lambda^n S + sum_j lambda^(n-1-j) k_j^T v_j
// as four products on the tensor cores (tcgen05 kind::f16, fp32 accumulators in TMEM): QK = Q K^T, O1 = Q S, DS = K'^T V
// with K'_j = lambda^(n-1-j) k_j, and O2 = P V with P = QK times the decays below the diagonal. Q, K and V arrive by TMA
// (128-byte swizzle, heads narrower than the padded width DP read as zero past their end).
//
// What is computed and goes back into a product (P, S, K') goes as 16-bit parts whose sum keeps enough of the fp32 value:
//  - bf16: P and S as two parts (2^-16 of a value, so that o keeps the error of its one rounding; one part each would add
//    1.4 times that rounding), K' as three (all 24 bits: the state is fp32 and sums K' over every chunk; with two parts
//    it was 2.4e-6 off, against 4.5e-7 for fp32 products).
//  - fp16: two parts are 22 bits, but only within the type's range, so each is scaled by a power of two that a maximum
//    gives: P by its row's, S and K' by their tile's, and K' has the decays counted from the chunk's last live token. The
//    scales go into the fp32 steps after the products. The maxima are those of the decayed values, so that a loud token
//    long ago takes no bits from the present (24 x 9600 tokens, cold caches: 761 us without the decays, 808 with). The maximum comes to 2^14 .. 2^15 and the second part ends at 2^-24: 22 bits
//    for values down to 2^17 below the maximum, 11 at 2^28. That far below, P and S are under the rounding of an fp16 output
//    beside the others; in K' it is a feature of k that small beside the chunk's largest.
//
// One CTA per (segment of a sequence, k/v head) walks the segment's chunks, and for each the G q heads of the group
// ("unit" u = (chunk, q head)). Roles: warps 0 and 2 MMA issue, warp 1 TMA, 8 warps turn QK into P (in place in TMEM, as the
// A operand of the last product) and join O1 and O2 into o, 16 warps hold S in registers and form K' and the S operand. S
// in registers stays fp32: lambda^n S + DS, once a chunk. The roles' loops are rolled: unrolled, their code did not stay in
// the instruction cache together and a unit took twice as long. The issuing warp stays converged
// (elect.sync): from one lane's branch each tcgen05.mma took 70 cycles to issue, more than a 128 x 64 x 16 product.
// A masked token, and a row past the segment's end, has its k and v rows taken as zero (K' zero, V zeroed in shared
// memory, its P column zero by selection, so that NaN and infinities there stay out); its o row is zero or not stored.
// A live token's NaN or infinity meets the rows before it in the same products (0 NaN) and makes them NaN. It also makes
// the state so, for good, which the state warps look for once the segment is done: chunks that hold such a token are then
// formed again token by token (redo_chunks; 1 to 2 % of a call without one). To keep it out of the products instead took 8
// to 12 % of every call (a selection above P's diagonal and a pass over each tile of V by a warp of its own).
//
// Bound by its roles' chain through a chunk and by shared memory's bandwidth, not by the products: DP 64 takes 4900 cycles a
// chunk and head, of which the products are 2400 (each operand's parts are products of their own). 24 sequences of 9600
// tokens, 16 heads of 64 (bf16, 1.9 GB): 667 us, 2.8 TB/s; 384 CTAs on 148 SMs are 2.6 rounds that take 3. DP 128 has
// shared memory for one stage only: one sequence of 28800 tokens, 12 heads of 128 (0.35 GB): 185 us, 62 of them the first
// pass for the parts' states. 37 sequences of 1 to 611 tokens, 4 heads of 96 x 72 shared by 3 (fp16): 81 us.
constexpr int kChunk = 128;
constexpr int kDaThreads = 896;
constexpr int kDaP = 4, kDaS = 12;  // first warps of the P and state roles

struct DaArgs {
  DattnArgs d;
  int seg_tokens;     // tokens of a segment (a multiple of kChunk), 0: a sequence is one segment
  int segs;           // the most segments of the call, and CTAs of a head
  float *seg_state;   // [segment][Hk][dk][dv]: a segment's own sum (kState), then the state before it
  int *err;
};

// the sequence, part, tokens and last-part flag of segment s: sequence i has max(1, ceil(length / seg_tokens)) segments,
// or none where the recurrent form has it, in order. One warp; false past the last segment.
__device__ bool find_segment(const DaArgs &a, int s, int &seq, int &part, long long &t0, long long &t1, bool &last) {
  const int lane = threadIdx.x % 32;
  long long b0, b1;
  if (!a.seg_tokens && !a.d.over) {
    if (s >= a.d.n) return false;
    seq = s; part = 0; last = true;
    seq_range(a.d, s, t0, t1);
    return true;
  }
  int base = 0;
  for (int i0 = 0; i0 < a.d.n; i0 += 32) {
    const int i = i0 + lane;
    int parts = 0;
    if (i < a.d.n) {
      seq_range(a.d, i, b0, b1);
      parts = a.d.over ? b1 - b0 > a.d.over : max(1, (int)((b1 - b0 + a.seg_tokens - 1) / a.seg_tokens));
    }
    int sum = parts;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, s < base + sum);
    if (hit) {
      const int l = __ffs(hit) - 1;
      seq = i0 + l;
      const int end = __shfl_sync(0xffffffffu, sum, l), np = __shfl_sync(0xffffffffu, parts, l);
      part = s - (base + end - np);
      last = part == np - 1;
      seq_range(a.d, seq, b0, b1);
      t0 = b0 + (long long)part * a.seg_tokens;
      t1 = last ? b1 : t0 + a.seg_tokens;
      return true;
    }
    base += __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}

// Shared memory and TMEM. A pass for the state alone has no Q and no S operand. Else, DP 128: one stage of Q, K, V, and the
// first part of K' in K's place (it waits for QK to have read K); DP 64: two stages (three of K), two QK / P regions, two sets of K', formed a chunk ahead.
template <int T, int DP, bool kState>
struct DaLayout {
  static constexpr int parts = T == 2 ? 3 : 2;      // of K'
  static constexpr bool in_place = DP == 128 && !kState;
  static constexpr int stages = in_place ? 1 : 2;    // Q and V tiles in flight
  static constexpr int kp_sets = DP == 64 ? 2 : 1;   // sets of K': with two it is formed a chunk ahead
  static constexpr int k_stages = DP == 64 ? 3 : stages;  // K tiles: the last to be free again (after DS) and the first needed
  static constexpr int qk_bufs = DP == 64 ? 2 : 1;  // QK / P regions in TMEM
  static constexpr uint32_t panel = kChunk * 128;   // 64 columns of a 128-row tile
  static constexpr uint32_t tile = kChunk * DP * 2;
  static constexpr uint32_t s_panel = DP * 128, s_tile = DP * DP * 2;
  static constexpr uint32_t q = 0, k = q + (kState ? 0 : stages * tile), v = k + k_stages * tile, kp = v + stages * tile,
                            st = kp + (in_place ? parts - 1 : kp_sets * parts) * tile, end = st + (kState ? 0 : 2 * s_tile);
  static constexpr uint32_t t_qk = 0, t_o1 = qk_bufs * 128, t_o2 = t_o1 + DP, t_ds = t_o2 + DP;  // TMEM columns
  // kState: the last part's second panel is read, not used
  static constexpr size_t smem = end + 1024 + (kState && DP == 64 ? panel : 0);
  static constexpr int scales = T == 1 ? (qk_bufs == 2 ? 4 : 2) : 1;  // P row scales: units until o has read them
  // part x of K' of set s
  static __device__ __forceinline__ uint32_t kpart(uint32_t base, int s, int x) {
    return in_place ? (x ? base + kp + (x - 1) * tile : base + k) : base + kp + (s % kp_sets * parts + x) * tile;
  }
};

// a place in a ring of N and the parity of its use
template <int N>
struct Ring {
  int at = 0, parity = 0;
  bool used = false;  // every place has been used once
  __device__ __forceinline__ void next() {
    if (N == 1 || ++at == N) {
      at = 0;
      parity ^= 1;
      used = true;
    }
  }
};

// the live tokens among a chunk's 128, bit j % 32 of word j / 32 (one warp; every lane gets all words)
__device__ __forceinline__ void live_words(const DattnArgs &a, long long t, int n, uint32_t (&w)[4]) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int b = 0; b < 4; b++) {
    const int j = 32 * b + lane;
    w[b] = __ballot_sync(0xffffffffu, j < n && (!a.live || a.live[t + j]));
  }
}
__device__ __forceinline__ uint32_t word_of(const uint32_t (&w)[4], int b) {
  return b == 0 ? w[0] : b == 1 ? w[1] : b == 2 ? w[2] : w[3];
}

// the power of two that brings a magnitude m to [2^14, 2^15), and its inverse; 1 where m is zero or not finite
__device__ __forceinline__ float scale_to_f16(float m, float &inv) {
  const int e = (int)(__float_as_uint(m) >> 23);
  if (e == 0 || e == 255) { inv = 1.f; return 1.f; }
  const int x = min(max(14 + 127 - e, -126), 126);
  inv = __uint_as_float((uint32_t)(127 - x) << 23);
  return __uint_as_float((uint32_t)(127 + x) << 23);
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// Pieces of 4 values among groups of L lanes: before, piece j of lane l is piece l % L of row j of its group; after, piece
// j of its own row (or back). A warp's memory accesses then cover L x 16 consecutive bytes of few rows.
template <int L>
__device__ __forceinline__ void turn_rows(float (&v)[4 * L]) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int b = 1; b < L; b <<= 1) {
    const bool up = lane & b;
#pragma unroll
    for (int j = 0; j < L; j++) {
      if (j & b) continue;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float got = __shfl_xor_sync(0xffffffffu, up ? v[4 * j + e] : v[4 * (j + b) + e], b);
        if (up) v[4 * j + e] = got;
        else v[4 * (j + b) + e] = got;
      }
    }
  }
}

__device__ __forceinline__ void sts128(uint32_t at, const uint32_t (&x)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
}

template <int T>
__device__ __forceinline__ bool no_number(elem_t<T> v) {
  return !(fabsf(Elem<T>::get(v)) < __int_as_float(0x7f800000));
}

// The outputs of the chunks from the first to the last that holds a live token whose k or v is not finite, by the
// definition: S_t = lambda S_(t-1) + k_t^T v_t from the segment's start (`from`, NULL: zero), o_t = scale q_t S_t. A warp
// has 4 columns of S at a time, a lane the rows lane + 32 p. All of the CTA's threads; span: two shared words.
template <int T>
__device__ __forceinline__ void redo_chunks(const DattnArgs &d, int hk, long long t0, long long t1, const float *from, float lam,
                                         int *span) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) { span[0] = 0x7fffffff; span[1] = -1; }
  __syncthreads();
  for (long long t = t0 + warp; t < t1; t += kDaThreads / 32) {
    if (d.live && !d.live[t]) continue;
    const elem_t<T> *k = (const elem_t<T> *)d.k + t * d.kts + (long long)hk * d.dk;
    const elem_t<T> *v = (const elem_t<T> *)d.v + t * d.vts + (long long)hk * d.dv;
    bool bad = false;
    for (int c = lane; c < d.dk; c += 32) bad |= no_number<T>(k[c]);
    for (int c = lane; c < d.dv; c += 32) bad |= no_number<T>(v[c]);
    if (bad) {
      atomicMin(&span[0], (int)((t - t0) / kChunk));
      atomicMax(&span[1], (int)((t - t0) / kChunk));
    }
  }
  __syncthreads();
  const long long first = t0 + (long long)span[0] * kChunk, end = min(t1, t0 + (long long)(span[1] + 1) * kChunk);
  for (int c0 = 4 * warp; c0 < d.dv && span[1] >= 0; c0 += kDaThreads / 8) {
    float S[4][4];
#pragma unroll
    for (int p = 0; p < 4; p++)
#pragma unroll
      for (int c = 0; c < 4; c++)
        S[p][c] = from && lane + 32 * p < d.dk ? from[(long long)(lane + 32 * p) * d.dv + c0 + c] : 0.f;
    for (long long t = t0; t < end; t++) {
      const bool live = !d.live || d.live[t];
      const elem_t<T> *k = (const elem_t<T> *)d.k + t * d.kts + (long long)hk * d.dk;
      const elem_t<T> *v = (const elem_t<T> *)d.v + t * d.vts + (long long)hk * d.dv + c0;
#pragma unroll
      for (int p = 0; p < 4; p++) {
        const float kk = live && lane + 32 * p < d.dk ? Elem<T>::get(k[lane + 32 * p]) : 0.f;
#pragma unroll
        for (int c = 0; c < 4; c++)
          S[p][c] = live && lane + 32 * p < d.dk ? fmaf(kk, Elem<T>::get(v[c]), lam * S[p][c]) : lam * S[p][c];
      }
      if (t < first || !live) continue;  // a dead token's o is zero already
      for (int g = 0; g < d.G; g++) {
        const elem_t<T> *q = (const elem_t<T> *)d.q + t * d.qts + (long long)(hk * d.G + g) * d.dk;
        elem_t<T> *o = (elem_t<T> *)d.o + t * d.ots + (long long)(hk * d.G + g) * d.dv + c0;
        float u[4] = {};
#pragma unroll
        for (int p = 0; p < 4; p++) {
          if (lane + 32 * p >= d.dk) continue;
          const float qq = Elem<T>::get(q[lane + 32 * p]);
#pragma unroll
          for (int c = 0; c < 4; c++) u[c] = fmaf(qq, S[p][c], u[c]);
        }
#pragma unroll
        for (int c = 0; c < 4; c++) {
#pragma unroll
          for (int m = 16; m; m >>= 1) u[c] += __shfl_xor_sync(0xffffffffu, u[c], m);
          if (lane == c) o[c] = Elem<T>::put(d.scale * u[c]);
        }
      }
    }
  }
}

template <int T, int DP, bool kState>
__global__ void __launch_bounds__(kDaThreads, 1) k_dattn_chunk(const __grid_constant__ CUtensorMap mq,
                                                              const __grid_constant__ CUtensorMap mk,
                                                              const __grid_constant__ CUtensorMap mv, const DaArgs a) {
  using L = DaLayout<T, DP, kState>;
  constexpr int NS = L::stages, NK = L::k_stages, NB = L::qk_bufs, PN = DP / 64;
  extern __shared__ uint8_t dsmem[];
  __shared__ __align__(8) unsigned long long b_qfull[NS], b_kfull[NK], b_vfull[NS], b_qempty[NS], b_kempty[NK],
      b_vempty[NS], b_qk[NB], b_p[NB], b_s, b_vfix[NS], b_kp[NS], b_kq, b_ds, b_o, b_oempty, b_max, b_row[4];
  __shared__ uint32_t tmem_s;
  __shared__ volatile int abort_s;
  __shared__ float s_pow[32 + 129];  // s_pow[32 + x] = lambda^x, 0 for x < 0
  __shared__ long long s_range[2];
  __shared__ int s_seg[3], s_span[2];
  __shared__ volatile int s_bad;  // the segment's state is not finite
  __shared__ float s_max[2][16], s_inv[2], s_dsc[2];  // fp16: the state warps' maxima, scales of S and of its sums by chunk
  __shared__ float s_pinv[L::scales][T == 1 ? kChunk : 1];  // fp16: the inverse row scales of P
  __shared__ float s_rowmax[T == 1 ? 2 : 1][2][T == 1 ? kChunk : 1];
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const DattnArgs &d = a.d;
  const int hk = blockIdx.y, G = kState ? 1 : d.G;
  launch_dependents();

  if (warp == 0) {
    int seq = 0, part = 0;
    long long t0 = 0, t1 = 0;
    bool last = false;
    const bool any = find_segment(a, blockIdx.x, seq, part, t0, t1, last);
    if (lane == 0) {
      s_range[0] = t0;
      s_range[1] = t1;
      s_seg[0] = any ? seq : -1;
      s_seg[1] = part;
      s_seg[2] = last;
      for (int s = 0; s < NS; s++) {
        mbar_init(smem_u32(&b_qfull[s]), 1); mbar_init(smem_u32(&b_vfull[s]), 1);
        mbar_init(smem_u32(&b_qempty[s]), 2); mbar_init(smem_u32(&b_vempty[s]), kState ? 1 : 2);
        mbar_init(smem_u32(&b_vfix[s]), 16); mbar_init(smem_u32(&b_kp[s]), 16);
      }
      for (int s = 0; s < NK; s++) { mbar_init(smem_u32(&b_kfull[s]), 1); mbar_init(smem_u32(&b_kempty[s]), kState ? 1 : 2); }
      for (int b = 0; b < NB; b++) { mbar_init(smem_u32(&b_qk[b]), 1); mbar_init(smem_u32(&b_p[b]), 8); }
      mbar_init(smem_u32(&b_s), 16); mbar_init(smem_u32(&b_ds), 1); mbar_init(smem_u32(&b_o), 2);
      mbar_init(smem_u32(&b_oempty), 8); mbar_init(smem_u32(&b_kq), 1);
      mbar_init(smem_u32(&b_max), 16);
      for (int w = 0; w < 4; w++) mbar_init(smem_u32(&b_row[w]), 2);
      abort_s = 0;
      s_bad = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else if (warp == 2) {
    for (int x = lane; x < 32 + 129; x += 32) s_pow[x] = x < 32 ? 0.f : d.pow[hk * kDattnPow + x - 32];
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_s, 0), base = (smem_u32(dsmem) + 1023u) & ~1023u;
  const long long t0 = s_range[0], t1 = s_range[1];
  const int seq = s_seg[0];
  // a segment's own sum is needed where another follows it
  const bool work = seq >= 0 && !(kState && s_seg[2]);
  const int nc = work ? (int)((t1 - t0 + kChunk - 1) / kChunk) : 0, nu = nc * G;
  const float *pw = s_pow + 32;
  // the state before the segment
  auto state_before = [&]() -> const float * {
    if (a.seg_tokens) return a.seg_state + ((long long)blockIdx.x * d.Hk + hk) * d.dk * d.dv;
    const long long slot = d.slot ? d.slot[seq] : seq;
    return d.s0 && slot >= 0 ? d.s0 + (slot * d.Hk + hk) * (long long)d.dk * d.dv : nullptr;
  };
  // where the segment's state goes
  auto state_after = [&]() -> float * {
    if (kState) return work ? a.seg_state + ((long long)blockIdx.x * d.Hk + hk) * d.dk * d.dv : nullptr;
    const long long slot = d.slot ? d.slot[seq] : seq;
    return s_seg[2] && d.s1 && slot >= 0 ? d.s1 + (slot * d.Hk + hk) * (long long)d.dk * d.dv : nullptr;
  };
  // a whole warp waits; false (and the error word set) when the time limit or another role's ran out
  auto wait = [&](unsigned long long &bar, int parity, int code) {
    if (__all_sync(0xffffffffu, mbar_try(smem_u32(&bar), parity))) return true;
    bool ok = mbar_wait_asleep(smem_u32(&bar), parity);
    ok = __all_sync(0xffffffffu, ok && !abort_s);
    if (!ok && lane == 0) {
      if (!abort_s) atomicExch(a.err, code);
      abort_s = 1;
    }
    return ok;
  };

  // o of unit u: this warp's 32 rows and CN columns from c0, 16 at a time. Two neighbouring lanes exchange halves of
  // their rows, so that a store covers whole sectors of 32 bytes: with 16 bytes of 32 rows a store it took 3300 cycles
  // a chunk of 128 x 128
  auto put_o = [&](int c, int g, int u, int c0) {
    constexpr int CN = DP / 2;
    const int r = 32 * (warp % 4) + lane;
    const long long t = t0 + (long long)c * kChunk;
    const int n = (int)min((long long)kChunk, t1 - t) - 32 * (warp % 4);  // this warp's rows inside the segment
    uint32_t alive = ~0u;
    if (d.live) alive = __ballot_sync(0xffffffffu, lane < n && d.live[t + r]);
    if (!wait(b_o, u & 1, BNNK_ERR_EPI_WAIT)) return false;
    tc_fence_after();
    float c1 = d.scale * pw[r + 1], c2 = 1.f;  // bf16: P has the scale already
    if constexpr (T == 1) {
      c1 *= s_inv[c & 1];
      c2 = d.scale * s_pinv[u % L::scales][r];
    }
    const uint32_t tq = tmem + c0 + ((uint32_t)((warp % 4) * 32) << 16);
    const int half = lane & 1, row0 = lane - half;
    elem_t<T> *o = (elem_t<T> *)d.o + (t + 32 * (warp % 4) + row0) * d.ots + (long long)(hk * G + g) * d.dv + c0 + half * 8;
#pragma unroll
    for (int j = 0; j < CN; j += 16) {
      uint32_t z[2][4];
#pragma unroll
      for (int k = 0; k < 2; k++) {
        uint32_t x[8], y[8];
        tmem_ld8(tq + L::t_o1 + j + 8 * k, x);
        tmem_ld8(tq + L::t_o2 + j + 8 * k, y);
        tmem_wait_ld(x, y);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float y0 = __uint_as_float(y[2 * e]), y1 = __uint_as_float(y[2 * e + 1]);
          z[k][e] = pack2f<T>(fmaf(c1, __uint_as_float(x[2 * e]), T == 1 ? c2 * y0 : y0),
                              fmaf(c1, __uint_as_float(x[2 * e + 1]), T == 1 ? c2 * y1 : y1));
        }
      }
      if (j + 16 == CN) {  // the last read: the next unit's products may be written
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&b_oempty));
      }
#pragma unroll
      for (int e = 0; e < 4; e++) {  // half k of this lane's row <-> this lane's half of row row0 + k
        const uint32_t got = __shfl_xor_sync(0xffffffffu, half ? z[0][e] : z[1][e], 1);
        if (half) z[0][e] = got;
        else z[1][e] = got;
      }
#pragma unroll
      for (int k = 0; k < 2; k++)
        if (row0 + k < n && c0 + j + half * 8 < d.dv)
          *reinterpret_cast<uint4 *>(o + k * d.ots + j) =
              (alive >> (row0 + k)) & 1 ? make_uint4(z[k][0], z[k][1], z[k][2], z[k][3]) : make_uint4(0, 0, 0, 0);
    }
    return true;
  };
  constexpr uint32_t bt = T - 1;
  constexpr uint32_t i_qk = idesc_16(bt, 128, 0, 0), i_qs = idesc_16(bt, DP, 0, 1), i_ds = idesc_16(bt, DP, 1, 1),
                     i_pv = idesc_16(bt, DP, 0, 1);
  // a descriptor's address is its low bits, in 16 bytes: K-major steps of 16 lie 32 bytes apart in a panel of 64,
  // MN-major steps 16 rows of 128 bytes
  auto kstep = [](int kk) { return (uint64_t)(((kk / 4) * L::panel + (kk % 4) * 32) >> 4); };
  constexpr uint64_t mnstep = 2048 >> 4;
  // V of chunk c for a product: its arrival, then the state warps' word that its dead rows are zero. The word alone would
  // not do: its parity says as much while the word on the tile's chunk before is still on its way, which nothing else that
  // this warp has waited for excludes. The tile's arrival does: the tile was free after that chunk's DS, which waited for
  // K', and the state warps give their word on K' after the one on V.
  auto wait_v = [&](int c, const Ring<NS> &rc) {
    const bool whole = t1 - (t0 + (long long)c * kChunk) >= kChunk && !d.live;
    if (!wait(b_vfull[rc.at], rc.parity, BNNK_ERR_MMA_WAIT)) return false;
    return whole || wait(b_vfix[rc.at], rc.parity, BNNK_ERR_MMA_WAIT);
  };

  if (warp == 1) {  // TMA
    Ring<NS> rq, rc;  // tiles of Q (one a unit), of V (one a chunk)
    Ring<NK> rk;      // of K
    bool ok = true;
    for (int c = 0; c < nc && ok; c++) {
      const int t = (int)(t0 + (long long)c * kChunk), s = rc.at;
      auto load_q = [&](int g) {
        if (rq.used && !(ok = wait(b_qempty[rq.at], rq.parity ^ 1, BNNK_ERR_TMA_WAIT))) return;
        if (elect_one()) {
          mbar_expect_tx(smem_u32(&b_qfull[rq.at]), L::tile);
#pragma unroll
          for (int p = 0; p < PN; p++)
            tma_load_3d(base + L::q + rq.at * L::tile + p * L::panel, &mq, smem_u32(&b_qfull[rq.at]), 64 * p, hk * G + g, t);
        }
        rq.next();
      };
      if (!kState) load_q(0);  // in the order in which the tiles are free again
      if (!ok || (rk.used && !(ok = wait(b_kempty[rk.at], rk.parity ^ 1, BNNK_ERR_TMA_WAIT)))) break;
      if (elect_one()) {
        mbar_expect_tx(smem_u32(&b_kfull[rk.at]), L::tile);
#pragma unroll
        for (int p = 0; p < PN; p++)
          tma_load_3d(base + L::k + rk.at * L::tile + p * L::panel, &mk, smem_u32(&b_kfull[rk.at]), 64 * p, hk, t);
      }
      rk.next();
      if (!ok || (rc.used && !(ok = wait(b_vempty[s], rc.parity ^ 1, BNNK_ERR_TMA_WAIT)))) break;
      if (elect_one()) {
        mbar_expect_tx(smem_u32(&b_vfull[s]), L::tile);
#pragma unroll
        for (int p = 0; p < PN; p++)
          tma_load_3d(base + L::v + s * L::tile + p * L::panel, &mv, smem_u32(&b_vfull[s]), 64 * p, hk, t);
      }
      for (int g = 1; g < G && ok; g++) load_q(g);
      rc.next();
    }
  } else if (warp == 0 || warp == 2) {  // MMA
    Ring<NS> kq, rq, rc;  // the next QK's Q tile; this unit's Q tile; this chunk's V tile and set of K'
    Ring<NK> kc, rn;      // the next QK's K tile; this chunk's
    Ring<NB> kb, rb;      // the next QK's region; this unit's
    Ring<1> ro, ru, rk;   // single barriers: a phase a unit (O1, O2), a phase a chunk
    int kg = 0, g = 0, c = 0;
    auto issue_qk = [&]() {
      if (!wait(b_qfull[kq.at], kq.parity, BNNK_ERR_MMA_WAIT)) return false;
      if (kg == 0 && !wait(b_kfull[kc.at], kc.parity, BNNK_ERR_MMA_WAIT)) return false;
      tc_fence_after();
      const uint64_t dq = smem_desc<128>(base + L::q + kq.at * L::tile), dk = smem_desc<128>(base + L::k + kc.at * L::tile);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; kk++)
          mma16_ss(tmem + L::t_qk + kb.at * 128, dq + kstep(kk), dk + kstep(kk), i_qk, kk != 0);
        mma_commit(smem_u32(&b_qk[kb.at]));
        mma_commit(smem_u32(&b_qempty[kq.at]));
        if (kg == G - 1) {
          mma_commit(smem_u32(&b_kempty[kc.at]));
          if (L::in_place) mma_commit(smem_u32(&b_kq));
        }
      }
      kq.next();
      kb.next();
      if (++kg == G) { kg = 0; kc.next(); }
      return true;
    };
    auto issue_o1 = [&](int u) {
      if (!wait(b_qfull[rq.at], rq.parity, BNNK_ERR_MMA_WAIT)) return false;
      if (g == 0 && !wait(b_s, rk.parity, BNNK_ERR_MMA_WAIT)) return false;
      if (u && !wait(b_oempty, ro.parity ^ 1, BNNK_ERR_MMA_WAIT)) return false;
      tc_fence_after();
      const uint64_t dq = smem_desc<128>(base + L::q + rq.at * L::tile), ds = smem_desc_mn(base + L::st, L::s_panel);
      if (elect_one()) {
#pragma unroll
        for (int part = 0; part < 2; part++)
#pragma unroll
          for (int kk = 0; kk < DP / 16; kk++)
            mma16_ss(tmem + L::t_o1, dq + kstep(kk), ds + (part * L::s_tile >> 4) + kk * mnstep, i_qs, (part | kk) != 0);
        mma_commit(smem_u32(&b_o));
        mma_commit(smem_u32(&b_qempty[rq.at]));
      }
      rq.next();
      ro.next();
      return true;
    };
    auto issue_ds = [&]() {
      const int s = rc.at;
      if (!wait_v(c, rc) || !wait(b_kp[s], rc.parity, BNNK_ERR_MMA_WAIT)) return false;
      // the chunk before's sum has been read: by the state warps' word that the S operand is there (which O1 waited for), or
      // where there is none by their word after the read (K' formed ahead says nothing about it)
      if (kState && c && !wait(b_s, rk.parity ^ 1, BNNK_ERR_MMA_WAIT)) return false;
      tc_fence_after();
      const uint64_t dk0 = smem_desc_mn(L::kpart(base, s, 0), L::panel), dk1 = smem_desc_mn(L::kpart(base, s, 1), L::panel);
      const uint64_t dv = smem_desc_mn(base + L::v + s * L::tile, L::panel);
      if (elect_one()) {
#pragma unroll
        for (int part = 0; part < L::parts; part++)
#pragma unroll
          for (int kk = 0; kk < 8; kk++)
            mma16_ss(tmem + L::t_ds, (part ? dk1 + ((part - 1) * L::tile >> 4) : dk0) + kk * mnstep, dv + kk * mnstep, i_ds,
                     (part | kk) != 0);
        mma_commit(smem_u32(&b_ds));
        mma_commit(smem_u32(&b_kempty[rn.at]));
        mma_commit(smem_u32(&b_vempty[s]));
      }
      return true;
    };
    auto issue_o2 = [&](int u) {
      const uint64_t dv = smem_desc_mn(base + L::v + rc.at * L::tile, L::panel);
      if (g == 0 && !wait_v(c, rc)) return false;
      if (u && !wait(b_oempty, ru.parity ^ 1, BNNK_ERR_MMA_WAIT)) return false;
      if (!wait(b_p[rb.at], rb.parity, BNNK_ERR_MMA_WAIT)) return false;
      tc_fence_after();
      if (elect_one()) {  // P: 16 columns j a block, its first parts in 8 TMEM columns, the second parts in the next 8
#pragma unroll
        for (int kk = 0; kk < 8; kk++)
#pragma unroll
          for (int part = 0; part < 2; part++)
            mma16_ts(tmem + L::t_o2, tmem + L::t_qk + rb.at * 128 + kk * 16 + part * 8, dv + kk * mnstep, i_pv,
                     (part | kk) != 0);
        mma_commit(smem_u32(&b_o));
        if (g == G - 1) mma_commit(smem_u32(&b_vempty[rc.at]));
      }
      rb.next();
      ru.next();
      return true;
    };
    // Two K tiles or more: one warp issues QK (a unit ahead) and O2, the other O1 and DS, so that the waits of one do not
    // hold up the other's products (24 x 9600 tokens, d 64: 710 us by one warp, 672 by two). One K tile: one warp, O2 after
    // DS, so that the next K is on its way meanwhile (28800 tokens, d 128: 181 us by one warp, 194 by two); the last O2, with
    // no next K, before DS.
    constexpr bool one = L::in_place;
    auto issue = [&](auto which) {  // each warp's own code: first QK and O2 (or all), or O1 and DS
      constexpr bool first = decltype(which)::value;
      bool ok = true;
      if constexpr (first) ok = nu == 0 || issue_qk();
      for (int u = 0; u < nu && ok; u++) {
        const bool last = g == G - 1;
        if constexpr (first && !one)
          if (u + 1 < nu && !(ok = issue_qk())) break;
        if constexpr (!kState && (!first || one))
          if (!(ok = issue_o1(u))) break;
        if constexpr (one) {
#pragma unroll 1
          for (int step = 0; step < 2 && ok; step++)
            if ((step == 0) == (u + 1 < nu)) ok = !last || issue_ds();
            else ok = issue_o2(u);
          if (!ok) break;
        } else if constexpr (first) {
          if (!(ok = issue_o2(u))) break;
        } else {
          if (last && !(ok = issue_ds())) break;
        }
        if (last) {
          g = 0;
          c++;
          rn.next();
          rk.next();
          rc.next();
        } else {
          g++;
        }
        if constexpr (one)
          if (u + 1 < nu) ok = issue_qk();
      }
    };
    if (warp == 0) {
      if constexpr (!kState) issue(std::true_type{});
    } else {
      if constexpr (!one) issue(std::false_type{});
    }
  } else if (warp >= kDaP && warp < kDaS) {
    // P: row i against the columns j <= i, blocks of 16 columns alternating between two warps
    const int qd = warp % 4, h = (warp - kDaP) / 4, i = 32 * qd + lane;
    float fixed[16];  // lambda^(15 - j)
#pragma unroll
    for (int j = 0; j < 16; j++) fixed[j] = pw[15 - j];
    int c = 0, g = 0, c_was = 0, g_was = 0;  // this unit's chunk and q head, and those of the unit before
    for (int u = 0; u < (kState ? 0 : nu); u++) {
      const int b = u % NB;
      const long long t = t0 + (long long)c * kChunk;
      const int n = (int)min((long long)kChunk, t1 - t);
      uint32_t lw[4] = {~0u, ~0u, ~0u, ~0u};
      if (n < kChunk || d.live) live_words(d, t, n, lw);
      if (!wait(b_qk[b], (u / NB) & 1, BNNK_ERR_EPI_WAIT)) break;
      tc_fence_after();
      const uint32_t tq = tmem + L::t_qk + b * 128 + ((uint32_t)(qd * 32) << 16);
      float sc = d.scale;
      const int blocks = 2 * qd + 2;  // those that reach the diagonal
      if constexpr (T == 1) {
        // the largest of the row's decayed products; the row's two warps a half each
        float m = 0.f;
#pragma unroll 1
        for (int blk = h; blk < blocks; blk += 2) {
          uint32_t x[16];
          tmem_ld16(tq + blk * 16, x);
          const uint32_t w = word_of(lw, blk / 2) >> (blk % 2 * 16);
          tmem_wait_ld(x);
          if ((w & 0xffffu) != 0xffffu) {
#pragma unroll
            for (int j = 0; j < 16; j++) x[j] = (w >> j) & 1 ? x[j] : 0u;
          }
          const float *f = pw + i - 16 * blk;  // the decays, as below
          float mb = 0.f;
          if (blk >= 2 * qd) {
#pragma unroll
            for (int j = 0; j < 16; j++) m = fmaxf(m, fabsf(__uint_as_float(x[j]) * f[-j]));
          } else {
#pragma unroll
            for (int j = 0; j < 16; j++) mb = fmaxf(mb, fabsf(__uint_as_float(x[j]) * fixed[j]));
            m = fmaxf(m, mb * f[-15]);
          }
        }
        s_rowmax[u & 1][h][i] = m;
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&b_row[qd]));
        if (!wait(b_row[qd], u & 1, BNNK_ERR_EPI_WAIT)) break;
        float inv;
        sc = scale_to_f16(fmaxf(m, s_rowmax[u & 1][h ^ 1][i]), inv);
        if (h == 0) s_pinv[u % L::scales][i] = inv;
      }
      uint32_t x[16];
      if (h < blocks) tmem_ld16(tq + h * 16, x);
#pragma unroll 1
      for (int blk = h; blk < blocks; blk += 2) {
        uint32_t p[16];
        const uint32_t w = word_of(lw, blk / 2) >> (blk % 2 * 16);
        // lambda^(i - j): off the diagonal lambda^(i - 16 blk - 15) lambda^(15 - j), which no power overflows and whose
        // second factor is the same for every row; on it from the table, 0 above
        const float *f = pw + i - 16 * blk;
        const bool diagonal = blk >= 2 * qd;
        const float f0 = diagonal ? sc : f[-15] * sc;
        tmem_wait_ld(x);
        if ((w & 0xffffu) != 0xffffu) {
#pragma unroll
          for (int j = 0; j < 16; j++) x[j] = (w >> j) & 1 ? x[j] : 0u;
        }
        if (diagonal) {
#pragma unroll
          for (int j = 0; j < 16; j++) x[j] = __float_as_uint(__uint_as_float(x[j]) * f[-j]);
        } else {
#pragma unroll
          for (int j = 0; j < 16; j++) x[j] = __float_as_uint(__uint_as_float(x[j]) * fixed[j]);
        }
#pragma unroll
        for (int j = 0; j < 16; j += 2)
          split2<T>(__uint_as_float(x[j]) * f0, __uint_as_float(x[j + 1]) * f0, p[j / 2], p[8 + j / 2]);
        if (blk + 2 < blocks) tmem_ld16(tq + (blk + 2) * 16, x);  // the next block, while this one is stored
        tmem_st16(tq + blk * 16, p);
      }
#pragma unroll
      for (int j = 0; j < 16; j++) x[j] = 0;
#pragma unroll 1
      for (int blk = blocks + h; blk < 8; blk += 2) tmem_st16(tq + blk * 16, x);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&b_p[b]));
      // o: of this unit where the next QK waits for its K; else of the unit before, whose products ran meanwhile
      if (L::in_place ? !put_o(c, g, u, h * (DP / 2)) : u && !put_o(c_was, g_was, u - 1, h * (DP / 2))) break;
      if (!L::in_place && u + 1 == nu) put_o(c, g, u, h * (DP / 2));
      c_was = c;
      g_was = g;
      if (++g == G) {
        g = 0;
        c++;
      }
    }
  } else if (warp >= kDaS && seq >= 0) {
    // the state: row r = dk index, DP / 4 columns from c0 in registers
    constexpr int HC = DP / 4;
    const int r = 32 * (warp % 4) + lane, c0 = (warp - kDaS) / 4 * HC, tid = threadIdx.x - 32 * kDaS;
    float S[HC];
    const float *from = kState ? nullptr : state_before();
    if (!kState && a.seg_tokens) wait_launch_before();  // the states before the segments
    // in memory order, a row's HC columns by LP neighbouring lanes: with 16 bytes of 32 rows an access, a state of 128 x 128
    // took 4100 cycles to load and as many to store
    constexpr int LP = HC / 4;
    const int mr = r - lane % LP, mc = c0 + lane % LP * 4;  // this lane's rows mr + j and columns there
#pragma unroll
    for (int j = 0; j < LP; j++) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (from && mr + j < d.dk && mc < d.dv) v = *reinterpret_cast<const float4 *>(from + (long long)(mr + j) * d.dv + mc);
      S[4 * j] = v.x; S[4 * j + 1] = v.y; S[4 * j + 2] = v.z; S[4 * j + 3] = v.w;
    }
    turn_rows<LP>(S);
    // the maximum over the role's threads; a buffer is written again two calls later, when every warp has arrived at
    // the call between and so has read it
    int calls = 0;
    bool ok = true;
    auto role_max = [&](float v) {
      v = warp_max(v);
      if (lane == 0) {
        s_max[calls & 1][warp - kDaS] = v;
        mbar_arrive(smem_u32(&b_max));
      }
      if (ok) ok = wait(b_max, calls & 1, BNNK_ERR_EPI_WAIT);
      return warp_max(s_max[calls++ & 1][lane % 16]);
    };
    auto put_state = [&](int c) {  // S before chunk c as the B operand of O1: row r, MN-major panels of 64 columns
      float sc = 1.f;
      if constexpr (T == 1) {
        float m = 0.f, inv;
#pragma unroll
        for (int j = 0; j < HC; j++) m = fmaxf(m, fabsf(S[j]));
        if (m == __int_as_float(0x7f800000)) {  // infinities are their columns' alone: the others' scale leaves them out
          m = 0.f;
#pragma unroll
          for (int j = 0; j < HC; j++) m = fmaxf(m, isinf(S[j]) ? 0.f : fabsf(S[j]));
        }
        sc = scale_to_f16(role_max(r < DP ? m : 0.f), inv);
        if (tid == 0) s_inv[c & 1] = inv;
      }
      if (r < DP) {
#pragma unroll
        for (int j = 0; j < HC; j += 8) {
          uint32_t h[4], l[4];
#pragma unroll
          for (int e = 0; e < 4; e++) split2<T>(S[j + 2 * e] * sc, S[j + 2 * e + 1] * sc, h[e], l[e]);
          const int col = c0 + j;
          const uint32_t at = base + L::st + (col / 64) * L::s_panel + r * 128 + ((((col % 64) / 8) ^ (r & 7)) << 4);
          sts128(at, h);
          sts128(at + L::s_tile, l);
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&b_s));
    };
    // the dead rows of V and K' of chunk c; false where a wait ran out. dsc: what the state's sum is multiplied by
    float dsc = 1.f;
    uint32_t lw[4] = {~0u, ~0u, ~0u, ~0u};
    auto dead = [&](int m) { return !((word_of(lw, 2 * m + tid / 256) >> (tid / 8 % 32)) & 1); };
    auto fix_v = [&](int c, const Ring<NS> &rc) {
      const int s = rc.at;
      const long long t = t0 + (long long)c * kChunk;
      const int n = (int)min((long long)kChunk, t1 - t);
      // 16-byte slots of the tiles, a row's 8 by 8 lanes: row tid / 8, then 64 rows on. A slot stays where it is, so the
      // tiles written here have the swizzle of the one they come from
      const bool whole = n == kChunk && !d.live;
      if (!whole) {
        live_words(d, t, n, lw);
        if (!(ok = wait(b_vfull[s], rc.parity, BNNK_ERR_EPI_WAIT))) return false;
        const uint32_t zero[4] = {0, 0, 0, 0};
#pragma unroll 1
        for (int m = 0; m < 2; m++)
          if (dead(m))
            for (int p = 0; p < PN; p++) sts128(base + L::v + s * L::tile + p * L::panel + (tid + 512 * m) * 16, zero);
        fence_async_smem();
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(smem_u32(&b_vfix[s]));
      return true;
    };
    auto make_kp = [&](int c, const Ring<NS> &rc, const Ring<NK> &rk) {
      const int s = rc.at;
      const int n = (int)min((long long)kChunk, t1 - (t0 + (long long)c * kChunk));
      if (!(ok = wait(b_kfull[rk.at], rk.parity, BNNK_ERR_EPI_WAIT))) return false;
      int from_j = n - 1;  // the token whose decay counts as 1
      float ksc = 1.f;
      auto load = [&](int m, int p, uint32_t (&x)[4]) {
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                     : "r"(base + L::k + rk.at * L::tile + p * L::panel + (tid + 512 * m) * 16)
                     : "memory");
      };
      if constexpr (T == 1) {
        float mx = 0.f;
        if (n < kChunk || d.live)
          from_j = lw[3] ? 127 - __clz(lw[3]) : lw[2] ? 95 - __clz(lw[2]) : lw[1] ? 63 - __clz(lw[1]) : lw[0] ? 31 - __clz(lw[0]) : 0;
#pragma unroll 1
        for (int m = 0; m < 2; m++)
          if (!dead(m)) {
            float rm = 0.f;
            for (int p = 0; p < PN; p++) {
              uint32_t x[4];
              load(m, p, x);
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const float2 f = unpack2<T>(x[e]);
                rm = fmaxf(rm, fmaxf(fabsf(f.x), fabsf(f.y)));
              }
            }
            mx = fmaxf(mx, rm * pw[from_j - tid / 8 - 64 * m]);
          }
        float inv;
        ksc = scale_to_f16(role_max(mx), inv);
        if (!ok) return false;
        if (tid == 0) s_dsc[c & 1] = inv * pw[n - 1 - from_j];
      }
      if (L::in_place && !(ok = wait(b_kq, c & 1, BNNK_ERR_EPI_WAIT))) return false;
#pragma unroll 1
      for (int m = 0; m < 2; m++) {
        const int row = tid / 8 + 64 * m;
        const bool off_row = dead(m);
        const float wt = off_row ? 0.f : pw[from_j - row] * ksc;
#pragma unroll
        for (int p = 0; p < PN; p++) {
          const uint32_t off = p * L::panel + (tid + 512 * m) * 16;
          uint32_t x[4], h[4], l[4], l2[4];
          load(m, p, x);
          if (off_row) x[0] = x[1] = x[2] = x[3] = 0;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float2 f = unpack2<T>(x[e]);
            if constexpr (L::parts == 3) split3<T>(f.x * wt, f.y * wt, h[e], l[e], l2[e]);
            else split2<T>(f.x * wt, f.y * wt, h[e], l[e]);
          }
          sts128(L::kpart(base, s, 0) + off, h);
          sts128(L::kpart(base, s, 1) + off, l);
          if constexpr (L::parts == 3) sts128(L::kpart(base, s, 2) + off, l2);
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&b_kp[s]));
      return true;
    };
    // one set of K' is formed when DS has read the last (in K's place also when the chunk's last QK has read K); of two
    // sets, one is formed a chunk ahead, while the products of this chunk run
    if (!kState && nc > 0) put_state(0);
    Ring<NS> rc;
    Ring<NK> rk;
    auto next_kp = [&](int c) {
      if (!fix_v(c, rc) || !make_kp(c, rc, rk)) return false;
      rc.next();
      rk.next();
      return true;
    };
    if (L::kp_sets == 2 && nc > 0 && ok) next_kp(0);
    for (int c = 0; c < nc && ok; c++) {
      const int n = (int)min((long long)kChunk, t1 - (t0 + (long long)c * kChunk));
      if (L::kp_sets == 1 ? !next_kp(c) : c + 1 < nc && !next_kp(c + 1)) break;
      if (!(ok = wait(b_ds, c & 1, BNNK_ERR_EPI_WAIT))) break;
      tc_fence_after();
      const float dec = pw[n];
      if constexpr (T == 1) dsc = s_dsc[c & 1];
      const uint32_t td = tmem + L::t_ds + c0 + ((uint32_t)((warp % 4) * 32) << 16);
#pragma unroll
      for (int j = 0; j < HC; j += 16) {
        uint32_t x[16];
        tmem_ld16(td + j, x);
        tmem_wait_ld(x);
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const float v = __uint_as_float(x[e]);
          S[j + e] = fmaf(dec, S[j + e], T == 1 ? v * dsc : v);
        }
      }
      tc_fence_before();
      if (kState) {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&b_s));
        continue;
      }
      if (c + 1 < nc) put_state(c + 1);  // the S operand's last reader, the chunk's last O1, comes before DS
    }
    {
      float *to = ok ? state_after() : nullptr;
      turn_rows<LP>(S);
      if constexpr (!kState) {
        float z = 0.f;
#pragma unroll
        for (int e = 0; e < HC; e++) z = fmaf(S[e], 0.f, z);
        if (z != 0.f && r < DP) s_bad = 1;
        asm volatile("bar.sync 1, 512;" ::: "memory");  // the state warps
      }
      // chunks formed again start from the state before the segment, which this one's place may be: until then it waits in
      // the S operand's place, which DS of the last chunk has come after
      if (!kState && s_bad && ok) to = reinterpret_cast<float *>(dsmem + (base - smem_u32(dsmem)) + L::st);
      if (to) {
#pragma unroll
        for (int j = 0; j < LP; j++)
          if (mr + j < d.dk && mc < d.dv)
            *reinterpret_cast<float4 *>(to + (long long)(mr + j) * d.dv + mc) =
                make_float4(S[4 * j], S[4 * j + 1], S[4 * j + 2], S[4 * j + 3]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  if constexpr (!kState)
    if (s_bad && !abort_s) {
      if (nc) redo_chunks<T>(d, hk, t0, t1, state_before(), pw[1], s_span);
      __syncthreads();  // the state before the segment has been read
      if (float *to = state_after())
        for (int e = threadIdx.x; e < d.dk * d.dv; e += kDaThreads)
          to[e] = reinterpret_cast<const float *>(dsmem + (base - smem_u32(dsmem)) + L::st)[e];
    }
}

// the states before each segment: S = s0, then S = lambda^seg_tokens S + (the segment's own sum), in place in seg_state.
// One thread per state element.
__global__ void __launch_bounds__(256) k_dattn_scan(const DaArgs a) {
  const DattnArgs &d = a.d;
  __shared__ int s_first, s_parts;
  __shared__ float s_dec;
  const int i = blockIdx.z, hk = blockIdx.y;
  launch_dependents();
  if (threadIdx.x < 32) {
    int before = 0, mine = 0;
    for (int j = threadIdx.x; j <= i; j += 32) {
      long long b0, b1;
      seq_range(d, j, b0, b1);
      const int parts = max(1, (int)((b1 - b0 + a.seg_tokens - 1) / a.seg_tokens));
      if (j < i) before += parts;
      else mine = parts;
    }
    for (int o = 16; o; o >>= 1) {
      before += __shfl_xor_sync(0xffffffffu, before, o);
      mine += __shfl_xor_sync(0xffffffffu, mine, o);
    }
    if (threadIdx.x == 0) {
      s_first = before;
      s_parts = min(mine, a.segs - before);  // offsets that do not ascend could ask for more
      // lambda^seg_tokens from the table's lambda^(128 2^k), as two floats each
      double dec = 1.0;
      const float *pk = d.pow + hk * kDattnPow + kDattnPow2;
      for (int k = 0, m = a.seg_tokens / kChunk; m; k++, m >>= 1)
        if (m & 1) dec *= (double)pk[2 * k] + (double)pk[2 * k + 1];
      s_dec = (float)dec;
    }
  }
  __syncthreads();
  const int e = blockIdx.x * 256 + threadIdx.x, size = d.dk * d.dv;
  if (e >= size) return;
  const long long slot = d.slot ? d.slot[i] : i;
  float S = d.s0 && slot >= 0 ? d.s0[(slot * d.Hk + hk) * (long long)size + e] : 0.f;
  float *p = a.seg_state + ((long long)s_first * d.Hk + hk) * size + e;
  const long long step = (long long)d.Hk * size;
  const int parts = s_parts;
  const float dec = s_dec;
  wait_launch_before();  // the segments' own sums
  for (int k0 = 0; k0 < parts; k0 += 8) {  // 8 loads in flight
    float own[8];
#pragma unroll
    for (int k = 0; k < 8; k++) own[k] = k0 + k < parts - 1 ? p[(k0 + k) * step] : 0.f;
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (k0 + k < parts) {
        p[(k0 + k) * step] = S;
        S = fmaf(dec, S, own[k]);
      }
  }
}

template <int T, int DP>
int run_chunk(const DaArgs &a, cudaStream_t st) {
  const DattnArgs &d = a.d;
  CUtensorMap mq, mk, mv;
  int e = encode_heads(&mq, d.q, T == 2, d.dk, d.H, d.tokens, d.qts, kChunk);
  if (!e) e = encode_heads(&mk, d.k, T == 2, d.dk, d.Hk, d.tokens, d.kts, kChunk);
  if (!e) e = encode_heads(&mv, d.v, T == 2, d.dv, d.Hk, d.tokens, d.vts, kChunk);
  if (e) return e;
  static SmemAttr attr_s, attr;
  const dim3 grid(a.segs, d.Hk);
  if (a.seg_tokens) {
    constexpr size_t smem = DaLayout<T, DP, true>::smem;
    e = attr_s.ensure(k_dattn_chunk<T, DP, true>, smem);
    if (e) return e;
    k_dattn_chunk<T, DP, true><<<grid, kDaThreads, smem, st>>>(mq, mk, mv, a);
    e = launch_early(k_dattn_scan, dim3((d.dk * d.dv + 255) / 256, d.Hk, d.n), 256, 0, st, a);
    if (e) return e;
  }
  constexpr size_t smem = DaLayout<T, DP, false>::smem;
  e = attr.ensure(k_dattn_chunk<T, DP, false>, smem);
  if (e) return e;
  if (a.seg_tokens) return launch_early(k_dattn_chunk<T, DP, false>, grid, kDaThreads, smem, st, mq, mk, mv, a);
  k_dattn_chunk<T, DP, false><<<grid, kDaThreads, smem, st>>>(mq, mk, mv, a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace bnn

using namespace bnn;

// Tokens of a segment, 0 for whole sequences. Whole sequences where they are enough CTAs for half of the SMs: one pass.
// Fewer: parts of about equal length, one per SM, whose states come from a first pass over K and V. 8 heads, d 64, us whole
// / in parts: 1 sequence of 2400 tokens 56 / 25, of 9600 185 / 39; 4 of 2400 57 / 41; 8 of 2400 59 / 69, of 9600 195 / 180;
// 12 of 9600 199 / 280; d 128: 1 of 2400 94 / 36. The lengths are known on the device alone: 8 even sequences lose 10 us
// by parts, a long one among 7 short ones gains 146.
static int segment_tokens(int n, int Hk, long long tokens) {
  const long long sms = num_sms(), ctas = (long long)n * Hk;
  if (ctas * 2 > sms) return 0;
  const long long parts = sms / Hk < 1 ? 1 : sms / Hk;  // of all sequences together
  const long long len = ((tokens + parts - 1) / parts + kChunk - 1) / kChunk * kChunk;
  return tokens <= (long long)n * len ? 0 : (int)len;
}

extern "C" long long bnnk_dattn_scratch_states(int n, int Hk, long long tokens) {
  // the most sequences that are split: no more than half of the SMs have, and of more than a chunk each on average
  long long most = num_sms() / (2 * Hk), parts = num_sms() / Hk;
  if (most > n) most = n;
  if (most > (tokens - 1) / kChunk) most = (tokens - 1) / kChunk;
  if (parts > tokens / kChunk) parts = tokens / kChunk;
  return most < 1 ? 0 : (most + parts + 1) * Hk;
}

extern "C" int bnnk_dattn(const bnnk_dattn_args *p, bnn_stream_t st) {
  if (p->n <= 0) return 0;
  const DattnArgs d = {p->n, p->H, p->Hk, p->H / p->Hk, p->dk, p->dv, p->tokens, p->cu, p->slot, p->live, p->q, p->k, p->v,
                       p->qts, p->kts, p->vts, p->s0, p->s1, p->o, p->ots, p->pow, p->scale, 0};
  const cudaStream_t s = (cudaStream_t)st;
  const bool wide = p->dk > 64 || p->dv > 64;
  DaArgs a = {d, segment_tokens(p->n, p->Hk, p->tokens), p->n, p->scratch, p->err};
  // The recurrent form for single tokens (cu NULL) and where the sequences are short on average: a token costs a CTA about
  // 2 us of latency, or a state's share of the SMs' arithmetic where CTAs are many; a chunk costs its 128 rows, filled or
  // not. Measured (8 heads, us, recurrent / chunk): 16 sequences, d 64, of 1 token 8 / 14, of 4 16.4 / 14.3, d 128, of 8
  // 26.6 / 18.4; 300 sequences, d 64, of 12 tokens 111 / 136, of 16 144 / 135, d 128, of 4 183 / 200, of 8 326 / 202.
  // Lengths are known on the device alone, and one of 1000 tokens would take the recurrent form 2 ms: those far above the
  // average go to the chunk form in a second launch, of as many CTAs a head as there can be such sequences (2 us for every
  // num_sms() of them that find none). Where the CTAs are few that costs what it saves, and the call's tokens may all be one
  // sequence's (d 64: 16 tokens of one sequence 35 us recurrent, 14.3 by chunks; of 16 8.3 and 14.4; 4 of one 14.3 and 14.3):
  // the recurrent form has up to 4 tokens of the whole call there, the chunk form the others. Callers that know of single
  // tokens have the step.
  const bool few = (long long)p->n * p->Hk <= num_sms();
  if (!p->cu || p->tokens <= (few ? 4ll : (wide ? 4ll : 12ll) * p->n)) {
    const int over = wide ? 32 : 64, warps = (p->dk + 15) / 16;
    if (p->cu && p->tokens > over) a.d.over = over;
    const dim3 grid(p->n, p->Hk, (p->dv + 31) / 32);
    const int e = p->type == 1 ? launch_early(k_dattn_rec<1>, grid, 32 * warps, 0, s, a.d)
                               : launch_early(k_dattn_rec<2>, grid, 32 * warps, 0, s, a.d);
    if (e || !a.d.over) return e;
    const long long longer = p->tokens / (over + 1);
    a.segs = longer < p->n ? (int)longer : p->n;
    a.seg_tokens = 0;
  } else if (a.seg_tokens) {
    a.segs += (int)(p->tokens / a.seg_tokens);
  }
  if (p->type == 1) return wide ? run_chunk<1, 128>(a, s) : run_chunk<1, 64>(a, s);
  return wide ? run_chunk<2, 128>(a, s) : run_chunk<2, 64>(a, s);
}
