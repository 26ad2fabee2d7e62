// A projection shared by all rows beside low-rank adapters, one of many for each row (bnn_lowrank):
//
//   y_r = W x_r + bias + h_r B_a^T,   h_r = s_a A_a x_r,   a = slot[r] (none where it is outside [0, slots))
//
// W [N][K], A [slots][rank][K], B [slots][N][rank]; sums in fp32. Two launches: h (k_lowrank_down), then y in one of three
// forms by the number of rows (one launch for one row); the second launch starts while the first runs (programmatic
// dependent launch) and waits for h only where it is used, after its sums over K.
#include <cuda.h>
#include <cuda_runtime.h>

#include "bnn_kernels.h"
#include "seq.cuh"
#include "smem_attr.cuh"
#include "sync.cuh"
#include "tc16.cuh"

namespace bnn {
namespace {

// D (16 x 8) += A (16 x 16) B (16 x 8), fp32 sums
template <int T>
__device__ __forceinline__ void mma_sync(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (T == 1)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ldg16(const void *p, bool in) {
  return in ? __ldg(reinterpret_cast<const uint4 *>(p)) : make_uint4(0, 0, 0, 0);
}

// ------------------------------------------------------------------ h = s_a A_a x
//
// One CTA per (16 MR rows, one of the adapters among them): the rows against the adapter's rank rows with warp-level matrix
// instructions (a product of 16 rows is too small for a 128-row tile, and bound by reading A and x), K in steps of 32
// dealt to 8 warps, their sums joined in shared memory in warp order. A lane's 16 bytes are 8 consecutive k of a row: the
// two instructions of a step take them in the same order from both operands, so their k are a permutation of the
// layout's, the same for both. Rows of other adapters are computed and dropped. Bound by latency: K over 8 warps is a
// few rounds of loads (9001 rows of 1536, rank 32, 1200 rows an adapter: 27 us, 1.1 TB/s).
constexpr int kDownRows = 16;

template <int T, int RT, int MR>  // RT: 8-wide tiles of the rank
__global__ void __launch_bounds__(256) k_lowrank_down(int rows, int K, const elem_t<T> *x, long long ldx,
                                                      const int32_t *slot, int slots, int rank, const elem_t<T> *A,
                                                      const float *scale, float *hid) {
  constexpr int R = kDownRows * MR;
  __shared__ float red[8][R][RT * 8 + 1];
  __shared__ int s_slot[R];
  wait_launch_before();  // the rows may be another launch's, and h is still read by this operator's last
  launch_dependents();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, q = lane % 4;
  const long long r0 = (long long)blockIdx.x * R;
  if (threadIdx.x < R) {
    int s = r0 + threadIdx.x < rows ? slot[r0 + threadIdx.x] : -1;
    s_slot[threadIdx.x] = s < slots ? s : -1;
  }
  __syncthreads();
  const int mine = lane < R ? s_slot[lane] : -1;
  // the first row of each adapter here
  const unsigned same = __match_any_sync(0xffffffffu, mine);
  unsigned first = __ballot_sync(0xffffffffu, mine >= 0 && __ffs(same) - 1 == lane);
  for (int e = 0; first; first &= first - 1, e++) {
    if (e % (int)gridDim.y != (int)blockIdx.y) continue;
    const int s = s_slot[__ffs(first) - 1];
    const elem_t<T> *a = A + (long long)s * rank * K;
    float acc[MR][RT][4] = {};
#pragma unroll(RT <= 2 ? 6 / MR + 1 : RT <= 4 ? 3 : 2)
    for (int k0 = 32 * warp; k0 < K; k0 += 256) {
      const int k = k0 + 8 * q;
      uint4 xa[MR], xb[MR];
#pragma unroll
      for (int m = 0; m < MR; m++) {
        const long long r = r0 + 16 * m + g;
        xa[m] = ldg16(x + r * ldx + k, r < rows && k < K);
        xb[m] = ldg16(x + (r + 8) * ldx + k, r + 8 < rows && k < K);
      }
#pragma unroll
      for (int j = 0; j < RT; j++) {
        const uint4 b = ldg16(a + (long long)(8 * j + g) * K + k, 8 * j + g < rank && k < K);
#pragma unroll
        for (int m = 0; m < MR; m++) {
          mma_sync<T>(acc[m][j], xa[m].x, xb[m].x, xa[m].y, xb[m].y, b.x, b.y);
          mma_sync<T>(acc[m][j], xa[m].z, xb[m].z, xa[m].w, xb[m].w, b.z, b.w);
        }
      }
    }
    __syncthreads();  // the sums of the adapter before have been read
#pragma unroll
    for (int m = 0; m < MR; m++)
#pragma unroll
      for (int j = 0; j < RT; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) red[warp][16 * m + g + 8 * (i / 2)][8 * j + 2 * q + i % 2] = acc[m][j][i];
    __syncthreads();
    const float f = scale ? scale[s] : 1.f;
    for (int i = threadIdx.x; i < R * rank; i += 256) {
      const int r = i / rank, c = i % rank;
      if (s_slot[r] != s) continue;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < 8; w++) v += red[w][r][c];
      hid[(r0 + r) * rank + c] = f * v;
    }
  }
}

// ------------------------------------------------------------------ up to 16 rows
//
// Bound by reading W (and the adapters' B) once, and by latency. One CTA per 16 rows of W: warp-level matrix
// instructions with W as the 16-row operand and 8 NT rows of x as the other, K dealt to 8 warps as above; the warps' sums
// are joined in shared memory, then each lane takes some rows' outputs of one column and adds their rank products with B
// from the rows' adapters (neighbouring lanes' rows of B are neighbours in memory; the loads of all of a lane's outputs
// are in flight together, the first of them before the wait for h).
// kOwn: the CTA forms h of its one row itself, while W is on its way: a second read of A from L2 by every CTA in place of
// a launch and its end (1 row, 1024 x 1024, calls one after another: 7.5 us, with the launch 9.7; 2 rows: 17.3 us, with the
// launch 11.3). 16 rows of W a CTA: with 32, which halve the reads of x, 8 rows of 6522 x 1024 took 15.4 us in place of
// 13.3. Against the next form at 16 rows: 14.2 us, 19.5 (6522 x 1024), 11.9 and 13.3 (1024 x 1024).
constexpr int kFewRows = 16, kOwnRows = 1;

template <int T, int OT, int NT, bool kOwn>
__global__ void __launch_bounds__(256) k_lowrank_few(const bnnk_lowrank_args p) {
  constexpr int P = 8 * NT + 1, CN = 16;
  __shared__ float red[8][CN][P];
  __shared__ __align__(16) float s_h[kOwn ? kOwnRows : 1][64];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, q = lane % 4;
  const int n0 = blockIdx.x * CN, K = p.K, rank = p.rank;
  if (kOwn) wait_launch_before();  // the only launch; else it follows the one that forms h, which has waited
  launch_dependents();
  const elem_t<T> *W = (const elem_t<T> *)p.w, *x = (const elem_t<T> *)p.x, *B = (const elem_t<T> *)p.b;
  float acc[NT][4] = {};
#pragma unroll 4
  for (int k0 = 32 * warp; k0 < K; k0 += 256) {
    const int k = k0 + 8 * q, n = n0 + g;
    const uint4 wa = ldg16(W + (long long)n * p.ldw + k, n < p.N && k < K);
    const uint4 wb = ldg16(W + (long long)(n + 8) * p.ldw + k, n + 8 < p.N && k < K);
#pragma unroll
    for (int j = 0; j < NT; j++) {
      const uint4 b = ldg16(x + (8 * j + g) * p.ldx + k, 8 * j + g < p.rows && k < K);
      mma_sync<T>(acc[j], wa.x, wb.x, wa.y, wb.y, b.x, b.y);
      mma_sync<T>(acc[j], wa.z, wb.z, wa.w, wb.w, b.z, b.w);
    }
  }
#pragma unroll
  for (int j = 0; j < NT; j++)
#pragma unroll
    for (int e = 0; e < 4; e++) red[warp][g + 8 * (e / 2)][8 * j + 2 * q + e % 2] = acc[j][e];
  constexpr int OUTS = (8 * NT * CN + 255) / 256, RSTEP = 256 / CN;  // a lane's rows: r0, r0 + RSTEP, ..
  const int c = threadIdx.x % CN, r0 = threadIdx.x / CN, n = n0 + c;
  float u[OUTS];
  int s[OUTS];
#pragma unroll
  for (int o = 0; o < OUTS; o++) {
    const int r = r0 + o * RSTEP;
    u[o] = 0.f;
    s[o] = p.slot && r < p.rows && n < p.N ? p.slot[r] : -1;
    if (s[o] >= p.slots) s[o] = -1;
  }
  if (kOwn) {
    for (int r = 0; r < p.rows; r++) {
      const int sr = p.slot[r];
      if (sr < 0 || sr >= p.slots) continue;
      const elem_t<T> *a = (const elem_t<T> *)p.a + (long long)sr * rank * K;
      float h[8] = {};  // rank indexes warp, warp + 8, ..
      for (int k = 8 * lane; k < K; k += 256) {
        float xv[8];
        load_elems<T, 8>(x + r * p.ldx + k, xv);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          if (warp + 8 * j >= rank) break;
          float av[8];
          load_elems<T, 8>(a + (long long)(warp + 8 * j) * K + k, av);
#pragma unroll
          for (int e = 0; e < 8; e++) h[j] = fmaf(xv[e], av[e], h[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if (warp + 8 * j >= rank) break;
#pragma unroll
        for (int o = 16; o; o >>= 1) h[j] += __shfl_xor_sync(0xffffffffu, h[j], o);
        if (lane == 0) s_h[r][warp + 8 * j] = h[j] * (p.scale ? p.scale[sr] : 1.f);
      }
    }
  }
  __syncthreads();
  if (p.slot) {
    for (int e = 0; e < rank; e += 8) {
      uint4 b[OUTS];
#pragma unroll
      for (int o = 0; o < OUTS; o++) b[o] = ldg16(B + ((long long)s[o] * p.N + n) * rank + e, s[o] >= 0);
      if (!kOwn && e == 0) wait_launch_before();
#pragma unroll
      for (int o = 0; o < OUTS; o++) {
        if (s[o] < 0) continue;
        const int r = r0 + o * RSTEP;
        const float *h = kOwn ? s_h[r] + e : p.hid + (long long)r * rank + e;
        const float4 h0 = *reinterpret_cast<const float4 *>(h), h1 = *reinterpret_cast<const float4 *>(h + 4);
        const float2 b0 = unpack2<T>(b[o].x), b1 = unpack2<T>(b[o].y), b2 = unpack2<T>(b[o].z), b3 = unpack2<T>(b[o].w);
        u[o] = fmaf(h0.x, b0.x, u[o]); u[o] = fmaf(h0.y, b0.y, u[o]);
        u[o] = fmaf(h0.z, b1.x, u[o]); u[o] = fmaf(h0.w, b1.y, u[o]);
        u[o] = fmaf(h1.x, b2.x, u[o]); u[o] = fmaf(h1.y, b2.y, u[o]);
        u[o] = fmaf(h1.z, b3.x, u[o]); u[o] = fmaf(h1.w, b3.y, u[o]);
      }
    }
  }
  const float bias = p.bias && n < p.N ? p.bias[n] : 0.f;
#pragma unroll
  for (int o = 0; o < OUTS; o++) {
    const int r = r0 + o * RSTEP;
    if (r >= p.rows || n >= p.N) continue;
    float v = bias;
#pragma unroll
    for (int w = 0; w < 8; w++) v += red[w][c][r];
    ((elem_t<OT> *)p.y)[r * p.ldy + n] = Elem<OT>::put(v + u[o]);
  }
}

// ------------------------------------------------------------------ 17 to 128 rows
//
// Still bound by reading W and, with an adapter a row, B: a tcgen05 tile of the (up to 64 of 128) rows and 16 GR columns a
// CTA, x and W streamed by TMA through a ring deep enough for the memory's latency, one thread issuing. Meanwhile 8 warps
// load the rows of B that the tile's outputs need (a thread 4 rows' outputs in each group of 16 columns), wait for h, and
// form the rank products in fp32 on the CUDA cores (with an adapter a row there is nothing for a matrix instruction to
// share); the accumulators then come from TMEM through shared memory to the threads that hold them. Four accumulators take
// a stage's four steps of 16: the tensor cores' fp32 sums lose a little at every step (K 1024 in one chain was 6.9e-7 off
// in fp32 outputs, against 2.6e-7 for a plain fp32 sum), so the chains are kept short.
// Class head of 64 stations with an adapter each (64 x 1024 x 6522, rank 16, fp32 logits): 14 us.
// More rows than 64 take one CTA per 64 of them. The many-row form gives each adapter of a tile its own steps; an adapter a
// row is its worst case, one adapter its best (1024 x 6522, rank 32, bf16 to fp32, cold caches, us, this form / that one: 128
// rows with an adapter each 48 / 143, 8 rows each 38 / 39, 64 each 38 / 26; 300 rows 91 / 206, 65 / 46, 63 / 28; 512 rows 136 /
// 296, 97 / 58, 97 / 30; fp16's that one 128 rows 108, 36, 26). 128 rows are the middle.
constexpr int kMidRows = 64, kMidMost = 128, kMidThreads = 320, kMidStages = 8;

struct MidArgs {
  bnnk_lowrank_args p;
  int nkb, stages;
  int *err;
};

template <int T, int OT, int GR>
__global__ void __launch_bounds__(kMidThreads, 1) k_lowrank_mid(const __grid_constant__ CUtensorMap mx,
                                                               const __grid_constant__ CUtensorMap mw, const MidArgs a) {
  constexpr int BN = 16 * GR, RI = kMidRows / 16;
  extern __shared__ uint8_t dsmem[];
  __shared__ __align__(8) unsigned long long b_full[kMidStages], b_empty[kMidStages], b_acc, b_out;
  __shared__ uint32_t tmem_s;
  __shared__ volatile int abort_s;
  __shared__ float s_y[kMidRows][BN + 1];
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const bnnk_lowrank_args &p = a.p;
  constexpr uint32_t a_bytes = 128 * 128, stage = (128 + BN) * 128, tmem_cols = BN == 48 ? 256 : 4 * BN;
  const int S = a.stages, n0 = blockIdx.x * BN, m0 = blockIdx.y * kMidRows;
  launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; s++) { mbar_init(smem_u32(&b_full[s]), 1); mbar_init(smem_u32(&b_empty[s]), 1); }
    mbar_init(smem_u32(&b_acc), 1);
    mbar_init(smem_u32(&b_out), 8);
    abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)),
                 "r"(tmem_cols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_s, 0), base = (smem_u32(dsmem) + 1023u) & ~1023u;
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
  if (warp == 0) {
    for (int kb = 0; kb < a.nkb; kb++) {
      const int s = kb % S;
      if (kb >= S && !wait(b_empty[s], (kb / S - 1) & 1, BNNK_ERR_TMA_WAIT)) break;
      const uint32_t st = base + s * stage, bar = smem_u32(&b_full[s]);
      if (elect_one()) {
        mbar_expect_tx(bar, kMidRows * 128 + BN * 128);  // the rows past 64 of the A tile are never written nor used
        tma_load_2d(st, &mx, bar, kb * 64, m0);
        tma_load_2d(st + a_bytes, &mw, bar, kb * 64, n0);
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = idesc_16(T - 1, BN, 0, 0);
    bool ok = true;
    for (int kb = 0; kb < a.nkb && ok; kb++) {
      const int s = kb % S;
      if (!(ok = wait(b_full[s], (kb / S) & 1, BNNK_ERR_MMA_WAIT))) break;
      tc_fence_after();
      const uint64_t da = smem_desc<128>(base + s * stage), db = smem_desc<128>(base + s * stage + a_bytes);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 4; kk++) mma16_ss(tmem + kk * BN, da + kk * 2, db + kk * 2, idesc, kb != 0);
        mma_commit(smem_u32(&b_empty[s]));
      }
    }
    if (ok && elect_one()) mma_commit(smem_u32(&b_acc));
  } else {
    const int tid = threadIdx.x - 64, c = tid % 16, r0 = m0 + tid / 16, rank = p.rank;
    const elem_t<T> *B = (const elem_t<T> *)p.b;
    float u[GR][RI] = {};
    int s[RI];
    if (p.slot) {
#pragma unroll
      for (int i = 0; i < RI; i++) {
        s[i] = r0 + 16 * i < p.rows ? p.slot[r0 + 16 * i] : -1;
        if (s[i] >= p.slots) s[i] = -1;
      }
      for (int e = 0; e < rank; e += 16) {  // 16 of the rank at a time; a rank of 8 more ends in a half
        uint4 b[GR][RI][2];
#pragma unroll
        for (int i = 0; i < RI; i++)
#pragma unroll
          for (int gr = 0; gr < GR; gr++) {
            const int n = n0 + 16 * gr + c;
            const elem_t<T> *bp = B + ((long long)s[i] * p.N + n) * rank + e;
            b[gr][i][0] = ldg16(bp, s[i] >= 0 && n < p.N);
            b[gr][i][1] = ldg16(bp + 8, s[i] >= 0 && n < p.N && e + 8 < rank);
          }
        if (e == 0) wait_launch_before();
#pragma unroll
        for (int i = 0; i < RI; i++) {
          if (s[i] < 0) continue;
          const float *h = p.hid + (long long)(r0 + 16 * i) * rank + e;
#pragma unroll
          for (int k = 0; k < 2; k++) {
            if (e + 8 * k >= rank) break;
            const float4 h0 = *reinterpret_cast<const float4 *>(h + 8 * k), h1 = *reinterpret_cast<const float4 *>(h + 8 * k + 4);
#pragma unroll
            for (int gr = 0; gr < GR; gr++) {
              const uint4 w = b[gr][i][k];
              const float2 b0 = unpack2<T>(w.x), b1 = unpack2<T>(w.y), b2 = unpack2<T>(w.z), b3 = unpack2<T>(w.w);
              float v = u[gr][i];
              v = fmaf(h0.x, b0.x, v); v = fmaf(h0.y, b0.y, v); v = fmaf(h0.z, b1.x, v); v = fmaf(h0.w, b1.y, v);
              v = fmaf(h1.x, b2.x, v); v = fmaf(h1.y, b2.y, v); v = fmaf(h1.z, b3.x, v); v = fmaf(h1.w, b3.y, v);
              u[gr][i] = v;
            }
          }
        }
      }
    }
    bool ok = wait(b_acc, 0, BNNK_ERR_EPI_WAIT);
    if (ok) {
      tc_fence_after();
      const int qd = warp % 4;
      if (qd < kMidRows / 32)  // the quarters that hold rows; the two warps of one share the groups
        for (int gr = (warp - 2) / 4; gr < GR; gr += 2) {
          const uint32_t tq = tmem + 16 * gr + ((uint32_t)(32 * qd) << 16);
          uint32_t x[16], y[16];
          float v[16];
          tmem_ld16(tq, x);
          tmem_ld16(tq + BN, y);
          tmem_wait_ld(x, y);
#pragma unroll
          for (int j = 0; j < 16; j++) v[j] = __uint_as_float(x[j]) + __uint_as_float(y[j]);
          tmem_ld16(tq + 2 * BN, x);
          tmem_ld16(tq + 3 * BN, y);
          tmem_wait_ld(x, y);
#pragma unroll
          for (int j = 0; j < 16; j++) s_y[32 * qd + lane][16 * gr + j] = v[j] + (__uint_as_float(x[j]) + __uint_as_float(y[j]));
        }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&b_out));
      ok = wait(b_out, 0, BNNK_ERR_EPI_WAIT);
    }
    if (ok) {
#pragma unroll
      for (int gr = 0; gr < GR; gr++) {
        const int n = n0 + 16 * gr + c;
        if (n >= p.N) continue;
        const float bias = p.bias ? p.bias[n] : 0.f;
#pragma unroll
        for (int i = 0; i < RI; i++) {
          const int r = r0 + 16 * i;
          if (r < p.rows) ((elem_t<OT> *)p.y)[(long long)r * p.ldy + n] = Elem<OT>::put(s_y[r - m0][16 * gr + c] + bias + u[gr][i]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols));
}

// ------------------------------------------------------------------ many rows
//
// A tcgen05 GEMM of 128-row tiles, y's accumulators in TMEM, with the adapters as more steps of the sum: for each
// adapter among the tile's rows (the list that 4 warps make from the rows' slots while W's steps run) the A operand is h
// in the rows of that adapter and zero in the others, the B operand B_a. h is fp32 and goes as 16-bit parts: three for
// bf16 (all 24 bits), two for fp16, which leave 2^-25 at most: 2^-23 of a row's largest |h| from 0.25 up. Slots of 64 / RB
// adapters share a stage (RB: the rank rounded up to 16, 32 or 64, a row of that many bytes swizzled as such).
// A tile of fp16 rows with an |h| past the type, or a row whose largest is below 0.25 (two parts would leave 1.7e-5 of an h of
// 1e-3), has kind::tf32 steps instead: h as two parts of 11 bits, which leave 2^-22 of it whatever its size, and B's values
// exact. 16 columns of the adapters back to back are a step: a row of A is 16 first parts and 16 second ones, a row of B 16
// values for both, made of the 16-bit ones that TMA puts behind them. 9001 x 1536 x 6144, rank 32, runs of 700, cold caches:
// 173 us, with 16-bit parts 158; 300 rows with an adapter each, 1024 x 6522, rank 16: 127 and 79.
//
// A NaN or an infinity in an adapter's B meets the zeros of the rows of others in the same products: y that is not finite
// where the row's own x and h are is formed again in fp32 when it is stored (row_product).
//
// One persistent CTA per SM, column tiles fastest. Warp 0 streams 64-wide steps of x and W, then the adapters' B, into a
// ring by TMA; warp 1 issues the MMAs into one of two accumulators; warps 2 .. 5 make the list and h's operand tiles;
// warps 6 .. 13 store y: accumulator rows through shared memory, so that a store covers 32 neighbouring words of a row at
// any row alignment; 16 bytes a lane where y's rows are whole 16 bytes.
// Bound by reading x and W from L2 (48 KB for 1040 cycles of products at 256 columns). 9001 x 1536 x 6144, fp16, calls apart
// with cold caches: 126 us without adapters, 1.35 PFLOP/s (the library's product: 123 us); with adapters of 700 rows and rank
// 32 158, 27 of them to form h; one call after another, at the clocks that lasting load leaves, 186. Tiles of 256 rows, which
// read half of W, left no TMEM for a second accumulator: 241 us in place of 212 at the time. Adapters that change from row to
// row: 331 us (bf16 373).
constexpr int kLrThreads = 448;
constexpr int kLrStages = 8;
constexpr int kLrPad = 20;  // words a row of the stores' shared memory: blocks of 16 words; 16-byte accesses meet no bank twice

struct LrArgs {
  bnnk_lowrank_args p;
  int nkb, bn, n_tiles, tiles, stages, tmem_cols;
  int na, acc_cols;  // accumulators of a tile (a power of two, the sum's steps in turn) and their columns
  int *err;
};

// the nearest tf32 (11 bits), ties away from zero; not for a NaN whose payload would carry over
__device__ __forceinline__ float to_tf32(float v) { return __uint_as_float((__float_as_uint(v) + 0x1000u) & 0xffffe000u); }

__device__ __forceinline__ bool any_not_finite(const float (&v)[8]) {
  float z = 0.f;
#pragma unroll
  for (int c = 0; c < 8; c++) z = fmaf(v[c], 0.f, z);
  return z != 0.f;
}
// whether row r's own inputs, its h or without an adapter its x, hold a NaN or an infinity
template <int T>
__device__ __forceinline__ bool row_not_finite(const bnnk_lowrank_args &p, long long r, int s) {
  float v[8];
  bool bad = false;
  if (s >= 0)
    for (int e = 0; e < p.rank; e += 8) {
      load_elems<0, 8>(p.hid + r * p.rank + e, v);
      bad |= any_not_finite(v);
    }
  else
    for (int k = 0; k < p.K; k += 8) {
      load_elems<T, 8>((const elem_t<T> *)p.x + r * p.ldx + k, v);
      bad |= any_not_finite(v);
    }
  return bad;
}
// y of row r, whose adapter is s, and column n
template <int T>
__device__ __forceinline__ float row_product(const bnnk_lowrank_args &p, long long r, int s, int n) {
  float sum = p.bias ? p.bias[n] : 0.f;
#pragma unroll 1
  for (int k = 0; k < p.K; k += 8) {
    float xv[8], wv[8];
    load_elems<T, 8>((const elem_t<T> *)p.x + r * p.ldx + k, xv);
    load_elems<T, 8>((const elem_t<T> *)p.w + n * p.ldw + k, wv);
#pragma unroll
    for (int c = 0; c < 8; c++) sum = fmaf(xv[c], wv[c], sum);
  }
  float u = 0.f;
  if (s >= 0)
#pragma unroll 1
    for (int e = 0; e < p.rank; e += 8) {
      float h[8], b[8];
      load_elems<0, 8>(p.hid + r * p.rank + e, h);
      load_elems<T, 8>((const elem_t<T> *)p.b + ((long long)s * p.N + n) * p.rank + e, b);
#pragma unroll
      for (int c = 0; c < 8; c++) u = fmaf(h[c], b[c], u);
    }
  return sum + u;
}

template <int T, int OT, int RB>
__global__ void __launch_bounds__(kLrThreads, 1) k_lowrank_many(const __grid_constant__ CUtensorMap mx,
                                                               const __grid_constant__ CUtensorMap mw,
                                                               const __grid_constant__ CUtensorMap mb,
                                                               const __grid_constant__ CUtensorMap mb8, const LrArgs a) {
  constexpr int PARTS = T == 2 ? 3 : 2, GS = 64 / RB;  // adapters a stage
  extern __shared__ uint8_t dsmem[];
  __shared__ __align__(8) unsigned long long b_full[kLrStages], b_empty[kLrStages], b_acc[2], b_accempty[2], b_list[2],
      b_listempty[2], b_place[kLrStages], b_base;
  __shared__ uint32_t tmem_s;
  __shared__ volatile int abort_s;
  __shared__ int s_n[2], s_list[2][128];
  __shared__ volatile uint8_t s_wide[2][4];  // tf32 steps, as warps 2 .. 5 found for their rows
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const bnnk_lowrank_args &p = a.p;
  const int S = a.stages, bn = a.bn;
  launch_dependents();
  const uint32_t a_bytes = 128 * 128, stage = (128 + bn) * 128;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; s++) { mbar_init(smem_u32(&b_full[s]), 5); mbar_init(smem_u32(&b_empty[s]), 1); mbar_init(smem_u32(&b_place[s]), 1); }
    for (int g = 0; g < 2; g++) {
      mbar_init(smem_u32(&b_acc[g]), 1);
      mbar_init(smem_u32(&b_accempty[g]), 8);
      mbar_init(smem_u32(&b_list[g]), 4);
      mbar_init(smem_u32(&b_listempty[g]), 6);
    }
    mbar_init(smem_u32(&b_base), 1);
    abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)),
                 "r"(a.tmem_cols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_s, 0), base = (smem_u32(dsmem) + 1023u) & ~1023u;
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
  const bool adapters = p.slot != nullptr;
  // a place in the ring of stages
  struct Place {
    int s = 0, parity = 0, used = 0;
    __device__ __forceinline__ void next(int S) {
      if (++s == S) { s = 0; parity ^= 1; used = 1; }
    }
  } at;
  // 8 columns of the list's adapters back to back: the adapter's place in the list, the columns' in the adapter
  struct Columns {
    int e = 0, off = 0;
    __device__ __forceinline__ void next(int rank) {
      if ((off += 8) == rank) off = 0, e++;
    }
  };
  int lt = 0;       // tiles done
  bool ok = true;
  // the stages that the tile's adapters take, and their kind (after list lt % 2 is made)
  auto extra = [&](int &n, bool &wide) {
    n = 0;
    wide = false;
    if (!adapters) return true;
    const int g = lt & 1;
    if (!wait(b_list[g], (lt >> 1) & 1, BNNK_ERR_TMA_WAIT)) return false;
    wide = T == 1 && (s_wide[g][0] | s_wide[g][1] | s_wide[g][2] | s_wide[g][3]);
    n = wide ? (s_n[g] * p.rank + 15) / 16 : (s_n[g] + GS - 1) / GS * PARTS;
    return true;
  };
  auto list_read = [&]() {
    __syncwarp();
    if (adapters && lane == 0) mbar_arrive(smem_u32(&b_listempty[lt & 1]));
  };

  if (warp == 0) {
    for (int t = blockIdx.x; t < a.tiles && ok; t += gridDim.x, lt++) {
      const int r0 = t / a.n_tiles * 128, n0 = t % a.n_tiles * bn, g = lt & 1;
      for (int kb = 0; kb < a.nkb; kb++, at.next(S)) {
        if (at.used && !(ok = wait(b_empty[at.s], at.parity ^ 1, BNNK_ERR_TMA_WAIT))) break;
        const uint32_t st = base + at.s * stage, bar = smem_u32(&b_full[at.s]);
        if (elect_one()) {
          mbar_expect_tx(bar, stage);
          asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], 4;" ::"r"(bar) : "memory");
          tma_load_2d(st, &mx, bar, kb * 64, r0);
          tma_load_2d(st + a_bytes, &mw, bar, kb * 64, n0);
        }
      }
      int n;
      bool wide;
      if (!ok || !(ok = extra(n, wide))) break;
      // the adapters' places: B here, b_place tells the warps that make A that a place is free for them (b_empty could not:
      // a parity tells one use from the next, not from the one after) and, for tf32 steps, that its 16-bit B is there
      Columns col;
      for (int k = 0; k < n; k++, at.next(S)) {
        if (at.used && !(ok = wait(b_empty[at.s], at.parity ^ 1, BNNK_ERR_TMA_WAIT))) break;
        const uint32_t st = base + at.s * stage + a_bytes, full = smem_u32(&b_full[at.s]), place = smem_u32(&b_place[at.s]);
        if (!wide) {
          const int e0 = k / PARTS * GS, here = min(GS, s_n[g] - e0);
          if (elect_one()) {
            mbar_arrive(place);
            mbar_expect_tx(full, here * bn * RB * 2);
            for (int e = 0; e < here; e++) tma_load_3d(st + e * bn * RB * 2, &mb, full, 0, n0, s_list[g][e0 + e]);
          }
        } else {
          const Columns c0 = col;
          col.next(p.rank);
          const Columns c1 = col;
          col.next(p.rank);
          const bool both = c1.e < s_n[g];
          if (elect_one()) {
            mbar_arrive(full);
            mbar_expect_tx(place, bn * (both ? 32 : 16));
            tma_load_3d(st + bn * 64, &mb8, place, c0.off, n0, s_list[g][c0.e]);
            if (both) tma_load_3d(st + bn * 80, &mb8, place, c1.off, n0, s_list[g][c1.e]);
          }
        }
      }
      list_read();
    }
  } else if (warp == 1) {
    const uint32_t idesc = idesc_16(T - 1, bn, 0, 0);
    int base_parity = 0;
    for (int t = blockIdx.x; t < a.tiles && ok; t += gridDim.x, lt++) {
      const int g = lt & 1;
      if (lt >= 2 && !(ok = wait(b_accempty[g], (lt / 2 - 1) & 1, BNNK_ERR_MMA_WAIT))) break;
      const uint32_t acc = tmem + g * a.na * a.acc_cols;
      for (int kb = 0; kb < a.nkb; kb++, at.next(S)) {
        if (!(ok = wait(b_full[at.s], at.parity, BNNK_ERR_MMA_WAIT))) break;
        tc_fence_after();
        const uint64_t da = smem_desc<128>(base + at.s * stage), db = smem_desc<128>(base + at.s * stage + a_bytes);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 4; kk++)
            mma16_ss(acc + (kk & (a.na - 1)) * a.acc_cols, da + kk * 2, db + kk * 2, idesc, kb != 0 || kk >= a.na);
          mma_commit(smem_u32(&b_empty[at.s]));
        }
      }
      int n;
      bool wide;
      if (!ok || !(ok = extra(n, wide))) break;
      const int used = n ? s_n[g] : 0;
      list_read();
      if (T == 1 && wide) {  // instructions of another kind: nothing says that they follow W's into the sum, so W's end first
        if (elect_one()) mma_commit(smem_u32(&b_base));
        if (!(ok = wait(b_base, base_parity, BNNK_ERR_MMA_WAIT))) break;
        base_parity ^= 1;
        tc_fence_after();
      }
      for (int k = 0; k < n; k++, at.next(S)) {
        if (!(ok = wait(b_full[at.s], at.parity, BNNK_ERR_MMA_WAIT))) break;
        tc_fence_after();
        const uint32_t st = base + at.s * stage;
        if (T == 1 && wide) {
          const uint64_t da = smem_desc<128>(st), db = smem_desc<64>(st + a_bytes);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 4; kk++) mma32_ss(acc, da + kk * 2, db + (kk & 1) * 2, idesc_tf32(bn), 1);
            mma_commit(smem_u32(&b_empty[at.s]));
          }
          continue;
        }
        const int here = min(GS, used - k / PARTS * GS);
        const uint64_t da = smem_desc<2 * RB>(st), db = smem_desc<2 * RB>(st + a_bytes);
        if (elect_one()) {
          for (int e = 0; e < here; e++)
#pragma unroll
            for (int kk = 0; kk < RB / 16; kk++)
              mma16_ss(acc, da + e * (128 * RB * 2 >> 4) + kk * 2, db + e * (bn * RB * 2 >> 4) + kk * 2, idesc, 1);
          mma_commit(smem_u32(&b_empty[at.s]));
        }
      }
      if (ok && elect_one()) mma_commit(smem_u32(&b_acc[g]));
    }
  } else if (warp < 6) {
    if (adapters) {
      const int row = threadIdx.x - 64;
      uint32_t place_parity = 0;  // by place
      auto wait_place = [&]() {
        if (!(ok = wait(b_place[at.s], (place_parity >> at.s) & 1, BNNK_ERR_TMA_WAIT))) return false;
        place_parity ^= 1u << at.s;
        return true;
      };
      wait_launch_before();
      for (int t = blockIdx.x; t < a.tiles && ok; t += gridDim.x, lt++) {
        const int r0 = t / a.n_tiles * 128, g = lt & 1;
        if (lt >= 2 && !(ok = wait(b_listempty[g], (lt / 2 - 1) & 1, BNNK_ERR_TMA_WAIT))) break;
        // the tile's adapters, in the order of their first rows: every warp makes the whole list from all 128 slots and
        // writes its own part of it
        int all[4], mine = -1, count = 0, before = 0;
        unsigned firsts[4];
#pragma unroll
        for (int w = 0; w < 4; w++) {
          const int r = r0 + 32 * w + lane;
          int s = r < p.rows ? p.slot[r] : -1;
          if (s >= p.slots) s = -1;
          all[w] = s;
          if (w == warp - 2) mine = s;
        }
#pragma unroll
        for (int w = 0; w < 4; w++) {
          const unsigned same = __match_any_sync(0xffffffffu, all[w]);  // every lane takes part, those without an adapter too
          bool first = all[w] >= 0 && __ffs(same) - 1 == lane;
#pragma unroll
          for (int v = 0; v < w; v++) {
            // neighbouring rows are mostly one request's: 32 rows all the same need one comparison
            const int s0 = __shfl_sync(0xffffffffu, all[v], 0);
            if (__all_sync(0xffffffffu, all[v] == s0)) first &= s0 != all[w];
            else
              for (int l = 0; l < 32; l++) first &= __shfl_sync(0xffffffffu, all[v], l) != all[w];
          }
          firsts[w] = __ballot_sync(0xffffffffu, first);
          if (w < warp - 2) before += __popc(firsts[w]);
          count += __popc(firsts[w]);
        }
        const unsigned own = firsts[0] * (warp == 2) | firsts[1] * (warp == 3) | firsts[2] * (warp == 4) | firsts[3] * (warp == 5);
        if ((own >> lane) & 1) s_list[g][before + __popc(own & ((1u << lane) - 1))] = mine;
        if (warp == 2 && lane == 0) s_n[g] = count;
        // this row's h, read while W's steps run
        float h[RB], most = 0.f;
#pragma unroll
        for (int c = 0; c < RB; c += 4) {
          float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
          if (mine >= 0 && c < p.rank) u = *reinterpret_cast<const float4 *>(p.hid + (long long)(r0 + row) * p.rank + c);
          h[c] = u.x, h[c + 1] = u.y, h[c + 2] = u.z, h[c + 3] = u.w;
        }
        if constexpr (T == 1) {
#pragma unroll
          for (int c = 0; c < RB; c++) most = fmaxf(most, fabsf(h[c]));
          const bool wide = (most > 0.f && most < 0.25f) || (most > 65504.f && most < __int_as_float(0x7f800000));
          const bool any = __any_sync(0xffffffffu, wide);
          if (lane == 0) s_wide[g][warp - 2] = any;
        }
        __threadfence_block();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&b_list[g]));
        int steps;
        bool wide;
        if (!(ok = extra(steps, wide))) break;
        // the ring's places of W's steps
        for (int kb = 0; kb < a.nkb; kb++) at.next(S);
        if constexpr (T == 1)
          if (wide) {
#pragma unroll
            for (int c = 0; c < RB; c++) h[c] = h[c] == h[c] ? h[c] : __uint_as_float(0x7fc00000u);  // for to_tf32
            uint8_t *ring = dsmem + (base - smem_u32(dsmem));
            Columns col;
#pragma unroll 1
            for (int k = 0; k < steps; k++, at.next(S)) {
              if (!wait_place()) break;
              uint8_t *st = ring + at.s * stage;
              int s[2], off[2];
              uint4 w[2][2];
#pragma unroll
              for (int j = 0; j < 2; j++, col.next(p.rank)) {
                s[j] = col.e < count ? s_list[g][col.e] : -1;
                off[j] = col.off;
#pragma unroll
                for (int q = 0; q < 2; q++) {
                  const int n = row + 128 * q;
                  w[j][q] = make_uint4(0, 0, 0, 0);
                  if (s[j] >= 0 && n < bn) w[j][q] = *reinterpret_cast<const uint4 *>(st + a_bytes + bn * 64 + (j * bn + n) * 16);
                }
              }
              // A: 128 bytes a row, first parts of 16 columns and second ones, 16-byte places with the 128-byte swizzle
#pragma unroll
              for (int j = 0; j < 2; j++) {
                uint8_t *ra = st + row * 128;
                const int sw = (row & 7) * 16;
                const bool on = s[j] >= 0 && s[j] == mine;
                float u[8] = {}, v[8] = {};
                if (__any_sync(0xffffffffu, on)) {
#pragma unroll
                  for (int i = 0; i < RB / 8; i++)
                    if (off[j] == 8 * i) {
#pragma unroll
                      for (int c = 0; c < 8; c++) v[c] = on ? h[8 * i + c] : 0.f;
                    }
#pragma unroll
                  for (int c = 0; c < 8; c++) {
                    u[c] = to_tf32(v[c]);
                    v[c] = to_tf32(v[c] - u[c]);
                  }
                }
#pragma unroll
                for (int i = 0; i < 2; i++) {
                  float4 *first = reinterpret_cast<float4 *>(ra + ((2 * j + i) * 16 ^ sw));
                  float4 *second = reinterpret_cast<float4 *>(ra + ((4 + 2 * j + i) * 16 ^ sw));
                  *first = make_float4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
                  *second = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                }
              }
              // B: 64 bytes a row, the 64-byte swizzle
#pragma unroll
              for (int q = 0; q < 2; q++) {
                const int n = row + 128 * q;
                if (n >= bn) break;
                uint8_t *rb = st + a_bytes + n * 64;
                const int sw = (n >> 1 & 3) * 16;
#pragma unroll
                for (int j = 0; j < 2; j++) {
                  const float2 b0 = unpack2<T>(w[j][q].x), b1 = unpack2<T>(w[j][q].y), b2 = unpack2<T>(w[j][q].z),
                               b3 = unpack2<T>(w[j][q].w);
                  *reinterpret_cast<float4 *>(rb + (2 * j * 16 ^ sw)) = make_float4(b0.x, b0.y, b1.x, b1.y);
                  *reinterpret_cast<float4 *>(rb + ((2 * j + 1) * 16 ^ sw)) = make_float4(b2.x, b2.y, b3.x, b3.y);
                }
              }
              fence_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(smem_u32(&b_full[at.s]));
            }
            if (!ok) break;
            list_read();
            continue;
          }
        for (int e0 = 0; e0 < count && ok; e0 += GS) {
          const int here = min(GS, count - e0);
          int my = -1;  // this row's adapter among the stage's
          for (int e = 0; e < here; e++)
            if (mine >= 0 && s_list[g][e0 + e] == mine) my = e;
#pragma unroll 1
          for (int part = 0; part < PARTS; part++, at.next(S)) {
            if (!wait_place()) break;
            const uint32_t st = base + at.s * stage;
#pragma unroll
            for (int c = 0; c < RB; c += 8) {
              uint32_t z[4] = {0, 0, 0, 0};
              if (my >= 0) {  // a part: what the parts before have left, rounded
#pragma unroll
                for (int i = 0; i < 4; i++) {
                  float &u = h[c + 2 * i], &v = h[c + 2 * i + 1];
                  z[i] = pack2f<T>(u, v);
                  const float2 f = unpack2<T>(z[i]);
                  u -= f.x, v -= f.y;
                }
              }
#pragma unroll 1
              for (int e = 0; e < here; e++) {
                const bool on = e == my;
                uint32_t off = e * 128 * RB * 2 + row * RB * 2 + c * 2;
                off ^= (off >> 3) & (RB == 64 ? 0x70 : RB == 32 ? 0x30 : 0x10);  // the swizzle of 2 RB bytes a row
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(st + off), "r"(on ? z[0] : 0),
                             "r"(on ? z[1] : 0), "r"(on ? z[2] : 0), "r"(on ? z[3] : 0)
                             : "memory");
              }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&b_full[at.s]));
          }
        }
        if (!ok) break;
        list_read();
      }
    }
  } else {
    // y: rows of this warp's TMEM quarter, blocks of 16 words a row alternating between two warps of a quarter
    constexpr int PW = OT == 0 ? 1 : 2, CW = 16 * PW;  // values a word, columns a block
    const int qd = warp % 4, h = (warp - 6) / 4;
    const uint32_t buf = base + S * stage + (warp - 6) * 32 * kLrPad * 4;
    const bool even = PW == 1 || (((uintptr_t)p.y | (uintptr_t)(p.ldy * 2)) & 3) == 0;  // word-aligned rows
    const bool bias16 = p.bias && ((uintptr_t)p.bias & 15) == 0;
    const bool wide = (((uintptr_t)p.y | (uintptr_t)(p.ldy * (4 / PW))) & 15) == 0;  // rows of whole 16 bytes
    for (int t = blockIdx.x; t < a.tiles; t += gridDim.x, lt++) {
      const int r0 = t / a.n_tiles * 128 + 32 * qd, n0 = t % a.n_tiles * bn, g = lt & 1;
      if (!wait(b_acc[g], (lt >> 1) & 1, BNNK_ERR_EPI_WAIT)) break;
      tc_fence_after();
      const uint32_t tq = tmem + g * a.na * a.acc_cols + ((uint32_t)(32 * qd) << 16);
      const int width = min(bn, p.N - n0), rows = min(32, p.rows - r0);
      int own_bad = -1, own = -1;  // this lane's row: row_not_finite (-1: not looked at yet), its adapter
#pragma unroll 1
      for (int c0 = h * CW; c0 < width; c0 += 2 * CW) {
#pragma unroll
        for (int w0 = 0; w0 < PW; w0++) {
          const int c = c0 + 16 * w0;
          if (c >= bn) break;
          uint32_t x[16];
          tmem_ld16(tq + c, x);
          tmem_wait_ld(x);
          float v[16];
#pragma unroll
          for (int j = 0; j < 16; j++) v[j] = __uint_as_float(x[j]);
          if (bias16 && c + 16 <= width) {
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
              const float4 u = __ldg(reinterpret_cast<const float4 *>(p.bias + n0 + c + j));
              v[j] += u.x, v[j + 1] += u.y, v[j + 2] += u.z, v[j + 3] += u.w;
            }
          } else if (p.bias) {
#pragma unroll
            for (int j = 0; j < 16; j++) v[j] += c + j < width ? __ldg(p.bias + n0 + c + j) : 0.f;
          }
          if (OT == 0)
            for (int k = 1; k < a.na; k++) {
              tmem_ld16(tq + k * a.acc_cols + c, x);
              tmem_wait_ld(x);
#pragma unroll
              for (int j = 0; j < 16; j++) v[j] += __uint_as_float(x[j]);
            }
          if (adapters) {
            float z = 0.f;
#pragma unroll
            for (int j = 0; j < 16; j++) z = fmaf(v[j], 0.f, z);
            if (__any_sync(0xffffffffu, z != 0.f)) {
              if (z != 0.f && lane < rows && own_bad < 0) {
                own = p.slot[r0 + lane];
                if (own >= p.slots) own = -1;
                own_bad = row_not_finite<T>(p, r0 + lane, own);
              }
#pragma unroll 1
              for (int j = 0; j < 16 && c + j < width; j++) {
                float u = 0.f;
#pragma unroll
                for (int i = 0; i < 16; i++) u = i == j ? v[i] : u;
                if (lane >= rows || own_bad || u * 0.f == 0.f) continue;
                u = row_product<T>(p, r0 + lane, own, n0 + c + j);
#pragma unroll
                for (int i = 0; i < 16; i++) v[i] = i == j ? u : v[i];
              }
            }
          }
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 16; j += 4 * PW) {
            uint32_t z[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
              z[i] = PW == 1 ? __float_as_uint(v[j + i]) : pack2f<T>(v[j + PW * i], v[j + PW * i + PW - 1]);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(buf + (lane * kLrPad + (16 * w0 + j) / PW) * 4),
                         "r"(z[0]), "r"(z[1]), "r"(z[2]), "r"(z[3])
                         : "memory");
          }
        }
        __syncwarp();
        if (wide && c0 + CW <= width) {
          char *y = (char *)p.y + ((long long)(r0 + lane / 4) * p.ldy + n0 + c0) * (4 / PW) + lane % 4 * 16;
#pragma unroll
          for (int r = lane / 4; r < 32; r += 8, y += 8 * p.ldy * (4 / PW)) {
            uint4 z;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(z.x), "=r"(z.y), "=r"(z.z), "=r"(z.w)
                         : "r"(buf + (r * kLrPad + lane % 4 * 4) * 4)
                         : "memory");
            if (r < rows) *reinterpret_cast<uint4 *>(y) = z;
          }
          __syncwarp();
          continue;
        }
        const int c = c0 + lane % 16 * PW;
        elem_t<OT> *y = (elem_t<OT> *)p.y + (long long)(r0 + lane / 16) * p.ldy + n0 + c;
#pragma unroll 4
        for (int r = lane / 16; r < rows; r += 2, y += 2 * p.ldy) {
          uint32_t z;
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(z) : "r"(buf + (r * kLrPad + lane % 16) * 4) : "memory");
          if constexpr (PW == 1) {
            if (c < width) *y = __uint_as_float(z);
          } else if (even && c + 1 < width) {
            *reinterpret_cast<uint32_t *>(y) = z;
          } else {
            if (c < width) reinterpret_cast<uint16_t *>(y)[0] = (uint16_t)z;
            if (c + 1 < width) reinterpret_cast<uint16_t *>(y)[1] = (uint16_t)(z >> 16);
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&b_accempty[g]));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols));
}

template <int T, int OT, int NT>
cudaError_t few_nt(const bnnk_lowrank_args &p, cudaStream_t st) {
  const dim3 grid((p.N + 15) / 16);
  if (p.slot && p.rows > kOwnRows) return launch_early(k_lowrank_few<T, OT, NT, false>, grid, 256, 0, st, p);
  if (p.slot) return launch_early(k_lowrank_few<T, OT, NT, true>, grid, 256, 0, st, p);
  k_lowrank_few<T, OT, NT, false><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError();
}

template <int T, int OT>
cudaError_t run_few(const bnnk_lowrank_args &p, cudaStream_t st) {
  return p.rows <= 8 ? few_nt<T, OT, 1>(p, st) : few_nt<T, OT, 2>(p, st);
}

template <int T, int OT, int GR>
int mid_groups(const bnnk_lowrank_args &p, int *err, cudaStream_t st) {
  constexpr int BN = 16 * GR;
  constexpr size_t stage = (128 + BN) * 128;
  MidArgs a = {p, (p.K + 63) / 64, kMidStages, err};
  constexpr size_t smem = kMidStages * stage + 1024;
  CUtensorMap mx, mw;
  int e = encode_rows16(&mx, p.x, T == 2, p.K, p.rows, p.ldx, 64, kMidRows, 128);
  if (!e) e = encode_rows16(&mw, p.w, T == 2, p.K, p.N, p.ldw, 64, BN, 128);
  static SmemAttr attr;
  if (!e) e = attr.ensure(k_lowrank_mid<T, OT, GR>, smem);
  if (e) return e;
  const dim3 grid((p.N + BN - 1) / BN, (p.rows + kMidRows - 1) / kMidRows);
  if (p.slot) return launch_early(k_lowrank_mid<T, OT, GR>, grid, kMidThreads, smem, st, mx, mw, a);
  k_lowrank_mid<T, OT, GR><<<grid, kMidThreads, smem, st>>>(mx, mw, a);
  return cudaGetLastError();
}

template <int T, int OT>
int run_mid(const bnnk_lowrank_args &p, int *err, cudaStream_t st) {
  // as few columns a CTA as fill the SMs once, up to 48 (64 rows of 6522 x 1024 with 16, 32, 48: 31.7, 24.0, 21.5 us)
  const int n = (p.N + 15) / 16 * ((p.rows + kMidRows - 1) / kMidRows), sms = num_sms();
  return n <= sms ? mid_groups<T, OT, 1>(p, err, st) : n <= 2 * sms ? mid_groups<T, OT, 2>(p, err, st)
                                                                    : mid_groups<T, OT, 3>(p, err, st);
}

template <int T, int OT, int RB>
int run_many(const bnnk_lowrank_args &p, int *err, cudaStream_t st) {
  LrArgs a = {};
  a.p = p;
  a.err = err;
  a.nkb = (p.K + 63) / 64;
  // fp32 outputs: the tensor cores' chains of fp32 sums kept to about 1024 values of K (one of 1024 was 6.9e-7 off, against
  // 2.6e-7 for a plain fp32 sum), for narrower tiles (2000 rows of 2720, us with 1, 2, 4 accumulators: K 512 25.6, 28.2,
  // 33.8, K 1536 35.8, 37.9, 50.2, K 4096 64.5, 68.9, 105); a 16-bit output's rounding hides them
  a.na = OT != 0 || p.K <= 512 ? 1 : p.K <= 2048 ? 2 : 4;
  // column tiles of at most 256 / na, of equal widths, narrower while there are fewer tiles than SMs
  const int n16 = (p.N + 15) & ~15, mt = (p.rows + 127) / 128, most = 256 / a.na;
  int nt = (n16 + most - 1) / most;
  while ((long long)mt * nt < num_sms() && ((n16 + nt) / (nt + 1) + 15) / 16 * 16 >= 32) nt++;
  a.bn = ((n16 + nt - 1) / nt + 15) & ~15;
  a.n_tiles = (p.N + a.bn - 1) / a.bn;
  if ((long long)mt * a.n_tiles > 0x7fffffffLL) return cudaErrorInvalidValue;
  a.tiles = mt * a.n_tiles;
  a.acc_cols = a.bn <= 32 ? 32 : a.bn <= 64 ? 64 : a.bn <= 128 ? 128 : 256;
  a.tmem_cols = 2 * a.na * a.acc_cols;
  const size_t stage = (size_t)(128 + a.bn) * 128, out = 8 * 32 * kLrPad * 4;
  const int s = (int)((227 * 1024 - 4096 - out) / stage);
  a.stages = s > kLrStages ? kLrStages : s;
  const size_t smem = a.stages * stage + out + 1024;
  CUtensorMap mx, mw, mb, mb8;
  int e = encode_rows16(&mx, p.x, T == 2, p.K, p.rows, p.ldx, 64, 128, 128);
  if (!e) e = encode_rows16(&mw, p.w, T == 2, p.K, p.N, p.ldw, 64, a.bn, 128);
  if (!e) e = encode_slots16(&mb, p.b, T == 2, p.rank, p.N, p.slots, RB, a.bn);
  if (!e) e = encode_slots16(&mb8, p.b, T == 2, p.rank, p.N, p.slots, 8, a.bn);
  static SmemAttr attr;
  if (!e) e = attr.ensure(k_lowrank_many<T, OT, RB>, smem);
  if (e) return e;
  const int grid = a.tiles < num_sms() ? a.tiles : num_sms();
  if (p.slot) return launch_early(k_lowrank_many<T, OT, RB>, dim3(grid), kLrThreads, smem, st, mx, mw, mb, mb8, a);
  k_lowrank_many<T, OT, RB><<<grid, kLrThreads, smem, st>>>(mx, mw, mb, mb8, a);
  return cudaGetLastError();
}

template <int T, int RT, int MR>
cudaError_t down_rows(const bnnk_lowrank_args &p, int adapters, cudaStream_t st) {
  return launch_early(k_lowrank_down<T, RT, MR>, dim3((p.rows + kDownRows * MR - 1) / (kDownRows * MR), adapters), 256, 0, st,
                      p.rows, p.K, (const elem_t<T> *)p.x, p.ldx, p.slot, p.slots, p.rank, (const elem_t<T> *)p.a, p.scale,
                      p.hid);
}

template <int T, int RT>
cudaError_t run_down(const bnnk_lowrank_args &p, cudaStream_t st) {
  // 32-row tiles halve the reads of A; 16 where rows are few, or the sums would not fit (700 rows an adapter, K 1536, rank
  // 32, us for the operator with 16 / 32: 300 rows 30.7 / 24.6, 9001 rows 171 / 164; 64 adapters, K 1024, rank 16, 64 rows
  // 13.6 / 16.6). As many CTAs a tile as its rows can have adapters while the tiles are few, two where they fill the SMs,
  // since most then hold one or two (an adapter a row, 300 rows, 2 / 16: 57 / 35; 700 rows an adapter, 9001 rows 164 / 180)
  const bool small = RT == 8 || p.rows <= kMidMost;
  const int tiles = (p.rows + (small ? 15 : 31)) / (small ? 16 : 32), share = 512 / tiles;
  const int y = share < 2 ? 2 : share > 16 ? 16 : share;
  return small ? down_rows<T, RT, 1>(p, y, st) : down_rows<T, RT, RT == 8 ? 1 : 2>(p, y, st);
}

template <int T>
int run_lowrank(const bnnk_lowrank_args &p, int *err, cudaStream_t st) {
  if (p.slot && p.rows > kOwnRows) {
    const cudaError_t e = p.rank <= 16 ? run_down<T, 2>(p, st) : p.rank <= 32 ? run_down<T, 4>(p, st) : run_down<T, 8>(p, st);
    if (e) return e;
  }
  if (p.rows <= kFewRows) return p.otype == 0 ? run_few<T, 0>(p, st) : run_few<T, T>(p, st);
  if (p.rows <= kMidMost) return p.otype == 0 ? run_mid<T, 0>(p, err, st) : run_mid<T, T>(p, err, st);
  if (p.otype == 0)
    return p.rank <= 16 ? run_many<T, 0, 16>(p, err, st) : p.rank <= 32 ? run_many<T, 0, 32>(p, err, st)
                                                                         : run_many<T, 0, 64>(p, err, st);
  return p.rank <= 16 ? run_many<T, T, 16>(p, err, st) : p.rank <= 32 ? run_many<T, T, 32>(p, err, st)
                                                                       : run_many<T, T, 64>(p, err, st);
}

}  // namespace
}  // namespace bnn

using namespace bnn;

extern "C" int bnnk_lowrank(const bnnk_lowrank_args *p, bnn_stream_t st) {
  if (p->rows <= 0) return 0;
  return p->type == 1 ? run_lowrank<1>(*p, p->err, (cudaStream_t)st) : run_lowrank<2>(*p, p->err, (cudaStream_t)st);
}
