/* The entry points of the operators over sequences of windows (include/bnneon_cuda.h): checks of arguments, the op
 * objects with their device tables and scratch, the launches (bnn_kernels.h). */
#include <cuda_runtime_api.h>
#include <math.h>
#include <stdlib.h>

#include "../../../include/bnneon_cuda.h"
#include "bnn_internal.h"

#define ERR bnn_set_error

static int launch_rc(const char *what, int e) {
  if (!e) return 0;
  ERR(BNN_ERR_WINDOW, "%s: CUDA error %d (%s)", what, e, cudaGetErrorString((cudaError_t)e));
  return -1;
}

/* device memory of an op; -1 with the error set */
static int dev_alloc(const char *what, void **p, size_t bytes) {
  const cudaError_t e = bnn_fail_dev_alloc() ? cudaErrorMemoryAllocation : cudaMalloc(p, bytes);
  if (!e) return 0;
  ERR(e == cudaErrorMemoryAllocation ? BNN_ERR_OOM : BNN_ERR_CPU, "%s: %zu bytes of device memory: CUDA error %d (%s)",
      what, bytes, (int)e, cudaGetErrorString(e));
  return -1;
}

/* an op's error word cleared, and table (NULL: none) copied to d_table; both have happened when it returns: the copies go
 * to the legacy stream, which streams made non-blocking do not wait for, and the first run may be on one of those */
static int dev_set(const char *what, int *err, float *d_table, const float *table, size_t bytes) {
  cudaError_t e = cudaMemset(err, 0, sizeof(int));
  if (!e && table) e = cudaMemcpy(d_table, table, bytes, cudaMemcpyHostToDevice);
  if (!e) e = cudaStreamSynchronize(cudaStreamLegacy);
  if (!e) return 0;
  ERR(BNN_ERR_CPU, "%s: CUDA error %d (%s)", what, (int)e, cudaGetErrorString(e));
  return -1;
}

static void *host_alloc(const char *what, size_t bytes) {
  void *p = bnn_fail_host_alloc() ? NULL : calloc(1, bytes);
  if (!p) ERR(BNN_ERR_OOM, "%s: out of memory", what);
  return p;
}

static int misaligned(const void *p) { return ((uintptr_t)p & 15) != 0; }
/* not where 4-byte values can be */
static int misaligned4(const void *p) { return ((uintptr_t)p & 3) != 0; }

/* a device word after all work issued so far, on streams that the copy alone would not wait for too */
static int read_word(const int *d) {
  int v = 0;
  if (d && (cudaDeviceSynchronize() || cudaMemcpy(&v, d, sizeof v, cudaMemcpyDeviceToHost))) return -1;
  return v;
}

/* ------------------------------------------------------------------ linear attention with decay */

struct bnn_dattn {
  int type, H, Hk, dk, dv, seqs;
  long long tokens;
  float scale;
  float *pow;      /* [Hk][kDattnPow] */
  float *scratch;  /* the states of the parts of long sequences */
  int *err;
};

bnn_dattn *bnn_dattn_new(int type, int heads, int kv_heads, int dk, int dv, const float *decay, float scale, int seqs,
                         long long tokens) {
  int ok = (type == BNN_T_F16 || type == BNN_T_BF16) && kv_heads >= 1 && kv_heads <= 65535 && heads >= kv_heads &&
           heads % kv_heads == 0 && dk >= 8 && dk <= 128 && dk % 8 == 0 && dv >= 8 && dv <= 128 && dv % 8 == 0 && decay &&
           isfinite(scale) && seqs >= 1 && tokens >= 1 && tokens < (1ll << 31);
  if (!ok) {
    ERR(BNN_ERR_USAGE, "bnn_dattn_new: type %d heads %d kv_heads %d dk %d dv %d scale %g seqs %d tokens %lld (type fp16 or "
        "bf16, heads a multiple of kv_heads, dk and dv multiples of 8 up to 128, a finite scale, at least one sequence "
        "and 1 .. 2^31 - 1 tokens)", type, heads, kv_heads, dk, dv, scale, seqs, tokens);
    return NULL;
  }
  for (int h = 0; h < kv_heads; h++)
    if (!(decay[h] >= 0.f && decay[h] <= 1.f)) {
      ERR(BNN_ERR_USAGE, "bnn_dattn_new: decay[%d] = %g (0 <= decay <= 1)", h, decay[h]);
      return NULL;
    }
  bnn_dattn *o = host_alloc("bnn_dattn_new", sizeof *o);
  if (!o) return NULL;
  o->type = type; o->H = heads; o->Hk = kv_heads; o->dk = dk; o->dv = dv; o->seqs = seqs; o->tokens = tokens;
  o->scale = scale;
  float *t = host_alloc("bnn_dattn_new", sizeof(float) * kDattnPow * kv_heads);
  const size_t bytes = sizeof(float) * kDattnPow * kv_heads;
  int bad = !t || dev_alloc("bnn_dattn_new", (void **)&o->pow, bytes) ||
            dev_alloc("bnn_dattn_new", (void **)&o->err, sizeof(int));
  const long long states = bad ? 0 : bnnk_dattn_scratch_states(seqs, kv_heads, tokens);
  if (states > 0) bad = dev_alloc("bnn_dattn_new", (void **)&o->scratch, sizeof(float) * states * dk * dv);
  if (!bad) {
    for (int h = 0; h < kv_heads; h++) {
        float *th = t + h * kDattnPow;
        for (int i = 0; i <= 128; i++) th[i] = (float)pow((double)decay[h], i);
        double p = pow((double)decay[h], 128.0);
        for (int k = 0; k < 25; k++, p *= p) {
          th[kDattnPow2 + 2 * k] = (float)p;
          th[kDattnPow2 + 2 * k + 1] = (float)(p - (double)(float)p);
        }
    }
    bad = dev_set("bnn_dattn_new", o->err, o->pow, t, bytes);
  }
  free(t);
  if (bad) { bnn_dattn_free(o); return NULL; }
  return o;
}

static int dattn_launch(const char *what, bnn_dattn *o, int n, long long tokens, const int32_t *d_cu,
                        const int32_t *d_slot, const uint8_t *d_live, const void *d_q, long long qts, const void *d_k,
                        long long kts, const void *d_v, long long vts, const float *d_s0, float *d_s1, void *d_o,
                        long long ots, void *stream) {
  if (!o || n < 0 || n > o->seqs || tokens < 0 || tokens > o->tokens) {
    ERR(BNN_ERR_USAGE, "%s: %d sequences of %lld tokens (capacity %d of %lld)", what, n, tokens, o ? o->seqs : 0,
        o ? o->tokens : 0);
    return -1;
  }
  if (n == 0) return 0;
  if (misaligned4(d_cu) || misaligned4(d_slot)) {
    ERR(BNN_ERR_USAGE, "%s: offsets %p, slots %p: not aligned to their elements", what, (const void *)d_cu,
        (const void *)d_slot);
    return -1;
  }
  if ((tokens > 0 && (!d_q || !d_k || !d_v || !d_o)) || misaligned(d_q) || misaligned(d_k) || misaligned(d_v) ||
      misaligned(d_o) || misaligned(d_s0) || misaligned(d_s1) || qts < (long long)o->H * o->dk || qts % 8 ||
      kts < (long long)o->Hk * o->dk || kts % 8 || vts < (long long)o->Hk * o->dv || vts % 8 ||
      ots < (long long)o->H * o->dv || ots % 8) {
    ERR(BNN_ERR_USAGE, "%s: q %p stride %lld, k %p stride %lld, v %p stride %lld, o %p stride %lld, states %p %p (16-byte "
        "aligned, token strides multiples of 8 that hold %d x %d, %d x %d, %d x %d and %d x %d elements)", what, d_q, qts,
        d_k, kts, d_v, vts, d_o, ots, (const void *)d_s0, (void *)d_s1, o->H, o->dk, o->Hk, o->dk, o->Hk, o->dv, o->H,
        o->dv);
    return -1;
  }
  const bnnk_dattn_args a = {o->type, n, o->H, o->Hk, o->dk, o->dv, tokens, d_cu, d_slot, d_live, d_q, d_k, d_v,
                             qts, kts, vts, d_s0, d_s1, d_o, ots, o->pow, o->scale, o->scratch, o->err};
  return launch_rc(what, bnnk_dattn(&a, (bnn_stream_t)stream));
}

int bnn_dattn_run(bnn_dattn *o, int n, long long tokens, const int32_t *d_cu, const int32_t *d_slot,
                  const uint8_t *d_live, const void *d_q, long long qts, const void *d_k, long long kts, const void *d_v,
                  long long vts, const float *d_s0, float *d_s1, void *d_o, long long ots, void *stream) {
  if (n > 0 && !d_cu) { ERR(BNN_ERR_USAGE, "bnn_dattn_run: no token offsets"); return -1; }
  return dattn_launch("bnn_dattn_run", o, n, tokens, d_cu, d_slot, d_live, d_q, qts, d_k, kts, d_v, vts, d_s0, d_s1, d_o,
                      ots, stream);
}

int bnn_dattn_step(bnn_dattn *o, int n, const int32_t *d_slot, const uint8_t *d_live, const void *d_q, long long qts,
                   const void *d_k, long long kts, const void *d_v, long long vts, const float *d_s0, float *d_s1,
                   void *d_o, long long ots, void *stream) {
  return dattn_launch("bnn_dattn_step", o, n, n, NULL, d_slot, d_live, d_q, qts, d_k, kts, d_v, vts, d_s0, d_s1, d_o, ots,
                      stream);
}

#define P(i) ((void *)(uintptr_t)w[i])
static int no_words(const char *what, const long long *w) {
  if (!w) ERR(BNN_ERR_USAGE, "%s: no arguments", what);
  return !w;
}
/* a count that an int does not hold is refused as a negative one */
static int count_of(long long v) { return v < 0 || v > 0x7fffffff ? -1 : (int)v; }

int bnn_dattn_run_words(bnn_dattn *o, const long long *w) {
  if (no_words("bnn_dattn_run_words", w)) return -1;
  return bnn_dattn_run(o, count_of(w[0]), w[1], P(2), P(3), P(4), P(5), w[6], P(7), w[8], P(9), w[10], P(11), P(12), P(13),
                       w[14], P(15));
}

int bnn_dattn_step_words(bnn_dattn *o, const long long *w) {
  if (no_words("bnn_dattn_step_words", w)) return -1;
  return bnn_dattn_step(o, count_of(w[0]), P(1), P(2), P(3), w[4], P(5), w[6], P(7), w[8], P(9), P(10), P(11), w[12],
                        P(13));
}

int bnn_dattn_error(bnn_dattn *o) { return o ? read_word(o->err) : -1; }

void bnn_dattn_free(bnn_dattn *o) {
  if (!o) return;
  cudaFree(o->pow);
  cudaFree(o->scratch);
  cudaFree(o->err);
  free(o);
}

/* ------------------------------------------------------------------ shared projection, low-rank adapters */

struct bnn_lowrank {
  bnnk_lowrank_args a;
  int rows;
};

bnn_lowrank *bnn_lowrank_new(int type, int out_type, int N, int K, const void *d_w, long long ldw, const float *d_bias,
                             int slots, int rank, const void *d_a, const void *d_b, const float *d_scale, int rows) {
  if ((type != BNN_T_F16 && type != BNN_T_BF16) || (out_type != BNN_T_F32 && out_type != type) || N < 1 || K < 8 ||
      K % 8 || N > (1 << 24) || K > (1 << 24) || !d_w || ldw < K || ldw % 8 || slots < 1 || rank < 8 || rank > 64 ||
      rank % 8 || !d_a || !d_b || rows < 1 || misaligned(d_w) || misaligned(d_a) || misaligned(d_b) ||
      misaligned4(d_bias) || misaligned4(d_scale)) {
    ERR(BNN_ERR_USAGE, "bnn_lowrank_new: type %d out %d N %d K %d ldw %lld slots %d rank %d rows %d w %p a %p b %p bias %p scale %p "
        "(type fp16 or bf16, out fp32 or the same, K and ldw >= K multiples of 8, N and K up to 2^24, rank a multiple of 8 in 8 "
        ".. 64, 16-byte aligned weights, bias and scale aligned to their elements)", type, out_type, N, K, ldw, slots, rank,
        rows, d_w, d_a, d_b, (const void *)d_bias, (const void *)d_scale);
    return NULL;
  }
  bnn_lowrank *o = host_alloc("bnn_lowrank_new", sizeof *o);
  if (!o) return NULL;
  o->rows = rows;
  o->a.type = type; o->a.otype = out_type; o->a.N = N; o->a.K = K; o->a.slots = slots; o->a.rank = rank;
  o->a.w = d_w; o->a.ldw = ldw; o->a.bias = d_bias; o->a.a = d_a; o->a.b = d_b; o->a.scale = d_scale;
  if (dev_alloc("bnn_lowrank_new", (void **)&o->a.hid, sizeof(float) * (size_t)rows * rank) ||
      dev_alloc("bnn_lowrank_new", (void **)&o->a.err, sizeof(int)) ||
      dev_set("bnn_lowrank_new", o->a.err, NULL, NULL, 0)) {
    bnn_lowrank_free(o);
    return NULL;
  }
  return o;
}

int bnn_lowrank_run(bnn_lowrank *o, int rows, const void *d_x, long long ldx, const int32_t *d_slot, void *d_y,
                    long long ldy, void *stream) {
  if (!o || rows < 0 || rows > o->rows || (rows > 0 && (!d_x || !d_y || ldx < o->a.K || ldx % 8 || ldy < o->a.N ||
                                                        misaligned(d_x) || misaligned4(d_slot) ||
                                                        ((uintptr_t)d_y & (o->a.otype ? 1 : 3))))) {
    ERR(BNN_ERR_USAGE, "bnn_lowrank_run: %d rows (capacity %d) x %p stride %lld (>= K %d, a multiple of 8, 16-byte "
        "aligned) y %p stride %lld (>= N %d) slots %p (y and slots aligned to their elements)", rows, o ? o->rows : 0, d_x,
        ldx, o ? o->a.K : 0, d_y, ldy, o ? o->a.N : 0, (const void *)d_slot);
    return -1;
  }
  if (rows == 0) return 0;
  bnnk_lowrank_args a = o->a;
  a.rows = rows;
  a.x = d_x;
  a.ldx = ldx;
  a.slot = d_slot;
  a.y = d_y;
  a.ldy = ldy;
  return launch_rc("bnn_lowrank_run", bnnk_lowrank(&a, (bnn_stream_t)stream));
}

int bnn_lowrank_run_words(bnn_lowrank *o, const long long *w) {
  if (no_words("bnn_lowrank_run_words", w)) return -1;
  return bnn_lowrank_run(o, count_of(w[0]), P(1), w[2], P(3), P(4), w[5], P(6));
}

int bnn_lowrank_error(bnn_lowrank *o) { return o ? read_word(o->a.err) : -1; }

void bnn_lowrank_free(bnn_lowrank *o) {
  if (!o) return;
  cudaFree(o->a.hid);
  cudaFree(o->a.err);
  free(o);
}

/* ------------------------------------------------------------------ norms around a block */

struct bnn_norm_gate {
  bnnk_norm_gate_args a;
};

bnn_norm_gate *bnn_norm_gate_new(int D, int x_type, int type, int norm, int gate, float eps, float alpha,
                                 const float *d_wpost, const float *d_bpost, const float *d_gamma, const float *d_wpre,
                                 const float *d_bpre) {
  if (D < 1 || D > (1 << 24) || type < BNN_T_F32 || type > BNN_T_BF16 || (x_type != BNN_T_F32 && x_type != type) ||
      (norm != BNN_NORM_RMS && norm != BNN_NORM_LAYER) || gate < BNN_GATE_NONE || gate > BNN_GATE_SILU || !(eps >= 0.f) ||
      !isfinite(eps) || !isfinite(alpha) || misaligned4(d_wpost) || misaligned4(d_bpost) || misaligned4(d_gamma) ||
      misaligned4(d_wpre) || misaligned4(d_bpre)) {
    ERR(BNN_ERR_USAGE, "bnn_norm_gate_new: D %d x_type %d type %d norm %d gate %d eps %g alpha %g (D in 1 .. 2^24, x_type "
        "fp32 or type, BNN_NORM_*, BNN_GATE_*, finite eps >= 0 and alpha, vectors aligned to their elements)", D, x_type,
        type, norm, gate, eps, alpha);
    return NULL;
  }
  bnn_norm_gate *o = host_alloc("bnn_norm_gate_new", sizeof *o);
  if (!o) return NULL;
  o->a.D = D; o->a.xtype = x_type; o->a.type = type; o->a.layer = norm; o->a.gate = gate; o->a.eps = eps;
  o->a.alpha = alpha; o->a.wpost = d_wpost; o->a.bpost = d_bpost; o->a.gamma = d_gamma; o->a.wpre = d_wpre;
  o->a.bpre = d_bpre;
  return o;
}

int bnn_norm_gate_run(bnn_norm_gate *o, int rows, const void *d_x, long long xs, const void *d_f, long long fs,
                      const void *d_g, long long gs, const uint8_t *d_live, void *d_xo, long long xos, void *d_h,
                      long long hs, void *stream) {
  const int D = o ? o->a.D : 0;
  if (!o || rows < 0 || (rows > 0 && (!d_x || xs < D || (d_f && (fs < D || (o->a.gate && (!d_g || gs < D)))) ||
                                      (!d_xo && !d_h) || (d_xo && xos < D) || (d_h && hs < D)))) {
    ERR(BNN_ERR_USAGE, "bnn_norm_gate_run: %d rows of %d, x %p stride %lld f %p stride %lld g %p stride %lld xo %p stride "
        "%lld h %p stride %lld (strides >= the width, g where f is given and the op has a gate, an output)", rows, D, d_x,
        xs, d_f, fs, d_g, gs, d_xo, xos, d_h, hs);
    return -1;
  }
  if (rows == 0) return 0;
  const uintptr_t xm = o->a.xtype ? 1 : 3, fm = o->a.type ? 1 : 3;
  if (((uintptr_t)d_x & xm) || ((uintptr_t)d_xo & xm) || ((uintptr_t)d_f & fm) || ((uintptr_t)d_g & fm) ||
      ((uintptr_t)d_h & fm)) {
    ERR(BNN_ERR_USAGE, "bnn_norm_gate_run: x %p f %p g %p xo %p h %p: not aligned to their elements", d_x, d_f, d_g, d_xo,
        d_h);
    return -1;
  }
  bnnk_norm_gate_args a = o->a;
  a.rows = rows;
  a.x = d_x; a.xs = xs; a.f = d_f; a.fs = fs; a.g = d_g; a.gs = gs; a.live = d_live;
  a.xo = d_xo; a.xos = xos; a.h = d_h; a.hs = hs;
  return launch_rc("bnn_norm_gate_run", bnnk_norm_gate(&a, (bnn_stream_t)stream));
}

int bnn_norm_gate_run_words(bnn_norm_gate *o, const long long *w) {
  if (no_words("bnn_norm_gate_run_words", w)) return -1;
  return bnn_norm_gate_run(o, count_of(w[0]), P(1), w[2], P(3), w[4], P(5), w[6], P(7), P(8), w[9], P(10), w[11], P(12));
}

void bnn_norm_gate_free(bnn_norm_gate *o) { free(o); }
