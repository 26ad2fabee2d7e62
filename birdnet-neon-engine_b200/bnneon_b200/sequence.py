"""Operators over sequences of windows (include/bnneon_cuda.h): linear attention with a decay per head, a shared
projection with low-rank adapters per row, and the norms, gate and residual around a block.

    from bnneon_b200 import sequence
    attn = sequence.DecayAttention("bf16", heads=8, dk=128, dv=128, decay=decay, seqs=64, tokens=1 << 16)
    attn.run(n, tokens, cu.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), s0, s1, stream=s)

Buffers are device pointers (ints, e.g. a torch tensor's data_ptr()) and `stream` a cudaStream_t as int (None = the
legacy default stream), as Model.infer_device takes them; calls are asynchronous. Strides default to packed rows.
An object's calls share its scratch: order them on one stream, or give each stream an object of its own.
"""
import struct

import numpy as np

from . import BnnError, last_error, load_library

TYPES = {"f32": 0, "f16": 1, "bf16": 2}
NORMS = {"rms": 0, "layer": 1}
GATES = {"none": 0, "sigmoid": 1, "silu": 2}

# a call's arguments as 64-bit words: ctypes takes about 0.1 us for each argument, more than a small call's launch
_WORDS = {n: struct.Struct(f"{n}q").pack for n in (7, 13, 14, 16)}


def _code(table, what, name):
    if name not in table:
        raise BnnError(f"{what} {name!r}: one of {', '.join(table)}", "USAGE")
    return table[name]


class _Op:
    """a library op object, freed with its Python object"""
    _free = None

    def __init__(self, lib):
        self.h = load_library(lib)
        self.op = None

    def _made(self, op):
        if not op:
            raise last_error(self.h)
        self.op = op

    def close(self):
        if self.op:
            getattr(self.h, self._free)(self.op)
            self.op = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:  # pylint: disable=broad-except
            pass


class DecayAttention(_Op):
    """S_t = decay S_(t-1) + k_t^T v_t, o_t = scale q_t S_t per sequence and head (bnn_dattn_*). decay: one float in
    [0, 1] per k/v head; seqs, tokens: the most of a call."""
    _free = "bnn_dattn_free"

    def __init__(self, dtype, heads, dk, dv, decay, kv_heads=None, scale=None, seqs=1, tokens=1, lib=None):
        super().__init__(lib)
        self.kv_heads = heads if kv_heads is None else kv_heads
        d = np.ascontiguousarray(decay, np.float32).reshape(-1)
        if d.size != self.kv_heads:
            raise BnnError(f"decay: {d.size} values for {self.kv_heads} k/v heads", "USAGE")
        self._made(self.h.bnn_dattn_new(_code(TYPES, "dtype", dtype), heads, self.kv_heads, dk, dv, d.ctypes.data,
                                        max(dk, 1) ** -0.5 if scale is None else scale, seqs, tokens))
        self.q_row, self.k_row, self.v_row, self.o_row = heads * dk, self.kv_heads * dk, self.kv_heads * dv, heads * dv

    def run(self, n, tokens, cu, q, k, v, o, s0=None, s1=None, slot=None, live=None, qts=None, kts=None, vts=None,
            ots=None, stream=None):
        """n sequences, sequence i the tokens cu[i] .. cu[i + 1] - 1"""
        if self.h.bnn_dattn_run_words(self.op, _WORDS[16](
                n, tokens, cu or 0, slot or 0, live or 0, q or 0, qts or self.q_row, k or 0, kts or self.k_row, v or 0,
                vts or self.v_row, s0 or 0, s1 or 0, o or 0, ots or self.o_row, stream or 0)):
            raise last_error(self.h)

    def step(self, n, q, k, v, o, s0=None, s1=None, slot=None, live=None, qts=None, kts=None, vts=None, ots=None,
             stream=None):
        """n sequences of one token each"""
        if self.h.bnn_dattn_step_words(self.op, _WORDS[14](
                n, slot or 0, live or 0, q or 0, qts or self.q_row, k or 0, kts or self.k_row, v or 0, vts or self.v_row,
                s0 or 0, s1 or 0, o or 0, ots or self.o_row, stream or 0)):
            raise last_error(self.h)

    @property
    def error(self):
        return self.h.bnn_dattn_error(self.op)


class LowRank(_Op):
    """y_r = W x_r + bias + scale[s] B[s] (A[s] x_r), s = slot[r] (bnn_lowrank_*). w, bias, a, b, scale: device pointers
    the caller keeps; rows: the most rows of a call."""
    _free = "bnn_lowrank_free"

    def __init__(self, dtype, out, N, K, w, bias, slots, rank, a, b, scale=None, rows=1, ldw=None, lib=None):
        super().__init__(lib)
        self._made(self.h.bnn_lowrank_new(_code(TYPES, "dtype", dtype), _code(TYPES, "out", out), N, K, w, ldw or K, bias,
                                          slots, rank, a, b, scale, rows))
        self.N, self.K = N, K

    def run(self, rows, x, slot, y, ldx=None, ldy=None, stream=None):
        if self.h.bnn_lowrank_run_words(self.op, _WORDS[7](rows, x or 0, ldx or self.K, slot or 0, y or 0, ldy or self.N,
                                                          stream or 0)):
            raise last_error(self.h)

    @property
    def error(self):
        return self.h.bnn_lowrank_error(self.op)


class NormGate(_Op):
    """u = norm(f) wpost + bpost; x' = x + alpha gamma act(g) u; h = norm(x') wpre + bpre (bnn_norm_gate_*). The vectors
    are fp32 device pointers the caller keeps, or None."""
    _free = "bnn_norm_gate_free"

    def __init__(self, D, xtype, dtype, norm="rms", gate="none", eps=1e-5, alpha=1.0, wpost=None, bpost=None, gamma=None,
                 wpre=None, bpre=None, lib=None):
        super().__init__(lib)
        self._made(self.h.bnn_norm_gate_new(D, _code(TYPES, "xtype", xtype), _code(TYPES, "dtype", dtype),
                                            _code(NORMS, "norm", norm), _code(GATES, "gate", gate), eps, alpha, wpost,
                                            bpost, gamma, wpre, bpre))
        self.D = D

    def run(self, rows, x, f, g, xo, h, live=None, xs=None, fs=None, gs=None, xos=None, hs=None, stream=None):
        D = self.D
        if self.h.bnn_norm_gate_run_words(self.op, _WORDS[13](
                rows, x or 0, xs or D, f or 0, fs or D, g or 0, gs or D, live or 0, xo or 0, xos or D, h or 0, hs or D,
                stream or 0)):
            raise last_error(self.h)
