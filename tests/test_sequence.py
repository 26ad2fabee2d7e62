"""The operators over sequences of windows (bnn_dattn_*, bnn_lowrank_*, bnn_norm_gate_*) against their definitions in 64
bits, and their refusals.

Tolerances, element by element. An output of t bits of significand is rounded once: u |want|, u = 2^-8 (bf16), 2^-11
(fp16), 2^-24 (fp32), and half the type's smallest step. A sum of n terms in fp32 is off by at most n 2^-24 times the sum
M of the terms' magnitudes. An fp32 factor that the tensor cores take as two 16-bit parts is off by the square of their
unit roundoff, 2^-16 for bf16: two such factors in a term (a chunk's products, the state before it) give 2^-15 M.
"""
import math

import numpy as np
import pytest

from bnneon_b200 import BnnError, last_error, load_library, sequence

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
TINY = {"bf16": 2.0 ** -134, "f16": 2.0 ** -25, "f32": 2.0 ** -150}


@pytest.fixture(scope="module")
def cuda():
    if not torch.cuda.is_available():
        pytest.fail("a GPU test ran without a visible CUDA device")
    torch.cuda.init()
    load_library()
    return torch.device("cuda")


def rand(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def check(got, want, slack, dtype, what):
    got, want = got.double(), want.double()
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    off = (got - want).abs() - (U[dtype] * want.abs() + TINY[dtype] + slack)
    assert float(off.max() if off.numel() else 0) <= 0, (
        f"{what}: {int((off > 0).sum())} of {off.numel()} beyond, worst by {float(off.max()):.3g} "
        f"(error {float((got - want).abs().max()):.3g})")


# ------------------------------------------------------------------ linear attention with decay


class Attention:
    """inputs of one call; tokens of dead rows hold NaN"""

    def __init__(self, dtype, H, Hk, dk, dv, lens, masked=0.0, states=None, seed=0, decay=None, row=0, k_scale=1.0):
        gen = generator(seed)
        self.dtype, self.H, self.Hk, self.dk, self.dv, self.lens = dtype, H, Hk, dk, dv, lens
        T = sum(lens)
        t = DT[dtype]
        # q, k and v as parts of one projection's rows, with `row` more elements a row
        width = H * dk + Hk * (dk + dv) + row
        buf = rand(gen, T + 1, width)[:T]
        buf[:, H * dk:H * dk + Hk * dk] *= k_scale
        self.buf = buf.to(t)
        self.q = self.buf[:, :H * dk].unflatten(1, (H, dk))
        self.k = self.buf[:, H * dk:(H + Hk) * dk].unflatten(1, (Hk, dk))
        self.v = self.buf[:, (H + Hk) * dk:(H + Hk) * dk + Hk * dv].unflatten(1, (Hk, dv))
        self.ts = width
        self.live = None
        if masked:
            self.live = torch.rand(T, device="cuda", generator=gen) >= masked
            self.buf[~self.live] = math.nan
        n = len(lens)
        self.cu = torch.tensor([0] + lens).cumsum(0).int().cuda()
        self.slot = torch.randperm(n + 3, device="cuda", generator=gen)[:n].int() if states is None else states.int()
        self.s0 = rand(gen, n + 3, Hk, dk, dv)
        self.decay = np.asarray(decay if decay is not None else 1 - 2.0 ** -np.linspace(0.5, 9, Hk), np.float32)
        self.scale = dk ** -0.5
        self.o = torch.full((T, H, dv), 7.0, device="cuda", dtype=t)

    def op(self, **kw):
        return sequence.DecayAttention(self.dtype, self.H, self.dk, self.dv, self.decay, kv_heads=self.Hk,
                                       scale=self.scale, seqs=max(1, len(self.lens)), tokens=max(1, sum(self.lens)), **kw)

    def run(self, op, s0=True, s1=None, slot=True, stream=None, step=False):
        args = [self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.o.data_ptr(),
                self.s0.data_ptr() if s0 else None, None if s1 is None else s1.data_ptr()]
        kw = dict(slot=self.slot.data_ptr() if slot else None, live=None if self.live is None else self.live.data_ptr(),
                  qts=self.ts, kts=self.ts, vts=self.ts, stream=stream)
        if step:
            op.step(len(self.lens), *args, **kw)
        else:
            op.run(len(self.lens), sum(self.lens), self.cu.data_ptr(), *args, **kw)

    def want(self, s0=True, slot=True):
        """(o, {sequence: state}) and the sums of their terms' magnitudes, token by token"""
        out, states = [], []
        lam = torch.from_numpy(self.decay.astype(np.float64)).cuda()[:, None, None]
        G = self.H // self.Hk
        t0 = 0
        o, mo = (torch.zeros(self.o.shape, dtype=torch.float64, device="cuda") for _ in range(2))
        for i, L in enumerate(self.lens):
            at = int(self.slot[i]) if slot else i
            S = self.s0[at].double() if s0 and at >= 0 else torch.zeros_like(self.s0[0], dtype=torch.float64)
            M = S.abs()
            for t in range(t0, t0 + L):
                S, M = lam * S, lam * M
                if self.live is None or bool(self.live[t]):
                    kv = self.k[t].double()[:, :, None] * self.v[t].double()[:, None, :]
                    S, M = S + kv, M + kv.abs()
                    q = self.q[t].double().view(self.Hk, G, self.dk)
                    o[t] = self.scale * torch.matmul(q, S).view(self.H, self.dv)
                    # the chunk form's terms are (q . k) v: their magnitude is at most |q| |k| |v| summed, as M has it
                    mo[t] = self.scale * torch.matmul(q.abs(), M).view(self.H, self.dv)
            states.append((S, M))
            t0 += L
        out = (o, mo)
        return out, states

    def check(self, s1, s0=True, slot=True, what=""):
        (o, mo), states = self.want(s0, slot)
        n = max(self.lens + [0]) + self.dk + 4
        rel = 2.0 ** -15 + n * 2.0 ** -24
        check(self.o, o, rel * mo, self.dtype, what + "o")
        if s1 is not None:
            for i, (S, M) in enumerate(states):
                at = int(self.slot[i]) if slot else i
                if at >= 0:
                    check(s1[at], S, rel * M, "f32", f"{what}state {i} of {self.lens[i]} tokens")


ATTENTION = [
    # dtype, heads, kv heads, dk, dv, lengths, share of masked tokens
    ("bf16", 2, 2, 128, 128, [1], 0),
    ("f16", 2, 2, 64, 64, [3, 0, 1, 17], 0),
    ("bf16", 2, 2, 128, 128, [128, 129, 127, 0, 255, 1, 300], 0),
    ("f16", 2, 2, 128, 128, [384, 63, 65], 0.2),
    ("bf16", 3, 1, 64, 64, [200, 130, 64], 0.1),
    ("f16", 6, 2, 96, 72, [150, 1, 290], 0.3),
    ("bf16", 4, 4, 40, 24, [333, 90], 0),
    ("f16", 1, 1, 8, 8, [513], 0),
    ("bf16", 8, 1, 72, 128, [140, 260], 0.5),
    ("f16", 2, 1, 128, 16, [700], 0),
    ("bf16", 1, 1, 128, 64, [2500], 0.05),
    ("bf16", 1, 1, 64, 128, [1900, 5], 0),
    ("f16", 20, 1, 32, 32, [131], 0.1),
]


@gpu
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_dattn_against_64_bits(cuda, case):
    dtype, H, Hk, dk, dv, lens, masked = ATTENTION[case]
    a = Attention(dtype, H, Hk, dk, dv, lens, masked, seed=case, row=8 * (case % 3))
    s1 = torch.full_like(a.s0, 9.0)
    op = a.op()
    a.run(op, s1=s1)
    a.check(s1)
    untouched = [i for i in range(len(a.s0)) if i not in set(a.slot.tolist())]
    assert bool((s1[untouched] == 9.0).all())
    assert op.error == 0
    # the same call again gives the same bits, in place too
    o, s = a.o.clone(), s1.clone()
    a.run(op, s1=s1)
    assert torch.equal(a.o, o) and torch.equal(s1, s)
    keep = a.s0.clone()
    a.run(op, s1=a.s0)
    assert torch.equal(a.o, o)
    assert torch.equal(a.s0[a.slot.long()], s[a.slot.long()])
    a.s0 = keep


MIXED = [
    # short sequences on average, some of them long: neighbours of the lengths where the forms change, empty ones
    ("bf16", 4, 2, 64, 64, [1] * 40 + [300] + [2] * 20 + [0] * 10 + [64, 65, 1, 66, 0] + [3] * 15, 0.1),
    ("f16", 2, 2, 40, 64, [0, 200] + [5] * 100, 0),
    ("bf16", 2, 2, 128, 128, [1] * 60 + [32, 33, 0, 140] + [1] * 60, 0),
    ("f16", 2, 2, 96, 72, [2] * 80 + [34], 0.2),
    ("bf16", 1, 1, 128, 64, [1, 0, 3], 0),
    ("f16", 3, 3, 64, 64, [1] * 5, 0),
]


@gpu
@pytest.mark.parametrize("case", range(len(MIXED)))
def test_dattn_long_among_short(cuda, case):
    dtype, H, Hk, dk, dv, lens, masked = MIXED[case]
    a = Attention(dtype, H, Hk, dk, dv, lens, masked, seed=100 + case)
    s1 = torch.full_like(a.s0, 9.0)
    op = a.op()
    a.run(op, s1=s1)
    a.check(s1)
    untouched = [i for i in range(len(a.s0)) if i not in set(a.slot.tolist())]
    assert bool((s1[untouched] == 9.0).all())
    assert op.error == 0
    o = a.o.clone()
    a.run(op, s1=a.s0)
    assert torch.equal(a.o, o) and torch.equal(a.s0[a.slot.long()], s1[a.slot.long()])


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads", [(2, 2, 128, 128), (8, 2, 64, 64), (3, 1, 96, 72), (12, 1, 8, 104), (1, 1, 24, 128)])
@pytest.mark.parametrize("n, masked", [(1, 0), (7, 0.4), (130, 0.1)])
def test_dattn_step(cuda, dtype, heads, n, masked):
    a = Attention(dtype, *heads, [1] * n, masked, seed=n)
    s1 = torch.zeros_like(a.s0)
    a.run(a.op(), s1=s1, step=True)
    a.check(s1)


@gpu
def test_dattn_states_optional(cuda):
    a = Attention("bf16", 2, 2, 64, 64, [140, 5, 0, 260], seed=3)
    op = a.op()
    s1 = torch.zeros_like(a.s0)
    a.run(op, s0=False, s1=s1)
    a.check(s1, s0=False, what="from zero: ")
    a.run(op)
    a.check(None, what="no state kept: ")
    a.run(op, s1=s1, slot=False)
    a.check(s1, slot=False, what="slots in order: ")
    a.slot = torch.tensor([2, -1, 0, -1], device="cuda").int()
    s1.fill_(5.0)
    a.run(op, s1=s1)
    a.check(s1, what="negative slots: ")
    assert bool((s1[1] == 5.0).all()) and bool((s1[3:] == 5.0).all())


@gpu
@pytest.mark.parametrize("decay", [[0.0, 1.0], [0.5, 2.0 ** -30], [1.0, 1.0 - 2.0 ** -24]])
def test_dattn_extreme_decays(cuda, decay):
    a = Attention("bf16", 2, 2, 64, 64, [300, 1, 129], seed=5, decay=decay)
    s1 = torch.zeros_like(a.s0)
    a.run(a.op(), s1=s1)
    a.check(s1)


@gpu
def test_dattn_all_masked(cuda):
    a = Attention("f16", 2, 2, 64, 64, [200, 1, 128], 0.5, seed=6)
    a.live.fill_(False)
    a.buf.fill_(math.inf)
    s1 = torch.zeros_like(a.s0)
    a.run(a.op(), s1=s1)
    assert bool((a.o == 0).all())
    a.check(s1)


@gpu
def test_dattn_neighbours_do_not_leak(cuda):
    """a sequence's results do not change when the tokens around it hold NaN"""
    a = Attention("bf16", 2, 2, 128, 128, [70, 77, 300], seed=7)
    s1 = torch.zeros_like(a.s0)
    op = a.op()
    a.run(op, s1=s1)
    o = a.o.clone()
    a.buf[:70] = math.nan
    a.buf[147:] = math.inf
    s2 = torch.zeros_like(a.s0)
    a.run(op, s1=s2)
    at = int(a.slot[1])
    assert torch.equal(a.o[70:147], o[70:147]) and torch.equal(s2[at], s1[at])


@gpu
def test_dattn_prompt_then_steps(cuda):
    """a prompt in one call, and the same tokens as a shorter prompt and single steps on its state"""
    a = Attention("bf16", 4, 2, 64, 64, [140], seed=8)
    whole = torch.zeros_like(a.s0)
    a.run(a.op(), s1=whole)
    want = a.o.clone()
    state = a.s0.clone()
    op = a.op()
    cu = torch.tensor([0, 130]).int().cuda()
    args = lambda t: (a.q[t].data_ptr(), a.k[t].data_ptr(), a.v[t].data_ptr(), a.o[t].data_ptr())  # noqa: E731
    kw = dict(slot=a.slot.data_ptr(), qts=a.ts, kts=a.ts, vts=a.ts)
    a.o.zero_()
    op.run(1, 130, cu.data_ptr(), *args(0), state.data_ptr(), state.data_ptr(), **kw)
    for t in range(130, 140):
        op.step(1, *args(t), state.data_ptr(), state.data_ptr(), **kw)
    a.check(state)
    assert float((a.o.double() - want.double()).abs().max()) < 0.1


@gpu
def test_dattn_many_tokens_few_heads(cuda):
    """long enough for the work to be split along the sequence; the definition in chunks of 64-bit products"""
    a = Attention("bf16", 1, 1, 64, 64, [20011, 3000], 0.05, seed=9)
    s1 = torch.zeros_like(a.s0)
    a.run(a.op(), s1=s1)
    a.check(s1)


@gpu
@pytest.mark.parametrize("dtype, heads, lens, masked", [("f16", (8, 8, 32, 32), [591] * 8, 0.1),
                                                        ("f16", (4, 2, 32, 32), [3000, 700], 0.0),
                                                        ("bf16", (8, 8, 64, 64), [1311] * 5, 0.1),
                                                        ("bf16", (2, 2, 128, 128), [2900, 17], 0.1),
                                                        ("f16", (3, 1, 96, 128), [1500, 2500], 0.1)])
def test_dattn_split_sequences_repeat(cuda, dtype, heads, lens, masked):
    """sequences in parts of several chunks, the same bits however the warps are timed against each other"""
    a = Attention(dtype, *heads, lens, masked, seed=12)
    s1 = torch.zeros_like(a.s0)
    op = a.op()
    a.run(op, s1=s1)
    o, s = a.o.clone(), s1.clone()
    a.check(s1)
    differ = torch.zeros((), device="cuda", dtype=torch.int64)
    for _ in range(200):
        a.run(op, s1=s1)
        differ += (a.o != o).sum() + (s1 != s).sum()
    assert int(differ) == 0 and op.error == 0


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_dattn_ends_inside_a_chunk_repeat(cuda, dtype):
    """heads up to 64, no mask, an end inside the third or a later chunk: the rows past it are the next sequence's (here
    NaN), and are zeroed in a tile that was used before; the same bits however the warps are timed against each other"""
    lens = [257, 300, 383, 511, 700] * 6
    a = Attention(dtype, 6, 6, 64, 64, [x for n in lens for x in (n, 130)], seed=15)
    odd = torch.cat([a.cu[i:i + 2] for i in range(0, 2 * len(lens), 2)])
    mine = torch.zeros(len(a.buf), dtype=torch.bool, device="cuda")
    for lo, hi in odd.view(-1, 2).tolist():
        mine[lo:hi] = True
    s1 = torch.zeros_like(a.s0)
    op = a.op()
    a.run(op, s1=s1)
    a.check(s1)
    o, s = a.o[mine].clone(), s1[a.slot[::2].long()].clone()
    a.buf[~mine] = math.nan
    differ = torch.zeros((), device="cuda", dtype=torch.int64)
    for _ in range(100):
        a.run(op, s1=s1)
        differ += (a.o[mine] != o).sum() + (s1[a.slot[::2].long()] != s).sum()
    assert int(differ) == 0 and op.error == 0


@gpu
@pytest.mark.parametrize("heads", [(2, 1, 64, 64), (1, 1, 128, 128), (3, 3, 40, 72)])
@pytest.mark.parametrize("masked", [0.0, 0.2])
def test_dattn_loud_tokens_long_ago(cuda, heads, masked):
    """fp16: a token 2^28 times as loud as the others, decayed to nothing 60 tokens later, takes nothing from the state and
    the outputs there. The scale brings the quiet outputs to about 1, the loud ones past the type"""
    lens = [128, 300, 77]
    a = Attention("f16", *heads, lens, masked, seed=16, decay=[0.5] * heads[1], k_scale=2.0 ** -13)
    a.scale = 1000.0
    loud = [0, 128, 128 + 140, 128 + 300 + 3]
    quiet = torch.ones(sum(lens), dtype=torch.bool, device="cuda")
    for t in loud:
        a.k[t] = (a.k[t].float() * 2.0 ** 28).clamp(-6e4, 6e4).half()
        quiet[t:t + 60] = False
    s1 = torch.zeros_like(a.s0)
    op = a.op()
    a.run(op, s0=False, s1=s1)
    (o, mo), states = a.want(s0=False)
    rel = 2.0 ** -15 + (max(lens) + a.dk + 4) * 2.0 ** -24
    check(a.o[quiet], o[quiet], rel * mo[quiet], "f16", "quiet o")
    for i, (S, M) in enumerate(states):
        check(s1[int(a.slot[i])], S, rel * M, "f32", f"state {i}")
    assert op.error == 0


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads, lens, bad", [((2, 2, 64, 64), [300, 140], [100, 257, 311]), ((3, 1, 96, 72), [300, 140], [0, 130, 299]),
                                              ((2, 1, 128, 128), [700], [127, 128, 640]), ((1, 1, 64, 64), [3000], [1500]),
                                              ((1, 1, 128, 64), [2500], [1000, 1001, 2499]), ((2, 2, 40, 24), [5, 9, 2], [6])])
@pytest.mark.parametrize("part", "qkv")
@pytest.mark.parametrize("value", [math.nan, -math.inf])
def test_dattn_live_tokens_without_numbers(cuda, dtype, heads, lens, bad, part, value):
    """a live token's NaN or infinity: other heads and other sequences keep their bits, the outputs and states that the
    definition has finite (those before the token, and columns that it does not reach) their values, the others are not
    finite"""
    a = Attention(dtype, *heads, lens, seed=17)
    op = a.op()
    s1 = torch.zeros_like(a.s0)
    a.run(op, s1=s1)
    o, s = a.o.clone(), s1.clone()
    x = {"q": a.q, "k": a.k, "v": a.v}[part]
    G, ends = a.H // a.Hk, a.cu.tolist()
    same = torch.full((sum(lens), a.H), True, device="cuda")
    for i, t in enumerate(bad):
        h = i % x.shape[1]
        x[t, h, (7 * i + 3) % x.shape[2]] = value
        first, end = max(e for e in ends if e <= t), min(e for e in ends if e > t)
        same[first:end, slice(h, h + 1) if part == "q" else slice(h * G, (h + 1) * G)] = False
    s1.zero_()
    a.s0, keep = a.s0.clone(), a.s0
    a.run(op, s1=a.s0)  # in place
    s1, a.s0 = a.s0, keep
    (want, mo), states = a.want()
    rel = 2.0 ** -15 + (max(lens) + a.dk + 4) * 2.0 ** -24

    def finite_ones(got, w, m, dt, what):
        fin = torch.isfinite(w)
        assert torch.equal(torch.isfinite(got), fin), what
        check(got[fin], w[fin], rel * m[fin], dt, what)

    finite_ones(a.o, want, mo, dtype, "o")
    for i, (S, M) in enumerate(states):
        finite_ones(s1[int(a.slot[i])], S, M, "f32", f"state {i}")
    assert torch.equal(a.o[same], o[same])
    if part == "q":
        assert torch.equal(s1[a.slot.long()], s[a.slot.long()])
    assert op.error == 0


@gpu
@pytest.mark.parametrize("dtype, adds", [("bf16", 24), ("f16", 16)])
@pytest.mark.parametrize("heads, lens", [((2, 2, 64, 64), [1000, 640]), ((2, 1, 128, 128), [1000, 640]), ((1, 1, 128, 128), [6000])])
def test_dattn_states_are_fp32(cuda, dtype, adds, heads, lens):
    """the states' error in rms: the products are exact but for the fp32 sums, a chunk's one chain of 8 steps for each of
    K's parts (three for bf16, two for fp16), of which the tensor cores cut off at most 2^-24 of the sum at a step. With a
    part less (16 or 11 bits of K') it would be above"""
    a = Attention(dtype, *heads, lens, seed=18, decay=[0.99] * heads[1])
    s1 = torch.zeros_like(a.s0)
    a.run(a.op(), s1=s1)
    _, states = a.want()
    for i, (S, _) in enumerate(states):
        assert float((s1[int(a.slot[i])].double() - S).norm() / S.norm()) < adds * 2.0 ** -24


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
def test_dattn_steps_after_a_prompt_against_64_bits(cuda, dtype, d):
    """outputs and state of single steps on the state that a prompt left, as of one sequence"""
    a = Attention(dtype, 4, 2, d, d, [140], 0.1, seed=19)
    state, op = a.s0.clone(), a.op()
    cu = torch.tensor([0, 130]).int().cuda()
    kw = dict(slot=a.slot.data_ptr(), qts=a.ts, kts=a.ts, vts=a.ts)

    def at(t):
        return [x[t].data_ptr() for x in (a.q, a.k, a.v, a.o)] + [state.data_ptr()] * 2

    op.run(1, 130, cu.data_ptr(), *at(0), live=a.live.data_ptr(), **kw)
    for t in range(130, 140):
        op.step(1, *at(t), live=a.live[t:].data_ptr(), **kw)
    a.check(state)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads", [(2, 1, 64, 64), (1, 1, 128, 72)])
@pytest.mark.parametrize("where", ["v", "s0"])
def test_dattn_infinite_columns_of_large_states(cuda, dtype, heads, where):
    """a column of the state that is infinite, from a v or from the state that a sequence starts with, leaves the other
    columns what they are, past fp16's largest value too"""
    a = Attention(dtype, *heads, [300, 200], seed=20)
    a.s0 *= 1e6
    a.q *= 2.0 ** -10
    if where == "v":
        a.v[10, 0, 3] = math.inf
    else:
        a.s0[int(a.slot[0]), 0, 5, 3] = math.inf
    s1, op = torch.zeros_like(a.s0), a.op()
    a.run(op, s1=s1)
    (want, mo), states = a.want()
    fin = torch.isfinite(want)
    rel = 2.0 ** -15 + (300 + a.dk + 4) * 2.0 ** -24
    assert torch.equal(torch.isfinite(a.o), fin)
    check(a.o[fin], want[fin], rel * mo[fin], dtype, "o")
    for i, (S, M) in enumerate(states):
        fin = torch.isfinite(S)
        assert torch.equal(torch.isfinite(s1[int(a.slot[i])]), fin)
        check(s1[int(a.slot[i])][fin], S[fin], rel * M[fin], "f32", f"state {i}")
    assert op.error == 0


@gpu
def test_dattn_scratch_is_what_calls_can_use(cuda):
    """none where no call has more tokens than a chunk; for any capacity, at least a state for each head and part of every
    call it allows. The parts of a call: those of `segment_tokens` in k_dattn.cu"""
    import ctypes  # pylint: disable=import-outside-toplevel
    states = load_library().bnnk_dattn_scratch_states
    states.restype, states.argtypes = ctypes.c_longlong, [ctypes.c_int, ctypes.c_int, ctypes.c_longlong]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert states(1, 8, 1) == 0 and states(1, 1, 128) == 0 and states(100, 16, 100) == 0

    def parts(n, hk, tokens):
        if n * hk * 2 > sms:
            return 0
        length = -(-(-(-tokens // max(1, sms // hk))) // 128) * 128
        return 0 if tokens <= n * length else n + tokens // length

    rng = np.random.default_rng(1)
    for _ in range(20000):
        hk, seqs, tokens = int(rng.integers(1, 100)), int(rng.integers(1, 160)), int(2 ** rng.uniform(0, 18))
        n, used = int(rng.integers(1, seqs + 1)), int(rng.integers(1, tokens + 1))
        for t in (used, tokens):
            assert parts(n, hk, t) * hk <= states(seqs, hk, tokens), (n, t, hk, seqs, tokens)


@gpu
def test_dattn_offsets_past_32_bits(cuda):
    """states and rows more than 2^32 bytes and 2^31 elements into their buffers"""
    torch.cuda.empty_cache()
    a = Attention("bf16", 16, 16, 128, 128, [130, 2], seed=10)
    per = 16 * 128 * 128
    pool = torch.empty((1 << 31) // per + 3, 16, 128, 128, device="cuda")
    at = [len(pool) - 1, len(pool) - 2]
    slot = torch.tensor(at).int().cuda()
    for i, s in enumerate(at):
        pool[s] = a.s0[i]
    stride = 1 << 24
    big = torch.empty(132 * stride + 4096, device="cuda", dtype=torch.bfloat16)
    q = big.as_strided((132, 2048), (stride, 1))
    q.copy_(a.q.reshape(132, 2048))
    op = a.op()
    op.run(2, 132, a.cu.data_ptr(), big.data_ptr(), a.k.data_ptr(), a.v.data_ptr(), a.o.data_ptr(), pool.data_ptr(),
           pool.data_ptr(), slot=slot.data_ptr(), qts=stride, kts=a.ts, vts=a.ts)
    a.slot = torch.tensor([0, 1]).int().cuda()
    s1 = torch.stack([pool[s] for s in at])
    a.check(s1)
    del pool, big, q
    torch.cuda.empty_cache()


@gpu
def test_operators_on_a_stream_of_their_own(cuda):
    """inputs written on a side stream, the calls on that stream, with work before them that a wrong stream would miss"""
    a = Attention("bf16", 2, 2, 64, 64, [150, 4], seed=11)
    op = a.op()
    s1 = torch.zeros_like(a.s0)
    a.run(op, s1=s1)
    want = a.o.clone()
    side = torch.cuda.Stream()
    keep = a.buf.clone()
    a.buf.zero_()
    a.o.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(10):
            big = big @ big * 1e-4
        a.buf.copy_(keep)
        a.run(op, s1=s1, stream=side.cuda_stream)
        got = a.o.clone()
    side.synchronize()
    assert torch.equal(got, want)


# ------------------------------------------------------------------ shared projection, low-rank adapters


def lowrank_case(dtype, out, rows, N, K, rank, slots, order, seed, bias=True, scale=True, xpad=0, ypad=0, wpad=0):
    gen, t = generator(seed), DT[dtype]
    x = rand(gen, rows, K + xpad).to(t)
    w = (rand(gen, N, K + wpad) * K ** -0.5).to(t)
    x[:, K:] = math.nan
    w[:, K:] = math.nan
    A, B = (rand(gen, slots, rank, K) * K ** -0.5).to(t), rand(gen, slots, N, rank).to(t)
    b = rand(gen, N) if bias else None
    s = torch.rand(slots, device="cuda", generator=gen) + 0.5 if scale else None
    if order == "none":
        slot = None
    elif order == "runs":
        slot = torch.sort(torch.randint(-1, slots, (rows,), device="cuda", generator=gen))[0].int()
    else:
        slot = torch.randint(-1, slots + 1, (rows,), device="cuda", generator=gen).int()  # slots: none, too
    y = torch.full((rows, N + ypad), 7.0, device="cuda", dtype=DT[out])
    op = sequence.LowRank(dtype, out, N, K, w.data_ptr(), None if b is None else b.data_ptr(), slots, rank, A.data_ptr(),
                          B.data_ptr(), None if s is None else s.data_ptr(), rows=rows, ldw=K + wpad)
    op.run(rows, x.data_ptr(), None if slot is None else slot.data_ptr(), y.data_ptr(), ldx=K + xpad, ldy=N + ypad)
    first = y.clone()
    op.run(rows, x.data_ptr(), None if slot is None else slot.data_ptr(), y.data_ptr(), ldx=K + xpad, ldy=N + ypad)
    assert torch.equal(first, y), "the same call again"
    assert op.error == 0
    xd, wd = x[:, :K].double(), w[:, :K].double()
    want, M = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if b is not None:
        want, M = want + b.double(), M + b.double().abs()
    if slot is not None:
        for a in range(slots):
            at = torch.nonzero(slot == a).flatten()
            f = 1.0 if s is None else s[a].double()
            want[at] += f * ((xd[at] @ A[a].double().t()) @ B[a].double().t())
            M[at] += f * ((xd[at].abs() @ A[a].double().abs().t()) @ B[a].double().abs().t())
    check(y[:, :N], want, (2.0 ** -15 + (K + rank + 4) * 2.0 ** -24) * M, out, "y")
    assert bool((y[:, N:] == 7.0).all()), "outside the rows"


LOWRANK = [
    # dtype, out, rows, N, K, rank, slots, order of the slots
    ("bf16", "bf16", 1, 1024, 1024, 16, 4, "any"),
    ("f16", "f32", 1, 61, 64, 8, 1, "any"),
    ("bf16", "f32", 5, 6522, 1024, 16, 5, "any"),
    ("f16", "f16", 16, 512, 1536, 64, 20, "any"),
    ("bf16", "bf16", 17, 129, 72, 24, 3, "any"),
    ("f16", "f32", 64, 1000, 520, 32, 64, "any"),
    ("bf16", "bf16", 128, 256, 256, 16, 2, "runs"),
    ("bf16", "f32", 300, 333, 200, 40, 7, "any"),
    ("f16", "f16", 1000, 1024, 1024, 16, 12, "runs"),
    ("bf16", "bf16", 2049, 640, 8, 8, 3, "runs"),
    ("f16", "f16", 129, 64, 128, 48, 130, "any"),
    ("bf16", "bf16", 257, 6522, 64, 56, 2, "any"),
    ("bf16", "f32", 31, 1, 40, 16, 2, "any"),
    ("f16", "f16", 77, 200, 96, 16, 2, "none"),
    ("bf16", "bf16", 2, 200, 96, 16, 2, "none"),
]


@gpu
@pytest.mark.parametrize("case", range(len(LOWRANK)))
def test_lowrank_against_64_bits(cuda, case):
    lowrank_case(*LOWRANK[case], seed=case, bias=case % 3 != 1, scale=case % 4 != 2, xpad=8 * (case % 2),
                 ypad=case % 5, wpad=8 * (case % 3))


LOWRANK_EDGES = [
    ("bf16", "bf16", 2, 77, 264, 64, 3, "any"),
    ("f16", "f16", 3, 128, 1000, 8, 3, "any"),
    ("bf16", "f32", 8, 40, 2048, 32, 9, "any"),
    ("f16", "f32", 9, 2500, 64, 24, 4, "any"),
    ("bf16", "bf16", 65, 300, 136, 64, 70, "any"),
    ("f16", "f32", 127, 6522, 128, 16, 200, "any"),
    ("bf16", "f32", 128, 50, 80, 48, 128, "any"),
    ("bf16", "bf16", 129, 300, 136, 64, 140, "any"),
    ("f16", "f16", 513, 260, 72, 24, 9, "any"),
    ("bf16", "f32", 300, 130, 2304, 64, 5, "runs"),
    ("f16", "f32", 200, 3000, 1024, 64, 3, "runs"),
    ("bf16", "bf16", 6000, 1000, 64, 64, 40, "runs"),
]


@gpu
@pytest.mark.parametrize("case", range(len(LOWRANK_EDGES)))
def test_lowrank_row_counts_where_forms_change(cuda, case):
    lowrank_case(*LOWRANK_EDGES[case], seed=50 + case, bias=case % 2 == 0, scale=case % 3 != 1, xpad=8 * (case % 3),
                 ypad=(0, 1, 8)[case % 3], wpad=8 * (case % 2))


@gpu
@pytest.mark.parametrize("rows", [1, 9, 50, 300])
@pytest.mark.parametrize("out", ["f16", "f32"])
def test_lowrank_fp16_h_past_the_type(cuda, rows, out):
    """h is fp32: rows whose h passes fp16's largest value keep it, beside rows of the same adapter whose h does not"""
    gen, K, N, rank, slots = generator(rows), 256, 200, 16, 3
    x = rand(gen, rows, K)
    x[::3] *= 300.0
    x, w = x.half(), (rand(gen, N, K) * 2.0 ** -4).half()
    A, B = rand(gen, slots, rank, K).half(), (rand(gen, slots, N, rank) * 2.0 ** -11).half()
    s = torch.full((slots,), 60.0, device="cuda")
    slot = torch.randint(-1, slots, (rows,), device="cuda", generator=gen).int()
    slot[0] = 0
    y = torch.empty(rows, N, device="cuda", dtype=DT[out])
    op = sequence.LowRank("f16", out, N, K, w.data_ptr(), None, slots, rank, A.data_ptr(), B.data_ptr(), s.data_ptr(),
                          rows=rows)
    op.run(rows, x.data_ptr(), slot.data_ptr(), y.data_ptr())
    assert op.error == 0
    xd, wd = x.double(), w.double()
    want, M = xd @ wd.t(), xd.abs() @ wd.abs().t()
    most = 0.0
    for a in range(slots):
        at = torch.nonzero(slot == a).flatten()
        if not len(at):
            continue
        h = 60.0 * (xd[at] @ A[a].double().t())
        most = max(most, float(h.abs().max()))
        want[at] += h @ B[a].double().t()
        M[at] += 60.0 * ((xd[at].abs() @ A[a].double().abs().t()) @ B[a].double().abs().t())
    assert most > 65504.0
    check(y, want, (2.0 ** -15 + (K + rank + 4) * 2.0 ** -24) * M, out, "y")


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 16, 128, 129, 500])
@pytest.mark.parametrize("scale", [1.0, 1e-2, 1e-4, 1e-6])
def test_lowrank_keeps_h_of_any_size(cuda, dtype, rows, scale):
    """h is fp32 however small and however many rows share the call. Without W: the error is that of the two sums, K and
    rank terms of 2^-24 each at worst, in rms no more than 2^-24 times the root of their number (2^-20), twice that where
    the tensor cores cut sums off"""
    gen, K, N, rank, slots = generator(rows), 256, 130, 24, 3
    x, w = rand(gen, rows, K).to(DT[dtype]), torch.zeros(N, K, device="cuda", dtype=DT[dtype])
    A, B = (rand(gen, slots, rank, K) * 2.0 ** -4).to(DT[dtype]), rand(gen, slots, N, rank).to(DT[dtype])
    s = torch.full((slots,), scale, device="cuda")
    slot = torch.randint(0, slots, (rows,), device="cuda", generator=gen).int()
    y = torch.empty(rows, N, device="cuda")
    op = sequence.LowRank(dtype, "f32", N, K, w.data_ptr(), None, slots, rank, A.data_ptr(), B.data_ptr(), s.data_ptr(),
                          rows=rows)
    op.run(rows, x.data_ptr(), slot.data_ptr(), y.data_ptr())
    h = torch.einsum("rk,rjk->rj", x.double(), A.double()[slot.long()]) * s.double()[0]
    want = torch.einsum("rj,rnj->rn", h, B.double()[slot.long()])
    assert float((y.double() - want).norm() / want.norm()) < 2.0 ** -19
    assert op.error == 0


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows, K, adds", [(12, 1024, 16), (64, 1024, 16), (128, 1024, 16), (300, 4096, 64)])
def test_lowrank_fp32_outputs_are_fp32(cuda, dtype, rows, K, adds):
    """the error in rms of fp32 outputs: of chains of so many steps of the tensor cores (K / 16 over the form's accumulators),
    which cut off up to 2^-24 of the sum at each, half of it on average"""
    gen, N, rank, slots = generator(rows), 260, 16, 4
    x, w = rand(gen, rows, K).to(DT[dtype]), (rand(gen, N, K) * K ** -0.5).to(DT[dtype])
    A, B = (rand(gen, slots, rank, K) * K ** -0.5).to(DT[dtype]), rand(gen, slots, N, rank).to(DT[dtype])
    slot = torch.randint(-1, slots, (rows,), device="cuda", generator=gen).int()
    y = torch.empty(rows, N, device="cuda")
    op = sequence.LowRank(dtype, "f32", N, K, w.data_ptr(), None, slots, rank, A.data_ptr(), B.data_ptr(), rows=rows)
    op.run(rows, x.data_ptr(), slot.data_ptr(), y.data_ptr())
    want = x.double() @ w.double().t()
    for a in range(slots):
        at = torch.nonzero(slot == a).flatten()
        want[at] += (x[at].double() @ A[a].double().t()) @ B[a].double().t()
    assert float((y.double() - want).norm() / want.norm()) < adds * 2.0 ** -25


@gpu
@pytest.mark.parametrize("rank, out", [(8, "f32"), (24, "f16"), (64, "f32")])
def test_lowrank_fp16_tiles_of_both_kinds(cuda, rank, out):
    """blocks of rows whose h is ordinary, small, past fp16 or absent, several tiles for each SM: every block to the
    accuracy of its own size"""
    gen, rows, K, N, slots = generator(rank), 5001, 64, 3000, 5
    size = torch.tensor([1.0, 1e-3, 1.0, 3e4, 1e-5, 0.0], device="cuda")[torch.arange(rows, device="cuda") // 100 % 6]
    x, w = rand(gen, rows, K).half(), (rand(gen, N, K) * 2.0 ** -3).half()
    A, B = (rand(gen, slots, rank, K) * 2.0 ** -3).half(), (rand(gen, slots, N, rank) * 2.0 ** -6).half()
    # the size by the adapter's scale: adapter 5 a + b has scale sizes[b]
    sizes = torch.tensor([1.0, 1e-3, 3e4, 1e-5], device="cuda")
    A4, B4 = A.repeat_interleave(4, 0).contiguous(), B.repeat_interleave(4, 0).contiguous()
    s = sizes.repeat(slots)
    which = torch.stack([(size == v).int() * i for i, v in enumerate(sizes)]).sum(0)
    slot = torch.randint(0, slots, (rows,), device="cuda", generator=gen) * 4 + which
    slot = torch.where(size == 0, -1, slot).int()
    y = torch.empty(rows, N, device="cuda", dtype=DT[out])
    op = sequence.LowRank("f16", out, N, K, w.data_ptr(), None, 4 * slots, rank, A4.data_ptr(), B4.data_ptr(), s.data_ptr(),
                          rows=rows)
    op.run(rows, x.data_ptr(), slot.data_ptr(), y.data_ptr())
    assert op.error == 0
    xd, wd = x.double(), w.double()
    want, M = xd @ wd.t(), xd.abs() @ wd.abs().t()
    for a in range(4 * slots):
        at = torch.nonzero(slot == a).flatten()
        want[at] += s[a].double() * ((xd[at] @ A4[a].double().t()) @ B4[a].double().t())
        M[at] += s[a].double() * ((xd[at].abs() @ A4[a].double().abs().t()) @ B4[a].double().abs().t())
    check(y, want, (K + rank + 8) * 2.0 ** -23 * M, out, "y")  # the tensor cores cut off: 2^-23 a term


@gpu
@pytest.mark.parametrize("dtype, out", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("rows", [1, 12, 100, 128, 129, 300, 1000])
@pytest.mark.parametrize("where, value", [("a", math.nan), ("b", math.nan), ("b", math.inf), ("x", math.nan), ("scale", math.inf)])
@pytest.mark.parametrize("size", [1.0, 1e-3])
def test_lowrank_values_that_are_no_numbers(cuda, dtype, out, rows, where, value, size):
    """what is not finite in one adapter or one row stays in its rows, whatever shares the call"""
    gen, K, N, rank, slots = generator(rows), 72, 300, 24, 6
    x, w = rand(gen, rows, K).to(DT[dtype]), rand(gen, N, K).to(DT[dtype])
    A, B = (rand(gen, slots, rank, K) * 2.0 ** -3).to(DT[dtype]), rand(gen, slots, N, rank).to(DT[dtype])
    bias, s = rand(gen, N), torch.full((slots,), size, device="cuda")
    slot = torch.randint(-1, slots, (rows,), device="cuda", generator=gen).int()
    slot[:2] = torch.tensor([1, 2][:rows]).int()
    {"a": A[1, 3], "b": B[1, 7:20], "x": x[rows // 2], "scale": s[1:2]}[where][..., 0] = value
    y = torch.full((rows, N), 7.0, device="cuda", dtype=DT[out])
    op = sequence.LowRank(dtype, out, N, K, w.data_ptr(), bias.data_ptr(), slots, rank, A.data_ptr(), B.data_ptr(),
                          s.data_ptr(), rows=rows)
    op.run(rows, x.data_ptr(), slot.data_ptr(), y.data_ptr())
    assert op.error == 0
    xd, wd = x.double(), w.double()
    want, M = xd @ wd.t() + bias.double(), xd.abs() @ wd.abs().t() + bias.double().abs()
    for a in range(slots):
        at = torch.nonzero(slot == a).flatten()
        want[at] += (s[a].double() * (xd[at] @ A[a].double().t())) @ B[a].double().t()
        M[at] += (s[a].double() * (xd[at].abs() @ A[a].double().abs().t())) @ B[a].double().abs().t()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(y), fin)
    check(y[fin], want[fin], (2.0 ** -15 + (K + rank + 4) * 2.0 ** -24) * M[fin], out, "y")


@gpu
def test_lowrank_adapter_replaced_between_runs(cuda):
    """the adapters are read by every run: one that is written in stream order counts from the next run on"""
    gen = generator(1)
    x, w = rand(gen, 40, 64).bfloat16(), rand(gen, 96, 64).bfloat16()
    A, B = rand(gen, 2, 8, 64).bfloat16(), rand(gen, 2, 96, 8).bfloat16()
    slot = torch.zeros(40, device="cuda").int()
    y = torch.empty(40, 96, device="cuda")
    op = sequence.LowRank("bf16", "f32", 96, 64, w.data_ptr(), None, 2, 8, A.data_ptr(), B.data_ptr(), rows=40)
    op.run(40, x.data_ptr(), slot.data_ptr(), y.data_ptr())
    before = y.clone()
    B[0] = 0
    op.run(40, x.data_ptr(), slot.data_ptr(), y.data_ptr())
    assert not torch.equal(before, y)
    xd, wd = x.double(), w.double()
    check(y, xd @ wd.t(), 2.0 ** -17 * (xd.abs() @ wd.abs().t()), "f32", "without the adapter")


# ------------------------------------------------------------------ norms around a block


def norm_case(D, xtype, dtype, norm, gate, rows, seed, masked=False, f=True, vectors="all", pad=0, inplace=False,
              offset=0, outputs="both"):
    gen, t, xt = generator(seed), DT[dtype], DT[xtype]

    def matrix(ty, scale=1.0, shift=0.0):
        flat = torch.full((rows * (D + pad) + offset,), math.nan, device="cuda", dtype=ty)
        m = flat[offset:].view(rows, D + pad)[:, :D]
        m.copy_((rand(gen, rows, D) * scale + shift).to(ty))
        return m

    x, ff, g = matrix(xt), matrix(t, 3.0, 0.5), matrix(t, 2.0)
    live = None
    if masked:
        live = torch.rand(rows, device="cuda", generator=gen) > 0.3
        ff[~live] = math.nan
        g[~live] = math.inf
    vec = {k: None for k in ("wpost", "bpost", "gamma", "wpre", "bpre")}
    if vectors == "all":
        vec = {k: rand(gen, D) for k in vec}
    eps, alpha = 1e-5, 0.7
    op = sequence.NormGate(D, xtype, dtype, norm, gate, eps, alpha, **{k: None if v is None else v.data_ptr()
                                                                         for k, v in vec.items()})
    x0, f0 = x.clone(), ff.clone()
    xo, h = (x, ff) if inplace else (matrix(xt), matrix(t))
    op.run(rows, x.data_ptr(), ff.data_ptr() if f else None, g.data_ptr() if gate != "none" else None,
           xo.data_ptr() if outputs != "h" else None, h.data_ptr() if outputs != "xo" else None,
           live=None if live is None else live.data_ptr(), xs=D + pad, fs=D + pad, gs=D + pad, xos=D + pad, hs=D + pad)

    def normed(v, m, w, b):
        """norm(v) w + b and the sum of its terms' magnitudes, m those of v"""
        mean = v.mean(-1, keepdim=True) if norm == "layer" else 0.0
        mm = m.mean(-1, keepdim=True) if norm == "layer" else 0.0
        r = 1 / torch.sqrt((v - mean).pow(2).mean(-1, keepdim=True) + eps)
        w = 1.0 if w is None else w.double()
        b = torch.zeros((), device="cuda").double() if b is None else b.double()
        return (v - mean) * r * w + b, (m + mm) * r * abs(w) + b.abs()

    y, my = x0.double(), x0.double().abs()
    if f:
        fd = f0.double()
        gd = g.double()
        if live is not None:
            fd = torch.where(live[:, None], fd, 0.0)
            gd = torch.where(live[:, None], gd, 0.0)
        u, mu = normed(fd, fd.abs(), vec["wpost"], vec["bpost"])
        act = {"none": torch.ones_like(gd), "sigmoid": torch.sigmoid(gd), "silu": gd * torch.sigmoid(gd)}[gate]
        coef = alpha * (1.0 if vec["gamma"] is None else vec["gamma"].double()) * act
        keep = torch.ones(rows, 1, device="cuda").double() if live is None else live[:, None].double()
        y, my = y + keep * coef * u, my + keep * coef.abs() * mu
    # the sums are trees: a thread's own terms, then the lanes and warps; 2^-19: the exponential and reciprocal
    rel = 2.0 ** -19 + (D / 32 + 64) * 2.0 ** -24
    if outputs != "h":
        check(xo, y, rel * my, xtype, "x'")
    if outputs != "xo":
        hh, mh = normed(y, my, vec["wpre"], vec["bpre"])
        if live is not None:
            hh, mh = torch.where(live[:, None], hh, 0.0), torch.where(live[:, None], mh, 0.0)
        # the statistics of h see x' off by rel my: relative to its norm, at most as much again
        check(h, hh, 4 * rel * mh * (1 + my.pow(2).mean(-1, keepdim=True).sqrt()
                                     / (y.pow(2).mean(-1, keepdim=True).sqrt() + 1e-30)), dtype, "h")


@gpu
@pytest.mark.parametrize("D", [1, 7, 8, 64, 250, 256, 1000, 1021, 1024, 1536, 2040, 2048, 2056, 5001, 8192, 8200, 20000])
@pytest.mark.parametrize("types", [("f32", "bf16"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("norm, gate", [("rms", "silu"), ("layer", "sigmoid")])
def test_norm_gate_widths(cuda, D, types, norm, gate):
    if norm == "layer" and D == 1:
        pytest.skip("a layer norm of one value is its bias")
    norm_case(D, *types, norm, gate, rows=5, seed=D, masked=D % 3 == 0)


@gpu
@pytest.mark.parametrize("case", [
    dict(D=1024, rows=3000), dict(D=1536, rows=2500, masked=True), dict(D=136, rows=9001), dict(D=1021, rows=1300),
    dict(D=200, rows=1301, pad=3), dict(D=512, rows=33, offset=1), dict(D=512, rows=33, pad=8, offset=8),
    dict(D=1024, rows=9, inplace=True), dict(D=999, rows=9, inplace=True), dict(D=9000, rows=9, inplace=True),
    dict(D=1024, rows=9, vectors="none"), dict(D=700, rows=20, f=False), dict(D=9001, rows=3, f=False, masked=True),
    dict(D=64, rows=1300, outputs="h"), dict(D=64, rows=1, outputs="xo"), dict(D=2000, rows=1, masked=True)])
@pytest.mark.parametrize("norm, gate, types", [("rms", "none", ("bf16", "bf16")), ("layer", "silu", ("f32", "f16"))])
def test_norm_gate_forms(cuda, case, norm, gate, types):
    kw = dict(case)
    norm_case(kw.pop("D"), *types, norm, gate, kw.pop("rows"), seed=3, **kw)


@gpu
@pytest.mark.parametrize("case", [
    dict(D=192, offset=1), dict(D=193), dict(D=1021, offset=5, masked=True), dict(D=1023, pad=6), dict(D=200, offset=4, pad=4),
    dict(D=2041, offset=7), dict(D=2042), dict(D=777, inplace=True, masked=True), dict(D=1024, offset=3, inplace=True),
    dict(D=300, offset=2, vectors="none", outputs="h"), dict(D=509, f=False, pad=1), dict(D=255, outputs="xo", masked=True)])
@pytest.mark.parametrize("norm, gate, types", [("rms", "silu", ("bf16", "bf16")), ("layer", "sigmoid", ("f32", "f16")),
                                               ("layer", "none", ("f32", "f32"))])
def test_norm_gate_rows_that_start_anywhere(cuda, case, norm, gate, types):
    kw = dict(case)
    norm_case(kw.pop("D"), *types, norm, gate, rows=1301, seed=4, **kw)


@gpu
@pytest.mark.parametrize("gate", ["sigmoid", "silu"])
@pytest.mark.parametrize("D", [64, 1021, 9001])
def test_norm_gate_fp32_gates_of_any_size(cuda, D, gate):
    """u is 1 everywhere, so that x' is the gate: of fp32 g to a few roundings (the exponential's 2 ulp, the quotient's 2, the
    products'), however large g is"""
    x, f = torch.zeros(800, D, device="cuda"), torch.ones(800, D, device="cuda")
    g = torch.linspace(-80.0, 80.0, 800 * D, device="cuda").view(800, D)
    xo = torch.empty_like(x)
    op = sequence.NormGate(D, "f32", "f32", "rms", gate, eps=0.0)
    op.run(800, x.data_ptr(), f.data_ptr(), g.data_ptr(), xo.data_ptr(), None)
    want = torch.sigmoid(g.double()) * (g.double() if gate == "silu" else 1.0)
    # the norm of ones: its sum is exact, its root's reciprocal 2 ulp
    check(xo, want, 8 * 2.0 ** -23 * want.abs(), "f32", "gate")


@gpu
def test_norm_gate_zero_rows_and_zero_values(cuda):
    op = sequence.NormGate(64, "f32", "bf16", "rms", "none")
    x = torch.zeros(4, 64, device="cuda")
    f = torch.zeros(4, 64, device="cuda").bfloat16()
    xo, h = torch.full_like(x, 3), torch.full_like(f, 3)
    op.run(0, None, None, None, None, None)
    op.run(4, x.data_ptr(), f.data_ptr(), None, xo.data_ptr(), h.data_ptr())
    assert bool((xo == 0).all()) and bool((h == 0).all())


@gpu
def test_station_context_example(cuda):
    """the operators together: whole recordings against window by window. The two ways round h, q, k, v, o and f to bf16
    (2^-8 each) at different sums: some roundings' difference, in logits of about the weights' size"""
    import importlib.util  # pylint: disable=import-outside-toplevel
    import os  # pylint: disable=import-outside-toplevel
    from conftest import REPO  # pylint: disable=import-outside-toplevel
    spec = importlib.util.spec_from_file_location("station_context", os.path.join(REPO, "examples", "station_context.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.main() < 8 * 2.0 ** -8


# ------------------------------------------------------------------ streams


def busy(ms=50):
    """work of about so many ms on the current stream"""
    torch.cuda._sleep(int(ms * 1.9e6))  # pylint: disable=protected-access


@gpu
def test_op_made_while_the_default_stream_is_busy(cuda):
    """an op's set-up is over when it exists: its first run may be on a side stream, and what the default stream still has
    to do must not write into the op's memory after that"""
    gen, K, N, rank = generator(2), 64, 96, 8
    w, A, B = rand(gen, N, K).bfloat16(), rand(gen, 2, rank, K).bfloat16(), rand(gen, 2, N, rank).bfloat16()
    side = torch.cuda.Stream()
    for rows in (1, 9, 50, 300):
        x, slot = rand(gen, rows, K).bfloat16(), torch.zeros(rows, device="cuda").int()
        outs = []
        for late in (False, True):
            y = torch.empty(rows, N, device="cuda")
            torch.cuda.synchronize()
            if late:
                busy()
            op = sequence.LowRank("bf16", "f32", N, K, w.data_ptr(), None, 2, rank, A.data_ptr(), B.data_ptr(), rows=rows)
            op.run(rows, x.data_ptr(), slot.data_ptr(), y.data_ptr(), stream=side.cuda_stream)
            side.synchronize()
            outs.append(y)
            torch.cuda.synchronize()
        assert torch.equal(*outs), rows
    a = Attention("bf16", 2, 2, 64, 64, [150, 4], seed=13)
    s1 = torch.zeros_like(a.s0)
    a.run(a.op(), s1=s1)
    want, state = a.o.clone(), s1.clone()
    a.o.zero_()
    torch.cuda.synchronize()
    busy()
    op = a.op()
    a.run(op, s1=s1, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(a.o, want) and torch.equal(s1, state)


@gpu
def test_error_word_waits_for_the_runs(cuda):
    """the error word is that of every run issued before, on a non-blocking stream too"""
    a = Attention("bf16", 2, 2, 64, 64, [150, 4], seed=14)
    att = a.op()
    w, y = torch.zeros(16, 64, device="cuda").bfloat16(), torch.empty(4, 16, device="cuda")
    low = sequence.LowRank("bf16", "f32", 16, 64, w.data_ptr(), None, 1, 8, w.data_ptr(), w.data_ptr(), rows=4)
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    for op, run in ((att, lambda: a.run(att, stream=side.cuda_stream)),
                    (low, lambda: low.run(4, w.data_ptr(), None, y.data_ptr(), stream=side.cuda_stream))):
        run()  # a kernel's first launch may wait for the device
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            busy()
            run()
            done.record()
        assert not done.query()
        assert op.error == 0 and done.query()


# ------------------------------------------------------------------ refusals (no GPU needed)


def usage(make, text):
    with pytest.raises(BnnError) as e:
        make()
    assert e.value.kind == "USAGE" and text in str(e.value), str(e.value)


P = 1 << 20  # a pointer that is never followed: the checks come first


@pytest.mark.parametrize("kw, text", [
    (dict(dtype="f32"), "type fp16 or bf16"), (dict(dtype="f64"), "one of"), (dict(heads=3, kv_heads=2), "multiple of kv_heads"),
    (dict(dk=12), "multiples of 8"), (dict(dv=136), "up to 128"), (dict(dk=0), "multiples of 8"),
    (dict(decay=[1.5, 0.5]), "decay[0] = 1.5"), (dict(decay=[0.5, math.nan]), "decay[1]"), (dict(decay=[0.5, -0.1]), "decay[1]"),
    (dict(decay=[0.5]), "1 values for 2"), (dict(scale=math.inf), "a finite scale"), (dict(seqs=0), "at least one sequence"),
    (dict(tokens=1 << 31), "2^31 - 1"), (dict(tokens=0), "1 .. 2^31 - 1")])
def test_dattn_new_refuses(kw, text):
    a = dict(dtype="bf16", heads=2, kv_heads=2, dk=64, dv=64, decay=[0.9, 0.5])
    a.update(kw)
    usage(lambda: sequence.DecayAttention(**a), text)


@pytest.mark.parametrize("kw, text", [
    (dict(dtype="f32"), "type fp16 or bf16"), (dict(out="f16"), "out fp32 or the same"), (dict(K=12), "multiples of 8"),
    (dict(N=0), "N 0"), (dict(rank=12), "rank a multiple of 8"), (dict(rank=72), "8 .. 64"), (dict(slots=0), "slots 0"),
    (dict(rows=0), "rows 0"), (dict(w=P + 2), "16-byte aligned"), (dict(a=None), "16-byte aligned"),
    (dict(b=P + 8), "16-byte aligned"), (dict(ldw=56), "ldw >= K"), (dict(ldw=68), "multiples of 8")])
def test_lowrank_new_refuses(kw, text):
    a = dict(dtype="bf16", out="bf16", N=10, K=64, w=P, bias=None, slots=2, rank=8, a=P, b=P, rows=4)
    a.update(kw)
    usage(lambda: sequence.LowRank(**a), text)


@pytest.mark.parametrize("kw, text", [
    (dict(D=0), "D in 1"), (dict(xtype="f16"), "x_type fp32 or type"), (dict(norm="max"), "one of"),
    (dict(gate="tanh"), "one of"), (dict(eps=-1.0), "eps >= 0"), (dict(eps=math.nan), "eps >= 0"),
    (dict(alpha=math.inf), "finite")])
def test_norm_gate_new_refuses(kw, text):
    a = dict(D=64, xtype="f32", dtype="bf16")
    a.update(kw)
    usage(lambda: sequence.NormGate(**a), text)


def test_norm_gate_run_refuses():
    op = sequence.NormGate(64, "f32", "bf16", "rms", "silu")
    ok = dict(rows=2, x=P, f=P, g=P, xo=P, h=P)
    for kw, text in [(dict(rows=-1), "-1 rows"), (dict(x=None), "strides"), (dict(g=None), "g where f is given"),
                     (dict(xo=None, h=None), "an output"), (dict(xs=63), "strides >= the width"),
                     (dict(hs=10), "strides >= the width"), (dict(x=P + 2), "not aligned"), (dict(h=P + 1), "not aligned")]:
        usage(lambda kw=kw: op.run(**dict(ok, **kw)), text)
    op.run(0, None, None, None, None, None)
    op.close()
    with pytest.raises(BnnError):
        op.run(**ok)


@gpu
def test_run_refuses(cuda):
    op = sequence.DecayAttention("bf16", 4, 64, 32, [0.9, 0.5], kv_heads=2, seqs=2, tokens=10)
    ok = dict(n=2, tokens=10, cu=P, q=P, k=P, v=P, o=P)
    for kw, text in [(dict(n=3), "capacity 2"), (dict(n=-1), "capacity"), (dict(tokens=11), "capacity"), (dict(cu=None), "offsets"),
                     (dict(q=None), "16-byte aligned"), (dict(k=P + 8), "16-byte aligned"), (dict(s0=P + 4), "16-byte aligned"),
                     (dict(qts=255), "token strides"), (dict(kts=132), "token strides"), (dict(ots=127), "token strides")]:
        usage(lambda kw=kw: op.run(**dict(ok, **kw)), text)
    usage(lambda: op.step(3, P, P, P, P), "capacity 2")
    op.run(0, 0, None, None, None, None, None)
    op.step(0, None, None, None, None)
    w = torch.zeros(10, 64, device="cuda").bfloat16()
    low = sequence.LowRank("bf16", "f32", 10, 64, w.data_ptr(), None, 1, 8, w.data_ptr(), w.data_ptr(), rows=4)
    ok = dict(rows=4, x=P, slot=P, y=P)
    for kw, text in [(dict(rows=5), "capacity 4"), (dict(rows=-1), "capacity"), (dict(x=None), "16-byte aligned"),
                     (dict(x=P + 8), "16-byte aligned"), (dict(ldx=60), ">= K"), (dict(ldy=9), ">= N"), (dict(y=P + 2), "y")]:
        usage(lambda kw=kw: low.run(**dict(ok, **kw)), text)
    low.run(0, None, None, None)


@gpu
def test_new_reports_out_of_memory(cuda):
    h = load_library()
    w = torch.zeros(10, 64, device="cuda").bfloat16()
    try:
        for k in (1, 2):
            h.bnn_debug_fail_alloc(0, k)
            with pytest.raises(BnnError) as e:
                sequence.DecayAttention("bf16", 2, 64, 64, [0.9, 0.5])
            assert e.value.kind == "OOM"
            h.bnn_debug_fail_alloc(0, k)
            with pytest.raises(BnnError) as e:
                sequence.LowRank("bf16", "f32", 10, 64, w.data_ptr(), None, 1, 8, w.data_ptr(), w.data_ptr())
            assert e.value.kind == "OOM"
        h.bnn_debug_fail_alloc(1, 0)
        with pytest.raises(BnnError) as e:
            sequence.NormGate(64, "f32", "bf16")
        assert e.value.kind == "OOM"
    finally:
        h.bnn_debug_fail_alloc(0, 0)


# ------------------------------------------------------------------ the entry points' two forms, captured calls


def block(seed=0, n=5, lens=(3, 140, 0, 1, 260)):
    """one of each operator with its buffers: (objects, calls by the plain entry points, calls by the Python methods)"""
    a = Attention("bf16", 2, 2, 64, 64, list(lens), 0.2, seed=seed)
    att, s1 = a.op(), torch.zeros_like(a.s0)
    gen = generator(seed)
    x, w = rand(gen, 40, 64).bfloat16(), rand(gen, 96, 64).bfloat16()
    A, B = rand(gen, 2, 8, 64).bfloat16(), rand(gen, 2, 96, 8).bfloat16()
    slot, y = torch.randint(-1, 2, (40,), device="cuda", generator=gen).int(), torch.zeros(40, 96, device="cuda")
    low = sequence.LowRank("bf16", "f32", 96, 64, w.data_ptr(), None, 2, 8, A.data_ptr(), B.data_ptr(), rows=40)
    r, f, g = rand(gen, 30, 72), rand(gen, 30, 72).bfloat16(), rand(gen, 30, 72).bfloat16()
    ro, h = torch.zeros_like(r), torch.zeros_like(f)
    norm = sequence.NormGate(72, "f32", "bf16", "layer", "silu")
    b = Attention("bf16", 2, 2, 64, 64, [1] * n, seed=seed + 1)
    bs1 = torch.zeros_like(b.s0)
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731

    def plain(st):
        c = att.h
        assert not c.bnn_dattn_run(att.op, len(lens), sum(lens), p(a.cu), p(a.slot), p(a.live), p(a.q), a.ts, p(a.k), a.ts,
                                   p(a.v), a.ts, p(a.s0), p(s1), p(a.o), 128, st)
        assert not c.bnn_dattn_step(att.op, n, p(b.slot), None, p(b.q), b.ts, p(b.k), b.ts, p(b.v), b.ts, p(b.s0), p(bs1),
                                    p(b.o), 128, st)
        assert not c.bnn_lowrank_run(low.op, 40, p(x), 64, p(slot), p(y), 96, st)
        assert not c.bnn_norm_gate_run(norm.op, 30, p(r), 72, p(f), 72, p(g), 72, None, p(ro), 72, p(h), 72, st)

    def methods(st):
        a.run(att, s1=s1, stream=st)
        b.run(att, s1=bs1, stream=st, step=True)
        low.run(40, p(x), p(slot), p(y), stream=st)
        norm.run(30, p(r), p(f), p(g), p(ro), p(h), stream=st)

    return (x, w, A, B, att, low, norm, slot), (a.o, s1, b.o, bs1, y, ro, h), plain, methods


@gpu
def test_plain_entry_points_give_what_the_methods_give(cuda):
    keep, outs, plain, methods = block()
    st = torch.cuda.current_stream().cuda_stream
    methods(st)
    want = [t.clone() for t in outs]
    for t in outs:
        t.zero_()
    plain(st)
    assert all(torch.equal(t, w) for t, w in zip(outs, want))
    del keep


@gpu
def test_calls_in_a_captured_graph(cuda):
    keep, outs, _, methods = block(seed=3)
    methods(torch.cuda.current_stream().cuda_stream)
    want = [t.clone() for t in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        methods(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        for t in outs:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t, w) for t, w in zip(outs, want))
    del keep


def test_counts_past_an_int_are_refused():
    norm = sequence.NormGate(64, "f32", "bf16")
    usage(lambda: norm.run((1 << 32) + 1, 4096, None, None, 4096, None), "-1 rows")


@pytest.mark.parametrize("vector", ["wpost", "bpost", "gamma", "wpre", "bpre"])
def test_norm_gate_new_refuses_misaligned_vectors(vector):
    usage(lambda: sequence.NormGate(64, "f32", "bf16", **{vector: P + 2}), "vectors aligned")


@pytest.mark.parametrize("kw", [dict(bias=P + 2), dict(scale=P + 1)])
def test_lowrank_new_refuses_misaligned_vectors(kw):
    a = dict(dtype="bf16", out="bf16", N=10, K=64, w=P, bias=P, slots=2, rank=8, a=P, b=P, scale=P, rows=4)
    usage(lambda: sequence.LowRank(**dict(a, **kw)), "aligned to their elements")


def test_words_entry_points_refuse_no_words():
    h = load_library()
    norm = sequence.NormGate(64, "f32", "bf16")
    for call, op in ((h.bnn_dattn_run_words, None), (h.bnn_dattn_step_words, None), (h.bnn_lowrank_run_words, None),
                     (h.bnn_norm_gate_run_words, norm.op)):
        assert call(op, None) == -1
        e = last_error(h)
        assert e.kind == "USAGE" and "no arguments" in str(e)


@gpu
def test_run_refuses_misaligned_offsets_and_slots(cuda):
    """on the host: in a kernel such an address would be a fault"""
    op = sequence.DecayAttention("bf16", 4, 64, 32, [0.9, 0.5], kv_heads=2, seqs=2, tokens=10)
    ok = dict(n=2, tokens=10, cu=P, q=P, k=P, v=P, o=P)
    for kw in (dict(cu=P + 2), dict(slot=P + 2), dict(slot=P + 1)):
        usage(lambda kw=kw: op.run(**dict(ok, **kw)), "not aligned to their elements")
    usage(lambda: op.step(1, P, P, P, P, slot=P + 3), "not aligned to their elements")
    w = torch.zeros(10, 64, device="cuda").bfloat16()
    low = sequence.LowRank("bf16", "f32", 10, 64, w.data_ptr(), None, 1, 8, w.data_ptr(), w.data_ptr(), rows=4)
    usage(lambda: low.run(4, P, P + 2, P), "aligned to their elements")
