"""Context across windows, for many stations at once.

The model scores windows one by one. This puts one block on its embeddings that looks back over the windows of a
station: norm, projection to q, k, v and a gate with the station's own low-rank adapter, linear attention with a decay
per head (its state is kept per station), output projection, norm, gate and residual, and a class head with the
station's adapter again. A recording goes through in one call; a live station adds a window at a time and gets what the
whole recording gives.

    python examples/station_context.py [package.bnpk]     (without one: a small synthetic v2.4 package)

The block's weights here are random: the program shows the calls and checks the two ways against each other.
"""
import os
import sys
import tempfile

import numpy as np
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(REPO, "birdnet-neon-engine_b200"))

from bnneon_b200 import Model, sequence, synth  # noqa: E402  pylint: disable=wrong-import-position

HEADS, RANK = 8, 16
BF16 = torch.bfloat16


class ContextBlock:
    """Weights, operators and the stations' states. rows, stations: the most windows and stations of a call."""

    def __init__(self, width, classes, stations, rows, seed=0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)

        def normal(*shape, scale=1.0, dtype=BF16):
            return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)

        self.width, self.classes, self.stations = width, classes, stations
        d = width // HEADS
        self.keep = []  # the operators hold pointers to the weights

        def lowrank(n, out):
            w = normal(n, width, scale=width ** -0.5)
            a, b = normal(stations, RANK, width, scale=width ** -0.5), normal(stations, n, RANK, scale=0.1 * RANK ** -0.5)
            bias = normal(n, scale=0.1, dtype=torch.float32)
            self.keep += [w, a, b, bias]
            return sequence.LowRank("bf16", out, n, width, w.data_ptr(), bias.data_ptr(), stations, RANK, a.data_ptr(),
                                    b.data_ptr(), rows=rows)

        ones = torch.ones(width, device="cuda")
        self.keep.append(ones)
        at = ones.data_ptr()
        self.norm = sequence.NormGate(width, "f32", "bf16", "rms", "silu", alpha=0.5, wpost=at, gamma=at, wpre=at)
        self.project, self.out, self.head = lowrank(4 * width, "bf16"), lowrank(width, "bf16"), lowrank(classes, "f32")
        decay = 1 - 2.0 ** -np.linspace(2, 9, HEADS)  # heads that look back some windows to some hundred
        self.attend = sequence.DecayAttention("bf16", HEADS, d, d, decay, seqs=stations, tokens=rows)
        self.state = torch.zeros(stations, HEADS, d, d, device="cuda")
        self.h, self.f, self.o = (torch.empty(rows, width, device="cuda", dtype=BF16) for _ in range(3))
        self.qkvg = torch.empty(rows, 4 * width, device="cuda", dtype=BF16)
        self.x2 = torch.empty(rows, width, device="cuda")
        self.logits = torch.empty(rows, classes, device="cuda")

    def __call__(self, x, station_of_row, live, stations, lengths=None):
        """x [rows][width] fp32: the stations' windows, one station's after another's (lengths), or one window a station
        (lengths None). live [rows]: False for a window that failed. Returns logits [rows][classes]."""
        w, n, s = self.width, x.shape[0], torch.cuda.current_stream().cuda_stream
        rows, alive = station_of_row.data_ptr(), live.data_ptr()
        self.norm.run(n, x.data_ptr(), None, None, None, self.h.data_ptr(), live=alive, stream=s)
        self.project.run(n, self.h.data_ptr(), rows, self.qkvg.data_ptr(), stream=s)
        q, k, v, gate = (self.qkvg.data_ptr() + 2 * w * i for i in range(4))  # parts of the projection's rows
        kw = dict(slot=stations.data_ptr(), live=alive, qts=4 * w, kts=4 * w, vts=4 * w, stream=s)
        at = self.state.data_ptr()
        if lengths is None:
            self.attend.step(n, q, k, v, self.o.data_ptr(), at, at, **kw)
        else:
            cu = torch.tensor([0] + lengths, device="cuda").cumsum(0).int()
            self.attend.run(len(lengths), n, cu.data_ptr(), q, k, v, self.o.data_ptr(), at, at, **kw)
        self.out.run(n, self.o.data_ptr(), rows, self.f.data_ptr(), stream=s)
        self.norm.run(n, x.data_ptr(), self.f.data_ptr(), gate, self.x2.data_ptr(), self.h.data_ptr(), live=alive,
                      gs=4 * w, stream=s)
        self.head.run(n, self.h.data_ptr(), rows, self.logits.data_ptr(), stream=s)
        return self.logits[:n].clone()


def main(package=None, lengths=(40, 17, 1, 25, 33, 8)):
    """Returns the largest difference of the two ways' logits, relative to their size."""
    lengths = list(lengths)
    with tempfile.TemporaryDirectory() as tmp:
        if package is None:
            package = os.path.join(tmp, "mini.bnpk")
            synth.make_package(package, seed=1, mini=True)
        with Model(package, batch=64) as m:
            width, classes = m.info.emb_dim, m.info.n_classes
            pcm = synth.audio(sum(lengths), seed=3, n_samples=m.info.n_samples, rate=m.info.sample_rate)
            _, emb = m.infer_batch(pcm)
    x = torch.from_numpy(emb).cuda()
    live = torch.ones(len(x), dtype=torch.bool, device="cuda")
    live[5] = live[lengths[0] + 3] = False  # two windows failed
    x[5] = float("nan")
    stations = torch.arange(len(lengths), device="cuda").int()
    of_row = stations.repeat_interleave(torch.tensor(lengths, device="cuda")).contiguous()

    block = ContextBlock(width, classes, len(lengths), len(x))
    whole = block(x, of_row, live, stations, lengths)

    block.state.zero_()
    start = np.concatenate([[0], np.cumsum(lengths)[:-1]])
    steps = torch.empty_like(whole)
    for t in range(max(lengths)):
        now = [i for i, n in enumerate(lengths) if t < n]
        at = torch.tensor([int(start[i]) + t for i in now], device="cuda")
        who = stations[now].contiguous()
        steps[at] = block(x[at].contiguous(), who, live[at].contiguous(), who)
    torch.cuda.synchronize()
    for op in (block.attend, block.project, block.out, block.head):
        if op.error:
            raise RuntimeError("a bounded device wait ran out")
    off = float((steps - whole).abs().max() / whole.abs().max())
    print(f"{len(lengths)} stations, {len(x)} windows: whole recordings against window by window, logits off by {off:.2g}")
    return off


if __name__ == "__main__":
    main(*sys.argv[1:2])
