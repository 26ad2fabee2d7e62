"""The operators over sequences of windows, as they are measured: decayed linear attention (prompts and single
tokens), a shared projection with low-rank adapters per row, and the norms, gate and residual around a block.

Sizes are those of window embeddings: 1024 (v2.4) or 1536 (Perch v2) values a window, the v2.4 class head of 6522
classes, recordings of one window to a day of 3 s windows, one live station to some hundreds. `run` computes the plain
forms in fp32 with torch operations, or (own = True) calls the library's operators.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CHUNK = 128


def listed():
    return [
        # one live station, one new window: the latency of a single call
        {"name": "step 1 station", "op": "step", "dtype": "bf16", "n": 1, "hk": 8, "g": 1, "dk": 128, "dv": 128,
         "masked": False},
        # a server with some hundred stations in step, windows of a few of them failed
        {"name": "step 300 stations", "op": "step", "dtype": "f16", "n": 300, "hk": 16, "g": 1, "dk": 64, "dv": 64,
         "masked": True},
        # one recording of an hour in 3 s windows
        {"name": "prompt 1 hour", "op": "prompt", "dtype": "bf16", "n": 1, "len": 1200, "ragged": False, "hk": 8, "g": 1,
         "dk": 128, "dv": 128, "masked": False},
        # a batch of short recordings of different lengths with failed windows, shared k/v heads, a narrow odd head
        {"name": "prompts ragged", "op": "prompt", "dtype": "f16", "n": 37, "len": 611, "ragged": True, "hk": 4, "g": 3,
         "dk": 96, "dv": 72, "masked": True},
        # a night of recordings from 24 stations
        {"name": "prompts night", "op": "prompt", "dtype": "bf16", "n": 24, "len": 9600, "ragged": False, "hk": 16,
         "g": 1, "dk": 64, "dv": 64, "masked": False},
        # one station's whole day
        {"name": "prompt 1 day", "op": "prompt", "dtype": "bf16", "n": 1, "len": 28800, "ragged": False, "hk": 12, "g": 1,
         "dk": 128, "dv": 128, "masked": False},
        # one live window through the block's projection
        {"name": "adapters 1 row", "op": "lowrank", "dtype": "bf16", "out": "bf16", "rows": 1, "K": 1024, "N": 1024,
         "rank": 16, "slots": 16, "run": 1},
        # 64 stations in step, each with its own adapter of the class head, fp32 logits
        {"name": "adapters class head", "op": "lowrank", "dtype": "bf16", "out": "f32", "rows": 64, "K": 1024, "N": 6522,
         "rank": 16, "slots": 64, "run": 1},
        # prompts of several stations through the projection to q, k, v and the gate
        {"name": "adapters prompts", "op": "lowrank", "dtype": "f16", "out": "f16", "rows": 9001, "K": 1536, "N": 6144,
         "rank": 32, "slots": 12, "run": 700},
        # one live window around a block
        {"name": "norms 1 row", "op": "norm", "dtype": "bf16", "xtype": "f32", "rows": 1, "D": 1024, "kind": "rms",
         "gate": "silu", "masked": False},
        # an odd width, 16-bit residual stream, layer norm, failed windows
        {"name": "norms odd width", "op": "norm", "dtype": "f16", "xtype": "f16", "rows": 3000, "D": 1021,
         "kind": "layer", "gate": "sigmoid", "masked": True},
        # a day's windows of one station around a block
        {"name": "norms prompts", "op": "norm", "dtype": "bf16", "xtype": "f32", "rows": 28800, "D": 1536, "kind": "rms",
         "gate": "silu", "masked": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "prompt", "prompt", "lowrank", "lowrank", "norm"])
    dtype = rng.choice(["bf16", "f16"])
    if op in ("step", "prompt"):
        case = {"op": op, "dtype": dtype, "hk": rng.choice([1, 2, 4, 8, 12, 16]), "g": rng.choice([1, 1, 2, 3, 4]),
                "dk": 8 * rng.randint(2, 16), "dv": 8 * rng.randint(2, 16), "masked": rng.random() < 0.5}
        if rng.random() < 0.5:
            case["dk"] = case["dv"] = rng.choice([32, 64, 128])
        if op == "step":
            return dict(case, n=_log(rng, 1, 400))
        n = _log(rng, 1, 64)
        heads = case["hk"] * max(1, case["g"])
        # at most the day-long prompt's tokens x head widths
        most = 28800 * 12 * 128 // (heads * max(case["dk"], case["dv"]) * n)
        return dict(case, n=n, len=_log(rng, 1, max(1, min(40000, most))), ragged=rng.random() < 0.7)
    if op == "lowrank":
        rows = _log(rng, 1, 8500)
        return {"op": op, "dtype": dtype, "out": rng.choice([dtype, "f32"]), "rows": rows, "K": 8 * _log(rng, 16, 192),
                "N": _log(rng, 64, 6144), "rank": 8 * rng.randint(1, 8), "slots": _log(rng, 1, 32),
                "run": _log(rng, 1, 1000)}
    return {"op": op, "dtype": dtype, "xtype": rng.choice(["f32", dtype]), "rows": _log(rng, 1, 28800),
            "D": _log(rng, 64, 1536), "kind": rng.choice(["rms", "layer"]), "gate": rng.choice(["silu", "sigmoid", "none"]),
            "masked": rng.random() < 0.3}


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _lengths(case):
    """the recordings' lengths: a case's own, the same for every seed, from nothing up to the longest"""
    if not case["ragged"]:
        return [case["len"]] * case["n"]
    r = torch.Generator()
    r.manual_seed(case["len"] * 1000 + case["n"])
    return torch.randint(0, case["len"] + 1, (case["n"],), generator=r).tolist()[:-1] + [case["len"]]


def _live(tokens, masked, gen):
    """failed windows: about one in ten, none where masked is false"""
    return torch.rand(tokens, device=DEV, generator=gen) > 0.1 if masked else None


def _attention_inputs(case, tokens, states, seed):
    gen, t = _generator(seed), DTYPES[case["dtype"]]
    hk, h, dk, dv = case["hk"], case["hk"] * case["g"], case["dk"], case["dv"]

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    s = {"q": normal(tokens, h, dk).to(t), "k": normal(tokens, hk, dk).to(t), "v": normal(tokens, hk, dv).to(t),
         # heads that look back a few windows to some thousands
         "decay": (1 - 2.0 ** -torch.linspace(1, 10, hk)).float(), "scale": dk ** -0.5,
         "s0": normal(states, hk, dk, dv), "live": _live(tokens, case["masked"], gen)}
    if s["live"] is not None:  # a failed window holds no number
        for name in "qkv":
            s[name][~s["live"]] = math.nan
    s["decay_gpu"] = s["decay"].to(DEV)
    # the stations' states lie in the pool in an order of their own
    s["slot"] = torch.randperm(states, device=DEV, generator=gen).int()
    return s


def _lowrank_inputs(case, seed):
    gen, t = _generator(seed), DTYPES[case["dtype"]]
    rows, K, N, rank, slots = (case[k] for k in ("rows", "K", "N", "rank", "slots"))

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    runs = (rows + case["run"] - 1) // case["run"]
    of_run = torch.randint(-1, slots, (runs,), device=DEV, generator=gen)  # -1: a station without an adapter
    if case["run"] == 1 and rows <= slots:
        of_run = torch.randperm(slots, device=DEV, generator=gen)[:rows]
    return {"x": normal(rows, K).to(t), "w": (normal(N, K) * K ** -0.5).to(t), "bias": normal(N) * 0.1,
            "a": (normal(slots, rank, K) * K ** -0.5).to(t), "b": (normal(slots, N, rank) * rank ** -0.5).to(t),
            "scale": torch.rand(slots, device=DEV, generator=gen) + 0.5,
            "slot": of_run.repeat_interleave(case["run"])[:rows].int().contiguous()}


def _norm_inputs(case, seed):
    gen, t = _generator(seed), DTYPES[case["dtype"]]
    rows, D = case["rows"], case["D"]

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    s = {"x": normal(rows, D).to(DTYPES[case["xtype"]]), "f": (normal(rows, D) * 3 + 0.5).to(t), "eps": 1e-5,
         "g": normal(rows, D).to(t) if case["gate"] != "none" else None, "alpha": 0.5,
         "gamma": torch.rand(D, device=DEV, generator=gen), "wpost": 1 + 0.2 * normal(D), "wpre": 1 + 0.2 * normal(D),
         "bpost": None, "bpre": None, "live": _live(rows, case["masked"], gen)}
    if case["kind"] == "layer":
        s["bpost"], s["bpre"] = 0.1 * normal(D), 0.1 * normal(D)
    if s["live"] is not None:
        s["f"][~s["live"]] = math.nan
    return s


def _inputs(case, seed):
    if case["op"] == "step":
        return _attention_inputs(case, case["n"], case["n"], seed)
    if case["op"] == "prompt":
        lens = _lengths(case)
        s = _attention_inputs(case, sum(lens), case["n"], seed)
        s["lens"] = lens
        s["cu"] = torch.tensor([0] + lens).cumsum(0).int().to(DEV)
        return s
    return _lowrank_inputs(case, seed) if case["op"] == "lowrank" else _norm_inputs(case, seed)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        _prepare_own(case, s)
    return s


def run(s):
    return (_RUN_OWN if own else _RUN_PLAIN)[s["case"]["op"]](s)


# ------------------------------------------------------------------ the library's operators


def _prepare_own(case, s):
    """the operator objects and output buffers that a program keeps"""
    import sys  # pylint: disable=import-outside-toplevel
    if "birdnet-neon-engine_b200" not in sys.path:
        sys.path.insert(0, "birdnet-neon-engine_b200")
    from bnneon_b200 import sequence  # pylint: disable=import-outside-toplevel
    t = DTYPES[case["dtype"]]
    if case["op"] in ("step", "prompt"):
        hk, h = case["hk"], case["hk"] * case["g"]
        s["op"] = sequence.DecayAttention(case["dtype"], h, case["dk"], case["dv"], s["decay"].numpy(), kv_heads=hk,
                                          scale=s["scale"], seqs=case["n"], tokens=s["q"].shape[0])
        s["o"] = torch.empty(s["q"].shape[0], h, case["dv"], dtype=t, device=DEV)
        s["s1"] = torch.empty_like(s["s0"])
    elif case["op"] == "lowrank":
        s["op"] = sequence.LowRank(case["dtype"], case["out"], case["N"], case["K"], s["w"].data_ptr(),
                                   s["bias"].data_ptr(), case["slots"], case["rank"], s["a"].data_ptr(),
                                   s["b"].data_ptr(), s["scale"].data_ptr(), rows=case["rows"])
        s["y"] = torch.empty(case["rows"], case["N"], dtype=DTYPES[case["out"]], device=DEV)
    else:
        s["op"] = sequence.NormGate(case["D"], case["xtype"], case["dtype"], case["kind"], case["gate"], s["eps"],
                                    s["alpha"], wpost=s["wpost"].data_ptr(), gamma=s["gamma"].data_ptr(),
                                    wpre=s["wpre"].data_ptr(), bpost=_at(s["bpost"]), bpre=_at(s["bpre"]))
        s["xo"], s["h"] = torch.empty_like(s["x"]), torch.empty_like(s["f"])


def _at(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_step(s):
    s["op"].step(s["q"].shape[0], s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["o"].data_ptr(),
                 s["s0"].data_ptr(), s["s1"].data_ptr(), slot=s["slot"].data_ptr(), live=_at(s["live"]), stream=_stream())
    return s["o"], s["s1"]


def _own_prompt(s):
    s["op"].run(len(s["lens"]), s["q"].shape[0], s["cu"].data_ptr(), s["q"].data_ptr(), s["k"].data_ptr(),
                s["v"].data_ptr(), s["o"].data_ptr(), s["s0"].data_ptr(), s["s1"].data_ptr(), slot=s["slot"].data_ptr(),
                live=_at(s["live"]), stream=_stream())
    return s["o"], s["s1"]


def _own_lowrank(s):
    s["op"].run(s["x"].shape[0], s["x"].data_ptr(), s["slot"].data_ptr(), s["y"].data_ptr(), stream=_stream())
    return s["y"]


def _own_norm(s):
    s["op"].run(s["x"].shape[0], s["x"].data_ptr(), s["f"].data_ptr(), _at(s["g"]), s["xo"].data_ptr(), s["h"].data_ptr(),
                live=_at(s["live"]), stream=_stream())
    return s["xo"], s["h"]


_RUN_OWN = {"step": _own_step, "prompt": _own_prompt, "lowrank": _own_lowrank, "norm": _own_norm}


# ------------------------------------------------------------------ the plain forms


def _plain_step(s):
    case = s["case"]
    n, hk, g = case["n"], case["hk"], case["g"]
    q, k, v, slot = s["q"].float(), s["k"].float(), s["v"].float(), s["slot"].long()
    live = torch.ones(n, dtype=torch.bool, device=DEV) if s["live"] is None else s["live"]
    q, k, v = (torch.where(live[:, None, None], t, 0.0) for t in (q, k, v))
    new = s["decay_gpu"][:, None, None] * s["s0"][slot] + k[..., :, None] * v[..., None, :]
    o = s["scale"] * torch.matmul(q.view(n, hk, g, -1), new)
    s1 = torch.empty_like(s["s0"])
    s1[slot] = new
    return o.view(n, hk * g, -1).to(s["q"].dtype), s1


def _plain_prompt(s):
    """chunked: products inside the chunks, a decayed sum over the chunks' states"""
    case = s["case"]
    n, hk, g, dk, dv = (case[k] for k in ("n", "hk", "g", "dk", "dv"))
    cu, slot, lam = s["cu"].long(), s["slot"].long(), s["decay_gpu"]
    chunks = max(1, -(-max(s["lens"]) // CHUNK))
    t = torch.arange(chunks * CHUNK, device=DEV)
    length = cu[1:] - cu[:-1]
    inside = t < length[:, None]
    tokens = s["q"].shape[0]
    at = torch.where(inside, cu[:-1, None] + t, tokens - 1)
    live = inside if s["live"] is None else inside & s["live"][at]
    keep = live[..., None, None]
    # [sequence][chunk][head][token][...], the q heads of one k/v head side by side
    q = torch.where(keep, s["q"][at].float(), 0.0).view(n, chunks, CHUNK, hk, g, dk).permute(0, 1, 3, 4, 2, 5)
    k = torch.where(keep, s["k"][at].float(), 0.0)
    v = torch.where(keep, s["v"][at].float(), 0.0)
    kc, vc = (x.view(n, chunks, CHUNK, hk, -1).transpose(2, 3) for x in (k, v))
    i = torch.arange(CHUNK, device=DEV)
    power = torch.where(i[:, None] >= i, lam[:, None, None] ** (i[:, None] - i).clamp(min=0), 0.0)
    p = torch.matmul(q, kc.transpose(-1, -2)[:, :, :, None]) * power[:, None]
    o = torch.matmul(p, vc[:, :, :, None])
    # the states before each chunk
    own_sum = torch.matmul((kc * lam[:, None, None] ** (CHUNK - 1 - i)[:, None]).transpose(-1, -2), vc)
    c = torch.arange(chunks, device=DEV)
    back = c[:, None] - 1 - c
    over = torch.where(back >= 0, lam[:, None, None] ** (CHUNK * back.clamp(min=0)), 0.0)
    s0 = s["s0"][slot]
    before = torch.matmul(over, own_sum.permute(0, 2, 1, 3, 4).reshape(n, hk, chunks, dk * dv)).view(n, hk, chunks, dk, dv)
    before = before + lam[:, None, None, None] ** (CHUNK * c)[:, None, None] * s0[:, :, None]
    o = o + lam[:, None, None, None] ** (i + 1)[:, None] * torch.matmul(q, before.transpose(1, 2)[:, :, :, None])
    o = (s["scale"] * o).permute(0, 1, 4, 2, 3, 5).reshape(n, chunks * CHUNK, hk * g, dv)
    out = o[inside].to(s["q"].dtype)
    # the states after the last token
    rest = (length[:, None] - 1 - t).clamp(min=0)
    w = lam ** rest[..., None]
    last = torch.matmul((k * w[..., None]).permute(0, 2, 3, 1), v.transpose(1, 2))
    s1 = torch.empty_like(s["s0"])
    s1[slot] = (lam ** length[:, None])[..., None, None] * s0 + last
    return out, s1


def _plain_lowrank(s):
    case = s["case"]
    x, slots, rank = s["x"].float(), case["slots"], case["rank"]
    hidden = torch.matmul(x, s["a"].float().view(slots * rank, -1).t()).view(-1, slots, rank)
    mine = torch.arange(slots, device=DEV) == s["slot"][:, None]
    hidden = (hidden * (mine * s["scale"])[..., None]).view(-1, slots * rank)
    up = s["b"].float().transpose(1, 2).reshape(slots * rank, -1)
    y = torch.matmul(x, s["w"].float().t()) + s["bias"] + torch.matmul(hidden, up)
    return y.to(DTYPES[case["out"]])


def _plain_norm(s):
    case = s["case"]

    def norm(v, w, b):
        if case["kind"] == "layer":
            v = v - v.mean(-1, keepdim=True)
        v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + s["eps"]) * w
        return v if b is None else v + b

    x, u = s["x"].float(), norm(s["f"].float(), s["wpost"], s["bpost"])
    if s["g"] is not None:
        g = s["g"].float()
        gate = 1 / (1 + torch.exp(-g))
        u = u * (g * gate if case["gate"] == "silu" else gate)
    x2 = x + s["alpha"] * s["gamma"] * u
    h = norm(x2, s["wpre"], s["bpre"])
    if s["live"] is not None:
        x2, h = torch.where(s["live"][:, None], x2, x), torch.where(s["live"][:, None], h, 0.0)
    return x2.to(s["x"].dtype), h.to(s["f"].dtype)


_RUN_PLAIN = {"step": _plain_step, "prompt": _plain_prompt, "lowrank": _plain_lowrank, "norm": _plain_norm}


# ------------------------------------------------------------------ the definitions in 64 bits


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] in ("step", "prompt"):
        return _exact_attention(case, s)
    return _exact_lowrank(case, s) if case["op"] == "lowrank" else _exact_norm(case, s)


def _exact_attention(case, s):
    """token by token: S = decay S + k^T v, o = scale q S"""
    n, hk, g = case["n"], case["hk"], case["g"]
    lens = s.get("lens", [1] * n)
    tokens = s["q"].shape[0]
    start = torch.tensor([0] + lens).cumsum(0)[:-1].to(DEV)
    length = torch.tensor(lens, device=DEV)
    ok = torch.ones(tokens, dtype=torch.bool, device=DEV) if s["live"] is None else s["live"]
    q, k, v = (torch.where(ok[:, None, None], s[x].double(), 0.0) for x in "qkv")
    state = s["s0"].double()[s["slot"].long()]
    lam = s["decay"].double().to(DEV)[:, None, None]
    o = torch.zeros(tokens, hk * g, case["dv"], dtype=torch.float64, device=DEV)
    # sequences in order of length, so that those at work at any time come first
    order = torch.argsort(length, descending=True)
    by_len = sorted(lens, reverse=True)
    state, start = state[order], start[order]
    m = n
    for t in range(by_len[0]):
        while by_len[m - 1] <= t:
            m -= 1
        at = start[:m] + t
        now = state[:m]
        now.mul_(lam).add_(k[at][..., :, None] * v[at][..., None, :])
        o[at] = s["scale"] * torch.einsum("nhgd,nhde->nhge", q[at].view(m, hk, g, -1), now).reshape(m, hk * g, -1)
    s1 = torch.empty_like(state)
    s1[s["slot"].long()[order]] = state
    return o, s1


def _exact_lowrank(case, s):
    x, slot = s["x"].double(), s["slot"].long()
    y = x @ s["w"].double().t() + s["bias"].double()
    for a in range(case["slots"]):
        rows = torch.nonzero(slot == a).flatten()
        if len(rows):
            y[rows] += s["scale"][a].double() * ((x[rows] @ s["a"][a].double().t()) @ s["b"][a].double().t())
    return y


def _exact_norm(case, s):
    def norm(v, w, b):
        if case["kind"] == "layer":
            v = v - v.mean(-1, keepdim=True)
        v = v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + s["eps"]) * w.double()
        return v if b is None else v + b.double()

    x = s["x"].double()
    u = norm(s["f"].double(), s["wpost"], s["bpost"])
    if case["gate"] != "none":
        g = s["g"].double()
        u = u * torch.sigmoid(g) * (g if case["gate"] == "silu" else 1.0)
    y = x + s["alpha"] * s["gamma"].double() * u
    h = norm(y, s["wpre"], s["bpre"])
    if s["live"] is not None:
        y, h = torch.where(s["live"][:, None], y, x), torch.where(s["live"][:, None], h, torch.zeros_like(h))
    return y, h


# ------------------------------------------------------------------ the work that cannot be left out


def work(case):
    if case["op"] in ("step", "prompt"):
        n, hk, g, dk, dv = (case[k] for k in ("n", "hk", "g", "dk", "dv"))
        tokens = n
        if case["op"] == "prompt":
            tokens = case["len"] * n if not case["ragged"] else case["len"] * (n - 1) // 2 + case["len"]
        moved = tokens * 2 * (hk * (dk + dv) + hk * g * (dk + dv) + (0.5 if case["masked"] else 0))
        # the state's update and its product with q, for each token
        return {"bytes": moved + 2 * 4 * n * hk * dk * dv, "flops": tokens * hk * (2 + 2 * g) * dk * dv}
    if case["op"] == "lowrank":
        rows, K, N, rank = (case[k] for k in ("rows", "K", "N", "rank"))
        used = min(case["slots"], -(-rows // case["run"]))
        out = 4 if case["out"] == "f32" else 2
        return {"bytes": 2 * (rows * K + N * K + used * rank * (K + N)) + rows * N * out + 4 * (N + rows),
                "flops": 2 * rows * (K * N + rank * (K + N))}
    rows, D = case["rows"], case["D"]
    x = 4 if case["xtype"] == "f32" else 2
    return {"bytes": rows * D * (2 * x + 2 + 2 + (2 if case["gate"] != "none" else 0)) + 12 * D,
            "flops": 16 * rows * D}
