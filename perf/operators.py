"""Grouped products and the 4-bit gallery: cases, plain forms and 64-bit definitions.

Four operators over rows that fall into groups of unequal sizes:

  affine  y_r = x_r W_e + b_e for the rows r of group e, optionally length-normalised
          (one pre-processing / projection matrix per recording or domain);
  score   S_e = G1_e G2_e^T, one block of log-likelihood ratios per group;
  gram    C_e = sum_r x_r x_r^T and F_e = sum_r x_r per group, in float64;
  q4      S_e = T_e Q_e^T + additive terms against a gallery whose rows are held as 4-bit codes with one
          scale per 32 coordinates.

`own` selects between elementary torch operations (False) and the calls of hyperion_amd.engine (True)."""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "fp64": torch.float64}
Q4_GROUP = 32


def listed():
    return [
        # a service that answers single requests: one or two vectors for each of a few domains
        dict(name="affine_requests", op="affine", groups=8, low=1, high=2, shape=1, d_in=512, d_out=200, lnorm=True,
             dtype="fp32", routed=True),
        # the recordings of a diarization batch, each with its own projection of odd width
        dict(name="affine_recordings", op="affine", groups=200, low=12, high=420, shape=2, d_in=200, d_out=77,
             lnorm=True, dtype="fp32", routed=False),
        # a large evaluation set of a few domains, vectors as a bf16 extractor leaves them on the device
        dict(name="affine_domains", op="affine", groups=6, low=9000, high=60000, shape=3, d_in=512, d_out=200,
             lnorm=False, dtype="bf16", routed=True),
        # the same from fp32 vectors, kept in order
        dict(name="affine_evaluation", op="affine", groups=24, low=2000, high=16000, shape=4, d_in=512, d_out=150,
             lnorm=False, dtype="fp32", routed=False),
        # one short recording with a few segments: latency
        dict(name="score_short", op="score", groups=3, low=2, high=40, shape=5, k=40, cross=False),
        # a batch of recordings, every segment against every other of its recording
        dict(name="score_recordings", op="score", groups=200, low=12, high=900, shape=6, k=150, cross=False),
        # trials of several domains: enrolment and test vectors of one domain against each other
        dict(name="score_domains", op="score", groups=12, low=300, high=20000, shape=7, k=150, cross=True),
        # moments of a few short recordings (the PCA of a recording)
        dict(name="gram_short", op="gram", groups=4, low=15, high=60, shape=8, d=128, dtype="fp32"),
        # moments of a batch of recordings
        dict(name="gram_recordings", op="gram", groups=200, low=12, high=900, shape=9, d=200, dtype="fp32"),
        # per-domain covariances of a training set held in double precision
        dict(name="gram_training", op="gram", groups=7, low=3000, high=30000, shape=10, d=512, dtype="fp64"),
        # one request against a gallery of a million
        dict(name="q4_million", op="q4", groups=1, low=1000000, high=1000000, shape=11, k=150, t_low=1, t_high=1),
        # partitions of a gallery, a handful of requests for each (some have none)
        dict(name="q4_partitions", op="q4", groups=40, low=500, high=30000, shape=12, k=150, t_low=0, t_high=40),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["affine", "score", "gram", "q4"])
        groups = _log_int(rng, 1, 300)
        low = _log_int(rng, 1, 500)
        high = max(low, _log_int(rng, 1, 20000))
        case = dict(op=op, groups=groups, low=low, high=high, shape=rng.randrange(1 << 30))
        if op == "affine":
            case.update(d_in=_log_int(rng, 40, 1024), d_out=_log_int(rng, 10, 512), lnorm=rng.random() < 0.5,
                        dtype=rng.choice(["fp32", "fp16", "bf16"]), routed=rng.random() < 0.5)
        elif op == "score":
            case.update(k=rng.randrange(10, 310), cross=rng.random() < 0.5)
        elif op == "gram":
            case.update(d=_log_int(rng, 20, 600), dtype=rng.choice(["fp32", "fp64"]))
        else:
            case.update(k=rng.randrange(10, 310), t_low=rng.randrange(0, 3), t_high=rng.randrange(3, 100))
        w = work(case)
        if all(w[key] <= max(work(c)[key] for c in listed() if c["op"] == op) for key in w):
            return case


# ---------------------------------------------------------------------------------------------- shapes
def _sizes(case):
    """Rows of every group; where there are several, one group in ten is empty and one in ten has one row."""
    rng = random.Random(case["shape"])
    sizes = []
    for _ in range(case["groups"]):
        n = _log_int(rng, case["low"], case["high"])
        if case["groups"] > 3 and case["low"] > 2:
            u = rng.random()
            n = 0 if u < 0.1 else 1 if u < 0.2 else n
        sizes.append(n)
    return sizes


def _other_sizes(case, sizes):
    """The other side of a product: the same rows, other rows of the same groups, or requests."""
    rng = random.Random(case["shape"] + 1)
    if case["op"] == "q4":
        t = [rng.randint(case["t_low"], case["t_high"]) for _ in sizes]
        return t if sum(t) else [1] + t[1:]
    if not case["cross"]:
        return list(sizes)
    return [max(1, n // rng.randint(2, 9)) for n in sizes]


def _offsets(sizes):
    out = [0]
    for n in sizes:
        out.append(out[-1] + n)
    return out


def _width(k):
    return (k + 2 + 7) // 8 * 8


def _blocks(a, b):
    return sum(x * y for x, y in zip(a, b))


def work(case):
    sizes = _sizes(case)
    n, used = sum(sizes), sum(1 for s in sizes if s)
    item = torch.empty(0, dtype=DTYPES[case.get("dtype", "fp32")]).element_size()
    if case["op"] == "affine":
        di, do = case["d_in"], case["d_out"]
        return {"bytes": n * di * item + used * (di + 1) * do * 4 + n * do * 4 + (4 * n if case["routed"] else 0),
                "flops": 2 * n * di * do}
    if case["op"] == "gram":
        d = case["d"]
        return {"bytes": n * d * item + len(sizes) * (d * d + d) * 8, "flops": n * d * (d + 1)}
    other = _other_sizes(case, sizes)
    cells, k = _blocks(sizes, other), case["k"]
    if case["op"] == "score":
        return {"bytes": 4 * ((n + sum(other)) * (k + 2) + cells), "flops": 2 * k * cells}
    live = sum(s for s, t in zip(sizes, other) if t)
    row = k / 2 + 2 * math.ceil(k / Q4_GROUP) + 4
    return {"bytes": int(live * row) + 4 * (sum(other) * (k + 2) + cells), "flops": 2 * k * cells}


# ---------------------------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    """Everything that is random, on the GPU, from the seed."""
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def spread(d):
        # coordinates of embeddings and latent vectors differ in scale by about a factor of ten
        return torch.exp(1.2 * (torch.rand(d, generator=gen, device="cuda") - 0.5) * 2)

    sizes = _sizes(case)
    n, E = sum(sizes), len(sizes)
    if case["op"] == "affine":
        di, do = case["d_in"], case["d_out"]
        x = (normal(n, di) * spread(di)).to(DTYPES[case["dtype"]])
        W = normal(E, di, do) * (spread(do) / math.sqrt(di))
        b = 0.3 * normal(E, do)
        order = torch.randperm(n, generator=gen, device="cuda") if case["routed"] else None
        return dict(x=x, W=W, b=b, order=order)
    if case["op"] == "gram":
        x = normal(n, case["d"]) * spread(case["d"]) + 0.5 * normal(1, case["d"])
        return dict(x=x.to(DTYPES[case["dtype"]]))
    other = _other_sizes(case, sizes)
    k, kp = case["k"], _width(case["k"])
    scale = spread(k)

    def packed(rows, enrol):
        G = torch.zeros(rows, kp, device="cuda")
        G[:, :k] = normal(rows, k) * scale
        G[:, k + (0 if enrol else 1)] = -0.25 * (G[:, :k] * G[:, :k]).sum(1) * (0.2 + 0.1 * normal(rows))
        G[:, k + (1 if enrol else 0)] = 1.0
        return G

    return dict(G1=packed(n, True), G2=packed(sum(other), False))


def _plain_q4(G, k):
    """4-bit codes (two to a byte, 8 stands for zero), scales and additive terms of packed rows.  The scale
    of 32 coordinates is the smallest bfloat16 number s with 7 s >= the largest magnitude, a code is the
    integer nearest to x / s, halves to even; 64 bits, because a quotient may lie next to a half."""
    n, ng = G.shape[0], (k + Q4_GROUP - 1) // Q4_GROUP
    codes = torch.empty(n, ng * Q4_GROUP // 2, dtype=torch.uint8, device=G.device)
    scales = torch.empty(n, ng, dtype=torch.float32, device=G.device)
    for r0 in range(0, n, 1 << 18):
        g = G[r0:r0 + (1 << 18), :k]
        x = torch.zeros(g.shape[0], ng * Q4_GROUP, dtype=torch.float64, device=G.device)
        x[:, :k] = g
        x = x.view(-1, ng, Q4_GROUP)
        top = x.abs().amax(2)
        s = (top / 7).float()
        s = (s.view(torch.int32) & -65536).view(torch.float32)
        up = ((s.view(torch.int32) >> 16) + 1 << 16).view(torch.float32)
        s = torch.where(7 * s.double() < top, up, s)
        c = torch.where(s[..., None] > 0, torch.round(x / s.double().clamp_min(1e-300)[..., None]), 0.0)
        u = (c + 8).to(torch.uint8).view(-1, ng * Q4_GROUP)
        codes[r0:r0 + g.shape[0]] = u[:, 0::2] | (u[:, 1::2] << 4)
        scales[r0:r0 + g.shape[0]] = s
    return codes, scales, G[:, k].clone()


def prepare(case, seed):
    sizes = _sizes(case)
    state = dict(_inputs(case, seed), case=case, sizes=sizes, off=_offsets(sizes))
    if case["op"] in ("score", "q4"):
        other = _other_sizes(case, sizes)
        state.update(other=other, off2=_offsets(other))
    if not own:
        if case["op"] == "q4":
            state["codes"], state["scales"], state["q"] = _plain_q4(state.pop("G1"), case["k"])
        return state
    from hyperion_amd import engine

    if case["op"] == "affine":
        order = state["order"]
        state["groups"] = engine.RowGroups(sizes, order=order)
        state["bank"] = engine.AffineBank(state.pop("W"), state.pop("b"))
    elif case["op"] == "gram":
        state["groups"] = engine.RowGroups(sizes)
    elif case["op"] == "score":
        rows = engine.RowGroups(sizes)
        cols = engine.RowGroups(other) if case["cross"] else rows
        state["pairs"] = engine.GroupPairs(rows, cols)
    else:
        state["gallery"] = engine.q4_rows(state.pop("G1"), case["k"], engine.RowGroups(sizes))
        state["pairs"] = engine.GroupPairs(engine.RowGroups(other), state["gallery"].groups)
    return state


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        from hyperion_amd import engine

        if op == "affine":
            return engine.grouped_affine(state["x"], state["groups"], state["bank"], lnorm=state["case"]["lnorm"])
        if op == "gram":
            return engine.grouped_gram64(state["x"], state["groups"])
        if op == "score":
            return engine.grouped_score(state["G1"], state["G2"], state["pairs"])
        return engine.q4_score(state["gallery"], state["G2"], state["pairs"])
    return {"affine": _run_affine, "gram": _run_gram, "score": _run_score, "q4": _run_q4}[op](state)


def _run_affine(s):
    x, off, order, case = s["x"], s["off"], s["order"], s["case"]
    y = torch.empty(x.shape[0], case["d_out"], device=x.device)
    for e in range(len(off) - 1):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        rows = slice(a, b) if order is None else order[a:b]
        z = torch.mm(x[rows].float(), s["W"][e]) + s["b"][e]
        if case["lnorm"]:
            z = z * (math.sqrt(case["d_out"]) / (torch.sqrt((z * z).sum(1, keepdim=True)) + 1e-10))
        y[rows] = z
    return y


def _run_gram(s):
    x, off = s["x"], s["off"]
    E, d = len(off) - 1, x.shape[1]
    C = torch.zeros(E, d, d, dtype=torch.float64, device=x.device)
    F = torch.zeros(E, d, dtype=torch.float64, device=x.device)
    for e in range(E):
        if off[e] < off[e + 1]:
            xe = x[off[e]:off[e + 1]].double()
            torch.mm(xe.t(), xe, out=C[e])
            F[e] = xe.sum(0)
    return C, F


def _run_score(s):
    off, off2 = s["off"], s["off2"]
    out = torch.empty(_blocks(s["sizes"], s["other"]), device=s["G1"].device)
    at = 0
    for e, (n1, n2) in enumerate(zip(s["sizes"], s["other"])):
        if n1 * n2:
            torch.mm(s["G1"][off[e]:off[e + 1]], s["G2"][off2[e]:off2[e + 1]].t(),
                     out=out[at:at + n1 * n2].view(n1, n2))
            at += n1 * n2
    return out


def _run_q4(s):
    off, off2, k = s["off"], s["off2"], s["case"]["k"]
    out = torch.empty(_blocks(s["sizes"], s["other"]), device=s["G2"].device)
    at = 0
    for e, (n, m) in enumerate(zip(s["sizes"], s["other"])):
        if n * m == 0:
            continue
        a, b = off[e], off[e + 1]
        codes = s["codes"][a:b]
        w = torch.stack((codes & 15, codes >> 4), dim=2).view(n, -1, Q4_GROUP).float() - 8
        w = (w * s["scales"][a:b, :, None]).view(n, -1)[:, :k]
        t = s["G2"][off2[e]:off2[e + 1]]
        blk = out[at:at + m * n].view(m, n)
        torch.mm(t[:, :k], w.t(), out=blk)
        blk += s["q"][a:b]
        blk += t[:, k + 1:k + 2]
        at += m * n
    return out


# ---------------------------------------------------------------------------------------------- definition
def exact(case, seed):
    """The same outputs in float64, group by group."""
    inp = _inputs(case, seed)
    sizes = _sizes(case)
    if case["op"] == "affine":
        X = inp["x"].double()
        if inp["order"] is not None:
            X = X[inp["order"]]
        parts = []
        for e, xe in enumerate(torch.split(X, sizes)):
            z = xe @ inp["W"][e].double() + inp["b"][e].double()
            if case["lnorm"]:
                z = math.sqrt(z.shape[1]) * z / (z.norm(dim=1, keepdim=True) + 1e-10)
            parts.append(z)
        Y = torch.cat(parts)
        if inp["order"] is not None:
            back = torch.empty_like(Y)
            back[inp["order"]] = Y
            Y = back
        return Y
    if case["op"] == "gram":
        xs = torch.split(inp["x"].double(), sizes)
        return (torch.stack([xe.t().contiguous() @ xe for xe in xs]), torch.stack([xe.sum(0) for xe in xs]))
    other, k = _other_sizes(case, sizes), case["k"]
    G1, G2 = inp["G1"].double(), inp["G2"].double()
    rows, cols = torch.split(G1, sizes), torch.split(G2, other)
    if case["op"] == "score":
        return torch.cat([(a @ b.t().contiguous()).flatten() for a, b in zip(rows, cols)])
    parts = []
    for a, t in zip(rows, cols):
        if t.shape[0] == 0 or a.shape[0] == 0:
            continue
        acc = a[:, k][None, :] + t[:, k + 1][:, None]
        for c0 in range(0, k, Q4_GROUP):
            g = a[:, c0:min(k, c0 + Q4_GROUP)]
            top = g.abs().amax(1)
            # smallest number of eight significant bits with 7 s >= top: mantissa as an integer in 128..255
            exp = torch.floor(torch.log2(top.clamp_min(1e-300) / 7)) - 7
            step = torch.exp2(exp)
            step = torch.where(top / 7 < 128 * step, step / 2, torch.where(top / 7 >= 256 * step, step * 2, step))
            m = torch.floor(top / 7 / step)
            m = torch.where(7 * m * step < top, m + 1, m)
            s = torch.where(7 * (m - 1) * step >= top, m - 1, m) * step
            c = torch.where(top[:, None] > 0, torch.round(g / s[:, None]), 0.0)
            acc = acc + t[:, c0:c0 + g.shape[1]] @ (c * s[:, None]).t().contiguous()
        parts.append(acc.flatten())
    return torch.cat(parts) if parts else torch.empty(0, dtype=torch.float64, device="cuda")
