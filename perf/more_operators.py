"""The dense end of a decode step around the quantized expert path, as a serving program calls it,
with the plain forms in elementary torch operations.

  kind "w4"      rows times a weight of 4-bit codes with a bf16 scale (and, where the checkpoint has
                 them, a zero point) per group of 32, 64 or 128 columns: y = x ((q - z) s)^T.
  kind "between" what stands between two blocks that are normed on both sides: the block's output is
                 normed, gated and added to the scaled residual, and the sum is normed for the next
                 block, into bf16 and / or MXFP8 rows.
  kind "sample"  next tokens from logits: temperature, min-p, top-k and top-p (in this order), drawn
                 with given uniform numbers; the tokens and their log probabilities.

`own` says whether run() calls this library's operators or computes the plain forms.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
BLOCK = 32         # columns that share a scale of MXFP8 rows
RANGE = 28.0       # tokens with less than e^-28 of the largest weight are not drawn
HIDDEN, SMALL_HIDDEN, VOCAB = 7168, 2048, 163840


def listed():
    return [
        # one token's gate and up projection, the finest groups: a matrix-vector product
        {"name": "w4_r1", "kind": "w4", "rows": 1, "n": 4096, "k": HIDDEN, "group": 32, "zeros": False,
         "f32": False},
        # a small model's projection of an odd width for a few sequences: latency counts
        {"name": "w4_r7_odd", "kind": "w4", "rows": 7, "n": 2051, "k": 1408, "group": 64, "zeros": True,
         "f32": False},
        # one token through the head, logits for the draw in fp32: the longest stream of weights
        {"name": "w4_head_r1", "kind": "w4", "rows": 1, "n": VOCAB, "k": HIDDEN, "group": 128,
         "zeros": False, "f32": True},
        # a decode batch through a small model's head
        {"name": "w4_head_r48", "kind": "w4", "rows": 48, "n": VOCAB, "k": SMALL_HIDDEN, "group": 128,
         "zeros": True, "f32": True},
        # a short ragged prompt through an MLP projection
        {"name": "w4_r333", "kind": "w4", "rows": 333, "n": 9728, "k": 2560, "group": 64, "zeros": False,
         "f32": False},
        # a full prefill chunk: the largest product
        {"name": "w4_r4096", "kind": "w4", "rows": 4096, "n": 4096, "k": HIDDEN, "group": 128,
         "zeros": True, "f32": False},
        # one token between two blocks of a decode step: latency alone
        {"name": "between_r1", "kind": "between", "rows": 1, "cols": HIDDEN, "x32": False, "post": True,
         "gate": "col", "scale": 1.0, "offset": False, "normed": True, "quant": False},
        # a small model's ragged chunk, a routed sum in fp32 with a gate per token and a scaled residual
        {"name": "between_r333_f32", "kind": "between", "rows": 333, "cols": SMALL_HIDDEN, "x32": True,
         "post": True, "gate": "row", "scale": 0.5, "offset": True, "normed": True, "quant": False},
        # a full prefill chunk with a gate per element, rows for bf16 and for MXFP8 products
        {"name": "between_r4096", "kind": "between", "rows": 4096, "cols": HIDDEN, "x32": False,
         "post": True, "gate": "full", "scale": 1.0, "offset": False, "normed": True, "quant": True},
        # one sequence's next token, all filters on: latency
        {"name": "sample_r1", "kind": "sample", "rows": 1, "vocab": VOCAB, "bf16": False, "top_k": True,
         "top_p": True, "min_p": False, "greedy": 0.0, "masked": 0.0},
        # a batch of a small odd vocabulary, bf16 logits (with their many ties), part of it masked
        {"name": "sample_r40_bf16", "kind": "sample", "rows": 40, "vocab": 32003, "bf16": True,
         "top_k": False, "top_p": True, "min_p": True, "greedy": 0.1, "masked": 0.3},
        # a full server's batch with every kind of request in it
        {"name": "sample_r256", "kind": "sample", "rows": 256, "vocab": VOCAB, "bf16": False,
         "top_k": True, "top_p": True, "min_p": True, "greedy": 0.1, "masked": 0.0},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["w4", "w4", "w4", "between", "between", "sample", "sample"])
    if kind == "w4":
        group = rng.choice([32, 64, 128])
        k = group * _log_int(rng, max(1, 256 // group), 8192 // group)
        n = _log_int(rng, 64, min(VOCAB, VOCAB * HIDDEN // k))
        n = n if rng.random() < 0.4 else 16 * ((n + 15) // 16)
        rows = _log_int(rng, 1, max(1, min(4096, 4096 * 4096 * HIDDEN // (n * k))))
        return {"kind": kind, "rows": rows, "n": n, "k": k, "group": group, "zeros": rng.random() < 0.5,
                "f32": rng.random() < 0.3}
    if kind == "between":
        cols = 32 * _log_int(rng, 4, 256)
        rows = _log_int(rng, 1, min(16384, 4096 * HIDDEN // cols))
        form = rng.choice(["both", "normed", "normed", "quant"])
        return {"kind": kind, "rows": rows, "cols": cols, "x32": rng.random() < 0.4,
                "post": rng.random() < 0.8, "gate": rng.choice(["none", "col", "row", "full"]),
                "scale": rng.choice([1.0, 1.0, 0.5, 0.83]), "offset": rng.random() < 0.4,
                "normed": form != "quant", "quant": form != "normed"}
    vocab = _log_int(rng, 500, VOCAB)
    return {"kind": kind, "rows": _log_int(rng, 1, 256), "vocab": vocab, "bf16": rng.random() < 0.4,
            "top_k": rng.random() < 0.6, "top_p": rng.random() < 0.6, "min_p": rng.random() < 0.4,
            "greedy": rng.choice([0.0, 0.2]), "masked": rng.choice([0.0, 0.0, 0.5])}


# ------------------------------------------------------------------ inputs, from the seed alone
def _gen(seed, stream):
    return torch.Generator(device="cuda").manual_seed(seed * 1013 + stream)


def _rows(g, rows, cols, std=1.0):
    """Hidden rows as a transformer has them: normal, with a few columns an order louder."""
    v = torch.randn(rows, cols, device="cuda", generator=g) * std
    loud = torch.rand(cols, device="cuda", generator=g) < 0.004
    return v * torch.where(loud, 12.0, 1.0)


def _logits(g, case):
    """A spread of all tokens, a handful that stand out, some masked."""
    rows, vocab = case["rows"], case["vocab"]
    v = torch.randn(rows, vocab, device="cuda", generator=g) * 2.2
    at = torch.randint(0, vocab, (rows, 12), device="cuda", generator=g)
    v.scatter_(1, at, 7 + 2 * torch.randn(rows, 12, device="cuda", generator=g))
    if case["masked"]:
        gone = torch.rand(rows, vocab, device="cuda", generator=g) < case["masked"]
        v.masked_fill_(gone, -math.inf)
    return v.to(torch.bfloat16) if case["bf16"] else v


def prepare(case, seed):
    s, kind, g = dict(case), case["kind"], _gen(seed, 1)
    if kind == "w4":
        n, k, groups = case["n"], case["k"], case["k"] // case["group"]
        s["x"] = _rows(g, case["rows"], k).to(torch.bfloat16)
        s["packed"] = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
        scales = torch.randn(n, groups, device="cuda", generator=g)
        s["scales"] = (scales.abs_() * (0.02 / 7)).to(torch.bfloat16)
        s["zero"] = (torch.randint(4, 12, (n, groups), dtype=torch.uint8, device="cuda", generator=g)
                     if case["zeros"] else None)
    elif kind == "between":
        rows, cols = case["rows"], case["cols"]
        x = _rows(g, rows, cols, 0.5)
        s["x"] = x if case["x32"] else x.to(torch.bfloat16)
        s["res"] = _rows(g, rows, cols, 2.0).to(torch.bfloat16)
        mean = 0.0 if case["offset"] else 1.0
        weight = lambda: (mean + 0.1 * torch.randn(cols, device="cuda", generator=g)).to(torch.bfloat16)  # noqa: E731
        s["pre_w"], s["post_w"] = weight(), weight() if case["post"] else None
        shape = {"none": None, "col": (cols,), "row": (rows, 1), "full": (rows, cols)}[case["gate"]]
        s["gate_v"] = (None if shape is None else
                       (0.5 + 0.3 * torch.randn(*shape, device="cuda", generator=g)).to(torch.bfloat16))
    else:
        rows = case["rows"]
        rand = lambda: torch.rand(rows, device="cuda", generator=g)  # noqa: E731
        s["logits"], s["u"] = _logits(g, case), rand()
        t = 0.5 + rand()
        s["temperature"] = torch.where(rand() < case["greedy"], 0.0, t)
        # a request without a filter has the value that leaves it out
        off = rand()
        k = torch.exp(rand() * math.log(400)).int()
        s["k_row"] = torch.where(off < 0.25, 0, k).int() if case["top_k"] else None
        s["p_row"] = torch.where(rand() < 0.25, 1.0, 0.6 + 0.39 * rand()) if case["top_p"] else None
        s["m_row"] = torch.where(rand() < 0.25, 0.0, 0.2 * rand()) if case["min_p"] else None
    if own:
        _prepare_own(s)
    return s


def _prepare_own(s):
    """What a program of this library keeps besides its inputs: packaged weights, output buffers,
    workspaces."""
    from pegainfer_amd import ops
    bf = dict(dtype=torch.bfloat16, device="cuda")
    if s["kind"] == "w4":
        s["w"] = ops.w4_pack(s.pop("packed"), s.pop("scales"), s.pop("zero"), group=s["group"])
        s["y"] = torch.empty(s["rows"], s["n"], device="cuda",
                             dtype=torch.float32 if s["f32"] else torch.bfloat16)
    elif s["kind"] == "between":
        rows, cols = s["rows"], s["cols"]
        s["sum"] = torch.empty(rows, cols, **bf)
        s["y"] = torch.empty(rows, cols, **bf) if s["normed"] else None
        s["q"] = ops.MxTensor.empty(rows, cols, ops.MxFormat.Fp8E4M3) if s["quant"] else None
    else:
        s["ws"] = ops.SampleWorkspace(s["rows"], s["vocab"])
        s["tokens"] = torch.empty(s["rows"], dtype=torch.int32, device="cuda")
        s["logprobs"] = torch.empty(s["rows"], device="cuda")


# ------------------------------------------------------------------ a pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from pegainfer_amd import ops
    if s["kind"] == "w4":
        ops.w4_gemm(s["w"], s["x"], s["y"])
        return s["y"]
    if s["kind"] == "between":
        ops.sandwich_rmsnorm(s["x"], s["res"], s["pre_w"], EPS, post_weight=s["post_w"], gate=s["gate_v"],
                             residual_scale=s["scale"], unit_offset=s["offset"], residual_out=s["sum"],
                             normed=s["y"], quantized=s["q"])
        q = s["q"]
        return [s["sum"], s["y"],
                (q.codes.view(torch.float8_e4m3fn), q.scales.view(torch.float8_e8m0fnu)) if q else None]
    ops.sample_tokens(s["ws"], s["logits"], s["u"], s["tokens"], temperature=s["temperature"],
                      top_k=s["k_row"], top_p=s["p_row"], min_p=s["m_row"], logprobs=s["logprobs"])
    return {"tokens": s["tokens"], "logprobs": s["logprobs"]}


# ------------------------------------------------------------------ the plain forms
def _weight(s):
    """(q - z) s in fp32, which holds it exactly."""
    n, half = s["packed"].shape
    q = torch.stack((s["packed"] & 15, s["packed"] >> 4), -1).reshape(n, 2 * half // s["group"], s["group"])
    z = 8.0 if s["zero"] is None else s["zero"].float().unsqueeze(-1)
    return ((q.float() - z) * s["scales"].float().unsqueeze(-1)).reshape(n, 2 * half)


def _scaled(v, e):
    """v * 2^e, exact."""
    return v * torch.exp2(e.double())


def _mxfp8(v):
    """Rows of 64 bits as E4M3 values and power-of-two scales: per block the smallest s >= -127 for
    which the largest magnitude over 2^s is at most 464, codes to nearest, ties to even."""
    rows, cols = v.shape
    b = v.reshape(rows, cols // BLOCK, BLOCK)
    amax = b.abs().amax(-1)
    m, e = torch.frexp(amax)
    s = e - 9 + (m > 464 / 512).to(e.dtype)
    s = torch.where(amax > 0, s, -127).clamp(min=-127)
    u = _scaled(b, -s.unsqueeze(-1)).reshape(rows, cols)
    step = torch.frexp(u).exponent.clamp(min=-5) - 4
    u = _scaled(torch.round(_scaled(u, -step)), step)
    return u.to(torch.float8_e4m3fn), (s + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _draw_plain(s):
    lg = s["logits"].float()
    rows, vocab = lg.shape
    lg = torch.where(torch.isnan(lg), -math.inf, lg)
    t = s["temperature"].double().unsqueeze(1)
    greedy = t <= 0
    t = torch.where(greedy, 1.0, t)
    # weights in 64 bits: the sums' borders decide tokens
    d = lg.double() - lg.amax(1, keepdim=True)
    least = -RANGE * t
    if s["m_row"] is not None:
        least = torch.maximum(least, t * torch.log(s["m_row"].double().unsqueeze(1)))
    w = torch.where(d >= least, torch.exp(d / t), 0.0)
    del d
    order = torch.sort(lg, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    k = torch.full_like(greedy, vocab, dtype=torch.int64)
    if s["k_row"] is not None:
        k = torch.where(s["k_row"].unsqueeze(1) > 0, s["k_row"].unsqueeze(1).long(), k)
    k = torch.where(greedy, 1, k)
    if s["k_row"] is not None or bool((s["greedy"] > 0)):
        ws = ws * (torch.arange(vocab, device=lg.device) < k)
    if s["p_row"] is not None:
        # of the mass that min-p and top-k left
        p = s["p_row"].double().unsqueeze(1)
        before = torch.cumsum(ws, 1) - ws
        ws = ws * ((before < p * ws.sum(1, keepdim=True)) | (p >= 1))
    w = torch.zeros_like(w).scatter_(1, order, ws)
    del order, ws
    cum = torch.cumsum(w, 1)
    total = cum[:, -1:]
    token = (cum <= s["u"].double().unsqueeze(1) * total).sum(1, keepdim=True).clamp(max=vocab - 1)
    logprob = torch.log(w.gather(1, token) / total)
    return {"tokens": token.squeeze(1).to(torch.int32), "logprobs": logprob.squeeze(1).float()}


def _run_plain(s):
    if s["kind"] == "w4":
        y = s["x"].float() @ _weight(s).T
        return y if s["f32"] else y.to(torch.bfloat16)
    if s["kind"] == "sample":
        return _draw_plain(s)
    # quantized values next to a rounding border decide in 64 bits
    up = torch.float64 if s["quant"] else torch.float32
    one = 1.0 if s["offset"] else 0.0
    y = s["x"].to(up)
    if s["post"]:
        y = y * torch.rsqrt((y * y).mean(1, keepdim=True) + EPS) * (one + s["post_w"].to(up))
    if s["gate_v"] is not None:
        y = y * s["gate_v"].to(up)
    v = s["scale"] * s["res"].to(up) + y
    z = v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * (one + s["pre_w"].to(up))
    return [v.to(torch.bfloat16), z.to(torch.bfloat16) if s["normed"] else None,
            _mxfp8(z) if s["quant"] else None]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "w4":
        r, n, k = case["rows"], case["n"], case["k"]
        per = 0.5 + (3 if case["zeros"] else 2) / case["group"]
        return {"bytes": n * k * per + 2.0 * r * k + (4.0 if case["f32"] else 2.0) * r * n,
                "flops": 2.0 * r * n * k}
    if case["kind"] == "between":
        rows, cols = case["rows"], case["cols"]
        n = float(rows) * cols
        per = (4 if case["x32"] else 2) + 4 + (2 if case["normed"] else 0) \
            + (1 + 1 / BLOCK if case["quant"] else 0)
        gate = {"none": 0, "col": 2 * cols, "row": 2 * rows, "full": 2 * n}[case["gate"]]
        return {"bytes": n * per + gate + (4 if case["post"] else 2) * cols, "flops": 11 * n}
    rows, vocab = case["rows"], case["vocab"]
    rows_of = 4 + 4 * (1 + case["top_k"] + case["top_p"] + case["min_p"]) + 8
    return {"bytes": float(rows) * (vocab * (2 if case["bf16"] else 4) + rows_of), "flops": 4.0 * rows * vocab}


# ------------------------------------------------------------------ the same in 64 bits
def _w4_exact(s):
    x, y = s["x"].double(), torch.empty(s["rows"], s["n"], dtype=torch.float64, device="cuda")
    step = max(1, (1 << 27) // s["k"])  # features at a time
    for at in range(0, s["n"], step):
        code = s["packed"][at:at + step]
        q = torch.empty(code.shape[0], s["k"], dtype=torch.float64, device="cuda")
        q[:, 0::2], q[:, 1::2] = (code % 16).double(), (code // 16).double()
        q -= 8.0 if s["zero"] is None else s["zero"][at:at + step].double().repeat_interleave(s["group"], 1)
        q *= s["scales"][at:at + step].double().repeat_interleave(s["group"], 1)
        y[:, at:at + step] = x @ q.T
    return y


def _mx_nearest(v):
    """The nearest E4M3 values, by search, and the scales, in 64 bits."""
    pos = [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)]
    grid = torch.tensor(pos[:-1], dtype=torch.float64, device=v.device)
    b = v.reshape(v.shape[0], -1, BLOCK)
    amax = b.abs().amax(-1)
    s = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -200) / 464)).clamp(min=-127)
    s = torch.where(amax <= 464 * torch.exp2(s), s, s + 1)  # where log2 rounded across a power of two
    s = torch.where((amax <= 464 * torch.exp2(s - 1)) & (s > -127), s - 1, s)
    a = (b.abs() / torch.exp2(s).unsqueeze(-1)).contiguous()
    hi = torch.searchsorted(grid, a).clamp(max=grid.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - grid[lo], grid[hi] - a
    pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return torch.copysign(grid[pick], b).reshape(v.shape), torch.exp2(s)


def _between_exact(s):
    x, res = s["x"].double(), s["res"].double()
    one, cols = float(s["offset"]), s["cols"]
    y = x if not s["post"] else x / (x.square().sum(1, keepdim=True) / cols + EPS).sqrt() * (s["post_w"].double() + one)
    v = res * s["scale"] + (y if s["gate_v"] is None else y * s["gate_v"].double())
    z = v / (v.square().sum(1, keepdim=True) / cols + EPS).sqrt() * (s["pre_w"].double() + one)
    return [v, z if s["normed"] else None, _mx_nearest(z) if s["quant"] else None]


def _sample_exact(s):
    """Row by row on the host, over the tokens that can be drawn alone."""
    tokens, logprobs = [], []
    every = s["logits"].float().cpu().numpy().astype(np.float64)
    host = {n: None if s[n] is None else s[n].cpu().numpy().astype(np.float64)
            for n in ("u", "temperature", "k_row", "p_row", "m_row")}
    for r, lg in enumerate(every):
        t = host["temperature"][r]
        d = lg - lg.max()
        ids = np.flatnonzero(d >= -RANGE * (t if t > 0 else 1.0))
        ids = ids[np.argsort(-d[ids], kind="stable")]
        if t <= 0:
            ids, t = ids[:1], 1.0
        if host["k_row"] is not None and host["k_row"][r] > 0:
            ids = ids[:int(host["k_row"][r])]
        w = np.exp(d[ids] / t)
        if host["m_row"] is not None:
            w = w[w >= host["m_row"][r]]
        if host["p_row"] is not None and host["p_row"][r] < 1:
            sums = np.concatenate(([0.0], np.cumsum(w)))
            w = w[:int(np.searchsorted(sums[:-1], host["p_row"][r] * sums[-1], side="left"))]
        ids = ids[:len(w)]
        back = np.argsort(ids)
        sums = np.cumsum(w[back])
        at = min(int(np.searchsorted(sums, host["u"][r] * sums[-1], side="right")), len(ids) - 1)
        tokens.append(int(ids[back][at]))
        logprobs.append(float(np.log(w[back][at] / sums[-1])))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32, device="cuda"),
            "logprobs": torch.tensor(logprobs, dtype=torch.float64, device="cuda")}


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"w4": _w4_exact, "between": _between_exact, "sample": _sample_exact}[case["kind"]](s)
