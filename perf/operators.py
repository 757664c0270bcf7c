"""Two operators of the logits path and the cases that stand for their use.

project  logits = x . W^T for weights held as 4-bit values with a scale (and,
         optionally, a minimum) per group of consecutive columns:
         w = s * (q - 8), or w = s * q + m with minimums.
draw     one token per row of logits from given uniforms: temperature, top-k,
         top-p and min-p over the descending order of the row (equal logits by
         ascending index), then the first token whose running mass reaches
         u times the kept mass; returns the token and its probability.

`run` computes them in plain torch, or, where `own` is true, through this
repository's engine. `exact` computes them in 64 bits.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the tiny configuration's output layer, one decode row: launch latency
        {"name": "project_tiny_1", "op": "project", "rows": 2000, "cols": 512, "group": 32, "mins": False,
         "nb": 1, "type": "f16", "scales": "f16", "out": "f32"},
        # one chat's decode step on the Llama-3 8B output layer
        {"name": "project_llama3_1", "op": "project", "rows": 128256, "cols": 4096, "group": 128, "mins": False,
         "nb": 1, "type": "bf16", "scales": "bf16", "out": "bf16"},
        # a few chats on a 2048-wide model; fp32 hidden states from a host-side
        # model, asymmetric groups of 64, fp32 logits for the sampler
        {"name": "project_2048_f32_4", "op": "project", "rows": 128256, "cols": 2048, "group": 64, "mins": True,
         "nb": 4, "type": "f32", "scales": "f16", "out": "f32"},
        # an odd vocabulary and width (the last group is short), seven chats
        {"name": "project_odd_7", "op": "project", "rows": 50257, "cols": 1696, "group": 128, "mins": True,
         "nb": 7, "type": "f16", "scales": "f16", "out": "f16"},
        # a serving batch on the Qwen2 vocabulary, groups of 32
        {"name": "project_qwen2_16", "op": "project", "rows": 151936, "cols": 4096, "group": 32, "mins": False,
         "nb": 16, "type": "bf16", "scales": "bf16", "out": "f32"},
        # the widest: 64 rows against an 8192-wide output layer
        {"name": "project_wide_64", "op": "project", "rows": 151936, "cols": 8192, "group": 128, "mins": True,
         "nb": 64, "type": "bf16", "scales": "f32", "out": "bf16"},
        # the tiny configuration: one row of 2000 logits, default chat settings
        {"name": "draw_tiny_1", "op": "draw", "rows": 1, "vocab": 2000, "type": "f32", "mode": "chat", "shape": "spread"},
        # one chat's decode step at the Llama-3 vocabulary
        {"name": "draw_llama3_1", "op": "draw", "rows": 1, "vocab": 128256, "type": "f32", "mode": "chat", "shape": "peaked"},
        # a batch of requests, each with settings of its own (some without top-k)
        {"name": "draw_mixed_256", "op": "draw", "rows": 256, "vocab": 128256, "type": "f32", "mode": "mixed", "shape": "spread"},
        # full-vocabulary nucleus at the Qwen2 vocabulary, logits of a bf16 projection
        {"name": "draw_nucleus_64", "op": "draw", "rows": 64, "vocab": 151936, "type": "bf16", "mode": "nucleus", "shape": "spread"},
        # grammar-constrained rows of an odd vocabulary: most logits are -inf
        {"name": "draw_masked_33", "op": "draw", "rows": 33, "vocab": 50257, "type": "f16", "mode": "minp", "shape": "masked"},
        # the largest: a shard of offline sampling, top-k 50
        {"name": "draw_offline_2048", "op": "draw", "rows": 2048, "vocab": 151936, "type": "bf16", "mode": "topk", "shape": "spread"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        rows = min(151936, _log_int(rng, 512, 152000))
        cols = 32 * _log_int(rng, 8, 192)
        return {"op": "project", "rows": rows, "cols": cols, "group": rng.choice([32, 64, 128, 256]),
                "mins": rng.random() < 0.5, "nb": _log_int(rng, 1, 64), "type": rng.choice(["f32", "f16", "bf16"]),
                "scales": rng.choice(["f32", "f16", "bf16"]), "out": rng.choice(["f32", "f16", "bf16"])}
    vocab = min(151936, _log_int(rng, 1000, 152000))
    kind = rng.choice(["f32", "f16", "bf16"])
    rows = _log_int(rng, 1, 4096 // SIZE[kind])
    return {"op": "draw", "rows": rows, "vocab": vocab, "type": kind,
            "mode": rng.choice(["chat", "mixed", "nucleus", "minp", "topk", "plain", "greedy"]),
            "shape": rng.choice(["spread", "peaked", "masked", "flat"])}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _prepare_project(case, g):
    rows, cols, group = case["rows"], case["cols"], case["group"]
    groups = -(-cols // group)
    lds = -(-rows // 8) * 8
    dev = "cuda"
    # quantised normal weights fill the 16 levels about evenly
    q = torch.randint(0, 256, (rows, cols // 2), generator=g, device=dev, dtype=torch.uint8)
    st = TYPES[case["scales"]]
    s = ((0.5 + torch.rand((groups, lds), generator=g, device=dev)) * (0.25 / math.sqrt(cols))).to(st)
    m = None
    if case["mins"]:
        m = (-s.float() * (8.0 + 2.0 * torch.rand((groups, lds), generator=g, device=dev) - 1.0)).to(st)[:, :rows]
    # RMS-normalised hidden states
    x = torch.randn((case["nb"], cols), generator=g, device=dev).to(TYPES[case["type"]])
    return {"case": case, "q": q, "s": s[:, :rows], "m": m, "x": x}


def _settings(case, g):
    """temperature, top-p, min-p and top-k of each row: three doubles and an int64."""
    n, mode, dev = case["rows"], case["mode"], "cuda"
    rec = torch.zeros((n, 4), dtype=torch.float64, device=dev)
    k = torch.zeros(n, dtype=torch.int64, device=dev)
    t, p, mp = 0.7, 1.0, 0.0
    if mode == "chat":
        p, mp, k = 0.95, 0.05, k + 40
    elif mode == "nucleus":
        t, p = 1.0, 0.99
    elif mode == "minp":
        t, mp = 1.0, 0.02
    elif mode == "topk":
        t, k = 1.0, k + 50
    elif mode == "plain":
        t = 1.0
    elif mode == "greedy":
        t = 0.0
    rec[:, 0], rec[:, 1], rec[:, 2] = t, p, mp
    if mode == "mixed":
        u = torch.rand((n, 4), generator=g, device=dev, dtype=torch.float64)
        rec[:, 0] = 0.5 + 0.7 * u[:, 0]
        rec[:, 1] = 0.8 + 0.2 * u[:, 1]
        rec[:, 2] = torch.where(u[:, 2] < 0.5, 0.0, 0.05)
        k = torch.tensor([0, 20, 50, 100], device=dev)[(4 * u[:, 3]).long()]
    rec.view(torch.int64)[:, 3] = k
    return rec


def _prepare_draw(case, g):
    n, V, dev = case["rows"], case["vocab"], "cuda"
    x = torch.randn((n, V), generator=g, device=dev)
    x *= 1.0 if case["shape"] == "flat" else 2.5
    if case["shape"] == "peaked":
        # a few tokens stand out, as in a trained model's rows
        at = torch.randint(0, V, (n, 24), generator=g, device=dev)
        x.scatter_add_(1, at, 6.0 + 6.0 * torch.rand((n, 24), generator=g, device=dev))
    elif case["shape"] == "masked":
        keep = torch.rand((n, V), generator=g, device=dev) < 0.02
        keep[:, 7] = True
        x = torch.where(keep, x, -math.inf)
    return {"case": case, "x": x.to(TYPES[case["type"]]), "settings": _settings(case, g),
            "u": torch.rand(n, generator=g, device=dev, dtype=torch.float64)}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_project(case, g) if case["op"] == "project" else _prepare_draw(case, g)


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------
def _weights(state, dtype):
    """The weight matrix [rows, cols] that the 4-bit values stand for."""
    c = state["case"]
    q = torch.stack((state["q"] & 15, state["q"] >> 4), 2).reshape(c["rows"], c["cols"]).to(dtype)
    s = state["s"].t().to(dtype).repeat_interleave(c["group"], 1)[:, :c["cols"]]
    if state["m"] is None:
        return (q - 8.0) * s
    return q * s + state["m"].t().to(dtype).repeat_interleave(c["group"], 1)[:, :c["cols"]]


def _plain_project(state):
    y = state["x"].float() @ _weights(state, torch.float32).t()
    return y.to(TYPES[state["case"]["out"]])


def _plain_draw(state):
    # 64 bits: the running masses are compared with borders
    V = state["x"].shape[1]
    rec = state["settings"]
    t, p, mp = rec[:, 0:1], rec[:, 1:2], rec[:, 2:3]
    k = rec.view(torch.int64)[:, 3:4]
    v, order = torch.sort(state["x"].float(), dim=1, descending=True, stable=True)
    v = v.double()
    rank = torch.arange(V, device=v.device)[None, :]
    e = torch.exp((v - v[:, :1]) / torch.where(t > 0, t, 1.0))
    e = torch.where((k <= 0) | (rank < k), e, 0.0)
    c = torch.cumsum(e, 1)
    keep = (p <= 0) | (p >= 1) | (c - e < p * c[:, -1:])
    keep &= (mp <= 0) | (e >= mp)
    keep[:, 0] = True
    e = torch.where(keep, e, 0.0)
    c = torch.cumsum(e, 1)
    total = c[:, -1:]
    at = (c < state["u"][:, None] * total).sum(1, keepdim=True)
    at = torch.minimum(at, (e > 0).sum(1, keepdim=True) - 1)
    at = torch.where(t > 0, at, 0)
    prob = torch.where(t > 0, e.gather(1, at) / total, 1.0)
    return order.gather(1, at)[:, 0], prob[:, 0].float()


_ENGINE = []


def _engine():
    """This repository's package and one engine, as a serving process keeps them."""
    if not _ENGINE:
        import __graft_entry__ as graft
        pkg = graft.load_package()
        _ENGINE.extend([pkg, pkg.Engine(0, max_rows=2048, max_vocab=1 << 18)])
    return _ENGINE


def run(state):
    project = state["case"]["op"] == "project"
    if own:
        pkg, eng = _engine()
        if project:
            w = pkg.G4Weights(state["q"], state["s"], state["m"], group=state["case"]["group"])
            return eng.g4_matmul(w, state["x"], out_dtype=TYPES[state["case"]["out"]], check=False)
        ids, probs, _ = eng.draw_batch(state["x"], state["settings"], state["u"], check=False)
        return ids, probs
    return _plain_project(state) if project else _plain_draw(state)


def work(case):
    if case["op"] == "project":
        rows, cols, nb = case["rows"], case["cols"], case["nb"]
        groups = -(-cols // case["group"])
        per = groups * SIZE[case["scales"]] * (2 if case["mins"] else 1)
        return {"bytes": rows * (cols // 2 + per) + nb * cols * SIZE[case["type"]] + nb * rows * SIZE[case["out"]],
                "flops": 2 * rows * cols * nb}
    # a logit is read once and compared or exponentiated once; the settings,
    # the uniform, the token and its probability are 52 bytes a row
    return {"bytes": case["rows"] * (case["vocab"] * SIZE[case["type"]] + 52), "flops": 2 * case["rows"] * case["vocab"]}


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------
def _exact_project(state):
    # group by group: s * sum (q - 8) x, or s * sum q x + m * sum x
    c = state["case"]
    x = state["x"].double()
    y = torch.zeros((c["nb"], c["rows"]), dtype=torch.float64, device=x.device)
    for g, lo in enumerate(range(0, c["cols"], c["group"])):
        xg = x[:, lo:lo + c["group"]]
        b = state["q"][:, lo // 2:(lo + xg.shape[1]) // 2]
        dot = xg[:, 0::2] @ (b % 16).double().t() + xg[:, 1::2] @ (b // 16).double().t()
        sg = state["s"][g].double()[None, :]
        total = xg.sum(1, keepdim=True)
        y += sg * (dot - 8.0 * total) if state["m"] is None else sg * dot + state["m"][g].double()[None, :] * total
    return y


def _exact_row(x, t, p, mp, k, u):
    """One row: (token, probability), by logarithms of the probabilities."""
    if t <= 0:
        return int((x == x.max()).nonzero()[0]), 1.0
    logp = torch.log_softmax(x / t, 0)
    value, index = torch.sort(-logp, stable=True)
    value = -value
    if 0 < k < value.numel():
        value, index = value[:k], index[:k]
    value = value - torch.logsumexp(value, 0)
    mass = torch.exp(value)
    n = mass.numel()
    if 0 < p < 1:
        n = min(n, int((torch.cumsum(mass, 0) < p).sum()) + 1)
    if mp > 0:
        n = min(n, max(1, int((value - value[0] >= math.log(mp)).sum())))
    run = torch.cumsum(mass[:n], 0)
    at = min(int((run < u * run[-1]).sum()), n - 1)
    return int(index[at]), float(mass[at] / run[-1])


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "project":
        return _exact_project(state)
    rec = state["settings"].tolist()
    ks = state["settings"].view(torch.int64)[:, 3].tolist()
    us = state["u"].tolist()
    got = [_exact_row(state["x"][r].double(), *rec[r][:3], ks[r], us[r]) for r in range(case["rows"])]
    dev = state["x"].device
    return (torch.tensor([a for a, _ in got], device=dev),
            torch.tensor([b for _, b in got], dtype=torch.float64, device=dev))
