"""Workloads of the transformer-step operators: what is timed and what its outputs are compared with.

Three families, all fp32 unless a case says otherwise:

  scores   attention scores -> probabilities (scale, tanh cap, distance bias, causal / prefix /
           document / length masks), and the gradient of that step
  norm     the norms around a residual block: y = x + scale * gate * N_post(f), h = N_pre(y),
           and all of its gradients
  clip     the norm of all gradients of a model, and their scaling down to a given norm

``run`` computes a case with elementary torch operations, or, where ``own`` is set, with the calls a
user makes of ctensor_b200.
"""
import math
import random

import torch

own = False


# ---- the cases ------------------------------------------------------------------------------------------
def listed():
    return [
        # One decoded token for eight requests of different lengths: latency counts.
        {"name": "scores-token", "op": "scores", "dir": "fwd", "batch": 8, "heads": 12, "queries": 1, "keys": 4097,
         "causal": True, "cap": 30.0, "slopes": False, "prefix": False, "docs": 0, "lengths": True},
        # One attention layer of a training step at the size of the framework's causal softmax workload:
        # several documents packed into a row, scores capped.
        {"name": "scores-packed-1024", "op": "scores", "dir": "fwd", "batch": 8, "heads": 12, "queries": 1024,
         "keys": 1024, "causal": True, "cap": 50.0, "slopes": False, "prefix": False, "docs": 5, "lengths": False},
        # The gradient of a longer layer: distance bias with learned slopes, a prompt that sees itself whole.
        {"name": "scores-prefix-grad-2048", "op": "scores", "dir": "bwd", "batch": 4, "heads": 16, "queries": 2048,
         "keys": 2048, "causal": True, "cap": 0.0, "slopes": True, "prefix": True, "docs": 0, "lengths": False},
        # A padded batch of odd sizes, both directions of attention, capped: the gradient.
        {"name": "scores-padded-grad-odd", "op": "scores", "dir": "bwd", "batch": 3, "heads": 5, "queries": 777,
         "keys": 1001, "causal": False, "cap": 30.0, "slopes": False, "prefix": False, "docs": 0, "lengths": True},
        # Eight tokens between two blocks while serving.
        {"name": "norm-token", "op": "norm", "dir": "fwd", "batch": 8, "rows": 1, "cols": 768, "post": "none",
         "pre": "layer", "gate": "none", "scale": 1.0},
        # Between two blocks of a training step, [8, 1024, 768], with a learned gate for each channel.
        {"name": "norm-layer-768", "op": "norm", "dir": "fwd", "batch": 8, "rows": 1024, "cols": 768, "post": "none",
         "pre": "layer", "gate": "channel", "scale": 1.0},
        # Norms on both sides of a wide block, the gate computed from each sequence's conditioning.
        {"name": "norm-sandwich-8192", "op": "norm", "dir": "fwd", "batch": 8, "rows": 1024, "cols": 8192,
         "post": "rms", "pre": "rms", "gate": "batch", "scale": 0.5},
        # The gradients of the second.
        {"name": "norm-layer-grad-768", "op": "norm", "dir": "bwd", "batch": 8, "rows": 1024, "cols": 768,
         "post": "none", "pre": "layer", "gate": "channel", "scale": 1.0},
        # The gradients of norms on both sides, with a gate for every token and channel; odd row count.
        {"name": "norm-sandwich-grad-5120", "op": "norm", "dir": "bwd", "batch": 3, "rows": 1367, "cols": 5120,
         "post": "rms", "pre": "rms", "gate": "full", "scale": 0.5},
        # The four tensors of a two-layer classifier in double precision: launch latency.
        {"name": "clip-mlp-double", "op": "clip", "model": "mlp", "width": 1024, "layers": 2, "vocab": 16,
         "double": True, "p": 2.0, "clipped": True},
        # 193 tensors, 202 million gradients, norm below the limit: nothing has to be scaled.
        {"name": "clip-below-202m", "op": "clip", "model": "transformer", "width": 1024, "layers": 12, "vocab": 50257,
         "double": False, "p": 2.0, "clipped": False},
        # 193 tensors, 1.07 billion gradients, scaled into the buffers that the optimizer reads.
        {"name": "clip-1b", "op": "clip", "model": "transformer", "width": 2560, "layers": 12, "vocab": 50257,
         "double": False, "p": 2.0, "clipped": True},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, evenly spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["scores", "norm", "clip"])
    if op == "scores":
        case = {"op": op, "dir": rng.choice(["fwd", "bwd"]), "batch": rng.randint(1, 9), "heads": rng.randint(1, 16)}
        most = 200_000_000 // (case["batch"] * case["heads"])
        case["queries"] = rng.choice([1, rng.randint(2, 9), _spread(rng, 10, 2048), _spread(rng, 10, 2048)])
        case["keys"] = _spread(rng, max(1, case["queries"] // 3), max(2, min(131072, most // case["queries"])))
        case["causal"] = rng.random() < 0.6
        case["cap"] = rng.choice([0.0, 30.0, 50.0])
        case["slopes"] = rng.random() < 0.3
        case["prefix"] = rng.random() < 0.3
        case["docs"] = rng.choice([0, 0, rng.randint(2, 9)])
        case["lengths"] = rng.random() < 0.4
        return case
    if op == "norm":
        case = {"op": op, "dir": rng.choice(["fwd", "bwd"]), "cols": _spread(rng, 32, 16384)}
        if rng.random() < 0.7:
            case["cols"] = -(-case["cols"] // 64) * 64
        tokens = _spread(rng, 1, 48_000_000 // case["cols"])
        case["batch"] = rng.randint(1, min(16, tokens))
        case["rows"] = max(1, tokens // case["batch"])
        case["post"] = rng.choice(["none", "layer", "rms"])
        case["pre"] = rng.choice(["layer", "rms"])
        case["gate"] = rng.choice(["none", "channel", "batch", "full", "token"])
        case["scale"] = rng.choice([1.0, 0.5, 0.22])
        return case
    case = {"op": op, "model": rng.choice(["ragged", "transformer"]), "double": rng.random() < 0.2,
            "p": rng.choice([2.0, 2.0, 1.0, math.inf]), "clipped": rng.random() < 0.7}
    if case["model"] == "ragged":
        case.update(width=_spread(rng, 1, 400_000), layers=rng.randint(1, 400), vocab=rng.randint(0, 10 ** 6))
    else:
        case.update(width=rng.randint(17, 1400), layers=rng.randint(1, 12), vocab=_spread(rng, 100, 60000))
    return case


# ---- inputs ---------------------------------------------------------------------------------------------
def _shapes(case):
    """The shapes of a model's parameters."""
    w, n, v = case["width"], case["layers"], case["vocab"]
    if case["model"] == "mlp":
        return [(w, w), (w,)] * (n - 1) + [(v, w), (v,)]
    if case["model"] == "ragged":      # n tensors of about w values each; v chooses the sizes
        r = random.Random(v)
        return [(r.choice([1, _spread(r, 1, 4 * w), _spread(r, 1, 4 * w)]),) for _ in range(n)]
    layer = [(w, w), (w,)] * 4 + [(4 * w, w), (4 * w,), (w, 4 * w), (w,)] + [(w,)] * 4
    return [(v, w)] + layer * n


def _key_lengths(case):
    """Valid keys of each sequence: from all of them down to about a third; a case decides them, not a seed."""
    B, K = case["batch"], case["keys"]
    return [max(1, K - (2 * K * b) // (3 * B)) for b in range(B)]


def _query_starts(case):
    """The queries of a sequence are its last positions."""
    n = _key_lengths(case) if case["lengths"] else [case["keys"]] * case["batch"]
    return [k - case["queries"] for k in n]


def _prefixes(case):
    return [(case["keys"] * (b + 1)) // (4 * case["batch"]) for b in range(case["batch"])]


def _documents(case):
    """Document numbers [B, K]: a few documents of unequal lengths one behind the other in every sequence."""
    K, n = case["keys"], case["docs"]
    j = torch.arange(K, dtype=torch.float64)
    rows = [torch.floor(n * ((j + 0.5) / K) ** (0.6 + 0.1 * (b % 8))).to(torch.int32) for b in range(case["batch"])]
    return torch.stack(rows)


def _admitted(case, device="cpu"):
    """Which keys a query may look at: bool [B, 1, Q, K]."""
    B, Q, K = case["batch"], case["queries"], case["keys"]
    j = torch.arange(K, device=device)[None, None, :]
    start = torch.tensor(_query_starts(case), device=device)[:, None, None]
    pos = start + torch.arange(Q, device=device)[None, :, None]
    ok = torch.ones(B, Q, K, dtype=torch.bool, device=device)
    if case["causal"]:
        see = j <= pos
        if case["prefix"]:
            see = see | (j < torch.tensor(_prefixes(case), device=device)[:, None, None])
        ok &= see
    if case["lengths"]:
        ok &= j < torch.tensor(_key_lengths(case), device=device)[:, None, None]
    if case["docs"]:
        docs = _documents(case).to(device)
        ok &= _query_docs(case, docs)[:, :, None] == docs[:, None, :]
    return ok[:, None]


def _query_docs(case, docs):
    start = torch.tensor(_query_starts(case), device=docs.device)[:, None]
    at = start + torch.arange(case["queries"], device=docs.device)[None, :]
    return torch.gather(docs, 1, at.clamp(0, case["keys"] - 1)).contiguous()


def _scores_state(case, g):
    B, H, Q, K = case["batch"], case["heads"], case["queries"], case["keys"]
    dev = "cuda"
    s = {"scores": torch.randn(B, H, Q, K, device=dev, generator=g) * 12.0,
         "start": torch.tensor(_query_starts(case), dtype=torch.int32, device=dev), "scale": 0.125}
    if case["lengths"]:
        s["lengths"] = torch.tensor(_key_lengths(case), dtype=torch.int32, device=dev)
    if case["prefix"]:
        s["prefix"] = torch.tensor(_prefixes(case), dtype=torch.int32, device=dev)
    if case["docs"]:
        s["key_docs"] = _documents(case).to(dev)
        s["query_docs"] = _query_docs(case, s["key_docs"])
    if case["slopes"]:
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device=dev, dtype=torch.float32) / H)
    if case["dir"] == "bwd":
        s["probs"] = _scores_forward(case, s)
        s["grad"] = torch.randn(B, H, Q, K, device=dev, generator=g) * 1e-2
    if own:
        import ctensor_b200 as ct
        s["rules"] = ct.ScoreRules(scale=s["scale"], cap=case["cap"], causal=case["causal"], query_start=s["start"],
                                   key_lengths=s.get("lengths"), prefix=s.get("prefix"), query_docs=s.get("query_docs"),
                                   key_docs=s.get("key_docs"), slopes=s.get("slopes"))
    return s


def _gate_shape(case):
    B, T, C = case["batch"], case["rows"], case["cols"]
    return {"channel": (C,), "batch": (B, 1, C), "full": (B, T, C), "token": (B, T, 1)}[case["gate"]]


def _norm_state(case, g):
    B, T, C = case["batch"], case["rows"], case["cols"]
    dev = "cuda"

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    # the residual stream has a few channels that are far larger than the others
    loud = 1.0 + 9.0 * (torch.rand(C, device=dev, generator=g) < 0.01)
    s = {"x": normal(B, T, C) * loud + 0.1, "f": normal(B, T, C) * 0.7}
    for side in ("pre", "post"):
        if case[side] != "none":
            s[side + "_weight"] = 1.0 + 0.02 * normal(C)
        if case[side] == "layer":
            s[side + "_bias"] = 0.02 * normal(C)
    if case["gate"] != "none":
        s["gate"] = 0.5 + 0.3 * normal(*_gate_shape(case))
    if case["dir"] == "bwd":
        s["y"], _, s["stats"] = _norm_forward(case, s)
        s["grad_y"] = normal(B, T, C) * 1e-3
        s["grad_h"] = normal(B, T, C) * 1e-3
    if own:
        import ctensor_b200 as ct
        kind = {"none": ct.NORM_NONE, "layer": ct.NORM_LAYER, "rms": ct.NORM_RMS}
        s["params"] = ct.ResidualNorm(post=kind[case["post"]], post_weight=s.get("post_weight"),
                                      post_bias=s.get("post_bias"), post_eps=EPS, pre=kind[case["pre"]],
                                      pre_weight=s.get("pre_weight"), pre_bias=s.get("pre_bias"), pre_eps=EPS,
                                      scale=case["scale"])
    return s


def _cut(case, flat=None):
    """The model's tensors as views of one flat buffer (made here if none is given): in a ragged model side
    by side, else each at a multiple of 128 elements with zeros between them."""
    step = 1 if case["model"] == "ragged" else 128
    starts, at = [], 0
    for shape in _shapes(case):
        starts.append(at)
        at += -(-math.prod(shape) // step) * step
    if flat is None:
        flat = torch.zeros(at, device="cuda", dtype=torch.float64 if case["double"] else torch.float32)
    return flat, [flat[a:a + math.prod(shape)].view(shape) for a, shape in zip(starts, _shapes(case))]


def _clip_state(case, g):
    s = {}
    s["flat"], grads = _cut(case)
    for i, t in enumerate(grads):
        t.normal_(generator=g).mul_(1e-3 * 2.0 ** (i % 5))
    s["grads"] = grads
    # a limit that every seed's gradients are above, or below: a norm's expected value times 0.4 or 4
    var = sum(t.numel() * (1e-3 * 2.0 ** (i % 5)) ** 2 for i, t in enumerate(grads))
    if case["p"] == 2.0:
        expected = math.sqrt(var)
    elif case["p"] == 1.0:
        expected = math.sqrt(2.0 / math.pi) * sum(t.numel() * 1e-3 * 2.0 ** (i % 5) for i, t in enumerate(grads))
    else:
        expected = 1e-3 * max(2.0 ** (i % 5) * math.sqrt(2.0 * math.log(2.0 * t.numel())) for i, t in enumerate(grads))
    s["max_norm"] = expected * (0.4 if case["clipped"] else 1e4)
    if own:
        import ctensor_b200 as ct
        s["list"] = ct.TensorList(grads)
    if case["clipped"]:
        s["flat_out"], s["out"] = _cut(case)
        if own:
            s["out_list"] = ct.TensorList(s["out"])
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"scores": _scores_state, "norm": _norm_state, "clip": _clip_state}[case["op"]](case, g)
    s["case"] = case
    return s


EPS = 1e-5


# ---- the plain forms ------------------------------------------------------------------------------------
def _mask(case, s):
    """The mask from the tensors that the call is given: bool [B, 1, Q, K]."""
    dev = s["start"].device
    j = torch.arange(case["keys"], device=dev)[None, None, :]
    ok = torch.ones(case["batch"], case["queries"], case["keys"], dtype=torch.bool, device=dev)
    if case["causal"]:
        see = j <= s["start"][:, None, None] + torch.arange(case["queries"], device=dev)[None, :, None]
        ok = see | (j < s["prefix"][:, None, None]) if case["prefix"] else see
    if case["lengths"]:
        ok = ok & (j < s["lengths"][:, None, None])
    if case["docs"]:
        ok = ok & (s["query_docs"][:, :, None] == s["key_docs"][:, None, :])
    return ok[:, None]


def _distance(case, s):
    """|position of the query - position of the key|: [B, 1, Q, K]."""
    dev = s["start"].device
    pos = s["start"][:, None] + torch.arange(case["queries"], device=dev)[None, :]
    return (pos[:, None, :, None] - torch.arange(case["keys"], device=dev)).abs()


def _scores_forward(case, s):
    t = s["scores"] * s["scale"]
    if case["cap"]:
        t = torch.tanh(t / case["cap"]) * case["cap"]
    if case["slopes"]:      # in 64 bits: the product of a far distance loses the score in 32
        t = t.double() - s["slopes"].double()[None, :, None, None] * _distance(case, s)
    ok = _mask(case, s)
    t = torch.where(ok, t, -math.inf)
    m = t.amax(dim=-1, keepdim=True)
    e = torch.exp((t - torch.where(m == -math.inf, 0.0, m)).float())
    z = e.sum(dim=-1, keepdim=True)
    return torch.where(z > 0, e / z, 0.0)


def _scores_backward(case, s):
    ok = _mask(case, s)
    p, grad = s["probs"], s["grad"]
    dp = torch.where(ok, grad, 0.0)
    dt = p * (dp - (p * dp).sum(dim=-1, keepdim=True))
    ds = dt * s["scale"]
    if case["cap"]:
        th = torch.tanh(s["scores"] * s["scale"] / case["cap"])
        ds = ds * (1.0 - th * th)
    ds = torch.where(ok, ds, 0.0)
    if not case["slopes"]:
        return [ds]
    return [ds, -(dt.double() * _distance(case, s)).sum(dim=(0, 2, 3)).float()]


def _norm_forward(case, s):
    x, f = s["x"], s["f"]
    stats = torch.zeros(x.shape[:-1] + (4,), device=x.device)
    stats[..., 1] = 1.0
    stats[..., 3] = 1.0

    def norm(v, side, at):
        kind = case[side]
        if kind == "none":
            return v
        if kind == "layer":
            mean = v.mean(dim=-1, keepdim=True)
            v = v - mean
            stats[..., at] = mean[..., 0]
        rstd = ((v * v).mean(dim=-1, keepdim=True) + EPS) ** -0.5
        stats[..., at + 1] = rstd[..., 0]
        v = v * rstd * s[side + "_weight"]
        return v + s[side + "_bias"] if kind == "layer" else v

    n = norm(f, "post", 0)
    y = x + (n * case["scale"] if case["gate"] == "none" else n * s["gate"] * case["scale"])
    return y, norm(y, "pre", 2), stats


def _norm_backward(case, s):
    f, y, stats = s["f"], s["y"], s["stats"]
    cols = y.shape[-1]
    out = {}

    def norm_grad(v, up, side, at):
        """The gradient of N(v) for an incoming gradient `up`, and those of its weight and bias."""
        kind = case[side]
        if kind == "none":
            return up
        rstd = stats[..., at + 1:at + 2]
        hat = (v - stats[..., at:at + 1]) * rstd if kind == "layer" else v * rstd
        out[side + "_weight"] = (up * hat).reshape(-1, cols).double().sum(dim=0).float()
        if kind == "layer":
            out[side + "_bias"] = up.reshape(-1, cols).double().sum(dim=0).float()
        a = up * s[side + "_weight"]
        d = a - hat * (a * hat).mean(dim=-1, keepdim=True)
        if kind == "layer":
            d = d - a.mean(dim=-1, keepdim=True)
        return d * rstd

    dx = s["grad_y"] + norm_grad(y, s["grad_h"], "pre", 2)
    dn = dx * case["scale"]
    if case["gate"] != "none":
        n = f
        if case["post"] != "none":
            n = (f - stats[..., 0:1]) * stats[..., 1:2] * s["post_weight"]
            if case["post"] == "layer":
                n = n + s["post_bias"]
        dg, gate = n * dn, s["gate"]
        out["gate"] = _fold(dg, _gate_shape(case))
        dn = dn * gate
    df = norm_grad(f, dn, "post", 0)
    return [dx, df] + [out[k] for k in NORM_GRADS if k in out]


NORM_GRADS = ("gate", "post_weight", "post_bias", "pre_weight", "pre_bias")


def _fold(t, shape):
    """The sum over the dims in which a tensor of `shape` was broadcast."""
    if len(shape) == 1:
        return t.double().sum(dim=(0, 1)).float()
    dims = [d for d in range(3) if shape[d] == 1 and t.shape[d] != 1]
    return t.double().sum(dim=dims, keepdim=True).float() if dims else t


def _clip_plain(case, s):
    p = case["p"]
    if p == math.inf:
        total = torch.stack([t.abs().amax() for t in s["grads"]]).amax().double()
    elif p == 1.0:
        total = torch.stack([t.double().abs().sum() for t in s["grads"]]).sum()
    else:
        total = torch.stack([t.double().square().sum() for t in s["grads"]]).sum().sqrt()
    dtype = s["grads"][0].dtype
    coef = torch.where((total > s["max_norm"]) & (total < math.inf), s["max_norm"] / total, 1.0).to(dtype)
    if not case["clipped"]:
        for t in s["grads"]:
            t.mul_(coef)
        return [total.to(dtype).reshape(1), s["flat"]]
    for t, o in zip(s["grads"], s["out"]):
        torch.mul(t, coef, out=o)
    return [total.to(dtype).reshape(1), s["flat_out"]]


# ---- one pass -------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "scores":
        return [_scores_forward(case, state)] if case["dir"] == "fwd" else _scores_backward(case, state)
    if case["op"] == "norm":
        return list(_norm_forward(case, state)) if case["dir"] == "fwd" else _norm_backward(case, state)
    return _clip_plain(case, state)


def _run_own(case, s):
    import ctensor_b200 as ct
    if case["op"] == "scores":
        if case["dir"] == "fwd":
            return [ct.score_softmax(s["scores"], s["rules"])]
        ds, slopes = ct.score_softmax_backward(s["grad"], s["probs"], s["rules"], scores=s["scores"] if case["cap"] else None,
                                               want_slopes=case["slopes"])
        return [ds, slopes] if case["slopes"] else [ds]
    if case["op"] == "norm":
        if case["dir"] == "fwd":
            return list(ct.residual_norm(s["x"], s["f"], s["params"], gate=s.get("gate")))
        g = ct.residual_norm_backward(s["f"], s["y"], s["stats"], s["params"], grad_y=s["grad_y"], grad_h=s["grad_h"],
                                      gate=s.get("gate"))
        return [g.x, g.f] + [getattr(g, k) for k in NORM_GRADS if getattr(g, k) is not None]
    norm = ct.clip_grad_norm(s["list"], s["max_norm"], p=case["p"], out=s.get("out_list"))
    return [norm, s["flat_out"] if case["clipped"] else s["flat"]]


# ---- what a pass cannot do without ----------------------------------------------------------------------
def work(case):
    if case["op"] == "scores":
        every = case["batch"] * case["heads"] * case["queries"] * case["keys"]
        seen = int(_admitted(case).sum()) * case["heads"]
        if case["dir"] == "fwd":
            return {"bytes": 4 * seen + 4 * every, "flops": seen * (12 if case["cap"] else 6)}
        reads = 12 if case["cap"] else 8
        return {"bytes": reads * seen + 4 * every, "flops": seen * (14 if case["cap"] else 6)}
    if case["op"] == "norm":
        rows, cols = case["batch"] * case["rows"], case["cols"]
        gate = 0 if case["gate"] == "none" else math.prod(_gate_shape(case))
        if case["dir"] == "fwd":      # x, f in; y, h out; four statistics a row
            return {"bytes": 16 * rows * cols + 16 * rows + 4 * gate + 8 * cols, "flops": 14 * rows * cols}
        return {"bytes": 24 * rows * cols + 16 * rows + 8 * gate + 16 * cols, "flops": 30 * rows * cols}
    n = sum(math.prod(s) for s in _shapes(case))
    size = 8 if case["double"] else 4
    return {"bytes": n * size * (2 if case["clipped"] else 1), "flops": n * (3 if case["clipped"] else 2)}


# ---- the definition in 64 bits --------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    return {"scores": _exact_scores, "norm": _exact_norm, "clip": _exact_clip}[case["op"]](case, state)


def _exact_scores(case, s):
    """Sequence by sequence, so that the 64-bit temporaries stay small."""
    B, H, Q, K = case["batch"], case["heads"], case["queries"], case["keys"]
    result = torch.empty(B, H, Q, K, dtype=torch.float64, device="cuda")
    slope_grad = torch.zeros(H, dtype=torch.float64, device="cuda")
    allowed = _admitted(case, "cuda")
    key_at = torch.arange(K, device="cuda", dtype=torch.float64)
    for b, start in enumerate(_query_starts(case)):
        away = (torch.arange(start, start + Q, device="cuda", dtype=torch.float64)[:, None] - key_at[None, :]).abs()
        closed = ~allowed[b, 0]
        for h in range(H):
            raw = s["scores"][b, h].double() * s["scale"]
            slow = torch.tanh(raw / case["cap"]) if case["cap"] else None
            if case["dir"] == "fwd":
                logit = raw if slow is None else case["cap"] * slow
                if case["slopes"]:
                    logit = logit - float(s["slopes"][h]) * away
                logit = logit.masked_fill(closed, -math.inf)
                top = logit.max(dim=1, keepdim=True).values
                weight = torch.exp(logit - top.masked_fill(top == -math.inf, 0.0))
                whole = weight.sum(dim=1, keepdim=True)
                result[b, h] = weight / whole.masked_fill(whole == 0.0, 1.0)
                continue
            prob = s["probs"][b, h].double()
            up = s["grad"][b, h].double().masked_fill(closed, 0.0)
            inner = prob * (up - torch.einsum("qk,qk->q", prob, up)[:, None])
            if case["slopes"]:
                slope_grad[h] -= torch.einsum("qk,qk->", inner, away)
            result[b, h] = (inner * s["scale"] if slow is None else inner * s["scale"] * (1.0 - slow ** 2)).masked_fill(closed, 0.0)
    return [result, slope_grad] if case["dir"] == "bwd" and case["slopes"] else [result]


def _exact_norm(case, s):
    """The forward pass written with variances; the gradients by differentiating it."""
    wide = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}

    def normed(v, kind, weight, bias):
        if kind == "none":
            return v
        centre = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
        spread = ((v - centre) ** 2).sum(-1, keepdim=True) / v.shape[-1]
        out = (v - centre) / torch.sqrt(spread + EPS) * weight
        return out if bias is None else out + bias

    def statistics(v, kind):
        if kind == "none":
            return [torch.zeros_like(v[..., 0]), torch.ones_like(v[..., 0])]
        centre = v.mean(-1) if kind == "layer" else torch.zeros_like(v[..., 0])
        return [centre, 1.0 / torch.sqrt(((v - centre[..., None]) ** 2).sum(-1) / v.shape[-1] + EPS)]

    if case["dir"] == "fwd":
        branch = normed(wide["f"], case["post"], wide.get("post_weight"), wide.get("post_bias"))
        y = wide["x"] + case["scale"] * wide.get("gate", 1.0) * branch
        h = normed(y, case["pre"], wide.get("pre_weight"), wide.get("pre_bias"))
        return [y, h, torch.stack(statistics(wide["f"], case["post"]) + statistics(y, case["pre"]), dim=-1)]
    names = ["f"] + [k for k in NORM_GRADS if k in wide]
    leaves = {k: wide[k].clone().requires_grad_() for k in names + ["y"]}
    h = normed(leaves["y"], case["pre"], leaves.get("pre_weight"), leaves.get("pre_bias"))
    through = torch.autograd.grad(h, [leaves["y"]] + [leaves[k] for k in ("pre_weight", "pre_bias") if k in leaves], wide["grad_h"])
    total = wide["grad_y"] + through[0]
    branch = case["scale"] * leaves.get("gate", 1.0) * normed(leaves["f"], case["post"], leaves.get("post_weight"), leaves.get("post_bias"))
    first = [k for k in ("f", "gate", "post_weight", "post_bias") if k in leaves]
    back = torch.autograd.grad(branch, [leaves[k] for k in first], total)
    return [total] + list(back) + list(through[1:])


def _exact_clip(case, s):
    wide = torch.float64
    if case["p"] == math.inf:
        total = max(float(t.abs().max()) for t in s["grads"])
    elif case["p"] == 1.0:
        total = math.fsum(float(t.abs().sum(dtype=wide)) for t in s["grads"])
    else:
        total = math.sqrt(math.fsum(float(torch.linalg.vector_norm(t, dtype=wide)) ** 2 for t in s["grads"]))
    factor = min(1.0, s["max_norm"] / total)
    flat = torch.zeros(s["flat"].numel(), dtype=wide, device="cuda")
    for t, o in zip(s["grads"], _cut(case, flat)[1]):
        o.copy_(t).mul_(factor)
    return [torch.tensor([total], dtype=wide), flat]
