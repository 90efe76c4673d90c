"""Plain 64-bit forms of the transformer-step operators and the rounding bounds their tests use.

Bounds count half steps of fp32, U = 2^-24 relative to the value rounded, and are worst cases of the
arithmetic that each operator documents, not fitted to results."""
import torch

U = 2.0 ** -24


# ---- scores ---------------------------------------------------------------------------------------------
def admitted(shape, rules, device):
    """bool [B, 1, Q, K]; ``rules``: the keyword arguments of ScoreRules."""
    B, _, Q, K = shape
    j = torch.arange(K, device=device)[None, None, :]
    pos = positions(shape, rules, device)[:, :, None]
    ok = torch.ones(B, Q, K, dtype=torch.bool, device=device)
    if rules.get("causal"):
        see = j <= pos
        if rules.get("prefix") is not None:
            see = see | (j < rules["prefix"].long()[:, None, None])
        ok = ok & see
    if rules.get("key_lengths") is not None:
        ok = ok & (j < rules["key_lengths"].long()[:, None, None])
    if rules.get("key_docs") is not None:
        ok = ok & (rules["query_docs"][:, :, None] == rules["key_docs"][:, None, :])
    return ok[:, None]


def positions(shape, rules, device):
    B, _, Q, K = shape
    start = rules.get("query_start")
    start = torch.full((B,), K - Q, device=device) if start is None else start.long()
    return start[:, None] + torch.arange(Q, device=device)[None, :]


def distance(shape, rules, device):
    pos = positions(shape, rules, device)
    return (pos[:, None, :, None] - torch.arange(shape[3], device=device)).abs().double()


def logits(s, rules):
    t = s * rules.get("scale", 1.0)
    if rules.get("cap"):
        t = rules["cap"] * torch.tanh(t / rules["cap"])
    if rules.get("slopes") is not None:
        t = t - rules["slopes"].to(t)[None, :, None, None] * distance(s.shape, rules, s.device)
    return t


def score_softmax(s, rules):
    """Differentiable in ``s`` (float64) and, given as float64 tensors, in the slopes."""
    ok = admitted(s.shape, rules, s.device)
    t = torch.where(ok, logits(torch.where(ok, s, torch.zeros((), dtype=s.dtype, device=s.device)), rules), -torch.inf)
    top = t.amax(-1, keepdim=True).detach() if s.shape[-1] else t
    e = torch.exp(t - torch.where(top == -torch.inf, 0.0, top))
    z = e.sum(-1, keepdim=True)
    return torch.where(ok, e / torch.where(z == 0.0, 1.0, z), 0.0)


def score_bound(s, p, rules):
    """|error| of a probability.  t: at most four roundings and a tanh within 2 steps (4 U) of a value no larger
    than T = |t| + bias, so t and the maximum are off by 8 U T each; their difference, of at most 2 T, is rounded
    (2 U T) and multiplied by log2(e), a rounded constant (4 U T): each exponential is off by 22 U T relative,
    the instruction for it by 2^-22 = 4 U, the sum (chains of at most 64 terms, then a tree of at most 13) by 77 U, reciprocal and
    product by 2 U."""
    ok = admitted(s.shape, rules, s.device)
    bare = {k: v for k, v in rules.items() if k != "slopes"}
    T = torch.where(ok, logits(torch.where(ok, s, 0.0), bare).abs(), 0.0)
    if rules.get("slopes") is not None:
        d = distance(s.shape, rules, s.device)
        d = torch.where(ok, d, torch.inf)
        near = d.amin(-1, keepdim=True)
        # the kernel measures distances from the nearest key that causal, prefix and length rules leave, at most
        # K - 1 away from the nearest admitted one
        d = torch.where(ok, d - torch.where(near == torch.inf, 0.0, near), 0.0)
        extra = s.shape[-1] if rules.get("key_docs") is not None else 0
        T = T + rules["slopes"].double().abs()[None, :, None, None] * (d + extra)
    top = T.amax(-1, keepdim=True)
    return p * U * (22.0 * top + 83.0) + 1e-37


def score_gradients(s, p, dp, rules):
    """(ds, dslopes, bound of ds, bound of dslopes) from the definition, in float64; `p` as given."""
    ok = admitted(p.shape, rules, p.device)
    scale = rules.get("scale", 1.0)
    dp, p = torch.where(ok, dp, 0.0), torch.where(ok, p, 0.0)
    D = (p * dp).sum(-1, keepdim=True)
    S = (p * dp).abs().sum(-1, keepdim=True)
    dt = p * (dp - D)
    # D: 77 roundings of partial sums no larger than S; the difference and the product two more
    dt_bound = p * U * (78.0 * S + 4.0 * (dp.abs() + D.abs()))
    slow = torch.ones_like(p)
    if rules.get("cap"):
        slow = torch.where(ok, 1.0 - torch.tanh(torch.where(ok, s, 0.0) * scale / rules["cap"]) ** 2, 0.0)
    ds = dt * scale * slow
    # the tanh is within 4 U of a value of at most 1, its argument within 3 U, squared and subtracted: 16 U
    bound = abs(scale) * (dt_bound + (16.0 * U + 3.0 * U) * dt.abs()) + 1e-37
    if rules.get("slopes") is None:
        return ds, None, bound, None
    d = distance(p.shape, rules, p.device)
    dslopes = -(d * dt).sum((0, 2, 3))
    # distance and product rounded, chains of at most 32 terms in fp32, fp64 from there, one rounding at the end
    dslopes_bound = (d * dt_bound + 36.0 * U * d * dt.abs()).sum((0, 2, 3)) + U * dslopes.abs()
    return ds, dslopes, bound, dslopes_bound


# ---- residual norm ----------------------------------------------------------------------------------------
def normed(v, kind, weight, bias, eps):
    if kind == 0:
        return v
    mean = v.mean(-1, keepdim=True) if kind == 1 else 0.0
    out = (v - mean) / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)
    if weight is not None:
        out = out * weight
    return out if bias is None else out + bias


def row_numbers(v, kind, eps):
    """(mean, rstd) of the rows, keepdim."""
    if kind == 0:
        return torch.zeros_like(v[..., :1]), torch.ones_like(v[..., :1])
    mean = v.mean(-1, keepdim=True) if kind == 1 else torch.zeros_like(v[..., :1])
    return mean, 1.0 / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)


def norm_bound(v, kind, weight, bias, eps):
    """|error| of N(v): the mean rounded once (U |mean|), rstd within 2 U, the difference, two products and
    the bias one each."""
    if kind == 0:
        return torch.zeros_like(v)
    mean, rstd = row_numbers(v, kind, eps)
    w = 1.0 if weight is None else weight.abs()
    b = 0.0 if bias is None else bias.abs()
    return U * (2.0 * mean.abs() * rstd * w + 6.0 * ((v - mean) * rstd).abs() * w + b + 1e-30)


def norm_gradient(v, up, up_bound, kind, weight, eps, rows_in_a_sum):
    """(dv, bound, {weight, bias gradients and bounds}) of N at v for the incoming gradient ``up`` that is known
    within ``up_bound``."""
    cols = v.shape[-1]
    if kind == 0:
        return up, up_bound, {}
    mean, rstd = row_numbers(v, kind, eps)
    hat = (v - mean) * rstd
    hat_bound = U * (5.0 * hat.abs() + 2.0 * mean.abs() * rstd)
    w = torch.ones(cols, dtype=v.dtype, device=v.device) if weight is None else weight
    a, a_bound = up * w, up_bound * w.abs() + U * (up * w).abs()
    m1 = a.mean(-1, keepdim=True) if kind == 1 else 0.0
    m2 = (a * hat).mean(-1, keepdim=True)
    # a thread's chain of at most 16 columns, then a tree of at most 13
    m1_bound = (a_bound + 30.0 * U * a.abs()).mean(-1, keepdim=True) if kind == 1 else 0.0
    m2_bound = (a_bound * hat.abs() + a.abs() * hat_bound + 31.0 * U * (a * hat).abs()).mean(-1, keepdim=True)
    inner = a - m1 - hat * m2
    size = a.abs() + (m1.abs() if kind == 1 else 0.0) + (hat * m2).abs()
    bound = rstd * (a_bound + m1_bound + hat_bound * m2.abs() + hat.abs() * m2_bound + 8.0 * U * size)
    flat = lambda t: t.reshape(-1, cols).sum(0)
    steps = (rows_in_a_sum + 4.0) * U
    sums = {"weight": (flat(up * hat), flat(up_bound * hat.abs() + up.abs() * hat_bound + steps * (up * hat).abs())),
            "bias": (flat(up), flat(up_bound + steps * up.abs()))}
    return rstd * inner, bound, sums


def fold_like(t, shape):
    while t.dim() > len(shape):
        t = t.sum(0)
    dims = [d for d in range(t.dim()) if shape[d] == 1 and t.shape[d] != 1]
    return t.sum(dims, keepdim=True) if dims else t


def residual_norm_gradients(f, y, pre, post, gate, scale, dy, dh, eps=1e-5):
    """All gradients and their bounds, {name: (value, bound)}, in float64.  pre / post: (kind, weight, bias)."""
    cols, rows = y.shape[-1], y[..., 0].numel()
    dy = torch.zeros_like(y) if dy is None else dy
    res = {}
    if pre[0]:
        g, b, sums = norm_gradient(y, dh, torch.zeros_like(dh), pre[0], pre[1], eps, rows)
        res.update({"pre_" + k: v for k, v in sums.items()})
    else:
        g, b = torch.zeros_like(y), torch.zeros_like(y)
    dx = dy + g
    dx_bound = b + 3.0 * U * (dx.abs() + g.abs())
    res["x"] = (dx, dx_bound)
    if f is None:
        return res
    factor = scale if gate is None else scale * gate
    dn, dn_bound = dx * factor, dx_bound * abs(factor) + 3.0 * U * (dx * factor).abs()
    if gate is not None:
        n = normed(f, post[0], post[1], post[2], eps)
        n_bound = norm_bound(f, post[0], post[1], post[2], eps)
        terms = scale * n * dx
        each = abs(scale) * (n_bound * dx.abs() + n.abs() * dx_bound) + 4.0 * U * terms.abs()
        res["gate"] = (fold_like(terms, gate.shape), fold_like(each + (rows + 34.0) * U * terms.abs(), gate.shape))
    df, df_bound, sums = norm_gradient(f, dn.expand_as(f), dn_bound.expand_as(f), post[0], post[1], eps, rows)
    res["f"] = (df, df_bound + 2.0 * U * df.abs())
    res.update({"post_" + k: v for k, v in sums.items()})
    return res
