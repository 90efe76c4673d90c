"""GPU tests of the transformer-step operators where their kernels' limits lie: clusters of CTAs, far documents, very
many rows, values near the ends of their types; against plain forms in 64 bits."""
import math

import pytest
import torch

import transformer_ref as ref
from test_gpu_transformer_ops import DEV, gen, ints, randn, vectors, within
from transformer_ref import U

pytestmark = pytest.mark.gpu


# ---- clusters of CTAs -------------------------------------------------------------------------------------
@pytest.mark.parametrize("keys", [5000, 30001, 140000])
def test_clusters_whose_ctas_have_nothing_to_load(ct, keys):
    """Rows in clusters (held and swept, both directions) of which most CTAs see no admitted key and so come to the
    cluster's first exchange as soon as they start, many launches in a row."""
    g = gen(keys)
    B, H = 6, 2
    s, dp = randn(g, B, H, 1, keys) * 3, randn(g, B, H, 1, keys)
    rules = {"scale": 0.5, "causal": True, "cap": 6.0, "key_lengths": ints([0, 1, 7, 600, 2100, keys]), "slopes": randn(g, H).abs() * 0.01}
    r = ct.ScoreRules(**rules)
    want = ref.score_softmax(s.double(), rules)
    runs = []
    for _ in range(20):
        p = ct.score_softmax(s, r)
        runs.append((p, *ct.score_softmax_backward(dp, p, r, scores=s, want_slopes=True)))
    p, ds, dslopes = runs[0]
    within(p, want, ref.score_bound(s.double(), want, rules), "probabilities")
    w, ws, bound, sbound = ref.score_gradients(s.double(), p.double(), dp.double(), rules)
    within(ds, w, bound, "score gradients")
    within(dslopes, ws, sbound, "slope gradients")
    assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(run, runs[0]))


@pytest.mark.parametrize("cols", [8196, 16388, 32768])
def test_clusters_of_norm_rows_many_times(ct, cols):
    """Rows in clusters, the last CTA's slice smaller than the others', many launches in a row."""
    g = gen(cols)
    x, f, dy, dh = (randn(g, 9, cols) for _ in range(4))
    pre, post = vectors(g, 2, True, False, cols), vectors(g, 2, True, False, cols)
    params = ct.ResidualNorm(pre=2, pre_weight=pre[1], post=2, post_weight=post[1])
    runs = []
    for _ in range(20):
        y, h, stats = ct.residual_norm(x, f, params)
        n = ct.residual_norm_backward(f, y, stats, params, grad_y=dy, grad_h=dh)
        runs.append((y, h, stats, n.x, n.f, n.pre_weight, n.post_weight))
    y = runs[0][0]
    want = x.double() + ref.normed(f.double(), 2, post[1].double(), None, 1e-5)
    within(y, want, ref.norm_bound(f.double(), 2, post[1].double(), None, 1e-5) + U * (4 * (want - x.double()).abs() + want.abs()), "y")
    grads = ref.residual_norm_gradients(f.double(), y.double(), (2, pre[1].double(), None), (2, post[1].double(), None), None, 1.0, dy.double(), dh.double())
    for name, t in zip(("x", "f", "pre_weight", "post_weight"), runs[0][3:]):
        within(t, grads[name][0], grads[name][1] + 1e-36, "gradient of " + name)
    assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(run, runs[0]))


# ---- the second launch of the norm gradients ----------------------------------------------------------------
@pytest.mark.parametrize("cols", [200, 4096])
@pytest.mark.parametrize("last", ["row", "value"])
def test_gate_gradients_that_need_no_second_launch(ct, cols, last):
    """No weights, and gate rows that end where a team's rows do on a machine of 148 SMs, so nothing is left to add
    up; what comes next in the stream reads the results at once."""
    g = gen(cols)
    sequences, rows = 296, 8
    x, f, dy, dh = (randn(g, sequences, rows, cols) for _ in range(4))
    gate = randn(g, sequences, 1, cols if last == "row" else 1)
    params = ct.ResidualNorm(pre=2, post=2)
    y, h, stats = ct.residual_norm(x, f, params, gate=gate)
    want = ref.residual_norm_gradients(f.double(), y.double(), (2, None, None), (2, None, None), gate.double(), 1.0, dy.double(), dh.double())
    torch.cuda.synchronize()
    for _ in range(20):
        n = ct.residual_norm_backward(f, y, stats, params, grad_y=dy, grad_h=dh, gate=gate)
        read = [t.clone() for t in (n.x, n.f, n.gate)]
        for t in (n.x, n.f, n.gate):
            t.fill_(math.nan)                            # the next call's results lie in the same memory
        for name, t in zip(("x", "f", "gate"), read):
            within(t, want[name][0], want[name][1] + 1e-36, "gradient of " + name)
        del n


# ---- distance bias with documents ----------------------------------------------------------------------------
def far_bound(s, p, rules):
    """|error| of a probability when the bias is counted from the nearest admitted key, documents among the rules or not.
    As ref.score_bound, but key by key: a logit t of a value and a bias of together T is off by 8 U T, its difference x to the
    maximum, rounded and multiplied by a rounded log2(e), by 3 U |x| more, an exponential by 4 U; a probability by
    that of its own key, that of the sum (each key's weighted with its probability), and 79 U for sum, reciprocal and product."""
    ok = ref.admitted(s.shape, rules, s.device)
    bare = {k: v for k, v in rules.items() if k != "slopes"}
    t = ref.logits(torch.where(ok, s, 0.0), bare)
    d = torch.where(ok, ref.distance(s.shape, rules, s.device), math.inf)
    near = d.amin(-1, keepdim=True)
    d = torch.where(ok, d - torch.where(near == math.inf, 0.0, near), 0.0)
    bias = rules["slopes"].double()[None, :, None, None] * d
    T = torch.where(ok, t.abs(), 0.0) + bias.abs()
    x = torch.where(ok, t - bias, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.where(ok, torch.where(top == -math.inf, 0.0, top) - x, 0.0)
    each = torch.where(ok, 8.0 * T + 3.0 * x + 4.0, 0.0)
    return p * U * (each + (p * each).sum(-1, keepdim=True) + 79.0) + 1e-37


def far_rules(g, H, Q, K):
    """Two sequences; in the first the queries see the 60 first keys only, in the second a few keys in every 1000th
    stretch, or none; slopes from 1/2 up."""
    docs = torch.full((2, K), 9, dtype=torch.int32, device=DEV)
    docs[0, :60] = 1
    docs[1, 7::1000] = 1
    docs[1, 8::1000] = 2
    who = torch.ones(2, Q, dtype=torch.int32, device=DEV)
    who[1, ::2], who[1, -1] = 2, 5
    return {"scale": 0.5, "query_docs": who, "key_docs": docs, "slopes": 0.5 + torch.rand(H, device=DEV, generator=g)}


@pytest.mark.parametrize("keys", [100, 700, 3001, 8192, 16384, 30001, 120000])
@pytest.mark.parametrize("cap", [0.0, 3.0])
def test_score_bias_of_far_documents(ct, keys, cap):
    g = gen(keys)
    B, H, Q = 2, 3, 5
    s = randn(g, B, H, Q, keys) * 3
    rules = dict(far_rules(g, H, Q, keys), cap=cap)
    for start in (None, ints([keys - 1, 0]), ints([2_000_000, -2_000_000])):
        if start is not None:
            rules["query_start"] = start
        p = ct.score_softmax(s, ct.ScoreRules(**rules))
        want = ref.score_softmax(s.double(), rules)
        within(p, want, far_bound(s.double(), want, rules), f"probabilities from {start}")


def test_score_bias_of_far_documents_beyond_exact_floats(ct):
    """Positions that Float32 does not tell apart."""
    g = gen(4)
    K = 20_000_001
    s = randn(g, 1, 1, 2, K)
    docs = torch.zeros(1, K, dtype=torch.int32, device=DEV)
    docs[0, 1001:1101] = 1
    rules = {"query_docs": ints([[1, 1]]), "key_docs": docs, "slopes": torch.full((1,), 0.3, device=DEV), "causal": True}
    p = ct.score_softmax(s, ct.ScoreRules(**rules))[..., :2000]
    assert float(p[..., :1001].sum()) == 0
    t = s[..., 1001:1101].double() - 0.3000000119 * torch.arange(99, -1, -1, device=DEV)
    want = torch.softmax(t, -1)
    within(p[..., 1001:1101], want, want * U * (22.0 * t.abs().amax(-1, keepdim=True) + 83.0), "probabilities")


@pytest.mark.parametrize("keys", [90, 1024, 1027, 5000, 16384, 30001, 120000])
@pytest.mark.parametrize("causal", [False, True])
def test_score_bias_in_packed_documents(ct, keys, causal):
    """Queries inside their documents: the keys next to them, which have most of the weight, keep all their bits."""
    g = gen(keys + 5)
    B, H, Q = 1, 2, 8
    s = randn(g, B, H, Q, keys)
    docs = (torch.arange(keys, device=DEV, dtype=torch.int32) * 3 // keys)[None].contiguous()
    at = keys - 3 * Q
    rules = {"causal": causal, "query_docs": docs[:, at:at + Q].contiguous(), "key_docs": docs, "query_start": ints([at]),
             "slopes": torch.tensor([0.5, 0.01], device=DEV)}
    p = ct.score_softmax(s, ct.ScoreRules(**rules))
    want = ref.score_softmax(s.double(), rules)
    within(p, want, far_bound(s.double(), want, rules), "probabilities")

@pytest.mark.parametrize("keys", [60, 700, 1001, 5000, 16384, 30001, 120000])
@pytest.mark.parametrize("docs", [False, True])
def test_slope_gradients_of_far_keys(ct, keys, docs):
    """A row's gradients of the logits add up to nothing, so the distance that all of its keys have in common does not
    count.  Probabilities that are multiples of 1/16 and add up to exactly one, so that it does not count in the
    formula in 64 bits either."""
    g = gen(keys + 1)
    B, H, Q = 2, 2, 3
    rules = far_rules(g, H, Q, keys) if docs else {"slopes": torch.rand(H, device=DEV, generator=g)}
    if not docs:
        rules["query_start"] = ints([3_000_000, -1_000_000])
    ok = ref.admitted((B, H, Q, keys), rules, DEV).expand(B, H, Q, keys)
    p = torch.zeros(B, H, Q, keys, device=DEV)
    for b in range(B):
        for h in range(H):
            for q in range(Q):
                allowed = ok[b, h, q].nonzero()[:, 0]
                if len(allowed):
                    pick = allowed[torch.randint(0, len(allowed), (16,), device=DEV, generator=g)]
                    p[b, h, q].index_put_((pick,), torch.full((16,), 1 / 16, device=DEV), accumulate=True)
    dp = randn(g, B, H, Q, keys)
    ds, dslopes = ct.score_softmax_backward(dp, p, ct.ScoreRules(**rules), want_slopes=True)
    w, ws, bound, _ = ref.score_gradients(p.double(), p.double(), dp.double(), rules)
    within(ds, w, bound, "score gradients")
    d = torch.where(ok, ref.distance(p.shape, rules, DEV), math.inf)
    near = d.amin(-1, keepdim=True)
    d = torch.where(ok, d - torch.where(near == math.inf, 0.0, near), 0.0)
    within(dslopes, ws, (d * (bound + 36.0 * U * w.abs())).sum((0, 2, 3)) + 2 * U * ws.abs(), "slope gradients")


# ---- column sums over very many rows ---------------------------------------------------------------------------
@pytest.mark.parametrize("what", ["bias", "gate", "all"])
@pytest.mark.parametrize("rows,cols", [(3_700_001, 4), (2_000_001, 68), (400_000, 260)])
def test_column_sums_over_many_rows(ct, what, rows, cols):
    """Ones among which every thousandth is 2^24: a Float32 sum that has met one of those loses the ones that follow.  At most
    240 rows and up to 16 such sums are added in Float32 (239 U + 15 U), the result is rounded (U)."""
    values = torch.ones(rows, 1, device=DEV)
    values[::1000] = 2.0 ** 24
    incoming = values.expand(rows, cols).contiguous()
    want = float(values.double().sum())
    one = torch.ones(cols, device=DEV)
    x = randn(gen(rows), rows, cols)
    near = lambda got: within(got, torch.full((cols,), want, device=DEV, dtype=torch.float64), torch.full((cols,), 260 * U * want, device=DEV, dtype=torch.float64), what)
    if what == "bias":
        params = ct.ResidualNorm(pre=1, pre_weight=one, pre_bias=one)
        _, _, stats = ct.residual_norm(x, None, params)
        near(ct.residual_norm_backward(None, x, stats, params, grad_h=incoming).pre_bias)
    elif what == "gate":
        params = ct.ResidualNorm(pre=0)
        f = torch.ones_like(x)
        y, _, stats = ct.residual_norm(x, f, params, gate=one)
        near(ct.residual_norm_backward(f, y, stats, params, grad_y=incoming, gate=one).gate)
    else:
        params = ct.ResidualNorm(pre=1, pre_weight=one, pre_bias=one, post=1, post_weight=one, post_bias=one)
        y, _, stats = ct.residual_norm(x, x, params, gate=one)
        near(ct.residual_norm_backward(x, y, stats, params, grad_y=x, grad_h=incoming, gate=one).pre_bias)


@pytest.mark.parametrize("gate", ["batch", "sequence", "token", "channel"])
@pytest.mark.parametrize("cols", [36, 7])
def test_more_teams_than_run_at_once(ct, gate, cols):
    """So many rows that teams come in several waves: gate rows shared inside and across teams, every gradient."""
    g = gen(cols)
    B, T = 1003, 1201
    x, f, dy, dh = (randn(g, B, T, cols) for _ in range(4))
    w = [1 + 0.3 * randn(g, cols) for _ in range(2)]
    shape = {"batch": (B, 1, cols), "sequence": (B, 1, 1), "token": (B, T, 1), "channel": (cols,)}[gate]
    gate = randn(g, *shape)
    params = ct.ResidualNorm(pre=2, pre_weight=w[0], post=2, post_weight=w[1], scale=0.5)
    y, _, stats = ct.residual_norm(x, f, params, gate=gate)
    got = ct.residual_norm_backward(f, y, stats, params, grad_y=dy, grad_h=dh, gate=gate)
    want = ref.residual_norm_gradients(f.double(), y.double(), (2, w[0].double(), None), (2, w[1].double(), None), gate.double(), 0.5, dy.double(), dh.double())
    for name in ("x", "f", "gate", "post_weight", "pre_weight"):
        value, bound = want[name]
        within(getattr(got, name), value, bound + 1e-36, "gradient of " + name)


# ---- norms of rows near the ends of Float32 -------------------------------------------------------------------
@pytest.mark.parametrize("cols", [20, 33, 768, 1001, 2048, 2052, 4100])
@pytest.mark.parametrize("gate", ["none", "full", "token"])
@pytest.mark.parametrize("size,weight", [(1e37, 50.0), (1e20, 1e20), (1e-30, 1e-12), (1e-38, 1.0)])
def test_rms_norms_of_extreme_rows(ct, cols, gate, size, weight):
    """Whatever the rows' size, only their direction counts: y, the next norm and df are those of rows of ordinary size."""
    g = gen(cols)
    B, T = 2, 3
    f = randn(g, B, T, cols) * size
    f[0, 0] = randn(g, cols)                             # an ordinary row among them
    shape = {"none": None, "full": (B, T, cols), "token": (B, T, 1)}[gate]
    gate = None if shape is None else randn(g, *shape).abs() + 0.5
    w = (1.0 + torch.rand(cols, device=DEV, generator=g)) * weight
    x = torch.zeros_like(f)
    params = ct.ResidualNorm(pre=2, pre_eps=0.0, post=2, post_weight=w, post_eps=0.0, scale=0.5)
    y, h, stats = ct.residual_norm(x, f, params, gate=gate)
    n = ref.normed(f.double(), 2, w.double(), None, 0.0)
    factor = 0.5 if gate is None else 0.5 * gate.double()
    want = factor * n
    within(y, want, abs(factor) * ref.norm_bound(f.double(), 2, w.double(), None, 0.0) + 4 * U * want.abs(), "y")
    want = ref.normed(y.double(), 2, None, None, 0.0)
    within(h, want, ref.norm_bound(y.double(), 2, None, None, 0.0) + U * want.abs(), "h")
    _, rstd = ref.row_numbers(f.double(), 2, 0.0)
    within(stats[..., 1], rstd[..., 0], 3 * U * rstd[..., 0], "rstd")


# ---- the exponential ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("keys", [2, 1026, 20001])
def test_score_exponential(ct, keys):
    """Differences x that are exact, from 1/8 to where results end: e^x within 1.25 |x| + 4 half steps, the
    sum of two, reciprocal and product one more each."""
    x = torch.arange(1, 8 * 104, device=DEV) / 8.0
    s = torch.full((1, 1, len(x), keys), -math.inf, device=DEV)
    s[0, 0, :, 0], s[0, 0, :, keys - 1] = 0.0, -x
    p = ct.score_softmax(s, ct.ScoreRules())[0, 0]
    e = torch.exp(-x.double())
    each = 1.25 * x.double() + 4
    want = e / (1 + e)
    slack = torch.where(e < 2.0 ** -125, 2.0 ** -125, 0.0)
    within(p[:, keys - 1], want, want * U * (each + each * e + 8) + slack, "the smaller one")
    within(p[:, 0], 1 / (1 + e), U * (each * e + 8), "the larger one")


# ---- clipping by very small factors ----------------------------------------------------------------------------
@pytest.mark.parametrize("size,limit,p,dtype", [(3e38, 0.5, 2, torch.float32), (1e30, 1e-12, 2, torch.float32), (3e38, 1e-35, 1, torch.float32),
                                                (1e35, 1e-20, math.inf, torch.float32), (1e300, 1e-15, math.inf, torch.float64),
                                                (1e303, 1e-10, 1, torch.float64), (1e10, 1e-12, 2, torch.float32)])
@pytest.mark.parametrize("out", [False, True])
def test_clip_by_very_small_factors(ct, size, limit, p, dtype, out):
    """The norm is finite and far above the limit: two roundings a value, the factor's and the product's."""
    g = gen(11)
    half = U if dtype == torch.float32 else 2.0 ** -53
    grads = [((torch.rand(n, device=DEV, generator=g, dtype=torch.float64) - 0.5) * 2 * size).to(dtype) for n in (1, 7, 9000, 20001)]
    flat = torch.cat(grads).double()
    unit = flat / flat.abs().max()                       # the sums of squares stay in range
    total = {1: unit.abs().sum(), 2: unit.square().sum().sqrt(), math.inf: unit.abs().max()}[p] * flat.abs().max()
    assert bool(total.isfinite())
    have = [t.clone() for t in grads]
    outs = [torch.empty(t.numel() + 3, device=DEV, dtype=dtype)[3 * (i % 2):][:t.numel()] for i, t in enumerate(grads)] if out else None
    n = ct.clip_grad_norm(have, limit, p, out=outs, norm=torch.empty(1, device=DEV, dtype=torch.float64))
    assert abs(float(n) - float(total)) <= 100 * 2.0 ** -53 * float(total)
    small = 2.0 ** -149 if dtype == torch.float32 else 2.0 ** -1074
    for a, b in zip(grads, outs if out else have):
        want = (a.double() / total) * limit              # in this order neither overflows nor vanishes
        within(b, want, (2.0 * half + 110 * 2.0 ** -53) * want.abs() + small, "clipped")


# ---- the cap's slope far beyond the cap ---------------------------------------------------------------------------
@pytest.mark.parametrize("keys", [64, 1001, 1024, 4096, 30001])
def test_gradients_of_scores_far_beyond_the_cap(ct, keys):
    """Scores of up to 40 caps: 1 - tanh^2 within (6.5 x + 12) half steps of itself (2 x of three rounded factors and 4 of the
    exponential, twice the reciprocal's 2 and the sum's 1, products), whatever is left of it."""
    g = gen(keys)
    s = (torch.rand(1, 2, 3, keys, device=DEV, generator=g) - 0.5) * 160.0
    p = torch.full_like(s, 1.0 / keys)
    dp = randn(g, 1, 2, 3, keys)
    rules = {"scale": 0.5, "cap": 1.0}
    ds, _ = ct.score_softmax_backward(dp, p, ct.ScoreRules(**rules), scores=s)
    x = s.double().abs() * 0.5
    slow = 4.0 * torch.exp(-2.0 * x) / (1.0 + torch.exp(-2.0 * x)) ** 2
    bare, _, bound, _ = ref.score_gradients(s.double(), p.double(), dp.double(), {"scale": 0.5})
    within(ds, bare * slow, bound * slow * 1.0001 + (6.5 * x + 14.0) * U * (bare * slow).abs() + 2.0 ** -126, "score gradients")


# ---- infinities and NaN in rows with norms on both sides ------------------------------------------------------
@pytest.mark.parametrize("cols", [8, 33, 768, 2048, 2052])
@pytest.mark.parametrize("kind", [1, 2])
def test_norms_of_rows_that_are_not_finite(ct, cols, kind):
    """What the formula says, at every width: an infinite entry of the stream leaves an RMS norm's other entries 0."""
    g = gen(cols)
    inf, nan = math.inf, math.nan
    x, f = randn(g, 8, cols), randn(g, 8, cols)
    f[:, 3] = 1.0
    for row, (where, value) in enumerate([(x, inf), (x, -inf), (x, nan), (f, inf), (f, -inf), (f, nan)]):
        where[row, 3] = value
    f[6, 3] = -1.0
    x[6, 3] = inf
    params = ct.ResidualNorm(pre=kind, post=kind, scale=0.5)
    y, h, _ = ct.residual_norm(x, f, params)
    want_y = x.double() + 0.5 * ref.normed(f.double(), kind, None, None, 1e-5)
    want_h = ref.normed(want_y, kind, None, None, 1e-5)
    for got, want in ((y, want_y), (h, want_h)):
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
        close = want.isfinite()
        assert bool(((got.double() - want)[close].abs() <= 1e-5 * (1 + want[close].abs())).all())


# ---- calls through the C functions that the Python binding does not make ------------------------------------------
def call_backward(ct, f, y, gate, stats, params, dy, dh, grads):
    """ctb_residual_norm_backward with the gradients in `grads` (name -> tensor) and no others, and a workspace of exactly
    the size that was asked for, with a guard behind it."""
    import ctypes
    L, raw = ct.lib(), ct._raw_view
    views = {k: raw(t) for k, t in grads.items()}
    c = ct.CResidualNormGrads(*(ct._address(views.get(n)) for n, _ in ct.CResidualNormGrads._fields_))
    yv, gv = raw(y), raw(gate)
    need = L.ctb_residual_norm_workspace_bytes(yv, gv)
    ws = torch.full((need + 1024,), 0xAB, dtype=torch.uint8, device=DEV)
    ct.check(L.ctb_residual_norm_backward(raw(f), yv, gv, raw(stats), params.c, raw(dy), raw(dh), ctypes.byref(c), ws.data_ptr(), need,
                                          torch.cuda.current_stream().cuda_stream))
    assert bool((ws[need:] == 0xAB).all()), "written behind the workspace"


WANTED = [("x",), ("gate",), ("f",), ("pre_weight",), ("post_weight", "post_bias"), ("pre_bias", "gate"), ("x", "f", "pre_weight"), ("x", "post_bias"),
          ("x", "f", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias")]


@pytest.mark.parametrize("wanted", WANTED, ids="-".join)
@pytest.mark.parametrize("cols", [96, 301, 2304, 5124])
@pytest.mark.parametrize("gate", ["channel", "batch", "sequence", "full"])
def test_some_of_the_norm_gradients(ct, wanted, cols, gate):
    """Any of the gradients without the others, at every 4-byte phase of what is written."""
    g = gen(cols)
    B, T = 6, 50
    x, f, dy, dh = (randn(g, B, T, cols) for _ in range(4))
    shape = {"channel": (cols,), "batch": (B, 1, cols), "sequence": (B, 1, 1), "full": (B, T, cols)}[gate]
    gate = randn(g, *shape)
    pre, post = vectors(g, 1, True, True, cols), vectors(g, 1, True, True, cols)
    params = ct.ResidualNorm(pre=1, pre_weight=pre[1], pre_bias=pre[2], post=1, post_weight=post[1], post_bias=post[2], scale=0.5)
    y, _, stats = ct.residual_norm(x, f, params, gate=gate)
    d = lambda v: tuple(t.double() if torch.is_tensor(t) else t for t in v)
    want = ref.residual_norm_gradients(f.double(), y.double(), d(pre), d(post), gate.double(), 0.5, dy.double(), dh.double())
    like = {"x": x, "f": f, "gate": gate, "post_weight": post[1], "post_bias": post[2], "pre_weight": pre[1], "pre_bias": pre[2]}
    for phase in (0, 3):
        flats = {n: torch.full((like[n].numel() + 8,), 7.0, device=DEV) for n in wanted}
        grads = {n: flats[n][phase:phase + like[n].numel()].view(like[n].shape) for n in wanted}
        call_backward(ct, f, y, gate, stats, params, dy, dh, grads)
        for n in wanted:
            within(grads[n], want[n][0], want[n][1] + 1e-36, "gradient of " + n)
            assert bool((flats[n][:phase] == 7).all()) and bool((flats[n][phase + like[n].numel():] == 7).all()), n


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 4), (149, 2050), (2400, 64), (300_000, 8), (5, 8200), (40_000, 12300)])
@pytest.mark.parametrize("norms", [(2, 2), (1, 1), (1, 0)], ids=str)
def test_workspace_of_the_size_asked_for(ct, rows, cols, norms):
    """The kernels stay inside the workspace, whichever of them runs and however many teams there are."""
    g = gen(rows)
    if rows * cols > 200_000_000:
        x = randn(g, 1, cols).expand(rows, cols).contiguous()
    else:
        x = randn(g, rows, cols)
    one = torch.ones(cols, device=DEV)
    for gate in (None, one, torch.ones(rows, 1, device=DEV)):
        params = ct.ResidualNorm(pre=norms[0], pre_weight=one, pre_bias=one if norms[0] == 1 else None, post=norms[1], post_weight=one if norms[1] else None)
        y, _, stats = ct.residual_norm(x, x, params, gate=gate)
        grads = {"x": torch.empty_like(x), "f": torch.empty_like(x), "pre_weight": torch.empty_like(one)}
        if norms[1]:
            grads["post_weight"] = torch.empty_like(one)
        if norms[0] == 1:
            grads["pre_bias"] = torch.empty_like(one)
        if gate is not None:
            grads["gate"] = torch.empty_like(gate)
        call_backward(ct, x, y, gate, stats, params, x, x, grads)
        got = ct.residual_norm_backward(x, y, stats, params, grad_y=x, grad_h=x, gate=gate)
        assert all(torch.equal(t, getattr(got, n)) for n, t in grads.items())


# ---- more elements than 32 bits count ---------------------------------------------------------------------------
def test_scores_of_more_than_2_31_elements(ct):
    B, H, Q, K = 1, 2, 34_000, 32_768
    s = torch.zeros(B, H, Q, K, device=DEV)
    g = gen(9)
    s[0, 1, -5:] = randn(g, 5, K) * 3
    rules = {"scale": 0.7, "causal": True, "query_start": ints([5])}
    p = ct.score_softmax(s, ct.ScoreRules(**rules))
    tail = dict(rules, query_start=ints([5 + Q - 5]))
    last = s[:, 1:, -5:].double()
    want = ref.score_softmax(last, tail)
    within(p[:, 1:, -5:], want, ref.score_bound(last, want, tail), "probabilities")
    assert float(p[0, 0, 0, :6].sum()) == pytest.approx(1.0, abs=8 * U) and float(p[0, 1, 10, 16:].abs().sum()) == 0.0
    dp = torch.zeros_like(s)
    dp[0, 1, -5:] = randn(g, 5, K)
    ds, _ = ct.score_softmax_backward(dp, p, ct.ScoreRules(**rules), out=s)
    w, _, bound, _ = ref.score_gradients(last, p[:, 1:, -5:].double(), dp[:, 1:, -5:].double(), tail)
    within(ds[:, 1:, -5:], w, bound, "score gradients")
    assert float(ds[0, 0].abs().amax()) == 0.0


@pytest.mark.parametrize("rows,cols", [(525_000, 4096), (263_000, 8196), (4_300_000, 501)])
@pytest.mark.parametrize("norms", [(2, 2), (1, 0)], ids=str)
def test_norms_of_more_than_2_31_elements(ct, rows, cols, norms):
    """All rows alike, so they all have the result of one row by itself."""
    g = gen(10)
    x, f, dy, dh, gate = (randn(g, 1, cols) for _ in range(5))
    w = 1 + 0.1 * randn(g, cols)
    params = ct.ResidualNorm(pre=norms[0], pre_weight=w, post=norms[1], post_weight=w if norms[1] else None)
    many = lambda t: t.expand(rows, t.shape[-1])
    one = ct.residual_norm(x, f, params, gate=gate)
    got = ct.residual_norm(many(x), many(f), params, gate=many(gate))
    at = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device=DEV)
    for a, b in zip(got, one):
        assert torch.equal(a[at], many(b)[at])
    del got, a
    y, h, stats = one
    one = ct.residual_norm_backward(f, y, stats, params, grad_y=dy, grad_h=dh, gate=gate)
    for fast in (True, False):                           # without grad_y the general kernel runs
        if not fast:
            one = ct.residual_norm_backward(f, y, stats, params, grad_h=dh, gate=gate)
        got = ct.residual_norm_backward(many(f), many(y), many(stats).contiguous(), params, grad_y=many(dy) if fast else None, grad_h=many(dh), gate=many(gate))
        for n in ("x", "f", "gate"):
            assert torch.equal(getattr(got, n)[at], many(getattr(one, n))[at]), n
        want = one.pre_weight.double() * rows
        within(got.pre_weight, want, 260 * U * want.abs() + 1e-30, "gradient of the weight")
        del got


def test_clipping_of_more_than_2_31_elements(ct):
    x = torch.ones(2_200_000_001, device=DEV)
    x[-5:] = torch.tensor([2.0, 4.0, 8.0, 16.0, 32.0], device=DEV)
    total = math.sqrt(2_200_000_001 - 5 + 4 + 16 + 64 + 256 + 1024)
    out = torch.empty(x.numel() + 1, device=DEV)[1:]
    for grads, outs in (([x], [out]), ([x], None)):
        got = float(ct.clip_grad_norm(grads, total / 2, out=outs, norm=torch.empty(1, device=DEV, dtype=torch.float64)))
        assert abs(got - total) <= 1e-12 * total
        y = out if outs else x
        assert y[-7:].tolist() == [0.5, 0.5, 1.0, 2.0, 4.0, 8.0, 16.0] and float(y[0]) == 0.5
        assert float(y[1_000_000_000:1_000_100_000].sum()) == 50_000.0
