"""GPU tests of the steps of a transformer block between its matrix products and of what stands between
the gradients and the optimizer: score_softmax, residual_norm, their gradients, grad_norm and
clip_grad_norm, against plain forms in 64 bits."""
import math

import pytest
import torch

import transformer_ref as ref
from transformer_ref import U

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def within(got, want, bound, what):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} outside their bounds; worst "
                                 f"{float(((got.double() - want).abs() / bound).nan_to_num(math.inf).max()):.3g} times the bound")


# ---- scores -------------------------------------------------------------------------------------------
def make_rules(kind, B, H, Q, K, seed=0):
    r = torch.Generator().manual_seed(seed + 17)
    pick = lambda lo, hi, *shape: torch.randint(lo, hi, shape, generator=r, dtype=torch.int32).to(DEV)
    rules = {"scale": 0.3}
    if "causal" in kind:
        rules["causal"] = True
    if "cap" in kind:
        rules["cap"] = 5.0
    if "start" in kind:          # some queries before every key, some far behind the last one
        rules["query_start"] = pick(-Q - 3, K + 40, B)
    if "prefix" in kind:
        rules["prefix"] = pick(-2, K + 2, B)
    if "lengths" in kind:
        rules["key_lengths"] = pick(0, K + 2, B)
    if "docs" in kind:
        rules["query_docs"], rules["key_docs"] = pick(0, 3, B, Q), pick(0, 4, B, K).sort(dim=1).values.contiguous()
    if "slopes" in kind:
        rules["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device=DEV, dtype=torch.float32) / H)
    return rules


KINDS = ["plain", "causal", "cap", "causal-start-slopes", "causal-prefix-lengths-cap", "docs", "docs-causal-lengths-slopes-cap-start",
         "slopes-start-lengths"]
SCORE_SHAPES = [(1, 1, 1, 1), (2, 3, 5, 1), (2, 3, 4, 7), (1, 2, 33, 128), (2, 2, 9, 253), (1, 3, 17, 512), (2, 2, 6, 1021), (1, 2, 3, 1024),
                (1, 2, 5, 2045), (1, 2, 3, 2048), (2, 1, 3, 4096), (1, 1, 3, 5001), (1, 2, 2, 8192), (1, 2, 3, 8193), (1, 1, 2, 40003)]


@pytest.mark.parametrize("shape", SCORE_SHAPES, ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_score_softmax_and_its_gradients(ct, shape, kind):
    B, H, Q, K = shape
    g = gen(K * 31 + Q)
    rules = make_rules(kind, B, H, Q, K, seed=K)
    s = randn(g, *shape) * 6.0
    ok = ref.admitted(shape, rules, DEV).expand(shape)
    masked = s.masked_fill(~ok, math.nan)                # masked places hold anything
    r = ct.ScoreRules(**rules)
    p = ct.score_softmax(masked, r)
    want = ref.score_softmax(s.double(), rules)
    within(p, want, ref.score_bound(s.double(), want, rules), "probabilities")
    assert not bool(p[~ok].any()) and not bool((~ok.any(-1) & (p.sum(-1) != 0)).any())

    dp = randn(g, *shape)
    slopes = "slopes" in rules
    ds, dslopes = ct.score_softmax_backward(dp.masked_fill(~ok, math.inf), p.masked_fill(~ok, math.nan), r,
                                            scores=masked if "cap" in rules else None, want_slopes=slopes)
    w, ws, bound, sbound = ref.score_gradients(s.double(), p.double(), dp.double(), rules)
    within(ds, w, bound, "score gradients")
    if slopes:
        within(dslopes, ws, sbound, "slope gradients")


@pytest.mark.parametrize("shape", [(2, 4, 37, 20001), (2, 4, 37, 16400), (2, 2, 10, 30001), (1, 3, 11, 20000), (1, 2, 2, 140000)], ids=str)
@pytest.mark.parametrize("kind", ["plain", "causal-prefix-lengths-cap", "docs", "docs-causal-lengths-slopes-cap-start"])
def test_score_long_rows(ct, shape, kind):
    """As many rows as CTAs run at once (each swept by one), and fewer (held or swept by clusters)."""
    test_score_softmax_and_its_gradients(ct, shape, kind)


@pytest.mark.parametrize("keys", [60, 128, 1000, 1001, 4096, 5000, 20000])
def test_score_special_values_in_documents(ct, keys):
    """Every third key in the query's document, with infinities and NaN there and elsewhere."""
    inf, nan = math.inf, math.nan
    g = gen(keys)
    docs = (torch.arange(keys, device=DEV, dtype=torch.int32) % 3)[None].contiguous()
    ok = docs[0] == 1
    s = randn(g, 1, 1, 5, keys)
    s[..., ~ok] = nan
    s[0, 0, 0, 4] = inf
    s[0, 0, 1, 4] = -inf
    s[0, 0, 2, 4] = nan
    s[0, 0, 3, ok] = -inf
    r = ct.ScoreRules(query_docs=ints([[1] * 5]), key_docs=docs)
    p = ct.score_softmax(s, r)[0, 0]
    assert not bool(p[:, ~ok].any())
    assert bool(p[0, ok].isnan().any()) and bool(p[2, ok].isnan().all()) and not bool(p[3].any())
    assert float(p[1, 4]) == 0.0
    for i in (1, 4):
        finite = ok & s[0, 0, i].isfinite()                    # -inf adds exactly nothing; the bound is one of finite logits
        t = s[0, 0, i, finite].double()[None, None, None]
        want = torch.softmax(t, -1)
        within(p[i, finite][None, None, None], want, ref.score_bound(t, want, {}), "probabilities")
    dp = randn(g, 1, 1, 5, keys)
    dp[0, 0, 0, 4], dp[0, 0, 0, 5] = inf, nan                  # one in the document, one outside
    q = p.clone().nan_to_num(0.25)[None, None]
    ds, _ = ct.score_softmax_backward(dp, q, r)
    assert not bool(ds[..., ~ok].any()) and bool(ds[0, 0, 1:].isfinite().all()) and not bool(ds[0, 0, 0, ok].isfinite().any())


def test_score_rows_of_many_sequences_and_a_long_cache(ct):
    """One query per sequence over 140,001 keys (a cluster of CTAs per row), ragged lengths."""
    g = gen(5)
    B, H, K = 3, 2, 140001
    s = randn(g, B, H, 1, K) * 4
    rules = {"scale": 1.0, "causal": True, "key_lengths": ints([1, 70002, K]), "query_start": ints([0, 70001, K - 1]), "cap": 8.0}
    p = ct.score_softmax(s, ct.ScoreRules(**rules))
    want = ref.score_softmax(s.double(), rules)
    within(p, want, ref.score_bound(s.double(), want, rules), "probabilities")
    assert float(p[0, :, 0, 0].sum()) == H
    dp = randn(g, B, H, 1, K)
    ds, _ = ct.score_softmax_backward(dp, p, ct.ScoreRules(**rules), scores=s)
    w, _, bound, _ = ref.score_gradients(s.double(), p.double(), dp.double(), rules)
    within(ds, w, bound, "score gradients")


@pytest.mark.parametrize("keys", [6, 515, 3000, 9000])
def test_score_strides_and_starts(ct, keys):
    """Views into wider buffers, heads and queries exchanged, rows at every 4-byte phase, strided tables."""
    g = gen(keys)
    B, H, Q = 2, 3, 4
    wide = randn(g, B, Q, H, keys + 9) * 3
    docs = torch.randint(0, 2, (B, 2 * keys), device=DEV, dtype=torch.int32, generator=g)
    rules = {"scale": 0.5, "cap": 4.0, "causal": True, "query_docs": ints([[0, 1, 0, 1], [1, 1, 0, 5]]), "key_docs": docs[:, ::2],
             "slopes": randn(g, 2 * H).abs()[::2]}
    for at in (0, 1, 2, 3, 5):
        s = wide[..., at:at + keys].permute(0, 2, 1, 3)
        flat = torch.zeros(B * H * Q * keys + 3, device=DEV)
        out = flat[at % 3:at % 3 + B * H * Q * keys].view(B, H, Q, keys)
        r = ct.ScoreRules(**rules)
        p = ct.score_softmax(s, r, out=out)
        want = ref.score_softmax(s.double(), rules)
        within(p, want, ref.score_bound(s.double(), want, rules), f"probabilities at {at}")
        assert float(flat[:at % 3].abs().sum()) == 0 and float(flat[at % 3 + out.numel():].abs().sum()) == 0
        dp = randn(g, B, Q, H, keys + 1)[..., 1:].permute(0, 2, 1, 3)
        ds, dslopes = ct.score_softmax_backward(dp, p, r, scores=s, want_slopes=True)
        w, ws, bound, sbound = ref.score_gradients(s.double(), p.double(), dp.double(), rules)
        within(ds, w, bound, "score gradients")
        within(dslopes, ws, sbound, "slope gradients")


def test_score_special_values(ct):
    inf, nan = math.inf, math.nan
    lowest = torch.finfo(torch.float32).min
    rows = torch.tensor([[1.0, -inf, 2.0, 0.5], [-inf, -inf, -inf, -inf], [nan, 1.0, 2.0, 3.0], [inf, 1.0, 2.0, 3.0],
                         [lowest, lowest, lowest, lowest], [3e38, -3e38, 0.0, 3e38]], device=DEV)
    for keys in (4, 700, 9000):
        s = torch.full((1, 1, 6, keys), nan, device=DEV)
        s[0, 0, :, :4] = rows
        rules = {"key_lengths": ints([4])}
        p = ct.score_softmax(s, ct.ScoreRules(**rules))[0, 0]
        assert float(p[:, 4:].abs().sum()) == 0
        assert float(p[0, 1]) == 0 and abs(float(p[0].sum()) - 1) < 8 * U
        assert float(p[1].abs().sum()) == 0                    # only -inf: nothing to attend to
        assert bool(p[2, :4].isnan().all()) and bool(p[3, :4].isnan().all())
        assert p[4, :4].tolist() == [0.25] * 4
        assert p[5, :4].tolist() == [0.5, 0.0, 0.0, 0.5]
        capped = ct.score_softmax(s, ct.ScoreRules(cap=2.0, **rules))[0, 0]
        assert bool(capped[3, :4].isfinite().all()) and abs(float(capped[3].sum()) - 1) < 8 * U
        assert capped[1, :4].tolist() == [0.25] * 4            # tanh brings -inf to -cap


def test_score_far_positions_keep_their_precision(ct):
    """A distance bias from queries a million positions behind their keys: only differences matter."""
    g = gen(3)
    s = randn(g, 1, 2, 3, 300)
    rules = {"scale": 1.0, "query_start": ints([1_000_000]), "slopes": torch.tensor([0.05, 0.5], device=DEV)}
    p = ct.score_softmax(s, ct.ScoreRules(**rules))
    want = ref.score_softmax(s.double(), rules)
    within(p, want, ref.score_bound(s.double(), want, rules), "probabilities")


def test_score_empty(ct):
    r = ct.ScoreRules(slopes=torch.ones(3, device=DEV))
    for shape in ((0, 3, 2, 4), (2, 3, 0, 4), (2, 3, 2, 0)):
        s = torch.zeros(shape, device=DEV)
        p = ct.score_softmax(s, r)
        ds, dslopes = ct.score_softmax_backward(s, p, r, want_slopes=True)
        assert p.shape == ds.shape == s.shape and dslopes.tolist() == [0.0] * 3


def test_score_gradient_against_differences(ct):
    g = gen(8)
    shape = (2, 2, 7, 19)
    rules = make_rules("docs-causal-slopes-cap", *shape)
    rules["query_docs"] = torch.zeros_like(rules["query_docs"])
    s, dp, way, away = randn(g, *shape), randn(g, *shape), randn(g, *shape).double(), randn(g, 2).double()
    r = ct.ScoreRules(**rules)
    p = ct.score_softmax(s, r)
    ds, dslopes = ct.score_softmax_backward(dp, p, r, scores=s, want_slopes=True)
    step = 1e-5

    def loss(t):
        moved = dict(rules, slopes=rules["slopes"].double() + t * away)
        return float((ref.score_softmax(s.double() + t * way, moved) * dp.double()).sum())
    slope = (loss(step) - loss(-step)) / (2 * step)
    got = float((ds.double() * way).sum() + (dslopes.double() * away).sum())
    # central differences: step^2 times third derivatives of a few hundred terms; gradients: fp32
    assert abs(got - slope) < 1e-5 * (1 + float((ds.double() * way).abs().sum() + (dslopes.double() * away).abs().sum()))


# ---- residual norm ----------------------------------------------------------------------------------------
GATES = ["none", "channel", "batch", "full", "token", "sequence", "one"]


def make_gate(g, kind, B, T, C):
    shape = {"none": None, "channel": (C,), "batch": (B, 1, C), "full": (B, T, C), "token": (B, T, 1), "sequence": (B, 1, 1), "one": (1,)}[kind]
    return None if shape is None else randn(g, *shape)


def check_norm(ct, x, f, pre, post, gate, scale, dy, dh):
    d = lambda t: None if t is None else t.double()
    params = ct.ResidualNorm(pre=pre[0], pre_weight=pre[1], pre_bias=pre[2], post=post[0], post_weight=post[1], post_bias=post[2], scale=scale)
    y, h, stats = ct.residual_norm(x, f, params, gate=gate)
    scale = float(torch.tensor(scale, dtype=torch.float32))
    if f is not None:
        n = ref.normed(f.double(), post[0], d(post[1]), d(post[2]), 1e-5)
        factor = scale if gate is None else scale * gate.double()
        want = x.double() + factor * n
        bound = abs(factor) * ref.norm_bound(f.double(), post[0], d(post[1]), d(post[2]), 1e-5) + U * (4 * (factor * n).abs() + want.abs())
        within(y, want, bound + 1e-37, "y")
    else:
        assert y is x
    if pre[0]:
        # h belongs to the y that was returned
        want = ref.normed(y.double(), pre[0], d(pre[1]), d(pre[2]), 1e-5)
        within(h, want, ref.norm_bound(y.double(), pre[0], d(pre[1]), d(pre[2]), 1e-5) + U * want.abs(), "h")
    else:
        assert h is None
    for v, kind, at in ((f, post[0], 0), (y, pre[0], 2)):
        mean, rstd = (torch.zeros_like(x[..., :1]), torch.ones_like(x[..., :1])) if v is None else ref.row_numbers(v.double(), kind, 1e-5)
        within(stats[..., at], mean[..., 0], U * mean[..., 0].abs() + 1e-12 * (0 if v is None else v.double().abs().mean(-1)), "mean")
        within(stats[..., at + 1], rstd[..., 0], 3 * U * rstd[..., 0], "rstd")
    got = ct.residual_norm_backward(f, y, stats, params, grad_y=dy, grad_h=dh, gate=gate)
    want = ref.residual_norm_gradients(d(f), y.double(), (pre[0], d(pre[1]), d(pre[2])), (post[0], d(post[1]), d(post[2])), d(gate), scale, d(dy), d(dh))
    for name in ("x", "f", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias"):
        t = getattr(got, name)
        given = {"x": x, "f": f, "gate": gate, "post_weight": post[1], "post_bias": post[2], "pre_weight": pre[1], "pre_bias": pre[2]}[name]
        assert (t is None) == (given is None), name
        if t is not None:
            assert t.shape == given.shape, name
            within(t, want[name][0], want[name][1] + 1e-36, "gradient of " + name)
    return y, h, stats, got


def vectors(g, kind, weighted, biased, C):
    return kind, (1 + 0.3 * randn(g, C)) if kind and weighted else None, (0.3 * randn(g, C)) if kind and biased else None


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("kinds", [(1, 0), (2, 0), (0, 1), (0, 2), (1, 1), (2, 2), (1, 2), (0, 0)], ids=str)
@pytest.mark.parametrize("shape", [(2, 5, 64), (3, 7, 300), (2, 3, 1001)], ids=str)
def test_residual_norm_kinds_and_gates(ct, shape, kinds, gate):
    B, T, C = shape
    g = gen(C + 7 * kinds[0] + kinds[1])
    x, f, dy, dh = (randn(g, *shape) + 0.5 for _ in range(4))
    pre, post = vectors(g, kinds[0], True, kinds[0] == 1, C), vectors(g, kinds[1], True, kinds[1] == 1, C)
    check_norm(ct, x, f, pre, post, make_gate(g, gate, B, T, C), 0.7, dy, dh if kinds[0] else None)


@pytest.mark.parametrize("cols", [1, 2, 3, 4, 31, 128, 255, 256, 257, 260, 512, 513, 768, 1024, 1025, 1028, 2048, 2050, 2052, 4096, 4100, 5120,
                                  8192, 8195, 8196, 16384, 16388, 32767, 32768])
@pytest.mark.parametrize("kinds", [(1, 1), (2, 2)], ids=str)
def test_residual_norm_widths(ct, cols, kinds):
    g = gen(cols)
    rows = 5 if cols > 4096 else 23
    x, f, dy, dh = (randn(g, 1, rows, cols) for _ in range(4))
    biased = kinds[0] == 1
    for gate in ("channel", "full"):
        check_norm(ct, x, f, vectors(g, kinds[0], True, biased, cols), vectors(g, kinds[1], True, biased, cols), make_gate(g, gate, 1, rows, cols), 0.5, dy, dh)


@pytest.mark.parametrize("cols", [63, 65, 127, 129, 301, 511, 1023, 1027, 1141, 2047, 3001, 4095, 4097])
@pytest.mark.parametrize("kinds", [(1, 0), (2, 1), (2, 2)], ids=str)
def test_residual_norm_odd_widths(ct, cols, kinds):
    """Rows that go element by element, at the ends of what each share of a thread holds."""
    g = gen(cols)
    rows = 5 if cols > 4096 else 41
    x, f, dy, dh = (randn(g, 1, rows, cols) for _ in range(4))
    for gate, biased in (("none", True), ("channel", False), ("full", True)):
        check_norm(ct, x, f, vectors(g, kinds[0], True, biased, cols), vectors(g, kinds[1], True, biased, cols), make_gate(g, gate, 1, rows, cols), 0.5, dy, dh)


@pytest.mark.parametrize("rows", [1, 2, 147, 300, 2500])
@pytest.mark.parametrize("cols", [48, 768, 1536, 3000])
def test_residual_norm_rows(ct, rows, cols):
    """Teams with one row, several rows, and gate rows that end inside a team's rows."""
    g = gen(rows)
    for B in (1, rows if rows < 10 else 7):
        T = rows // B if rows % B == 0 else rows
        x, f, dy, dh = (randn(g, B, T, cols) for _ in range(4))
        for gate in ("batch", "sequence"):
            check_norm(ct, x, f, vectors(g, 1, True, True, cols), vectors(g, 2, True, False, cols), make_gate(g, gate, B, T, cols), 1.0, dy, dh)


def test_residual_norm_many_gate_rows(ct):
    """A gate row for every three rows: more gate rows than teams, and none of a multiple of them."""
    g = gen(77)
    x, f, dy, dh = (randn(g, 1111, 3, 260) for _ in range(4))
    for gate in ("batch", "sequence"):
        check_norm(ct, x, f, vectors(g, 2, True, False, 260), vectors(g, 2, True, False, 260), make_gate(g, gate, 1111, 3, 260), 0.25, dy, dh)


def test_residual_norm_without_a_block_output(ct):
    g = gen(2)
    for C in (768, 77):
        x, dy, dh = (randn(g, 9, C) for _ in range(3))
        for kind in (1, 2):
            check_norm(ct, x, None, vectors(g, kind, True, True, C), (0, None, None), None, 1.0, dy, dh)
            check_norm(ct, x, None, vectors(g, kind, False, False, C), (0, None, None), None, 1.0, None, dh)


def test_residual_norm_strides(ct):
    """Columns of a wider buffer, gate rows inside a [B, 6 C] projection, rows at odd 4-byte phases."""
    g = gen(4)
    B, T, C = 3, 5, 132
    wide, ada = randn(g, B, T, 3 * C + 1), randn(g, B, 6 * C)
    for at in (0, C, C + 1):
        f = wide[..., at:at + C]
        gate = ada[:, None, 2 * C:3 * C]
        x, dh = randn(g, B, T, C), randn(g, B, T, 2 * C)[..., C:]
        check_norm(ct, x, f, vectors(g, 1, True, True, C), vectors(g, 2, True, True, C), gate, 1.5, randn(g, B, T, C), dh)
    check_norm(ct, x, f, vectors(g, 1, True, True, C), vectors(g, 2, True, True, C), ada[:, None, 1:2], 1.5, None, dh)


def test_residual_norm_large_mean(ct):
    """A mean a thousand times the deviation: the statistics do not cancel."""
    g = gen(6)
    x, f, dy, dh = (randn(g, 4, 1000) + off for off in (1000.0, -500.0, 0.0, 0.0))
    check_norm(ct, x, f, vectors(g, 1, True, True, 1000), vectors(g, 1, True, True, 1000), None, 1.0, dy, dh)


@pytest.mark.parametrize("cols", [200, 1000, 1024, 2040, 4096])
@pytest.mark.parametrize("part", [1.0, 1.0 - 2.0 ** -12])
def test_residual_norm_of_a_stream_that_cancels(ct, cols, part):
    """The block takes back all, or nearly all, of the stream: the next norm magnifies what is left."""
    g = gen(cols)
    f = randn(g, 6, cols)
    x = -part * f / torch.sqrt((f.double() ** 2).mean(-1, keepdim=True) + 1e-5).float()
    check_norm(ct, x, f, (2, None, None), (2, None, None), None, 1.0, randn(g, 6, cols), randn(g, 6, cols))


@pytest.mark.parametrize("cols", [20, 1000, 4100])
@pytest.mark.parametrize("kind", [1, 2])
def test_residual_norm_huge_and_tiny_rows(ct, cols, kind):
    """Rows whose mean square is beyond Float32 on either side are normed like any other."""
    g = gen(cols)
    for size in (1e20, 1e-25):
        x = randn(g, 3, cols) * size
        _, h, _ = ct.residual_norm(x, None, ct.ResidualNorm(pre=kind, pre_eps=0.0))
        want = ref.normed(x.double(), kind, None, None, 0.0)
        within(h, want, ref.norm_bound(x.double(), kind, None, None, 0.0) + U * want.abs(), f"rows of {size}")


def test_residual_norm_empty(ct):
    C = 12
    w = torch.ones(C, device=DEV)
    params = ct.ResidualNorm(pre_weight=w, pre_bias=w, post=ct.NORM_RMS, post_weight=w)
    x = torch.zeros(2, 0, C, device=DEV)
    gate = torch.ones(2, 1, C, device=DEV)
    y, h, stats = ct.residual_norm(x, x.clone(), params, gate=gate)
    assert y.shape == h.shape == x.shape and stats.shape == (2, 0, 4)
    got = ct.residual_norm_backward(x, y, stats, params, grad_y=x, grad_h=x, gate=gate)
    for t in (got.gate, got.post_weight, got.pre_weight, got.pre_bias):
        assert float(t.abs().sum()) == 0


def test_residual_norm_gradient_against_differences(ct):
    g = gen(12)
    B, T, C = 2, 3, 20
    x, f, dy, dh = (randn(g, B, T, C) for _ in range(4))
    pre, post, gate = vectors(g, 1, True, True, C), vectors(g, 2, True, True, C), randn(g, B, 1, C)
    params = ct.ResidualNorm(pre=1, pre_weight=pre[1], pre_bias=pre[2], post=2, post_weight=post[1], post_bias=post[2], scale=0.5)
    y, h, stats = ct.residual_norm(x, f, params, gate=gate)
    got = ct.residual_norm_backward(f, y, stats, params, grad_y=dy, grad_h=dh, gate=gate)
    inputs = {"x": x, "f": f, "gate": gate, "post_weight": post[1], "post_bias": post[2], "pre_weight": pre[1], "pre_bias": pre[2]}
    ways = {k: randn(g, *v.shape).double() for k, v in inputs.items()}
    step = 1e-5

    def loss(t):
        m = {k: v.double() + t * ways[k] for k, v in inputs.items()}
        yy = m["x"] + 0.5 * m["gate"] * ref.normed(m["f"], 2, m["post_weight"], m["post_bias"], 1e-5)
        return float((yy * dy).sum() + (ref.normed(yy, 1, m["pre_weight"], m["pre_bias"], 1e-5) * dh).sum())
    slope = (loss(step) - loss(-step)) / (2 * step)
    terms = {k: getattr(got, k).double() * ways[k] for k in inputs}
    assert abs(sum(float(t.sum()) for t in terms.values()) - slope) < 1e-5 * (1 + sum(float(t.abs().sum()) for t in terms.values()))


# ---- gradient norm and clipping ------------------------------------------------------------------------------
def model(g, sizes, dtype=torch.float32, scale=1.0):
    return [(randn(g, n).to(dtype) * scale) for n in sizes]


def norm_of(tensors, p):
    flat = torch.cat([t.double().reshape(-1) for t in tensors]) if tensors else torch.zeros(1, dtype=torch.float64)
    return float(flat.abs().max()) if p == math.inf else float(flat.abs().sum()) if p == 1 else float(flat.square().sum().sqrt())


SIZES = [[1], [3], [8192], [8193, 1, 8191], [1000003], [5, 0, 70000, 1, 33], [17] * 300, [9] * 2100]


@pytest.mark.parametrize("p", [1, 2, math.inf])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_clip_grad_norm(ct, sizes, p, dtype):
    g = gen(len(sizes))
    grads = model(g, sizes, dtype)
    half = U if dtype == torch.float32 else 2.0 ** -53
    slack = 64 * 2.0 ** -53               # the fp64 sum: chains of a few dozen, then trees
    total = norm_of(grads, p)
    n = ct.grad_norm(grads, p)
    assert n.dtype == dtype and abs(float(n) - total) <= (half + slack) * total
    for limit, out in ((0.5 * total, False), (0.5 * total, True), (2 * total, False), (2 * total, True), (0.0, True), (math.inf, False)):
        have = [t.clone() for t in grads]
        outs = [torch.full_like(t, 7.0) for t in grads] if out else None
        n = ct.clip_grad_norm(have, limit, p, out=outs)
        assert abs(float(n) - total) <= (half + slack) * total
        factor = limit / total if limit < total else 1.0
        for a, b in zip(grads, outs if out else have):
            within(b, a.double() * factor, (2.1 * half + slack) * (a.double() * factor).abs(), "clipped") if factor < 1 else None
            assert factor < 1 or torch.equal(a, b)
        if out:
            assert all(torch.equal(a, b) for a, b in zip(grads, have))


def test_clip_starts_at_every_phase(ct):
    """Tensors at every 4-byte phase of one buffer, outputs at another phase: neighbours keep their values."""
    g = gen(1)
    for n in (1, 7, 30, 8190, 20000):
        for at in range(9):
            flat = randn(g, n + 20)
            keep = flat.clone()
            view = flat[at:at + n]
            total = norm_of([view], 2)
            target = torch.zeros(n + 30, device=DEV)
            got = ct.clip_grad_norm([view], total / 4, out=[target[3 + at // 2:3 + at // 2 + n]])
            assert abs(float(got) - total) <= 2 * U * total
            within(target[3 + at // 2:3 + at // 2 + n], view.double() / 4, 3 * U * view.double().abs() / 4, "out of place")
            assert float(target.abs().sum()) == pytest.approx(float(target[3 + at // 2:3 + at // 2 + n].abs().sum()))
            ct.clip_grad_norm([view], total / 4)
            within(view, keep[at:at + n].double() / 4, 3 * U * keep[at:at + n].double().abs() / 4, "in place")
            assert torch.equal(flat[:at], keep[:at]) and torch.equal(flat[at + n:], keep[at + n:])


@pytest.mark.parametrize("count", [128, 129, 384, 385, 1024, 1025])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_clip_many_ragged_tensors_side_by_side(ct, count, dtype):
    """Views of one buffer, so at every phase, up to a little more than the longest list of a launch and up to
    two stretches of whole vectors; in place and out of place, at the same and at another phase."""
    g = gen(count)
    half = U if dtype == torch.float32 else 2.0 ** -53
    slack = 64 * 2.0 ** -53
    lengths = [(1, 3, 8, 31, 1023, 8191, 8192, 8193, 16384, 16385, 24577, 33001)[(7 * i) % 12 if i % 9 == 0 else i % 5] for i in range(count)]
    flat = torch.randn(sum(lengths), device=DEV, generator=g, dtype=dtype)
    views = lambda buf, lead: list(buf[lead:lead + flat.numel()].split(lengths))
    total = norm_of([flat], 2)
    want = flat.double() / 4
    for lead in (0, 3):
        target = torch.full((flat.numel() + 8,), 5.0, device=DEV, dtype=dtype)
        n = ct.clip_grad_norm(views(flat, 0), total / 4, out=views(target, lead))
        assert abs(float(n) - total) <= (half + slack) * total
        within(target[lead:lead + flat.numel()], want, (2.1 * half + slack) * want.abs(), "out of place")
        assert bool((target[:lead] == 5).all()) and bool((target[lead + flat.numel():] == 5).all())
    keep = flat.clone()
    ct.clip_grad_norm(views(flat, 0), total * 2)
    assert torch.equal(flat, keep)
    ct.clip_grad_norm(views(flat, 0), total / 4)
    within(flat, want, (2.1 * half + slack) * want.abs(), "in place")


def test_clip_mixed_types_permuted_views_and_one_tensor_twice(ct):
    g = gen(9)
    a, b = randn(g, 40, 50).t(), randn(g, 30, 20).double()
    total = norm_of([a, b], 2)
    n = ct.clip_grad_norm(ct.TensorList([a, b]), total / 3)
    assert n.dtype == torch.float64 and abs(float(n) - total) < 1e-13 * total
    assert abs(norm_of([a, b], 2) - total / 3) < 3 * U * total
    twice = ct.grad_norm([a, a])                             # counted as often as it is named
    assert abs(float(twice) - math.sqrt(2) * norm_of([a], 2)) <= 2 * U * float(twice)
    with pytest.raises(ct.CtbError):
        ct.clip_grad_norm([a, a], 1.0)
    outs = [torch.empty(50, 40, device=DEV).t().contiguous().t() for _ in range(2)]
    ct.clip_grad_norm([a, a], math.inf, out=outs)            # the gradient's strides; named twice, written apart
    assert all(torch.equal(o, a) for o in outs)
    with pytest.raises(ct.CtbError):                         # other strides than the gradient's
        ct.clip_grad_norm([a], 1.0, out=[torch.empty(50, 40, device=DEV)])


def test_clip_extremes_and_values_that_are_not_finite(ct):
    for scale in (1e-30, 1e25):                               # squares beyond fp32 on either side
        t = torch.full((1000,), scale, device=DEV)
        want = float(t[0].double()) * math.sqrt(1000)
        assert abs(float(ct.grad_norm([t])) - want) <= 2 * U * want
    for bad in (math.inf, -math.inf, math.nan):
        for p in (1, 2, math.inf):
            t = torch.ones(9000, device=DEV)
            t[8500] = bad
            n = float(ct.clip_grad_norm([t], 0.5, p))
            assert math.isnan(n) if math.isnan(bad) else n == math.inf
            assert float(t[0]) == 1.0 and (math.isnan(float(t[8500])) or float(t[8500]) == bad)
    z = torch.zeros(100, device=DEV)
    assert float(ct.clip_grad_norm([z], 0.0)) == 0.0
    empty = torch.full((1,), 5.0, device=DEV)
    assert float(ct.grad_norm([], norm=empty)) == 0.0
    assert float(ct.grad_norm([torch.zeros(0, device=DEV)])) == 0.0


def test_clip_is_the_same_every_time(ct):
    g = gen(21)
    grads = model(g, [100003, 77, 5000000])
    runs = []
    for _ in range(3):
        out = [torch.empty_like(t) for t in grads]
        n = ct.clip_grad_norm(grads, 1.0, out=out)
        runs.append([n] + out)
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


# ---- streams, graphs, together --------------------------------------------------------------------------------
def step(ct, w, grads):
    """Forward and backward of the steps between the products of one block."""
    p = ct.score_softmax(w["s"], w["rules"])
    y, h, stats = ct.residual_norm(w["x"], w["f"], w["norm"], gate=w["gate"])
    ds, dslopes = ct.score_softmax_backward(w["dp"], p, w["rules"], scores=w["s"], want_slopes=True)
    n = ct.residual_norm_backward(w["f"], y, stats, w["norm"], grad_y=w["dy"], grad_h=w["dh"], gate=w["gate"])
    outs = [dslopes, n.gate, n.post_weight, n.pre_weight, n.pre_bias]
    total = ct.clip_grad_norm(outs, 0.1)
    return [p, y, h, stats, ds, n.x, n.f, total] + outs


def inputs(ct, seed):
    g = gen(seed)
    C = 260
    w = {"s": randn(g, 2, 3, 40, 90), "dp": randn(g, 2, 3, 40, 90), "x": randn(g, 2, 40, C), "f": randn(g, 2, 40, C), "dy": randn(g, 2, 40, C),
         "dh": randn(g, 2, 40, C), "gate": randn(g, 2, 1, C)}
    w["rules"] = ct.ScoreRules(scale=0.5, cap=3.0, causal=True, slopes=torch.rand(3, device=DEV, generator=g), prefix=ints([3, 40]))
    w["norm"] = ct.ResidualNorm(pre_weight=randn(g, C), pre_bias=randn(g, C), post=ct.NORM_RMS, post_weight=randn(g, C), scale=0.5)
    return w


def test_side_stream_graph_and_two_graphs_at_once(ct):
    a, b = inputs(ct, 1), inputs(ct, 2)
    want = {id(w): [t.clone() for t in step(ct, w, None)] for w in (a, b)}
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st, w in zip(streams, (a, b)):
        with torch.cuda.stream(st):
            got = step(ct, w, None)
        st.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want[id(w)]))
    graphs = []
    for w in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(ct, w, None)
        graphs.append((graph, outs))
    for _ in range(3):                                         # both in flight, each with workspaces of its own
        for st, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for w, (_, outs) in zip((a, b), graphs):
        assert all(torch.equal(x, y) for x, y in zip(outs, want[id(w)]))
    a["s"].copy_(b["s"])                                       # a replay sees new contents
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1][0], ct.score_softmax(b["s"], a["rules"]))


def test_clusters_in_a_graph(ct):
    """Rows that take a cluster of CTAs, first met while capturing, on a stream of their own."""
    g = gen(3)
    C = 12300
    x, f, dy, dh, w = randn(g, 2, 70, C), randn(g, 2, 70, C), randn(g, 2, 70, C), randn(g, 2, 70, C), randn(g, C)
    norm = ct.ResidualNorm(pre=ct.NORM_RMS, pre_weight=w, post=ct.NORM_RMS, post_weight=w)
    s, dp = randn(g, 1, 2, 1, 30000), randn(g, 1, 2, 1, 30000)
    rules = ct.ScoreRules(slopes=torch.rand(2, device=DEV, generator=g))

    def run():
        y, h, stats = ct.residual_norm(x, f, norm)
        n = ct.residual_norm_backward(f, y, stats, norm, grad_y=dy, grad_h=dh)
        p = ct.score_softmax(s, rules)
        return [y, h, n.x, n.f, n.pre_weight, n.post_weight, p, *ct.score_softmax_backward(dp, p, rules, want_slopes=True)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in outs]
    assert all(torch.equal(a, b) for a, b in zip(got, run()))


def test_a_training_step_of_a_block(ct):
    """Attention and a feed-forward product between pre and post norms, cross-entropy, every gradient, the
    clipping and an Adam step, against the same network differentiated in 64 bits."""
    g = gen(33)
    B, H, T, D, V = 2, 2, 12, 8, 11
    C = H * D
    shapes = {"wq": (C, C), "wk": (C, C), "wv": (C, C), "wo": (C, C), "wu": (C, C), "head": (C, V)}
    prm = {k: randn(g, *s) * 0.3 for k, s in shapes.items()}
    prm.update({k: 1 + 0.1 * randn(g, C) for k in ("n1", "n2", "n3", "p1", "p2")})
    prm.update({"b1": 0.1 * randn(g, C), "gate": 0.5 + 0.1 * randn(g, C), "slopes": torch.rand(H, device=DEV, generator=g)})
    x = randn(g, B, T, C)
    labels = torch.randint(0, V, (B * T,), device=DEV, generator=g, dtype=torch.int32)
    docs = ints([[0] * 5 + [1] * 7, [0] * 12])
    scale = 1 / math.sqrt(D)
    mm = ct.matmul
    flat = lambda t: t.reshape(B * T, -1)
    heads = lambda t: ct.contiguous(t.view(B, T, H, D).permute(0, 2, 1, 3)).view(B * H, T, D)
    back = lambda t: ct.contiguous(t.view(B, H, T, D).permute(0, 2, 1, 3)).view(B, T, C)
    tr = lambda t: ct.contiguous(t.transpose(-1, -2))

    rules = ct.ScoreRules(scale=scale, cap=3.0, causal=True, query_docs=docs, key_docs=docs, slopes=prm["slopes"])
    entry = ct.ResidualNorm(pre_weight=prm["n1"], pre_bias=prm["b1"])
    middle = ct.ResidualNorm(post=ct.NORM_RMS, post_weight=prm["p1"], pre=ct.NORM_RMS, pre_weight=prm["n2"], scale=0.5)
    final = ct.ResidualNorm(post=ct.NORM_RMS, post_weight=prm["p2"], pre=ct.NORM_RMS, pre_weight=prm["n3"])
    _, h1, st1 = ct.residual_norm(x, None, entry)
    q, k, v = (heads(mm(flat(h1), prm[w])) for w in ("wq", "wk", "wv"))
    s = mm(q, tr(k)).view(B, H, T, T)
    p = ct.score_softmax(s, rules)
    a = back(mm(p.view(B * H, T, T), v))
    f1 = mm(flat(a), prm["wo"]).view(B, T, C)
    y1, h2, st2 = ct.residual_norm(x, f1, middle, gate=prm["gate"])
    u = mm(flat(h2), prm["wu"])
    f2 = ct.unary(ct.RELU, u).view(B, T, C)
    y2, h3, st3 = ct.residual_norm(y1, f2, final)
    lg = mm(flat(h3), prm["head"])
    loss = ct.cross_entropy(lg, labels)

    dlg = ct.cross_entropy_backward(lg, labels, 1.0 / (B * T))
    grads = {"head": mm(tr(flat(h3)), dlg)}
    g3 = ct.residual_norm_backward(f2, y2, st3, final, grad_h=mm(dlg, tr(prm["head"])).view(B, T, C))
    du = ct.binary(ct.MUL, flat(g3.f), ct.unary(ct.GT_S, u, 0.0))
    grads["wu"] = mm(tr(flat(h2)), du)
    g2 = ct.residual_norm_backward(f1, y1, st2, middle, grad_y=g3.x, grad_h=mm(du, tr(prm["wu"])).view(B, T, C), gate=prm["gate"])
    grads["wo"] = mm(tr(flat(a)), flat(g2.f))
    da = heads(mm(flat(g2.f), tr(prm["wo"])).view(B, T, C))
    dv = mm(tr(p.view(B * H, T, T)), da)
    ds, grads["slopes"] = ct.score_softmax_backward(mm(da, tr(v)).view(B, H, T, T), p, rules, scores=s, want_slopes=True)
    ds = ds.view(B * H, T, T)
    dh = torch.zeros_like(h1)
    for name, t in (("wq", mm(ds, k)), ("wk", mm(tr(ds), q)), ("wv", dv)):
        t = flat(back(t))
        grads[name] = mm(tr(flat(h1)), t)
        ct.accumulate_grad(dh, mm(t, tr(prm[name])).view(B, T, C))
    g1 = ct.residual_norm_backward(None, x, st1, entry, grad_y=g2.x, grad_h=dh)
    grads.update(n1=g1.pre_weight, b1=g1.pre_bias, p1=g2.post_weight, n2=g2.pre_weight, gate=g2.gate, p2=g3.post_weight, n3=g3.pre_weight)

    w = {k: t.double().requires_grad_() for k, t in prm.items()}
    xd = x.double().requires_grad_()
    r = {"scale": scale, "cap": 3.0, "causal": True, "query_docs": docs, "key_docs": docs, "slopes": w["slopes"]}
    hd = ref.normed(xd, 1, w["n1"], w["b1"], 1e-5)
    qd, kd, vd = ((hd @ w[n]).view(B, T, H, D).transpose(1, 2) for n in ("wq", "wk", "wv"))
    ad = (ref.score_softmax(qd @ kd.transpose(-1, -2), r) @ vd).transpose(1, 2).reshape(B, T, C)
    yd = xd + 0.5 * w["gate"] * ref.normed(ad @ w["wo"], 2, w["p1"], None, 1e-5)
    yd2 = yd + ref.normed((ref.normed(yd, 2, w["n2"], None, 1e-5) @ w["wu"]).relu(), 2, w["p2"], None, 1e-5)
    ld = torch.nn.functional.cross_entropy((ref.normed(yd2, 2, w["n3"], None, 1e-5) @ w["head"]).reshape(B * T, V), labels.long())
    ld.backward()
    ld = ld.detach()
    assert abs(float(loss) - float(ld)) < 2e-5 * float(ld)      # the loss's own 1e-5, and fp32 products
    for name, t in grads.items():
        want = w[name].grad
        # chains of some 40 fp32 operations with sums of up to 24 terms: 1e-5 of the largest gradient
        assert float((t.double() - want).abs().max()) < 1e-5 * float(want.abs().max()), name
    assert float((g1.x.double() - xd.grad).abs().max()) < 1e-5 * float(xd.grad.abs().max())

    order = sorted(grads)
    total = ct.clip_grad_norm([grads[n] for n in order], 0.05)
    want = math.sqrt(sum(float(w[n].grad.square().sum()) for n in order))
    assert abs(float(total) - want) < 1e-5 * want and want > 0.05
    for n in order:
        clipped = w[n].grad * (0.05 / want)
        assert float((grads[n].double() - clipped).abs().max()) < 2e-5 * float(clipped.abs().max()), n
        before = prm[n].clone()
        m, vv = torch.zeros_like(before), torch.zeros_like(before)
        ct.adam_step(prm[n], grads[n], m, vv, lr=1e-3, step=1)
        assert float((prm[n] - before).abs().max()) <= 1.0001e-3
