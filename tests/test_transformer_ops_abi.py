"""CPU tests of the transformer-step entry points: what they refuse, with which status and message, and that
well-formed calls fail loudly without a CUDA device and leave their outputs alone."""
import ctypes
import math

import numpy as np
import pytest

import ctensor_b200 as ct

NULL, SHAPE, DTYPE, ARG, CUDA, WORKSPACE, LIMIT = 1, 2, 3, 5, 6, 7, 8


@pytest.fixture(scope="module")
def L():
    return ct.lib()


CODES = {np.dtype(np.float32): ct.F32, np.dtype(np.float64): ct.F64, np.dtype(np.int32): ct.I32, np.dtype(np.int64): ct.I64}


class Arr:
    """A numpy array and its C view."""

    def __init__(self, shape, dtype=np.float32, of=None):
        self.a = np.zeros(shape, dtype) if of is None else of
        self.v = ct.make_view(self.a.ctypes.data, CODES[self.a.dtype], self.a.shape, [s // self.a.itemsize for s in self.a.strides])


def address(x):
    return None if x is None else ctypes.addressof(x.v)


def v(x):
    return None if x is None else x.v


def refused(status, want, text):
    assert status == want, (status, ct.lib().ctb_last_error())
    assert text in ct.lib().ctb_last_error().decode(), ct.lib().ctb_last_error()


def rules(scale=1.0, cap=0.0, causal=0, query_start=None, key_lengths=None, prefix=None, query_docs=None, key_docs=None, slopes=None):
    return ct.CScoreRules(scale, cap, causal, 0, *(address(t) for t in (query_start, key_lengths, prefix, query_docs, key_docs, slopes)))


def params(post=0, pre=1, post_eps=1e-5, pre_eps=1e-5, scale=1.0, post_weight=None, post_bias=None, pre_weight=None, pre_bias=None):
    return ct.CResidualNormParams(post, pre, post_eps, pre_eps, scale, *(address(t) for t in (post_weight, post_bias, pre_weight, pre_bias)))


def grads_of(**kw):
    return ct.CResidualNormGrads(*(address(kw.get(n)) for n, _ in ct.CResidualNormGrads._fields_))


def needs_no_gpu(L):
    if L.ctb_device_count() > 0:
        pytest.skip("a CUDA device is present")


def test_struct_sizes():
    assert ctypes.sizeof(ct.CScoreRules) == 8 + 8 + 4 + 4 + 6 * 8
    assert ctypes.sizeof(ct.CResidualNormParams) == 4 + 4 + 3 * 8 + 4 * 8
    assert ctypes.sizeof(ct.CResidualNormGrads) == 7 * 8


def test_score_softmax_refusals(L):
    s, o = Arr((2, 3, 4, 5)), Arr((2, 3, 4, 5))
    i2, f3 = Arr((2,), np.int32), Arr((3,))
    call = lambda r, s=s, o=o: L.ctb_score_softmax(v(s), ctypes.byref(r) if r else None, v(o), None)
    refused(call(rules(), s=None), NULL, "null input")
    refused(call(None), NULL, "null rules")
    refused(call(rules(), s=Arr((2, 3, 4, 5), np.float64)), DTYPE, "Float32")
    refused(call(rules(), s=Arr((6, 4, 5))), SHAPE, "4D")
    refused(call(rules(), s=Arr(0, of=np.zeros((2, 3, 5, 4), np.float32).transpose(0, 1, 3, 2))), SHAPE, "contiguous")
    refused(call(rules(), o=Arr((2, 3, 4, 6))), SHAPE, "elements")
    refused(call(rules(), o=s), ARG, "overlaps")
    refused(call(rules(scale=math.nan)), ARG, "scale")
    refused(call(rules(scale=1e39)), ARG, "scale")
    refused(call(rules(cap=-1.0)), ARG, "cap")
    refused(call(rules(cap=math.inf)), ARG, "cap")
    refused(call(rules(cap=1e-300)), ARG, "cap")
    refused(call(rules(query_start=Arr((2,), np.int64))), DTYPE, "query_start")
    refused(call(rules(key_lengths=Arr((3,), np.int32))), SHAPE, "key_lengths")
    refused(call(rules(prefix=Arr((2, 1), np.int32))), SHAPE, "prefix")
    refused(call(rules(slopes=Arr((2,)))), SHAPE, "slopes")
    refused(call(rules(slopes=Arr((3,), np.int32))), DTYPE, "slopes")
    refused(call(rules(query_docs=Arr((2, 4), np.int32))), ARG, "together")
    refused(call(rules(query_docs=Arr((2, 4), np.int32), key_docs=Arr((2, 4), np.int32))), SHAPE, "key_docs")
    refused(call(rules(slopes=f3), o=Arr(0, of=np.lib.stride_tricks.as_strided(f3.a, (2, 3, 4, 5), (240, 80, 20, 4)))), ARG, "overlaps")
    needs_no_gpu(L)
    o.a[:] = 7
    assert call(rules(causal=1, query_start=i2, slopes=f3)) == CUDA and np.all(o.a == 7)


def test_score_softmax_backward_refusals(L):
    shape = (2, 3, 4, 5)
    g, p, s, o, sl, gs = Arr(shape), Arr(shape), Arr(shape), Arr(shape), Arr((3,)), Arr((3,))
    ws = np.zeros(8192, np.uint8)

    def call(r, g=g, p=p, s=s, o=o, gs=None, ws=None, nbytes=0):
        return L.ctb_score_softmax_backward(v(g), v(p), v(s), ctypes.byref(r), v(o), v(gs), ws, nbytes, None)
    refused(call(rules(), g=Arr((2, 3, 4, 6))), SHAPE, "shapes differ")
    refused(call(rules(), g=None), NULL, "null gradient")
    refused(call(rules(cap=1.0), s=None), NULL, "scores are needed")
    refused(call(rules(cap=1.0), s=Arr((2, 3, 4, 6))), SHAPE, "shapes differ")
    refused(call(rules(), o=g), ARG, "overlaps")
    refused(call(rules(), gs=gs), ARG, "without slopes")
    refused(call(rules(slopes=sl), gs=Arr((2,))), SHAPE, "elements")
    refused(call(rules(slopes=sl), gs=Arr(0, of=o.a.reshape(-1)[:3])), ARG, "overlap")
    need = L.ctb_score_softmax_workspace_bytes(v(p))
    assert need >= 2 * 3 * 4 * 8
    at = ws.ctypes.data + (-ws.ctypes.data) % 256
    refused(call(rules(slopes=sl), gs=gs, ws=at, nbytes=need - 1), WORKSPACE, "needed")
    refused(call(rules(slopes=sl), gs=gs, ws=at + 8, nbytes=need), WORKSPACE, "aligned")
    needs_no_gpu(L)
    assert call(rules(slopes=sl), gs=gs, ws=at, nbytes=need) == CUDA
    assert call(rules()) == CUDA


def test_residual_norm_refusals(L):
    x, f, y, h, w = Arr((2, 3, 8)), Arr((2, 3, 8)), Arr((2, 3, 8)), Arr((2, 3, 8)), Arr((8,))
    raw = np.zeros(64, np.float32)
    start = (-raw.ctypes.data) % 16 // 4
    stats = Arr(0, of=raw[start:start + 24])

    def call(p, x=x, f=f, gate=None, y=y, h=h, stats=stats):
        return L.ctb_residual_norm(v(x), v(f), v(gate), ctypes.byref(p) if p else None, v(y), v(h), v(stats), None)
    refused(call(params(), x=None), NULL, "null input")
    refused(call(None), NULL, "null parameters")
    refused(call(params(), x=Arr((2, 3, 8), np.float64)), DTYPE, "Float32")
    refused(call(params(), f=Arr((6, 8))), SHAPE, "shapes differ")
    refused(call(params(), x=Arr(0, of=np.zeros((2, 8, 3), np.float32).transpose(0, 2, 1))), SHAPE, "last dim")
    refused(call(params(), x=Arr(0, of=np.zeros((3, 2, 8), np.float32).transpose(1, 0, 2))), SHAPE, "fixed distance")
    refused(call(params(pre=3)), ARG, "unknown norm")
    refused(call(params(pre_eps=-1.0)), ARG, "eps")
    refused(call(params(scale=math.inf)), ARG, "scale")
    refused(call(params(pre_weight=Arr((7,)))), SHAPE, "weights")
    refused(call(params(pre_weight=Arr((8,), np.float64))), DTYPE, "weights")
    refused(call(params(post_weight=w)), ARG, "without its norm")
    refused(call(params(pre=0), h=h), ARG, "pre norm")
    refused(call(params(), h=None), ARG, "pre norm")
    refused(call(params(), y=None), ARG, "block output")
    refused(call(params(), f=None), ARG, "block output")
    refused(call(params(), f=None, y=None, gate=w), ARG, "without a block output")
    refused(call(params(post=1), f=None, y=None), ARG, "without a block output")
    refused(call(params(), gate=Arr((2, 3, 5))), SHAPE, "Shape mismatch")
    refused(call(params(), gate=Arr((1, 3, 8))), SHAPE, "come after")
    refused(call(params(), gate=Arr((2, 1, 8), np.int32)), DTYPE, "gate")
    refused(call(params(), y=x), ARG, "overlaps")
    refused(call(params(), h=y), ARG, "two outputs overlap")
    refused(call(params(), stats=Arr((5, 4))), SHAPE, "elements")
    refused(call(params(), stats=Arr(0, of=raw[start + 1:start + 25])), ARG, "16-byte")
    refused(L.ctb_residual_norm(Arr((1, 32769)).v, None, None, ctypes.byref(params()), None, Arr((1, 32769)).v, None, None), LIMIT, "32768")
    needs_no_gpu(L)
    y.a[:] = 7
    for gate in (None, w, Arr((2, 1, 8)), Arr((2, 3, 1)), Arr((1,)), Arr((2, 3, 8))):
        assert call(params(post=2, post_weight=w), gate=gate) == CUDA
    assert np.all(y.a == 7)


def test_residual_norm_backward_refusals(L):
    shape = (2, 3, 8)
    f, y, dy, dh, w, gate = Arr(shape), Arr(shape), Arr(shape), Arr(shape), Arr((8,)), Arr((2, 1, 8))
    raw = np.zeros(64, np.float32)
    start = (-raw.ctypes.data) % 16 // 4
    stats = Arr(0, of=raw[start:start + 24])
    dx, df, dw, dgate = Arr(shape), Arr(shape), Arr((8,)), Arr((2, 1, 8))

    def call(p, out, f=f, y=y, gate=gate, stats=stats, dy=dy, dh=dh, ws=None, nbytes=0):
        return L.ctb_residual_norm_backward(v(f), v(y), v(gate), v(stats), ctypes.byref(p), v(dy), v(dh), ctypes.byref(out) if out else None, ws, nbytes, None)
    full = grads_of(x=dx, f=df, gate=dgate, pre_weight=dw)
    refused(call(params(), full, y=None), NULL, "null input")
    refused(call(params(), None), NULL, "no output")
    refused(call(params(), grads_of()), NULL, "no output")
    refused(call(params(), full, dh=None), ARG, "goes with a pre norm")
    refused(call(params(pre=0), grads_of(x=dx)), ARG, "goes with a pre norm")
    refused(call(params(pre=0), grads_of(x=dx), dh=None, dy=None), NULL, "null gradient")
    refused(call(params(), full, dy=Arr((2, 3, 9))), SHAPE, "shapes differ")
    refused(call(params(), full, stats=None), NULL, "null view")
    refused(call(params(), grads_of(x=dx, gate=dgate), gate=None), ARG, "did not go in")
    refused(call(params(), grads_of(post_weight=dw)), ARG, "did not go in")
    refused(call(params(), grads_of(f=df), f=None, gate=None), ARG, "did not go in")
    refused(call(params(), grads_of(gate=Arr((2, 3, 8)))), SHAPE, "elements")
    refused(call(params(), grads_of(x=dx, f=dx)), ARG, "two outputs overlap")
    refused(call(params(), grads_of(x=dy)), ARG, "overlaps an input")
    need = L.ctb_residual_norm_workspace_bytes(v(y), v(gate))
    assert need > 0
    ws = np.zeros(need + 512, np.uint8)
    at = ws.ctypes.data + (-ws.ctypes.data) % 256
    refused(call(params(), full, ws=at, nbytes=need - 1), WORKSPACE, "needed") if L.ctb_device_count() else None
    refused(call(params(), full, ws=at + 16, nbytes=need), WORKSPACE, "aligned")
    needs_no_gpu(L)
    assert call(params(), full, ws=at, nbytes=need) == CUDA


def test_clip_refusals(L):
    a, b, n = Arr((4, 3)), Arr((5,)), Arr((1,))

    def lst(*arrs):
        return (ctypes.POINTER(ct.View) * max(1, len(arrs)))(*[ctypes.pointer(x.v) if x else None for x in arrs])

    def clip(arrs, limit=1.0, p=2.0, outs=None, norm=n, ws=None, nbytes=0, count=None):
        return L.ctb_clip_grad_norm(lst(*arrs) if arrs is not None else None, len(arrs or ()) if count is None else count, limit, p,
                                    None if outs is None else lst(*outs), v(norm), ws, nbytes, None)
    refused(clip([a, b], limit=-1.0), ARG, "max_norm")
    refused(clip([a, b], limit=math.nan), ARG, "max_norm")
    for p in (0.0, 3.0, -math.inf, math.nan):
        refused(clip([a, b], p=p), ARG, "p must be")
    refused(clip([a, None]), NULL, "null gradient")
    refused(clip(None, count=2), NULL, "null gradient list")
    refused(clip([a], count=-1), ARG, "negative count")
    refused(clip([Arr((3,), np.int32)]), DTYPE, "Float32 or Double64")
    refused(clip([Arr(0, of=np.zeros((4, 6), np.float32)[:, ::2])]), SHAPE, "dense")
    refused(clip([a], norm=None), NULL, "null view")
    refused(clip([a], norm=Arr((2,))), SHAPE, "one element")
    refused(clip([a], norm=Arr((1,), np.int32)), DTYPE, "norm")
    refused(clip([a, a]), ARG, "overlaps")
    refused(clip([a, b], outs=[Arr((4, 3)), a]), SHAPE, "shape and strides")
    refused(clip([a], outs=[a]), ARG, "overlaps")
    refused(clip([a, b], outs=[Arr((4, 3)), None]), NULL, "null view")
    refused(clip([a], outs=[Arr((4, 3), np.float64)]), DTYPE, "dtype")
    refused(clip([a], norm=Arr(0, of=a.a.reshape(-1)[2:3])), ARG, "overlaps")
    odd = np.zeros(64, np.uint8)
    start = odd.ctypes.data + (-odd.ctypes.data) % 16 + 2
    bad = Arr((4,))
    bad.v = ct.make_view(start, ct.F32, (4,), (1,))
    refused(clip([bad]), ARG, "misaligned")
    need = L.ctb_grad_norm_workspace_bytes(2)
    assert need > 0 and L.ctb_grad_norm_workspace_bytes(0) == 0 and L.ctb_grad_norm_workspace_bytes(5000) > need
    ws = np.zeros(need + 512, np.uint8)
    at = ws.ctypes.data + (-ws.ctypes.data) % 256
    refused(clip([a, b], ws=at, nbytes=8), WORKSPACE, "needed")
    refused(clip([a, b], ws=at + 4, nbytes=need), WORKSPACE, "aligned")
    needs_no_gpu(L)
    a.a[:] = 7
    assert clip([a, b]) == CUDA and clip([a, b], ws=at, nbytes=need) == CUDA and clip([a, a], outs=[Arr((4, 3)), Arr((4, 3))]) == CUDA
    assert L.ctb_grad_norm(lst(a, a), 2, 2.0, n.v, None, 0, None) == CUDA and np.all(a.a == 7)
