"""The language-model operators without a GPU: refusals of the Python entry points and of the C ABI
(all of them before anything is launched), and the rotary tables."""
import ctypes
import math

import numpy as np
import pytest

from ad_b200 import ops
from ad_b200 import runtime as rt

A = ops.DeviceArray


def arr(shape, dtype="float32", strides=None, device=0, ptr=4096):
    return A(ptr, shape, dtype, strides, device)


# ------------------------------------------------------------------ rotary tables

def test_rotary_table_against_complex_powers():
    cos, sin = ops.rotary_table(300, 64)
    assert cos.shape == sin.shape == (300, 32) and cos.dtype == np.float32
    step = np.exp(1j * 10000.0 ** (-np.arange(32) / 32))
    turn = np.stack([step ** p for p in range(300)])
    # a power of 300 factors in 64 bits, rounded once to 32
    assert np.abs(cos - turn.real).max() <= 2.0 ** -24 and np.abs(sin - turn.imag).max() <= 2.0 ** -24


def frequencies(cos, sin):
    return np.arctan2(sin[1].astype(np.float64), cos[1].astype(np.float64))


def test_rotary_table_scalings():
    plain = frequencies(*ops.rotary_table(2, 64))
    linear = frequencies(*ops.rotary_table(2, 64, scaling="linear", factor=4.0))
    np.testing.assert_allclose(linear, plain / 4, rtol=1e-6)
    raised = frequencies(*ops.rotary_table(2, 64, scaling="base", factor=4.0))
    np.testing.assert_allclose(raised[0], plain[0], rtol=1e-6)
    np.testing.assert_allclose(raised[-1], plain[-1] / 4, rtol=1e-6)
    cos, sin = ops.rotary_table(2, 64, scaling="parts", factor=4.0, original=2048)
    gain = 1 + 0.1 * math.log(4.0)
    np.testing.assert_allclose(np.hypot(cos, sin), gain, rtol=1e-6)
    f = frequencies(cos, sin)
    turns = 2048 * plain / (2 * math.pi)
    np.testing.assert_allclose(f[turns >= 32], plain[turns >= 32], rtol=1e-6)
    np.testing.assert_allclose(f[turns <= 1], plain[turns <= 1] / 4, rtol=1e-6)
    between = (turns > 1) & (turns < 32)
    assert between.any() and (f[between] < plain[between]).all() and (f[between] > plain[between] / 4).all()


def test_rotary_table_edges():
    assert ops.rotary_table(0, 8)[0].shape == (0, 4)
    assert ops.rotary_table(5, 0)[0].shape == (5, 0)
    for bad in (dict(positions=4, rotary=3), dict(positions=-1, rotary=4), dict(positions=4, rotary=4, base=0.0),
                dict(positions=4, rotary=4, factor=0.0), dict(positions=4, rotary=4, scaling="odd"),
                dict(positions=4, rotary=4, scaling="parts", factor=2.0)):
        with pytest.raises(ValueError):
            ops.rotary_table(**bad)


# ------------------------------------------------------------------ refusals in Python

def rotary_args(**kw):
    a = dict(q=arr((2, 3, 4, 8)), k=arr((2, 3, 2, 8)), cos=arr((16, 4)), sin=arr((16, 4)),
             positions=arr((2, 3), "int64"), out=(arr((2, 3, 4, 8)), arr((2, 3, 2, 8))))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,error,text", [
    (dict(q=np.zeros((2, 3, 4, 8), np.float32)), TypeError, "device array"),
    (dict(q=3), TypeError, "device array"),
    (dict(q=arr((2, 3, 4, 8), "int64")), TypeError, "float32, bfloat16 or float16"),
    (dict(q=arr((2, 3, 4, 8), device=-1)), ValueError, "not in device memory"),
    (dict(q=arr((2, 3, 4, 8), strides=(192, 64, 16, 2))), ValueError, "adjacent"),
    (dict(q=arr((3, 8))), ValueError, "expected"),
    (dict(k=arr((2, 3, 2, 8), "bfloat16")), TypeError, "k"),
    (dict(k=arr((2, 3, 2, 16))), ValueError, "k: 2 x 3 tokens of 16"),
    (dict(k=arr((2, 3, 2, 8), device=1)), ValueError, "device 1"),
    (dict(cos=arr((16, 5)), sin=arr((16, 5))), ValueError, "10 rotated elements in a head of 8"),
    (dict(sin=arr((15, 4))), ValueError, "cos, sin"),
    (dict(cos=arr((16, 4), "bfloat16"), sin=arr((16, 4), "bfloat16")), TypeError, "cos"),
    (dict(cos=arr((16, 4), strides=(8, 1))), ValueError, "adjacent"),
    (dict(positions=arr((2, 3))), TypeError, "int64 or int32"),
    (dict(positions=arr((3, 2), "int64")), ValueError, "positions"),
    (dict(layout="pairs"), ValueError, "layout"),
    (dict(out=None), ValueError, "have to be given"),
    (dict(out=(arr((2, 3, 4, 8)), None)), ValueError, "one array for q and one for k"),
    (dict(out=(arr((2, 3, 4, 9)), arr((2, 3, 2, 8)))), ValueError, "shape"),
    (dict(out=(arr((2, 3, 4, 8), strides=(0, 32, 8, 1)), arr((2, 3, 2, 8)))), ValueError, "share memory"),
])
def test_rotary_refuses(kw, error, text):
    with pytest.raises(error, match=text):
        ops.rotary(**rotary_args(**kw))


def norm_args(**kw):
    a = dict(x=arr((6, 8)), z=arr((6, 8)), after_weight=arr((8,)), before_weight=arr((8,)),
             out=(arr((6, 8)), arr((6, 8)), arr((6, 4))))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,error,text", [
    (dict(kind="batch"), ValueError, "kind"),
    (dict(x=arr((6, 8), "int32")), TypeError, "x"),
    (dict(x=arr((), "float32")), ValueError, "scalar"),
    (dict(z=arr((6, 9))), ValueError, "z: shape"),
    (dict(z=arr((6, 8), "float16")), TypeError, "z"),
    (dict(x=arr((6, 8), strides=(16, 2))), ValueError, "adjacent"),
    (dict(x=arr((2, 3, 8), strides=(100, 8, 1)), z=arr((2, 3, 8))), ValueError, "evenly spaced"),
    (dict(after_weight=arr((7,))), ValueError, "after_weight: 7 elements"),
    (dict(after_weight=arr((8,), "bfloat16")), TypeError, "weights"),
    (dict(before_weight=arr((8,), strides=(2,))), ValueError, "adjacent"),
    (dict(after_weight=None, after_bias=arr((8,))), ValueError, "bias"),
    (dict(gate=arr((4, 8))), ValueError, "gate: 4 rows"),
    (dict(gate=arr((6, 7))), ValueError, "gate"),
    (dict(gate=arr((0, 8))), ValueError, "gate"),
    (dict(out=None), ValueError, "have to be given"),
    (dict(out=(arr((6, 8)), None, arr((6, 4)))), ValueError, "y goes with"),
    (dict(out=(arr((6, 8), strides=(4, 1)), arr((6, 8)), arr((6, 4)))), ValueError, "overlap"),
    (dict(out=(arr((6, 8)), arr((6, 8)), arr((6, 3)))), ValueError, "stats"),
    (dict(stream=5, out=None), ValueError, "have to be given"),
])
def test_block_norm_refuses(kw, error, text):
    with pytest.raises(error, match=text):
        ops.block_norm(**norm_args(**kw))


@pytest.mark.parametrize("kw,error,text", [
    (dict(dy=None), ValueError, "dy goes with"),
    (dict(dh=arr((6, 9))), ValueError, "dh"),
    (dict(stats=arr((6, 3))), ValueError, "stats"),
    (dict(out=None), ValueError, "have to be given"),
    (dict(workspace=None), ValueError, "have to be given"),
    (dict(out=(arr((6, 8)), arr((6, 8)), arr((6, 8)), arr((8,)), arr((8,)), None, None)), ValueError, "gate"),
    (dict(out=(arr((6, 8)), arr((6, 8)), None, arr((9,)), arr((8,)), None, None)), ValueError, "after_weight"),
])
def test_block_norm_grad_refuses(kw, error, text):
    a = dict(dh=arr((6, 8)), dy=arr((6, 8)), x=arr((6, 8)), z=arr((6, 8)), after_weight=arr((8,)),
             before_weight=arr((8,)), stats=arr((6, 4)), workspace=arr((1 << 20,)),
             out=(arr((6, 8)), arr((6, 8)), None, arr((8,)), arr((8,)), None, None))
    a.update(kw)
    with pytest.raises(error, match=text):
        ops.block_norm_grad(**a)


@pytest.mark.parametrize("kw,error,text", [
    (dict(logits=arr((4, 10), "int64")), TypeError, "logits"),
    (dict(logits=arr((4, 0))), ValueError, "empty vocabulary"),
    (dict(logits=arr((4, 10), strides=(20, 2))), ValueError, "adjacent"),
    (dict(logits=arr((4, 10), strides=(5, 1))), ValueError, "overlap"),
    (dict(tokens=arr((4,))), TypeError, "tokens"),
    (dict(tokens=arr((5,), "int64")), ValueError, "tokens: 5 elements"),
    (dict(tokens=arr((4,), "int64", device=1)), ValueError, "device 1"),
    (dict(scale=0.0), ValueError, "scale"),
    (dict(scale=math.inf), ValueError, "scale"),
    (dict(scale=math.nan), ValueError, "scale"),
    (dict(top=33, logits=arr((4, 100))), ValueError, "top"),
    (dict(top=11), ValueError, "top"),
    (dict(top=-1), ValueError, "top"),
    (dict(), ValueError, "have to be given"),
    (dict(top=2, out=(arr((4,)), arr((4,)), arr((4, 4)), arr((4, 2)), arr((4, 2)))), TypeError, "top_index"),
    (dict(top=2, out=(arr((4,)), arr((4,)), arr((4, 4)), None, None)), ValueError, "missing"),
])
def test_token_logprobs_refuses(kw, error, text):
    a = dict(logits=arr((4, 10)), tokens=arr((4,), "int64"))
    a.update(kw)
    with pytest.raises(error, match=text):
        ops.token_logprobs(**a)


def test_token_logprobs_grad_refuses():
    for kw, error in ((dict(stats=arr((4, 3))), ValueError), (dict(g_logp=arr((4,), "bfloat16")), TypeError),
                      (dict(out=arr((4, 10), "bfloat16")), TypeError), (dict(out=None), ValueError)):
        a = dict(logits=arr((4, 10)), tokens=arr((4,), "int64"), stats=arr((4, 4)), out=arr((4, 10)))
        a.update(kw)
        with pytest.raises(error):
            ops.token_logprobs_grad(**a)


# ------------------------------------------------------------------ refusals of the C ABI

def refused(rc, text):
    assert rc != 0
    assert text in rt.lib().ad_last_error(), rt.lib().ad_last_error()


def test_c_entries_refuse():
    L = rt.lib()
    st = (ctypes.c_int64 * 3)(24, 8, 8)
    p = 4096

    def rotary(dtype=0, q=p, dim=8, rotary=4, layout=0, tokens=3, cos=p):
        return L.ad_rotary(-1, dtype, q, st, p, st, 1, None, None, None, None, 0, 1, tokens, dim, rotary, layout, 0,
                           cos, p, 16, p, 1, 3, 1, None)

    refused(rotary(dtype=7), b"element type")
    refused(rotary(q=None), b"null operand")
    refused(rotary(rotary=3), b"cannot be rotated")
    refused(rotary(rotary=10), b"cannot be rotated")
    refused(rotary(layout=2), b"layout")
    refused(rotary(tokens=-1), b"negative")
    refused(rotary(cos=None), b"null operand")
    assert rotary(tokens=0) == 0  # nothing to do

    def norm(dtype=0, wtype=0, kind=0, x=p, gate=None, per=0, rows=4, width=8, eps=1e-5, h=p, y=p, stats=p, ba=None, wa=p):
        return L.ad_block_norm(-1, dtype, wtype, kind, x, 8, p, 8, gate, 8, per, 0, wa, ba, p, None, 1.0, eps, rows,
                               width, h, 8, y, 8, stats, None)

    refused(norm(dtype=3), b"element type")
    refused(norm(wtype=1), b"weights of type")
    refused(norm(kind=2), b"unknown norm")
    refused(norm(x=None), b"null operand")
    refused(norm(width=0), b"rows of 0")
    refused(norm(width=40000), b"rows of 40000")
    refused(norm(gate=p, per=3), b"share gates")
    refused(norm(eps=-1.0), b"eps")
    refused(norm(y=None), b"null or unaligned")
    refused(norm(stats=p + 4), b"null or unaligned")
    refused(norm(wa=None, ba=p), b"bias without")
    assert norm(rows=0) == 0

    def logp(dtype=0, logits=p, ld=10, rows=4, vocab=10, scale=1.0, top=0, stats=p):
        return L.ad_token_logprobs(-1, dtype, logits, ld, rows, vocab, p, 1, scale, top, p, p, stats, p, p, None)

    refused(logp(dtype=-1), b"element type")
    refused(logp(logits=None), b"null operand")
    refused(logp(logits=p + 2), b"unaligned")
    refused(logp(ld=9), b"overlap")
    refused(logp(vocab=0), b"rows of 0 logits")
    refused(logp(scale=-1.0), b"positive")
    refused(logp(top=11), b"alternatives")
    refused(logp(stats=None), b"null or unaligned")
    assert logp(rows=0) == 0


@pytest.mark.parametrize("kw,error,text", [
    (dict(g=arr((4, 8), "int64")), TypeError, "g"),
    (dict(g=arr((8,))), ValueError, "expected"),
    (dict(steps=33), ValueError, "steps"),
    (dict(coefficients=[(1.0, 2.0, 3.0)] * 4), ValueError, "coefficients"),
    (dict(coefficients=[(1.0, 2.0)] * 5), ValueError, "coefficients"),
    (dict(out=arr((4, 9))), ValueError, "out"),
    (dict(out=arr((4, 8), strides=(0, 1))), ValueError, "share memory"),
    (dict(out=None), ValueError, "have to be given"),
    (dict(workspace=None), ValueError, "have to be given"),
    (dict(workspace=arr((4,))), rt.ADError, "bytes of workspace"),
    (dict(workspace=arr((1 << 20,), ptr=4100)), rt.ADError, "256-byte aligned"),
    (dict(coefficients=(50.0, 0.0, 0.0)), rt.ADError, "past 1024"),
    (dict(coefficients=(math.nan, 0.0, 0.0)), rt.ADError, "not a number"),
    (dict(eps=-1.0), rt.ADError, "eps"),
    (dict(g=arr((4, 70000)), out=arr((4, 70000))), rt.ADError, "at most"),
])
def test_orthogonalize_refuses(kw, error, text):
    a = dict(g=arr((4, 8)), out=arr((4, 8), "bfloat16"), workspace=arr((1 << 20,)))
    a.update(kw)
    with pytest.raises(error, match=text):
        ops.orthogonalize(**a)
