"""Embeddings, feed-forward blocks, log probabilities of a linear layer and gradient clipping without a
GPU: refusals of the Python entry points and of the C ABI (all of them before anything is launched)."""
import ctypes
import math

import numpy as np
import pytest

from ad_b200 import ops
from ad_b200 import runtime as rt

P = 1 << 20


def arr(shape, dtype="bfloat16", strides=None, device=0, ptr=P):
    return ops.DeviceArray(ptr, shape, dtype, strides, device)


def far(k, shape, dtype="bfloat16", strides=None, device=0):
    """An array in a place of its own."""
    return arr(shape, dtype, strides, device, (k + 2) << 24)


# ------------------------------------------------------------------ embeddings

@pytest.mark.parametrize("kw,error,text", [
    (dict(table=np.zeros((4, 8), np.float32)), TypeError, "device array"),
    (dict(table=far(0, (4, 8), "int32")), TypeError, "table"),
    (dict(table=far(0, (8,))), ValueError, "table"),
    (dict(table=far(0, (0, 8))), ValueError, "table"),
    (dict(table=far(0, (4, 8), strides=(16, 2))), ValueError, "adjacent"),
    (dict(tokens=far(1, (3,), "float32")), TypeError, "tokens"),
    (dict(tokens=far(1, (3,), "int64", strides=(2,))), ValueError, "adjacent"),
    (dict(tokens=far(1, (3,), "int64", device=1)), ValueError, "device 1"),
    (dict(scale=math.nan), ValueError, "scale"),
    (dict(scale=math.inf), ValueError, "scale"),
    (dict(out=None), ValueError, "have to be given"),
    (dict(out=far(2, (3, 9))), ValueError, "out: shape"),
    (dict(out=far(2, (3, 8), "float32")), TypeError, "out"),
    (dict(out=far(2, (3, 8), strides=(4, 1))), ValueError, "overlap"),
    (dict(out=far(0, (3, 8))), rt.ADError, "overlap operands or one another"),
])
def test_embed_refuses(kw, error, text):
    a = dict(tokens=far(1, (3,), "int64"), table=far(0, (4, 8)), out=far(2, (3, 8)))
    a.update(kw)
    with pytest.raises(error, match=text):
        ops.embed(**a)


@pytest.mark.parametrize("kw,error,text", [
    (dict(dy=far(0, (3, 8), "int64")), TypeError, "dy"),
    (dict(tokens=far(1, (4,), "int64")), ValueError, "tokens"),
    (dict(tokens=far(1, (3,), "uint8")), TypeError, "tokens"),
    (dict(vocab=0), ValueError, "vocab"),
    (dict(scale=-math.inf), ValueError, "scale"),
    (dict(out=None), ValueError, "have to be given"),
    (dict(workspace=None), ValueError, "have to be given"),
    (dict(out=None, accumulate=True), ValueError, "out has to be given"),
    (dict(out=far(2, (5, 8), "float16")), TypeError, "out"),
    (dict(out=far(2, (6, 8))), ValueError, "out"),
    (dict(out=far(2, (5, 8), strides=(7, 1))), ValueError, "overlap"),
    (dict(out=far(0, (5, 8))), rt.ADError, "overlap operands or one another"),
    (dict(workspace=far(3, (8,))), rt.ADError, "bytes of workspace"),
    (dict(workspace=arr((1 << 20,), ptr=(9 << 24) + 64)), rt.ADError, "256-byte aligned"),
    (dict(workspace=far(2, (1 << 20,))), rt.ADError, "overlap operands or one another"),
])
def test_embed_grad_refuses(kw, error, text):
    a = dict(dy=far(0, (3, 8)), tokens=far(1, (3,), "int64"), vocab=5, out=far(2, (5, 8)), workspace=far(3, (1 << 20,)))
    a.update(kw)
    with pytest.raises(error, match=text):
        ops.embed_grad(**a)


def test_workspace_queries_name_what_is_no_array():
    x, w = far(0, (4, 16)), far(1, (24, 16))
    for call, name in ((lambda: ops.linear_logprobs_workspace(x, 3), "weight"), (lambda: ops.linear_logprobs_workspace(3, w), "x"),
                       (lambda: ops.feed_forward_workspace(x, w, w, 3), "w_down"),
                       (lambda: ops.feed_forward_workspace(x, w, w, far(2, (16, 24)), dy=3), "dy")):
        with pytest.raises(TypeError, match=f"{name}: expected a device array"):
            call()


def test_embed_grad_workspace_grows():
    sizes = [ops.embed_grad_workspace(n, 1000, 64) for n in (0, 1, 100, 2048, 2049, 100000)]
    assert sizes[0] == 0 and sizes == sorted(sizes) and len(set(sizes)) == len(sizes)


# ------------------------------------------------------------------ log probabilities of a linear layer

def linear(**kw):
    a = dict(x=far(0, (4, 16)), weight=far(1, (10, 16)), tokens=far(2, (4,), "int64"),
             out=(far(3, (4,), "float32"), far(4, (4,), "float32"), far(5, (4, 2), "float32")),
             workspace=far(6, (1 << 20,)))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,error,text", [
    (dict(x=far(0, (4, 16), "float32")), TypeError, "x: expected bfloat16 or float16"),
    (dict(x=3), TypeError, "device array"),
    (dict(x=far(0, (4, 16), device=-1)), ValueError, "not in device memory"),
    (dict(x=far(0, (4, 16), strides=(8, 1))), ValueError, "x: rows overlap"),
    (dict(x=far(0, (4, 0)), weight=far(1, (10, 0))), ValueError, "empty"),
    (dict(weight=far(1, (0, 16))), ValueError, "empty"),
    (dict(weight=far(1, (10, 16), "float16")), TypeError, "weight"),
    (dict(weight=far(1, (10, 15))), ValueError, "weight: shape"),
    (dict(weight=far(1, (160,))), ValueError, "weight"),
    (dict(weight=far(1, (10, 16), strides=(1, 10))), ValueError, "adjacent"),
    (dict(tokens=far(2, (5,), "int64")), ValueError, "tokens"),
    (dict(tokens=far(2, (4,))), TypeError, "tokens"),
    (dict(scale=0.0), ValueError, "scale"),
    (dict(scale=math.inf), ValueError, "scale"),
    (dict(out=None), ValueError, "have to be given"),
    (dict(workspace=None), ValueError, "have to be given"),
    (dict(out=(far(3, (4,)), far(4, (4,), "float32"), far(5, (4, 2), "float32"))), TypeError, "out logp"),
    (dict(out=(far(3, (4,), "float32"), far(4, (4,), "float32"), far(5, (4, 3), "float32"))), ValueError, "out stats"),
    (dict(out=(far(3, (4,), "float32"), far(3, (4,), "float32"), far(5, (4, 2), "float32"))), rt.ADError, "overlap operands or one another"),
    (dict(out=(far(0, (4,), "float32"), far(4, (4,), "float32"), far(5, (4, 2), "float32"))), rt.ADError, "overlap operands or one another"),
])
def test_linear_logprobs_refuses(kw, error, text):
    with pytest.raises(error, match=text):
        ops.linear_logprobs(**linear(**kw))


@pytest.mark.parametrize("kw,error,text", [
    (dict(stats=far(5, (4, 4), "float32")), ValueError, "stats"),
    (dict(g_logp=far(7, (4,))), TypeError, "g_logp"),
    (dict(g_lse=far(8, (5,), "float32")), ValueError, "g_lse"),
    (dict(out=None), ValueError, "have to be given"),
    (dict(out=None, accumulate=True), ValueError, "out has to be given"),
    (dict(out=(far(9, (4, 16), "float32"), far(10, (10, 16)))), TypeError, "out x"),
    (dict(out=(far(9, (4, 16)), far(10, (10, 16), "float16"))), TypeError, "out weight"),
    (dict(out=(far(9, (4, 16)), far(10, (10, 17)))), ValueError, "out weight"),
    (dict(out=(far(0, (4, 16)), far(10, (10, 16)))), rt.ADError, "overlap operands or one another"),
    (dict(out=(far(9, (4, 16)), far(1, (10, 16)))), rt.ADError, "overlap operands or one another"),
])
def test_linear_logprobs_grad_refuses(kw, error, text):
    a = linear(stats=far(5, (4, 2), "float32"), g_logp=far(7, (4,), "float32"), g_lse=far(8, (4,), "float32"),
               out=(far(9, (4, 16)), far(10, (10, 16))))
    a.update(kw)
    with pytest.raises(error, match=text):
        ops.linear_logprobs_grad(**a)


# ------------------------------------------------------------------ feed-forward blocks

def ffn(**kw):
    a = dict(x=far(0, (4, 16)), w_gate=far(1, (24, 16)), w_up=far(2, (24, 16)), w_down=far(3, (16, 24)),
             out=(far(4, (4, 16)), None, None), workspace=far(7, (1 << 20,)))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,error,text", [
    (dict(act="tanh"), ValueError, "act"),
    (dict(x=far(0, (4, 16), "float32")), TypeError, "x: expected bfloat16 or float16"),
    (dict(x=far(0, (4, 16), strides=(0, 1))), ValueError, "x: rows overlap"),
    (dict(x=far(0, (4, 0))), ValueError, "empty"),
    (dict(w_gate=far(1, (24, 15))), ValueError, "w_gate: shape"),
    (dict(w_gate=far(1, (24, 16), "float16")), TypeError, "w_gate"),
    (dict(w_up=far(2, (25, 16))), ValueError, "w_up: shape"),
    (dict(w_up=far(2, (24, 16), strides=(1, 24))), ValueError, "adjacent"),
    (dict(w_down=far(3, (24, 16))), ValueError, "w_down: shape"),
    (dict(w_down=far(3, (16, 24), device=1)), ValueError, "device 1"),
    (dict(out=None), ValueError, "have to be given"),
    (dict(workspace=None), ValueError, "have to be given"),
    (dict(keep=True), ValueError, "go with keep"),
    (dict(out=(far(4, (4, 16)), far(5, (4, 24), "float32"), None)), ValueError, "go with keep"),
    (dict(keep=True, out=(far(4, (4, 16)), far(5, (4, 24)), far(6, (4, 24), "float32"))), TypeError, "out gate"),
    (dict(keep=True, out=(far(4, (4, 16)), far(5, (4, 24), "float32"), far(5, (4, 24), "float32"))), rt.ADError, "overlap operands or one another"),
    (dict(out=(far(0, (4, 16)), None, None)), rt.ADError, "overlap operands or one another"),
])
def test_feed_forward_refuses(kw, error, text):
    with pytest.raises(error, match=text):
        ops.feed_forward(**ffn(**kw))


@pytest.mark.parametrize("kw,error,text", [
    (dict(dy=far(8, (4, 15))), ValueError, "dy: shape"),
    (dict(dy=far(8, (4, 16), strides=(0, 1))), ValueError, "dy: rows overlap"),
    (dict(gate=far(5, (4, 24))), TypeError, "gate"),
    (dict(up=far(6, (4, 23), "float32")), ValueError, "up: shape"),
    (dict(out=None, accumulate=True), ValueError, "out has to be given"),
    (dict(out=(far(9, (4, 16)), far(10, (24, 16)), far(11, (24, 16), "float32"), far(12, (16, 24)))), TypeError, "one type"),
    (dict(out=(far(9, (4, 16)), far(10, (24, 16)), far(10, (24, 16)), far(12, (16, 24)))), rt.ADError, "overlap operands or one another"),
    (dict(out=(far(9, (4, 16)), far(10, (24, 16)), far(11, (24, 16)), far(3, (16, 24)))), rt.ADError, "overlap operands or one another"),
])
def test_feed_forward_grad_refuses(kw, error, text):
    a = ffn(dy=far(8, (4, 16)), gate=far(5, (4, 24), "float32"), up=far(6, (4, 24), "float32"),
            out=(far(9, (4, 16)), far(10, (24, 16)), far(11, (24, 16)), far(12, (16, 24))))
    a.update(kw)
    with pytest.raises(error, match=text):
        ops.feed_forward_grad(**a)


def test_columns_of_one_array_are_apart():
    """Results that are columns of one array side by side share no memory, although their ranges do: with
    a device these calls run, without one they get as far as looking for it."""
    def call(gate, up):
        if rt.device_count():
            return ""
        with pytest.raises(rt.ADError) as e:
            ops.feed_forward(**ffn(keep=True, out=(far(4, (4, 16)), gate, up)))
        return str(e.value)

    left = arr((4, 24), "float32", strides=(50, 1), ptr=P << 9)
    assert "overlap" not in call(left, arr((4, 24), "float32", strides=(50, 1), ptr=(P << 9) + 96))
    assert "overlap" not in call(left, arr((4, 24), "float32", strides=(50, 1), ptr=(P << 9) + 104))
    if not rt.device_count():
        assert "overlap" in call(left, arr((4, 24), "float32", strides=(50, 1), ptr=(P << 9) + 108))
        assert "overlap" in call(left, arr((4, 24), "float32", strides=(50, 1), ptr=(P << 9) + 92))
        assert "overlap" in call(left, arr((4, 24), "float32", strides=(49, 1), ptr=(P << 9) + 96))


# ------------------------------------------------------------------ clipping

def clip(**kw):
    a = dict(grads=[far(0, (4, 8)), far(1, (7,), "float32")], max_norm=1.0, norm=far(2, (1,), "float32"),
             workspace=far(3, (1 << 20,)))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,error,text", [
    (dict(grads=[]), ValueError, "no arrays"),
    (dict(grads=[far(0, (4,)), 3]), TypeError, r"grads\[1\]"),
    (dict(grads=[far(0, (4,), "int32")]), TypeError, r"grads\[0\]"),
    (dict(grads=[far(0, (4,), device=-1)]), ValueError, "not in device memory"),
    (dict(grads=[far(0, (4,)), far(1, (4,), device=1)]), ValueError, "device 1"),
    (dict(grads=[far(0, (4, 8), strides=(9, 1))]), ValueError, "adjacent"),
    (dict(grads=[far(0, (4, 8), strides=(0, 1))]), ValueError, "adjacent"),
    (dict(max_norm=-1.0), ValueError, "max_norm"),
    (dict(max_norm=math.nan), ValueError, "max_norm"),
    (dict(norm=None), ValueError, "have to be given"),
    (dict(workspace=None), ValueError, "have to be given"),
    (dict(norm=far(2, (1,))), TypeError, "norm"),
    (dict(norm=far(2, (2,), "float32")), ValueError, "norm"),
    (dict(out=[far(4, (4, 8))]), ValueError, "1 arrays for 2"),
    (dict(out=[far(4, (4, 8)), 5]), TypeError, r"out\[1\]"),
    (dict(out=[far(4, (4, 8)), far(5, (7,))]), ValueError, r"out\[1\]"),
    (dict(out=[far(4, (4, 8), strides=(1, 4)), far(5, (7,), "float32")]), ValueError, r"out\[0\]"),
    (dict(workspace=far(3, (8,))), rt.ADError, "bytes of workspace"),
    # an array that comes twice would be scaled twice
    (dict(grads=[far(0, (4, 8)), far(0, (4, 8))]), rt.ADError, "overlap"),
    (dict(grads=[far(0, (4, 8)), arr((8,), ptr=(2 << 24) + 32)]), rt.ADError, "overlap"),
    (dict(out=[far(4, (4, 8)), far(0, (7,), "float32")]), rt.ADError, "overlap"),
    (dict(norm=far(0, (1,), "float32")), rt.ADError, "overlap"),
    (dict(workspace=far(1, (1 << 20,))), rt.ADError, "overlap"),
])
def test_clip_norm_refuses(kw, error, text):
    with pytest.raises(error, match=text):
        ops.clip_norm(**clip(**kw))


def test_clip_norm_takes_any_order_of_axes():
    for shape, strides in (((4, 8), (8, 1)), ((4, 8), (1, 4)), ((2, 3, 4), (1, 8, 2)), ((5, 1), (1, 77)), ((), ()), ((0, 3), (3, 1))):
        x = arr(shape, strides=strides)
        assert ops._dense_array(x, "x")[1] == math.prod(shape)


# ------------------------------------------------------------------ refusals of the C ABI

def refused(rc, text):
    assert rc != 0
    assert text in rt.lib().ad_last_error(), rt.lib().ad_last_error()


def test_c_entries_refuse():
    L = rt.lib()
    p = P

    def embed(dtype=1, tokens=p, rows=4, table=p, ldt=8, vocab=5, width=8, scale=1.0, y=p, ldy=8):
        return L.ad_embed(-1, dtype, tokens, 1, rows, table, ldt, vocab, width, scale, y, ldy, None)

    refused(embed(dtype=3), b"element type")
    refused(embed(tokens=None), b"null operand")
    refused(embed(tokens=p + 4), b"not aligned")
    refused(embed(y=p + 1), b"not aligned")
    refused(embed(ldy=7), b"overlap")
    refused(embed(vocab=0), b"tokens")
    refused(embed(rows=-1), b"rows")
    refused(embed(scale=math.inf), b"scale")
    refused(embed(rows=(1 << 30) + 1), b"at most")
    assert embed(rows=0) == 0 and embed(width=0) == 0

    def embed_grad(dtype=1, dy=p, rows=4, vocab=5, width=8, out_type=1, out=p, ldo=8, acc=0, ws=p, bytes=1 << 20):
        return L.ad_embed_grad(-1, dtype, dy, 8, p, 1, rows, vocab, width, 1.0, out_type, out, ldo, acc, ws, bytes, None)

    refused(embed_grad(out_type=2), b"type 2")
    refused(embed_grad(out=None), b"null")
    refused(embed_grad(dy=p + 1), b"not aligned")
    refused(embed_grad(ldo=7), b"overlap")
    refused(embed_grad(ws=None), b"bytes of workspace")
    refused(embed_grad(ws=p + 128), b"bytes of workspace")
    refused(embed_grad(bytes=100), b"bytes of workspace")
    assert embed_grad(width=0) == 0 and embed_grad(rows=0, acc=1) == 0
    n = rt.c_size_t()
    refused(L.ad_embed_grad_workspace(4, 0, 8, ctypes.byref(n)), b"tokens")
    refused(L.ad_embed_grad_workspace(4, 5, 8, None), b"null operand")

    def linear(dtype=1, x=p, ldx=16, w=p, ldw=16, rows=4, width=16, vocab=10, tokens=p, scale=1.0, logp=p, stats=p):
        return L.ad_linear_logprobs(-1, dtype, x, ldx, w, ldw, rows, width, vocab, tokens, 1, scale, logp, p, stats, p, 1 << 30, None)

    refused(linear(dtype=0), b"element type")
    refused(linear(x=None), b"null operand")
    refused(linear(x=p + 1), b"not aligned")
    refused(linear(stats=p + 4), b"not aligned")
    refused(linear(tokens=p + 4), b"not aligned")
    refused(linear(ldx=15), b"overlap")
    refused(linear(ldw=15), b"overlap")
    refused(linear(width=0), b"rows of 0")
    refused(linear(vocab=0), b"0 tokens")
    refused(linear(rows=(1 << 24) + 1), b"at most")
    refused(linear(scale=-1.0), b"scale")
    refused(linear(scale=math.nan), b"scale")
    assert linear(rows=0) == 0
    refused(L.ad_linear_logprobs_workspace(-1, 1, p, 16, p, 16, 4, 0, 10, 0, ctypes.byref(n)), b"rows of 0")

    def linear_grad(dw_type=1, dx=p, dw=p, lddw=16, rows=4, acc=0):
        return L.ad_linear_logprobs_grad(-1, 1, p, 16, p, 16, rows, 16, 10, p, 1, 1.0, p, None, None, dx, 16, dw_type, dw, lddw, acc,
                                         p, 1 << 30, None)

    refused(linear_grad(dw_type=2), b"type 2")
    refused(linear_grad(dw=None), b"null")
    refused(linear_grad(dx=None), b"null operand")
    refused(linear_grad(lddw=15), b"overlap")
    assert linear_grad(rows=0, acc=1) == 0

    def ffn(dtype=1, act=0, x=p, ldx=16, wg=p, ldd=24, rows=4, width=16, hidden=24, y=p, gate=None, up=None):
        return L.ad_feed_forward(-1, dtype, act, x, ldx, wg, 16, p, 16, p, ldd, rows, width, hidden, y, 16, gate, 24, up, 24,
                                 p, 1 << 30, None)

    refused(ffn(dtype=0), b"element type")
    refused(ffn(act=4), b"activation")
    refused(ffn(act=-1), b"activation")
    refused(ffn(x=None), b"null operand")
    refused(ffn(y=p + 1), b"not aligned")
    refused(ffn(gate=p), b"kept together")
    refused(ffn(gate=p + 2, up=p), b"not aligned")
    refused(ffn(ldx=15), b"overlap")
    refused(ffn(ldd=23), b"overlap")
    refused(ffn(hidden=0), b"0 hidden")
    refused(ffn(width=(1 << 20) + 1), b"at most")
    assert ffn(rows=0) == 0

    def ffn_grad(dw_type=1, dy=p, gate=p, dx=p, dwg=p, rows=4, acc=0):
        return L.ad_feed_forward_grad(-1, 1, 0, dy, 16, p, 16, p, 16, p, 16, p, 24, gate, 24, p, 24, rows, 16, 24, dx, 16, dw_type,
                                      dwg, 16, p, 16, p, 24, acc, p, 1 << 30, None)

    refused(ffn_grad(dw_type=2), b"type 2")
    refused(ffn_grad(dwg=None), b"null")
    refused(ffn_grad(dy=None), b"null operand")
    refused(ffn_grad(gate=p + 2), b"not aligned")
    assert ffn_grad(rows=0, acc=1) == 0

    def clip(count=1, inp=p, n=4, dtype=1, max_norm=1.0, norm=2 * p, ws=3 * p, bytes=1 << 20):
        one = (ctypes.c_void_p * 1)(inp)
        return L.ad_clip_norm(-1, count, one, one, (ctypes.c_int64 * 1)(n), (ctypes.c_int * 1)(dtype), max_norm, norm, ws, bytes, None)

    refused(clip(count=-1), b"arrays")
    refused(clip(inp=None), b"null operand")
    refused(clip(inp=p + 1), b"not aligned")
    refused(clip(n=-1), b"elements")
    refused(clip(dtype=3), b"element type")
    refused(clip(max_norm=-1.0), b"max_norm")
    refused(clip(max_norm=math.nan), b"max_norm")
    refused(clip(norm=None), b"norm")
    refused(clip(ws=None), b"bytes of workspace")
    refused(clip(bytes=100), b"bytes of workspace")
    refused(clip(norm=p), b"overlap")
