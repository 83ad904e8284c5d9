"""Refusals of the language-model operators at the edges of what they take: all of them before anything
is launched, so they need no GPU."""
import ctypes

import pytest

from ad_b200 import ops
from ad_b200 import runtime as rt

from .test_ops_host import arr, norm_args, refused, rotary_args

P = 4096


def entries():
    """(name, call of the C entry with addresses by name, {name: bytes its address has to be a multiple of})
    for bfloat16 operands with float32 weights, and for float32 ones."""
    L = rt.lib()
    st = (ctypes.c_int64 * 3)(24, 8, 8)
    for dtype, size in ((0, 4), (1, 2)):
        for wide in (1, 0):
            yield ("ad_rotary", lambda a, t=dtype, w=wide: L.ad_rotary(
                -1, t, a["q"], st, a["q_out"], st, 1, a["k"], st, a["k_out"], st, 1, 1, 3, 8, 4, 0, 0, a["cos"], a["sin"],
                16, a["positions"], w, 3, 1, None),
                dict(q=size, q_out=size, k=size, k_out=size, cos=4, sin=4, positions=8 if wide else 4))
            yield ("ad_token_logprobs", lambda a, t=dtype, w=wide: L.ad_token_logprobs(
                -1, t, a["logits"], 10, 4, 10, a["tokens"], w, 1.0, 2, a["logp"], a["entropy"], a["stats"], a["top_logp"],
                a["top_index"], None),
                dict(logits=size, tokens=8 if wide else 4, logp=4, entropy=4, stats=16, top_logp=4, top_index=8))
            yield ("ad_token_logprobs_grad", lambda a, t=dtype, w=wide: L.ad_token_logprobs_grad(
                -1, t, a["logits"], 10, 4, 10, a["tokens"], w, 1.0, a["stats"], a["g_logp"], a["g_entropy"], a["grad"], 10,
                None), dict(logits=size, tokens=8 if wide else 4, stats=16, g_logp=4, g_entropy=4, grad=size))
        for wtype, wsize in ((0, 4), (dtype, size)):
            weights = {k: wsize for k in ("wa", "ba", "wb", "bb")}
            yield ("ad_block_norm", lambda a, t=dtype, w=wtype: L.ad_block_norm(
                -1, t, w, 1, a["x"], 8, a["z"], 8, a["gate"], 8, 2, 1, a["wa"], a["ba"], a["wb"], a["bb"], 1.0, 1e-5, 4, 8,
                a["h"], 8, a["y"], 8, a["stats"], None),
                dict(x=size, z=size, gate=size, h=size, y=size, stats=16, **weights))
            yield ("ad_block_norm_grad", lambda a, t=dtype, w=wtype: L.ad_block_norm_grad(
                -1, t, w, 1, a["dh"], 8, a["dy"], 8, a["x"], 8, a["z"], 8, a["gate"], 8, 2, 1, a["wa"], a["ba"], a["wb"],
                a["bb"], 1.0, P, 4, 8, a["dx"], 8, a["dz"], 8, a["dgate"], 8, a["dwa"], a["dba"], a["dwb"],
                a["dbb"], P, 1 << 20, None),
                dict(dh=size, dy=size, x=size, z=size, gate=size, dx=size, dz=size, dgate=size, **weights,
                     **{"d" + k: wsize for k in weights}))
        coef = (ctypes.c_float * 3)(1.5, -0.5, 0.0)
        yield ("ad_orthogonalize", lambda a, t=dtype: L.ad_orthogonalize(
            -1, t, a["g"], 1, 4, 8, 0, 8, 1, 1, coef, 0.0, t, a["out"], 0, 8, 1, P, 1 << 20, None), dict(g=size, out=size))


def test_c_entries_refuse_unaligned_operands():
    """An address that is not a multiple of the element's size would be a fault of the device."""
    for who, call, sizes in entries():
        for name, size in sizes.items():
            for off in (1, size // 2, size - 1):
                refused(call({k: P + (off if k == name else 0) for k in sizes}), b"aligned")
                assert rt.lib().ad_last_error().startswith(who.encode())


def test_device_arrays_refuse_unaligned_addresses():
    for kw in (dict(q=arr((2, 3, 4, 8), ptr=P + 2)), dict(positions=arr((2, 3), "int64", ptr=P + 4)),
               dict(sin=arr((16, 4), ptr=P + 1))):
        with pytest.raises(rt.ADError, match="aligned"):
            ops.rotary(**rotary_args(**kw))
    with pytest.raises(rt.ADError, match="aligned"):
        ops.orthogonalize(arr((4, 8), "bfloat16", ptr=P + 1), out=arr((4, 8), "bfloat16"), workspace=arr((1 << 20,)))


def test_arrays_without_elements_and_single_rows():
    """Strides that nothing follows are not looked at."""
    for shape, strides, want in (((2, 0, 8), (8, 8, 1), (0, 8, 8)), ((0, 3, 8), (24, 8, 1), (0, 8, 8)),
                                 ((3, 0, 2, 8), (16, 16, 8, 1), (0, 8, 8)), ((2, 0, 5, 8), (1, 7, 3, 1), (0, 8, 8)),
                                 ((1, 8), (2 ** 40, 1), (1, 8, 8)), ((1, 1, 8), (3, 2 ** 40, 1), (1, 8, 8)),
                                 ((2, 3, 0), (3, 1, 1), (6, 0, 0))):
        assert ops._rows(arr(shape, strides=strides), "x") == want
    x = arr((2, 0, 8), strides=(8, 8, 1))
    h, y, _ = ops.block_norm(x, x, arr((8,)), arr((8,)), gate=x, out=(x, x, arr((0, 4))))
    assert h is x and y is x
    none = arr((2, 0), strides=(1, 1))
    out = ops.TokenLogprobs(none, none, arr((0, 4)), None, None)
    r = ops.token_logprobs(x, arr((2, 0), "int64", strides=(1, 1)), out=out)
    assert r.logp is none
    assert ops.token_logprobs_grad(x, arr((2, 0), "int64", strides=(1, 1)), arr((0, 4)), out=x) is x


@pytest.mark.parametrize("what", [None, 3, "text", [1.0], object()])
def test_operands_that_are_no_arrays(what):
    """A TypeError that names the operand, wherever one has to be given."""
    def no(name, call, **kw):
        with pytest.raises(TypeError, match=name + ": expected a device array"):
            call(**kw)

    for name in ("q", "cos", "sin", "positions"):
        no(name, ops.rotary, **rotary_args(**{name: what}))
    for name in ("x", "z"):
        no(name, ops.block_norm, **norm_args(**{name: what}))
    no("out h", ops.block_norm, **norm_args(out=(what, arr((6, 8)), arr((6, 4)))))
    no("out stats", ops.block_norm, **norm_args(out=(arr((6, 8)), arr((6, 8)), what)))
    grads = (arr((6, 8)), arr((6, 8)), None, arr((8,)), arr((8,)), None, None)
    args = dict(dh=arr((6, 8)), dy=arr((6, 8)), x=arr((6, 8)), z=arr((6, 8)), after_weight=arr((8,)),
                before_weight=arr((8,)), stats=arr((6, 4)), workspace=arr((1 << 20,)), out=grads)
    for name in ("dh", "x", "z", "stats"):
        no(name, ops.block_norm_grad, **{**args, name: what})
    for name in ("logits", "tokens"):
        no(name, ops.token_logprobs, **{**dict(logits=arr((4, 10)), tokens=arr((4,), "int64")), name: what})
    for name in ("logits", "tokens", "stats"):
        no(name, ops.token_logprobs_grad,
           **{**dict(logits=arr((4, 10)), tokens=arr((4,), "int64"), stats=arr((4, 4)), out=arr((4, 10))), name: what})
    no("g", ops.orthogonalize, g=what)
    if what is not None:
        no("k", ops.rotary, **rotary_args(k=what))
        no("gate", ops.block_norm, **norm_args(gate=what))
        no("before_weight", ops.block_norm, **norm_args(before_weight=what))
        no("dy", ops.block_norm_grad, **{**args, "dy": what})
        no("workspace", ops.orthogonalize, g=arr((4, 8)), out=arr((4, 8)), workspace=what)
