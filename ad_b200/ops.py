"""Operators of language models on the caller's device memory.

* ``rotary`` / ``rotary_table``: rotary positions of queries and keys
* ``block_norm`` / ``block_norm_grad``: the norm after a block, its gate, the scaled residual sum
  and the norm before the next block
* ``token_logprobs`` / ``token_logprobs_grad``: log probabilities of given tokens, entropy and the
  best alternatives of rows of logits
* ``orthogonalize``: Newton-Schulz orthogonalisation of matrix updates

Operands are device arrays: torch CUDA tensors, or ``DeviceArray`` views of memory from
``runtime.Context.malloc`` (this module imports no framework by itself).  Elements are float32,
bfloat16 or float16.  A call checks its arguments (``TypeError``, ``ValueError``), launches and
returns without waiting; errors of the library are ``runtime.ADError``.

Results are new torch tensors unless ``out`` gives arrays to write.  The launch goes to torch's
current stream on the operands' device, or to ``stream`` (a cudaStream_t as an integer, or an object
with a ``cuda_stream`` attribute); on a stream that is not the current one, and with ``DeviceArray``
operands, all results (and the workspace, where there is one) have to be given, because torch's
allocator hands out memory for its current stream.  Sums are held in 32 bits or more and results do
not depend on scheduling.

Results are not recorded for automatic differentiation, also where operands require gradients: a
training step calls the gradients' entry points itself, or from ``torch.autograd.Function``s as
``examples/lm_step.py`` does.  The streams of a ``runtime.Context`` neither wait for the legacy default
stream, on which calls with ``DeviceArray`` operands go by default, nor it for them: such a program
waits with ``Context.sync`` before a call that reads what the context wrote, and for the stream of the
call before the context goes on.
"""
import ctypes
import math
import sys
from typing import NamedTuple, Optional, Sequence

import numpy as np

from . import runtime as rt

F32, BF16, F16 = 0, 1, 2
_FLOATS = {"float32": F32, "bfloat16": BF16, "float16": F16}
_INTS = {"int64": 1, "int32": 0}
_SIZES = (4, 2, 2)
_codes: dict = {}  # dtype object -> (kind, code)


class DeviceArray:
    """A view of device memory: address, shape, element type ("float32", "bfloat16", "float16",
    "int32", "int64"), strides in elements (row-major when left out) and device index."""

    __slots__ = ("ptr", "shape", "dtype", "strides", "device")

    def __init__(self, ptr: int, shape: Sequence[int], dtype: str = "float32",
                 strides: Optional[Sequence[int]] = None, device: int = 0):
        self.ptr = int(ptr)
        self.shape = tuple(int(s) for s in shape)
        if strides is None:
            strides, n = [], 1
            for s in reversed(self.shape):
                strides.append(n)
                n *= s
            strides = strides[::-1]
        self.strides = tuple(int(s) for s in strides)
        if len(self.strides) != len(self.shape):
            raise ValueError(f"{len(self.strides)} strides for {len(self.shape)} axes")
        self.dtype = dtype
        self.device = device

    def data_ptr(self) -> int:
        return self.ptr

    def stride(self):
        return self.strides

    def get_device(self) -> int:
        return self.device


def _code(x, name):
    """("f" or "i", type code) of an array's elements."""
    try:
        return _codes[x.dtype]
    except (KeyError, TypeError):
        pass
    except AttributeError:
        raise TypeError(f"{name}: expected a device array, got {type(x).__name__}") from None
    if not hasattr(x, "data_ptr"):
        raise TypeError(f"{name}: expected a device array, got {type(x).__name__}")
    s = str(x.dtype).replace("torch.", "")
    c = ("f", _FLOATS[s]) if s in _FLOATS else ("i", _INTS[s]) if s in _INTS else ("?", s)
    _codes[x.dtype] = c
    return c


def _float(x, name):
    kind, code = _code(x, name)
    if kind != "f":
        raise TypeError(f"{name}: expected float32, bfloat16 or float16 elements, got {x.dtype}")
    return code


def _integer(x, name):
    kind, code = _code(x, name)
    if kind != "i":
        raise TypeError(f"{name}: expected int64 or int32 elements, got {x.dtype}")
    return code


def _typed(x, code, name):
    if _float(x, name) != code:
        raise TypeError(f"{name}: expected {list(_FLOATS)[code]} elements, got {x.dtype}")


def _on(device, x, name):
    if x.get_device() != device:
        raise ValueError(f"{name}: on device {x.get_device()}, not on device {device}")


def _device(x, name):
    d = x.get_device()
    if d < 0:
        raise ValueError(f"{name}: not in device memory")
    return d


# What the checks of a call found, by the layouts of its operands (shapes, strides, types, devices)
# and its options: a program makes the same calls again and again.
_checked: dict = {}


def _layout(x):
    return None if x is None else (x.shape, x.stride(), x.dtype, x.get_device())


def _remember(key, found):
    if len(_checked) >= 4096:
        _checked.clear()
    _checked[key] = found
    return found


_lib = None


def _entry(name):
    """A function of the library, bound once."""
    global _lib
    if _lib is None:
        _lib = rt.lib()
    return getattr(_lib, name)


_torch = None


def _stream(device, stream, x, allocates):
    """The cudaStream_t to launch on; refuses to allocate for a stream that is not torch's current."""
    global _torch
    if isinstance(x, DeviceArray):
        current = None
    else:
        if _torch is None:
            _torch = sys.modules["torch"]
        current = _torch._C._cuda_getCurrentRawStream(device)
    if stream is None:
        s = current
        if s is None:
            s = 0
    else:
        s = getattr(stream, "cuda_stream", stream)
    if allocates and s != current:
        raise ValueError("results (and workspace) have to be given for a DeviceArray or a stream that is not the "
                         "current one")
    return s


def _empty(shape, like, dtype=None):
    return _torch.empty(shape, dtype=like.dtype if dtype is None else getattr(_torch, dtype), device=like.device)


def _empty_rows(x):
    """A row-major array like x."""
    return _torch.empty_like(x) if x.is_contiguous() else _empty(x.shape, x)


def _rows(x, name):
    """(rows, width, elements from row to row) of an array seen as rows of its last axis."""
    shape, st = x.shape, x.stride()
    n = len(shape)
    if n == 0:
        raise ValueError(f"{name}: a scalar has no rows")
    width = shape[-1]
    if width > 1 and st[-1] != 1:
        raise ValueError(f"{name}: a row's elements have to be adjacent (stride {st[-1]})")
    if n == 2:
        return shape[0], width, st[0] if shape[0] > 1 else width
    if n == 1:
        return 1, width, width
    if 0 in shape:  # no elements: strides say nothing
        return math.prod(shape[:-1]), width, width
    rows, ld = 1, None
    for i in range(n - 2, -1, -1):
        if shape[i] != 1:
            if ld is None:
                ld = st[i]
            elif st[i] != ld * rows:
                raise ValueError(f"{name}: rows are not evenly spaced (strides {tuple(st)})")
            rows *= shape[i]
    return rows, width, width if ld is None else ld


def _apart(ld, rows, width, name):
    if rows > 1 and ld < width:
        raise ValueError(f"{name}: rows overlap (stride {ld}, width {width})")


def _flat(x, n, name):
    """A vector of n adjacent elements (of any shape)."""
    shape, st = x.shape, x.stride()
    size = 1
    for i in range(len(shape) - 1, -1, -1):
        if shape[i] > 1 and size and st[i] != size:
            raise ValueError(f"{name}: elements have to be adjacent")
        size *= shape[i]
    if size != n:
        raise ValueError(f"{name}: {size} elements, expected {n}")


def _same_shape(x, shape, name):
    if tuple(x.shape) != tuple(shape):
        raise ValueError(f"{name}: shape {tuple(x.shape)}, expected {tuple(shape)}")


# ------------------------------------------------------------------ rotary positions

def rotary_table(positions: int, rotary: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 original: int = 0, low: float = 1.0, high: float = 32.0):
    """Cosines and sines, float32 numpy arrays [positions][rotary / 2], for ``rotary`` elements of a
    head, computed in 64 bits.  Pair i turns by base^(-2 i / rotary) a position.  ``scaling`` for
    contexts ``factor`` times as long as those trained on:

    * "linear": every frequency divided by the factor
    * "base": the base raised so that the slowest pair is divided by the factor, the fastest unchanged
    * "parts": pairs that turn at least ``high`` times over the ``original`` length keep their
      frequency, those that turn at most ``low`` times have it divided, others in between; cosines
      and sines are multiplied by 1 + 0.1 ln(factor), which sharpens the attention
    """
    if positions < 0 or rotary < 0 or rotary % 2:
        raise ValueError(f"rotary_table: {positions} positions, {rotary} elements (an even number)")
    if not factor > 0 or not base > 0:
        raise ValueError(f"rotary_table: factor {factor}, base {base}: positive numbers are wanted")
    half = rotary // 2
    i = np.arange(half, dtype=np.float64)
    gain = 1.0
    if scaling == "base" and rotary > 2:
        base = base * factor ** (rotary / (rotary - 2))
    elif scaling not in ("none", "linear", "base", "parts"):
        raise ValueError(f"rotary_table: unknown scaling {scaling!r}")
    freq = base ** (-2.0 * i / max(rotary, 1))
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "parts":
        if original <= 0 or not 0 <= low < high:
            raise ValueError(f"rotary_table: original length {original}, turns {low} to {high}")
        turns = original * freq / (2 * math.pi)
        keep = np.clip((turns - low) / (high - low), 0.0, 1.0)
        freq = freq * keep + freq / factor * (1.0 - keep)
        gain = 1.0 + 0.1 * math.log(factor) if factor > 1 else 1.0
    angle = np.arange(positions, dtype=np.float64)[:, None] * freq[None, :]
    return (gain * np.cos(angle)).astype(np.float32), (gain * np.sin(angle)).astype(np.float32)


_LAYOUTS = {"half": 0, "interleaved": 1}
_Strides = ctypes.c_int64 * 3


def _heads(x, name, sequences=None, tokens=None, dim=None):
    """(sequences, tokens, heads, dim, strides of the first three) of [B, T, H, D] or [T, H, D]."""
    shape, st = x.shape, x.stride()
    if len(shape) == 3:
        shape, st = (1, *shape), (0, *st)
    elif len(shape) != 4:
        raise ValueError(f"{name}: expected [sequences, tokens, heads, dim] or [tokens, heads, dim], got {tuple(shape)}")
    b, t, h, d = shape
    if d > 1 and st[3] != 1:
        raise ValueError(f"{name}: a head's elements have to be adjacent (stride {st[3]})")
    if tokens is not None and (b, t, d) != (sequences, tokens, dim):
        raise ValueError(f"{name}: {b} x {t} tokens of {d} elements, expected {sequences} x {tokens} of {dim}")
    return b, t, h, d, _Strides(st[0], st[1], st[2])


def _rotary_operands(q, k, cos, sin, positions, layout):
    if layout not in _LAYOUTS:
        raise ValueError(f"layout: {layout!r} is not one of {list(_LAYOUTS)}")
    dt = _float(q, "q")
    dev = _device(q, "q")
    b, t, hq, d, sq = _heads(q, "q")
    _typed(cos, F32, "cos")
    _typed(sin, F32, "sin")
    half = cos.shape[1] if len(cos.shape) == 2 else -1
    if half < 0 or tuple(cos.shape) != tuple(sin.shape):
        raise ValueError(f"cos, sin: shapes {tuple(cos.shape)} and {tuple(sin.shape)}, expected [rows, rotary / 2] twice")
    if 2 * half > d:
        raise ValueError(f"cos: {2 * half} rotated elements in a head of {d}")
    p64 = _integer(positions, "positions")
    ps, pst = positions.shape, positions.stride()
    if len(ps) == 2 and (ps[0] == b or ps[0] == 1) and ps[1] == t:
        p_seq, p_tok = (pst[0] if ps[0] == b else 0), pst[1]
    elif len(ps) == 1 and ps[0] == t:
        p_seq, p_tok = 0, pst[0]
    else:
        raise ValueError(f"positions: shape {tuple(ps)}, expected {(b, t)} or {(t,)}")
    for x, name in ((cos, "cos"), (sin, "sin")):
        _flat(x, cos.shape[0] * half, name)
        _on(dev, x, name)
    _on(dev, positions, "positions")
    hk, sk = 0, None
    if k is not None:
        _typed(k, dt, "k")
        _on(dev, k, "k")
        _, _, hk, _, sk = _heads(k, "k", b, t, d)
    return dev, dt, b, t, hq, hk, d, sq, sk, half, p64, p_seq, p_tok


def rotary(q, k, cos, sin, positions, *, layout: str = "half", inverse: bool = False, out=None, stream=None):
    """Rotary positions of queries ``q`` and keys ``k`` ([sequences, tokens, heads, dim] or [tokens,
    heads, dim], any strides with a head's elements adjacent; ``k`` may be None).  ``cos`` and ``sin``:
    float32 tables [table rows, rotary / 2] (``rotary_table``; rows may be none); the first ``rotary`` elements of each
    head turn, the others are copied.  ``positions``: int64 or int32, [sequences, tokens] or [tokens]
    for all sequences; outside the table they make NaNs.  ``inverse`` turns back, which is also the
    gradient.  ``out``: (q, k) to write, which may be the operands themselves.  Returns (q, k)."""
    try:
        key = (layout, _layout(q), _layout(k), _layout(cos), _layout(sin), _layout(positions))
        found = _checked.get(key)
    except (AttributeError, TypeError):  # not all of them device arrays: refused below
        key = found = None
    if found is None:
        found = _remember(key, _rotary_operands(q, k, cos, sin, positions, layout))
    dev, dt, b, t, hq, hk, d, sq, sk, half, p64, p_seq, p_tok = found
    s = _stream(dev, stream, q, out is None)
    if out is None:
        yq = _torch.empty_like(q)
        yk = _torch.empty_like(k) if k is not None else None
    else:
        yq, yk = out if isinstance(out, (tuple, list)) else (out, None)
        if yq is None or (yk is None) != (k is None):
            raise ValueError("out: expected one array for q and one for k")
    for y, x, name in ((yq, q, "out for q"), (yk, k, "out for k")):
        if y is not None and out is not None:
            _typed(y, dt, name)
            _same_shape(y, x.shape, name)
            _on(dev, y, name)
            if any(n > 1 and not m for n, m in zip(y.shape, y.stride())):
                raise ValueError(f"{name}: elements share memory (strides {tuple(y.stride())})")
    oq = sq if yq.stride() == q.stride() else _heads(yq, "out for q")[4]
    ok = None if yk is None else sk if yk.stride() == k.stride() else _heads(yk, "out for k")[4]
    rt.check(_entry("ad_rotary")(
        dev, dt, q.data_ptr(), sq, yq.data_ptr(), oq, hq, k.data_ptr() if k is not None else None, sk,
        yk.data_ptr() if yk is not None else None, ok, hk, b, t, d, 2 * half, _LAYOUTS[layout], inverse,
        cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(), p64, p_seq, p_tok, s))
    return yq, yk


# ------------------------------------------------------------------ norms around a block

_KINDS = {"rms": 0, "layer": 1}


def _norm_operands(x, z, after, before, gate, after_bias, before_bias, kind):
    try:
        key = (kind, _layout(x), _layout(z), _layout(after), _layout(before), _layout(gate), _layout(after_bias),
               _layout(before_bias))
        found = _checked.get(key)
    except (AttributeError, TypeError):  # not all of them device arrays: refused below
        key = found = None
    return found or _remember(key, _check_norm_operands(x, z, after, before, gate, after_bias, before_bias, kind))


def _check_norm_operands(x, z, after, before, gate, after_bias, before_bias, kind):
    """Checks what both directions take: (device, dtype, wtype, rows, width, ldx, ldz, ldg, rows a gate)."""
    if kind not in _KINDS:
        raise ValueError(f"kind: {kind!r} is not one of {list(_KINDS)}")
    dt = _float(x, "x")
    dev = _device(x, "x")
    rows, width, ldx = _rows(x, "x")
    _typed(z, dt, "z")
    _same_shape(z, x.shape, "z")
    _on(dev, z, "z")
    ldz = _rows(z, "z")[2]
    wt = None
    for v, name in ((after, "after_weight"), (before, "before_weight"), (after_bias, "after_bias"),
                    (before_bias, "before_bias")):
        if v is not None:
            c = _float(v, name)
            if wt is None:
                wt = c
            if c != wt or (c != F32 and c != dt):
                raise TypeError(f"{name}: weights and biases are all float32 or all of the elements' type")
            _flat(v, width, name)
            _on(dev, v, name)
    if (after_bias is not None and after is None) or (before_bias is not None and before is None):
        raise ValueError("a bias needs the weight of its norm")
    ldg = per = 0
    if gate is not None:
        _typed(gate, dt, "gate")
        _on(dev, gate, "gate")
        groups, gwidth, ldg = _rows(gate, "gate")
        if gwidth != width or groups < 1 and rows or groups and rows % groups:
            raise ValueError(f"gate: {groups} rows of {gwidth} elements for {rows} rows of {width}")
        per = rows // groups if groups else 0
    return dev, dt, F32 if wt is None else wt, rows, width, ldx, ldz, ldg, per


def _ptr(x):
    return None if x is None else x.data_ptr()


def block_norm(x, z, after_weight, before_weight, *, gate=None, after_bias=None, before_bias=None, kind: str = "rms",
               gate_sigmoid: bool = False, residual_scale: float = 1.0, eps: float = 1e-5, out=None, stream=None):
    """The glue between two blocks in one pass over memory, for the residual stream ``x`` and a block's
    output ``z`` ([..., width], up to 32768 wide)::

        u = norm(z) * after_weight + after_bias        (z itself when after_weight is None)
        h = residual_scale * x + act(gate) * u         (without the factor when gate is None)
        y = norm(h) * before_weight + before_bias      (None when before_weight is None)

    ``kind``: "rms" or "layer".  ``gate``: [..., width] for every value, [groups, width] with equal
    numbers of consecutive rows sharing a gate row, or [width] for all; act is the sigmoid when
    ``gate_sigmoid``.  Weights and biases are float32 or of the elements' type.  Returns (h, y,
    stats); ``stats`` (float32 [rows, 4]) is for ``block_norm_grad``.  ``out``: the three to write."""
    dev, dt, wt, rows, width, ldx, ldz, ldg, per = _norm_operands(
        x, z, after_weight, before_weight, gate, after_bias, before_bias, kind)
    s = _stream(dev, stream, x, out is None)
    if out is None:
        h = _empty_rows(x)
        y = None if before_weight is None else _empty_rows(x)
        stats = x.new_empty((rows, 4), dtype=_torch.float32)
        ldh = ldy = width
    else:
        h, y, stats = out
        if (y is None) != (before_weight is None):
            raise ValueError("out: y goes with before_weight")
        ldh = ldy = 0
        _typed(h, dt, "out h")
        for v, name in ((h, "out h"), (y, "out y")):
            if v is not None:
                _typed(v, dt, name)
                _same_shape(v, x.shape, name)
                _on(dev, v, name)
        ldh = _rows(h, "out h")[2]
        _apart(ldh, rows, width, "out h")
        if y is not None:
            ldy = _rows(y, "out y")[2]
            _apart(ldy, rows, width, "out y")
        _typed(stats, F32, "out stats")
        _flat(stats, rows * 4, "out stats")
        _on(dev, stats, "out stats")
    rt.check(_entry("ad_block_norm")(
        dev, dt, wt, _KINDS[kind], x.data_ptr(), ldx, z.data_ptr(), ldz, _ptr(gate), ldg, per, gate_sigmoid,
        _ptr(after_weight), _ptr(after_bias), _ptr(before_weight), _ptr(before_bias), residual_scale, eps, rows, width,
        h.data_ptr(), ldh, _ptr(y), ldy, stats.data_ptr(), s))
    return h, y, stats


class BlockNormGrads(NamedTuple):
    """Gradients of ``block_norm``'s operands; None where there was no operand."""
    x: object
    z: object
    gate: object
    after_weight: object
    before_weight: object
    after_bias: object
    before_bias: object


def block_norm_grad_workspace(rows: int, width: int, gate_rows: int = 0, device: int = -1) -> int:
    """Bytes of workspace that ``block_norm_grad`` needs for a gate of ``gate_rows`` rows (0: none)."""
    n = rt.c_size_t()
    rt.check(rt.lib().ad_block_norm_grad_workspace(device, rows, width, rows // gate_rows if gate_rows else 0,
                                                   ctypes.byref(n)), "ad_block_norm_grad_workspace")
    return n.value


def block_norm_grad(dh, dy, x, z, after_weight, before_weight, stats, *, gate=None, after_bias=None, before_bias=None,
                    kind: str = "rms", gate_sigmoid: bool = False, residual_scale: float = 1.0, eps: float = 1e-5,
                    out=None, workspace=None, stream=None):
    """The gradients of ``block_norm``'s operands from those of its results (``dy`` is None without a
    ``before_weight``), its operands and its ``stats``: a ``BlockNormGrads``, gradients of weights and
    biases in their type (``eps`` went into ``stats``), zeros where there are no rows.  ``out``: a
    ``BlockNormGrads`` to write; ``workspace``: adjacent elements of any type,
    ``block_norm_grad_workspace`` bytes or more."""
    dev, dt, wt, rows, width, ldx, ldz, ldg, per = _norm_operands(
        x, z, after_weight, before_weight, gate, after_bias, before_bias, kind)
    if (dy is None) != (before_weight is None):
        raise ValueError("dy goes with before_weight")
    lds = []
    for v, name in ((dh, "dh"), (dy, "dy")):
        if v is None and name == "dy":
            lds.append(0)
            continue
        _typed(v, dt, name)
        _same_shape(v, x.shape, name)
        _on(dev, v, name)
        lds.append(_rows(v, name)[2])
    _typed(stats, F32, "stats")
    _flat(stats, rows * 4, "stats")
    _on(dev, stats, "stats")
    s = _stream(dev, stream, x, out is None or workspace is None)
    weights = (after_weight, before_weight, after_bias, before_bias)
    if out is None:
        g = BlockNormGrads(_empty_rows(x), _empty_rows(x), None if gate is None else _empty_rows(gate),
                           *(None if v is None else _empty_rows(v) for v in weights))
        lddx = lddz = lddg = width
    else:
        g = BlockNormGrads(*out)
        lddx = lddz = lddg = 0
        for v, like, name in zip(g, (x, z, gate, *weights), BlockNormGrads._fields):
            if (v is None) != (like is None):
                raise ValueError(f"out {name}: goes with its operand")
            if v is not None:
                _typed(v, _float(like, name), "out " + name)
                _same_shape(v, like.shape, "out " + name)
                _on(dev, v, "out " + name)
        lddx, lddz = _rows(g.x, "out x")[2], _rows(g.z, "out z")[2]
        _apart(lddx, rows, width, "out x")
        _apart(lddz, rows, width, "out z")
        if gate is not None:
            gr, _, lddg = _rows(g.gate, "out gate")
            _apart(lddg, gr, width, "out gate")
        for v, name in zip(g[3:], BlockNormGrads._fields[3:]):
            if v is not None:
                _flat(v, width, "out " + name)
    need = block_norm_grad_workspace(rows, width, rows // per if per else 0, dev)
    if workspace is None:
        workspace = _empty((need,), x, "uint8")
        have = need
    else:
        have = _nbytes(workspace, "workspace")
        _on(dev, workspace, "workspace")
    rt.check(_entry("ad_block_norm_grad")(
        dev, dt, wt, _KINDS[kind], dh.data_ptr(), lds[0], _ptr(dy), lds[1], x.data_ptr(), ldx, z.data_ptr(), ldz,
        _ptr(gate), ldg, per, gate_sigmoid, _ptr(after_weight), _ptr(after_bias), _ptr(before_weight),
        _ptr(before_bias), residual_scale, stats.data_ptr(), rows, width, g.x.data_ptr(), lddx, g.z.data_ptr(), lddz,
        _ptr(g.gate), lddg, _ptr(g.after_weight), _ptr(g.after_bias), _ptr(g.before_weight), _ptr(g.before_bias),
        workspace.data_ptr(), have, s))
    if rows == 0 and gate is not None:  # a sum over no rows for each row of the gate
        groups, _, lddg = _rows(g.gate, "out gate")
        rt.check(_entry("ad_clear_rows")(dev, g.gate.data_ptr(), lddg * _SIZES[dt], width * _SIZES[dt], groups, s))
    return g


def _nbytes(x, name):
    """Bytes of an array of adjacent elements of any type."""
    _code(x, name)
    n = 1
    for s in x.shape:
        n *= s
    _flat(x, n, name)
    if isinstance(x, DeviceArray):
        sizes = {"uint8": 1, "int8": 1, "bfloat16": 2, "float16": 2, "float32": 4, "int32": 4, "int64": 8}
        if x.dtype not in sizes:
            raise TypeError(f"{name}: unknown element type {x.dtype}")
        return n * sizes[x.dtype]
    return n * x.element_size()


# ------------------------------------------------------------------ token log probabilities

class TokenLogprobs(NamedTuple):
    """Results of ``token_logprobs``: float32 [rows] twice, float32 [rows, 4] for the gradient (its
    last column: the log of the sum of exp(scale * logits)), float32 and int64 [rows, top] or None."""
    logp: object
    entropy: object
    stats: object
    top_logp: object
    top_index: object


def _logit_operands(logits, tokens, scale):
    if not 0 < scale < math.inf:
        raise ValueError(f"scale: {scale} is not a positive number")
    try:
        key = (_layout(logits), _layout(tokens))
        found = _checked.get(key)
    except (AttributeError, TypeError):  # not both of them device arrays: refused below
        key = found = None
    return found or _remember(key, _check_logit_operands(logits, tokens))


def _check_logit_operands(logits, tokens):
    dt = _float(logits, "logits")
    dev = _device(logits, "logits")
    rows, vocab, ld = _rows(logits, "logits")
    _apart(ld, rows, vocab, "logits")
    t64 = _integer(tokens, "tokens")
    _flat(tokens, rows, "tokens")
    _on(dev, tokens, "tokens")
    if vocab < 1:
        raise ValueError("logits: an empty vocabulary")
    return dev, dt, rows, vocab, ld, t64


def token_logprobs(logits, tokens, *, top: int = 0, scale: float = 1.0, out=None, stream=None) -> TokenLogprobs:
    """For each row of ``scale * logits`` ([..., vocab]; ``scale`` is the reciprocal temperature): the
    log probability of its entry of ``tokens`` (int64 or int32; 0 for a negative one, NaN for one past
    the vocabulary), the entropy of the row's distribution, and the ``top`` (at most 32) most likely
    tokens with their log probabilities, the lower index first among equal logits.  Logits of -inf are
    masked; a row with nothing else has log probabilities of -inf, entropy 0 and no gradient.  Any other
    mask has a probability of 0 beside larger logits, and a finite log probability while 32 bits hold it.
    ``out``: a ``TokenLogprobs`` to write."""
    dev, dt, rows, vocab, ld, t64 = _logit_operands(logits, tokens, scale)
    if not 0 <= top <= min(32, vocab):
        raise ValueError(f"top: {top} alternatives of {vocab} (at most 32)")
    s = _stream(dev, stream, logits, out is None)
    if out is None:
        shape, new, f32 = logits.shape[:-1], logits.new_empty, _torch.float32
        stats = new((rows, 4), dtype=f32)
        r = TokenLogprobs(new(shape, dtype=f32), new(shape, dtype=f32), stats,
                          new((*shape, top), dtype=f32) if top else None,
                          new((*shape, top), dtype=_torch.int64) if top else None)
    else:
        r = TokenLogprobs(*out)
        for v, n, name in ((r.logp, 1, "logp"), (r.entropy, 1, "entropy"), (r.stats, 4, "stats"),
                           (r.top_logp, top, "top_logp"), (r.top_index, top, "top_index")):
            if n:
                if v is None:
                    raise ValueError(f"out: {name} is missing")
                if name == "top_index":
                    if _integer(v, "out " + name) != 1:
                        raise TypeError(f"out {name}: expected int64 elements, got {v.dtype}")
                else:
                    _typed(v, F32, "out " + name)
                _flat(v, rows * n, "out " + name)
                _on(dev, v, "out " + name)
    rt.check(_entry("ad_token_logprobs")(
        dev, dt, logits.data_ptr(), ld, rows, vocab, tokens.data_ptr(), t64, scale, top, r.logp.data_ptr(),
        r.entropy.data_ptr(), r.stats.data_ptr(), _ptr(r.top_logp) if top else None,
        _ptr(r.top_index) if top else None, s))
    return r


def token_logprobs_grad(logits, tokens, stats, g_logp=None, g_entropy=None, *, scale: float = 1.0, out=None,
                        stream=None):
    """The gradient of ``logits`` (in their type) from those of ``token_logprobs``'s ``logp`` and
    ``entropy`` (float32, one a row; None: zeros), its operands and its ``stats``.  ``out``: the array
    to write, which may be ``logits`` itself."""
    dev, dt, rows, vocab, ld, t64 = _logit_operands(logits, tokens, scale)
    for v, n, name in ((stats, 4, "stats"), (g_logp, 1, "g_logp"), (g_entropy, 1, "g_entropy")):
        if v is not None or n == 4:
            _typed(v, F32, name)
            _flat(v, rows * n, name)
            _on(dev, v, name)
    s = _stream(dev, stream, logits, out is None)
    if out is None:
        out = _empty_rows(logits)
        ldo = vocab
    else:
        _typed(out, dt, "out")
        _same_shape(out, logits.shape, "out")
        _on(dev, out, "out")
        ldo = _rows(out, "out")[2]
        _apart(ldo, rows, vocab, "out")
    rt.check(_entry("ad_token_logprobs_grad")(
        dev, dt, logits.data_ptr(), ld, rows, vocab, tokens.data_ptr(), t64, scale, stats.data_ptr(), _ptr(g_logp),
        _ptr(g_entropy), out.data_ptr(), ldo, s))
    return out


# ------------------------------------------------------------------ orthogonalised updates

NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)  # a quintic that brings singular values near 1 in a few steps


def orthogonalize_workspace(count: int, rows: int, cols: int) -> int:
    """Bytes of workspace that ``orthogonalize`` needs."""
    n = rt.c_size_t()
    rt.check(rt.lib().ad_orthogonalize_workspace(count, rows, cols, ctypes.byref(n)), "ad_orthogonalize_workspace")
    return n.value


def orthogonalize(g, *, steps: int = 5, coefficients=NEWTON_SCHULZ, eps: float = 1e-7, out=None, workspace=None,
                  stream=None):
    """Newton-Schulz orthogonalisation of an update: of each matrix of ``g`` ([rows, cols] or [count,
    rows, cols], any strides), X = G / (|G| + eps), then ``steps`` times X = a X + (b A + c A A) X with
    A = X X^T (taken from the side with fewer rows).  ``coefficients``: (a, b, c), or one such triple a
    step.  Products have operands of 11 bits and sums of 32, so the result is within about 1e-3
    (norm-wise) of the exact iteration, in float32 too; it is bfloat16, or of ``out``'s type.  A zero
    matrix gives zeros, whatever ``eps`` is, one with a NaN or an infinity NaNs.  X's elements are held to
    about 2e-12, which is more than 1e-3 of a matrix with a norm below 1e-6 ``eps``.  ``workspace``:
    adjacent elements at a 256-byte boundary, ``orthogonalize_workspace`` bytes or more.  Blocks of the kernel wait
    for one another; where such a wait took longer than 2 s the result is NaNs, and no error is raised."""
    dt = _float(g, "g")
    dev = _device(g, "g")
    shape, st = g.shape, g.stride()
    if len(shape) == 2:
        count, (rows, cols), sb, (sr, sc) = 1, shape, 0, st
    elif len(shape) == 3:
        (count, rows, cols), (sb, sr, sc) = shape, st
    else:
        raise ValueError(f"g: expected [rows, cols] or [count, rows, cols], got {tuple(shape)}")
    if not 0 <= steps <= 32:
        raise ValueError(f"steps: {steps} (0 to 32)")
    coef = list(coefficients)
    if len(coef) == 3 and not hasattr(coef[0], "__len__"):
        coef = coef * steps
    else:
        if len(coef) != steps or any(len(c) != 3 for c in coef):
            raise ValueError(f"coefficients: expected a triple, or {steps} of them")
        coef = [v for c in coef for v in c]
    s = _stream(dev, stream, g, out is None or workspace is None)
    if out is None:
        out = _empty(shape, g, "bfloat16")
    ot = _float(out, "out")
    _same_shape(out, shape, "out")
    _on(dev, out, "out")
    so = out.stride()
    if any(n > 1 and not m for n, m in zip(shape, so)):
        raise ValueError(f"out: elements share memory (strides {tuple(so)})")
    need = orthogonalize_workspace(count, rows, cols)
    if workspace is None:
        workspace = _empty((need,), g, "uint8")
        have = need
    else:
        have = _nbytes(workspace, "workspace")
        _on(dev, workspace, "workspace")
    rt.check(_entry("ad_orthogonalize")(
        dev, dt, g.data_ptr(), count, rows, cols, sb, sr, sc, steps, (rt.c_float * max(1, len(coef)))(*coef), eps, ot,
        out.data_ptr(), so[0] if len(so) == 3 else 0, so[-2], so[-1], workspace.data_ptr(), have, s))
    return out
