"""Operators of language models at the edges of what they take (B200 only).  The 64-bit
implementations and the bounds' derivation are those of test_gpu_ops."""
import math
import threading

import pytest

from .test_gpu_ops import (N_SOFT, block_operands, check_block, check_logprobs, check_orthogonal, dtype, logprobs64,
                           orthogonal64, rand, seeded, update, within)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops():
    from ad_b200 import ops as o
    return o


@pytest.mark.parametrize("t", ["float32", "bfloat16"])
@pytest.mark.parametrize("scale", [0.7, 1.0, 1.25])
@pytest.mark.parametrize("base", [3e4, 5e5, 2e6, 1e8, 1e9, 1e10, 1e12, 1e20, 9e29, 1.1e30, 1e37])
@pytest.mark.parametrize("vocab", [50, 20000])
def test_token_logprobs_of_large_logits(ops, t, scale, base, vocab):
    """Rows that are large throughout, rows masked with a finite value that is not the type's lowest, and
    rows of such a mask alone."""
    gen = seeded(vocab, len(t), math.log2(base), 100 * scale)
    logits = rand(gen, (12, vocab), t, 2.0)
    for r, b in ((0, base), (4, -base)):
        logits[r] = b                                    # nothing but the mask
        logits[r + 1, :vocab - 9] = b                    # the mask first (or far ahead of the rest)
        logits[r + 2, 5::3] = b                          # in between
        steps = torch.randint(0, 4, (vocab,), generator=gen)
        near = torch.full((vocab,), b, dtype=dtype(t))   # some neighbouring values
        spacing = torch.nextafter(near.abs().double().to(dtype(t)), torch.tensor(math.inf, dtype=dtype(t))) - near.abs()
        logits[r + 3] = (near.double() + steps * spacing.double()).to(dtype(t)).cuda()
    logits[8, ::2], logits[8, 1::2] = base, -base        # both signs
    logits[9] = -math.inf
    logits[9, 3] = -base                                 # one value left
    logits[10, :vocab // 2], logits[10, vocab // 2:] = -base, -base / 2
    tokens = torch.randint(0, vocab, (12,), generator=gen)
    tokens[9] = 3
    g, e = rand(gen, (12,), "float32"), rand(gen, (12,), "float32", 0.1)
    r, _ = check_logprobs(ops, logits, tokens.cuda(), scale, 7, t, g, e)
    lse = logprobs64(logits, tokens, scale, 0)["lse"]
    within(r.stats[:, 3].cpu(), lse, lse.abs() + 4 + math.log(vocab), N_SOFT, "float32")


@pytest.mark.parametrize("t", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("scale", [0.6, 1.0, 1.25])
@pytest.mark.parametrize("vocab", [40, 3000])
def test_token_logprobs_of_lowest_values(ops, t, scale, vocab):
    """Tokens masked with the type's lowest value that are asked for, and alternatives that reach such
    values: finite where 32 bits hold them."""
    gen = seeded(vocab, len(t), 10 * scale)
    low = torch.finfo(dtype(t)).min
    logits = rand(gen, (6, vocab), t, 2.0)
    logits[:, 4:] = low                  # four values left
    logits[1, :4] += 1000                # a larger maximum
    logits[2, 5] = -math.inf
    if t != "float16":
        logits[3, 0] = 1e30              # far above everything
        logits[4, 0] = -low              # the largest there is
    tokens = torch.tensor([vocab - 1, 17, 5, 9, 20, 0])
    r = ops.token_logprobs(logits, tokens.cuda(), top=10, scale=scale)
    w = logprobs64(logits, tokens, scale, 10)
    for got, want in ((r.logp, w["logp"]), (r.top_logp, w["top"])):
        want = want.float().double()     # past the range of 32 bits: infinite
        within(got.cpu(), want, want.abs().nan_to_num(posinf=0.0) + 4 + math.log(vocab), N_SOFT, "float32")
    assert torch.equal(r.top_index[[0, 1, 3, 4, 5]].cpu(), w["index"][[0, 1, 3, 4, 5]])
    if t == "float16" or scale <= 1.0:
        assert torch.isfinite(r.logp[[0, 1]]).all()


@pytest.mark.parametrize("t", ["float32", "bfloat16"])
@pytest.mark.parametrize("scale", [1.0, 1.25])
def test_token_logprobs_grad_of_rows_at_the_lowest_value(ops, t, scale):
    """A row whose values are all the type's lowest has a gradient like any row of equal values, also
    where the log of its sum lies past the range of 32 bits; one of -inf has none."""
    vocab = 70
    logits = torch.full((3, vocab), torch.finfo(dtype(t)).min, device="cuda", dtype=dtype(t))
    logits[1] = 0.5
    logits[2] = -math.inf
    tokens = torch.tensor([3, 3, 3], device="cuda")
    g, e = torch.full((3,), -0.5, device="cuda"), torch.full((3,), 0.25, device="cuda")
    _, d = check_logprobs(ops, logits, tokens, scale, 2, t, g, e)
    assert d[:2].all() and not d[2].any()


def test_token_logprobs_largest_scale(ops):
    """Factors up to the largest number of 32 bits: equal values share, a larger one takes all."""
    logits = torch.zeros(4, 100, device="cuda")
    logits[1, 7] = 1.0
    logits[2] = -3.0
    logits[3] = 1e-30
    logits[3, 9] = 2e-30
    for scale in (1e30, 2.3e38, 2.4e38, 3.4e38):
        r = ops.token_logprobs(logits, torch.tensor([7, 7, 0, 9], device="cuda"), top=1, scale=scale)
        want = torch.tensor([-math.log(100), 0.0, -math.log(100), 0.0], dtype=torch.float64)
        if scale < 1e31:  # the fourth row's values lie 1 apart
            want[3] = 1.0 - math.log(math.e + 99)
        within(r.logp.cpu(), want, torch.full((4,), 5.0, dtype=torch.float64), N_SOFT, "float32")
        assert r.top_index[:, 0].tolist() == [0, 7, 0, 9]


def test_block_norm_threads_of_different_widths(ops):
    """Widths that share a kernel but not its amount of shared memory, launched from threads side by side
    (the library's calls leave Python's lock to the others)."""
    from ad_b200 import runtime as rt
    L, failed = rt.lib(), []

    def loop(width, calls):
        try:
            stream = torch.cuda.Stream()
            d = block_operands(ops, 2, width, "bfloat16", "bfloat16", "rms", "none")
            h, y, st = ops.block_norm(d["x"], d["z"], d["wa"], d["wb"])
            want = ops.block_norm_grad(d["dh"], d["dy"], d["x"], d["z"], d["wa"], d["wb"], st)
            g = [torch.empty_like(v) for v in want if v is not None]
            ws = torch.empty(ops.block_norm_grad_workspace(2, width), dtype=torch.uint8, device="cuda")
            torch.cuda.synchronize()
            p = {k: None if v is None else v.data_ptr() for k, v in d.items()}
            args = (0, ops.BF16, ops.BF16, 0, p["dh"], width, p["dy"], width, p["x"], width, p["z"], width, None, 0, 0, 0,
                    p["wa"], None, p["wb"], None, 1.0, st.data_ptr(), 2, width, g[0].data_ptr(), width, g[1].data_ptr(),
                    width, None, 0, g[2].data_ptr(), None, g[3].data_ptr(), None, ws.data_ptr(), ws.numel(),
                    stream.cuda_stream)
            for _ in range(calls):
                rt.check(L.ad_block_norm_grad(*args))
            stream.synchronize()
            assert all(torch.equal(u, v) for u, v in zip(g, [v for v in want if v is not None]))
        except BaseException as e:  # noqa: BLE001  (handed to the test's own thread)
            failed.append(e)

    threads = [threading.Thread(target=loop, args=(w, 20000)) for w in (4096, 2304, 3200, 2560)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


@pytest.mark.parametrize("t,wt", [("float32", "float32"), ("bfloat16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("width,gate", [(6145, "none"), (6400, "three"), (7168, "none"), (7172, "row"), (7680, "three"),
                                        (8192, "none"), (8192, "row"), (8193, "three")])
def test_block_norm_wide_rows(ops, t, wt, kind, width, gate):
    """Widths whose weights and rows to come would not all fit a multiprocessor's shared memory, and
    those whose gradients give 16 or 32 elements to a thread."""
    d = block_operands(ops, 6, width, t, wt, kind, gate)
    check_block(ops, d, t, wt, kind, gate == "row", 1.0)


def test_block_norm_wide_rows_of_many_blocks(ops):
    d = block_operands(ops, 700, 8192, "float32", "float32", "rms", "many")
    check_block(ops, d, "float32", "float32", "rms", True, 0.5)


def test_a_refused_call_leaves_nothing_to_the_next(ops):
    """The error of one call is not reported by the next one, which works."""
    import ctypes
    from ad_b200 import runtime as rt
    x, w = torch.randn(5, 64, device="cuda"), torch.ones(64, device="cuda")
    q = torch.randn(1, 5, 2, 32, device="cuda")
    cos, sin = (torch.from_numpy(v).cuda() for v in ops.rotary_table(8, 32))
    pos = torch.arange(5, device="cuda")
    tok = torch.arange(5, device="cuda")
    stats = ops.block_norm(x, x, w, w)[2]
    calls = [lambda: ops.rotary(q, None, cos, sin, pos), lambda: ops.rotary(q, None, cos, sin, pos, layout="interleaved"),
             lambda: ops.rotary(q[..., 1:31], None, cos[:, :15].contiguous(), sin[:, :15].contiguous(), pos),
             lambda: ops.block_norm(x, x, w, w), lambda: ops.block_norm_grad(x, x, x, x, w, w, stats),
             lambda: ops.token_logprobs(x, tok),
             lambda: ops.token_logprobs_grad(x, tok, ops.token_logprobs(x, tok).stats),
             lambda: ops.orthogonalize(x), lambda: ops.orthogonalize(x, steps=0)]
    L = rt.lib()
    st = (ctypes.c_int64 * 3)(64, 64, 32)
    for call in calls:
        refused = L.ad_rotary(99, 0, q.data_ptr(), st, q.data_ptr(), st, 2, None, None, None, None, 0, 1, 5, 32, 32, 0, 0,
                              cos.data_ptr(), sin.data_ptr(), 8, pos.data_ptr(), 1, 0, 1, None)
        assert refused and b"ad_rotary" in L.ad_last_error()
        call()
    torch.cuda.synchronize()


# Of a sigmoid's share: exp to 2 ulp (4 E), 1 + exp (4 E carried on and a rounding), the quotient to 2 ulp,
# a product: 14 E.  Its slope is the product of two shares, times two factors: 32 E.  16-bit elements
# take an exp of 2 + 1.2 |x| ulp, 50 at most here: 100 E more a share, far below their own rounding.
@pytest.mark.parametrize("t,n_act,n_slope", [("float32", 14, 32), ("bfloat16", 114, 232), ("float16", 114, 232)])
@pytest.mark.parametrize("shape", [(12, 256), (12, 100), (6, 333)])
def test_block_norm_saturated_gates(ops, t, n_act, n_slope, shape):
    """h = sigmoid(gate) z alone, and the gate's gradient, relative to their own size."""
    rows, width = shape
    gen = seeded(rows, width, len(t))
    signs = torch.tensor([12.0, -12.0, 20.0, -20.0, 5.0, -40.0])
    gate = (signs.repeat(rows * width)[:rows * width].reshape(rows, width) + torch.rand(rows, width, generator=gen)).to(dtype(t)).cuda()
    z, dh = rand(gen, shape, t, 1.0, 3.0), rand(gen, shape, t, 1.0, 3.0)
    opts = dict(gate=gate, gate_sigmoid=True, residual_scale=0.0)
    x = torch.zeros_like(z)
    h, _, st = ops.block_norm(x, z, None, None, **opts)
    g = ops.block_norm_grad(dh, None, x, z, None, None, st, **opts)
    big = gate.double()
    act, rest = torch.sigmoid(big), torch.sigmoid(-big)
    within(h, act * z.double(), act * z.double().abs(), n_act, t)
    within(g.z, act * dh.double(), act * dh.double().abs(), n_act, t)
    slope = act * rest * z.double() * dh.double()
    within(g.gate, slope, slope.abs(), n_slope, t)
    shared = ops.block_norm_grad(dh, None, x, z, None, None, st, gate=gate[:1], gate_sigmoid=True, residual_scale=0.0)
    slope = (act * rest)[:1] * z.double() * dh.double()
    within(shared.gate, slope.sum(0, keepdim=True), slope.abs().sum(0, keepdim=True), n_slope + rows, t)
    gate[0] = math.inf
    gate[1] = -math.inf
    h, _, st = ops.block_norm(x, z, None, None, **opts)
    g = ops.block_norm_grad(dh, None, x, z, None, None, st, **opts)
    assert torch.equal(h[0], z[0]) and not h[1].any() and not g.gate[:2].any() and torch.equal(g.z[0], dh[0])


@pytest.mark.parametrize("shape", [(16,), (1, 16), (3, 16)])
@pytest.mark.parametrize("t", ["float32", "bfloat16"])
def test_block_norm_grad_of_a_gate_without_rows(ops, shape, t):
    """A gate shared by no rows has a gradient of zeros, whatever was in its memory."""
    x = torch.ones((0, 16), device="cuda", dtype=dtype(t))
    w, gate = torch.ones(16, device="cuda"), torch.ones(shape, device="cuda", dtype=dtype(t))
    h, y, stats = ops.block_norm(x, x, w, w, gate=gate)
    torch.full((1 << 16,), math.nan, device="cuda")  # what the allocator may hand out again
    g = ops.block_norm_grad(x, x, x, x, w, w, stats, gate=gate)
    assert g.gate.shape == shape and not g.gate.any()
    wide = torch.full((shape[0] if len(shape) > 1 else 1, 40), math.nan, device="cuda", dtype=dtype(t))
    room = wide[:, 5:21].reshape(shape) if len(shape) == 1 else wide[:, 5:21]
    out = ops.BlockNormGrads(x, x, room, *(torch.full((16,), math.nan, device="cuda") for _ in range(2)), None, None)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    ops.block_norm_grad(x, x, x, x, w, w, stats, gate=gate, out=out, workspace=torch.empty(0, device="cuda"), stream=s)
    s.synchronize()
    assert not room.any() and not out.after_weight.any() and not out.before_weight.any()
    assert torch.isnan(wide[:, :5]).all() and torch.isnan(wide[:, 21:]).all()


def test_clear_rows_refuses(ops):
    from ad_b200 import runtime as rt
    x = torch.ones(4, 8, device="cuda")
    for args in ((16, 32, 4), (32, -1, 4), (32, 32, -1)):
        with pytest.raises(rt.ADError, match="ad_clear_rows"):
            rt.check(rt.lib().ad_clear_rows(0, x.data_ptr(), *args, None))
    assert x.all()


@pytest.mark.parametrize("eps", [0.0, 1e-38, 1e-7])
def test_orthogonalize_zero_matrices(ops, eps):
    g = update(seeded(50), 3, 70, 100, "noise", "float32")
    g[1] = 0
    y = ops.orthogonalize(g, eps=eps)
    assert not y[1].any() and torch.isfinite(y).all() and y[0].any() and y[2].any()
    assert not ops.orthogonalize(g[1:2], eps=eps, steps=0).any()


@pytest.mark.parametrize("norm", [1e-42, 1e-40, 1e-36, 3e-35, 1e-34, 1e-30, 1e30, 1e38])
@pytest.mark.parametrize("rows,cols", [(60, 50), (33, 129)])
def test_orthogonalize_any_scale(ops, norm, rows, cols):
    """Scales at which the reciprocal of the norm does not fit 32 bits, or only as a subnormal number."""
    gen = seeded(51, rows, cols)
    g = torch.randn(2, rows, cols, generator=gen, dtype=torch.float64)
    g[0] = torch.linalg.qr(g[0]).Q if rows >= cols else torch.linalg.qr(g[0].T).Q.T
    g *= norm / g.square().sum((1, 2), keepdim=True).sqrt()
    g[1, 0, 0] = norm      # one value that 32 bits hold however small the others are
    g = g.float().cuda()
    check_orthogonal(ops.orthogonalize(g, eps=0.0), orthogonal64(g, 5, [ops.NEWTON_SCHULZ] * 5, 0.0), 5, "bfloat16")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,r", [(32, 16), (32, 32), (33, 18), (32, 12)])
def test_rotary_empty_tables(ops, layout, d, r):
    """With tables of no rows every position lies outside them."""
    q = torch.ones(1, 3, 2, d, device="cuda")
    none = torch.empty(0, r // 2, device="cuda")
    y, _ = ops.rotary(q, None, none, none, torch.arange(3, device="cuda"), layout=layout)
    assert torch.isnan(y[..., :r]).all() and torch.equal(y[..., r:], q[..., r:])
