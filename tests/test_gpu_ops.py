"""Operators of language models against plain 64-bit implementations (B200 only).

Bounds are derived from the arithmetic, not from runs: `U[t]` is the unit roundoff of the result's
type, E = 2^-24 that of 32 bits; a value computed by n operations in 32 bits from terms of total
magnitude `mag` may be off by n E mag, and is rounded once to its type."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

E = 2.0 ** -24
U = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 1e-37, "bfloat16": 1e-37, "float16": 2.0 ** -24}  # spacing of the smallest numbers


@pytest.fixture(scope="module")
def ops():
    from ad_b200 import ops as o
    return o


def dtype(name):
    return getattr(torch, name)


def within(got, want, mag, n, t):
    """|got - want| <= one rounding to type t + n E mag; NaN and infinities in the same places."""
    got = got.double()
    assert got.shape == want.shape
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    bound = 1.01 * U[t] * want.abs() + n * E * mag + TINY[t]
    worst = ((got - want).abs() / bound)[fine]
    assert worst.numel() == 0 or float(worst.max()) <= 1.0, float(worst.max())


def rand(gen, shape, t, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * std + mean).to(dtype(t)).cuda()


def seeded(*key):
    return torch.Generator().manual_seed(sum((i + 1) * int(k) for i, k in enumerate(key)))


# ------------------------------------------------------------------ rotary

def rotary64(x, cos, sin, pos, half, layout, inverse):
    x = x.double().clone()
    ok = (pos >= 0) & (pos < cos.shape[0])
    at = pos.clamp(0, max(cos.shape[0] - 1, 0))
    c, s = cos.double()[at], sin.double()[at]
    c, s = (torch.where(ok[..., None], v, math.nan)[:, :, None] for v in (c, s))
    if inverse:
        s = -s
    iu = torch.arange(half) if layout == "half" else torch.arange(0, 2 * half, 2)
    iv = iu + (half if layout == "half" else 1)
    u, v = x[..., iu], x[..., iv]
    mag = x.abs()
    mag[..., iu] = mag[..., iv] = (u.abs() * 1.2 + v.abs() * 1.2)  # |cos|, |sin| <= 1.2 with any gain used here
    x[..., iu], x[..., iv] = u * c - v * s, v * c + u * s
    return x, mag


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("t", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("b,n,hq,hk,d,r", [
    (1, 1, 1, 1, 2, 2), (3, 1, 8, 2, 64, 64), (2, 37, 4, 4, 128, 64), (1, 130, 5, 1, 80, 80), (2, 9, 3, 3, 96, 30),
    (2, 5, 2, 1, 33, 18), (1, 4, 2, 2, 24, 0), (1, 3, 64, 8, 256, 250), (2, 3, 1, 1, 1030, 1030)])
def test_rotary(ops, layout, t, b, n, hq, hk, d, r):
    gen = seeded(b, n, hq, hk, d, r)
    cos, sin = (torch.from_numpy(v).cuda() for v in ops.rotary_table(200, r))
    pos = torch.randint(0, 200, (b, n), generator=gen)
    q, k = rand(gen, (b, n, hq, d), t), rand(gen, (b, n, hk, d), t)
    for inverse in (False, True):
        yq, yk = ops.rotary(q, k, cos, sin, pos.cuda(), layout=layout, inverse=inverse)
        for y, x in ((yq, q), (yk, k)):
            want, mag = rotary64(x.cpu(), cos.cpu(), sin.cpu(), pos, r // 2, layout, inverse)
            within(y.cpu(), want, mag, 3, t)
            assert torch.equal(y[..., r:], x[..., r:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,r", [(64, 64), (64, 22), (40, 40)])
def test_rotary_strides_types_and_in_place(ops, layout, d, r):
    gen = seeded(d, r, 7)
    cos, sin = (torch.from_numpy(v).cuda() for v in ops.rotary_table(64, r))
    store = rand(gen, (2, 6, 19, d + 3), "bfloat16")
    q = store[:, :4, :, 1:d + 1].transpose(1, 2)      # heads first, unaligned, gaps
    k = store[:, 4:, :, 3:].transpose(1, 2)
    pos32 = torch.randint(0, 64, (19,), generator=gen, dtype=torch.int32)
    pos = pos32.long().expand(2, 19)
    want = [rotary64(x.cpu(), cos.cpu(), sin.cpu(), pos, r // 2, layout, False) for x in (q, k)]
    yq, yk = ops.rotary(q, k, cos, sin, pos32.cuda(), layout=layout)
    for y, w in ((yq, want[0]), (yk, want[1])):
        within(y.cpu(), *w, 3, "bfloat16")
    before = store.clone()
    zq, zk = ops.rotary(q, k, cos, sin, pos32.cuda(), layout=layout, out=(q, k))
    assert zq is q and zk is k and torch.equal(q, yq) and torch.equal(k, yk)
    assert torch.equal(store[:, :4, :, 0], before[:, :4, :, 0]) and torch.equal(store[:, 4:, :, :3], before[:, 4:, :, :3])
    assert torch.equal(store[:, :4, :, d + 1:], before[:, :4, :, d + 1:])


def test_rotary_unknown_positions_and_values(ops):
    cos, sin = (torch.from_numpy(v).cuda() for v in ops.rotary_table(16, 4))
    q = torch.ones(1, 5, 2, 8, device="cuda")
    q[0, 1, 0, 0] = math.inf
    q[0, 2, 1, 7] = math.nan
    pos = torch.tensor([[0, 3, 15, 16, -1]])
    y, none = ops.rotary(q, None, cos, sin, pos.cuda())
    assert none is None
    want, mag = rotary64(q.cpu(), cos.cpu(), sin.cpu(), pos, 2, "half", False)
    assert torch.isnan(y[0, 3:, :, :4]).all() and torch.isfinite(y[0, 3:, :, 4:]).all()
    assert torch.equal(torch.isnan(y.cpu()), torch.isnan(want))
    assert torch.equal(torch.isinf(y.cpu()), torch.isinf(want))
    within(y[0, 0].cpu(), want[0, 0], mag[0, 0], 3, "float32")


def test_rotary_empty(ops):
    cos, sin = (torch.from_numpy(v).cuda() for v in ops.rotary_table(16, 4))
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        q = torch.ones(shape, device="cuda")
        y, _ = ops.rotary(q, None, cos, sin, torch.zeros(shape[:2], dtype=torch.int64, device="cuda"))
        assert y.shape == q.shape


def test_rotary_turns_back(ops):
    """The inverse of the rotation gives the operand again: cos^2 + sin^2 is 1 within 3 E."""
    gen = seeded(5)
    cos, sin = (torch.from_numpy(v).cuda() for v in ops.rotary_table(4000, 64))
    q = rand(gen, (1, 4000, 2, 64), "float32")
    pos = torch.arange(4000, device="cuda")
    y, _ = ops.rotary(q, None, cos, sin, pos, layout="interleaved")
    z, _ = ops.rotary(y, None, cos, sin, pos, layout="interleaved", inverse=True)
    pair = q.reshape(1, 4000, 2, 32, 2).double().abs().sum(-1, keepdim=True).expand(-1, -1, -1, -1, 2).reshape(q.shape)
    within(z, q.double(), pair, 12, "float32")


# ------------------------------------------------------------------ norms around a block

def norm64(v, w, b, kind, eps):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    r = (((v - mean) ** 2).mean(-1, keepdim=True) + eps) ** -0.5
    n = (v - mean) * r
    y = n if w is None else n * w
    # terms that make up a value, each as large as it can be
    mag = (v.abs() + v.abs().mean(-1, keepdim=True)) * r
    mag = mag if w is None else mag * w.abs()
    if b is not None:
        y, mag = y + b, mag + b.abs()
    return y, n, r, mag


def block64(d, kind, sigmoid, scale, eps):
    x, z, gate = d["x"].double(), d["z"].double(), d.get("gate")
    w = {k: None if d.get(k) is None else d[k].double() for k in ("wa", "wb", "ba", "bb")}
    if w["wa"] is None:
        u, nz, rz, mu = z, None, None, z.abs()
    else:
        u, nz, rz, mu = norm64(z, w["wa"], w["ba"], kind, eps)
    act = slope = torch.ones_like(x)
    if gate is not None:
        per = x.shape[0] // gate.shape[0]
        g = gate.double().repeat_interleave(per, 0)
        act = torch.sigmoid(g) if sigmoid else g
        slope = act * (1 - act) if sigmoid else torch.ones_like(g)
    h = scale * x + act * u
    mh = abs(scale) * x.abs() + act.abs() * mu
    if w["wb"] is None:
        return dict(h=h, mh=mh, u=u, mu=mu, act=act, slope=slope, nz=nz, rz=rz)
    y, nh, rh, _ = norm64(h, w["wb"], w["bb"], kind, eps)
    my = (mh + mh.mean(-1, keepdim=True)) * rh
    my = (my + nh.abs() * (my * nh.abs()).mean(-1, keepdim=True)) * w["wb"].abs() + (0 if w["bb"] is None else w["bb"].abs())
    return dict(h=h, mh=mh, y=y, my=my, u=u, mu=mu, act=act, slope=slope, nz=nz, rz=rz, nh=nh, rh=rh)


def block_operands(ops, rows, width, t, wt, kind, gate, after=True, before=True, bias=None):
    gen = seeded(rows, width, len(t), len(wt), len(kind), len(gate))
    bias = kind == "layer" if bias is None else bias
    groups = {"none": 0, "row": rows, "one": 1, "three": 3, "many": rows // 2}[gate]
    d = dict(x=rand(gen, (rows, width), t, 2.0), z=rand(gen, (rows, width), t, 0.7, 0.3))
    d["gate"] = rand(gen, (groups, width), t, 1.0, 0.4) if groups else None
    d["wa"] = rand(gen, (width,), wt, 0.2, 1.0) if after else None
    d["wb"] = rand(gen, (width,), wt, 0.2, 1.0) if before else None
    d["ba"] = rand(gen, (width,), wt, 0.1) if after and bias else None
    d["bb"] = rand(gen, (width,), wt, 0.1) if before and bias else None
    d["dh"] = rand(gen, (rows, width), t, 0.1)
    d["dy"] = rand(gen, (rows, width), t, 0.1) if before else None
    return d


def run_block(ops, d, kind, sigmoid, scale, eps, grad=True, **kw):
    opts = dict(gate=d["gate"], after_bias=d["ba"], before_bias=d["bb"], kind=kind, gate_sigmoid=sigmoid,
                residual_scale=scale, eps=eps)
    h, y, stats = ops.block_norm(d["x"], d["z"], d["wa"], d["wb"], **opts)
    g = ops.block_norm_grad(d["dh"], d["dy"], d["x"], d["z"], d["wa"], d["wb"], stats, **opts) if grad else None
    return h, y, g


# Operations on the way of a value in the widest case: a row's sum is made of at most 32 additions
# in a thread and 10 across threads, the rest are single operations.
N_ROW = 60
N_GRAD = 3 * N_ROW


def check_block(ops, d, t, wt, kind, sigmoid, scale, eps=1e-5):
    h, y, g = run_block(ops, d, kind, sigmoid, scale, eps)
    r = block64(d, kind, sigmoid, scale, eps)
    within(h, r["h"], r["mh"], N_ROW, t)
    if d["wb"] is not None:
        within(y, r["y"], r["my"], 2 * N_ROW, t)
    else:
        assert y is None
    rows, width = d["x"].shape
    layer = kind == "layer"

    def through(v, mv, n, rr):  # gradient through a norm, and the magnitude of its terms
        out = v - n * (v * n).mean(-1, keepdim=True)
        big = n.abs() + 1  # the normalised row's own error goes with the mean
        mag = mv + big * (mv * big).mean(-1, keepdim=True)
        if layer:
            out, mag = out - v.mean(-1, keepdim=True), mag + mv.mean(-1, keepdim=True)
        return rr * out, rr * mag

    total, mt = d["dh"].double(), d["dh"].double().abs()
    if d["wb"] is not None:
        v = d["dy"].double() * d["wb"].double()
        # how far nh may be off counts through mh
        grow = 1 + r["rh"] * r["mh"]
        a, ma = through(v, v.abs() * grow, r["nh"], r["rh"])
        total, mt = total + a, mt + ma * (1 + (r["rh"] * r["mh"]).mean(-1, keepdim=True))
    within(g.x, scale * total, abs(scale) * mt, N_GRAD, t)
    du, mdu = total * r["act"], mt * r["act"].abs()
    if d["wa"] is not None:
        wa = d["wa"].double()
        growz = 1 + r["rz"] * d["z"].double().abs()
        a, ma = through(du * wa, mdu * wa.abs() * growz, r["nz"], r["rz"])
        within(g.z, a, ma * (1 + growz.mean(-1, keepdim=True)), N_GRAD, t)
    else:
        within(g.z, du, mdu, N_GRAD, t)
    n_sum = N_GRAD + rows  # a column's sum: as many additions as rows at most
    if d["gate"] is not None:
        per = rows // d["gate"].shape[0]
        dg, mg = total * r["u"] * r["slope"], mt * (r["mu"] + r["u"].abs()) * (r["slope"].abs() + 1e-3)
        dg, mg = (v.reshape(-1, per, width).sum(1) for v in (dg, mg))
        within(g.gate, dg, mg, n_sum if per > 1 else N_GRAD, t)
    else:
        assert g.gate is None
    if d["wa"] is not None:
        within(g.after_weight, (du * r["nz"]).sum(0), (mdu * (r["nz"].abs() + growz)).sum(0), n_sum, wt)
    if d["wb"] is not None:
        dy = d["dy"].double()
        within(g.before_weight, (dy * r["nh"]).sum(0), (dy.abs() * (r["nh"].abs() + grow)).sum(0), n_sum, wt)
    for got, want, mag, like in ((g.after_bias, du, mdu, d["ba"]), (g.before_bias, d["dy"], None, d["bb"])):
        assert (got is None) == (like is None)
        if got is not None:
            within(got, want.double().sum(0), (want if mag is None else mag).double().abs().sum(0), n_sum, wt)


@pytest.mark.parametrize("t,wt", [("float32", "float32"), ("bfloat16", "float32"), ("bfloat16", "bfloat16"),
                                  ("float16", "float16")])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,width,gate,sigmoid,scale", [
    (1, 1, "none", False, 1.0), (6, 8, "row", True, 0.5), (6, 1024, "three", False, 1.0), (300, 256, "one", True, 1.0),
    (1000, 100, "many", False, -0.7), (12, 1023, "three", True, 2.0), (9, 4096, "row", False, 1.0),
    (7, 5000, "none", False, 1.0), (6, 8200, "three", True, 1.0), (3, 9001, "row", True, 1.0)])
def test_block_norm(ops, t, wt, kind, rows, width, gate, sigmoid, scale):
    d = block_operands(ops, rows, width, t, wt, kind, gate)
    check_block(ops, d, t, wt, kind, sigmoid, scale)


@pytest.mark.parametrize("after,before", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("gate", ["none", "row", "three"])
def test_block_norm_without_norms(ops, after, before, gate):
    d = block_operands(ops, 33, 200, "float32", "float32", "layer", gate, after, before)
    check_block(ops, d, "float32", "float32", "layer", False, 1.0)


def test_block_norm_rms_with_bias(ops):
    d = block_operands(ops, 10, 96, "bfloat16", "float32", "rms", "row", bias=True)
    check_block(ops, d, "bfloat16", "float32", "rms", True, 1.0)


def test_block_norm_many_rows(ops):
    """More rows than blocks; the sums of the weights over all of them."""
    d = block_operands(ops, 5000, 64, "float32", "float32", "layer", "many")
    check_block(ops, d, "float32", "float32", "layer", True, 1.0)


def test_block_norm_strides(ops):
    """Rows with gaps and an odd first element; the result the same as from rows without."""
    d = block_operands(ops, 20, 130, "bfloat16", "bfloat16", "rms", "row")
    s = dict(d)
    for k in ("x", "z", "gate", "dh", "dy"):
        wide = torch.full((20, 140), 9.0, device="cuda", dtype=torch.bfloat16)
        wide[:, 3:133] = d[k]
        s[k] = wide[:, 3:133]
    for a, b in zip(run_block(ops, d, "rms", True, 1.0, 1e-5), run_block(ops, s, "rms", True, 1.0, 1e-5)):
        for u, v in zip(a if isinstance(a, tuple) else (a,), b if isinstance(b, tuple) else (b,)):
            assert (u is None) == (v is None) and (u is None or torch.equal(u, v))


def test_block_norm_given_results(ops):
    d = block_operands(ops, 12, 256, "float32", "float32", "layer", "three")
    h, y, stats = ops.block_norm(d["x"], d["z"], d["wa"], d["wb"], gate=d["gate"], kind="layer")
    g = ops.block_norm_grad(d["dh"], d["dy"], d["x"], d["z"], d["wa"], d["wb"], stats, gate=d["gate"], kind="layer")
    n = ops.block_norm_grad_workspace(12, 256, 3, 0)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    room = ops.BlockNormGrads(*(None if v is None else torch.full_like(v, math.nan) for v in g))
    g2 = ops.block_norm_grad(d["dh"], d["dy"], d["x"], d["z"], d["wa"], d["wb"], stats, gate=d["gate"], kind="layer",
                             out=room, workspace=ws)
    assert all(v is r and torch.equal(v, u) for v, r, u in zip(g2, room, g) if v is not None)
    x, z = d["x"].clone(), d["z"].clone()
    h2, y2, _ = ops.block_norm(x, z, d["wa"], d["wb"], gate=d["gate"], kind="layer", out=(x, z, torch.empty_like(stats)))
    assert h2 is x and torch.equal(h2, h) and torch.equal(y2, y)


def test_block_norm_differences(ops):
    """Gradients against central differences of the 64-bit loss sum(h a) + sum(y b): step 1e-4, whose
    square times the third derivatives here (of order 10) is far below the bound of 1e-4."""
    d = block_operands(ops, 6, 12, "float32", "float32", "layer", "three")
    _, _, g = run_block(ops, d, "layer", True, 0.8, 1e-5)
    names = dict(x="x", z="z", gate="gate", wa="after_weight", wb="before_weight", ba="after_bias", bb="before_bias")
    d64 = {k: v.double() for k, v in d.items()}

    def loss(e):
        r = block64(e, "layer", True, 0.8, 1e-5)
        return float((r["h"] * e["dh"]).sum() + (r["y"] * e["dy"]).sum())

    for k, field in names.items():
        flat = getattr(g, field).double().reshape(-1)
        for i in range(0, flat.numel(), max(1, flat.numel() // 9)):
            step = torch.zeros(flat.numel(), dtype=torch.float64, device="cuda")
            step[i] = 1e-4
            step = step.reshape(d64[k].shape)
            diff = (loss({**d64, k: d64[k] + step}) - loss({**d64, k: d64[k] - step})) / 2e-4
            assert abs(diff - float(flat[i])) <= 1e-4 * (1 + abs(diff)), (k, i)


def test_block_norm_zero_rows_and_infinities(ops):
    """A row of zeros has a norm of zeros; an infinity spoils its own row alone."""
    d = block_operands(ops, 4, 64, "bfloat16", "float32", "rms", "none")
    clean = run_block(ops, d, "rms", False, 1.0, 1e-5)
    d["z"][1] = 0
    d["x"][1] = 0
    d["z"][2, 5] = math.inf
    h, y, g = run_block(ops, d, "rms", False, 1.0, 1e-5)
    assert not h[1].any() and not y[1].any()
    for r in (0, 3):
        assert torch.equal(h[r], clean[0][r]) and torch.equal(y[r], clean[1][r]) and torch.equal(g.z[r], clean[2].z[r])
    assert torch.isnan(y[2]).all()


def test_block_norm_no_rows(ops):
    d = {k: torch.ones((0, 16), device="cuda") for k in ("x", "z", "dh", "dy")}
    w = torch.ones(16, device="cuda")
    h, y, stats = ops.block_norm(d["x"], d["z"], w, w)
    g = ops.block_norm_grad(d["dh"], d["dy"], d["x"], d["z"], w, w, stats)
    assert h.shape == (0, 16) and not g.after_weight.any() and not g.before_weight.any()


# ------------------------------------------------------------------ token log probabilities

def logprobs64(logits, tokens, scale, top, g=None, e=None):
    x = scale * logits.double().cpu()
    tokens = tokens.cpu()
    m = x.amax(-1, keepdim=True)
    empty = m[:, 0] == -math.inf
    m = torch.where(torch.isinf(m) & (m < 0), 0.0, m)
    ex = torch.exp(x - m)
    s = ex.sum(-1, keepdim=True)
    lse = m + torch.log(s)
    # not x - lse: beside the lowest value of 32 bits the logarithm would be lost even in 64
    lp = torch.where(empty[:, None], -math.inf, (x - m) - torch.log(s))
    p = torch.where(empty[:, None], 0.0, ex / s)
    ent = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    has = (tokens >= 0) & (tokens < x.shape[1])
    at = torch.where(has, tokens, 0).long()
    logp = lp.gather(1, at[:, None])[:, 0]
    logp = torch.where(has, logp, torch.where(tokens < 0, 0.0, math.nan))
    order = torch.sort(logits.double().cpu(), dim=-1, descending=True, stable=True).indices[:, :top]
    out = dict(logp=logp, entropy=ent, top=lp.gather(1, order), index=order, lse=lse[:, 0], p=p, lp=lp, empty=empty)
    if g is not None:
        g, e = (v.double().cpu()[:, None] for v in (g, e))
        gg = torch.where((tokens >= 0)[:, None], g, 0.0)
        flat = torch.where(p > 0, lp, 0.0)
        d = -p * (gg + e * (flat + ent[:, None]))
        mag = p * (gg.abs() + e.abs() * (flat.abs() + ent[:, None]))
        hot = torch.zeros_like(p)
        hot[has & ~empty, at[has & ~empty]] = 1.0
        # the exponent's own rounding grows with its distance from the largest
        out.update(grad=scale * (d + hot * gg), mag=scale * (mag * (4 + flat.abs()) + hot * gg.abs()))
    return out


# ex2.approx: 2 units in the last place; the exponent's factor and product: 2 roundings of up to
# its magnitude, counted through (4 + |log p|); a thread's sum of up to 128 such values and the joins.
N_SOFT = 200


def check_logprobs(ops, logits, tokens, scale, top, t, g=None, e=None):
    r = ops.token_logprobs(logits, tokens, top=top, scale=scale)
    w = logprobs64(logits, tokens, scale, top, g, e)
    ln_s = w["entropy"] + 4
    within(r.logp.cpu(), w["logp"], ln_s + torch.nan_to_num(w["logp"], neginf=0.0).abs(), N_SOFT, "float32")
    within(r.entropy.cpu(), w["entropy"], ln_s, N_SOFT, "float32")
    if top:
        assert torch.equal(r.top_index.cpu(), w["index"])
        within(r.top_logp.cpu(), w["top"], ln_s[:, None] + torch.nan_to_num(w["top"], neginf=0.0).abs(), N_SOFT, "float32")
    else:
        assert r.top_logp is None and r.top_index is None
    if g is not None:
        d = ops.token_logprobs_grad(logits, tokens, r.stats, g, e, scale=scale)
        within(d.cpu(), w["grad"], w["mag"], N_SOFT, t)
        return r, d
    return r, None


@pytest.mark.parametrize("t", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,vocab,top,scale", [
    (1, 1, 1, 1.0), (2, 3, 3, 0.5), (5, 31, 0, 1.0), (3, 100, 32, 2.0), (64, 1000, 5, 1.0), (300, 517, 4, 0.7),
    (1, 50001, 20, 1.25), (4, 131072, 32, 1.0), (150, 8191, 1, 1.0), (2, 32000, 0, 1.0)])
def test_token_logprobs(ops, t, rows, vocab, top, scale):
    gen = seeded(rows, vocab, top)
    logits = rand(gen, (rows, vocab), t, 3.0)
    tokens = torch.randint(0, vocab, (rows,), generator=gen)
    tokens[::7] = logits[::7].float().argmax(-1).cpu()
    if rows > 2:
        tokens[2] = -1
    g, e = rand(gen, (rows,), "float32"), rand(gen, (rows,), "float32", 0.1)
    check_logprobs(ops, logits, tokens.cuda(), scale, top, t, g, e)


@pytest.mark.parametrize("t", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab,top", [(300, 7), (20000, 32)])
def test_token_logprobs_ties(ops, t, vocab, top):
    """Many equal logits: the lower index first; zeros of both signs are equal."""
    gen = seeded(vocab, top)
    logits = torch.randint(-3, 3, (40, vocab), generator=gen).to(dtype(t)).cuda()
    logits[0] = 0
    logits[1] = 0
    logits[1, 1::2] = -0.0
    logits[2] = -5
    logits[2, vocab - 40:] = 4
    logits[3] = torch.arange(vocab).to(dtype(t)).cuda()
    logits[4] = -torch.arange(vocab).to(dtype(t)).cuda()
    tokens = torch.randint(0, vocab, (40,), generator=gen).cuda()
    check_logprobs(ops, logits, tokens, 1.0, top, t)


@pytest.mark.parametrize("t", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("vocab", [50, 40000])
def test_token_logprobs_masks(ops, t, vocab):
    """-inf and the type's lowest value as masks, rows with one value left, with nothing left, and all
    at the lowest value; the gradient of masked logits is zero."""
    gen = seeded(vocab, 3)
    logits = rand(gen, (8, vocab), t, 2.0)
    low = torch.finfo(dtype(t)).min
    logits[0, ::2] = -math.inf
    logits[1, 1::2] = low
    logits[2] = -math.inf
    logits[3] = -math.inf
    logits[3, vocab - 1] = 1.5
    logits[4] = low
    logits[5, :vocab - 3] = -math.inf
    logits[6] = low
    logits[6, 7] = -math.inf
    tokens = torch.tensor([1, 0, 5, vocab - 1, 3, 0, 7, -4]).cuda()
    g, e = rand(gen, (8,), "float32"), rand(gen, (8,), "float32", 0.1)
    r, d = check_logprobs(ops, logits, tokens, 1.0, 5, t, g, e)
    assert not d[2].any() and not d[0, ::2].any()
    assert float(r.logp[2]) == -math.inf and float(r.entropy[2]) == 0 and float(r.stats[2, 3]) == -math.inf


def test_token_logprobs_nan_and_bad_tokens(ops):
    logits = torch.randn(4, 600, device="cuda")
    logits[1, 33] = math.nan
    tokens = torch.tensor([600, 5, 2, -1], device="cuda", dtype=torch.int32)
    r = ops.token_logprobs(logits, tokens, top=3)
    d = ops.token_logprobs_grad(logits, tokens, r.stats, torch.ones(4, device="cuda"))
    assert torch.isnan(r.logp[:2]).all() and torch.isfinite(r.logp[2:]).all() and float(r.logp[3]) == 0
    assert torch.isnan(r.entropy[1]) and torch.isfinite(r.entropy[0])
    assert torch.isnan(d[:2]).all() and torch.isfinite(d[2:]).all() and not d[3].any()
    few = torch.full((1, 4), math.nan, device="cuda")
    few[0, 2] = 1.0
    r = ops.token_logprobs(few, torch.zeros(1, dtype=torch.int64, device="cuda"), top=3)
    assert r.top_index.tolist() == [[2, -1, -1]]


def test_token_logprobs_strides_and_in_place(ops):
    """Rows with a gap and an odd start; the gradient in place and in rows aligned otherwise."""
    gen = seeded(9)
    wide = rand(gen, (37, 1013), "bfloat16", 2.0)
    logits = wide[:, 5:1006]
    tokens = torch.randint(0, 1001, (37,), generator=gen).cuda()
    g, e = rand(gen, (37,), "float32"), rand(gen, (37,), "float32", 0.1)
    r, d = check_logprobs(ops, logits, tokens, 1.0, 4, "bfloat16", g, e)
    alone, _ = check_logprobs(ops, logits.contiguous(), tokens, 1.0, 4, "bfloat16", g, e)
    assert torch.equal(r.top_index, alone.top_index)
    before = wide.clone()
    got = ops.token_logprobs_grad(logits, tokens, r.stats, g, e, out=logits)
    assert got is logits and torch.equal(logits, d)
    assert torch.equal(wide[:, :5], before[:, :5]) and torch.equal(wide[:, 1006:], before[:, 1006:])


def test_token_logprobs_differences(ops):
    """Against central differences of the 64-bit loss sum(logp g) + sum(entropy e)."""
    gen = seeded(11)
    logits = rand(gen, (3, 20), "float32", 1.5)
    tokens = torch.tensor([3, 0, 19]).cuda()
    g, e = rand(gen, (3,), "float32"), rand(gen, (3,), "float32")
    r = ops.token_logprobs(logits, tokens, scale=0.8)
    d = ops.token_logprobs_grad(logits, tokens, r.stats, g, e, scale=0.8).double().cpu()

    def loss(x):
        w = logprobs64(x, tokens, 0.8, 0)
        return float((w["logp"] * g.double().cpu()).sum() + (w["entropy"] * e.double().cpu()).sum())

    x = logits.double().cpu()
    for i in range(60):
        step = torch.zeros(60, dtype=torch.float64)
        step[i] = 1e-4
        diff = (loss(x + step.reshape(3, 20)) - loss(x - step.reshape(3, 20))) / 2e-4
        assert abs(diff - float(d.reshape(-1)[i])) <= 1e-5 * (1 + abs(diff))


def test_token_logprobs_empty(ops):
    logits = torch.empty((0, 10), device="cuda")
    tokens = torch.empty((0,), dtype=torch.int64, device="cuda")
    r = ops.token_logprobs(logits, tokens, top=2)
    assert r.logp.shape == (0,) and r.top_index.shape == (0, 2)
    assert ops.token_logprobs_grad(logits, tokens, r.stats).shape == (0, 10)


# ------------------------------------------------------------------ memory, streams, repeats

def test_device_array_of_the_context(ops):
    """Memory of the framework's own context, on its stream 0 by way of the legacy stream."""
    import numpy as np
    from ad_b200 import runtime as rt
    ctx = rt.Context(0)
    try:
        x = np.random.default_rng(0).standard_normal((6, 50)).astype(np.float32)
        tok = np.arange(6, dtype=np.int64)
        p = ctx.malloc(x.nbytes), ctx.malloc(tok.nbytes), ctx.malloc(4 * 6 * 6)
        ctx.h2d(p[0], x.ctypes.data, x.nbytes)
        ctx.h2d(p[1], tok.ctypes.data, tok.nbytes)
        ctx.sync()
        A = ops.DeviceArray
        out = ops.TokenLogprobs(A(p[2], (6,)), A(p[2] + 24, (6,)), A(p[2] + 48, (6, 4)), None, None)
        ops.token_logprobs(A(p[0], (6, 50)), A(p[1], (6,), "int64"), out=out)
        got = np.empty((36,), np.float32)
        torch.cuda.synchronize()
        ctx.d2h(got.ctypes.data, p[2], got.nbytes)
        ctx.sync()
        w = logprobs64(torch.from_numpy(x), torch.from_numpy(tok), 1.0, 0)
        within(torch.from_numpy(got[:6]), w["logp"], w["entropy"] + 4 + w["logp"].abs(), N_SOFT, "float32")
        for q in p:
            ctx.free(q)
    finally:
        ctx.close()


def test_other_streams(ops):
    """On a stream that is current, and on one that is named with results given."""
    x = torch.randn(64, 512, device="cuda")
    w = torch.ones(512, device="cuda")
    h, y, st = ops.block_norm(x, x, w, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        h2, y2, _ = ops.block_norm(x, x, w, w)
    out = (torch.empty_like(x), torch.empty_like(x), torch.empty_like(st))
    s.wait_stream(torch.cuda.current_stream())
    ops.block_norm(x, x, w, w, out=out, stream=s)
    s.synchronize()
    assert torch.equal(h2, h) and torch.equal(y2, y) and torch.equal(out[1], y)
    with pytest.raises(ValueError, match="have to be given"):
        ops.block_norm(x, x, w, w, stream=s)


def test_graph_capture_and_repeats(ops):
    """Calls can be captured; the same operands give the same bits again."""
    x = torch.randn(500, 3000, device="cuda", dtype=torch.bfloat16)
    tok = torch.randint(0, 3000, (500,), device="cuda")
    g = torch.randn(500, device="cuda")

    def step():
        r = ops.token_logprobs(x, tok, top=7)
        return [*r, ops.token_logprobs_grad(x, tok, r.stats, g)]

    first = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    graph.replay()
    torch.cuda.synchronize()
    again = step()
    for a, b, c in zip(first, held, again):
        assert torch.equal(a, b) and torch.equal(a, c)


# ------------------------------------------------------------------ orthogonalised updates

def orthogonal64(g, steps, coef, eps):
    out = []
    for x in g.double():
        x = x / (x.square().sum().sqrt() + eps)
        for k in range(steps):
            a, b, c = coef[k]
            if x.shape[0] <= x.shape[1]:
                p = x @ x.T
                x = a * x + (b * p + c * (p @ p)) @ x
            else:
                p = x.T @ x
                x = a * x + x @ (b * p + c * (p @ p))
        out.append(x)
    return torch.stack(out)


# A step rounds three operands (X, A, B) to 11 bits: 2^-11 / sqrt(3) of their norms each (the
# root mean square of the rounding), added up over the steps as if none cancelled; then the result.
def check_orthogonal(got, want, steps, t):
    rms = 3 * steps * 2.0 ** -11 / math.sqrt(3) + U[t] / math.sqrt(3) + 2.0 ** -20
    for a, b in zip(got.double(), want):
        assert float((a - b).norm()) <= rms * float(b.norm()) + 1e-30, (float((a - b).norm() / b.norm()), rms)


def update(gen, count, rows, cols, kind, t):
    r = min(rows, cols)
    if kind == "noise":
        g = torch.randn(count, rows, cols, generator=gen, dtype=torch.float64)
    elif kind == "decay":
        g = (torch.randn(count, rows, r, generator=gen, dtype=torch.float64) / torch.arange(1, r + 1)) @ torch.randn(
            count, r, cols, generator=gen, dtype=torch.float64)
    else:
        g = torch.randn(count, rows, 1, generator=gen, dtype=torch.float64) @ torch.randn(
            count, 1, cols, generator=gen, dtype=torch.float64)
    return (1e-3 * g).to(dtype(t)).cuda()


@pytest.mark.parametrize("kind", ["noise", "decay", "rank one"])
@pytest.mark.parametrize("t", ["float32", "bfloat16"])
@pytest.mark.parametrize("count,rows,cols", [(1, 128, 128), (3, 64, 256), (2, 300, 130), (1, 513, 1000), (2, 7, 5),
                                             (1, 1, 70), (1, 90, 1), (5, 129, 127), (1, 1100, 400)])
def test_orthogonalize(ops, kind, t, count, rows, cols):
    gen = seeded(count, rows, cols, len(kind))
    g = update(gen, count, rows, cols, kind, t)
    want = orthogonal64(g, 5, [ops.NEWTON_SCHULZ] * 5, 1e-7)
    check_orthogonal(ops.orthogonalize(g), want, 5, "bfloat16")
    out = torch.full((count, rows, cols), math.nan, device="cuda")
    assert ops.orthogonalize(g, out=out) is out
    check_orthogonal(out, want, 5, "float32")


def test_orthogonalize_steps_and_coefficients(ops):
    gen = seeded(40)
    g = update(gen, 2, 200, 310, "noise", "float32")
    cubic, quintic = (1.5, -0.5, 0.0), (3.4445, -4.7750, 2.0315)
    for coef in ([], [quintic], [quintic] * 3 + [cubic] * 5, [(2.0, -1.5, 0.5)] * 12):
        out = torch.empty((2, 200, 310), device="cuda")
        ops.orthogonalize(g, steps=len(coef), coefficients=coef, out=out)
        check_orthogonal(out, orthogonal64(g, len(coef), coef, 1e-7), len(coef), "float32")
    # enough steps bring every singular value to 1
    s = torch.linalg.svdvals(ops.orthogonalize(g, steps=13, coefficients=[quintic] * 5 + [cubic] * 8,
                                               out=torch.empty((2, 200, 310), device="cuda")))
    assert float((s - 1).abs().max()) < 0.01


def test_orthogonalize_strides(ops):
    gen = seeded(41)
    wide = update(gen, 3, 150, 210, "noise", "float32")
    want = ops.orthogonalize(wide[:, :133, 3:100].contiguous())
    assert torch.equal(ops.orthogonalize(wide[:, :133, 3:100]), want)
    turned = wide[:, :133, 3:100].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ops.orthogonalize(turned), want)
    spread = torch.zeros(3, 266, 194, device="cuda")
    spread[:, ::2, ::2] = wide[:, :133, 3:100]
    assert torch.equal(ops.orthogonalize(spread[:, ::2, ::2]), want)
    out = torch.zeros(3, 97, 140, device="cuda", dtype=torch.bfloat16)
    ops.orthogonalize(wide[:, :133, 3:100], out=out[:, :, :133].transpose(1, 2))
    assert torch.equal(out[:, :, :133].transpose(1, 2), want) and not out[:, :, 133:].any()
    assert torch.equal(ops.orthogonalize(wide[1, :133, 3:100]), want[1])
    # one matrix for all of a batch
    same = ops.orthogonalize(wide[:1, :133, 3:100].expand(3, 133, 97))
    assert torch.equal(same[2], want[0])


def test_orthogonalize_zero_nan_and_scale(ops):
    gen = seeded(42)
    g = update(gen, 5, 140, 96, "noise", "float32")
    clean = ops.orthogonalize(g)
    g[1] = 0
    g[2, 5, 7] = math.nan
    g[3, 0, 0] = math.inf
    y = ops.orthogonalize(g)
    assert not y[1].any() and torch.isnan(y[2]).any() and torch.isnan(y[3]).any()
    assert torch.equal(y[0], clean[0]) and torch.equal(y[4], clean[4])
    for big in (1e30, 1e-25):  # squares out of the range of 32 bits
        z = ops.orthogonalize(g[:1] * big, eps=0.0)
        check_orthogonal(z, orthogonal64(g[:1] * big, 5, [ops.NEWTON_SCHULZ] * 5, 0.0), 5, "bfloat16")


def test_orthogonalize_given_workspace_and_repeats(ops):
    gen = seeded(43)
    g = update(gen, 2, 257, 640, "decay", "bfloat16")
    first = ops.orthogonalize(g)
    n = ops.orthogonalize_workspace(2, 257, 640)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(first)
    for _ in range(2):
        ops.orthogonalize(g, out=out, workspace=ws)
        assert torch.equal(out, first)
    assert ops.orthogonalize(g[:0]).shape == (0, 257, 640)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.orthogonalize(g)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, first)


@pytest.mark.parametrize("count,rows,cols", [(6, 1024, 2048), (5, 2100, 1001), (74, 257, 300), (1, 2048, 2040),
                                             (40, 300, 520)])
def test_orthogonalize_large(ops, count, rows, cols):
    """Sizes that each of the tilings is chosen for."""
    gen = seeded(count, rows, cols)
    g = update(gen, count, rows, cols, "decay", "float32")
    g += 1e-5 * torch.randn(g.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    check_orthogonal(ops.orthogonalize(g), orthogonal64(g, 5, [ops.NEWTON_SCHULZ] * 5, 1e-7), 5, "bfloat16")


# ------------------------------------------------------------------ together

def test_language_model_step(ops):
    """The example's gradients against the same model in plain 64-bit torch, and its loss over 40 steps:
    it starts above that of guessing (ln 61 = 4.1) and all but the second token can be foretold."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "lm_step.py")
    spec = importlib.util.spec_from_file_location("lm_step", path)
    lm = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(lm)
    model = lm.Model(vocab=61, width=64, heads=4, hidden=128, layers=2, length=16)
    tokens = torch.randint(0, 61, (5, 16), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    model.loss(tokens).backward()

    def plain(p):  # the parameters in 64 bits
        def norm(v, w):
            return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5) * w

        def turn(v):
            u, w = v[..., :8], v[..., 8:]
            c, s = model.cos.double()[:16, None], model.sin.double()[:16, None]
            return torch.cat((u * c - w * s, w * c + u * s), -1)

        x = p["embedding"][tokens].reshape(80, 64)
        y = norm(x, p["first"])
        for m, v6 in zip(p["matrices"], p["vectors"]):
            q, k, v = (t.reshape(5, 16, 4, 16) for t in (y @ m["qkv"].T).chunk(3, -1))
            s = torch.einsum("bthd,bshd->bhts", turn(q), turn(k)) / 4 + model.mask.double()
            z = torch.einsum("bhts,bshd->bthd", s.softmax(-1), v).reshape(80, 64) @ m["out"].T
            x = x + torch.sigmoid(v6[4]) * norm(z, v6[0])
            y = norm(x, v6[1])
            x = x + torch.sigmoid(v6[5]) * norm(torch.relu(y @ m["up"].T) @ m["down"].T, v6[2])
            y = norm(x, v6[3])
        lp = torch.log_softmax(y @ p["embedding"].T, -1).reshape(5, 16, 61)[:, :-1]
        return -lp.gather(-1, tokens[:, 1:, None]).sum() / 75

    p = dict(embedding=model.embedding, first=model.first, matrices=model.matrices, vectors=model.vectors)
    double = lambda t: t.detach().double().requires_grad_()  # noqa: E731
    p64 = dict(embedding=double(p["embedding"]), first=double(p["first"]),
               matrices=[{k: double(v) for k, v in m.items()} for m in p["matrices"]],
               vectors=[[double(v) for v in layer] for layer in p["vectors"]])
    plain(p64).backward()
    pairs = [(p["embedding"], p64["embedding"]), (p["first"], p64["first"])]
    pairs += [(a[k], b[k]) for a, b in zip(p["matrices"], p64["matrices"]) for k in a]
    pairs += [(a, b) for x, y in zip(p["vectors"], p64["vectors"]) for a, b in zip(x, y)]
    for a, b in pairs:
        # two layers of products and norms in 32 bits: some thousand roundings on the way, norm-wise
        assert float((a.grad.double() - b.grad).norm()) <= 2000 * E * float(b.grad.norm())
    losses = lm.main(40)
    assert losses[0] > 4.0 and losses[-1] < 0.5 * losses[0]


# ------------------------------------------------------------------ far apart and many

def test_offsets_past_32_bits(ops):
    """Rows (tokens, matrices) 2^31 elements apart give the bits of rows side by side."""
    far = 2 ** 31
    store = torch.empty(far + 70000, dtype=torch.bfloat16, device="cuda")
    gen = seeded(77)
    near = rand(gen, (2, 1000), "bfloat16", 2.0)
    x = store.as_strided((2, 1000), (far, 1))
    x.copy_(near)
    tok = torch.tensor([3, 999], device="cuda")
    a, b = ops.token_logprobs(x, tok, top=4), ops.token_logprobs(near, tok, top=4)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    g = torch.ones(2, device="cuda")
    assert torch.equal(ops.token_logprobs_grad(x, tok, a.stats, g), ops.token_logprobs_grad(near, tok, b.stats, g))
    cos, sin = (torch.from_numpy(v).cuda() for v in ops.rotary_table(8, 40))
    q, pos = x.view(1, 2, 1, 1000)[..., :40], torch.tensor([2, 5], device="cuda")
    assert torch.equal(ops.rotary(q, None, cos, sin, pos)[0], ops.rotary(q.contiguous(), None, cos, sin, pos)[0])
    m = store.as_strided((2, 20, 50), (far, 50, 1))
    assert torch.equal(ops.orthogonalize(m), ops.orthogonalize(m.contiguous()))
    rows = store.as_strided((2, 1000), (far - 8, 1))
    rows.copy_(near)
    w = torch.ones(1000, device="cuda")
    h, y, st = ops.block_norm(rows, near, w, w)
    h2, y2, st2 = ops.block_norm(near, near, w, w)
    assert torch.equal(h, h2) and torch.equal(y, y2)
    dg, dg2 = (ops.block_norm_grad(near, near, v, near, w, w, s) for v, s in ((rows, st), (near, st2)))
    assert all(u is None or torch.equal(u, v) for u, v in zip(dg, dg2))


def test_many_short_rows(ops):
    """More rows than a grid's second axis holds."""
    gen = seeded(78)
    logits = rand(gen, (70001, 9), "float32", 2.0)
    tok = torch.randint(-1, 9, (70001,), generator=gen).cuda()
    check_logprobs(ops, logits, tok, 1.0, 2, "float32", torch.ones(70001, device="cuda"), torch.ones(70001, device="cuda"))
    d = block_operands(ops, 70002, 8, "float32", "float32", "rms", "many")
    check_block(ops, d, "float32", "float32", "rms", False, 1.0)
    cos, sin = (torch.from_numpy(v).cuda() for v in ops.rotary_table(4, 4))
    q = rand(gen, (70001, 1, 1, 4), "float16")
    pos = torch.randint(0, 4, (70001, 1), generator=gen)
    y, _ = ops.rotary(q, None, cos, sin, pos.cuda())
    want, mag = rotary64(q.cpu(), cos.cpu(), sin.cpu(), pos, 2, "half", False)
    within(y.cpu(), want, mag, 3, "float16")
