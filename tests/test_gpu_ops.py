"""The operators on device tensors (vadc_amd/ops.py) against their definitions in float64, on the device.

Tolerances.  u = 2^-24 is half a float32 step, eps / 2 half a step of the output's type; a sum of n products in float32, in any order, is off by at most (n + 1) u sum |products|.
An activation here changes by at most 1.13 times its argument's change (gelu) and is itself good to a few float32 steps."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTS = ("none", "relu", "silu", "gelu", "sigmoid")


@pytest.fixture(scope="module")
def ops():
    from vadc_amd import ops
    return ops


def gen(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=g, device="cuda")


def act64(y, name):
    return {"none": lambda a: a, "relu": torch.relu, "silu": lambda a: a * torch.sigmoid(a), "gelu": lambda a: a * torch.special.ndtr(a), "sigmoid": torch.sigmoid}[name](y)


def half_step(y, dtype):
    """half a step of `dtype` at y: relative, or half of its smallest number (fp16's subnormals)"""
    return y.abs() * (torch.finfo(dtype).eps / 2) + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def within(got, want, tol):
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got.double()), torch.isnan(want))
    off = (got.double() - want).abs()
    bad = (off > tol) & torch.isfinite(want)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, the worst by {(off / tol)[bad].max().item():.3g} times its tolerance"


# ---------------------------------------------------------------------------------------------------------------- linear

def linear64(x, w, b, act, r, first):
    y = x.double() @ w.double().T
    if b is not None:
        y = y + b.double()
    if r is not None and first:
        y = y + r.double()
    y = act64(y, act)
    return y + r.double() if r is not None and not first else y


def linear_tol(x, w, b, r, want, dtype):
    mass = x.double().abs() @ w.double().abs().T
    for t in (b, r):
        if t is not None:
            mass = mass + t.double().abs()
    # K products, bias, residual (two sums); operands in three bfloat16 parts (float32 inputs) leave at most 3 u of a product out; the activation: 8 u of its value and of 1
    return 1.13 * (x.shape[-1] + 8) * U * mass + 8 * U * (want.abs() + 1) + half_step(want, dtype)


LINEAR_SIZES = [(1, 1, 1), (2, 3, 5), (1, 64, 64), (1, 2048, 130), (7, 1000, 33), (16, 512, 512), (17, 100, 33), (33, 264, 1), (64, 128, 512), (65, 129, 257), (130, 72, 200), (128, 256, 256),
                (257, 520, 514), (300, 63, 128), (1111, 40, 72), (600, 1032, 640), (513, 4096, 130)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, k, n", LINEAR_SIZES)
def test_linear(ops, m, k, n, dtype):
    dt, rnd = TYPES[dtype], gen(m * 7919 + k * 31 + n)
    i = m + k + n
    act, mode = ACTS[i % 5], ("none", "after", "before")[i % 3]
    x, w = rnd(m, k).to(dt), (rnd(n, k) * k ** -0.5).to(dt)
    b = rnd(n).to(dt) if i % 4 else None
    r = rnd(m, n).to(dt) if mode != "none" else None
    got = ops.linear(x, w, bias=b, activation=act, residual=r, residual_first=mode == "before")
    want = linear64(x, w, b, act, r, mode == "before")
    within(got, want, linear_tol(x, w, b, r, want, dt))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, k, n", [(100, 640, 70), (100, 513, 70), (90, 1153, 200), (1700, 200, 1800), (1700, 201, 1800), (3000, 200, 4000), (3000, 65, 4000), (8200, 129, 4100), (8200, 136, 4100)])
def test_linear_several_tiles_a_workgroup(ops, m, k, n, dtype):
    """more tiles than workgroups, groups of waves with unequal shares of k; odd k: rows at every alignment"""
    dt, rnd = TYPES[dtype], gen(m + k)
    x, w, b = rnd(m, k).to(dt), (rnd(n, k) * k ** -0.5).to(dt), rnd(n).to(dt)
    want = linear64(x, w, b, "relu", None, False)
    within(ops.linear(x, w, bias=b, activation="relu"), want, linear_tol(x, w, b, None, want, dt))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, k, n", [(100, 131, 70), (300, 515, 140), (2000, 67, 3000), (9000, 65, 4000)])
def test_linear_part_of_a_piece(ops, m, k, n, dtype):
    """16-byte aligned rows that end inside 16 bytes; what lies behind their ends is NaN"""
    dt, rnd = TYPES[dtype], gen(m + k)
    x, w = torch.full((m, k + 8 - k % 8), math.nan, dtype=dt, device="cuda"), torch.full((n, k + 16 - k % 8), math.nan, dtype=dt, device="cuda")
    x[:, :k], w[:, :k] = rnd(m, k).to(dt), (rnd(n, k) * k ** -0.5).to(dt)
    x, w = x[:, :k], w[:, :k]
    want = linear64(x, w, None, "none", None, False)
    within(ops.linear(x, w), want, linear_tol(x, w, None, None, want, dt))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset, gap", [(0, 0), (1, 0), (1, 2), (3, 1), (0, 1), (2, 2)])
@pytest.mark.parametrize("m, n", [(1, 37), (16, 16), (17, 90), (32, 33), (33, 70), (64, 129), (65, 20), (1025, 1900)])
def test_linear_any_alignment(ops, m, n, offset, gap, dtype):
    """rows that begin and end anywhere, k's from one up; what lies around them is NaN"""
    dt, rnd = TYPES[dtype], gen(m + n)
    for k in (1, 3, 7, 8, 9, 15, 17, 63, 64, 65, 127, 129) if m > 1000 else (1, 2, 5, 7, 8, 9, 16, 31, 63, 64, 65, 127, 128, 129, 511, 513, 575, 577, 1031, 1217):
        x, w = (torch.full((offset + r * (k + gap),), math.nan, dtype=dt, device="cuda")[offset:].view(r, k + gap)[:, :k] for r in (m, n))
        x.copy_(rnd(m, k))
        w.copy_(rnd(n, k) * k ** -0.5)
        want = linear64(x, w, None, "none", None, False)
        within(ops.linear(x, w), want, linear_tol(x, w, None, None, want, dt))


def test_linear_rows_far_apart(ops):
    """rows further apart than 32-bit offsets within a tile reach"""
    m, n, k, rnd = 70, 200, 131, gen(5)
    x = torch.empty(m, 4_200_001, dtype=torch.bfloat16, device="cuda")[:, :k]
    x.copy_(rnd(m, k))
    w = rnd(n, k).bfloat16()
    want = linear64(x, w, None, "none", None, False)
    within(ops.linear(x, w), want, linear_tol(x, w, None, None, want, torch.bfloat16))
    want = linear64(w, x, None, "none", None, False)
    within(ops.linear(w, x), want, linear_tol(w, x, None, None, want, torch.bfloat16))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("mode", ("none", "after", "before"))
@pytest.mark.parametrize("m", (3, 40, 300))
def test_linear_epilogues(ops, m, mode, act):
    rnd = gen(m)
    x, w, b, r = rnd(m, 96).bfloat16(), rnd(136, 96).bfloat16() * 0.3, rnd(136).bfloat16(), rnd(m, 136).bfloat16()
    r = None if mode == "none" else r
    got = ops.linear(x, w, bias=b, activation=act, residual=r, residual_first=mode == "before")
    want = linear64(x, w, b, act, r, mode == "before")
    within(got, want, linear_tol(x, w, b, r, want, torch.bfloat16))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, k, n, off", [(5, 64, 40, 1), (200, 128, 96, 1), (200, 128, 96, 4), (1, 256, 64, 3), (140, 131, 67, 0)])
def test_linear_strides(ops, m, k, n, off, dtype):
    """rows inside wider tensors, at addresses that are aligned to the element only; what lies between the rows of the output stays"""
    dt, rnd = TYPES[dtype], gen(k + off)
    x, w, r = rnd(m, k + 9).to(dt)[:, off:off + k], rnd(n, k + 5).to(dt)[:, off:off + k], rnd(m, n + 3).to(dt)[:, off % 3:off % 3 + n]
    wide = torch.full((m, n + 7), 77.0, dtype=dt, device="cuda")
    out = wide[:, off:off + n]
    assert ops.linear(x, w, residual=r, out=out) is out
    want = linear64(x, w, None, "none", r, False)
    within(out, want, linear_tol(x, w, None, r, want, dt))
    wide[:, off:off + n] = 77.0
    assert (wide == 77.0).all()


def test_linear_leading_dimensions_in_place_and_empty(ops):
    rnd = gen(5)
    x, w, b = rnd(3, 4, 24), rnd(8, 24), rnd(8)
    want = linear64(x, w, b, "none", None, False)
    tol = linear_tol(x, w, b, None, want, torch.float32)
    within(ops.linear(x, w, bias=b), want, tol)
    within(ops.linear(x[0, 0], w, bias=b), want[0, 0], tol[0, 0])
    r = rnd(3, 4, 8)
    want2 = linear64(x, w, b, "silu", r, False)
    assert ops.linear(x, w, bias=b, activation="silu", residual=r, out=r) is r                    # the residual stream, in place
    within(r, want2, linear_tol(x, w, b, r, want2, torch.float32) + 8 * U * tol)
    assert ops.linear(x[:0], w).shape == (0, 4, 8) and ops.linear(x, w[:0]).shape == (3, 4, 0)
    assert torch.equal(ops.linear(x[..., :0], w[:, :0], bias=b), b.expand(3, 4, 8))               # a sum of nothing
    with pytest.raises(ValueError, match="overlaps"):
        ops.linear(x[..., :8], w[:, :8], out=x[..., 4:12])
    with pytest.raises(ValueError, match="rows"):
        ops.linear(rnd(6, 5, 24)[:, :4][::2], w, out=torch.empty(3, 4, 8, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", (2, 70, 200))
def test_linear_infinities_and_nan(ops, m, dtype):
    """an infinity or NaN reaches the outputs that its row or feature makes, as in the definition, and no other"""
    dt, rnd = TYPES[dtype], gen(m)
    x, w = rnd(m, 128).to(dt), rnd(80, 128).to(dt)
    x[0, 3], x[1, 64] = math.inf, math.nan
    w[7, 5] = -math.inf
    got, want = ops.linear(x, w).double(), linear64(x, w, None, "none", None, False)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    ok = torch.isfinite(want)
    x[0, 3] = x[1, 64] = w[7, 5] = 0
    within(torch.where(ok, got, 0.0), torch.where(ok, want, 0.0), linear_tol(x, w, None, None, want, dt).nan_to_num(1e300, 1e300, 1e300))


def test_linear_float32_range(ops):
    """float32 operands near the ends of their range: products that fit are right, also where a factor is over bfloat16's largest rounded-to-nearest value"""
    x = torch.full((150, 64), 3.4e38, device="cuda")
    w = torch.full((96, 64), 2.0 ** -30, device="cuda")
    want = linear64(x, w, None, "none", None, False)
    within(ops.linear(x, w), want, linear_tol(x, w, None, None, want, torch.float32))
    x = torch.full((150, 64), 2.0 ** -60 * 1.2345678, device="cuda")
    want = linear64(x, w, None, "none", None, False)
    within(ops.linear(x, w), want, 1.13 * 72 * U * want.abs() + 2.0 ** -24 * want.abs())


# ------------------------------------------------------------------------------------------------------------ group norm

def norm64(x, groups, w, b, eps, act, gate, lengths):
    n, l, c = x.shape
    out = torch.zeros(n, l, c, dtype=torch.float64, device="cuda")
    spread = torch.zeros_like(out)
    for i in range(n) if l > 1 else (slice(0, n),):
        j = slice(i, i + 1) if l > 1 else i
        live = l if lengths is None or l == 1 else max(0, min(l, int(lengths[i])))
        if not live:
            continue
        v = x[j, :live].double().unflatten(2, (groups, c // groups))
        mean, var = v.mean(dim=(1, 3), keepdim=True), v.var(dim=(1, 3), keepdim=True, correction=0)
        r = 1 / (var + eps).sqrt()
        y, s = ((v - mean) * r).flatten(2), ((v - mean).abs() * r + v.abs().amax(dim=(1, 3), keepdim=True) * r).flatten(2)
        if w is not None:
            y, s = y * w.double(), s * w.double().abs()
        if b is not None:
            y = y + b.double()
        out[j, :live], spread[j, :live] = y, s
    g = act64(gate.double(), act) if gate is not None else 1.0
    want = out * g if gate is not None else act64(out, act)
    return want, spread * (g.abs() if gate is not None else 1.13), out


def norm_tol(want, spread, dtype, chain):
    """mean and variance come out of a chain of at most `chain` merges of sets, each good to 4 u of the largest value (mean) and of itself (variance); y's own steps: 8 u"""
    return (4 * chain + 8) * U * spread + 12 * U * (want.abs() + 1) + half_step(want, dtype)


NORM_SIZES = [(1, 1, 1, 1), (1, 1, 8, 8), (5, 1, 12, 3), (3, 1, 2048, 16), (70, 1, 384, 12), (9, 1, 4096, 1), (2, 1, 20000, 4), (33, 1, 130, 10), (2, 7, 6, 2), (3, 50, 64, 8), (2, 333, 384, 12),
              (1, 2049, 20, 4), (4, 1000, 32, 32), (1, 5000, 8, 1), (2, 64, 1032, 1), (3, 3, 7, 1), (1, 20011, 24, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, l, c, groups", NORM_SIZES)
def test_group_norm(ops, n, l, c, groups, dtype):
    dt, rnd = TYPES[dtype], gen(n + l + c)
    i = n + l + c
    x = (rnd(n, l, c) * (1 + rnd(c).abs()) + 3 * rnd(c)).to(dt)
    w, b = (rnd(c).to(dt) if i % 3 else None), (rnd(c).to(dt) if i % 4 else None)
    gate = rnd(n, l, c).to(dt) if i % 2 else None
    act = ACTS[i % 5]
    want, spread, _ = norm64(x, groups, w, b, 1e-5, act, gate, None)
    chain = l * (c // groups) // 256 + 24
    within(ops.group_norm(x, groups, weight=w, bias=b, activation=act, gate=gate), want, norm_tol(want, spread, dt, chain))
    if l == 1:
        g2 = None if gate is None else gate[:, 0]
        within(ops.group_norm(x[:, 0], groups, weight=w, bias=b, activation=act, gate=g2), want[:, 0], norm_tol(want, spread, dt, chain)[:, 0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("l, c, groups", [(40, 24, 3), (700, 64, 4), (5000, 40, 1), (1, 48, 6)])
def test_group_norm_lengths_and_strides(ops, l, c, groups, dtype):
    """sequences of none, one, some and all positions inside wider tensors; NaN behind them is not read, and the output's rows behind them stay"""
    dt, rnd = TYPES[dtype], gen(l)
    lengths = torch.tensor([l, 0, 1, l // 2 + 1, -3, l + 100], dtype=torch.int32, device="cuda")
    n = len(lengths)
    x = (rnd(n, l + 2, c + 5) + 1).to(dt)[:, 1:l + 1, 3:c + 3]
    gate = rnd(n, l, c + 1).to(dt)[:, :, 1:]
    w, b = rnd(c).to(dt), rnd(c).to(dt)
    live = torch.arange(l, device="cuda")[None] < lengths[:, None]
    x[~live], gate[~live] = math.nan, math.nan
    for kw in (dict(gate=gate, activation="silu"), dict(activation="relu")):
        wide = torch.full((n, l, c + 3), 55.0, dtype=dt, device="cuda")
        out = ops.group_norm(x, groups, weight=w, bias=b, lengths=lengths, out=wide[:, :, 2:c + 2], **kw)
        seq = norm64(x, groups, w, b, 1e-5, kw["activation"], kw.get("gate"), lengths) if l > 1 else norm64(x.nan_to_num(), groups, w, b, 1e-5, kw["activation"], kw["gate"].nan_to_num() if "gate" in kw else None, None)
        want, spread, _ = seq
        within(out[live], want[live], norm_tol(want, spread, dt, l * (c // groups) // 256 + 24)[live])
        out[live] = 55.0
        assert (wide == 55.0).all()
        fresh = ops.group_norm(x, groups, weight=w, bias=b, lengths=lengths, **kw)
        assert (fresh[~live] == 0).all() and not torch.isnan(fresh).any()


def test_group_norm_far_mean_constant_and_in_place(ops):
    rnd = gen(3)
    x = rnd(2, 3000, 16) * 0.01 + 1000                               # the mean is 1e5 deviations from zero: no digits of the variance may go
    want, _, _ = norm64(x, 2, None, None, 1e-5, "none", None, None)
    chain = 3000 * 8 // 256 + 24
    # rounding of a deviation from the mean: the mean is off by 4 u chain / sqrt-free worst case of 1000, over a spread of 0.01
    within(ops.group_norm(x, 2), want, torch.full_like(want, 4 * chain * U * 1000 / 0.01 + 1e-5))
    off = (ops.group_norm(x, 2).double() - want).norm() / want.norm()
    assert off < 2 * 1000 * U / 0.01, off                            # one rounding of the mean, as a rule
    flat = torch.full((2, 40, 12), 3.25, device="cuda")
    assert torch.equal(ops.group_norm(flat, 3), torch.zeros_like(flat))
    for shape in ((40, 64), (3, 500, 64)):
        y, gate = rnd(*shape), rnd(*shape)
        want = ops.group_norm(y, 4, gate=gate, activation="silu")
        first, second = y.clone(), gate.clone()
        assert torch.equal(ops.group_norm(first, 4, gate=gate, activation="silu", out=first), want)
        assert torch.equal(ops.group_norm(y, 4, gate=second, activation="silu", out=second), want)
    bad = rnd(3, 50, 8)
    bad[1, 7, 5] = math.inf
    got = ops.group_norm(bad, 2)
    assert torch.isnan(got[1, :, 4:]).all() and torch.isfinite(got[1, :, :4]).all() and torch.isfinite(got[[0, 2]]).all()


# ----------------------------------------------------------------------------------------------------------- gated delta

def delta64(q, k, v, g, beta, state, scale, normalize, lengths):
    b, t, hk, dk = q.shape
    h = v.shape[2]
    S, out = state.double().clone(), torch.zeros(v.shape, dtype=torch.float64, device="cuda")
    most = S.norm(dim=2).amax(-1)                                    # the largest column of each state so far
    q, k = q.double(), k.double()
    if normalize:
        q, k = (a / (a.square().sum(-1, keepdim=True) + 1e-6).sqrt() for a in (q, k))
    q, k = (a.repeat_interleave(h // hk, dim=2) for a in (q, k))
    for i in range(t):
        live = torch.ones(b, dtype=torch.bool, device="cuda") if lengths is None else i < lengths
        d = S * g[:, i].double().exp()[..., None, None]
        u = beta[:, i].double()[..., None] * (v[:, i].double() - (d * k[:, i, :, :, None]).sum(2))
        d = d + k[:, i, :, :, None] * u[:, :, None]
        S = torch.where(live[:, None, None, None], d, S)
        out[:, i] = torch.where(live[:, None, None], scale * (S * q[:, i, :, :, None]).sum(2), 0.0)
        most = torch.maximum(most, torch.where(live[:, None], S.norm(dim=2).amax(-1) + v[:, i].double().abs().amax(-1), most))
    return out, S, most


def delta_tol(out, most, t, dk, scale, q_norm, dtype):
    """With |k| <= 1, 0 <= beta <= 1 and decay <= 1 a step is a contraction, so errors add: a step rounds sums of dk products and a handful of factors, a block of 64 steps also sums of
    64 products, twice (the triangular inverse, whose entries are at most 1): (dk + 160) u of the largest column and value a step, on the state and on u."""
    state = 2 * (dk + 160) * t * U * most[..., None, None]
    o = abs(scale) * q_norm * (state[..., 0] + (dk + 160) * U * most[..., None])
    return half_step(out, dtype) + o[:, None], state


def delta_inputs(seed, b, t, hk, h, dk, dv, dt, normalize):
    rnd = gen(seed)
    q, k, v = rnd(b, t, hk, dk), rnd(b, t, hk, dk), rnd(b, t, h, dv)
    if not normalize:
        q, k = (a / (a.norm(dim=-1, keepdim=True) * 1.02) for a in (q, k))
    g = -torch.nn.functional.softplus(rnd(b, t, h)) * torch.exp(2 * rnd(h) - 2)
    return q.to(dt), k.to(dt), v.to(dt), g, torch.sigmoid(rnd(b, t, h)), rnd(b, h, dk, dv)


def check_delta(ops, q, k, v, g, beta, state, normalize, lengths=None, scale=None, out=None):
    b, t, hk, dk = q.shape
    s = dk ** -0.5 if scale is None else scale
    mine = state.clone()
    got = ops.gated_delta(q, k, v, g, beta, mine, scale=scale, normalize=normalize, lengths=lengths, out=out)
    clean = [a if lengths is None else a.nan_to_num() for a in (q, k, v, g, beta)]
    want, S, most = delta64(*clean, state, s, normalize, lengths)
    q_norm = 1.0 if normalize else clean[0].double().norm(dim=-1).max().item()
    tol_o, tol_s = delta_tol(want, most, t, dk, s, q_norm, v.dtype)
    live = torch.ones(b, t, dtype=torch.bool, device="cuda") if lengths is None else torch.arange(t, device="cuda")[None] < lengths[:, None]
    within(got[live], want[live], tol_o.expand_as(want)[live])
    within(mine, S, tol_s.expand_as(S))
    # far inside the worst case, as sums of independent roundings are
    assert (mine.double() - S).norm() <= 3e-6 * S.norm() + 1e-30
    return got, mine


DELTA_SIZES = [(1, 1, 1, 1, 1, 1), (3, 1, 2, 4, 64, 64), (2, 1, 1, 3, 48, 80), (2, 2, 1, 1, 128, 128), (1, 5, 1, 2, 33, 17), (2, 17, 2, 2, 64, 64), (1, 64, 1, 1, 64, 64), (2, 65, 1, 2, 128, 64),
               (1, 130, 3, 6, 48, 80), (2, 200, 1, 1, 24, 37), (1, 257, 2, 2, 128, 128), (1, 70, 1, 1, 200, 40), (1, 127, 1, 4, 256, 16), (1, 300, 1, 1, 100, 128), (5, 128, 1, 1, 8, 8), (1, 1000, 1, 1, 64, 32)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("normalize", (True, False))
@pytest.mark.parametrize("b, t, hk, h, dk, dv", DELTA_SIZES)
def test_gated_delta(ops, b, t, hk, h, dk, dv, normalize, dtype):
    check_delta(ops, *delta_inputs(t + dk, b, t, hk, h, dk, dv, TYPES[dtype], normalize), normalize, scale=None if t % 2 else 0.7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t, dk, dv", [(1, 32, 32), (9, 20, 12), (150, 64, 64), (130, 48, 80)])
def test_gated_delta_lengths_and_strides(ops, t, dk, dv, dtype):
    """streams of none, one, some and all steps; q, k, v as slices of one projection, states inside a wider pool; NaN behind a stream's steps is not read, nothing behind them is written"""
    dt, b, hk, h = TYPES[dtype], 6, 2, 4
    lengths = torch.tensor([t, 0, 1, t // 2 + 1, -1, t + 9], dtype=torch.int32, device="cuda")
    q, k, v, g, beta, state = delta_inputs(t, b, t, hk, h, dk, dv, dt, True)
    live = torch.arange(t, device="cuda")[None] < lengths[:, None]
    for a in (q, k, v, g, beta):
        a[~live] = math.nan
    both = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2), v.flatten(2)[..., :3]], dim=2)
    q2, k2, v2 = (both[..., lo:lo + heads * d].unflatten(2, (heads, d)) for lo, heads, d in ((0, hk, dk), (hk * dk, hk, dk), (2 * hk * dk, h, dv)))
    wide = torch.full((b, t, h, dv + 2), 9.0, dtype=dt, device="cuda")
    gb = torch.cat([g, beta], dim=2)
    got, mine = check_delta(ops, q2, k2, v2, gb[..., :h], gb[..., h:], state, True, lengths=lengths, out=wide[..., 1:dv + 1])
    assert torch.equal(mine[1], state[1]) and torch.equal(mine[4], state[4])
    plain_state = state.clone()
    fresh = ops.gated_delta(q, k, v, g, beta, plain_state, normalize=True, lengths=lengths)
    assert torch.equal(fresh[live], got[live]) and (fresh[~live] == 0).all() and torch.equal(plain_state, mine)
    got[live] = 9.0
    assert (wide == 9.0).all()
    pool = torch.full((b, h + 1, dk, dv), 4.0, device="cuda")
    pool[:, :h] = state
    ops.gated_delta(q, k, v, g, beta, pool[:, :h], normalize=True, lengths=lengths)
    assert torch.equal(pool[:, :h], mine) and (pool[:, h] == 4.0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_delta_steps_and_blocks_agree(ops, dtype):
    """one call over all steps, calls of unequal numbers of steps, and one call per step: the state carries on"""
    q, k, v, g, beta, state = delta_inputs(11, 3, 150, 1, 2, 64, 48, TYPES[dtype], True)
    want, S, most = delta64(q, k, v, g, beta, state, 0.125, True, None)
    tol_o, tol_s = delta_tol(want, most, 150, 64, 0.125, 1.0, TYPES[dtype])
    for cuts in ([0, 150], [0, 64, 65, 130, 150], list(range(151))):
        s, outs = state.clone(), []
        for lo, hi in zip(cuts, cuts[1:]):
            outs.append(ops.gated_delta(*(a[:, lo:hi] for a in (q, k, v, g, beta)), s, normalize=True))
        within(torch.cat(outs, 1), want, tol_o.expand_as(want))
        within(s, S, tol_s.expand_as(S))


@pytest.mark.parametrize("t", (1, 3, 100))
def test_gated_delta_extreme_gates(ops, t):
    """decays of 0 and of e^-inf, gates of 0 and 1, keys of zero: exact where the formula is"""
    q, k, v, g, beta, state = delta_inputs(2, 2, t, 1, 2, 32, 32, torch.float32, True)
    zero = torch.zeros_like(beta)
    s = state.clone()
    ops.gated_delta(q, k, v, zero, zero, s, normalize=True)          # nothing decays, nothing is written
    assert torch.equal(s, state)
    g2, s = zero.clone(), state.clone()
    g2[:, t // 2] = -math.inf                                        # all that came before is forgotten
    check_delta(ops, q, k, v, g2, beta, state, True)
    g2[:, t // 2], g2[:, -1] = -1e30, -88.0
    check_delta(ops, q, k, v, g2, beta, state, True)
    check_delta(ops, q, torch.zeros_like(k), v, g, beta, state, True)
    check_delta(ops, q, k, v, -20 * torch.ones_like(g), torch.ones_like(beta), state, True)
    # one direction again and again, at full strength: the triangular inverse at its worst
    one = k[:, :1].expand_as(k).contiguous()
    check_delta(ops, q, one, v, zero, torch.ones_like(beta), state, True)


def test_gated_delta_nan_stays_in_its_stream_and_head(ops):
    q, k, v, g, beta, state = delta_inputs(4, 3, 90, 2, 2, 64, 32, torch.bfloat16, True)
    want, S, _ = delta64(q, k, v, g, beta, state, 0.125, True, None)
    v[1, 40, 1, 5], state[2, 0, 3, 7] = math.nan, math.inf
    got = ops.gated_delta(q, k, v, g, beta, state, normalize=True)
    ok = torch.ones(3, 2, dtype=torch.bool)
    ok[1, 1] = ok[2, 0] = False
    assert torch.isfinite(got.transpose(1, 2)[ok]).all() and torch.isfinite(state[ok]).all()
    assert torch.isnan(state[1, 1, :, 5]).all() and torch.isnan(got[1, 89, 1, 5])
    assert torch.isfinite(got[1, :40, 1]).all()


# -------------------------------------------------------------------------------------------------------------- together

class Layer:
    """a streaming layer: x + out(norm(delta(project(x)))), its state carried from call to call"""

    def __init__(self, ops, dt, width=192, heads=4, dk=32, dv=48, streams=5):
        rnd = gen(21)
        self.ops, self.heads, self.dk, self.dv = ops, heads, dk, dv
        self.sizes = (heads // 2 * dk, heads // 2 * dk, heads * dv)
        self.w_in = (rnd(sum(self.sizes), width) * width ** -0.5).to(dt)
        self.w_gate, self.b_gate = (rnd(heads * dv, width) * width ** -0.5).to(dt), rnd(heads * dv).to(dt) * 0.1
        self.w_beta = (rnd(heads, width) * width ** -0.5).to(dt)
        self.w_out = (rnd(width, heads * dv) * (heads * dv) ** -0.5).to(dt)
        self.norm = (1 + 0.1 * rnd(heads * dv)).to(dt)
        self.state = torch.zeros(streams, heads, dk, dv, device="cuda")

    def __call__(self, x):
        ops, h = self.ops, self.heads
        q, k, v = ops.linear(x, self.w_in, activation="silu").split(self.sizes, dim=-1)
        beta = ops.linear(x, self.w_beta, activation="sigmoid").float()
        gate = ops.linear(x, self.w_gate, bias=self.b_gate)
        o = ops.gated_delta(q.unflatten(2, (h // 2, self.dk)), k.unflatten(2, (h // 2, self.dk)), v.unflatten(2, (h, self.dv)), -0.2 * beta, beta, self.state, normalize=True)
        o = ops.group_norm(o.reshape(-1, h * self.dv), h, weight=self.norm, gate=gate.reshape(-1, h * self.dv), activation="silu")
        return ops.linear(o.reshape(x.shape[0], x.shape[1], -1), self.w_out, residual=x)

    def definition(self, x):
        """the same in float64, each tensor between two operators rounded as the layer rounds it"""
        dt, h, b, t = x.dtype, self.heads, x.shape[0], x.shape[1]
        cast = lambda a: a.to(dt)  # noqa: E731
        q, k, v = cast(linear64(x, self.w_in, None, "silu", None, False)).split(self.sizes, dim=-1)
        beta = cast(linear64(x, self.w_beta, None, "sigmoid", None, False)).float()
        gate = cast(linear64(x, self.w_gate, self.b_gate, "none", None, False))
        o, S, _ = delta64(q.unflatten(2, (h // 2, self.dk)), k.unflatten(2, (h // 2, self.dk)), v.unflatten(2, (h, self.dv)), -0.2 * beta, beta, torch.zeros_like(self.state), self.dk ** -0.5, True, None)
        o, _, _ = norm64(cast(o).reshape(b * t, 1, -1), h, self.norm, None, 1e-5, "silu", gate.reshape(b * t, 1, -1), None)
        return linear64(cast(o).reshape(b, t, -1), self.w_out, None, "none", x, False), S


@pytest.mark.parametrize("dtype", TYPES)
def test_streaming_layer(ops, dtype):
    """the operators as they are used together: all steps in one call, and one call per step, give the definition's outputs and state"""
    dt = TYPES[dtype]
    x = gen(8)(5, 140, 192).to(dt)
    layer = Layer(ops, dt)
    want, S = layer.definition(x)
    # four roundings of dt lie between x and the output, each of a value near 1 in size that later products average: 8 half steps of the output's scale
    tol = 8 * torch.finfo(dt).eps / 2 * want.abs().amax() + 2e-5
    within(layer(x), want, tol.expand_as(want))
    assert (layer.state.double() - S).norm() <= (torch.finfo(dt).eps + 1e-5) * S.norm()
    layer.state.zero_()
    steps = torch.cat([layer(x[:, i:i + 1].contiguous()) for i in range(140)], 1)
    within(steps, want, tol.expand_as(want))
    assert (layer.state.double() - S).norm() <= (torch.finfo(dt).eps + 1e-5) * S.norm()


@pytest.mark.parametrize("t", (1, 100))
def test_captured_and_replayed(ops, t):
    """a layer captured into a graph: each replay is the eager call's result, bit for bit, with eager work in between; a second graph of the same layer keeps to its own workspace"""
    layer = Layer(ops, torch.bfloat16)
    xs = [gen(30 + i)(5, t, 192).bfloat16() for i in range(4)]
    x = xs[0].clone()
    layer(x)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = layer(x)
        graphs.append((g, y))
    for i in range(8):
        before = torch.randn_like(layer.state)
        layer.state.copy_(before)
        x.copy_(xs[i % 4])
        want = layer(x)
        end = layer.state.clone()
        layer.state.copy_(before)
        g, y = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(layer.state, end), i


def test_norm_long_captured(ops):
    rnd = gen(6)
    x = rnd(2, 9000, 64)
    lengths = torch.tensor([9000, 4001], dtype=torch.int32, device="cuda")
    ops.group_norm(x, 8, lengths=lengths)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.group_norm(x, 8, lengths=lengths)
    for i in range(4):
        x.copy_(rnd(2, 9000, 64))
        want = ops.group_norm(x, 8, lengths=lengths)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), i


def test_streams_at_once_and_the_same_bits_twice(ops):
    """calls on two streams of the caller at the same time, and a call again: the same bits"""
    q, k, v, g, beta, state = delta_inputs(9, 4, 300, 2, 4, 64, 64, torch.bfloat16, True)
    x, w = gen(2)(700, 512).bfloat16(), gen(3)(384, 512).bfloat16()
    z = gen(4)(3, 3000, 96)

    def work():
        s = state.clone()
        return ops.gated_delta(q, k, v, g, beta, s, normalize=True), s, ops.linear(x, w, activation="gelu"), ops.group_norm(z, 4)

    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(work())
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_an_engine_runs_beside_the_operators(ops, weights_blob):
    """an engine's probabilities are the same bits with the operators' work on the device at the same time"""
    import numpy as np
    from vadc_amd import synth
    from vadc_amd.engine import Engine

    pcm = synth.make_streams(32, 6, seed0=4)
    eng = Engine(weights_blob, max_streams=32, max_chunks_per_call=6, device=0)
    want = eng.run(pcm)
    layer, x = Layer(ops, torch.bfloat16), gen(1)(5, 64, 192).bfloat16()
    first = layer(x)
    for _ in range(3):
        eng.reset_streams()
        for _ in range(20):
            layer(x)
        assert np.array_equal(eng.run(pcm), want)
    layer.state.zero_()
    assert torch.equal(layer(x), first)
    eng.close()


def test_long_offsets(ops):
    """element offsets over 2^31: the last rows of a tensor of 5 GB"""
    rows, wide = 70000, 40000
    x = torch.empty(rows, wide, dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 2 ** 31
    x[-3:, :64] = gen(5)(3, 64).bfloat16()
    w = gen(6)(32, 64).bfloat16()
    want = linear64(x[-3:, :64], w, None, "none", None, False)
    tol = linear_tol(x[-3:, :64], w, None, None, want, torch.bfloat16)
    x[:-3, :64] = 0
    got = ops.linear(x[:, :64], w)
    within(got[-3:], want, tol)
    assert (got[:-3] == 0).all()
    out = torch.empty(rows, wide, dtype=torch.bfloat16, device="cuda")
    y = ops.group_norm(x[:, :64], 2, out=out[:, :64])
    nw, spread, _ = norm64(x[-3:, None, :64], 2, None, None, 1e-5, "none", None, None)
    within(y[-3:], nw[:, 0], norm_tol(nw, spread, torch.bfloat16, 24)[:, 0])
    q = x[None, -70:, :32].unflatten(2, (1, 32))
    k = x[None, -70:, 32:64].unflatten(2, (1, 32))
    v = x.view(1, rows, 1, wide)[:, -70:, :, :48]
    v.copy_(gen(7)(1, 70, 1, 48))
    state = gen(8)(1, 1, 32, 48)
    check_delta(ops, q, k, v, torch.full((1, 70, 1), -0.1, device="cuda"), torch.full((1, 70, 1), 0.5, device="cuda"), state, True)


def test_slices_of_a_long_call(ops):
    """more streams, sequences or rows than one launch takes: the last, short slice takes the form of the others (on its own it would choose another, whose workspace nobody gave)"""
    for t in (1, 12, 30):
        q, k, v, g, beta, state = delta_inputs(t, 2049, t, 1, 4, 8, 12, torch.float32, True)
        check_delta(ops, q, k, v, g, beta, state, True)
    x = torch.empty(4097, 64, 1024, dtype=torch.bfloat16, device="cuda")
    x.copy_(gen(1)(1, 64, 1024) + torch.arange(4097, device="cuda")[:, None, None] % 5)
    got = ops.group_norm(x, 1024)
    for rows in (slice(0, 3), slice(4094, 4097)):
        want, spread, _ = norm64(x[rows], 1024, None, None, 1e-5, "none", None, None)
        within(got[rows], want, norm_tol(want, spread, torch.bfloat16, 64))
    del x, got
    x, w = gen(2)(70001, 8).half(), gen(3)(1024, 8).half()
    want = linear64(x, w, None, "none", None, False)
    within(ops.linear(x, w), want, linear_tol(x, w, None, None, want, torch.float16))


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_of_no_features(ops, dtype):
    """a sum of nothing, in every form"""
    dt, b = TYPES[dtype], gen(1)(200).to(TYPES[dtype])
    for m in (1, 40, 300, 20000):
        x = torch.empty(m, 0, dtype=dt, device="cuda")
        assert torch.equal(ops.linear(x, torch.empty(200, 0, dtype=dt, device="cuda"), bias=b), b.expand(m, 200))


def test_broadcast_inputs(ops):
    """rows, heads and streams that are one piece of memory"""
    rnd = gen(4)
    x, w, r = rnd(1, 64).bfloat16().expand(300, 64), rnd(96, 64).bfloat16(), rnd(1, 96).bfloat16().expand(300, 96)
    want = linear64(x, w, None, "none", r, False)
    within(ops.linear(x, w, residual=r), want, linear_tol(x, w, None, r, want, torch.bfloat16))
    z = rnd(1, 64).expand(50, 64)
    want, spread, _ = norm64(z[:, None], 4, None, None, 1e-5, "none", None, None)
    within(ops.group_norm(z, 4), want[:, 0], norm_tol(want, spread, torch.float32, 24)[:, 0])
    q, k, v, g, beta, state = delta_inputs(3, 2, 70, 2, 4, 32, 32, torch.bfloat16, True)
    check_delta(ops, q[:, :, :1].expand(2, 70, 2, 32), k[:1].expand(2, 70, 2, 32), v[:, :, :1].expand(2, 70, 4, 32), g, beta, state, True)


# ------------------------------------------------------------------------------------------- what the interface promises

@pytest.mark.parametrize("dtype", ("f16", "bf16"))
@pytest.mark.parametrize("normalize", (True, False))
@pytest.mark.parametrize("b, t, hk, h, dk, dv", DELTA_SIZES + [(2, 1000, 1, 2, 128, 64)])
def test_gated_delta_rounds_an_output_once(ops, b, t, hk, h, dk, dv, normalize, dtype):
    """sums and states are float32 whatever the type: the 16-bit call's outputs are the float32 call's on the same values, rounded once, and its states the same bits"""
    q, k, v, g, beta, state = delta_inputs(t + dv, b, t, hk, h, dk, dv, TYPES[dtype], normalize)
    mine, wide = state.clone(), state.clone()
    got = ops.gated_delta(q, k, v, g, beta, mine, normalize=normalize)
    want = ops.gated_delta(q.float(), k.float(), v.float(), g, beta, wide, normalize=normalize)
    assert torch.equal(got, want.to(got.dtype)) and torch.equal(mine, wide)


@pytest.mark.parametrize("normalize", (True, False))
@pytest.mark.parametrize("b, t, hk, h, dk, dv", DELTA_SIZES + [(2, 1000, 1, 2, 128, 64)])
def test_gated_delta_float32_outputs_are_as_good_as_the_state(ops, b, t, hk, h, dk, dv, normalize):
    """an output is a sum over the state's rows through q: it has the state's relative error (3e-6 of the norm, as check_delta's) and that of its own dk + 64 terms, rounded
    independently: sqrt(dk + 64) half steps, 18 u = 1.1e-6 at most"""
    q, k, v, g, beta, state = delta_inputs(t + dk + 1, b, t, hk, h, dk, dv, torch.float32, normalize)
    want, _, _ = delta64(q, k, v, g, beta, state, 0.5, normalize, None)
    got = ops.gated_delta(q, k, v, g, beta, state, scale=0.5, normalize=normalize)
    assert (got.double() - want).norm() <= 4.1e-6 * want.norm()


@pytest.mark.parametrize("act", ("sigmoid", "silu"))
def test_float32_sigmoid_far_from_zero(ops, act):
    """the activation's own error in float32 steps, where 1 + e^-y is all exponential: an exponential and a reciprocal of 1 step each, 1 + e and y sigmoid rounded (half a step each), and what is
    left of e^-y's own corrections, 1 step -- 4 steps of 2 u relative; beyond its range it ends at 0 and 1"""
    one = torch.ones(1, 1, device="cuda")
    y = torch.linspace(-79, 79, 160001, device="cuda")
    for rows, part in ((1, slice(None)), (300, slice(0, 9000)), (300, slice(75000, 84000))):
        got, want = ops.linear(one.expand(rows, 1), y[part, None], activation=act)[rows // 2], act64(y[part].double(), act)
        assert ((got.double() - want).abs() <= 4 * 2 * U * want.abs()).all()
    y = torch.tensor([-math.inf, -3e38, -1000.0, -200.0, 200.0, 3e38, math.inf, math.nan], device="cuda")
    got = ops.linear(one, y[:, None], activation="sigmoid")[0]
    assert torch.equal(got[:7], torch.tensor([0.0, 0.0, 0.0, 0.0, 1.0, 1.0, 1.0], device="cuda")) and torch.isnan(got[7])
    got = ops.linear(one, y[1:7, None], activation="silu")[0]
    assert torch.equal(got, torch.tensor([0.0, 0.0, 0.0, 200.0, 3e38, math.inf], device="cuda"))


def test_outputs_in_the_rows_of_an_operand(ops):
    """x and out, x and gate, v and out side by side in the same wide rows"""
    rnd = gen(12)
    rows = rnd(70, 32 + 48)
    x, out, w = rows[:, :32], rows[:, 32:], rnd(48, 32)
    want = ops.linear(x.clone(), w)
    assert torch.equal(ops.linear(x, w, out=out), want) and torch.equal(rows[:, 32:], want)
    rows = rnd(3, 40, 3, 24)
    want = ops.group_norm(rows[:, :, 0].clone(), 4, gate=rows[:, :, 1].clone())
    assert torch.equal(ops.group_norm(rows[:, :, 0], 4, gate=rows[:, :, 1], out=rows[:, :, 2]), want)
    q, k, v, g, beta, state = delta_inputs(6, 2, 70, 1, 2, 16, 24, torch.float32, True)
    rows = torch.cat([v, v], 3)
    mine = state.clone()
    want = ops.gated_delta(q, k, v, g, beta, state, normalize=True)
    assert torch.equal(ops.gated_delta(q, k, rows[..., :24], g, beta, mine, normalize=True, out=rows[..., 24:]), want) and torch.equal(mine, state)


@pytest.mark.parametrize("t", (1, 40))
def test_gated_delta_refuses_a_state_over_its_inputs(ops, t):
    """views of one pool: values inside the states are refused, with and without an output given; beside them they are taken"""
    q, k, v, g, beta, state = delta_inputs(7, 2, t, 1, 2, 16, 24, torch.float32, True)
    part = 2 * 16 * 24
    pool = torch.zeros(2, part + t * 48, device="cuda")
    s = pool[:, :part].view(2, 2, 16, 24)
    s.copy_(state)
    over = pool.as_strided((2, t, 2, 24), (part + t * 48, 48, 24, 1), part - 1)
    for out in (None, torch.empty_like(v)):
        with pytest.raises(ValueError, match="state overlaps v"):
            ops.gated_delta(q, k, over, g, beta, s, out=out)
    assert torch.equal(s, state)
    beside = pool[:, part:].view(2, t, 2, 24)
    beside.copy_(v)
    assert torch.equal(ops.gated_delta(q, k, beside, g, beta, s, normalize=True), ops.gated_delta(q, k, v, g, beta, state, normalize=True)) and torch.equal(s, state)


@pytest.mark.parametrize("t", (1, 40))
def test_writes_in_place_are_seen_by_autograd(ops, t):
    """a graph that saved a tensor which a call then writes raises in its backward, as with torch's own in-place operations, also through a view; a tensor of torch's inference mode is taken"""
    rnd = gen(13)
    q, k, v, g, beta, state = delta_inputs(8, 2, t, 1, 2, 16, 24, torch.float32, True)
    x, w, z = rnd(30, 16), rnd(24, 16), rnd(30, 24)
    for written, call in ((state, lambda: ops.gated_delta(q, k, v, g, beta, state, normalize=True)), (state, lambda: ops.gated_delta(q, k, v, g, beta, state[:], normalize=True)),
                          (v, lambda: ops.gated_delta(q, k, v.clone(), g, beta, state, normalize=True, out=v)), (z, lambda: ops.linear(x, w, residual=z, out=z)), (z, lambda: ops.group_norm(z, 4, out=z)),
                          (z, lambda: ops.linear(x[:10], w, out=z[:10]))):
        weight = torch.ones_like(written, requires_grad=True)
        loss = (written * weight).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    before = (q._version, x._version, w._version)
    ops.linear(x, w)
    ops.gated_delta(q, k, v, g, beta, state, normalize=True)
    assert (q._version, x._version, w._version) == before
    with torch.inference_mode():
        s = state.clone()
        assert torch.equal(ops.gated_delta(q, k, v, g, beta, s, normalize=True), ops.gated_delta(q, k, v, g, beta, state, normalize=True))


def test_tangents_are_refused(ops):
    from torch.autograd import forward_ad

    rnd = gen(14)
    x, w = rnd(5, 16), rnd(8, 16)
    q, k, v, g, beta, state = delta_inputs(8, 2, 3, 1, 2, 16, 24, torch.float32, True)
    with forward_ad.dual_level():
        assert torch.equal(ops.linear(x, w), ops.linear(x, w))       # no tangent: taken
        dual = {a: forward_ad.make_dual(b, torch.ones_like(b)) for a, b in (("x", x), ("w", w), ("state", state), ("g", g))}
        with torch.no_grad():
            for call in (lambda: ops.linear(dual["x"], w), lambda: ops.linear(x, dual["w"]), lambda: ops.group_norm(dual["x"], 2), lambda: ops.gated_delta(q, k, v, g, beta, dual["state"]),
                         lambda: ops.gated_delta(q, k, v, dual["g"], beta, state)):
                with pytest.raises(ValueError, match="forward-mode"):
                    call()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("normalize", (True, False))
@pytest.mark.parametrize("t, at, dk, dv", [(1, 0, 32, 24), (6, 2, 64, 32), (6, 5, 40, 3), (90, 40, 64, 32), (90, 89, 128, 40), (90, 0, 100, 17), (40, 30, 200, 24)])
def test_gated_delta_what_is_not_finite(ops, t, at, dk, dv, normalize, dtype):
    """one value that is not finite, in each operand, in either form: NaN in its column (a key or gate: all columns; a query: its own outputs) of its head from its step on, every other bit as without it"""
    q, k, v, g, beta, state = delta_inputs(t + dk, 2, t, 2, 4, dk, dv, TYPES[dtype], normalize)
    clean = state.clone()
    want = ops.gated_delta(q, k, v, g, beta, clean, normalize=normalize)
    for value in (math.inf, -math.inf, math.nan):
        for name in ("q", "k", "v", "g", "beta", "state"):
            if name == "g" and value == -math.inf:
                continue                             # a state that is forgotten
            a = dict(q=q.clone(), k=k.clone(), v=v.clone(), g=g.clone(), beta=beta.clone(), state=state.clone())
            outs, states = torch.zeros_like(want, dtype=torch.bool), torch.zeros_like(state, dtype=torch.bool)
            if name in ("q", "k"):
                a[name][1, at, 1, 7] = value         # the heads 2 and 3
                outs[1, at:(at + 1 if name == "q" else t), 2:] = True
                states[1, 2:] = name == "k"
            elif name == "v":
                a[name][1, at, 1, 2] = value
                outs[1, at:, 1, 2], states[1, 1, :, 2] = True, True
            elif name == "state":
                a[name][1, 1, 5, 2] = value
                outs[1, :, 1, 2], states[1, 1, :, 2] = True, True
            else:
                a[name][1, at, 1] = value
                outs[1, at:, 1], states[1, 1] = True, True
            got = ops.gated_delta(a["q"], a["k"], a["v"], a["g"], a["beta"], a["state"], normalize=normalize)
            assert torch.equal(torch.isnan(got), outs) and torch.equal(torch.isnan(a["state"]), states), (name, value)
            assert torch.equal(got[~outs], want[~outs]) and torch.equal(a["state"][~states], clean[~states]), (name, value)


# float32 products in tiles, both sizes of them: far from the sizes where a narrower form takes over (512 blocks of 64 rows x 16 features) and from each other (200 tiles of 128 x 128)
PARTS_SIZES = [(1025, 1900), (2049, 2500)]


@pytest.mark.parametrize("m, n", PARTS_SIZES)
@pytest.mark.parametrize("k", (128, 131))
def test_linear_float32_tiles_infinities_and_nan(ops, m, n, k):
    """an infinity or NaN reaches the outputs of its row or feature, as in the definition, and no other"""
    rnd = gen(m + k)
    x, w = rnd(m, k), rnd(n, k)
    x[0, 3], x[1, 64], x[m - 1, k - 1], x[700, 0] = math.inf, math.nan, -math.inf, math.inf
    w[7, 5], w[n - 1, k - 1], w[70, 3] = -math.inf, math.nan, 0.0    # (infinity times zero)
    got, want = ops.linear(x, w).double(), linear64(x, w, None, "none", None, False)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    ok = torch.isfinite(want)
    x, w = x.nan_to_num(0, 0, 0), w.nan_to_num(0, 0, 0)
    within(torch.where(ok, got, 0.0), torch.where(ok, want, 0.0), linear_tol(x, w, None, None, torch.where(ok, want, 0.0), torch.float32))


@pytest.mark.parametrize("m, n", PARTS_SIZES)
def test_linear_float32_tiles_range(ops, m, n):
    """operands near the ends of the range.  An operand's three bfloat16 parts end at bfloat16's smallest number, 2^-133: what is left of it is at most half of that, 2^-134 times the other factor"""
    w = torch.full((n, 64), 2.0 ** -30, device="cuda")
    x = torch.full((m, 64), 3.4e38, device="cuda")
    want = linear64(x, w, None, "none", None, False)
    within(ops.linear(x, w), want, linear_tol(x, w, None, None, want, torch.float32))
    w = gen(m)(n, 64) * 2.0 ** 40
    for e in (-60, -100, -108, -112, -116, -120, -126, -130, -140):
        x = gen(n)(m, 64) * 2.0 ** e
        want = linear64(x, w, None, "none", None, False)
        tol = (64 + 8) * U * (x.double().abs() @ w.double().abs().T) + 2.0 ** -134 * w.double().abs().sum(1)
        within(ops.linear(x, w), want, tol)
        within(ops.linear(w, x), want.T, tol.T)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("mode", ("none", "after", "before"))
@pytest.mark.parametrize("m, n", PARTS_SIZES)
def test_linear_float32_tiles_epilogues(ops, m, n, mode, act):
    rnd = gen(m)
    x, w, b, r = rnd(m, 96), rnd(n, 96) * 0.3, rnd(n), rnd(m, n)
    r = None if mode == "none" else r
    want = linear64(x, w, b, act, r, mode == "before")
    tol = linear_tol(x, w, b, r, want, torch.float32)
    within(ops.linear(x, w, bias=b, activation=act, residual=r, residual_first=mode == "before"), want, tol)
    if r is not None:                                # in place, and in rows that are further apart
        wide = torch.empty(m, n + 5, device="cuda")[:, 3:n + 3]
        wide.copy_(r)
        within(ops.linear(x, w, bias=b, activation=act, residual=wide, residual_first=mode == "before", out=wide), want, tol)


@pytest.mark.parametrize("dtype", TYPES)
def test_gelu_keeps_its_negative_tail(ops, dtype):
    """relative, down to y = -12 (fp16: to its smallest numbers): the argument y / sqrt 2 and its constant are rounded, which erfc takes 2 (y / sqrt 2)^2 times, 2 y^2 u; erfc itself is good to 16
    steps of 2 u, two products to u each; then half a step of the output's type"""
    dt = TYPES[dtype]
    y = torch.linspace(-12, 12, 48001, device="cuda").to(dt)
    one = torch.ones(1, 1, dtype=dt, device="cuda")
    want = 0.5 * y.double() * torch.special.erfc(-y.double() / 2 ** 0.5)
    for rows, part in ((1, slice(None)), (300, slice(0, 9000)), (300, slice(20000, 29000))):
        got = ops.linear(one.expand(rows, 1), y[part, None], activation="gelu")[rows // 2]
        tol = (2 * y[part].double() ** 2 + 34) * U * want[part].abs()
        within(got, want[part], tol * (1 + torch.finfo(dt).eps) + half_step(want[part], dt))
    far = torch.tensor([-math.inf, -100.0, 100.0, math.inf, math.nan], dtype=dt, device="cuda")
    got = ops.linear(one, far[:, None], activation="gelu")[0]
    assert got[1] == 0 and got[2] == 100 and got[3] == math.inf and torch.isnan(got[4])
