"""Work of the operators on device tensors (vadc_amd/ops.py): what a streaming layer with a recurrent state runs per call.

    linear       y = act(x W^T + b) + r                      the projections around the recurrence
    gated_delta  S_t = a_t S_{t-1} + k_t u_t^T, ...          the recurrence, one state per stream, one step or many per call
    group_norm   y = (x - mean) / sqrt(var + eps) w + b      per head behind the recurrence (gated), per sequence in an encoder

A case is one call.  `run` computes it in plain torch (float32, rounded once at the end) or, with `own`, through vadc_amd.ops;
`exact` gives the definition's values in float64.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------------------------------------------------------- cases

def _linear(m, k, n, dtype, bias, act, residual, **kw):
    return dict(op="linear", m=m, k=k, n=n, dtype=dtype, bias=bias, act=act, residual=residual, **kw)


def _norm(n, l, c, groups, dtype, act, gate, ragged, **kw):
    return dict(op="group_norm", n=n, l=l, c=c, groups=groups, dtype=dtype, act=act, gate=gate, ragged=ragged, **kw)


def _delta(b, t, hk, h, dk, dv, dtype, normalize, ragged, **kw):
    return dict(op="gated_delta", b=b, t=t, hk=hk, h=h, dk=dk, dv=dv, dtype=dtype, normalize=normalize, ragged=ragged, **kw)


def listed():
    return [
        # one stream's projection at one step: the weights are read once, latency counts
        _linear(1, 2048, 2048, "bf16", True, "silu", "none", name="linear 1 row bf16"),
        # one step of 256 streams (the benchmark's stream count) through an output projection
        _linear(256, 2048, 2048, "f16", True, "none", "after", name="linear 256 rows f16"),
        # an odd batch with sizes that are no multiple of a tile; the residual enters in front of the activation, as in a conv block
        _linear(1111, 1000, 1537, "bf16", True, "gelu", "before", name="linear odd bf16"),
        # the float32 input projection of 512 gate rows from 128 features, 4096 streams x 24 steps
        _linear(98304, 128, 512, "f32", True, "none", "none", name="linear gates f32"),
        # a wide projection over a long batch of steps
        _linear(8192, 4096, 4096, "bf16", True, "silu", "after", name="linear large bf16"),
        # the heads' norm with its gate, one step of 256 streams
        _norm(256, 1, 2048, 16, "bf16", "silu", True, False, name="norm heads 256 steps"),
        # an encoder's feature sequences, channels last, of unequal lengths
        _norm(6, 20011, 384, 12, "f32", "silu", False, True, name="norm long ragged f32"),
        # the heads' norm with its gate, many steps of many streams
        _norm(49152, 1, 4096, 32, "bf16", "silu", True, False, name="norm heads large"),
        # one stream, one step
        _delta(1, 1, 16, 16, 128, 128, "bf16", True, False, name="delta one step"),
        # one step of 4096 streams: the states are read and written once
        _delta(4096, 1, 4, 4, 64, 64, "bf16", True, False, name="delta 4096 streams"),
        # 61 streams of unequal lengths, odd head sizes, float32
        _delta(61, 333, 3, 6, 48, 80, "f32", True, True, name="delta ragged f32"),
        # one long stream: two value heads to a key head
        _delta(2, 8192, 16, 32, 128, 128, "bf16", True, False, name="delta long"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("linear", "group_norm", "gated_delta"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    odd = rng.random() < 0.4
    if op == "linear":
        m = _log(rng, 1, 16384)
        k, n = (_log(rng, 64, 4096) for _ in range(2))
        if not odd:
            k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
        while m * k * n > (2 ** 37 if dtype != "f32" else 2 ** 34):
            m = max(1, m // 2)
        return _linear(m, k, n, dtype, rng.random() < 0.8, rng.choice(("none", "relu", "silu", "gelu", "sigmoid")), rng.choice(("none", "after", "before")))
    if op == "group_norm":
        groups = rng.choice((1, 4, 8, 12, 16, 32))
        c = groups * (_log(rng, 3, 128) if odd else 8 * _log(rng, 1, 16))
        heads = rng.random() < 0.5
        n, l = (_log(rng, 1, 65536), 1) if heads else (_log(rng, 1, 64), _log(rng, 2, 32768))
        while n * l * c > 2 ** 26:
            n, l = (max(1, n // 2), l) if n > 1 else (n, max(1, l // 2))
        return _norm(n, l, c, groups, dtype, rng.choice(("none", "relu", "silu", "gelu", "sigmoid")), heads, not heads and rng.random() < 0.5)
    hk = rng.choice((1, 2, 3, 4, 8, 16))
    h = hk * rng.choice((1, 1, 2, 4))
    dk, dv = (_log(rng, 24, 128), _log(rng, 24, 128)) if odd else (rng.choice((64, 128)), rng.choice((64, 128)))
    b, t = (_log(rng, 1, 4096), 1) if rng.random() < 0.4 else (_log(rng, 1, 256), _log(rng, 2, 8192))
    while b * h * dk * dv > 2 ** 26 or b * t * h * (dk + dv) > 2 ** 26:
        b, t = (max(1, b // 2), t) if b > 1 else (b, max(1, t // 2))
    return _delta(b, t, hk, h, dk, dv, dtype, rng.random() < 0.7, t > 1 and rng.random() < 0.4)


# --------------------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(g, n, longest):
    """unequal lengths, the longest and (of four or more) an empty one among them"""
    v = torch.randint(1, longest + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
    v[0] = longest
    if n >= 4:
        v[n // 2] = 0
    return v


def prepare(case, seed):
    g, dt = _gen(seed), TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = dict(case)
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = randn(m, k).to(dt)
        s["weight"] = (randn(n, k) * k ** -0.5).to(dt)
        s["bias"] = (randn(n) * 0.1).to(dt) if case["bias"] else None
        s["res"] = randn(m, n).to(dt) if case["residual"] != "none" else None
    elif case["op"] == "group_norm":
        n, l, c = case["n"], case["l"], case["c"]
        s["x"] = (randn(n, l, c) * (0.5 + torch.rand(c, generator=g, device="cuda")) + 0.7 * randn(c)).to(dt)   # channels differ in mean and scale
        s["weight"] = (1 + 0.1 * randn(c)).to(dt)
        s["bias"] = (0.1 * randn(c)).to(dt)
        s["gate"] = randn(n, l, c).to(dt) if case["gate"] else None
        s["lengths"] = _lengths(g, n, l) if case["ragged"] else None
        s["out"] = torch.zeros(n, l, c, dtype=dt, device="cuda") if case["ragged"] else None
    else:
        b, t, hk, h, dk, dv = (case[w] for w in ("b", "t", "hk", "h", "dk", "dv"))
        k = randn(b, t, hk, dk)
        q = randn(b, t, hk, dk)
        if not case["normalize"]:                    # keys of length one at most, as the recurrence needs them
            k = k / (k.norm(dim=-1, keepdim=True) * 1.01)
            q = q / q.norm(dim=-1, keepdim=True)
        s["q"], s["k"], s["v"] = q.to(dt), k.to(dt), randn(b, t, h, dv).to(dt)
        rate = torch.exp(torch.empty(h, device="cuda").uniform_(math.log(0.01), math.log(1.0), generator=g))    # heads forget at rates of their own
        s["log_decay"] = -rate * torch.nn.functional.softplus(randn(b, t, h))
        s["beta"] = torch.sigmoid(randn(b, t, h))
        s["state"] = 0.1 * randn(b, h, dk, dv)
        s["lengths"] = _lengths(g, b, t) if case["ragged"] else None
        s["out"] = torch.zeros(b, t, h, dv, dtype=dt, device="cuda") if case["ragged"] else None
    return s


# ---------------------------------------------------------------------------------------------------- the plain form

def _act(y, name):
    if name == "relu":
        return torch.clamp(y, min=0)
    if name == "silu":
        return y / (1 + torch.exp(-y))
    if name == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-y))
    return y


def _plain_linear(s):
    y = s["x"].float() @ s["weight"].float().T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["residual"] == "before":
        y = y + s["res"].float()
    y = _act(y, s["act"])
    if s["residual"] == "after":
        y = y + s["res"].float()
    return y.to(s["x"].dtype)


def _plain_norm(s):
    x, groups = s["x"], s["groups"]
    n, l, c = x.shape
    v = x.float().reshape(n, l, groups, c // groups)
    if s["lengths"] is None:
        mean = v.mean(dim=(1, 3), keepdim=True)
        d = v - mean
        var = (d * d).mean(dim=(1, 3), keepdim=True)
    else:
        live = (torch.arange(l, device=x.device)[None, :] < s["lengths"][:, None])[:, :, None, None]
        count = (s["lengths"].float() * (c // groups)).clamp(min=1)[:, None, None, None]
        mean = torch.where(live, v, 0.0).sum(dim=(1, 3), keepdim=True) / count
        d = torch.where(live, v - mean, 0.0)
        var = (d * d).sum(dim=(1, 3), keepdim=True) / count
    y = (d / torch.sqrt(var + 1e-5)).reshape(n, l, c) * s["weight"].float() + s["bias"].float()
    y = y * _act(s["gate"].float(), s["act"]) if s["gate"] is not None else _act(y, s["act"])
    y = y.to(x.dtype)
    if s["lengths"] is None:
        return y
    s["out"].copy_(torch.where(live[:, :, :, 0], y, s["out"]))
    return s["out"]


def _plain_delta(s):
    """The recurrence in blocks of 64 steps.  With G the running sum of log_decay inside a block, A[i, j] = beta_i e^(G_i - G_j) k_i.k_j below the diagonal,
    the updates are U = (I + A)^-1 diag(beta) (V - diag(e^G) K S), the outputs diag(e^G) Q S + tril(e^(G_i - G_j) q_i.k_j) U."""
    q, k, v, state = s["q"], s["k"], s["v"], s["state"]
    b, t, hk, dk = q.shape
    h, dv = v.shape[2], v.shape[3]
    q, k, w = q.float(), k.float(), v.float()
    if s["normalize"]:
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + 1e-6)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    q = (q * dk ** -0.5).repeat_interleave(h // hk, dim=2)
    k = k.repeat_interleave(h // hk, dim=2)
    decay, beta = s["log_decay"], s["beta"]
    if s["lengths"] is not None:                     # a step that is not there changes nothing
        live = torch.arange(t, device=q.device)[None, :, None] < s["lengths"][:, None, None]
        decay, beta = torch.where(live, decay, 0.0), torch.where(live, beta, 0.0)
    size = min(64, t)
    blocks = -(-t // size)

    def cut(a):                                      # [b, t, h, d] -> [b, h, blocks, size, d]
        a = torch.nn.functional.pad(a, (0, 0, 0, 0, 0, blocks * size - t))
        return a.reshape(b, blocks, size, h, -1).permute(0, 3, 1, 2, 4).contiguous()

    q, k, w = cut(q), cut(k), cut(w)
    total = cut(decay[..., None])[..., 0].double().cumsum(-1)
    beta = cut(beta[..., None])
    between = torch.exp((total[..., :, None] - total[..., None, :]).clamp(max=700)).float()
    kt = k.transpose(-1, -2).contiguous()
    power = -torch.tril(beta * between * (k @ kt), -1).double()
    eye = torch.eye(size, device=q.device, dtype=torch.float64)
    inverse, reach = eye + power, 2
    while reach < size:                              # 1 + p + p^2 + ... as (1 + p)(1 + p^2)(1 + p^4) ...
        power = power @ power
        inverse = inverse + inverse @ power
        reach *= 2
    inverse = inverse.float()
    inner = torch.tril(between * (q @ kt))
    gain = torch.exp(total).float()[..., None]
    rest = torch.exp(total[..., -1:] - total).float()[..., None]
    end = torch.exp(total[..., -1]).float()[..., None, None]
    outs, S = [], state
    for i in range(blocks):
        u = inverse[:, :, i] @ (beta[:, :, i] * (w[:, :, i] - gain[:, :, i] * (k[:, :, i] @ S)))
        outs.append(gain[:, :, i] * (q[:, :, i] @ S) + inner[:, :, i] @ u)
        S = end[:, :, i] * S + (rest[:, :, i] * k[:, :, i]).transpose(-1, -2) @ u
    state.copy_(S)
    o = torch.stack(outs, 2).permute(0, 2, 3, 1, 4).reshape(b, blocks * size, h, dv)[:, :t].to(v.dtype)
    if s["lengths"] is not None:
        s["out"].copy_(torch.where(live[..., None], o, s["out"]))
        o = s["out"]
    return o.contiguous(), state


# ------------------------------------------------------------------------------------------------------------ one pass

def run(s):
    if own:
        from vadc_amd import ops

        if s["op"] == "linear":
            return ops.linear(s["x"], s["weight"], bias=s["bias"], activation=s["act"], residual=s["res"], residual_first=s["residual"] == "before")
        if s["op"] == "group_norm":
            return ops.group_norm(s["x"], s["groups"], weight=s["weight"], bias=s["bias"], activation=s["act"], gate=s["gate"], lengths=s["lengths"], out=s["out"])
        o = ops.gated_delta(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], s["state"], normalize=s["normalize"], lengths=s["lengths"], out=s["out"])
        return o, s["state"]
    if s["op"] == "linear":
        return _plain_linear(s)
    return _plain_norm(s) if s["op"] == "group_norm" else _plain_delta(s)


def work(case):
    w = BYTES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": w * (m * k + n * k + m * n * (2 if case["residual"] != "none" else 1) + (n if case["bias"] else 0)), "flops": 2 * m * k * n}
    if case["op"] == "group_norm":
        e = case["n"] * case["l"] * case["c"]
        if case["ragged"]:
            e //= 2                                  # lengths are uniform up to the longest
        return {"bytes": w * (e * (3 if case["gate"] else 2) + 2 * case["c"]), "flops": 10 * e}
    b, t, hk, h, dk, dv = (case[x] for x in ("b", "t", "hk", "h", "dk", "dv"))
    steps = b * t // (2 if case["ragged"] else 1)
    return {"bytes": steps * (w * (2 * hk * dk + 2 * h * dv) + 8 * h) + 8 * b * h * dk * dv, "flops": steps * h * 7 * dk * dv}


# ------------------------------------------------------------------------------------- the definition, step by step, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    functions = {"none": lambda a: a, "relu": torch.relu, "silu": lambda a: a * torch.sigmoid(a), "sigmoid": torch.sigmoid,
                 "gelu": lambda a: a * torch.special.ndtr(a)}
    act = functions[case["act"]] if "act" in case else None
    if case["op"] == "linear":
        rows = []
        for x, r in zip(s["x"].split(16384), (s["res"] if s["res"] is not None else s["x"]).split(16384)):
            a = torch.mm(x.double(), s["weight"].double().t())
            if case["bias"]:
                a += s["bias"].double()
            if case["residual"] == "none":
                rows.append(act(a))
            else:
                rows.append(act(a + r.double()) if case["residual"] == "before" else act(a) + r.double())
        return torch.cat(rows)
    if case["op"] == "group_norm":
        out = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
        size = case["c"] // case["groups"]
        if case["l"] == 1:
            pieces = [(slice(i, i + 8192), slice(0, 1)) for i in range(0, case["n"], 8192)]
        else:
            pieces = [(slice(i, i + 1), slice(0, int(s["lengths"][i]) if case["ragged"] else case["l"])) for i in range(case["n"])]
        for rows, steps in pieces:
            x = s["x"][rows, steps].double()
            if not x.numel():
                continue
            grouped = x.unflatten(2, (case["groups"], size)).transpose(1, 2).flatten(2)
            var, mean = torch.var_mean(grouped, dim=2, correction=0)
            wide = [a.repeat_interleave(size, dim=1)[:, None] for a in (mean, var)]
            y = (x - wide[0]) * torch.rsqrt(wide[1] + 1e-5) * s["weight"].double() + s["bias"].double()
            out[rows, steps] = y * act(s["gate"][rows, steps].double()) if case["gate"] else act(y)
        return out
    b, t, hk, h, dk, dv = (case[w] for w in ("b", "t", "hk", "h", "dk", "dv"))
    S, last = s["state"].double(), s["lengths"]
    out = torch.zeros(b, t, h, dv, dtype=torch.float64, device="cuda")
    for i in range(t):
        q, k = s["q"][:, i].double(), s["k"][:, i].double()
        if case["normalize"]:
            q, k = (a * torch.rsqrt(a.square().sum(2, keepdim=True) + 1e-6) for a in (q, k))
        q, k = (a[:, :, None].expand(b, hk, h // hk, dk).reshape(b, h, dk, 1) for a in (q, k))
        now = S * s["log_decay"][:, i].double().exp()[..., None, None]
        u = s["beta"][:, i].double()[..., None] * (s["v"][:, i].double() - (now * k).sum(2))
        now = now + k * u[:, :, None]
        o = (now * q).sum(2) / math.sqrt(dk)
        if last is None:
            S, out[:, i] = now, o
        else:
            there = (i < last)[:, None, None]
            S, out[:, i] = torch.where(there[..., None], now, S), torch.where(there, o, 0.0)
    return out, S
