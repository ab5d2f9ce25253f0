"""The sequence operators and their gradients in 64 bits, position by position from the formulas,
and what rounding may move a result by.

Every function also runs on magnitudes (`mag=True`): each product and sum of absolute values, so that
a value whose computation passes k roundings of unit u lies within k u times its magnitude. A
rounding is off by at most u = 2^-24 (float32) or 2^-53 (float64) relative to its value.
"""

import numpy as np

import rustautograd_amd as rg

UNIT = {"float32": 2.0 ** -24, "float64": 2.0 ** -53}


def sigmoid(v):
    return 1.0 / (1.0 + np.exp(-v))


def softplus(v):
    return np.maximum(v, 0.0) + np.log1p(np.exp(-np.abs(v)))


def _ends(lengths, batch, length):
    return [length] * batch if lengths is None else [min(max(int(n), 0), length) for n in lengths]


def conv(x, w, bias, state, lengths, silu, dy, dnext, mag=False):
    """{y, next, dx, dw, dbias, dstate}; `dnext` may be None."""
    A = np.abs if mag else (lambda v: v)
    b, t, d = x.shape
    k = w.shape[0]
    past = np.concatenate([np.zeros((b, k - 1, d)) if state is None else state, x], 1).astype(np.float64)
    y, nxt = np.zeros((b, t, d)), np.zeros((b, k - 1, d))
    dpast, dw, db = np.zeros_like(past), np.zeros(w.shape), np.zeros(d)
    for i, n in enumerate(_ends(lengths, b, t)):
        row = past[i].copy()
        row[k - 1 + n:] = 0.0  # not read
        for s in range(n):
            pre = sum(w[j] * row[s + j] for j in range(k)) + (0.0 if bias is None else bias)
            g = sigmoid(pre)
            size = sum(np.abs(w[j] * row[s + j]) for j in range(k)) + (0.0 if bias is None else np.abs(bias))
            # The slope of silu is at most 1.1, so a result moves by at most that times what pre does.
            y[i, s] = (1.1 * size if silu else size) if mag else (pre * g if silu else pre)
            slope = g * (1.0 + pre * (1.0 - g)) if silu else np.ones(d)
            # The slope itself moves by at most half of what pre moves.
            gp = np.abs(dy[i, s]) * (np.abs(slope) + 0.5 * size + 1.0) if mag else dy[i, s] * slope
            db += gp
            for j in range(k):
                dw[j] += gp * A(row[s + j])
                dpast[i, s + j] += gp * A(w[j])
        nxt[i] = A(row[n:n + k - 1])
        if dnext is not None:
            dpast[i, n:n + k - 1] += A(dnext[i])
    return {"y": y, "next": nxt, "dx": dpast[:, k - 1:], "dw": dw, "dbias": db, "dstate": dpast[:, :k - 1]}


def conv_roundings(x, w):
    """Products and sums of an output, its activation, and the sums over the batch of dw."""
    return 2 * w.shape[0] + 24 + x.shape[0] * x.shape[1]


def scan(x, dt, a, b, c, d, z, state, lengths, soft, dy, dlast, mag=False):
    """{y, last, dx, ddt, da, db, dc, dd, dz, dstate}; b and c are [batch, length, groups, states]."""
    A = np.abs if mag else (lambda v: v)
    n_b, length, width = x.shape
    states, groups = a.shape[1], b.shape[2]
    per = width // groups
    out = {"y": np.zeros(x.shape), "last": np.zeros((n_b, width, states)), "dx": np.zeros(x.shape), "ddt": np.zeros(x.shape), "da": np.zeros(a.shape),
           "db": np.zeros(b.shape), "dc": np.zeros(c.shape), "dd": np.zeros(width), "dz": np.zeros(x.shape), "dstate": np.zeros((n_b, width, states))}
    for i, n in enumerate(_ends(lengths, n_b, length)):
        h = [A(np.zeros((width, states)) if state is None else state[i].astype(np.float64))]
        steps, decays, ys, gates = [], [], [], []
        for t in range(n):
            step = softplus(dt[i, t].astype(np.float64)) if soft else dt[i, t].astype(np.float64)
            e = np.exp(step[:, None] * a)
            bt, ct = (A(np.repeat(v[i, t], per, 0)) for v in (b, c))
            h.append(e * h[-1] + A((step * x[i, t])[:, None]) * bt)
            y = (ct * h[-1]).sum(-1) + (0.0 if d is None else A(d * x[i, t]))
            gate = 1.0 if z is None else z[i, t] * sigmoid(z[i, t].astype(np.float64))
            steps.append(step), decays.append(e), ys.append(y), gates.append(gate)
            out["y"][i, t] = y * A(gate)
        out["last"][i] = h[-1]
        back = np.zeros((width, states)) if dlast is None else A(dlast[i].astype(np.float64))
        for t in reversed(range(n)):
            bt, ct = (A(np.repeat(v[i, t], per, 0)) for v in (b, c))
            step, u = A(steps[t]), A(x[i, t].astype(np.float64))
            gy = A(dy[i, t] * gates[t])
            if z is not None:
                s = sigmoid(z[i, t].astype(np.float64))
                out["dz"][i, t] = A(dy[i, t]) * ys[t] * A(s * (1.0 + z[i, t] * (1.0 - s)) + (1.0 if mag else 0.0))
            g = back + gy[:, None] * ct
            p = decays[t] * h[t]
            sum_b, sum_a = (g * bt).sum(-1), (g * p * A(a)).sum(-1)
            out["dx"][i, t] = step * sum_b + (0.0 if d is None else gy * A(d))
            out["ddt"][i, t] = (u * sum_b + sum_a) * (sigmoid(dt[i, t].astype(np.float64)) if soft else 1.0)
            out["da"] += g * p * step[:, None]
            for q in range(groups):
                ch = slice(q * per, (q + 1) * per)
                out["db"][i, t, q] = (g * (step * u)[:, None])[ch].sum(0)
                out["dc"][i, t, q] = (gy[:, None] * h[t + 1])[ch].sum(0)
            out["dd"] += gy * u
            back = g * decays[t]
        out["dstate"][i] = back
    return out


def scan_roundings(x, dt, a, soft):
    """A state passes as many steps as the sequence has, forward and back, each rounding the decay (its
    exponent, of relative error 6 u, counts |dt a| times), the products and the sum; outputs sum over
    the states, the gradients of the maps over the channels and those of a and d over the batch."""
    step = softplus(dt.astype(np.float64)) if soft else np.abs(dt.astype(np.float64))
    exponent = float(np.nanmax(step) * np.abs(a).max())
    return (6.0 * exponent + 8.0) * 2 * x.shape[1] + a.shape[1] + x.shape[2] + x.shape[0] * x.shape[1] + 60


def rotary(x, gain, pos, sections, turn, base, eps, dy, mag=False):
    """{y, dx, dgain}."""
    b, t, heads, hd = x.shape
    half = turn // 2
    x, dy = x.astype(np.float64), dy.astype(np.float64)
    pos = np.broadcast_to(pos, (b, t)).astype(np.longdouble)
    inverse = np.longdouble(base) ** (-2 * np.arange(half, dtype=np.longdouble) / np.longdouble(max(turn, 1)))
    turns = pos[..., None] * inverse
    cs, sn = np.cos(turns).astype(np.float64)[:, :, None], np.sin(turns).astype(np.float64)[:, :, None]
    A = np.abs if mag else (lambda v: v)
    cs, sn = A(cs) + (1.0 if mag else 0.0), A(sn) + (1.0 if mag else 0.0)  # an angle's own error counts as one more
    sign = 1.0 if mag else -1.0

    def turned(v, back):
        f, s = v[..., :half], v[..., half:turn]
        k = -sign if back else sign
        k = 1.0 if mag else k
        return np.concatenate([f * cs + k * s * sn, s * cs + (1.0 if mag else -k) * f * sn, v[..., turn:]], -1)

    y, dx, dgain = A(x).copy(), A(dy).copy(), np.zeros((len(sections), hd))
    at = 0
    for row, n in enumerate(sections):
        ch = slice(at, at + n)
        v, g = x[:, :, ch], dy[:, :, ch]
        r = 1.0 / np.sqrt((v * v).mean(-1, keepdims=True) + eps) if gain is not None else np.ones(v.shape[:-1] + (1,))
        scale = gain[row].astype(np.float64) if gain is not None else np.ones(hd)
        xhat, scale = A(v) * r, A(scale)
        y[:, :, ch] = turned(xhat * scale, False)
        u = turned(A(g), True)
        dgain[row] = (u * xhat).sum((0, 1, 2))
        mean = (u * scale * xhat).mean(-1, keepdims=True)
        dx[:, :, ch] = r * (u * scale + (1.0 if mag else -1.0) * xhat * mean) if gain is not None else u
        at += n
    return {"y": y, "dx": dx, "dgain": dgain}


def rotary_roundings(x):
    """Sums over the head for the mean square and the mean, some twenty products and the sine and cosine
    (four units each), and dgain's sum over the positions and heads."""
    return 3 * x.shape[3] + 40 + x.shape[0] * x.shape[1] * x.shape[2]


def agree(got, want, size, roundings, dtype, what=""):
    """|got - want| <= roundings * u * size, elementwise, with one step of the smallest normal number."""
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, f"{what}: shape {got.shape}, not {want.shape}"
    assert np.isfinite(got).all(), f"{what}: {np.count_nonzero(~np.isfinite(got))} values are not finite"
    room = roundings * UNIT[dtype] * size + np.finfo(dtype).tiny
    off = np.abs(got - want)
    if not (off <= room).all():
        j = int(np.argmax(off - room))
        raise AssertionError(f"{what}[{j}]: {got.ravel()[j]!r}, not {want.ravel()[j]!r}: off by {off.ravel()[j]:.3e}, room for {room.ravel()[j]:.3e}")


# ---- cases ------------------------------------------------------------------------------------------

# batch, length, width, taps, flags: b bias, s state, l lengths, a activation
CONV_CASES = [(1, 1, 1, 2, ""), (2, 1, 8, 4, "bsa"), (1, 5, 4, 8, "ba"), (2, 7, 64, 3, "bsl"), (3, 33, 65, 4, "bsla"), (1, 32, 256, 4, "a"),
              (2, 70, 260, 5, "sla"), (4, 31, 10, 6, "la"), (2, 129, 12, 7, "bsa"), (1, 3, 516, 8, "bsla"), (5, 40, 77, 2, "bsla")]
# batch, length, width, states, groups, flags: d skip, z gate, s state, l lengths, p softplus
SCAN_CASES = [(1, 1, 1, 1, 1, ""), (2, 1, 8, 4, 1, "dzsp"), (1, 2, 64, 16, 1, "dz"), (2, 15, 65, 16, 1, "dzslp"), (1, 16, 64, 3, 1, "s"),
              (2, 17, 63, 8, 1, "zlp"), (1, 33, 6, 5, 3, "dsp"), (3, 40, 200, 8, 2, "dslp"), (1, 48, 130, 13, 2, "dzp"), (2, 31, 40, 24, 1, "dzslp"),
              (1, 20, 33, 33, 1, "dzs"), (2, 18, 36, 64, 4, "dzslp"), (1, 100, 16, 16, 1, "dzsp"), (2, 64, 4, 17, 2, "zp"), (1, 70, 132, 16, 1, "dzp"),
              (1, 300, 5, 16, 1, "dzsp"), (2, 523, 8, 4, 1, "dzslp")]
# batch, length, sections, passing heads, head, rotary dims, flags: g gain, p own positions, t shared ones, f first ones
ROTARY_CASES = [(1, 1, (1,), 0, 2, 2, "g"), (2, 1, (4, 2), 2, 64, 64, "gp"), (1, 5, (3,), 1, 8, 8, ""), (2, 9, (6, 2), 2, 44, 22, "gp"),
                (1, 33, (1, 1), 0, 16, 0, "g"), (2, 7, (2, 3), 0, 128, 128, "gt"), (1, 3, (5,), 0, 256, 256, "gp"), (1, 4, (2,), 1, 250, 250, "g"),
                (3, 40, (8, 8), 8, 32, 32, "gp"), (1, 6, (1, 2, 3, 1), 0, 10, 6, "gp"), (2, 65, (7,), 0, 24, 8, "p"), (3, 17, (2, 1), 1, 32, 16, "gf")]


def lengths_of(batch, length):
    """Full, empty, one token, then others."""
    return np.array([[length, 0, 1, (length + 1) // 2, length - 1][i % 5] for i in range(batch)], np.int32)


def conv_inputs(case, dtype, seed=0):
    b, t, d, k, flags = case
    r = np.random.default_rng(seed)
    f = lambda *s, m=1.0: (m * r.standard_normal(s)).astype(dtype)  # noqa: E731
    v = {"x": f(b, t, d), "w": f(k, d, m=0.5), "bias": f(d, m=0.3) if "b" in flags else None, "state": f(b, k - 1, d) if "s" in flags else None,
         "dy": f(b, t, d), "dnext": f(b, k - 1, d)}
    return v, lengths_of(b, t) if "l" in flags else None, "a" in flags


def scan_inputs(case, dtype, seed=0):
    b, t, d, n, g, flags = case
    r = np.random.default_rng(seed)
    f = lambda *s, m=1.0: (m * r.standard_normal(s)).astype(dtype)  # noqa: E731
    step = r.uniform(0.01, 0.4, (b, t, d))
    v = {"x": f(b, t, d), "dt": (np.log(np.expm1(step)) if "p" in flags else step).astype(dtype),
         "a": (-np.arange(1, n + 1) * np.exp(0.1 * r.standard_normal((d, n))) * min(1.0, 16.0 / n)).astype(dtype), "b": f(b, t, g, n), "c": f(b, t, g, n),
         "d": f(d) if "d" in flags else None, "z": f(b, t, d) if "z" in flags else None, "state": f(b, d, n) if "s" in flags else None,
         "dy": f(b, t, d), "dlast": f(b, d, n)}
    return v, lengths_of(b, t) if "l" in flags else None, "p" in flags


def rotary_inputs(case, dtype, seed=0):
    b, t, sections, passing, hd, turn, flags = case
    r = np.random.default_rng(seed)
    heads = sum(sections) + passing
    f = lambda *s: r.standard_normal(s).astype(dtype)  # noqa: E731
    pos = None
    if "f" in flags:
        pos = r.integers(-5, 2000000, (b, 1)).astype(np.int32)
    elif "p" in flags:
        pos = (r.integers(-5, 2000000, (b, 1)) + np.arange(t)).astype(np.int32)
    elif "t" in flags:
        pos = (700 + 3 * np.arange(t)).astype(np.int32)
    return {"x": f(b, t, heads, hd), "gain": f(len(sections), hd) if "g" in flags else None, "dy": f(b, t, heads, hd)}, pos


def fill_outside(v, lengths, names):
    """NaN in what the padded positions hold."""
    for i, n in enumerate(lengths):
        for name in names:
            if v[name] is not None:
                v[name][i, n:] = np.nan


def _differentiated(fn, inputs, device):
    """fn(dict of tracers) -> (results, scalar): its results and gradients for the floating inputs."""
    def program(given):
        (_, results), grads = rg.value_and_grad(fn, has_aux=True)(given)
        return results, grads
    tree = {k: rg.tensor(v) for k, v in inputs.items() if v is not None}
    c = rg.compile(lambda g: program(g), (tree,), validate="none", device=device)
    results, grads = c(tree)
    return [r.numpy() for r in results], {k: g.numpy() for k, g in grads.items()}


def check_conv(case, dtype, device):
    v, lengths, silu = conv_inputs(case, dtype)
    dnext = v["dnext"]
    want = conv(v["x"], v["w"], v["bias"], v["state"], lengths, silu, v["dy"], dnext)
    size = conv(v["x"], v["w"], v["bias"], v["state"], lengths, silu, v["dy"], dnext, mag=True)
    k = conv_roundings(v["x"], v["w"])
    if lengths is not None:
        fill_outside(v, lengths, ["x"])
    dy, dn = rg.tensor(v["dy"]), rg.tensor(dnext)

    def fn(g):
        y, nxt = rg.causal_conv(g["x"], g["w"], g.get("bias"), g.get("state"), lengths, "silu" if silu else None)
        return (y * dy).sum() + (nxt * dn).sum(), (y, nxt)

    (y, nxt), grads = _differentiated(fn, {n: v[n] for n in ("x", "w", "bias", "state")}, device)
    agree(y, want["y"], size["y"], k, dtype, "y")
    assert np.array_equal(nxt, want["next"].astype(dtype))
    for name, g in grads.items():
        agree(g, want["d" + name], size["d" + name], k, dtype, "d" + name)


def check_scan(case, dtype, device, with_last=True, joined=False):
    v, lengths, soft = scan_inputs(case, dtype)
    dlast = v["dlast"] if with_last else None
    args = (v["x"], v["dt"], v["a"], v["b"], v["c"], v["d"], v["z"], v["state"], lengths, soft, v["dy"], dlast)
    want, size = scan(*args), scan(*args, mag=True)
    k = scan_roundings(v["x"], v["dt"], v["a"], soft)
    if lengths is not None:
        fill_outside(v, lengths, ["x", "dt", "b", "c", "z"])
    dy, dl = rg.tensor(v["dy"]), rg.tensor(v["dlast"])

    if joined:
        v["b"], v["c"] = np.concatenate([v["b"], v["c"]], 2), None
        want["db"], size["db"] = (np.concatenate([w["db"], w["dc"]], 2) for w in (want, size))

    def fn(g):
        y, last = rg.selective_scan(g["x"], g["dt"], g["a"], g["b"], g.get("c"), g.get("d"), g.get("z"), g.get("state"), lengths, soft)
        return (y * dy).sum() + ((last * dl).sum() if with_last else 0.0), (y, last)

    (y, last), grads = _differentiated(fn, {n: v[n] for n in ("x", "dt", "a", "b", "c", "d", "z", "state")}, device)
    agree(y, want["y"], size["y"], k, dtype, "y")
    agree(last, want["last"], size["last"], k, dtype, "last")
    for name, g in grads.items():
        agree(g, want["d" + name], size["d" + name], k, dtype, "d" + name)


def log_inputs(case, dtype):
    """Inputs of a scan whose rates are given as logarithms and whose steps have a bias, and what the
    formulas then take: the steps before the softplus, and the rates. The sum of a step is off by a
    rounding of |dt| + |bias|, which moves the step by up to that times its value (without a softplus
    all are positive), and a rate by the four units of its exponential: every position's error grows
    by less than (|dt| + |bias| + 4) / 6 of that which scan_roundings counts."""
    v, lengths, soft = scan_inputs(case, dtype)
    r = np.random.default_rng(1)
    bias = (r.standard_normal(case[2]) if soft else r.uniform(0.0, 0.1, case[2])).astype(dtype)
    if soft:
        v["dt"] = v["dt"] - bias
    v["dt_bias"], v["a"] = bias, np.log(-v["a"])
    raw, rates = v["dt"].astype(np.float64) + bias, -np.exp(v["a"].astype(np.float64))
    grown = 1.0 + (float((np.abs(v["dt"]) + np.abs(bias)).max()) + 4.0) / 6.0
    return v, lengths, soft, raw, rates, grown * scan_roundings(v["x"], raw, rates, soft)


def check_scan_of_logs(case, dtype, device, joined=False):
    v, lengths, soft, raw, rates, k = log_inputs(case, dtype)
    args = (v["x"], raw, rates, v["b"], v["c"], v["d"], v["z"], v["state"], lengths, soft, v["dy"], v["dlast"])
    want, size = scan(*args), scan(*args, mag=True)
    for w, sign in ((want, 1.0), (size, -1.0)):
        w["da"], w["ddt_bias"] = sign * w["da"] * rates, w["ddt"].sum((0, 1))
    if lengths is not None:
        fill_outside(v, lengths, ["x", "dt", "b", "c", "z"])
    dy, dl = rg.tensor(v["dy"]), rg.tensor(v["dlast"])
    if joined:
        v["b"], v["c"] = np.concatenate([v["b"], v["c"]], 2), None
        want["db"], size["db"] = (np.concatenate([w["db"], w["dc"]], 2) for w in (want, size))

    def fn(g):
        y, last = rg.selective_scan(g["x"], g["dt"], g["a"], g["b"], g.get("c"), g.get("d"), g.get("z"), g.get("state"), lengths, soft, g["dt_bias"], True)
        return (y * dy).sum() + (last * dl).sum(), (y, last)

    (y, last), grads = _differentiated(fn, {n: v[n] for n in ("x", "dt", "a", "b", "c", "d", "z", "state", "dt_bias")}, device)
    agree(y, want["y"], size["y"], k, dtype, "y")
    agree(last, want["last"], size["last"], k, dtype, "last")
    for name, g in grads.items():
        agree(g, want["d" + name], size["d" + name], k, dtype, "d" + name)


def check_rotary(case, dtype, device):
    b, t, sections, passing, hd, turn, flags = case
    v, pos = rotary_inputs(case, dtype)
    at = np.arange(t) if pos is None else pos + np.arange(t) if pos.shape == (b, 1) else pos
    args = (v["x"], v["gain"], at, sections, turn, 10000.0, 1e-6, v["dy"])
    want, size = rotary(*args), rotary(*args, mag=True)
    k = rotary_roundings(v["x"])
    dy = rg.tensor(v["dy"])

    def fn(g):
        y = rg.rotary_norm(g["x"], g.get("gain"), pos, sections, turn)
        return (y * dy).sum(), (y,)

    (y,), grads = _differentiated(fn, {n: v[n] for n in ("x", "gain")}, device)
    agree(y, want["y"], size["y"], k, dtype, "y")
    if passing:
        assert np.array_equal(y[:, :, sum(sections):], v["x"][:, :, sum(sections):])
        assert np.array_equal(grads["x"][:, :, sum(sections):], v["dy"][:, :, sum(sections):])
    for name, g in grads.items():
        agree(g, want["d" + name], size["d" + name], k, dtype, "d" + name)
