"""Cases for the kernels that the sequence operators run on at larger sizes, which kernel a size runs
on, and what rounding may move a scan's results by, position by position."""

import ctypes

import numpy as np

import sequence_reference as ref

F32, F64 = 0, 1  # rg_dtype
_CODE = {"float32": F32, "float64": F64}


# ---- which kernel a size runs on: the launchers' own arithmetic, which needs no device ---------------

def _ask(name, args, dtype, sizes, result=ctypes.c_uint32):
    """`rgk::name(dtype, const args&)`, whose structure begins with `sizes`."""
    from rustautograd_amd import _native
    f = getattr(ctypes.CDLL(_native.HIP_LIBRARY), f"_ZN3rgk{len(name)}{name}EiRKNS_{len(args)}{args}E")
    f.restype = result
    block = (ctypes.c_uint32 * 128)(*sizes)
    return f(ctypes.c_int(_CODE[dtype]), ctypes.byref(block))


def conv_form(case, dtype):
    """(channels a lane, positions a run) of a convolution."""
    batch, length, width, taps, _ = case
    blocks, rows = (_ask(n, "ConvArgs", dtype, (batch, length, width, taps), t) for n, t in (("conv_blocks", ctypes.c_uint64), ("conv_grad_rows", ctypes.c_uint32)))
    (run,) = [r for r in (1, 4, 8) if batch * -(-length // (4 * r)) == rows and (r == 1) == (length <= 4)]
    (lane,) = [v for v in (1, 2, 4) if rows * -(-width // (64 * v)) == blocks and width % v == 0]
    return lane, run


def scan_chunks(case, dtype):
    """(chunks a sequence, blocks of the gradient over them, positions a chunk)."""
    batch, length, width, states, groups, _ = case
    sizes = (batch, length, width, states, groups, groups)
    tiles = _ask("scan_group_tiles", "ScanArgs", dtype, sizes)
    chunks = _ask("scan_blocks", "ScanArgs", dtype, sizes, ctypes.c_uint64) // (batch * groups * tiles)
    marks = -(-length // 16)
    return chunks, _ask("scan_rows", "ScanArgs", dtype, sizes) // batch, 16 * -(-marks // chunks)


def rotary_blocks(case, dtype):
    """Blocks of the gradient, each a partial row of the gain's."""
    batch, length, sections, passing, head, turn = case[:6]
    return _ask("rotary_grad_rows", "RotaryArgs", dtype, (batch, length, sum(sections) + passing, head, turn, len(sections)))


# ---- convolutions --------------------------------------------------------------------------------------

# As ref.CONV_CASES, with the form that each dtype takes: lanes past the width, runs past the length,
# a second block of channels, and the widest taps with the widest form.
CONV_SIZES = [((16, 1001, 5, 4, "bsl"), (1, 8), (1, 8)), ((16, 1001, 5, 8, "sa"), (1, 8), (1, 8)), ((16, 2021, 130, 8, "bsla"), (2, 8), (2, 8)),
              ((16, 2021, 130, 3, "bl"), (2, 8), (2, 8)), ((16, 2021, 260, 4, "bsl"), (4, 8), (2, 8)), ((16, 2021, 260, 8, "bsla"), (4, 8), (2, 8)),
              ((16, 2021, 260, 2, "a"), (4, 8), (2, 8))]


def conv_whole(case, dtype, seed=0):
    """Operands of whole numbers, whose sums are exact in the dtype (below 2^24)."""
    v, lengths, silu = ref.conv_inputs(case, dtype, seed)
    r = np.random.default_rng(seed + 1)
    return {k: None if a is None else r.integers(-3, 4, a.shape).astype(dtype) for k, a in v.items()}, lengths, silu


def conv(x, w, bias, state, lengths, silu, dy, dnext):
    """Results and gradients in 64 bits, all positions at once, and the magnitudes that their roundings
    count on (as ref.conv with mag=True)."""
    b, t, d = x.shape
    k = w.shape[0]
    n = np.array(ref._ends(lengths, b, t))
    inside = (np.arange(t)[None] < n[:, None])[:, :, None]
    past = np.concatenate([np.zeros((b, k - 1, d)) if state is None else state, np.where(inside, x, 0.0)], 1).astype(np.float64)
    w, dy = w.astype(np.float64), np.where(inside, dy, 0.0).astype(np.float64)
    own = 0.0 if bias is None else bias.astype(np.float64)
    pre = sum(w[j] * past[:, j:j + t] for j in range(k)) + own
    much = sum(np.abs(w[j] * past[:, j:j + t]) for j in range(k)) + np.abs(own)
    g = ref.sigmoid(pre)
    slope = g * (1.0 + pre * (1.0 - g)) if silu else np.ones_like(pre)
    out, size = {}, {}
    out["y"], size["y"] = np.where(inside, pre * g if silu else pre, 0.0), np.where(inside, (1.1 if silu else 1.0) * much, 0.0)
    ends = n[:, None] + np.arange(k - 1)
    out["next"] = np.take_along_axis(past, ends[:, :, None], 1)
    for to, gp, wk, p, more in ((out, dy * slope, w, past, dnext), (size, np.abs(dy) * (np.abs(slope) + 0.5 * much + 1.0), np.abs(w), np.abs(past), np.abs(dnext))):
        dpast = np.zeros_like(past)
        for j in range(k):
            dpast[:, j:j + t] += wk[j] * gp
        for i in range(b):
            dpast[i, n[i]:n[i] + k - 1] += more[i]
        to["dx"], to["dstate"], to["dbias"] = np.where(inside, dpast[:, k - 1:], 0.0), dpast[:, :k - 1], gp.sum((0, 1))
        to["dw"] = np.stack([(gp * p[:, j:j + t]).sum((0, 1)) for j in range(k)])
    return out, size


# ---- scans -----------------------------------------------------------------------------------------------

# As ref.SCAN_CASES, with chunks and blocks of the gradient in float32: more than 32 chunks, blocks of
# several chunks with two and four states a lane and with four in sixteen lanes.
SCAN_SIZES = [((2, 2003, 5, 4, 1, "dzslp"), 42, 42), ((1, 2003, 3, 16, 1, "zp"), 42, 42), ((4, 523, 32, 16, 32, "dzslp"), 7, 4), ((4, 523, 32, 7, 32, "zs"), 7, 4),
              ((4, 523, 32, 40, 32, "dlp"), 7, 4), ((8, 200, 64, 13, 64, "dzp"), 3, 1)]


def scan(x, dt, a, b, c, d, z, state, lengths, soft, dy, dlast, dtype, chunk):
    """({results and gradients}, {what rounding may move each value by}), in 64 bits.

    The second follows every rounding of unit u through the recurrence, so that an error fades as the
    states do. A step's softplus is within 8 u of itself (exponential 4, logarithm 3, their sum 1). A
    decay e^(dt a) has an exponent that the product, the rate's factor and the step move by
    |dt a| times their units, and a power of two within 2 u; where chunks are joined, the sum over
    the steps of a chunk has as many roundings as positions, `chunk`, each of which moves the decay
    over it by up to |sum dt a| u: `chunk` u |dt a| a position, which the decay's own exponent
    counts here; the join's other roundings (5 u) are fewer than the 3 u of its 16 positions or
    more. A gate is within 12 u. Sums over n values count n u of their magnitudes."""
    u = ref.UNIT[dtype]
    x, dt, a, b, c, d, z, state, dy, dlast = (None if v is None else v.astype(np.float64) for v in (x, dt, a, b, c, d, z, state, dy, dlast))
    n_b, length, width = x.shape
    states, per = a.shape[1], width // b.shape[2]
    inside = (np.arange(length)[None] < np.array(ref._ends(lengths, n_b, length))[:, None])[:, :, None]
    x, dt, dy, b, c = (np.where(inside if v.ndim == 3 else inside[..., None], v, 0.0) for v in (x, dt, dy, b, c))
    step = np.where(inside, ref.softplus(dt) if soft else dt, 0.0)
    es = 8 * u if soft else 0.0
    spread = lambda v: np.repeat(v, per, 2)  # noqa: E731
    bt, ct = spread(b), spread(c)
    e = np.exp(step[..., None] * a)
    rel = np.where(inside[..., None], np.abs(step[..., None] * a) * ((chunk + 6) * u + es) + 3 * u, 0.0)
    d = np.zeros(width) if d is None else d
    sig = None if z is None else ref.sigmoid(np.where(inside, z, 0.0))
    z = None if z is None else np.where(inside, z, 0.0)
    gate = np.ones_like(x) if z is None else z * sig
    gate_u = 0.0 if z is None else 12 * u
    h, eh = np.zeros((n_b, length + 1, width, states)), np.zeros((n_b, length + 1, width, states))
    if state is not None:
        h[:, 0] = state
    p, ep = np.zeros_like(e), np.zeros_like(e)
    for t in range(length):
        p[:, t] = e[:, t] * h[:, t]
        ep[:, t] = e[:, t] * eh[:, t] + np.abs(p[:, t]) * rel[:, t]
        add = (step[:, t] * x[:, t])[..., None] * bt[:, t]
        h[:, t + 1] = p[:, t] + add
        eh[:, t + 1] = ep[:, t] + np.abs(add) * (es + 3 * u) + np.where(inside[:, t, :, None], u * np.abs(p[:, t]), 0.0)
    A = np.abs
    raw = (ct * h[:, 1:]).sum(-1) + d * x
    eraw = (A(ct) * eh[:, 1:]).sum(-1) + (states + 4) * u * (A(ct * h[:, 1:]).sum(-1) + A(d * x))
    want = {"y": np.where(inside, raw * gate, 0.0), "last": h[:, length]}
    room = {"y": np.where(inside, eraw * A(gate) + (gate_u + u) * A(raw * gate), 0.0), "last": eh[:, length]}
    if z is not None:
        slope = sig * (1.0 + z * (1.0 - sig))
        want["dz"] = dy * raw * slope
        room["dz"] = A(dy) * (eraw * A(slope) + A(raw) * (12 * u * A(slope) + 10 * u * (1.0 + A(z)) * sig)) + 3 * u * A(want["dz"])
    gy = dy * gate
    egy = (gate_u + 2 * u) * A(gy)
    back, eback = np.zeros((n_b, width, states)), np.zeros((n_b, width, states))
    if dlast is not None:
        back = dlast.copy()
    G, eG = np.zeros_like(e), np.zeros_like(e)
    for t in reversed(range(length)):
        term = gy[:, t, :, None] * ct[:, t]
        G[:, t] = back + term
        eG[:, t] = eback + egy[:, t, :, None] * A(ct[:, t]) + np.where(inside[:, t, :, None], 2 * u * (A(back) + A(term)), 0.0)
        back = e[:, t] * G[:, t]
        eback = e[:, t] * eG[:, t] + A(back) * np.where(inside[:, t, :, None], rel[:, t] + u, 0.0)
    want["dstate"], room["dstate"] = back, eback
    sum_b, esum_b = (G * bt).sum(-1), (eG * A(bt)).sum(-1) + (states + 3) * u * A(G * bt).sum(-1)
    sum_a = (G * p * a).sum(-1)
    esum_a = ((eG * A(p) + A(G) * ep) * A(a)).sum(-1) + (states + 5) * u * A(G * p * a).sum(-1)
    want["dx"] = step * sum_b + gy * d
    room["dx"] = step * esum_b + es * A(step * sum_b) + A(d) * egy + 3 * u * (A(step * sum_b) + A(gy * d))
    part = x * sum_b + sum_a
    epart = A(x) * esum_b + esum_a + 2 * u * (A(x * sum_b) + A(sum_a))
    soft_slope = ref.sigmoid(dt) if soft else np.ones_like(dt)
    want["ddt"] = np.where(inside, part * soft_slope, 0.0)
    room["ddt"] = np.where(inside, epart * soft_slope + 10 * u * A(part * soft_slope), 0.0)
    far = (length + n_b + 64) * u
    s4 = step[..., None]
    want["da"] = (G * p * s4).sum((0, 1))
    room["da"] = ((eG * A(p) + A(G) * ep) * s4 + (es + 3 * u) * A(G * p * s4)).sum((0, 1)) + far * A(G * p * s4).sum((0, 1))
    drive = (step * x)[..., None]
    grouped = lambda v: v.reshape(n_b, length, width // per, per, states).sum(3)  # noqa: E731
    want["db"], want["dc"] = grouped(G * drive), grouped(gy[..., None] * h[:, 1:])
    room["db"] = grouped(eG * A(drive) + A(G * drive) * (es + (per + 6) * u))
    room["dc"] = grouped(egy[..., None] * A(h[:, 1:]) + A(gy[..., None]) * eh[:, 1:] + (per + 6) * u * A(gy[..., None] * h[:, 1:]))
    want["dd"] = (gy * x).sum((0, 1))
    room["dd"] = (egy * A(x) + far * A(gy * x)).sum((0, 1))
    return want, room


def near(got, want, room, dtype, what):
    """Within the room, a hundredth of it more for products of errors, and what results below the
    smallest normal numbers lose."""
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, f"{what}: shape {got.shape}, not {want.shape}"
    off = np.abs(got - want)
    allowed = 1.01 * room + 100 * float(np.finfo(dtype).tiny) + ref.UNIT[dtype] * np.abs(want)
    if not (off <= allowed).all():
        j = int(np.argmax(np.where(np.isfinite(off), off / allowed, np.inf)))
        raise AssertionError(f"{what}[{j}]: {got.ravel()[j]!r}, not {want.ravel()[j]!r}: off by {off.ravel()[j]:.3e}, room for {allowed.ravel()[j]:.3e}")


def check_scan(case, dtype, device, chunk, with_last=True):
    import rustautograd_amd as rg
    v, lengths, soft = ref.scan_inputs(case, dtype)
    want, room = scan(*(v[k] for k in ("x", "dt", "a", "b", "c", "d", "z", "state")), lengths, soft, v["dy"], v["dlast"] if with_last else None, dtype, chunk)
    if lengths is not None:
        ref.fill_outside(v, lengths, ["x", "dt", "b", "c", "z"])
    dy, dl = rg.tensor(v["dy"]), rg.tensor(v["dlast"])

    def fn(g):
        y, last = rg.selective_scan(g["x"], g["dt"], g["a"], g["b"], g["c"], g.get("d"), g.get("z"), g.get("state"), lengths, soft)
        return (y * dy).sum() + ((last * dl).sum() if with_last else 0.0), (y, last)

    (y, last), grads = ref._differentiated(fn, {n: v[n] for n in ("x", "dt", "a", "b", "c", "d", "z", "state")}, device)
    near(y, want["y"], room["y"], dtype, "y")
    near(last, want["last"], room["last"], dtype, "last")
    for name, g in grads.items():
        near(g, want["d" + name], room["d" + name], dtype, "d" + name)
