"""Attention with shaped scores and over a paged cache from the formulas in 64 bits, and for every
value how far roundings of half a step may move it.

With u half a step of the type: a sum of n products is off by at most (n + 2) u of the sum of their
sizes, in whatever order it is formed. A score is such a sum over the head, multiplied by the scale and
log2(e) (rounded), capped (tanh of the scaled sum, within 6 u of itself) and lowered by the slope's
product: `off_s`. A weight is the power of two of the score less the row's logarithm: it moves by the
error of both, which is at most `off_s` over the row twice, by the rounding of that difference, and by
the rounding of the sum over the row. Errors of products and differences follow by their derivatives."""

import math

import numpy as np

import rustautograd_amd as rg

# (batch, length, heads, key heads, head, what, cap): j one operand of q, k and v, c causal, s slopes, d documents, p prefix, l lengths
CASES = [
    (1, 1, 1, 1, 1, "c", 0), (2, 1, 2, 1, 8, "jcs", 5.0), (1, 2, 1, 1, 3, "", 0), (2, 15, 3, 3, 16, "jc", 0), (1, 31, 4, 2, 31, "csl", 3.0),
    (3, 32, 2, 1, 32, "jcdl", 0), (2, 33, 6, 2, 33, "cdp", 8.0), (1, 63, 1, 1, 64, "jp", 0), (2, 64, 4, 4, 64, "jcs", 20.0), (3, 65, 4, 1, 44, "cpl", 4.0),
    (2, 100, 2, 2, 65, "d", 0), (1, 130, 3, 1, 96, "jcsdpl", 6.0), (2, 200, 2, 1, 64, "jcdl", 10.0), (1, 129, 1, 1, 100, "cs", 0), (1, 70, 2, 1, 128, "jcp", 30.0),
    (1, 97, 2, 2, 130, "cl", 0), (1, 50, 2, 1, 256, "jcsd", 12.0), (4, 40, 8, 2, 24, "jcsdl", 0), (5, 70, 2, 2, 20, "sdpl", 2.0),
]
# (batch, new, heads, key heads, head, page, table pages, what, cap): j one operand, s slopes, l lengths
PAGED = [
    (1, 1, 1, 1, 1, 1, 3, "", 0), (2, 1, 4, 1, 16, 8, 5, "js", 0), (3, 1, 8, 2, 64, 24, 20, "jl", 10.0), (2, 3, 6, 3, 40, 7, 13, "sl", 4.0), (1, 17, 2, 1, 33, 16, 9, "j", 0),
    (4, 1, 16, 1, 64, 64, 12, "js", 20.0), (2, 70, 4, 2, 64, 64, 6, "jl", 0), (1, 1, 8, 2, 128, 100, 41, "s", 0), (2, 5, 3, 1, 96, 32, 11, "jsl", 7.0), (1, 2, 2, 2, 256, 5, 60, "j", 0),
    (1, 1, 2, 1, 64, 256, 24, "js", 0), (3, 40, 1, 1, 130, 10, 9, "l", 3.0), (2, 20, 4, 2, 100, 9, 50, "js", 5.0), (2, 30, 2, 1, 128, 33, 12, "jl", 0),
    (1, 20, 4, 2, 40, 8, 5, "js", 0),
]
# Enough blocks for the device's other forms: 64 rows a block, a group's heads in one part, and in two of four.
LARGE = [(8, 256, 16, 4, 32, "jcsl", 5.0), (8, 250, 16, 16, 64, "jcp", 0), (8, 256, 32, 16, 16, "cd", 9.0), (8, 256, 32, 8, 20, "jcs", 0), (2, 300, 64, 64, 50, "jd", 0)]


def inputs(case, dtype, seed=0):
    b, t, h, g, hd, what, _ = case
    r = np.random.default_rng(1000 * seed + b * 7919 + t * 31 + h * 17 + g * 5 + hd)
    v = {k: r.standard_normal((b, t, n, hd)).astype(dtype) * dtype.type(1.2) for k, n in (("q", h), ("k", g), ("v", g))}
    v["dy"] = r.standard_normal((b, t, h, hd)).astype(dtype)
    v["slopes"] = np.exp2(-np.arange(1, h + 1) * 4.0 / h).astype(dtype) if "s" in what else None
    v["documents"] = v["prefix"] = v["lengths"] = None
    if "d" in what:
        ids = 5 - np.sort(r.integers(0, 3, (b, t)), axis=1)
        ids[:, t // 2:t // 2 + 3] = -2  # a few that belong to none
        v["documents"] = ids.astype(np.int32)
    if "p" in what:
        v["prefix"] = r.integers(0, t + 1, b).astype(np.int32)
    if "l" in what:
        n = r.integers(0, t + 1, b).astype(np.int32)
        n[0] = t
        if b > 2:
            n[1], n[2] = 0, 2 * t  # none, and more than there are
        v["lengths"] = n
    return v


def inside(case, v):
    b, t = case[:2]
    ok = np.ones((b, t), bool)
    if v["lengths"] is not None:
        ok &= np.arange(t) < v["lengths"][:, None]
    if v["documents"] is not None:
        ok &= v["documents"] >= 0
    return ok


def seen(case, v):
    b, t = case[:2]
    at = np.arange(t)
    s = np.broadcast_to((at[None] <= at[:, None]) if "c" in case[5] else np.ones((t, t), bool), (b, t, t)).copy()
    if v["prefix"] is not None:
        s |= at[None, None] < v["prefix"][:, None, None]
    if v["documents"] is not None:
        s &= v["documents"][:, :, None] == v["documents"][:, None, :]
    ok = inside(case, v)
    return s & ok[:, :, None] & ok[:, None, :]


def head(q, k, v, see, distance, scale, cap, slope, u, dy=None):
    """Values of one head and how far they may be off, in 64 bits: (y, off y) or, with a cotangent,
    (dq, dk, dv, dslope) and theirs."""
    q, k, v = (np.where(np.isfinite(x), x, 0.0).astype(np.float64) for x in (q, k, v))
    n, length = q.shape[1], k.shape[0]
    dot, size = scale * (q @ k.T), abs(scale) * (np.abs(q) @ np.abs(k).T)
    off = (n + 5) * u * size
    if cap:
        t = np.tanh(dot / cap)
        off_t = off / cap + 6 * u * np.abs(t)
        s, bend, off_bend = cap * t, 1 - t * t, 2 * np.abs(t) * off_t + 3 * u
        off = cap * off_t + 2 * u * np.abs(s)
    else:
        s, bend, off_bend = dot, np.ones_like(dot), np.zeros_like(dot)
    off = off + 4 * u * np.abs(slope) * distance + u * (np.abs(s) + np.abs(slope) * distance)
    s = np.where(see, s - slope * distance, -np.inf)
    any_ = see.any(1)
    top = np.where(any_, s.max(1, initial=-np.inf), 0.0)
    e = np.exp(s - top[:, None])
    z = np.where(any_, e.sum(1), 1.0)
    p = e / z[:, None]
    gap = np.where(see, np.abs(s - top[:, None]) + np.log(z)[:, None] + np.abs(top)[:, None], 0.0)
    rel = 2 * np.where(see, off, 0.0).max(1, initial=0.0)[:, None] + 4 * u * gap + (length + 12) * u
    y = p @ v
    off_y = (p * (rel + (length + 4) * u)) @ np.abs(v) + u * np.abs(y)
    if dy is None:
        return y, off_y
    dy = np.where(np.isfinite(dy), dy, 0.0).astype(np.float64)
    dp, size_dp = dy @ v.T, np.abs(dy) @ np.abs(v).T
    d = (y * dy).sum(1)[:, None]
    off_dp = (n + 3) * u * size_dp + (n + 3) * u * (np.abs(y) * np.abs(dy)).sum(1)[:, None] + (off_y * np.abs(dy)).sum(1)[:, None]
    ds = p * (dp - d)
    off_ds = p * (np.abs(dp - d) * (rel + 3 * u) + off_dp)
    du, off_du = ds * bend, off_ds * bend + np.abs(ds) * (off_bend + 2 * u)
    total = len(q) + length + 6
    sums = lambda w, off_w, x: (w @ x, off_w @ np.abs(x) + total * u * (np.abs(w) @ np.abs(x)))
    dq, off_dq = sums(du, off_du, k)
    dk, off_dk = sums(du.T, off_du.T, q)
    dv, off_dv = sums(p.T, (p * rel).T, dy)
    dslope = -(ds * distance).sum()
    off_slope = (off_ds * distance).sum() + 2 * total * u * (np.abs(ds) * distance).sum()
    return (scale * dq, scale * dk, dv, dslope), (abs(scale) * off_dq, abs(scale) * off_dk, off_dv, off_slope)


def expected(case, v, dtype, grad):
    """Every result and its bound, as dicts."""
    b, t, h, g, hd, _, cap = case
    u = np.finfo(dtype).eps / 2
    see, scale, distance = seen(case, v), 1 / math.sqrt(hd), np.abs(np.arange(t)[:, None] - np.arange(t)).astype(float)
    names = ("q", "k", "v", "slopes") if grad else ("y",)
    shapes = {"q": (b, t, h, hd), "k": (b, t, g, hd), "v": (b, t, g, hd), "slopes": (h,), "y": (b, t, h, hd)}
    want, off = ({n: np.zeros(shapes[n]) for n in names} for _ in range(2))
    for i in range(b):
        for j in range(h):
            of = j // (h // g)
            slope = 0.0 if v["slopes"] is None else float(v["slopes"][j])
            x, o = head(v["q"][i, :, j], v["k"][i, :, of], v["v"][i, :, of], see[i], distance, scale, cap, slope, u, v["dy"][i, :, j] if grad else None)
            for into, part in ((want, x), (off, o)):
                if not grad:
                    into["y"][i, :, j] = part
                    continue
                into["q"][i, :, j] += part[0]
                into["k"][i, :, of] += part[1]
                into["v"][i, :, of] += part[2]
                into["slopes"][j] += part[3]
    return want, off


def agree(got, want, off, dtype, what):
    assert got.dtype == dtype and got.shape == want.shape, what
    bound = off + np.finfo(dtype).eps / 2 * np.abs(want) + np.finfo(dtype).tiny
    far = ~(np.abs(got - want) <= bound)  # NaN is far
    assert not far.any(), f"{what}: {int(far.sum())} of {far.size} off, first at {np.argwhere(far)[0]}: {got[far][0]} for {want[far][0]} within {bound[far][0]}"


def call(case, x, v):
    _, _, h, g, _, what, cap = case
    q, k, val = (x["x"], None, None) if "j" in what else (x["q"], x["k"], x["v"])
    return rg.attention(q, k, val, heads=(h, g) if "j" in what else None, causal="c" in what, cap=cap or None, slopes=x.get("slopes"),
                        documents=v["documents"], prefix=v["prefix"], lengths=v["lengths"])


def given(case, v):
    """The differentiable operands as tensors, NaN in what lies outside."""
    ok = inside(case, v)
    x = {}
    for k in ("q", "k", "v", "dy"):
        x[k] = v[k].copy()
        x[k][~ok] = np.nan
    dy = x.pop("dy")
    if "j" in case[5]:
        x = {"x": np.concatenate([x["q"], x["k"], x["v"]], axis=2)}
    if v["slopes"] is not None:
        x["slopes"] = v["slopes"]
    return {k: rg.tensor(a) for k, a in x.items()}, rg.tensor(dy)


def check(case, dtype, device):
    dtype = np.dtype(dtype)
    v = inputs(case, dtype)
    x, dy = given(case, v)
    program = rg.compile(lambda x: call(case, x, v), (x,), validate="none", device=device)
    want, off = expected(case, v, dtype, False)
    agree(program(x).numpy(), want["y"], off["y"], dtype, "y")
    slopes = rg.compile(lambda x, dy: rg.grad(lambda x: (call(case, x, v) * dy).sum())(x), (x, dy), validate="none", device=device)
    got = {k: t.numpy() for k, t in slopes(x, dy).items()}
    want, off = expected(case, v, dtype, True)
    h, g = case[2:4]
    if "j" in case[5]:
        got["q"], got["k"], got["v"] = np.split(got.pop("x"), [h, h + g], axis=2)
    for k in got:
        agree(got[k], want[k], off[k], dtype, "d" + k)


def check_each_alone(case, dtype, device):
    """The gradient in one operand alone is that of all of them."""
    dtype = np.dtype(dtype)
    case = (*case[:5], case[5].replace("j", ""), case[6])
    v = inputs(case, dtype)
    x, dy = {k: rg.tensor(v[k]) for k in ("q", "k", "v", "slopes")}, rg.tensor(v["dy"])
    grads = lambda names: rg.compile(lambda x: rg.grad(lambda part: (call(case, {**x, **part}, v) * dy).sum())({k: x[k] for k in names}), (x,), validate="none", device=device)(x)
    want = grads(tuple(x))
    for k in x:
        assert np.array_equal(grads((k,))[k].numpy(), want[k].numpy()), k


# Of CASES, and where values that are no numbers stand: their place as a share of the length.
ODD = [(CASES[i], at) for i, at in ((5, 0.3), (6, 0.9), (8, 0.6), (9, 0.2), (11, 0.7), (12, 0.3), (14, 0.5), (15, 0.4), (16, 0.8))] + [(LARGE[1], 0.5), (LARGE[3], 0.9)]


def check_odd(case, at, bad, dtype, device):
    """Infinities and NaN in one position of the first sequence reach what sees it and nothing else: its key
    and value the queries that see it and, through them, the keys that those see; its query and the
    gradient of its result the keys that it sees."""
    dtype = np.dtype(dtype)
    case = (*case[:5], case[5].replace("j", ""), case[6])
    v, see, p = inputs(case, dtype), seen(case, inputs(case, dtype)), int(at * case[1])
    assert see[0, p, p]
    program = rg.compile(lambda x: call(case, x, v), ({k: rg.tensor(v[k]) for k in ("q", "k", "v", "slopes") if v[k] is not None},), validate="none", device=device)

    def agrees(got, want, off, reached, what):
        agree(np.where(reached[..., None, None], dtype.type(0), got), np.where(reached[..., None, None], 0.0, want), off, dtype, what)
        if np.isnan(bad):
            assert np.isnan(got[reached]).all(), what

    for where in (("k", "v"), ("v",), ("q", "dy"), ("dy",)):
        x = {k: v[k].copy() for k in ("q", "k", "v", "dy", "slopes") if v[k] is not None}
        for k in where:
            x[k][0, p, :, 1:] = bad
        dy, x = rg.tensor(x["dy"]), {k: rg.tensor(a) for k, a in x.items() if k != "dy"}
        queries = np.zeros(see.shape[:2], bool)
        queries[0] = see[0, :, p] if "v" in where else np.arange(case[1]) == p
        keys = (see & queries[:, :, None]).any(1)
        y, want, off = program(x).numpy(), *expected(case, v, dtype, False)
        if "dy" in where:
            agrees(y, want["y"], off["y"], queries & ("q" in where), "y")
        else:
            column = 0 if "k" in where else 1  # of values alone the others' columns are as they were
            agree(y[..., :column], want["y"][..., :column], off["y"][..., :column], dtype, "y")
            agrees(y[..., column:], want["y"][..., column:], off["y"][..., column:], queries, "y")
        grads = rg.compile(lambda x, dy: rg.grad(lambda x: (call(case, x, v) * dy).sum())(x), (x, dy), validate="none", device=device)(x, dy)
        want, off = expected(case, v, dtype, True)
        for k, reached in (("q", queries), ("k", keys)):
            agrees(grads[k].numpy(), want[k], off[k], reached, "d" + k)
        got = grads["v"].numpy()
        agree(np.where(keys[..., None, None], dtype.type(0), got), np.where(keys[..., None, None], 0.0, want["v"]), off["v"], dtype, "dv")


# ---- over a paged cache ------------------------------------------------------------------------------

def paged_inputs(case, dtype, seed=0):
    b, t, h, g, hd, page, n, what, _ = case
    r = np.random.default_rng(seed + b * 7919 + t * 31 + h * 17 + hd)
    v = {k: r.standard_normal((b, t, m, hd)).astype(dtype) for k, m in (("q", h), ("k", g), ("v", g))}
    pages = b * n + 2
    v["k_pages"], v["v_pages"] = (r.standard_normal((pages, page, g, hd)).astype(dtype) for _ in range(2))
    v["table"] = r.permutation(pages)[:b * n].reshape(b, n).astype(np.int32)
    room = n * page
    v["first"] = r.integers(0, max(1, room - t + 1), b).astype(np.int32)
    v["first"][0] = max(0, room - t)  # a full table
    if b > 1:
        v["first"][-1] = 0
    v["slopes"] = np.exp2(-np.arange(1, h + 1) * 6.0 / h).astype(dtype) if "s" in what else None
    v["lengths"] = None
    if "l" in what:
        v["lengths"] = r.integers(0, t + 1, b).astype(np.int32)
        v["lengths"][0] = t
    return v


def paged_expected(case, v, dtype):
    b, t, h, g, hd, page, n, _, cap = case
    u, scale, room, pages = np.finfo(dtype).eps / 2, 1 / math.sqrt(hd), n * page, len(v["k_pages"])
    y, off = np.zeros((b, t, h, hd)), np.zeros((b, t, h, hd))
    k_pages, v_pages = v["k_pages"].copy(), v["v_pages"].copy()

    def place(i, p):
        return None if p >= room or not 0 <= v["table"][i, p // page] < pages else (v["table"][i, p // page], p % page)

    for i in range(b):
        first, count = max(0, int(v["first"][i])), t if v["lengths"] is None else min(max(0, int(v["lengths"][i])), t)
        old = [p for p in range(min(first, room)) if place(i, p)]
        at = np.array(old + [first + j for j in range(count)])
        keys, values = (np.concatenate([np.array([pages_[place(i, p)] for p in old]).reshape(-1, g, hd), new[i, :count]])
                        for pages_, new in ((v["k_pages"], v["k"]), (v["v_pages"], v["v"])))
        distance = (first + np.arange(count))[:, None] - at[None]
        for j in range(h if count else 0):
            of = j // (h // g)
            slope = 0.0 if v["slopes"] is None else float(v["slopes"][j])
            y[i, :count, j], off[i, :count, j] = head(v["q"][i, :count, j], keys[:, of], values[:, of], distance >= 0, np.abs(distance).astype(float), scale, cap, slope, u)
        for j in range(count):
            if place(i, first + j):
                k_pages[place(i, first + j)], v_pages[place(i, first + j)] = v["k"][i, j], v["v"][i, j]
    return y, off, k_pages, v_pages


def paged_call(case, x):
    _, _, h, g, _, _, _, what, cap = case
    q, k, v = (x["x"], None, None) if "j" in what else (x["q"], x["k"], x["v"])
    return rg.paged_attention(q, k, v, heads=(h, g) if "j" in what else None, cache=(x["k_pages"], x["v_pages"]), table=x["table"], first=x["first"],
                              lengths=x.get("lengths"), cap=cap or None, slopes=x.get("slopes"))


def paged_given(case, v):
    x = {k: a for k, a in v.items() if a is not None}
    if "j" in case[7]:
        x["x"] = np.concatenate([x.pop("q"), x.pop("k"), x.pop("v")], axis=2)
    return {k: rg.tensor(a) for k, a in x.items()}


def check_paged(case, dtype, device, change=None):
    dtype = np.dtype(dtype)
    v = paged_inputs(case, dtype)
    if change:
        change(v)
    x = paged_given(case, v)
    program = rg.compile(lambda x: paged_call(case, x), (x,), validate="none", device=device)
    y, (k_pages, v_pages) = program(x)
    want, off, want_k, want_v = paged_expected(case, v, dtype)
    agree(y.numpy(), want, off, dtype, "y")
    assert np.array_equal(k_pages.numpy(), want_k, equal_nan=True) and np.array_equal(v_pages.numpy(), want_v, equal_nan=True)
    assert np.array_equal(x["k_pages"].numpy(), v["k_pages"], equal_nan=True)


def past_the_table(v):
    """More positions before the new tokens than the table has room for."""
    v["first"][0] = v["table"].shape[1] * v["k_pages"].shape[1] + 5


def strange_tables(v):
    """Entries that are no page, a first position past the table, and one before it begins."""
    v["table"][0, 0] = -1
    v["table"][0, -1] = 1 << 30
    v["first"][0] += 1  # the last new token has no row
    if len(v["first"]) > 1:
        v["table"][-1, :] = np.iinfo(np.int32).min
        v["first"][-1] = -3


def check_odd_token(case, bad, dtype, device):
    """Infinities and NaN in the last new token of the first sequence reach its own row alone."""
    dtype = np.dtype(dtype)
    case = (*case[:7], case[7].replace("j", ""), case[8])
    v = paged_inputs(case, dtype)
    clean = paged_expected(case, v, dtype)
    last = case[1] - 1
    for where in (("k", "v"), ("v",)):
        x = {k: a.copy() for k, a in v.items() if a is not None}
        for k in where:
            x[k][0, last] = bad
        y, (k_pages, v_pages) = rg.compile(lambda x: paged_call(case, x), (paged_given(case, x),), validate="none", device=device)(paged_given(case, x))
        got, want = y.numpy(), clean[0].copy()
        assert not np.isfinite(got[0, last]).any()
        got[0, last] = want[0, last] = 0
        agree(got, want, clean[1], dtype, "y")
        assert np.isfinite(k_pages.numpy()).all() == ("k" not in where) and not np.isfinite(v_pages.numpy()).all()
