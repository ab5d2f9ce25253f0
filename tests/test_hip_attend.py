"""The kernels of attention with shaped scores, of its paged form and of the joint norm on the device:
values and gradients against the formulas in 64 bits, captured and replayed step loops against the
same steps one by one, and the operators run together."""

import numpy as np
import pytest

import rustautograd_amd as rg
from rustautograd_amd import nn, optim, random
import attention_reference as ref

pytestmark = pytest.mark.gpu
F = np.float32


def _takes(head, dtype):
    """The device takes float64 heads of up to 128 values and says so of others."""
    return dtype == "float32" or head <= 128


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", ref.CASES, ids=str)
def test_attention(case, dtype):
    if _takes(case[4], dtype):
        ref.check(case, dtype, "hip")
    else:
        with pytest.raises(rg.DiagnosticError, match="at most 128"):
            ref.check(case, dtype, "hip")


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", ref.PAGED, ids=str)
def test_paged_attention(case, dtype):
    if _takes(case[4], dtype):
        ref.check_paged(case, dtype, "hip")
    else:
        with pytest.raises(rg.DiagnosticError, match="at most 128"):
            ref.check_paged(case, dtype, "hip")


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("case, at", ref.ODD, ids=str)
def test_what_is_no_number_reaches_what_sees_it(case, at, bad, dtype):
    if not _takes(case[4], dtype):
        pytest.skip("refused")
    ref.check_odd(case, at, bad, dtype, "hip")


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("case", [ref.PAGED[i] for i in (3, 4, 6, 9, 11, 13)], ids=str)
def test_a_token_that_is_no_number(case, bad, dtype):
    if not _takes(case[4], dtype):
        pytest.skip("refused")
    ref.check_odd_token(case, bad, dtype, "hip")


@pytest.mark.parametrize("case", [ref.CASES[i] for i in (6, 11, 18)], ids=str)
def test_a_gradient_alone(case):
    case = (*case[:5], case[5] + "s" * ("s" not in case[5]), case[6])
    ref.check_each_alone(case, "float32", "hip")


@pytest.mark.parametrize("case", [ref.PAGED[i] for i in (1, 2, 3, 6)], ids=str)
def test_pages_that_are_not_there(case):
    ref.check_paged(case, "float32", "hip", ref.strange_tables)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", [ref.PAGED[i] for i in (1, 3, 14)], ids=str)
def test_positions_past_the_table(case, dtype):
    ref.check_paged(case, dtype, "hip", ref.past_the_table)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", ref.LARGE, ids=str)
def test_attention_of_many_blocks(case, dtype):
    ref.check(case, dtype, "hip")


@pytest.mark.parametrize("length, heads", [(4500, 8), (8400, 2)])
def test_documents_over_many_stages(length, heads):
    """Stages without a document of the block's are left out, also past the 64 that are looked at at
    once; one document comes back at the end."""
    r = np.random.default_rng(length)
    case = (1, length, heads, 1, 16, "jcsd", 3.0)
    ids = np.repeat(np.arange(length // 40 + 1), r.integers(1, 80, length // 40 + 1))[:length]
    ids = np.concatenate([ids, np.full(length - len(ids), ids.max() + 1)]).astype(np.int32)
    ids[-20:] = 0
    ids[500:700] = -1
    v = {k: r.standard_normal((1, length, n, 16)).astype(F) for k, n in (("q", heads), ("k", 1), ("v", 1), ("dy", heads))}
    v.update(slopes=np.exp2(-np.arange(1, heads + 1.0)).astype(F), documents=ids[None], prefix=None, lengths=None)
    x, dy = ref.given(case, v)
    y = rg.compile(lambda x: ref.call(case, x, v), (x,), validate="none")(x).numpy()
    grads = rg.compile(lambda x, dy: rg.grad(lambda x: (ref.call(case, x, v) * dy).sum())(x), (x, dy), validate="none")(x, dy)
    dx = np.split(grads["x"].numpy(), [heads, heads + 1], axis=2)
    u, dtype, slopes, off_slopes = np.finfo(F).eps / 2, np.dtype(F), np.zeros(heads), np.zeros(heads)
    for d in np.unique(ids):
        at = np.flatnonzero(ids == d)
        if d < 0:
            assert not y[0, at].any() and not any(g[0, at].any() for g in dx)
            continue
        apart = at[:, None] - at[None]
        want, off = {n: np.zeros((len(at), 16)) for n in "kv"}, {n: np.zeros((len(at), 16)) for n in "kv"}
        for h in range(heads):
            args = v["q"][0, at, h], v["k"][0, at, 0], v["v"][0, at, 0], apart >= 0, np.abs(apart).astype(float), 0.25, 3.0, float(v["slopes"][h]), u
            ref.agree(y[0, at, h], *ref.head(*args), dtype, "y")
            g, o = ref.head(*args, v["dy"][0, at, h])
            ref.agree(dx[0][0, at, h], g[0], o[0], dtype, "dq")
            for n, k in (("k", 1), ("v", 2)):
                want[n] += g[k]
                off[n] += o[k]
            slopes[h] += g[3]
            off_slopes[h] += o[3]
        ref.agree(dx[1][0, at, 0], want["k"], off["k"], dtype, "dk")
        ref.agree(dx[2][0, at, 0], want["v"], off["v"], dtype, "dv")
    ref.agree(grads["slopes"].numpy(), slopes, off_slopes, dtype, "dslopes")


def test_pages_past_32_bits():
    """A cache of 4.9 GB each way, made on the device, whose last pages the table names: the rows that a
    small cache of the same values gives."""
    r = np.random.default_rng(5)
    page, g, hd, pages = 256, 4, 64, 18700
    x, base = (rg.tensor(r.standard_normal(s).astype(F)) for s in ((1, 1, 3 * g, hd), (1, page, g, hd)))
    names = [pages - 1, 3, pages - 2]

    def step(x, base, table, which):
        cache = tuple(base * s + (which * 2.0 ** -15).reshape(-1, 1, 1, 1) for s in (1.0, -0.5))
        return rg.paged_attention(x, cache=cache, table=table, first=np.array([700], np.int32), heads=(g, g))[0]

    def at(table, which):
        args = x, base, rg.tensor(np.array([table], np.int32)), rg.tensor(np.array(which, F))
        return rg.compile(step, args, validate="none")(*args).numpy()

    # One split more or less sums in another order: a few roundings of values near 1.
    np.testing.assert_allclose(at(names, np.arange(pages)), at([0, 1, 2], names), rtol=0, atol=2e-6)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("sizes", [(1,), (3, 16384, 16385), (100000, 1, 7), tuple(range(1, 131)), tuple(range(4090, 4400))], ids=len)
def test_norm(sizes, dtype):
    r = np.random.default_rng(len(sizes))
    parts = [r.standard_normal(n).astype(dtype) for n in sizes]
    got = float(optim.gradient_norm([rg.tensor(p) for p in parts]))
    want = np.sqrt(sum((p.astype(np.longdouble) ** 2).sum() for p in parts))
    # Sums of squares in 64 bits: at most the number of terms in roundings of 2^-53, far below one of
    # float32; the root halves them.
    assert abs(got - want) <= (np.finfo(dtype).eps + sum(sizes) * 2.0 ** -53) * want


# ---- step loops ---------------------------------------------------------------------------------------

def _tokens(seed=0, batch=3, dtype="float32"):
    """A cache, the tokens to go on from, and a step that reads and appends and makes the next tokens."""
    r = np.random.default_rng(seed)
    h, g, hd, page, n = 4, 2, 24, 7, 6
    pages = r.permutation(batch * n + 1)[:batch * n].reshape(batch, n).astype(np.int32)
    state = {"x": r.standard_normal((batch, 1, h + 2 * g, hd)), "k": r.standard_normal((batch * n + 1, page, g, hd)),
             "v": r.standard_normal((batch * n + 1, page, g, hd)), "first": np.array([20, 0, 6][:batch], np.int32)}
    state = {k: rg.tensor(v if v.dtype == np.int32 else v.astype(dtype)) for k, v in state.items()}
    data = {"table": rg.tensor(pages), "drive": rg.tensor(r.standard_normal((batch, 1, h + 2 * g, hd)).astype(dtype))}

    def step(s, data):
        y, (k, v) = rg.paged_attention(s["x"], cache=(s["k"], s["v"]), table=data["table"], first=s["first"], heads=(h, g), cap=9.0)
        x = rg.tanh(0.5 * rg.concatenate([y, y], axis=2) + data["drive"])
        return {"x": x, "k": k, "v": v, "first": s["first"] + 1}

    return state, data, step


def _same(got, want):
    for k in want:
        assert np.array_equal(got[k].numpy(), want[k].numpy(), equal_nan=True), k


def _one_by_one(step, state, data, steps):
    program = rg.compile(step, (state, data), validate="none")
    for _ in range(steps):
        out = program(state, data)
        state = out[0] if isinstance(out, tuple) else out
    return state


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("kind", ["carried", "watched", "read twice"])
def test_a_cache_carried_by_a_loop(kind, dtype, monkeypatch):
    """The loop writes new rows where the pages are, unless something else reads them; either way it does
    what single calls do, in one run and in several, also of an odd number of steps."""
    state, data, plain = _tokens(dtype=dtype)
    seen = {"carried": lambda s, new: new["x"].sum(), "watched": lambda s, new: (new["x"].sum() + s["k"].sum(), s["v"]),
            "read twice": lambda s, new: (rg.paged_attention(s["x"], cache=(s["k"], s["k"]), table=data["table"], first=s["first"], heads=(4, 2))[0]).sum()}[kind]

    def step(s, data):
        new = plain(s, data)
        return new, seen(s, new)

    want = _one_by_one(step, state, data, 7)
    program = rg.compile(step, (state, data), validate="none")
    _same(rg.run(program, state, [data], steps=7).state, want)
    now = state
    for steps in (3, 1, 2, 1):
        now = rg.run(program, now, [data], steps=steps).state
        float(rg.ones(5).sum())  # the program's own work between
    _same(now, want)
    monkeypatch.setenv("RG_HIP_GRAPHS", "0")
    _same(rg.run(program, state, [data], steps=7).state, want)


def test_a_cache_in_a_loop_that_stops():
    """A value that is not finite ends the run after its step; the pages are those of that step."""
    state, data, plain = _tokens(1)

    def step(s, data):
        new = plain(s, data)
        return new, 1.0 / (24 - new["first"][0]).cast("float32")

    program = rg.compile(step, (state, data), validate="none")
    r = rg.run(program, state, [data], steps=90)
    assert len(r.history["aux"]) == 4
    _same(r.state, _one_by_one(plain, state, data, 4))


def test_cycled_tables_and_batches():
    """A table for every step: rows go where the step's own table says."""
    state, data, step = _tokens(2)
    other = {**data, "table": rg.tensor(data["table"].numpy()[::-1].copy())}
    program = rg.compile(step, (state, data), validate="none")
    want = state
    for k in range(5):
        want = program(want, (data, other)[k % 2])
    _same(rg.run(program, state, [data, other], steps=5).state, want)


def test_rows_written_twice_keep_the_later_sequence():
    for seed in range(3):
        case = (6, 3, 2, 1, 16, 4, 3, "j", 0)

        def share(v):
            r = np.random.default_rng(seed)
            v["table"][:] = r.integers(0, 5, v["table"].shape)
            v["first"][:] = r.integers(0, 10, 6)

        v = ref.paged_inputs(case, np.dtype("float32"))
        share(v)
        x = ref.paged_given(case, v)
        _, (k, held) = rg.compile(lambda x: ref.paged_call(case, x), (x,), validate="none")(x)
        _, _, want_k, want_v = ref.paged_expected(case, v, np.dtype("float32"))
        assert np.array_equal(k.numpy(), want_k) and np.array_equal(held.numpy(), want_v)


def test_training_loop_with_every_mask_and_the_clip():
    """Captured and replayed steps against the same steps one by one."""
    case = (3, 75, 4, 2, 40, "jcsdpl", 7.0)
    v = ref.inputs(case, np.dtype("float32"))
    x = {"x": rg.tensor(np.concatenate([v["q"], v["k"], v["v"]], axis=2)), "slopes": rg.tensor(v["slopes"])}
    t = rg.tensor(v["dy"])

    def step(s, t):
        def loss(s):
            off = ref.call(case, s, v) - t
            return (off * off).sum()

        value, grads = rg.value_and_grad(loss)(s)
        grads, norm = optim.clip_gradients(grads, 3.0)
        return {k: s[k] - 0.05 * grads[k] for k in s}, (value, norm)

    program = rg.compile(step, (x, t), validate="none")
    run = rg.run(program, x, [t], steps=6)
    s, losses, norms = x, [], []
    for _ in range(6):
        s, (value, norm) = program(s, t)
        losses.append(float(value))
        norms.append(float(norm))
    _same(run.state, s)
    assert run.history["aux.0"] == losses and run.history["aux.1"] == norms
    _same(rg.run(program, x, [t], steps=6).state, s)


def test_attention_inside_a_scan_body():
    case = (2, 37, 2, 1, 32, "jcd", 4.0)
    v = ref.inputs(case, np.dtype("float32"))
    x = rg.tensor(np.concatenate([v["q"], v["k"], v["v"]], axis=2))
    body = lambda c, _: (rg.concatenate([ref.call(case, {"x": c}, v), c[:, :, 2:]], axis=2), c[:, :, :1].sum())
    direct = x
    for _ in range(3):
        direct = rg.compile(lambda c: body(c, None)[0], (direct,), validate="none")(direct)
    looped, _ = rg.compile(lambda c: rg.scan(body, c, rg.zeros(3)), (x,), validate="none")(x)
    assert np.array_equal(looped.numpy(), direct.numpy())


def test_tokens_continue_what_attention_reads_at_once():
    """Prompt in a chunk, then token by token over the pages: the rows of one attention over all."""
    r = np.random.default_rng(4)
    b, t, h, g, hd, page = 2, 45, 4, 2, 32, 8
    x = r.standard_normal((b, t, h + 2 * g, hd)).astype(F)
    slopes = rg.tensor(np.array([0.5, 0.2, 0.1, 0.05], F))
    whole = rg.attention(rg.tensor(x), heads=(h, g), cap=6.0, slopes=slopes).numpy()
    cache = tuple(rg.zeros((b * 6, page, g, hd)) for _ in range(2))
    table = rg.tensor(r.permutation(b * 6).reshape(b, 6).astype(np.int32))
    out, at = [], 0
    for n in (30, 1, 1, 5, 1, 7):
        first = rg.tensor(np.full(b, at, np.int32))
        y, cache = rg.paged_attention(rg.tensor(x[:, at:at + n].copy()), cache=cache, table=table, first=first, heads=(h, g), cap=6.0, slopes=slopes)
        out.append(y.numpy())
        at += n
    case = (b, t, h, g, hd, "jcs", 6.0)
    v = {"q": x[:, :, :h], "k": x[:, :, h:h + g], "v": x[:, :, h + g:], "slopes": slopes.numpy(), "documents": None, "prefix": None, "lengths": None}
    want, off = ref.expected(case, v, np.dtype("float32"), False)
    ref.agree(np.concatenate(out, axis=1), want["y"], off["y"], np.dtype("float32"), "y")
    ref.agree(whole, want["y"], off["y"], np.dtype("float32"), "y")


def test_a_block_trained_and_then_served():
    """A block of grouped, capped, turned heads under documents trains with the clip, and is then read
    over pages, a prompt and single tokens in a captured loop; the device against the oracle."""
    block = nn.TransformerBlock(48, 6, mlp_ratio=2, kv_heads=2, cap=5.0, rotary=True, distance=True)
    params = block.init(random.key(1))
    r = np.random.default_rng(6)
    x, t = (rg.tensor(r.standard_normal((3, 40, 48)).astype(F)) for _ in range(2))
    docs = np.sort(r.integers(0, 3, (3, 40)), axis=1).astype(np.int32)
    opt = optim.sgd(0.1)

    def step(s, data):
        x, t = data
        value, grads = rg.value_and_grad(lambda p: nn.mse_loss(block(p, x, documents=docs), t))(s["p"])
        grads, norm = optim.clip_gradients(grads, 0.2)
        p, o = opt.update(grads, s["o"], s["p"])
        return {"p": p, "o": o}, (value, norm)

    def token(s, data):
        y, cache = block.extend(data["p"], s["x"], s["cache"])
        return {"x": rg.tanh(y), "cache": cache}

    got = {}
    for device in ("hip", "cpu"):
        start = {"p": params, "o": opt.init(params)}
        run = rg.run(rg.compile(step, (start, (x, t)), validate="none", device=device), start, [(x, t)], steps=3)
        trained = run.state["p"]
        lengths = np.array([40, 17, 0], np.int32)
        read = rg.compile(lambda p, x: block.extend(p, x, block.state(3, 60, page=7), lengths), (trained, x), validate="none", device=device)
        _, cache = read(trained, x)
        s = {"x": x[:, :1], "cache": cache}
        served = rg.run(rg.compile(token, (s, {"p": trained}), validate="none", device=device), s, [{"p": trained}], steps=9).state
        got[device] = [np.array(run.history["aux.0"]), np.array(run.history["aux.1"]), served["x"].numpy(), served["cache"]["k"].numpy()]
        assert served["cache"]["pos"].numpy().tolist() == [49, 26, 9]
    # float32 through three updates and nine tokens of two norms and four products each.
    for a, b in zip(got["hip"], got["cpu"]):
        np.testing.assert_allclose(a, b, rtol=1e-4, atol=1e-5)


def test_a_decoder_of_several_layers_carries_its_caches():
    """Three blocks, each with pages of its own, token by token: one captured loop and single calls."""
    blocks = [nn.TransformerBlock(32, 4, kv_heads=2, cap=7.0, rotary=True) for _ in range(3)]
    params = [b.init(k) for b, k in zip(blocks, random.split(random.key(3), 3))]

    def step(s, data):
        x, caches = s["x"], []
        for block, p, cache in zip(blocks, data, s["caches"]):
            x, cache = block.extend(p, x, cache)
            caches.append(cache)
        return {"x": rg.tanh(x), "caches": caches}

    start = {"x": random.normal(random.key(4), (2, 1, 32)), "caches": [b.state(2, 40, page=6) for b in blocks]}
    run = rg.run(rg.compile(step, (start, params), validate="none"), start, [params], steps=21).state
    want = _one_by_one(step, start, params, 21)
    _same({"x": run["x"]}, {"x": want["x"]})
    for got, cache in zip(run["caches"], want["caches"]):
        _same(got, cache)
        assert cache["pos"].numpy().tolist() == [21, 21]


def test_standard_validation_on_the_device():
    block = nn.TransformerBlock(32, 4, cap=5.0, kv_heads=2)
    params = block.init(random.key(1))
    x = random.normal(random.key(2), (2, 20, 32))
    docs = np.array([[1] * 20, [2] * 15 + [-1] * 5], np.int32)
    program = rg.compile(lambda p: rg.value_and_grad(lambda p: (block(p, x, documents=docs) ** 2.0).mean())(p), (params,), validate="standard")
    assert program.report["status"] == "ok", program.report
