"""The sequence operators' kernels on the device: values and gradients against the formulas in 64
bits, captured and replayed step loops against the same steps one by one, bodies of control flow, and
the three operators run together as the layers call them."""

import numpy as np
import pytest

import rustautograd_amd as rg
from rustautograd_amd import nn, random
import sequence_reference as ref

pytestmark = pytest.mark.gpu
F = np.float32


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", ref.CONV_CASES, ids=str)
def test_conv(case, dtype):
    ref.check_conv(case, dtype, "hip")


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", ref.SCAN_CASES, ids=str)
def test_scan(case, dtype):
    ref.check_scan(case, dtype, "hip")


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("with_last", [True, False])
def test_scan_of_many_groups_over_long_sequences(dtype, with_last):
    """Enough channels and positions that a block of the gradient takes two chunks of the forward pass, and
    the last block one."""
    ref.check_scan((4, 523, 32, 3, 32, "dzslp"), dtype, "hip", with_last=with_last)


@pytest.mark.parametrize("case", [ref.SCAN_CASES[i] for i in (2, 7, 12, 16)], ids=str)
def test_scan_whose_last_state_nobody_reads(case):
    ref.check_scan(case, "float32", "hip", with_last=False)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", [ref.SCAN_CASES[i] for i in (1, 3, 7, 11, 12, 16)], ids=str)
def test_scan_of_maps_in_one_operand(case, dtype):
    ref.check_scan(case, dtype, "hip", joined=True)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", ref.SCAN_CASES, ids=str)
def test_scan_of_logarithms_with_a_bias(case, dtype):
    ref.check_scan_of_logs(case, dtype, "hip", joined=case[1] % 2 == 0)


def test_rates_of_logarithms_at_their_ends():
    """A logarithm of minus infinity keeps the state, one past the type's exponential forgets it at once."""
    a = np.array([[-np.inf], [200.0], [np.inf]], F)
    state = np.array([[[0.5], [0.5], [0.5]]], F)
    for length in (3, 40):  # a few positions, and tiles
        x, dt, b = np.zeros((1, length, 3), F), np.full((1, length, 3), 0.25, F), np.ones((1, length, 1, 1), F)
        y, last = rg.selective_scan(*(rg.tensor(v) for v in (x, dt, a, b, b)), state=rg.tensor(state), log_rates=True)
        assert np.array_equal(y.numpy()[0], np.tile(np.array([0.5, 0.0, 0.0], F), (length, 1)))
        assert last.numpy().ravel().tolist() == [0.5, 0.0, 0.0]


FEW = [(1, 1, 1, 1, 1, ""), (3, 1, 70, 16, 1, "dzsp"), (2, 3, 130, 16, 2, "dzsp"), (5, 4, 33, 13, 1, "zslp"), (2, 2, 20, 64, 4, "dslp"), (2, 1, 9, 32, 1, "s"),
       (5, 4, 40, 8, 2, "dzslp")]


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", FEW, ids=str)
def test_single_tokens_and_a_few(case, dtype):
    """Without a gradient, up to four positions run on a kernel of their own."""
    v, lengths, soft = ref.scan_inputs(case, dtype)
    args = (v["x"], v["dt"], v["a"], v["b"], v["c"], v["d"], v["z"], v["state"], lengths, soft, v["dy"], None)
    want, size, k = ref.scan(*args), ref.scan(*args, mag=True), ref.scan_roundings(v["x"], v["dt"], v["a"], soft)
    if lengths is not None:
        ref.fill_outside(v, lengths, ["x", "dt", "b", "c", "z"])
    given = {n: rg.tensor(v[n]) for n in ("x", "dt", "a", "b", "c", "d", "z", "state") if v[n] is not None}
    program = rg.compile(lambda g: rg.selective_scan(g["x"], g["dt"], g["a"], g["b"], g["c"], g.get("d"), g.get("z"), g.get("state"), lengths, soft), (given,),
                         validate="none")
    y, last = program(given)
    ref.agree(y.numpy(), want["y"], size["y"], k, dtype, "y")
    ref.agree(last.numpy(), want["last"], size["last"], k, dtype, "last")


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", FEW, ids=str)
def test_a_few_positions_of_logarithms_with_a_bias(case, dtype):
    v, lengths, soft, raw, rates, k = ref.log_inputs(case, dtype)
    args = (v["x"], raw, rates, v["b"], v["c"], v["d"], v["z"], v["state"], lengths, soft, v["dy"], None)
    want, size = ref.scan(*args), ref.scan(*args, mag=True)
    if lengths is not None:
        ref.fill_outside(v, lengths, ["x", "dt", "b", "c", "z"])
    given = {n: rg.tensor(v[n]) for n in ("x", "dt", "a", "b", "c", "d", "z", "state", "dt_bias") if v[n] is not None}
    program = rg.compile(lambda g: rg.selective_scan(g["x"], g["dt"], g["a"], g["b"], g["c"], g.get("d"), g.get("z"), g.get("state"), lengths, soft,
                                                     g["dt_bias"], True), (given,), validate="none")
    y, last = program(given)
    ref.agree(y.numpy(), want["y"], size["y"], k, dtype, "y")
    ref.agree(last.numpy(), want["last"], size["last"], k, dtype, "last")


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", ref.ROTARY_CASES, ids=str)
def test_rotary(case, dtype):
    ref.check_rotary(case, dtype, "hip")


def _inputs(case, names):
    v, lengths, soft = ref.scan_inputs(case, "float32")
    return {k: rg.tensor(v[k]) for k in names if v[k] is not None}, v, lengths, soft


def test_infinite_rates_and_values_stay_where_they_are():
    """A rate of minus infinity forgets the state at once; an infinite input reaches the positions after
    it in its own channel and sequence, and no other; padded NaN reaches none."""
    v, lengths, _ = ref.scan_inputs((2, 21, 6, 4, 1, "l"), "float32")
    v["a"][1] = -np.inf
    v["x"][0, 5, 3] = np.inf
    lengths = np.array([21, 9], np.int32)
    ref.fill_outside(v, lengths, ["x", "dt", "b", "c"])
    args = [rg.tensor(v[k]) for k in ("x", "dt", "a", "b", "c")]
    y, last = (o.numpy() for o in rg.compile(lambda *a: rg.selective_scan(*a, lengths=lengths), tuple(args), validate="none")(*args))
    clean = np.ones((2, 21, 6), bool)
    clean[0, 5:, 3] = False
    assert np.isfinite(y[clean]).all() and not np.isfinite(y[~clean]).any()
    assert (y[1, 9:] == 0).all()
    want = v["dt"][0, :, 1] * v["x"][0, :, 1] * (v["b"] * v["c"])[0, :, 0].sum(-1)
    # No state: four products and sums, of magnitudes that the same sum of absolute values bounds.
    size = np.abs(v["dt"][0, :, 1] * v["x"][0, :, 1]) * np.abs(v["b"] * v["c"])[0, :, 0].sum(-1)
    ref.agree(y[0, :, 1], want.astype(np.float64), size.astype(np.float64), 24, "float32", "forgetting channel")


def test_a_rate_that_is_nan_stays_in_its_channel_and_group():
    """Channel 0's rate reaches its own results and the gradients of its group's maps, no others, also
    where the last tile of channels is not full."""
    v, _, _ = ref.scan_inputs((1, 40, 6, 4, 2, ""), "float32")
    v["a"][0, 0] = np.nan
    dy = rg.tensor(v["dy"])

    def program(g):
        return rg.grad(lambda g: (rg.selective_scan(g["x"], g["dt"], g["a"], g["b"], g["c"])[0] * dy).sum())(g)

    given = {k: rg.tensor(v[k]) for k in ("x", "dt", "a", "b", "c")}
    grads = {k: g.numpy() for k, g in rg.compile(program, (given,), validate="none")(given).items()}
    assert np.isfinite(grads["b"][:, :, 1]).all() and np.isfinite(grads["c"][:, :, 1]).all()
    for k in ("x", "dt"):
        assert np.isfinite(grads[k][..., 1:]).all() and not np.isfinite(grads[k][..., 0]).any()
    assert np.isfinite(grads["a"][1:]).all()


@pytest.mark.parametrize("dtype", ["float32", "float64"])
def test_states_that_grow_past_what_one_factor_holds(dtype):
    """Growing states over many chunks. Channel 0 starts empty and its inputs begin late: it is 0 until
    then. Channel 1 holds 1e-30 and grows by e^96 within a stretch of 32 positions (e^1200 from
    1e-300 in 64 bits): more than one factor of its type holds, the state itself does not overflow."""
    v, _, _ = ref.scan_inputs((1, 523, 2, 4, 1, "s"), dtype)
    grow = 3.0 if dtype == "float32" else 37.5
    v["a"][:] = 1.0
    v["dt"][0, :, 0], v["x"][0, :, 0] = 1.0, 0.0
    v["x"][0, 510:, 0] = 1.0
    v["dt"][0, :, 1], v["dt"][0, 32:64, 1], v["x"][0, :, 1] = 0.0, grow, 0.0
    v["state"][0, 0], v["state"][0, 1] = 0.0, 1e-30 if dtype == "float32" else 1e-300
    v["dy"][:], v["dlast"][:] = 0.0, 0.0
    v["dy"][0, 505:, 1] = 1e-30 if dtype == "float32" else 1e-300
    args = (v["x"], v["dt"], v["a"], v["b"], v["c"], None, None, v["state"], None, False, v["dy"], None)
    want, size = ref.scan(*args), ref.scan(*args, mag=True)
    k = ref.scan_roundings(v["x"], v["dt"], v["a"], False)
    dy = rg.tensor(v["dy"])

    def program(g):
        def loss(g):
            y, last = rg.selective_scan(g["x"], g["dt"], g["a"], g["b"], g["c"], state=g["state"])
            return (y * dy).sum(), (y, last)
        (_, results), grads = rg.value_and_grad(loss, has_aux=True)(g)
        return results, grads["state"]

    given = {n: rg.tensor(v[n]) for n in ("x", "dt", "a", "b", "c", "state")}
    (y, last), dstate = rg.compile(program, (given,), validate="none")(given)
    assert (y.numpy()[0, :510, 0] == 0.0).all() and (dstate.numpy()[0, 0] == 0.0).all()
    ref.agree(y.numpy(), want["y"], size["y"], k, dtype, "y")
    ref.agree(last.numpy(), want["last"], size["last"], k, dtype, "last")
    ref.agree(dstate.numpy(), want["dstate"], size["dstate"], k, dtype, "dstate")


@pytest.mark.parametrize("optimize", ["none", "standard"])
def test_gradients_asked_for_one_by_one(optimize):
    """A scan differentiated once for each argument: as differentiated for both at once."""
    v, _, _ = ref.scan_inputs((2, 40, 4, 3, 1, ""), "float32")
    x, dt, a, b, c, dy = (rg.tensor(v[k]) for k in ("x", "dt", "a", "b", "c", "dy"))

    def loss(x, dt):
        return (rg.selective_scan(x, dt, a, b, c)[0] * dy).sum()

    apart = rg.compile(lambda x, dt: rg.value_and_grad(loss, argnums=(0, 1))(x, dt)[1], (x, dt), validate="none", optimize=optimize)(x, dt)
    both = rg.compile(lambda t: rg.grad(lambda t: loss(*t))(t), ((x, dt),), validate="none", optimize=optimize)((x, dt))
    for one, other in zip(apart, both):
        assert np.array_equal(one.numpy(), other.numpy())


def test_activations_at_their_ends():
    """SiLU and softplus far out: 0 and the value itself, infinities as the limits have them, NaN as NaN."""
    far = np.array([-np.inf, -1e30, -200.0, -90.0, 0.0, 90.0, 1e30, np.inf, np.nan], F)
    x = rg.tensor(far.reshape(1, 9, 1))
    unit = rg.tensor(np.array([[0.0], [1.0]], F))
    y = rg.compile(lambda v: rg.causal_conv(v, unit, activation="silu")[0], (x,), validate="none")(x).numpy().ravel()
    # A product with the tap of 0 makes the infinite neighbours NaN; the finite positions stay.
    assert np.abs(y[2:4]).max() <= 200.0 * 1e-37 and y[4] == 0.0 and y[5] == 90.0 and y[6] == F(1e30) and np.isnan(y[8])
    one = rg.tensor(np.ones((1, 9, 1), F))
    dt = rg.tensor(np.array([-np.inf, -1e30, -200.0, -30.0, 0.0, 30.0, 1e30, 3.0, -5.0], F).reshape(1, 9, 1))
    run = rg.compile(lambda d: rg.selective_scan(one, d, rg.tensor(np.full((1, 1), -np.inf, F)), rg.ones((1, 9, 1)), rg.ones((1, 9, 1)), softplus=True)[0], (dt,),
                     validate="none")
    # With nothing kept, y is the step itself: log(1 + e^v), four roundings.
    want = np.logaddexp(0.0, dt.numpy().ravel().astype(np.float64))
    got = run(dt).numpy().ravel()
    assert np.abs(got[:3]).max() <= 1e-40
    ref.agree(got[3:], want[3:], want[3:], 8, "float32", "softplus")


def _steps(program, state, data, n):
    """The state after n calls of `program`, one by one, and their scalars."""
    seen = []
    for _ in range(n):
        state, aux = program(state, data)
        seen.append([float(a) for a in (aux if isinstance(aux, tuple) else (aux,))])
    return state, np.array(seen)


def _same(a, b):
    if isinstance(a, dict):
        return a.keys() == b.keys() and all(_same(a[k], b[k]) for k in a)
    return np.array_equal(a.numpy(), b.numpy(), equal_nan=True)


def test_a_replayed_training_loop_is_its_steps_one_by_one():
    """Every operator's gradient in one step, run as captured graphs and call by call: the same bits, also
    on a second run of the same program after other work."""
    layer = nn.SelectiveSSM(24, states=8, dt_rank=3, groups=2, rotary=True)
    attn = nn.MultiHeadAttention(24, 2, qk_norm=True, rotary=10000.0)
    params = {"ssm": layer.init(random.key(0)), "attn": attn.init(random.key(1))}
    r = np.random.default_rng(0)
    data = (rg.tensor(r.standard_normal((2, 37, 24)).astype(F)), rg.tensor(r.standard_normal((2, 37, 24)).astype(F)))
    mask = rg.tril(37)

    def loss(p, x, t):
        h = x + attn(p["attn"], x, mask)
        return nn.mse_loss(h + layer(p["ssm"], h), t)

    def step(p, batch):
        value, grads = rg.value_and_grad(loss)(p, *batch)
        return rg.tree.map(lambda a, g: a - 0.1 * g, p, grads), value

    program = rg.compile(step, (params, data), validate="none")
    want, seen = _steps(program, params, data, 7)
    for _ in range(2):
        got = rg.run(program, params, [data], steps=7)
        assert _same(got.state, want)
        assert np.array_equal(np.array(got.history["aux"], F), seen[:, 0].astype(F))
    assert seen[-1, 0] < seen[0, 0]


def test_a_replayed_token_loop_is_its_tokens_one_by_one():
    layer = nn.SelectiveSSM(16, states=16, rotary=True)
    params = layer.init(random.key(2))
    state = {"x": rg.tensor(np.random.default_rng(1).standard_normal((3, 1, 16)).astype(F)), **layer.state(3)}

    def step(s, p):
        y, carried = layer.extend(p, s["x"], {k: s[k] for k in ("conv", "scan", "pos")})
        return {"x": rg.tanh(y + s["x"]), **carried}, (y.sum(),)

    program = rg.compile(step, (state, params), validate="none")
    want, _ = _steps(program, state, params, 70)
    for _ in range(2):
        got = rg.run(program, state, [params], steps=70)
        assert _same(got.state, want)
        assert got.state["pos"].tolist() == [70, 70, 70]


def test_prompts_and_tokens_agree():
    """A prompt read at once, and the same positions in parts down to single tokens: the same sums in the
    same order, but for parts' own tiles; bound as the scan's, twice over."""
    case = (2, 50, 70, 16, 1, "dzp")
    given, v, _, _ = _inputs(case, ("x", "dt", "a", "b", "c", "d", "z"))
    whole = rg.compile(lambda g: rg.selective_scan(g["x"], g["dt"], g["a"], g["b"], g["c"], g["d"], g["z"], softplus=True), (given,), validate="none")
    y, last = whole(given)
    args = (v["x"], v["dt"], v["a"], v["b"], v["c"], v["d"], v["z"], None, None, True, v["dy"], None)
    size = ref.scan(*args, mag=True)
    k = 2 * ref.scan_roundings(v["x"], v["dt"], v["a"], True)
    state, parts, lo = rg.zeros((2, 70, 16)), [], 0
    for n in (17, 1, 1, 2, 3, 5, 21):
        part = {q: rg.tensor(t.numpy()[:, lo:lo + n]) if q in ("x", "dt", "b", "c", "z") else t for q, t in given.items()}
        out, state = rg.compile(lambda g, s: rg.selective_scan(g["x"], g["dt"], g["a"], g["b"], g["c"], g["d"], g["z"], s, softplus=True), (part, state),
                                validate="none")(part, state)
        parts.append(out.numpy())
        lo += n
    ref.agree(np.concatenate(parts, 1), y.numpy().astype(np.float64), size["y"], k, "float32", "y")
    ref.agree(state.numpy(), last.numpy().astype(np.float64), size["last"], k, "float32", "state")


def test_inside_control_flow():
    """Tokens through a `scan` body, whose slots and workspace are the enclosing program's, with gradients."""
    r = np.random.default_rng(4)
    x = rg.tensor(r.standard_normal((6, 2, 3, 8)).astype(F))
    w = rg.tensor((0.5 * r.standard_normal((3, 8))).astype(F))

    def looped(w, x):
        def body(s, v):
            y, s = rg.causal_conv(v, w, state=s, activation="silu")
            return s, y
        _, ys = rg.scan(body, rg.zeros((2, 2, 8)), x)
        return (ys * ys).sum()

    def at_once(w, x):
        rows = x.transpose(1, 0, 2, 3).reshape(2, 18, 8)
        y, _ = rg.causal_conv(rows, w, activation="silu")
        return (y * y).sum()

    a, b = (rg.compile(lambda *v: rg.value_and_grad(f)(*v), (w, x), validate="none")(w, x) for f in (looped, at_once))
    # One sum of 288 squares and of their slopes, in another order: 288 u of the sum of magnitudes.
    assert abs(float(a[0]) - float(b[0])) <= 288 * 2.0 ** -24 * float(b[0])
    assert np.allclose(a[1].numpy(), b[1].numpy(), rtol=0, atol=400 * 2.0 ** -24 * 36 * np.abs(x.numpy()).max() ** 2)


def test_two_programs_at_once_keep_to_their_own_buffers():
    """Programs of the same operators with other sizes and data, called in turn."""
    programs = []
    for k, case in enumerate([(2, 130, 70, 16, 1, "dz"), (1, 40, 200, 16, 1, "dz")]):
        given, v, _, _ = _inputs(case, ("x", "dt", "a", "b", "c", "d", "z"))

        def fn(g):
            return rg.grad(lambda q: (rg.selective_scan(q["x"], q["dt"], q["a"], q["b"], q["c"], q["d"], q["z"])[0] ** 2.0).sum())(g)
        programs.append((rg.compile(fn, (given,), validate="none"), given))
    first = [p(g) for p, g in programs]
    for _ in range(3):
        assert all(_same(p(g), want) for (p, g), want in zip(programs, first))


def test_the_oracle_agrees_at_standard_validation():
    """compile(validate="standard") holds the device against the CPU oracle."""
    layer = nn.SelectiveSSM(16, states=8, rotary=True)
    params = layer.init(random.key(5))
    x = rg.tensor(np.random.default_rng(7).standard_normal((2, 19, 16)).astype(F))
    c = rg.compile(lambda p, v: rg.value_and_grad(lambda q: (layer(q, v) ** 2.0).sum())(p), (params, x))
    assert c.report.ok, c.report


# Batch, length, sections, passing heads, head, rotary dims. The walkers do not divide the tokens: some
# have none in the last round, in the second of three or more walks or in the only one.
WALKS = [(1, 5, (2, 1), 0, 8, 8), (2, 9, (3,), 2, 4, 2), (3, 701, (3,), 2, 256, 2), (3, 5001, (4, 3), 3, 8, 8), (3, 5001, (4, 3), 3, 8, 2)]


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", WALKS, ids=str)
def test_rotary_without_eps_over_many_tokens(case, dtype):
    """Heads of +1 and -1 have a root mean square of 1, without `eps` exactly; whole numbers for the rest,
    and a position of 0, keep every sum exact (below 2^24): results and gradients are equal, not near."""
    b, t, sections, passing, hd, turn = case
    r = np.random.default_rng(11)
    used = sum(sections)
    x = (2 * r.integers(0, 2, (b, t, used + passing, hd)) - 1).astype(dtype)
    dy, gain = (r.integers(-2, 3, s).astype(dtype) for s in (x.shape, (len(sections), hd)))
    start, weight = rg.tensor(np.zeros(t, np.int32)), rg.tensor(dy)

    def program(given):
        def loss(g):
            y = rg.rotary_norm(g["x"], g["gain"], start, sections, turn, eps=0.0)
            return (y * weight).sum(), y
        (_, y), grads = rg.value_and_grad(loss, has_aux=True)(given)
        return y, grads

    given = {"x": rg.tensor(x), "gain": rg.tensor(gain)}
    y, grads = rg.compile(program, (given,), validate="none")(given)
    rows = np.concatenate([np.repeat(gain, sections, 0), np.ones((passing, hd), dtype)])
    assert np.array_equal(y.numpy(), x * rows)
    u = dy * rows
    mean = (u * x).sum(-1, keepdims=True) / hd
    mean[:, :, used:] = 0.0
    assert np.array_equal(grads["x"].numpy(), u - x * mean)
    ends = np.cumsum(sections)
    want = np.stack([(dy * x)[:, :, e - n:e].sum((0, 1, 2), dtype=np.float64) for n, e in zip(sections, ends)])
    assert np.array_equal(grads["gain"].numpy(), want.astype(dtype))


def _far_below(dtype):
    """Values whose exponential is 0 in the type: SiLU and its slope are 0 there."""
    return np.array([-110.0 if dtype == "float32" else -750.0, -1e4, -1e30, -1e37, np.finfo(dtype).min], dtype)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
def test_silu_of_a_convolution_far_below_zero(dtype):
    far = _far_below(dtype)
    x = np.ones((1, 12, 3), dtype)
    x[0, 2:7, 1] = far[::-1]  # the one before the next ordinary position, which its product with a slope keeps finite, last
    weight = rg.tensor(np.full(x.shape, 2.0, dtype))
    w = np.concatenate([np.zeros((1, 3)), np.ones((1, 3))]).astype(dtype)

    def program(given):
        def loss(g):
            y = rg.causal_conv(g["x"], g["w"], g["b"], activation="silu")[0]
            return (y * weight).sum(), y
        (_, y), grads = rg.value_and_grad(loss, has_aux=True)(given)
        return y, grads

    given = {"x": rg.tensor(x), "w": rg.tensor(w), "b": rg.zeros(3, dtype)}
    y, grads = rg.compile(program, (given,), validate="none")(given)
    s = ref.sigmoid(1.0)
    want, slope = np.full(x.shape, s), np.full(x.shape, 2.0 * s * (2.0 - s))
    want[0, 2:7, 1] = slope[0, 2:7, 1] = 0.0
    ref.agree(y.numpy(), want, np.abs(want), 24, dtype, "y")
    ref.agree(grads["x"].numpy(), slope, np.abs(slope), 40, dtype, "dx")
    # Sums of twelve terms of up to 40 roundings.
    ref.agree(grads["b"].numpy(), slope.sum((0, 1)), slope.sum((0, 1)), 60, dtype, "db")
    assert (y.numpy()[0, 2:7, 1] == 0.0).all() and (grads["x"].numpy()[0, 2:7, 1] == 0.0).all()
    want_w = np.stack([(slope[0, 1:] * x[0, :-1]).sum(0), (slope[0] * x[0]).sum(0)])
    assert np.isfinite(grads["w"].numpy()).all()
    keep = np.array([True, False, True])
    ref.agree(grads["w"].numpy()[:, keep], want_w[:, keep], want_w[:, keep], 60, dtype, "dw")
    ref.agree(grads["w"].numpy()[1, 1], want_w[1, 1], want_w[1, 1], 60, dtype, "dw of the far channel")


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("length", [8, 40])
def test_a_gate_closed_with_the_lowest_values(length, dtype):
    """A gate far below zero closes: its positions give 0 and pass no gradient, others are as ever."""
    far = _far_below(dtype)
    v, _, _ = ref.scan_inputs((2, length, 6, 4, 1, "dzp"), dtype)
    v["z"][1, 2:7, 3] = far
    v["z"][0, 1:6, 0] = far
    shut = v["z"] <= far.max()
    args = (v["x"], v["dt"], v["a"], v["b"], v["c"], v["d"], v["z"], None, None, True, v["dy"], None)
    with np.errstate(over="ignore"):
        want, size, k = ref.scan(*args), ref.scan(*args, mag=True), ref.scan_roundings(v["x"], v["dt"], v["a"], True)
    weight = rg.tensor(v["dy"])

    def fn(g):
        y = rg.selective_scan(g["x"], g["dt"], g["a"], g["b"], g["c"], g["d"], g["z"], softplus=True)[0]
        return (y * weight).sum(), (y,)

    (y,), grads = ref._differentiated(fn, {n: v[n] for n in ("x", "dt", "a", "b", "c", "d", "z")}, "hip")
    ref.agree(y, want["y"], size["y"], k, dtype, "y")
    assert (y[shut] == 0.0).all() and (grads["z"][shut] == 0.0).all()
    for n, g in grads.items():
        ref.agree(g, want["d" + n], size["d" + n], k, dtype, "d" + n)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
def test_a_token_s_gate_closed_with_the_lowest_values(dtype):
    far = _far_below(dtype)
    v, _, _ = ref.scan_inputs((1, 1, 7, 4, 1, "dz"), dtype)
    v["z"][0, 0, 1:6] = far
    given = {n: rg.tensor(v[n]) for n in ("x", "dt", "a", "b", "c", "d", "z")}
    y = rg.compile(lambda g: rg.selective_scan(g["x"], g["dt"], g["a"], g["b"], g["c"], g["d"], g["z"])[0], (given,), validate="none")(given).numpy()
    assert (y[0, 0, 1:6] == 0.0).all() and np.isfinite(y).all() and (y[0, 0, [0, 6]] != 0.0).all()


@pytest.mark.parametrize("dtype, width, rate, step", [("float32", 66, 200.0, 1e-3), ("float32", 65, 150.0, 1e-3), ("float64", 33, 1200.0, 1e-4)])
def test_channels_that_do_not_fill_a_vector_beside_a_growing_one(dtype, width, rate, step):
    """The last tile's first channel grows, by little in each of its small steps; the lanes past the last
    channel, which have no step, leave the gradients of the maps alone."""
    case = (2, 40, width, 4, 1, "zp")
    v, _, _ = ref.scan_inputs(case, dtype)
    last = 64 if dtype == "float32" else 32
    v["a"][last] = rate
    v["dt"][:, :, last] = np.log(np.expm1(step))
    args = (v["x"], v["dt"], v["a"], v["b"], v["c"], None, v["z"], None, None, True, v["dy"], None)
    want, size = ref.scan(*args), ref.scan(*args, mag=True)
    k = ref.scan_roundings(v["x"], v["dt"], v["a"], True)
    weight = rg.tensor(v["dy"])

    def fn(g):
        y = rg.selective_scan(g["x"], g["dt"], g["a"], g["b"], g["c"], z=g["z"], softplus=True)[0]
        return (y * weight).sum(), (y,)

    (y,), grads = ref._differentiated(fn, {n: v[n] for n in ("x", "dt", "a", "b", "c", "z")}, "hip")
    ref.agree(y, want["y"], size["y"], k, dtype, "y")
    for n, g in grads.items():
        ref.agree(g, want["d" + n], size["d" + n], k, dtype, "d" + n)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("length, width, padded", [(5, 6, False), (37, 8, False), (37, 5, True)])
def test_infinities_at_the_end_of_a_convolution(dtype, length, width, padded):
    """The last input meets the last tap alone and the first tap the positions up to the last: gradients that
    no formula multiplies with an infinite value are finite, and exact for whole numbers."""
    r = np.random.default_rng(3)
    x, w, dy = (r.integers(-3, 4, s).astype(dtype) for s in ((2, length, width), (3, width), (2, length, width)))
    lengths = np.array([length, length - 2], np.int32) if padded else None
    weight = rg.tensor(dy)
    ends = [length, length - 2] if padded else [length, length]

    def grads(x, w):
        given = {"x": rg.tensor(x), "w": rg.tensor(w)}
        program = rg.compile(lambda g: rg.grad(lambda g: (rg.causal_conv(g["x"], g["w"], lengths=lengths)[0] * weight).sum())(g), (given,), validate="none")
        return {n: g.numpy() for n, g in program(given).items()}

    clean = grads(x, w)
    for i, n in enumerate(ends):
        far = x.copy()
        far[i, n - 1, 0] = np.inf
        got = grads(far, w)
        assert np.array_equal(got["w"][:2], clean["w"][:2]) and np.array_equal(got["w"][:, 1:], clean["w"][:, 1:])
        assert np.array_equal(got["x"], clean["x"])
    wide = w.copy()
    wide[0, 1] = np.inf
    got = grads(x, wide)
    for i, n in enumerate(ends):
        # The last two inputs before a sequence's end meet the first tap at no position; padded ones none.
        assert np.array_equal(got["x"][i, n - 2:], clean["x"][i, n - 2:])
        assert np.array_equal(got["x"][i, :, [0, *range(2, width)]], clean["x"][i, :, [0, *range(2, width)]])


@pytest.mark.parametrize("dtype, eps", [("float32", 1e-40), ("float32", 2e-38), ("float64", 1e-300)])
def test_heads_of_zeros_under_the_smallest_eps(dtype, eps):
    """They stay zeros, and their gradient is the cotangent over the root of `eps`."""
    dy = np.random.default_rng(0).integers(-3, 4, (2, 3, 2, 4)).astype(dtype)
    x, gain, weight = rg.zeros((2, 3, 2, 4), dtype), rg.ones((1, 4), dtype), rg.tensor(dy)

    def program(given):
        def loss(g):
            y = rg.rotary_norm(g["x"], g["gain"], rotary_dims=0, eps=eps)
            return (y * weight).sum(), y
        (_, y), grads = rg.value_and_grad(loss, has_aux=True)(given)
        return y, grads

    y, grads = rg.compile(program, ({"x": x, "gain": gain},), validate="none")({"x": x, "gain": gain})
    assert (y.numpy() == 0.0).all() and (grads["gain"].numpy() == 0.0).all()
    want = dy.astype(np.float64) / np.sqrt(np.float64(np.dtype(dtype).type(eps)))
    ref.agree(grads["x"].numpy(), want, np.abs(want), 8, dtype, "dx")
