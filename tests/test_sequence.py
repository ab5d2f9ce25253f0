"""The sequence operators through the engine on the CPU oracle: values and gradients against the
formulas in 64 bits, gradients against differences, refusals, and the layers that call them."""

import os
import re

import numpy as np
import pytest

import rustautograd_amd as rg
from rustautograd_amd import nn, random
import sequence_reference as ref

F = np.float32


def _t(*shape, dtype=F):
    return rg.tensor(np.ones(shape, dtype))


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", ref.CONV_CASES, ids=str)
def test_conv(case, dtype):
    ref.check_conv(case, dtype, "cpu")


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", ref.SCAN_CASES[:-2], ids=str)
def test_scan(case, dtype):
    ref.check_scan(case, dtype, "cpu")


@pytest.mark.parametrize("case", [ref.SCAN_CASES[i] for i in (1, 3, 7, 11)], ids=str)
def test_scan_of_maps_in_one_operand(case):
    ref.check_scan(case, "float32", "cpu", joined=True)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", [ref.SCAN_CASES[i] for i in (0, 1, 3, 7, 9, 12)], ids=str)
def test_scan_of_logarithms_with_a_bias(case, dtype):
    ref.check_scan_of_logs(case, dtype, "cpu")


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", ref.ROTARY_CASES, ids=str)
def test_rotary(case, dtype):
    ref.check_rotary(case, dtype, "cpu")


def test_device_plans_run_the_same_operators():
    ref.check_conv(ref.CONV_CASES[4], "float32", "cpu_devplan")
    ref.check_scan(ref.SCAN_CASES[3], "float32", "cpu_devplan")
    ref.check_scan(ref.SCAN_CASES[7], "float32", "cpu_devplan", with_last=False)
    ref.check_scan_of_logs(ref.SCAN_CASES[3], "float32", "cpu_devplan", joined=True)
    ref.check_rotary(ref.ROTARY_CASES[3], "float32", "cpu_devplan")


# ---- gradients against differences -------------------------------------------------------------------

def _by_differences(fn, inputs, step=1e-6):
    """Central differences of fn's scalar along one direction an input, against its gradients; both
    in float64, whose truncation (step^2) and rounding (1e-16 / step) leave about 1e-9 of the size."""
    value = rg.compile(fn, tuple(rg.tensor(v) for v in inputs), validate="none")
    slopes = rg.compile(lambda *v: rg.value_and_grad(fn, argnums=tuple(range(len(v))))(*v)[1], tuple(rg.tensor(v) for v in inputs), validate="none")
    grads = slopes(*[rg.tensor(v) for v in inputs])
    r = np.random.default_rng(5)
    for k, v in enumerate(inputs):
        way = r.standard_normal(v.shape)
        ends = []
        for s in (step, -step):
            moved = list(inputs)
            moved[k] = v + s * way
            ends.append(float(value(*[rg.tensor(m) for m in moved])))
        want = (ends[0] - ends[1]) / (2 * step)
        got = float((grads[k].numpy() * way).sum())
        assert abs(got - want) <= 1e-7 * max(1.0, abs(want)), (k, got, want)


def test_conv_gradients_are_the_differences():
    v, n, _ = ref.conv_inputs((3, 6, 4, 4, "bsla"), "float64")
    _by_differences(lambda x, w, b, s: sum((o * o).sum() for o in rg.causal_conv(x, w, b, s, n, "silu")), [v[k] for k in ("x", "w", "bias", "state")])


def test_scan_gradients_are_the_differences():
    v, n, _ = ref.scan_inputs((3, 9, 4, 3, 2, "dzslp"), "float64")
    _by_differences(lambda x, dt, a, b, c, d, z, s: sum((o * o).sum() for o in rg.selective_scan(x, dt, a, b, c, d, z, s, n, softplus=True)),
                    [v[k] for k in ("x", "dt", "a", "b", "c", "d", "z", "state")])


def test_scan_of_logarithms_gradients_are_the_differences():
    v, n, _, _, _, _ = ref.log_inputs((3, 9, 4, 3, 2, "dzslp"), "float64")
    _by_differences(lambda x, dt, a, b, c, e: sum((o * o).sum() for o in rg.selective_scan(x, dt, a, b, c, lengths=n, softplus=True, dt_bias=e, log_rates=True)),
                    [v[k] for k in ("x", "dt", "a", "b", "c", "dt_bias")])


def test_rotary_gradients_are_the_differences():
    v, pos = ref.rotary_inputs((2, 3, (2, 1), 1, 6, 4, "gp"), "float64")
    weight = rg.tensor(v["dy"])
    _by_differences(lambda x, g: (rg.rotary_norm(x, g, pos, (2, 1), 4) ** 2.0 * weight).sum(), [v["x"], v["gain"]])


def test_a_shared_input_gets_both_gradients():
    """The same value as two operands: its gradient is the sum of theirs."""
    v, _, _ = ref.scan_inputs((1, 5, 4, 4, 1, ""), "float64")
    x, dt, a, b = (rg.tensor(v[k]) for k in ("x", "dt", "a", "b"))
    one = rg.grad(lambda m: rg.selective_scan(x, dt, a, m, m)[0].sum())(b).numpy()
    two = rg.grad(lambda p: rg.selective_scan(x, dt, a, p["b"], p["c"])[0].sum())({"b": b, "c": b})
    assert np.allclose(one, two["b"].numpy() + two["c"].numpy(), rtol=1e-14)


def test_a_gradient_of_a_gradient_is_refused():
    x, w = _t(1, 4, 2), _t(2, 2)
    with pytest.raises(rg.DiagnosticError, match="GRAD_UNSUPPORTED"):
        rg.grad(lambda v: rg.grad(lambda u: (rg.causal_conv(u, w, activation="silu")[0] ** 2.0).sum())(v).sum())(x)
    with pytest.raises(rg.DiagnosticError, match="GRAD_UNSUPPORTED"):
        rg.grad(lambda v: (rg.grad(lambda u: (rg.rotary_norm(u) ** 2.0).sum())(v) ** 2.0).sum())(_t(1, 4, 1, 2))


# ---- refusals ------------------------------------------------------------------------------------------

def _scan(x=(2, 3, 4), dt=(2, 3, 4), a=(4, 5), b=(2, 3, 1, 5), c=(2, 3, 1, 5), **more):
    return rg.selective_scan(_t(*x), _t(*dt), _t(*a), _t(*b), _t(*c), **more)


@pytest.mark.parametrize("call, code, cause", [
    (lambda: rg.causal_conv(_t(2, 3), _t(2, 3)), "SHAPE_MISMATCH", "x_must_be_batch_length_width"),
    (lambda: rg.causal_conv(_t(2, 3, 4), _t(1, 4)), "SHAPE_MISMATCH", "taps_must_be_two_to_eight"),
    (lambda: rg.causal_conv(_t(2, 3, 4), _t(9, 4)), "SHAPE_MISMATCH", "taps_must_be_two_to_eight"),
    (lambda: rg.causal_conv(_t(2, 3, 4), _t(4, 3)), "SHAPE_MISMATCH", "weights_must_be_taps_width"),
    (lambda: rg.causal_conv(_t(2, 0, 4), _t(2, 4)), "SHAPE_MISMATCH", "empty_operand"),
    (lambda: rg.causal_conv(_t(2, 3, 4), _t(2, 4), _t(3)), "SHAPE_MISMATCH", "bias_must_be_width"),
    (lambda: rg.causal_conv(_t(2, 3, 4), _t(4, 4), state=_t(2, 2, 4)), "SHAPE_MISMATCH", "state_must_be_batch_taps_less_one_width"),
    (lambda: rg.causal_conv(_t(2, 3, 4), _t(2, 4), lengths=[1, 2, 3]), "SHAPE_MISMATCH", "lengths_must_be_one_per_sequence"),
    (lambda: rg.causal_conv(_t(2, 3, 4), _t(2, 4), lengths=rg.tensor(np.ones(2, F))), "DTYPE_MISMATCH", "lengths_and_positions_must_be_int32"),
    (lambda: rg.causal_conv(_t(2, 3, 4), _t(2, 4, dtype=np.float64)), "DTYPE_MISMATCH", "implicit_promotion_not_allowed"),
    (lambda: rg.causal_conv(_t(2, 3, 4, dtype=np.int32), _t(2, 4, dtype=np.int32)), "UNSUPPORTED_DTYPE", "operation_is_float_only_cast_first"),
    (lambda: rg.causal_conv(_t(2, 3, 4), _t(2, 4), activation="relu"), "INVALID_ARGUMENT", "activation_must_be_none_or_silu"),
    (lambda: _scan(dt=(2, 3, 1)), "SHAPE_MISMATCH", "dt_shape_differs_from_x"),
    (lambda: _scan(a=(3, 5)), "SHAPE_MISMATCH", "a_must_be_width_by_at_most_64_states"),
    (lambda: _scan(a=(4, 65), b=(2, 3, 1, 65), c=(2, 3, 1, 65)), "SHAPE_MISMATCH", "a_must_be_width_by_at_most_64_states"),
    (lambda: _scan(b=(2, 3, 3, 5), c=(2, 3, 3, 5)), "SHAPE_MISMATCH", "b_must_be_batch_length_groups_states_with_groups_dividing_the_width"),
    (lambda: _scan(c=(2, 3, 2, 5)), "SHAPE_MISMATCH", "c_shape_differs_from_b"),
    (lambda: rg.selective_scan(_t(2, 3, 4), _t(2, 3, 4), _t(4, 5), _t(2, 3, 3, 5)), "SHAPE_MISMATCH",
     "b_must_be_batch_length_groups_states_with_groups_dividing_the_width"),
    (lambda: rg.rotary_norm(_t(2, 3, 4, 6), positions=[[0], [1], [2]]), "SHAPE_MISMATCH", "positions_must_be_length_or_batch_length"),
    (lambda: _scan(d=_t(5)), "SHAPE_MISMATCH", "d_must_be_width"),
    (lambda: _scan(z=_t(2, 3, 5)), "SHAPE_MISMATCH", "z_shape_differs_from_x"),
    (lambda: _scan(dt_bias=_t(5)), "SHAPE_MISMATCH", "dt_bias_must_be_width"),
    (lambda: _scan(state=_t(2, 5, 4)), "SHAPE_MISMATCH", "state_must_be_batch_width_states"),
    (lambda: rg.rotary_norm(_t(2, 3, 4)), "SHAPE_MISMATCH", "x_must_be_batch_length_heads_head"),
    (lambda: rg.rotary_norm(_t(2, 3, 4, 5), rotary_dims=4), "SHAPE_MISMATCH", "head_must_be_even_and_at_most_256"),
    (lambda: rg.rotary_norm(_t(2, 3, 4, 258)), "SHAPE_MISMATCH", "head_must_be_even_and_at_most_256"),
    (lambda: rg.rotary_norm(_t(2, 3, 4, 6), rotary_dims=3), "SHAPE_MISMATCH", "rotary_dims_must_be_even_and_within_the_head"),
    (lambda: rg.rotary_norm(_t(2, 3, 4, 6), rotary_dims=8), "SHAPE_MISMATCH", "rotary_dims_must_be_even_and_within_the_head"),
    (lambda: rg.rotary_norm(_t(2, 3, 4, 6), rotary_dims=-2), "INVALID_ARGUMENT", "sections_and_rotary_dims_must_not_be_negative"),
    (lambda: rg.rotary_norm(_t(2, 3, 4, 6), sections=(3, 2)), "SHAPE_MISMATCH", "sections_must_be_one_to_four_within_the_heads"),
    (lambda: rg.rotary_norm(_t(2, 3, 4, 6), sections=(1, 0)), "INVALID_ARGUMENT", "sections_and_rotary_dims_must_not_be_negative"),
    (lambda: rg.rotary_norm(_t(2, 3, 4, 6), gain=_t(2, 6)), "SHAPE_MISMATCH", "gain_must_be_sections_head"),
    (lambda: rg.rotary_norm(_t(2, 3, 4, 6), positions=[0, 1]), "SHAPE_MISMATCH", "positions_must_be_length_or_batch_length"),
    (lambda: rg.rotary_norm(_t(2, 3, 4, 6), base=0.0), "INVALID_ARGUMENT", "base_must_be_positive_and_eps_not_negative"),
    (lambda: rg.rotary_norm(_t(2, 3, 4, 6), eps=-1.0), "INVALID_ARGUMENT", "base_must_be_positive_and_eps_not_negative"),
])
def test_refusals(call, code, cause):
    with pytest.raises(rg.DiagnosticError) as e:
        call()
    assert e.value.diagnostic["code"] == code, e.value.diagnostic
    assert cause in str(e.value.diagnostic), e.value.diagnostic


@pytest.mark.parametrize("optimize", ["none", "standard"])
def test_gradients_asked_for_one_by_one_share_the_kept_states(optimize):
    """One scan differentiated once for each argument: each of its results is in the plan once."""
    v, _, _ = ref.scan_inputs((2, 40, 4, 3, 1, ""), "float32")
    x, dt, a, b, c = (rg.tensor(v[k]) for k in ("x", "dt", "a", "b", "c"))
    p = rg.compile(lambda x, dt: rg.value_and_grad(lambda *s: rg.selective_scan(*s, a, b, c)[0].sum(), argnums=(0, 1))(x, dt), (x, dt),
                   validate="none", optimize=optimize)
    (scan,) = [s for s in p.plan_summary() if s.get("op") == "selective_scan"]
    assert [k for k, _ in scan["outs"]] == [0, 2]


# ---- plans, validation, layers -----------------------------------------------------------------------

def test_a_result_nobody_reads_has_no_slot():
    x, w = _t(1, 4, 8), _t(2, 8)
    c = rg.compile(lambda v: rg.causal_conv(v, w)[0], (x,), validate="none", device="cpu_devplan")
    (step,) = [s for s in c.plan_summary() if s.get("op") == "causal_conv"]
    assert [k for k, _ in step["outs"]] == [0]


def test_equal_calls_are_one_operator():
    x, w = _t(1, 4, 8), _t(2, 8)
    c = rg.compile(lambda v: rg.causal_conv(v, w)[0] + rg.causal_conv(v, w)[0] + rg.causal_conv(v, w, activation="silu")[0], (x,), validate="none")
    assert sum(s.get("op") == "causal_conv" for s in c.plan_summary()) == 2


def test_validation_names_the_operator_that_turns_bad():
    v, _, _ = ref.scan_inputs((1, 6, 2, 4, 1, "d"), "float32")
    v["a"][0, 0] = 300.0  # a growing state overflows
    args = [rg.tensor(v[k]) for k in ("x", "dt", "a", "b", "c")]
    args[1] = rg.tensor(np.full((1, 6, 2), 1.0, F))
    c = rg.compile(lambda *a: rg.selective_scan(*a)[0], tuple(args), validate="none")
    found = c.check(*args)
    assert not found.ok and "selective_scan" in str(found)


def test_profile_prices_the_operators():
    v, _, _ = ref.scan_inputs((1, 6, 2, 4, 1, "d"), "float32")
    args = tuple(rg.tensor(v[k]) for k in ("x", "dt", "a", "b", "c"))
    c = rg.compile(lambda *a: rg.selective_scan(*a)[0], args, validate="none")
    assert "selective_scan" in str(c.profile(*args, repeats=1))


@pytest.mark.parametrize("optimize", ["search", "search-linear", "standard", "none"])
@pytest.mark.parametrize("device", ["cpu", "cpu_devplan"])
def test_thorough_validation_and_every_optimizer(device, optimize):
    """Differences on the float64 shadow graph, the optimizer's check, and plans with the operators in
    the graph that the matrix search rewrites."""
    layer, params = _ssm()
    attn = nn.MultiHeadAttention(12, 2, qk_norm=True, rotary=100.0)
    weights = attn.init(random.key(1))
    x = rg.tensor(np.random.default_rng(0).standard_normal((2, 5, 12)).astype(F))
    mask = rg.tril(5)

    def step(p, v):
        return rg.value_and_grad(lambda q: (layer(q["ssm"], v + attn(q["attn"], v, mask)) ** 2.0).mean())(p)

    c = rg.compile(step, ({"ssm": params, "attn": weights}, x), validate="thorough", device=device, optimize=optimize)
    assert c.report["status"] == "ok", c.report


def _ssm(dtype="float32", **more):
    layer = nn.SelectiveSSM(12, states=6, taps=3, dt_rank=2, rotary=True, groups=2, dtype=dtype, **more)
    return layer, layer.init(random.key(3))


def test_a_prompt_read_at_once_or_token_by_token():
    """The same positions through one call, through two, and one token at a time: the states and results
    agree to the roundings of the parts, which run the same formulas (float64: 1e-12 of the size)."""
    layer, params = _ssm("float64")
    x = np.random.default_rng(0).standard_normal((2, 9, 12))
    whole, end = layer.extend(params, rg.tensor(x))
    state, parts = None, []
    for lo, hi in [(0, 4), (4, 5), (5, 6), (6, 9)]:
        y, state = layer.extend(params, rg.tensor(x[:, lo:hi]), state)
        parts.append(y.numpy())
    assert np.allclose(np.concatenate(parts, 1), whole.numpy(), rtol=0, atol=1e-12)
    assert state["pos"].tolist() == end["pos"].tolist() == [9, 9]
    for k in ("conv", "scan"):
        assert np.allclose(state[k].numpy(), end[k].numpy(), rtol=0, atol=1e-12)
    fresh, _ = layer.extend(params, rg.tensor(x), layer.state(2))
    assert np.allclose(fresh.numpy(), whole.numpy(), rtol=0, atol=1e-12)


def test_a_padded_batch_reads_as_its_sequences_alone():
    layer, params = _ssm("float64")
    x = np.random.default_rng(1).standard_normal((3, 7, 12))
    lengths = [7, 0, 4]
    y, state = layer.extend(params, rg.tensor(x), lengths=[11, -3, 4])  # read as within 0 .. 7
    assert state["pos"].tolist() == lengths
    for i, n in enumerate(lengths):
        assert (y.numpy()[i, n:] == 0.0).all()
        if n:
            alone, s = layer.extend(params, rg.tensor(x[i:i + 1, :n]))
            assert np.allclose(alone.numpy()[0], y.numpy()[i, :n], rtol=0, atol=1e-12)
            assert np.allclose(s["scan"].numpy()[0], state["scan"].numpy()[i], rtol=0, atol=1e-12)
        else:
            assert (state["scan"].numpy()[i] == 0.0).all() and (state["conv"].numpy()[i] == 0.0).all()


def test_layer_checks():
    with pytest.raises(ValueError, match="groups"):
        nn.SelectiveSSM(4, width=9, groups=2)
    with pytest.raises(ValueError, match="odd number of states"):
        nn.SelectiveSSM(4, states=5, rotary=True)
    layer = nn.SelectiveSSM(8)
    params = layer.init(random.key(0))
    step = np.log1p(np.exp(params["dt"]["b"].numpy()))
    assert params["in"]["w"].shape == (8, 16) and step.min() > 0.0009 and step.max() < 0.11
    assert layer(params, _t(1, 3, 8)).shape == (1, 3, 8)


def test_attention_with_normed_and_turned_heads():
    """Equal queries and keys are turned apart by their distance alone: attention with `rotary` is the
    same wherever the positions start; and the options leave the plain layer as it was."""
    x = rg.tensor(np.random.default_rng(2).standard_normal((2, 6, 16)))
    plain = nn.MultiHeadAttention(16, 4, dtype="float64")
    params = plain.init(random.key(1))
    assert set(params) == {"qkv", "out"}
    layer = nn.MultiHeadAttention(16, 4, dtype="float64", qk_norm=True, rotary=10000.0)
    own = layer.init(random.key(1))
    assert own["gain"].shape == (2, 4) and np.array_equal(own["qkv"]["w"].numpy(), params["qkv"]["w"].numpy())
    here = layer(own, x, rg.tril(6, "float64")).numpy()
    far = layer(own, x, rg.tril(6, "float64"), positions=rg.tensor((np.arange(6) + 4000).astype(np.int32))).numpy()
    # Angles of 4000 carry about 4000 u = 5e-13 more error.
    assert np.allclose(here, far, rtol=0, atol=1e-11)
    assert not np.allclose(here, plain(params, x, rg.tril(6, "float64")).numpy(), atol=1e-6)


def test_attention_options_keep_the_fused_attention():
    """The turned projection is read in place by the fused attention step, forward and backward."""
    layer, mask = nn.MultiHeadAttention(64, 2, qk_norm=True, rotary=10000.0), rg.tril(32)
    params = layer.init(random.key(0))
    x = rg.tensor(np.random.default_rng(0).standard_normal((2, 32, 64)).astype(F))
    c = rg.compile(lambda p, v: rg.value_and_grad(lambda q: (layer(q, v, mask) ** 2.0).sum())(p), (params, x), validate="none", device="cpu_devplan")
    kinds = [s["kind"] for s in c.plan_summary()]
    assert sum("attn" in k or "attention" in k for k in kinds) == 2, kinds
    block = nn.TransformerBlock(64, 2, qk_norm=True, rotary=100.0)
    assert block(block.init(random.key(0)), x, mask).shape == x.shape


def test_attention_turned_by_the_usual_base():
    """`rotary=True` is the base that `rotary_norm` has by default, not a base of 1."""
    x = rg.tensor(np.random.default_rng(4).standard_normal((1, 5, 8)).astype(F))
    layers = [nn.MultiHeadAttention(8, 2, rotary=r) for r in (True, 10000.0, 1.0, False, None)]
    params = layers[0].init(random.key(0))
    usual, same, other, off, none = (layer(params, x).numpy() for layer in layers)
    assert np.array_equal(usual, same) and not np.array_equal(usual, other)
    assert np.array_equal(off, none) and not np.array_equal(usual, off)
    block = [nn.TransformerBlock(8, 2, rotary=r) for r in (True, 10000.0)]
    params = block[0].init(random.key(1))
    assert np.array_equal(block[0](params, x).numpy(), block[1](params, x).numpy())


def test_layers_refuse_sizes_that_their_operators_do():
    """When they are made, not at their first call."""
    for states in (1, 5, 66, 0):
        with pytest.raises(ValueError, match="states"):
            nn.SelectiveSSM(8, states=states)
    for taps in (1, 9):
        with pytest.raises(ValueError, match="taps"):
            nn.SelectiveSSM(8, taps=taps)
    for options in ({"qk_norm": True}, {"rotary": 100.0}):
        for d, heads in ((6, 2), (516, 2)):
            with pytest.raises(ValueError, match="head"):
                nn.MultiHeadAttention(d, heads, **options)
    nn.MultiHeadAttention(6, 2)
    nn.MultiHeadAttention(512, 2, qk_norm=True, rotary=True)


def test_an_eps_that_float32_does_not_hold_is_refused():
    """It would be 0 there, and the norm of a head of zeros NaN."""
    zeros, gain = np.zeros((1, 2, 1, 4)), np.ones((1, 4))
    with pytest.raises(rg.DiagnosticError, match="eps_rounds_to_zero_in_the_dtype"):
        rg.rotary_norm(rg.tensor(zeros.astype(F)), rg.tensor(gain.astype(F)), eps=1e-50)
    for dtype, eps in (("float32", 1e-40), ("float64", 1e-50)):
        assert (rg.rotary_norm(rg.tensor(zeros.astype(dtype)), rg.tensor(gain.astype(dtype)), eps=eps).numpy() == 0.0).all()
    # Heads that are only turned have no norm, and no use for it.
    assert (rg.rotary_norm(rg.tensor(zeros.astype(F)), eps=1e-50).numpy() == 0.0).all()


def test_the_polynomial_of_the_logarithm_is_as_exact_as_its_comment_says():
    """The float32 kernels' log(1 + u) with the source's coefficients, every step rounded once: 48 bits of
    a product and a sum in 64 bits lose less than 2^-52 before the rounding to 24."""
    path = os.path.join(os.path.dirname(rg.__file__), "csrc", "hip", "sequence.hip")
    with open(path) as f:
        source = f.read()
    stated = float(re.search(r"([\d.]+) x 2\^-24 off at most", source).group(1))
    body = re.search(r"float log1p_\(float u\) \{(.*?)\n\}", source, re.S).group(1)
    first, *others = (np.float64(F(v)) for v in re.findall(r"(-?0\.\d+)f", body))
    assert len(others) == 8

    def rounded(v):
        return v.astype(F).astype(np.float64)

    worst = 0.0
    for exponent in range(-27, 0):
        start = int(F(2.0 ** exponent).view(np.int32))
        for low in range(start, start + 2 ** 23, 2 ** 21):
            u = np.arange(low, low + 2 ** 21 + 1, 1 if exponent >= -2 else 7, dtype=np.int32).view(F).astype(np.float64)
            p = np.full_like(u, first)
            for c in others:
                p = rounded(p * u + c)
            got = rounded(rounded(u * p) * u + u)
            want = np.log1p(u)
            worst = max(worst, float((np.abs(got - want) / want).max()) * 2.0 ** 24)
    assert stated - 0.02 <= worst <= stated, worst
