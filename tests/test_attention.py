"""Attention with shaped scores, its paged form and the joint norm through the engine on the CPU
oracle: values and gradients against the formulas in 64 bits, gradients against differences, and
refusals."""

import numpy as np
import pytest

import rustautograd_amd as rg
from rustautograd_amd import optim
import attention_reference as ref

F = np.float32


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", ref.CASES, ids=str)
def test_attention(case, dtype):
    ref.check(case, dtype, "cpu")


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", ref.PAGED, ids=str)
def test_paged_attention(case, dtype):
    ref.check_paged(case, dtype, "cpu")


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("case, at", ref.ODD[:-2], ids=str)
def test_what_is_no_number_reaches_what_sees_it(case, at, bad, dtype):
    ref.check_odd(case, at, bad, dtype, "cpu")


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("case", [ref.PAGED[i] for i in (3, 4, 6, 9, 11, 13)], ids=str)
def test_a_token_that_is_no_number(case, bad, dtype):
    ref.check_odd_token(case, bad, dtype, "cpu")


@pytest.mark.parametrize("case", [ref.CASES[i] for i in (6, 11, 18)], ids=str)
def test_a_gradient_alone(case):
    case = (*case[:5], case[5] + "s" * ("s" not in case[5]), case[6])
    ref.check_each_alone(case, "float32", "cpu")


@pytest.mark.parametrize("case", [ref.PAGED[i] for i in (1, 2, 3, 6)], ids=str)
def test_pages_that_are_not_there(case):
    ref.check_paged(case, "float32", "cpu", ref.strange_tables)


@pytest.mark.parametrize("case", [ref.PAGED[i] for i in (1, 3, 14)], ids=str)
def test_positions_past_the_table(case):
    ref.check_paged(case, "float32", "cpu", ref.past_the_table)


def test_device_plans_run_the_same_operators():
    ref.check(ref.CASES[11], "float32", "cpu_devplan")
    ref.check(ref.CASES[12], "float64", "cpu_devplan")
    ref.check_paged(ref.PAGED[3], "float32", "cpu_devplan")


def _by_differences(fn, inputs, step=1e-6):
    """Central differences of fn's scalar along one direction an input; both sides in float64, whose
    truncation (step^2) and rounding (1e-16 / step) leave about 1e-9 of the size."""
    tensors = tuple(rg.tensor(v) for v in inputs)
    value = rg.compile(fn, tensors, validate="none")
    grads = rg.compile(lambda *v: rg.value_and_grad(fn, argnums=tuple(range(len(v))))(*v)[1], tensors, validate="none")(*tensors)
    r = np.random.default_rng(5)
    for k, v in enumerate(inputs):
        way = r.standard_normal(v.shape)
        ends = []
        for s in (step, -step):
            moved = list(inputs)
            moved[k] = v + s * way
            ends.append(float(value(*[rg.tensor(m) for m in moved])))
        want, got = (ends[0] - ends[1]) / (2 * step), float((grads[k].numpy() * way).sum())
        assert abs(got - want) <= 1e-7 * max(1.0, abs(want)), (k, got, want)


@pytest.mark.parametrize("case", [ref.CASES[i] for i in (6, 11, 17, 18)], ids=str)
def test_gradients_are_the_differences(case):
    case = (*case[:5], case[5].replace("j", "") + ("" if "s" in case[5] else "s"), case[6])
    v = ref.inputs(case, np.dtype("float64"))
    dy = rg.tensor(v["dy"])
    fn = lambda q, k, val, s: (ref.call(case, {"q": q, "k": k, "v": val, "slopes": s}, v) * dy).sum()
    _by_differences(fn, [v["q"], v["k"], v["v"], v["slopes"]])


def test_norm_gradient_is_the_difference():
    r = np.random.default_rng(1)
    parts = [r.standard_normal(s) for s in ((), (3,), (2, 5), (1, 4, 2))]
    _by_differences(lambda *v: rg.sin(optim.gradient_norm(list(v)) * 1.7), parts)
    zero = [rg.zeros((2, 3)), rg.zeros(4)]
    grads = rg.grad(lambda g: optim.gradient_norm(g))(zero)
    assert all((g.numpy() == 0).all() for g in grads)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
def test_norm_and_clip(dtype):
    r = np.random.default_rng(2)
    tree = {"a": r.standard_normal((5, 7)).astype(dtype), "b": [r.standard_normal(n).astype(dtype) for n in (1, 3, 400)]}
    flat = np.concatenate([tree["a"].ravel(), *tree["b"]]).astype(np.float64)
    given = rg.tree.map(rg.tensor, tree)
    for most in (0.5, 1e6):
        clipped, norm = rg.compile(lambda g: optim.clip_gradients(g, most), (given,), validate="none")(given)
        want = np.sqrt((flat ** 2).sum())
        # The squares are summed in 64 bits; one rounding of the root, one of the factor, one of the product.
        u = np.finfo(dtype).eps / 2
        assert abs(float(norm) - want) <= 2 * u * want
        scaled = flat * min(1.0, most / want)
        got = np.concatenate([x.numpy().ravel() for x in rg.tree.leaves(clipped)])
        assert (np.abs(got - scaled) <= 5 * u * np.abs(scaled)).all()
        if most > want:
            assert np.array_equal(got.astype(np.float64), flat)


def test_norm_of_values_whose_squares_do_not_fit():
    assert float(optim.gradient_norm([rg.tensor(np.full((4,), 1e30, F))])) == F(2e30)
    assert float(optim.gradient_norm([rg.tensor(np.full((4,), 1e-30, F))])) == F(2e-30)


@pytest.mark.parametrize("bad, clipped", [(np.inf, [0.0, np.nan]), (np.nan, [np.nan, np.nan])])
def test_clip_where_the_norm_is_no_number(bad, clipped):
    got, norm = optim.clip_gradients([rg.tensor(np.array([1.0, bad], F))], 1.0)
    assert np.array_equal(got[0].numpy(), np.array(clipped, F), equal_nan=True)
    assert np.array_equal(norm.numpy(), F(bad), equal_nan=True)


def _code(fn):
    with pytest.raises(rg.DiagnosticError) as e:
        fn()
    return e.value.diagnostic["code"]


def _t(*shape, dtype=F):
    return rg.tensor(np.ones(shape, dtype))


def _i(*values):
    return rg.tensor(np.array(values, np.int32))


def test_refusals():
    q, k = _t(2, 5, 4, 8), _t(2, 5, 2, 8)
    docs, wrong = rg.zeros((2, 5), "int32"), [
        (lambda: rg.attention(q, k, _t(2, 5, 2, 7)), "SHAPE_MISMATCH"),
        (lambda: rg.attention(q, _t(2, 6, 2, 8), _t(2, 6, 2, 8)), "SHAPE_MISMATCH"),
        (lambda: rg.attention(q, _t(2, 5, 3, 8), _t(2, 5, 3, 8)), "SHAPE_MISMATCH"),
        (lambda: rg.attention(q, k), "INVALID_ARGUMENT"),
        (lambda: rg.attention(q, None, k), "INVALID_ARGUMENT"),
        (lambda: rg.attention(q), "INVALID_ARGUMENT"),
        (lambda: rg.attention(q, heads=(2, 2)), "SHAPE_MISMATCH"),
        (lambda: rg.attention(q, heads=(0, 2)), "INVALID_ARGUMENT"),
        (lambda: rg.attention(q, heads=(4,)), "INVALID_ARGUMENT"),
        (lambda: rg.attention(q, k, k, heads=(4, 2)), "INVALID_ARGUMENT"),
        (lambda: rg.attention(_t(5, 4, 8), _t(5, 4, 8), _t(5, 4, 8)), "SHAPE_MISMATCH"),
        (lambda: rg.attention(_t(1, 2, 1, 257), _t(1, 2, 1, 257), _t(1, 2, 1, 257)), "SHAPE_MISMATCH"),
        (lambda: rg.attention(q, k, k, cap=0.0), "INVALID_ARGUMENT"),
        (lambda: rg.attention(q, k, k, cap=-3.0), "INVALID_ARGUMENT"),
        (lambda: rg.attention(q, k, k, cap=float("nan")), "INVALID_ARGUMENT"),
        (lambda: rg.attention(q, k, k, cap=float("inf")), "INVALID_ARGUMENT"),
        (lambda: rg.attention(q, k, k, cap=1e-40), "INVALID_ARGUMENT"),
        (lambda: rg.attention(q, k, k, scale=float("inf")), "INVALID_ARGUMENT"),
        (lambda: rg.attention(q, k, k, slopes=_t(2)), "SHAPE_MISMATCH"),
        (lambda: rg.attention(q, k, k, slopes=_t(4, dtype=np.float64)), "DTYPE_MISMATCH"),
        (lambda: rg.attention(q, k, _t(2, 5, 2, 8, dtype=np.float64)), "DTYPE_MISMATCH"),
        (lambda: rg.attention(q, k, k, documents=rg.zeros((2, 5))), "DTYPE_MISMATCH"),
        (lambda: rg.attention(q, k, k, documents=rg.zeros((2, 4), "int32")), "SHAPE_MISMATCH"),
        (lambda: rg.attention(q, k, k, prefix=_i(1)), "SHAPE_MISMATCH"),
        (lambda: rg.attention(q, k, k, lengths=_i(1, 2, 3)), "SHAPE_MISMATCH"),
        (lambda: rg.attention(docs.reshape(2, 5, 1, 1), docs.reshape(2, 5, 1, 1), docs.reshape(2, 5, 1, 1)), "UNSUPPORTED_DTYPE"),
    ]
    for n, (fn, code) in enumerate(wrong):
        assert _code(fn) == code, n


def test_scales_that_float32_does_not_hold_are_refused():
    q, k = rg.ones((1, 4, 2, 8)), rg.ones((1, 4, 2, 8))
    for kw in ({"scale": 1e31}, {"cap": 1e-31}, {"cap": 1e31}, {"scale": 1e10, "cap": 1e-25}):
        with pytest.raises(rg.DiagnosticError, match="INVALID_ARGUMENT"):
            rg.attention(q, k, k, **kw)
    assert np.isfinite(rg.attention(q, k, k, scale=1e5, cap=1e-20).numpy()).all()


def test_paged_refusals():
    x, pages, table, first = _t(2, 1, 8, 8), _t(6, 4, 2, 8), rg.zeros((2, 3), "int32"), _i(1, 2)
    call = lambda x=x, cache=(pages, pages), table=table, first=first, heads=(4, 2), **kw: rg.paged_attention(x, cache=cache, table=table, first=first, heads=heads, **kw)
    assert call()[0].shape == (2, 1, 4, 8)
    for n, (fn, code) in enumerate([
        (lambda: call(cache=(pages,)), "INVALID_ARGUMENT"),
        (lambda: call(cache=(pages, _t(6, 5, 2, 8))), "SHAPE_MISMATCH"),
        (lambda: call(cache=(_t(6, 4, 1, 8), _t(6, 4, 1, 8))), "SHAPE_MISMATCH"),
        (lambda: call(cache=(pages, _t(6, 4, 2, 8, dtype=np.float64))), "DTYPE_MISMATCH"),
        (lambda: call(table=rg.zeros((3, 3), "int32")), "SHAPE_MISMATCH"),
        (lambda: call(table=rg.zeros((2, 3))), "DTYPE_MISMATCH"),
        (lambda: call(first=_i(1)), "SHAPE_MISMATCH"),
        (lambda: call(first=rg.zeros((2,))), "DTYPE_MISMATCH"),
        (lambda: call(lengths=_i(1)), "SHAPE_MISMATCH"),
        (lambda: call(heads=None), "INVALID_ARGUMENT"),
        (lambda: call(cap=0.0), "INVALID_ARGUMENT"),
        (lambda: rg.grad(lambda x: call(x=x)[0].sum())(x), "GRAD_UNSUPPORTED"),
    ]):
        assert _code(fn) == code, n


def test_second_derivatives_are_refused():
    q = _t(1, 3, 1, 4)
    inner = lambda q: rg.grad(lambda q: rg.attention(q, q, q).sum())(q).sum()
    assert _code(lambda: rg.grad(inner)(q)) == "GRAD_UNSUPPORTED"


def test_norm_refusals():
    assert _code(lambda: optim.gradient_norm([rg.zeros(3, "int32")])) == "UNSUPPORTED_DTYPE"
    assert _code(lambda: optim.gradient_norm([rg.zeros(3), rg.zeros(3, "float64")])) == "DTYPE_MISMATCH"
    with pytest.raises(ValueError):
        optim.gradient_norm([])
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            optim.clip_gradients([rg.zeros(3)], bad)


def test_shared_operands_add_their_gradients():
    """One tensor as queries, keys and values: the sum of the three gradients."""
    r = np.random.default_rng(3)
    x, dy = rg.tensor(r.standard_normal((2, 9, 2, 6))), rg.tensor(r.standard_normal((2, 9, 2, 6)))
    parts = rg.grad(lambda p: (rg.attention(p[0], p[1], p[2], cap=3.0) * dy).sum())([x, x, x])
    whole = rg.grad(lambda x: (rg.attention(x, x, x, cap=3.0) * dy).sum())(x)
    np.testing.assert_allclose(whole.numpy(), sum(p.numpy() for p in parts), rtol=1e-13, atol=1e-15)


# ---- layers --------------------------------------------------------------------------------------------

def _layer(**kw):
    from rustautograd_amd import nn, random
    layer = nn.MultiHeadAttention(24, 6, dtype="float64", init=nn.normal_init(0.4), **kw)
    return layer, layer.init(random.key(3))


LAYERS = [{}, {"rotary": True, "qk_norm": True}, {"kv_heads": 2, "cap": 4.0, "distance": True}, {"kv_heads": 3, "rotary": True}]


@pytest.mark.parametrize("kw", LAYERS, ids=str)
def test_a_layer_read_in_chunks_is_the_layer_at_once(kw):
    """In float64: sums in other orders leave about 1e-15, of which each layer makes a few."""
    layer, params = _layer(**kw)
    r = np.random.default_rng(7)
    x = r.standard_normal((2, 11, 24))
    whole = (layer(params, rg.tensor(x)) if layer.shaped else layer(params, rg.tensor(x), mask=rg.tril(11, "float64"))).numpy()
    state, out, at = layer.state(2, 13, page=4), [], 0
    for n in (5, 1, 1, 4):
        y, state = layer.extend(params, rg.tensor(x[:, at:at + n].copy()), state)
        out.append(y.numpy())
        at += n
    np.testing.assert_allclose(np.concatenate(out, 1), whole, rtol=1e-12, atol=1e-13)
    assert state["pos"].numpy().tolist() == [11, 11]


def test_a_padded_prompt_goes_on_as_if_it_were_alone():
    layer, params = _layer(kv_heads=2, cap=4.0, rotary=True)
    r = np.random.default_rng(8)
    x, after = r.standard_normal((2, 6, 24)), r.standard_normal((2, 1, 24))
    y, state = layer.extend(params, rg.tensor(x), layer.state(2, 9, page=2), lengths=np.array([3, 9], np.int32))
    assert state["pos"].numpy().tolist() == [3, 6]
    np.testing.assert_array_equal(y.numpy()[0, 3:], np.broadcast_to(params["out"]["b"].numpy(), (3, 24)))
    y, state = layer.extend(params, rg.tensor(after), state)
    for b, n in ((0, 3), (1, 6)):
        alone = np.concatenate([x[b:b + 1, :n], after[b:b + 1]], axis=1)
        np.testing.assert_allclose(y.numpy()[b, 0], layer(params, rg.tensor(alone)).numpy()[0, -1], rtol=1e-12, atol=1e-13)


def test_plain_masks_as_the_layers_own():
    """Documents, a prefix and lengths against the same layer under the mask that they stand for."""
    layer, params = _layer()
    r = np.random.default_rng(9)
    x = rg.tensor(r.standard_normal((2, 8, 24)))
    at = np.arange(8)
    causal = at[None] <= at[:, None]
    docs = np.array([[4, 4, 4, 7, 7, 7, 7, 7], [1, 1, 2, 2, 2, 3, 3, 3]], np.int32)
    same = docs[:, :, None] == docs[:, None, :]
    prefix = np.array([3, 6], np.int32)
    early = at[None, None] < prefix[:, None, None]
    for got, mask in ((layer(params, x, documents=docs), causal & same), (layer(params, x, prefix=prefix), causal | early),
                      (layer(params, x, documents=docs, prefix=prefix), (causal | early) & same)):
        want = layer(params, x, mask=rg.tensor(mask[:, None].astype(np.float64)))
        np.testing.assert_allclose(got.numpy(), want.numpy(), rtol=1e-12, atol=1e-13)
    got = layer(params, x, lengths=np.array([5, 8], np.int32)).numpy()
    want = layer(params, x, mask=rg.tensor(causal.astype(np.float64))).numpy()
    np.testing.assert_allclose(got[0, :5], want[0, :5], rtol=1e-12, atol=1e-13)
    np.testing.assert_allclose(got[1], want[1], rtol=1e-12, atol=1e-13)


@pytest.mark.parametrize("optimize", ["search", "search-linear", "standard", "none"])
@pytest.mark.parametrize("device", ["cpu", "cpu_devplan"])
def test_block_trains_with_the_clip_and_passes_thorough_validation(device, optimize):
    """A block's gradients against differences on the float64 shadow graph, as thorough validation takes
    them, the clip within; plans with the operators in the graph that the matrix search rewrites."""
    from rustautograd_amd import nn, random
    block = nn.TransformerBlock(16, 4, mlp_ratio=2, kv_heads=2, cap=4.0, distance=True)
    params = block.init(random.key(1))
    x, t = (random.normal(random.key(k), (2, 6, 16)) for k in (2, 3))
    opt = optim.adamw(1e-3)
    docs = np.array([[0, 0, 0, 1, 1, 1], [0, 0, 0, 0, 0, -1]], np.int32)

    def step(state, t):
        loss = lambda p: nn.mse_loss(block(p, x, documents=docs), t)
        value, grads = rg.value_and_grad(loss)(state["p"])
        grads, norm = optim.clip_gradients(grads, 0.01)
        p, o = opt.update(grads, state["o"], state["p"])
        return {"p": p, "o": o}, (value, norm)

    program = rg.compile(step, ({"p": params, "o": opt.init(params)}, t), validate="thorough", device=device, optimize=optimize)
    assert program.report["status"] == "ok", program.report
    r = rg.run(program, {"p": params, "o": opt.init(params)}, [t], steps=3)
    assert r.status == "completed" and np.isfinite(r.history["aux.0"]).all()


def test_profile_prices_the_operators():
    q = _t(1, 6, 2, 4)
    program = rg.compile(lambda q: (rg.attention(q, q, q).sum(), optim.gradient_norm([q])), (q,), validate="none")
    said = str(program.profile(q, repeats=1))
    assert "attention" in said and "joint_norm" in said


def test_layer_refusals():
    from rustautograd_amd import nn, random
    for kw in ({"kv_heads": 4}, {"kv_heads": 0}, {"cap": 0.0}, {"cap": -1.0}):
        with pytest.raises(ValueError):
            nn.MultiHeadAttention(24, 6, **kw)
    layer = nn.MultiHeadAttention(24, 6, cap=3.0, dropout_rate=0.1)
    params, x = layer.init(random.key(0)), rg.zeros((1, 4, 24))
    with pytest.raises(ValueError):
        layer(params, x, mask=rg.tril(4))
    with pytest.raises(ValueError):
        layer(params, x, key=random.key(1))
    with pytest.raises(ValueError):
        layer.state(0, 5)
    ahead = nn.MultiHeadAttention(24, 6, causal=False)
    with pytest.raises(ValueError):
        ahead.extend(ahead.init(random.key(0)), x, ahead.state(1, 8))
