"""The sequence operators' kernels at the sizes where they take other forms: several channels a lane and
long runs of the convolution, many chunks and blocks of several chunks of the scan."""

import numpy as np
import pytest

import rustautograd_amd as rg
from rustautograd_amd import random
import sequence_reference as ref
import sequence_sizes as sizes

pytestmark = pytest.mark.gpu


def _conv(v, lengths, silu):
    dy, dn = rg.tensor(v["dy"]), rg.tensor(v["dnext"])

    def fn(g):
        y, nxt = rg.causal_conv(g["x"], g["w"], g.get("bias"), g.get("state"), lengths, "silu" if silu else None)
        return (y * dy).sum() + (nxt * dn).sum(), (y, nxt)

    (y, nxt), grads = ref._differentiated(fn, {n: v[n] for n in ("x", "w", "bias", "state")}, "hip")
    return {"y": y, "next": nxt, **{"d" + n: g for n, g in grads.items()}}


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case, f32, f64", sizes.CONV_SIZES, ids=str)
def test_conv_of_whole_numbers(case, f32, f64, dtype):
    """Every sum is exact: equal, not near."""
    v, lengths, _ = sizes.conv_whole(case, dtype)
    want, _ = sizes.conv(v["x"], v["w"], v["bias"], v["state"], lengths, False, v["dy"], v["dnext"])
    assert np.abs(want["dw"]).max() < 2.0 ** 24
    if lengths is not None:
        v["x"][:] = np.where((np.arange(case[1])[None] < lengths[:, None])[:, :, None], v["x"], np.nan)
    for name, got in _conv(v, lengths, False).items():
        assert np.array_equal(got, want[name].astype(dtype)), name


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case, f32, f64", [c for c in sizes.CONV_SIZES if "a" in c[0][4]], ids=str)
def test_conv_with_silu(case, f32, f64, dtype):
    v, lengths, _ = ref.conv_inputs(case, dtype)
    want, size = sizes.conv(v["x"], v["w"], v["bias"], v["state"], lengths, True, v["dy"], v["dnext"])
    if lengths is not None:
        ref.fill_outside(v, lengths, ["x"])
    # Products and sums of an output and its activation; for dw and dbias a run and the rows that are folded, too.
    k = 2 * case[3] + 24
    rows = (f32 if dtype == "float32" else f64)[1] + 4 + case[0] * -(-case[1] // 32)
    for name, got in _conv(v, lengths, True).items():
        if name == "next":
            assert np.array_equal(got, want["next"].astype(dtype))
        else:
            ref.agree(got, want[name], size[name], k + (rows if name in ("dw", "dbias") else 0), dtype, name)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", ref.SCAN_CASES, ids=str)
def test_scan_within_its_roundings(case, dtype):
    sizes.check_scan(case, dtype, "hip", sizes.scan_chunks(case, dtype)[2])


@pytest.mark.parametrize("with_last", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case, chunks, blocks", sizes.SCAN_SIZES, ids=str)
def test_scan_of_many_chunks(case, chunks, blocks, dtype, with_last):
    sizes.check_scan(case, dtype, "hip", sizes.scan_chunks(case, dtype)[2], with_last)


def test_a_scan_of_many_chunks_inside_control_flow():
    """A `scan` body whose operator is cut into chunks, in the enclosing program's workspace: the bits of
    the same steps written out, forward and back."""
    case = (2, 300, 6, 16, 1, "zs")
    assert sizes.scan_chunks(case, "float32")[0] > 1
    v = [ref.scan_inputs(case, "float32", seed)[0] for seed in range(3)]
    fixed = {k: rg.tensor(v[0][k]) for k in ("a", "d") if v[0][k] is not None}
    stacked = {k: rg.tensor(np.stack([w[k] for w in v])) for k in ("x", "dt", "b", "c", "z")}
    weight = rg.tensor(np.stack([w["dy"] for w in v]))
    start = rg.tensor(v[0]["state"])

    def step(h, p):
        y, h = rg.selective_scan(p["x"], p["dt"], fixed["a"], p["b"], p["c"], z=p["z"], state=h)
        return h, y

    def looped(g):
        last, ys = rg.scan(step, g["state"], {k: g[k] for k in stacked})
        return (ys * weight).sum() + last.sum(), (ys, last)

    def written_out(g):
        h, ys = g["state"], []
        for i in range(3):
            h, y = step(h, {k: g[k][i] for k in stacked})
            ys.append(y.reshape(1, *y.shape))
        ys = rg.concatenate(ys, 0)
        return (ys * weight).sum() + h.sum(), (ys, h)

    inputs = {**{k: t.numpy() for k, t in stacked.items()}, "state": start.numpy()}
    (one, other) = (ref._differentiated(f, inputs, "hip") for f in (looped, written_out))
    for got, want in zip(one[0], other[0]):
        assert np.array_equal(got, want)
    for k in inputs:
        assert np.array_equal(one[1][k], other[1][k]), k


def _long_maps(joined):
    """Gradients of the maps of a scan of 2137153 positions, 17 channels (two tiles, each a partial row) and
    63 states, less those that the formulas give. Rates of minus infinity and whole numbers keep every
    value exact: db = c sum dy x, dc = b sum dy x. Made and compared on the device."""
    length, width, states = 2 ** 21 + 40001, 17, 63

    def whole(key, shape):
        return rg.floor(random.uniform(key, shape) * 5.0) - 2.0

    def program(key):
        keys = random.split(key, 4)
        x, dy = (whole(k, (1, length, width)) for k in keys[:2])
        b, c = (whole(k, (1, length, 1, states)) for k in keys[2:])
        dt, rates = rg.broadcast_to(rg.ones((1,)), x.shape), rg.tensor(np.full((width, states), -np.inf, np.float32))
        maps = (rg.concatenate([b, c], 2), None) if joined else (b, c)
        given = {k: m for k, m in zip("bc", maps) if m is not None}
        grads = rg.grad(lambda g: (rg.selective_scan(x, dt, rates, g["b"], g.get("c"))[0] * dy).sum())(given)
        sums = (x * dy).sum(-1).reshape(1, length, 1, 1)
        wants = (rg.concatenate([c, b], 2) * sums,) if joined else (c * sums, b * sums)
        return [rg.abs(g - w).max() for g, w in zip((grads[k] for k in sorted(grads)), wants)], rg.abs(grads["b"]).max()

    key = random.key(0)
    return rg.compile(program, (key,), validate="none")(key)


def test_folds_that_do_not_fit_one_launch():
    """Two gradients of 1.35e8 values each: the threads that fold both are more than a launch may have."""
    off, most = _long_maps(joined=False)
    assert [float(v) for v in off] == [0.0, 0.0] and float(most) > 20.0


def test_a_fold_that_no_launch_holds_is_refused():
    """One gradient of 2.7e8 values, an odd multiple of two."""
    with pytest.raises(rg.DiagnosticError, match="exceeds the launch limit"):
        _long_maps(joined=True)
