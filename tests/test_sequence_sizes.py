"""The larger sequence cases without a device: which kernel each runs on, the references against the
position-by-position ones, and that the scan's bounds are fine enough to find a wrong carry."""

import numpy as np
import pytest

import sequence_reference as ref
import sequence_sizes as sizes
from test_hip_sequence import WALKS


@pytest.mark.parametrize("case, f32, f64", sizes.CONV_SIZES, ids=str)
def test_convolutions_run_in_the_forms_they_are_meant_for(case, f32, f64):
    assert sizes.conv_form(case, "float32") == f32 and sizes.conv_form(case, "float64") == f64


def test_convolutions_of_few_positions_run_one_at_a_time():
    assert [sizes.conv_form((2, t, 7, 4, ""), "float32") for t in (1, 4, 17)] == [(1, 1), (1, 1), (1, 4)]


@pytest.mark.parametrize("case, chunks, blocks", sizes.SCAN_SIZES, ids=str)
def test_scans_are_cut_as_meant(case, chunks, blocks):
    for dtype in ("float32", "float64"):
        assert sizes.scan_chunks(case, dtype)[:2] == (chunks, blocks)


def test_rotations_walk_several_tokens():
    """A block's groups of lanes are at most 64: fewer of them than heads of tokens, which they do not divide."""
    for case in WALKS[2:]:
        for dtype in ("float32", "float64"):
            batch, length, sections, passing, head, _ = case
            blocks, heads = sizes.rotary_blocks(case, dtype), sum(sections) + passing
            assert blocks == 512 and batch * length * heads > blocks * (64 if head == 8 else 4)


@pytest.mark.parametrize("case", ref.CONV_CASES, ids=str)
def test_the_convolution_at_once_is_that_by_positions(case):
    v, lengths, silu = ref.conv_inputs(case, "float64")
    args = (v["x"], v["w"], v["bias"], v["state"], lengths, silu, v["dy"], v["dnext"])
    out, size = sizes.conv(*args)
    for got, want in ((out, ref.conv(*args)), (size, ref.conv(*args, mag=True))):
        for name in got:
            assert np.allclose(got[name], want[name], rtol=1e-12, atol=1e-12), name


@pytest.mark.parametrize("with_last", [True, False])
@pytest.mark.parametrize("case", ref.SCAN_CASES, ids=str)
def test_the_scan_at_once_is_that_by_positions(case, with_last):
    v, lengths, soft = ref.scan_inputs(case, "float64")
    args = (*(v[k] for k in ("x", "dt", "a", "b", "c", "d", "z", "state")), lengths, soft, v["dy"], v["dlast"] if with_last else None)
    got, room = sizes.scan(*args, "float64", 64)
    want = ref.scan(*args)
    for name in got:
        assert np.allclose(got[name], want[name], rtol=1e-11, atol=1e-11), name
        assert (room[name] >= 0.0).all()


@pytest.mark.parametrize("case", [ref.SCAN_CASES[i] for i in (3, 6, 7, 12, 15, 16)], ids=str)
@pytest.mark.parametrize("dtype", ["float32", "float64"])
def test_scan_within_its_roundings(case, dtype):
    sizes.check_scan(case, dtype, "cpu", sizes.scan_chunks(case, dtype)[2])


@pytest.mark.parametrize("case", [ref.SCAN_CASES[15], ref.SCAN_CASES[16]], ids=str)
def test_the_bounds_find_a_wrong_carry(case):
    """A state carried into the sequence's second half wrong by a thousandth of itself, or a gradient
    carried back out of it so: found in the results of the half that takes it."""
    v, lengths, soft = ref.scan_inputs(case, "float32")
    chunk, cut = sizes.scan_chunks(case, "float32")[2], case[1] // 2
    names = ("x", "dt", "a", "b", "c", "d", "z")
    ends = np.full(case[0], case[1]) if lengths is None else lengths
    want, room = sizes.scan(*(v[k] for k in names), v["state"], ends, soft, v["dy"], v["dlast"], "float32", chunk)

    def half(span, state, ends, dlast):
        part = [v[k][:, span] if k in ("x", "dt", "b", "c", "z") and v[k] is not None else v[k] for k in names]
        return sizes.scan(*part, state, np.clip(ends, 0, None), soft, v["dy"][:, span], dlast, "float32", chunk)[0]

    early, late = slice(0, cut), slice(cut, None)
    first = half(early, v["state"], np.minimum(ends, cut), None)
    for wrong in (1.0, 1.001):
        second = half(late, wrong * first["last"], ends - cut, v["dlast"])
        for k in ("y", "ddt"):
            assert np.any(np.abs(second[k] - want[k][:, late]) > 1.01 * room[k][:, late]) == (wrong != 1.0), (k, wrong)
    for wrong in (1.0, 1.001):
        again = half(early, v["state"], np.minimum(ends, cut), wrong * half(late, first["last"], ends - cut, v["dlast"])["dstate"])
        for k in ("dx", "ddt"):
            assert np.any(np.abs(again[k] - want[k][:, early]) > 1.01 * room[k][:, early]) == (wrong != 1.0), (k, wrong)
