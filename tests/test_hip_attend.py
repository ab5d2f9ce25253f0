"""The kernels of attention with shaped scores, of its paged form and of the joint norm on the device:
values and gradients against the formulas in 64 bits, captured and replayed step loops against the
same steps one by one, and the operators run together."""

import numpy as np
import pytest

import rustautograd_amd as rg
from rustautograd_amd import optim
import attention_reference as ref

pytestmark = pytest.mark.gpu
F = np.float32


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", ref.CASES, ids=str)
def test_attention(case, dtype):
    ref.check(case, dtype, "hip")


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", ref.PAGED, ids=str)
def test_paged_attention(case, dtype):
    ref.check_paged(case, dtype, "hip")


@pytest.mark.parametrize("case", [ref.PAGED[i] for i in (1, 2, 3, 6)], ids=str)
def test_pages_that_are_not_there(case):
    ref.check_paged(case, "float32", "hip", ref.strange_tables)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("sizes", [(1,), (3, 16384, 16385), (100000, 1, 7), tuple(range(1, 131))], ids=len)
def test_norm(sizes, dtype):
    r = np.random.default_rng(len(sizes))
    parts = [r.standard_normal(n).astype(dtype) for n in sizes]
    got = float(optim.gradient_norm([rg.tensor(p) for p in parts]))
    want = np.sqrt(sum((p.astype(np.longdouble) ** 2).sum() for p in parts))
    # Sums of squares in 64 bits: at most the number of terms in roundings of 2^-53, far below one of
    # float32; the root halves them.
    assert abs(got - want) <= (np.finfo(dtype).eps + sum(sizes) * 2.0 ** -53) * want
