"""The cases of decoder_parts.py do tell three bf16 parts from two, on the CPU."""
import numpy as np
import pytest

import decoder_parts as deep
from test_gpu_decoder import KERNELS, cross_spec


def test_parts_are_exact():
    rng = np.random.default_rng(1)
    x = np.ldexp(rng.standard_normal(100000), rng.integers(-60, 60, 100000)).astype(np.float32)
    assert (sum(p.astype(np.float64) for p in deep.parts(x, 3)) == x).all()
    assert (np.abs(sum(p.astype(np.float64) for p in deep.parts(x, 2)) - x) <= 2.0 ** -17 * np.abs(x)).all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("case", deep.CASES)
def test_two_parts_are_noticed(kernel, case):
    spec = cross_spec(*KERNELS[kernel])
    q, k, v, _ = deep.inputs(spec, case, np.random.default_rng(60))
    want, off = deep.want(spec, case, q, k, v)
    three, two = (np.abs(deep.simulate(spec, case, q, k, v, n) - want) for n in (3, 2))
    # Three parts leave nothing but what the simulation rounds (the scaled query, and p to FP32).
    assert (three <= 0.5 * off).all()
    # Two are out of bounds, by far for some and, but for p, whose bits are as they come, for many.
    assert (two > 1.5 * off).any()
    if case != "p":
        assert (two > off).mean() > 0.4
