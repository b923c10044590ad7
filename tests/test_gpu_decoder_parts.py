"""Attention of a decoder's step where every one of an operand's 24 bits counts (decoder_parts.py), on every kernel."""
import numpy as np
import pytest

import decoder_parts as deep
import jade_hip
import test_gpu_decoder as base

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel", base.KERNELS)
@pytest.mark.parametrize("case", deep.CASES)
def test_no_part_is_lost(runtime, kernel, case):
    spec = base.cross_spec(*base.KERNELS[kernel])
    assert jade_hip.spec_describe(spec)["launch"]["kernel"] == kernel
    q, k, v, lengths = deep.inputs(spec, case, np.random.default_rng(60))
    want, off = deep.want(spec, case, q, k, v)
    got = base.run(runtime, spec, {"q": q, "k": k, "v": v, "lengths": lengths})["out"]
    base.within(got, want, off)


@pytest.mark.parametrize("nodes,dim", [(3, 64), (9, 128), (20, 60), (40, 64), (20, 96), (70, 90), (30, 128), (128, 128)])
def test_no_part_of_a_drafted_value_is_lost(runtime, nodes, dim):
    # Nodes that see themselves alone: an output is the node's value.
    rng = np.random.default_rng(61)
    spec = base.tree_spec(2, 2, 2, nodes, 5, dim)
    x = base.tree_inputs(rng, spec, [0, 0], [[-1] * nodes] * 2)
    x["v_draft"] = deep.deep(rng, x["v_draft"].size).reshape(x["v_draft"].shape)
    want = x["v_draft"].astype(np.float64)
    base.within(base.run(runtime, spec, x)["out"], want, 2 * base.dec.U * np.abs(want))
