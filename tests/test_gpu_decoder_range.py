"""Operands at the ends of FP32's range in the attention of a decoder's step, on every kernel: bf16 parts have to carry
them as FP32 does, or what they do not carry has to be noticed and done in FP32. The operands are chosen so that FP32 sums
are exact or one key takes all, so the tolerances are a few roundings."""
import numpy as np
import pytest

import decoder_oracle as dec
import jade_hip
import test_gpu_decoder as base

pytestmark = pytest.mark.gpu

KERNELS = base.KERNELS


def query_of(dim):
    """A query element that is eight bits after the kernels' scaling, log2(e) / sqrt(dim)."""
    scale = np.float32(1) / np.sqrt(np.float32(dim)) * np.float32(1.44269504088896340736)
    for bits in range(128, 256):
        want = np.float32(bits * 2.0 ** 51)
        for q in (want / scale, np.nextafter(want / scale, np.float32(0)), np.nextafter(want / scale, np.float32(np.inf))):
            if q * scale == want:
                return q
    raise AssertionError(dim)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("single", [True, False])
def test_scores_of_minus_ten_to_the_36(runtime, kernel, single):
    # Scores that FP32 holds, but not times 2^24 (the scale of Q's parts), all their products of one sign. One key has
    # the least of them by a factor of two, or is the only one: its weight is 1, all others are 0, the output is its
    # value. Off by the division: 2.
    spec = base.cross_spec(*KERNELS[kernel])
    assert jade_hip.spec_describe(spec)["launch"]["kernel"] == kernel
    rng = np.random.default_rng(50)
    b, n = spec["batch"], spec["keys"]
    lengths = [1] * b if single else [n, n - 1, max(2, n // 2)] + [n] * (b - 3)
    x = base.cross_inputs(rng, spec, lengths)
    wins = [int(rng.integers(0, length)) for length in lengths]
    x["q"][:] = query_of(spec["dim"])
    x["k"][:] = -(2.0 ** 58)
    for i, win in enumerate(wins):
        x["k"][i, :, win] = -(2.0 ** 57)
    got = base.run(runtime, spec, x)["out"].reshape(x["q"].shape)
    group = spec["heads"] // spec["kv_heads"]
    for i, win in enumerate(wins):
        want = np.repeat(x["v"][i, :, win], group, axis=0)[:, None, :].astype(np.float64)
        want = np.broadcast_to(want, got[i].shape)
        base.within(got[i], want, 2 * dec.U * np.abs(want))


@pytest.mark.parametrize("heads", [5, 20, 40, 300])
@pytest.mark.parametrize("dim", [64, 96, 100, 128])
@pytest.mark.parametrize("keys", [7, 300])
def test_scores_whose_dims_cancel(runtime, heads, dim, keys):
    # The first key's score is -2a + a + a = 0 like all others', in exact steps, but -2a times 2^24 is past FP32's
    # range. So all weights are 1 and the output is the mean, which the first key's value dominates.
    rng = np.random.default_rng(51)
    spec = base.cross_spec(1, heads, 1, 1, keys, dim)
    x = base.cross_inputs(rng, spec, [keys])
    x["q"][:] = query_of(dim)
    x["k"][:] = 0
    x["k"][0, 0, 0, [0, 16, 32]] = [-(2.0 ** 46), 2.0 ** 45, 2.0 ** 45]
    x["v"][0, 0, 0] += np.float32(keys)
    values = x["v"][0, 0].astype(np.float64)
    want = np.broadcast_to(values.mean(axis=0), (heads, 1, dim))
    # One rounding a key, and as in attend() 16 for joining and dividing.
    off = dec.U * (keys + 16) * np.broadcast_to(np.abs(values).mean(axis=0), want.shape)
    base.within(base.run(runtime, spec, x)["out"], want[None], off[None])


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("every", [1, 4])
def test_values_below_bf16s_least(runtime, kernel, every):
    # Values of 2^-138, in all dims or in every fourth: bf16's smallest number is 2^-133. Queries of zeros weigh all
    # keys 1, and sums of subnormal numbers are exact, so an output is off by the division and its own rounding.
    spec = base.cross_spec(*KERNELS[kernel])
    rng = np.random.default_rng(52)
    b, n = spec["batch"], spec["keys"]
    lengths = [n, n - 1, 1] + [n] * (b - 3)
    x = base.cross_inputs(rng, spec, lengths)
    x["q"][:] = 0
    x["v"][..., ::every] = (1 + np.abs(x["v"][..., ::every])) * np.float32(2.0 ** -138)
    got = base.run(runtime, spec, x)["out"].reshape(x["q"].shape)
    group = spec["heads"] // spec["kv_heads"]
    for i, length in enumerate(lengths):
        values = np.repeat(x["v"][i, :, :length].astype(np.float64), group, axis=0)
        want = np.broadcast_to(values.mean(axis=1, keepdims=True), got[i].shape)[..., ::every]
        base.within(got[i][..., ::every], want, 4 * dec.U * want + 2.0 ** -149)


@pytest.mark.parametrize("nodes,dim", [(7, 64), (20, 64), (20, 96), (40, 128), (100, 80), (33, 50)])
def test_drafted_values_below_bf16s_least(runtime, nodes, dim):
    # A chain over an empty cache: node n's output is the mean of the values up to it.
    rng = np.random.default_rng(53)
    spec = base.tree_spec(2, 2, 2, nodes, 64, dim)
    x = base.tree_inputs(rng, spec, [0, 0], [[n - 1 for n in range(nodes)]] * 2)
    x["q"][:] = 0
    x["v_draft"] = ((1 + np.abs(x["v_draft"])) * np.float32(2.0 ** -138)).astype(np.float32)
    want = np.cumsum(x["v_draft"].astype(np.float64), axis=2) / np.arange(1, nodes + 1)[:, None]
    base.within(base.run(runtime, spec, x)["out"], want, 4 * dec.U * want + 2.0 ** -149)


@pytest.mark.parametrize("kernel", KERNELS)
def test_values_of_zero(runtime, kernel):
    # Not to be taken for values that the parts lost: plain zeros, some dims of them or all.
    spec = base.cross_spec(*KERNELS[kernel])
    rng = np.random.default_rng(54)
    lengths = [spec["keys"]] * spec["batch"]
    x = base.cross_inputs(rng, spec, lengths)
    x["v"][..., 1::2] = 0
    got = base.run(runtime, spec, x)["out"].reshape(x["q"].shape)
    part = dict(spec, batch=2)
    want, off = dec.cross(part, x["q"][:2], x["k"][:2], x["v"][:2], lengths)
    base.within(got[:2], want, off)
    assert (got[..., 1::2] == 0).all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("scale", [2.0 ** 90, 2.0 ** 108])
def test_values_whose_scaled_sums_overflow(runtime, kernel, scale):
    # V's parts carry values times 2^24: these, or sums of them, pass FP32's range there, but not as they are.
    spec = base.cross_spec(*KERNELS[kernel])
    rng = np.random.default_rng(55)
    lengths = [spec["keys"]] * spec["batch"]
    x = base.cross_inputs(rng, spec, lengths)
    x["v"] = (x["v"] * np.float32(scale)).astype(np.float32)
    want, off = dec.cross(dict(spec, batch=3), x["q"][:3], x["k"][:3], x["v"][:3], lengths)
    got = base.run(runtime, spec, x)["out"].reshape(x["q"].shape)
    base.within(got[:3], want, off)
    assert np.isfinite(got).all()


@pytest.mark.parametrize("nodes,dim", [(5, 64), (20, 128), (40, 64), (30, 90), (70, 128), (130, 50)])
def test_large_drafted_values_stay_with_those_who_see_them(runtime, nodes, dim):
    # Two branches; the second's values and keys are 2^108 and its queries as small, the first's are ordinary.
    rng = np.random.default_rng(56)
    half = nodes // 2
    spec = base.tree_spec(1, 2, 1, nodes, 90, dim)
    x = base.tree_inputs(rng, spec, [77], [[n - 1 for n in range(half)] + [-1] + list(range(half, nodes - 1))])
    for name, scale in (("v_draft", 2.0 ** 108), ("k_draft", 2.0 ** 60), ("q", 2.0 ** -60)):
        x[name][:, :, half:] *= np.float32(scale)
    want, off = base.tree_want(spec, x)
    base.within(base.run(runtime, spec, x)["out"], want, off)
