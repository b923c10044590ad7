"""Attention of a decoder's step where a run of the ragged kernels has many tiles: sums carried from tile to tile, units
cut in their midst and joined, units that a run has to itself, cuts moved to a unit's end. Every kernel, against 64 bits
(decoder_units.py)."""
import numpy as np
import pytest

import jade_hip
import test_gpu_decoder as base
from decoder_units import Cuts, check

pytestmark = pytest.mark.gpu


def rising(rng, spec, x):
    """Scores of the cached keys that rise, fall or do neither along the keys, by 12 powers of two: the running maximum
    moves in some tiles and not in others."""
    names = ("q", "k_cache") if "nodes" in spec else ("q", "k")
    most = spec["capacity"] if "nodes" in spec else spec["keys"]
    ramp = np.linspace(-1, 1, most, dtype=np.float32)
    q, k = (base.dec.by_token(x[n], spec["token_major"]) for n in names)  # [batch, rows, heads, dim]
    q[..., 0] = 2
    for b in range(spec["batch"]):
        k[b, :, :, 0] = (b % 3 - 1) * np.float32(12 * np.log(2) / 4 * np.sqrt(spec["dim"])) * ramp[:, None]
    return x


# (batch, heads, kv_heads, queries, keys, dim): few long units, cut in their midst. `keys` is all of the first sequence.
LONG = {"attention_ragged_d64": (3, 24, 12, 5, 6000, 39), "attention_ragged_d128": (3, 24, 12, 8, 6000, 80),
        "attention_ragged_parts_d64_r32": (3, 32, 16, 12, 6000, 32), "attention_ragged_parts_d64_r64": (4, 24, 12, 20, 5000, 31),
        "attention_ragged_parts_d96_r32": (3, 32, 16, 9, 5000, 80), "attention_ragged_parts_d96_r64": (3, 16, 16, 50, 5000, 95),
        "attention_ragged_parts_d128_r32": (3, 32, 16, 10, 5000, 128), "attention_ragged_parts_d128_r64": (3, 24, 12, 27, 5000, 99)}


@pytest.mark.parametrize("kernel", LONG)
@pytest.mark.parametrize("token_major", [False, True])
def test_long_units_cut_in_their_midst(runtime, kernel, token_major):
    spec = base.cross_spec(*LONG[kernel], token_major)
    keys = spec["keys"]
    lengths = [keys, 0, keys * 2 // 3 + 1, keys // 2 + 7][:spec["batch"]]
    cuts = Cuts(spec, lengths)
    assert cuts.kernel == kernel and cuts.chunk >= 3 and cuts.inside > 100 and cuts.longest >= 3
    rng = np.random.default_rng(70)
    x = rising(rng, spec, base.cross_inputs(rng, spec, lengths))
    got = base.run(runtime, spec, x, repeats=2)["out"]
    check(spec, x, got, [(b, kv) for b in range(spec["batch"]) for kv in range(0, spec["kv_heads"], 3)])


# Very many short units: a run has four or more of them, and its cuts go to their ends.
SHORT = {"attention_ragged_d64": (440, 10, 5, 7, 230, 12), "attention_ragged_d128": (440, 10, 5, 4, 230, 67),
         "attention_ragged_parts_d64_r32": (720, 8, 4, 12, 330, 13), "attention_ragged_parts_d64_r64": (95, 10, 5, 95, 330, 63),
         "attention_ragged_parts_d96_r32": (360, 8, 4, 11, 330, 66), "attention_ragged_parts_d96_r64": (95, 5, 5, 190, 330, 91),
         "attention_ragged_parts_d128_r32": (360, 8, 4, 10, 330, 98), "attention_ragged_parts_d128_r64": (95, 10, 5, 95, 330, 127)}


def short_lengths(rng, batch, most):
    """Mostly of 60% of the keys or more, some empty, of one key or of any number."""
    kind = rng.random(batch)
    return [int(n) for n in np.where(kind < 0.1, 0, np.where(kind < 0.15, 1, np.where(
        kind < 0.3, rng.integers(0, most + 1, batch), rng.integers(most * 6 // 10, most + 1, batch))))]


@pytest.mark.parametrize("kernel", SHORT)
def test_short_units_in_runs_of_many(runtime, kernel):
    spec = base.cross_spec(*SHORT[kernel])
    rng = np.random.default_rng(71)
    lengths = short_lengths(rng, spec["batch"], spec["keys"])
    cuts = Cuts(spec, lengths)
    assert cuts.kernel == kernel and cuts.chunk >= 12 and cuts.moved > 50 and cuts.whole > 500
    x = rising(rng, spec, base.cross_inputs(rng, spec, lengths))
    got = base.run(runtime, spec, x, repeats=2)["out"]
    assert (got.reshape(x["q"].shape)[np.array(lengths) == 0] == 0).all()
    units = [(b, kv) for b in range(spec["batch"]) for kv in range(spec["kv_heads"])]
    check(spec, x, got, units[::7] + units[-3:])


@pytest.mark.parametrize("kernel,shape", [("attention_ragged_d64", (420, 10, 5, 3, 900, 10)),
                                          ("attention_ragged_parts_d64_r32", (720, 8, 4, 12, 900, 7)),
                                          ("attention_ragged_parts_d64_r64", (95, 10, 5, 95, 1500, 14))])
def test_long_sequences_among_short_ones(runtime, kernel, shape):
    # Cuts inside the units of the long ones, cuts at unit ends among the short ones.
    spec = base.cross_spec(*shape)
    rng = np.random.default_rng(75)
    lengths = np.array(short_lengths(rng, spec["batch"], 200))
    lengths[5::31] = spec["keys"] - 3
    cuts = Cuts(spec, lengths)
    assert cuts.kernel == kernel and cuts.moved > 20 and cuts.inside > 20 and cuts.whole > 200
    x = rising(rng, spec, base.cross_inputs(rng, spec, lengths))
    got = base.run(runtime, spec, x)["out"]
    units = [(b, kv) for b in range(spec["batch"]) for kv in range(spec["kv_heads"])]
    check(spec, x, got, sorted(set(units[::9] + [u for u in units if lengths[u[0]] > 200])))


# (batch, heads, kv_heads, nodes, capacity, dim)
TREES = {"attention_ragged_d64": [(2, 24, 12, 5, 9000, 40), (440, 10, 5, 3, 170, 30)],
         "attention_ragged_d128": [(2, 24, 12, 8, 9000, 128), (440, 10, 5, 4, 170, 72)],
         "attention_ragged_parts_d64_r32": [(2, 32, 16, 15, 7000, 64), (640, 8, 4, 9, 250, 21)],
         "attention_ragged_parts_d64_r64": [(2, 32, 16, 130, 2000, 40), (125, 10, 5, 70, 250, 14)],
         "attention_ragged_parts_d96_r32": [(2, 32, 16, 13, 5000, 90), (320, 8, 4, 11, 250, 66)],
         "attention_ragged_parts_d96_r64": [(2, 32, 16, 40, 3000, 96), (125, 10, 5, 70, 250, 70)],
         "attention_ragged_parts_d128_r32": [(2, 32, 16, 10, 5000, 100), (320, 8, 4, 14, 250, 110)],
         "attention_ragged_parts_d128_r64": [(2, 32, 16, 150, 1500, 128), (130, 10, 5, 40, 250, 97)]}


@pytest.mark.parametrize("kernel", TREES)
@pytest.mark.parametrize("many", [False, True])
def test_trees_behind_many_tiles(runtime, kernel, many):
    spec = base.tree_spec(*TREES[kernel][many], token_major=not many)
    rng = np.random.default_rng(72)
    most = spec["capacity"]
    lengths = short_lengths(rng, spec["batch"], most) if many else [most, most // 3]
    cuts = Cuts(spec, lengths)
    assert cuts.kernel == kernel and (cuts.moved > 20 and cuts.whole > 200 if many else cuts.inside > 100 and cuts.longest >= 3)
    x = rising(rng, spec, base.tree_inputs(rng, spec, lengths))
    got = base.run(runtime, spec, x, repeats=2)["out"]
    units = [(b, kv) for b in range(spec["batch"]) for kv in range(spec["kv_heads"])]
    check(spec, x, got, units[::11] + units[-2:] if many else units[::3])


@pytest.mark.parametrize("kernel", base.KERNELS)
@pytest.mark.parametrize("token_major", [False, True])
def test_every_sequence_of_every_kernel(runtime, kernel, token_major):
    # As test_every_kernel_of_attention_cross, whose lengths these are, but each sequence and head against 64 bits.
    spec = base.cross_spec(*base.KERNELS[kernel], token_major)
    rng = np.random.default_rng(73)
    lengths = [spec["keys"], 0, 1, 32, 33][:spec["batch"]] + [int(n) for n in rng.integers(0, spec["keys"] + 1, spec["batch"])]
    x = base.cross_inputs(rng, spec, lengths[:spec["batch"]])
    got = base.run(runtime, spec, x)["out"]
    check(spec, x, got, [(b, kv) for b in range(spec["batch"]) for kv in range(spec["kv_heads"])])


@pytest.mark.parametrize("queries,dim,kernel", [(1, 9, "attention_ragged_d64"), (20, 9, "attention_ragged_parts_d64_r32"),
                                                (40, 13, "attention_ragged_parts_d64_r64"), (40, 101, "attention_ragged_parts_d128_r64")])
def test_thousands_of_sequences_on_the_ragged_kernels(runtime, queries, dim, kernel):
    batch = 3000
    rng = np.random.default_rng(74)
    spec = base.cross_spec(batch, 1, 1, queries, 150, dim)
    assert jade_hip.spec_describe(spec)["launch"]["kernel"] == kernel
    lengths = np.where(rng.random(batch) < 0.7, 0, rng.integers(0, 151, batch))
    x = base.cross_inputs(rng, spec, lengths)
    got = base.run(runtime, spec, x)["out"]
    assert (got.reshape(x["q"].shape)[lengths == 0] == 0).all()
    check(spec, x, got, [(b, 0) for b in np.flatnonzero(lengths)[::3]] + [(0, 0), (63, 0), (64, 0), (65, 0), (2999, 0)])
