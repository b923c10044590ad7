"""decoder_units.py agrees with decoder_oracle.py and tells a wrong tile from a right one, on the CPU."""
import numpy as np
import pytest

import decoder_oracle as dec
import decoder_units as units
import test_gpu_decoder as base
from test_gpu_decoder_runs import LONG, rising


@pytest.mark.parametrize("token_major", [False, True])
def test_units_are_the_oracles_rows(token_major):
    rng = np.random.default_rng(1)
    cross = base.cross_spec(2, 6, 2, 5, 70, 20, token_major)
    x = base.cross_inputs(rng, cross, [70, 0])
    tree = base.tree_spec(2, 6, 2, 9, 50, 20, token_major)
    y = base.tree_inputs(rng, tree, [50, 0], [[n - 1 for n in range(8)] + [-2], [-1, 0, 0, 5, -2, 2, 1, 6, 3]])
    for spec, z, (want, off) in ((cross, x, dec.cross(cross, x["q"], x["k"], x["v"], x["lengths"])),
                                 (tree, y, base.tree_want(tree, y))):
        want, off = dec.by_token(want, token_major), dec.by_token(off, token_major)
        for b in range(2):
            for kv in range(2):
                got, bound = units.unit(spec, z, b, kv)
                mine = want[b][:, 3 * kv:3 * kv + 3].swapaxes(0, 1)
                assert np.abs(got - mine).max() < 1e-13
                assert np.allclose(bound, off[b][:, 3 * kv:3 * kv + 3].swapaxes(0, 1), rtol=1e-9, atol=0)


@pytest.mark.parametrize("kernel", LONG)
def test_a_lost_tile_is_noticed(kernel):
    spec = dict(base.cross_spec(*LONG[kernel]), kv_heads=2, heads=2 * LONG[kernel][1] // LONG[kernel][2], batch=3)
    rng = np.random.default_rng(2)
    keys, tile = spec["keys"], 128 if "parts" in kernel else 64
    x = rising(rng, spec, base.cross_inputs(rng, spec, [keys] * 3))
    for b in range(3):  # scores that fall, level ones and scores that rise: the tile with the largest, or any
        want, off = units.unit(spec, x, b, 0)
        q = np.concatenate(x["q"][b, :spec["heads"] // 2]).astype(np.float64)
        lost = np.s_[:tile] if b == 0 else np.s_[keys // 2:keys // 2 + tile] if b == 1 else np.s_[-tile:]
        k, v = (np.delete(x[n][b, 0].astype(np.float64), lost, axis=0) for n in "kv")
        wrong = units.attend(q, k, v)[0].reshape(want.shape)
        assert (np.abs(wrong - want) > off).mean() > 0.5


def test_cuts():
    # 4 heads of 3 tiles in 512 runs: a tile each; 2048 heads of 3 tiles: 12 a run, whole units all.
    spec = base.cross_spec(1, 4, 4, 1, 130, 16)
    few = units.Cuts(spec, [130])
    assert (few.kernel, few.chunk, few.moved, few.inside, few.whole, few.longest) == ("attention_ragged_d64", 1, 0, 8, 0, 1)
    many = units.Cuts(dict(spec, batch=512), [130] * 512)
    assert (many.chunk, many.moved, many.inside, many.whole, many.longest) == (12, 0, 0, 2048, 3)
    odd = units.Cuts(dict(spec, batch=600), [130] * 600)
    assert odd.chunk == 15 and odd.inside == 0
    odd = units.Cuts(dict(spec, batch=560), [130] * 560)
    assert odd.chunk == 14 and odd.moved > 300 and odd.inside == 0 and odd.whole == 2240
