"""The operators of a decoder's step (rotary, qk_norm_rotary, attention_tree, cache_append, attention_cross) on the
GPU against 64-bit restatements (decoder_oracle.py), with its derived bounds."""
import numpy as np
import pytest

import decoder_oracle as dec
import jade_hip

pytestmark = pytest.mark.gpu


def run(runtime, spec, inputs, repeats=1):
    """One dispatch; `inputs` by binding name. Returns the written bindings by name."""
    kernel = runtime.compile(spec)
    bufs = {}
    for b in kernel.bindings:
        bufs[b["name"]] = runtime.resident(inputs[b["name"]]) if b["name"] in inputs else runtime.alloc(b["elements"])
        assert len(bufs[b["name"]]) == b["elements"]
    runtime.execute([(kernel, [bufs[b["name"]] for b in kernel.bindings])], repeats)
    got = {b["name"]: runtime.download(bufs[b["name"]]) for b in kernel.bindings if b["write"]}
    for b in bufs.values():
        b.free()
    kernel.release()
    return got


def within(got, want, off):
    got = got.reshape(want.shape).astype(np.float64)
    assert np.isfinite(got).all()
    over = np.abs(got - want) - off
    assert over.max() <= 0, (np.unravel_index(over.argmax(), over.shape), over.max(), off.max())


def normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def shape_of(token_major, batch, heads, rows, dim):
    return (batch, rows, heads, dim) if token_major else (batch, heads, rows, dim)


# ---- rotary -----------------------------------------------------------------------------------------------

SCALED = {"factor": 8.0, "context": 8192.0, "low_turns": 1.0, "high_turns": 4.0, "magnitude": 1.25}


def rotary_spec(batch, seq, heads, dim, part, interleaved=False, inverse=False, token_major=True, out_token_major=False,
                **more):
    return {"op": "rotary", "batch": batch, "seq": seq, "heads": heads, "dim": dim, "rotary_dim": part,
            "interleaved": interleaved, "inverse": inverse, "token_major": token_major,
            "out_token_major": out_token_major, "base": 10000.0, **more}


# Whole float4s (each lane count), parts of the head, odd and scalar heads, more heads than a wave takes.
@pytest.mark.parametrize("batch,seq,heads,dim,part", [
    (2, 3, 5, 128, 128), (1, 1, 1, 2, 2), (3, 7, 9, 80, 32), (2, 5, 3, 80, 20), (1, 9, 40, 64, 64), (1, 4, 2, 512, 512),
    (1, 3, 7, 256, 64), (2, 2, 3, 10, 4), (1, 65, 2, 33, 16), (2, 300, 33, 32, 16), (1, 2, 3, 510, 506), (1, 3, 2, 8, 8),
    (4, 600, 6, 96, 96)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", [(True, False), (False, False), (False, True), (True, True)])
def test_rotary(runtime, batch, seq, heads, dim, part, interleaved, layout):
    rng = np.random.default_rng(dim * seq + part)
    spec = rotary_spec(batch, seq, heads, dim, part, interleaved, token_major=layout[0], out_token_major=layout[1])
    x = normal(rng, *shape_of(layout[0], batch, heads, seq, dim))
    positions = (rng.integers(0, 100000, (batch, 1)) + np.arange(seq)).astype(np.float32)
    got = run(runtime, spec, {"x": x, "positions": positions})["out"]
    want, size = dec.rotate(spec, dec.by_token(x.astype(np.float64), layout[0]), positions)
    want, size = dec.by_token(want, layout[1]), dec.by_token(size, layout[1])
    within(got, want, dec.ROTARY_BOUND * size)  # copied dims are equal


@pytest.mark.parametrize("more", [{"factor": 4.0}, SCALED])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary_scaled_far_and_odd_positions(runtime, more, inverse):
    rng = np.random.default_rng(5)
    positions = np.array([[0.0, 0.5, -3.25, 2.0 ** 24 - 1, 1e6, 123457.0, 1e9, -1e7]], np.float32)
    spec = rotary_spec(1, 8, 4, 128, 128, inverse=inverse, **more)
    x = normal(rng, 1, 8, 4, 128)
    got = run(runtime, spec, {"x": x, "positions": positions})["out"]
    want, size = dec.rotate(spec, x.astype(np.float64), positions, inverse)
    # The oracle's own angles carry 2^-53 of a 10^9 radian angle: 1.1e-7.
    far = np.abs(positions.reshape(1, 8, 1, 1)) * 2.0 ** -52
    within(got, dec.by_token(want, False), dec.by_token((dec.ROTARY_BOUND + far) * size, False))


def test_rotary_inverse_is_the_gradient_and_undoes(runtime):
    rng = np.random.default_rng(7)
    spec = rotary_spec(2, 33, 3, 80, 48, out_token_major=True)
    x, g = normal(rng, 2, 33, 3, 80), normal(rng, 2, 33, 3, 80)
    positions = rng.integers(0, 5000, (2, 33)).astype(np.float32)
    y = run(runtime, spec, {"x": x, "positions": positions})["out"].reshape(x.shape)
    back = dict(spec, inverse=True)
    dx = run(runtime, back, {"x": g, "positions": positions})["out"].reshape(x.shape)
    # <R x, g> = <x, R^T g>, element by element of x's direction: differences of a linear map.
    for _ in range(8):
        at = tuple(rng.integers(0, n) for n in x.shape)
        moved = x.copy()
        moved[at] += 1.0
        dy = run(runtime, spec, {"x": moved, "positions": positions})["out"].reshape(x.shape).astype(np.float64) - y
        # Two outputs change; each y is off by ROTARY_BOUND (|a| + |b| <= 12) on both sides of the difference.
        assert abs((dy * g).sum() - dx[at] * (moved[at].astype(np.float64) - x[at])) <= 2 * 2 * 12 * 5 * dec.ROTARY_BOUND
    again = run(runtime, back, {"x": y, "positions": positions})["out"].reshape(x.shape)
    assert np.abs(again - x).max() <= 2 * 2 * 12 * dec.ROTARY_BOUND


def test_rotary_position_that_is_not_finite_spoils_its_own_token_only(runtime):
    rng = np.random.default_rng(8)
    spec = rotary_spec(1, 3, 2, 16, 8, out_token_major=True)
    x = normal(rng, 1, 3, 2, 16)
    got = run(runtime, spec, {"x": x, "positions": np.array([1.0, np.nan, np.inf])})["out"].reshape(x.shape)
    assert np.isnan(got[0, 1:, :, :8]).all()
    assert (got[..., 8:] == x[..., 8:]).all() and np.isfinite(got[0, 0]).all()


# ---- qk_norm_rotary ---------------------------------------------------------------------------------------

def norm_spec(batch, seq, heads, kv_heads, dim, part, interleaved=False, token_major=True, out_token_major=False, **more):
    return {"op": "qk_norm_rotary", "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary_dim": part, "interleaved": interleaved, "token_major": token_major,
            "out_token_major": out_token_major, "epsilon": 1e-6, "base": 10000.0, **more}


@pytest.mark.parametrize("batch,seq,heads,kv_heads,dim,part", [
    (2, 3, 8, 2, 128, 128), (16, 1, 32, 8, 128, 64), (1, 5, 3, 3, 80, 80), (1, 7, 5, 1, 37, 20), (2, 2, 1, 3, 64, 32),
    (1, 2, 2, 1, 512, 256), (1, 700, 12, 4, 96, 96), (3, 3, 2, 2, 3, 2)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", [(True, False), (False, True)])
def test_qk_norm_rotary(runtime, batch, seq, heads, kv_heads, dim, part, interleaved, layout):
    rng = np.random.default_rng(dim + seq)
    spec = norm_spec(batch, seq, heads, kv_heads, dim, part, interleaved, *layout, **SCALED)
    x = {"q": 3 * normal(rng, *shape_of(layout[0], batch, heads, seq, dim)),
         "k": 3 * normal(rng, *shape_of(layout[0], batch, kv_heads, seq, dim)),
         "q_weight": 1 + 0.3 * normal(rng, dim), "k_weight": 1 + 0.3 * normal(rng, dim),
         "positions": rng.integers(0, 10000, (batch, seq)).astype(np.float32)}
    got = run(runtime, spec, x)
    for name in "qk":
        y = dec.norm(dec.by_token(x[name].astype(np.float64), layout[0]), x[name + "_weight"].astype(np.float64), 1e-6)
        want, size = dec.rotate(spec, y, x["positions"])
        off = np.where(size > 0, (dec.NORM_BOUND + dec.ROTARY_BOUND) * size, dec.NORM_BOUND * np.abs(y))
        within(got[name + "_out"], dec.by_token(want, layout[1]), dec.by_token(off, layout[1]))


def test_qk_norm_rotary_zero_and_tiny_heads(runtime):
    spec = norm_spec(1, 2, 2, 1, 64, 64, out_token_major=True)
    x = {"q": np.zeros((1, 2, 2, 64), np.float32), "k": np.full((1, 2, 1, 64), 1e-20, np.float32),
         "q_weight": np.ones(64), "k_weight": np.ones(64), "positions": np.array([[3.0, 4.0]])}
    got = run(runtime, spec, x)
    assert (got["q_out"] == 0).all()
    assert np.abs(got["k_out"]).max() < 1e-16  # the epsilon holds the norm


# ---- attention over an encoder's states ------------------------------------------------------------------

def cross_spec(batch, heads, kv_heads, queries, keys, dim, token_major=False):
    return {"op": "attention_cross", "batch": batch, "heads": heads, "kv_heads": kv_heads, "queries": queries,
            "keys": keys, "dim": dim, "token_major": token_major}


def cross_inputs(rng, spec, lengths):
    tm = spec["token_major"]
    b, d = spec["batch"], spec["dim"]
    return {"q": normal(rng, *shape_of(tm, b, spec["heads"], spec["queries"], d)),
            "k": normal(rng, *shape_of(tm, b, spec["kv_heads"], spec["keys"], d)),
            "v": normal(rng, *shape_of(tm, b, spec["kv_heads"], spec["keys"], d)),
            "lengths": np.array(lengths, np.float32)}


@pytest.mark.parametrize("batch,heads,kv_heads,queries,keys,dim", [
    (1, 1, 1, 1, 1, 1), (2, 4, 2, 1, 64, 64), (3, 6, 2, 5, 65, 80), (2, 2, 2, 16, 63, 128), (2, 8, 1, 2, 200, 128),
    (1, 8, 2, 4, 513, 96), (2, 4, 4, 33, 70, 64), (1, 3, 1, 11, 130, 37), (2, 2, 1, 50, 129, 128), (1, 2, 2, 7, 1531, 80),
    (1, 1, 1, 3, 100, 3), (2, 5, 5, 1, 300, 126), (1, 2, 1, 150, 90, 40)])
@pytest.mark.parametrize("token_major", [False, True])
def test_attention_cross(runtime, batch, heads, kv_heads, queries, keys, dim, token_major):
    rng = np.random.default_rng(keys + dim)
    spec = cross_spec(batch, heads, kv_heads, queries, keys, dim, token_major)
    lengths = [keys, max(1, keys - 17), keys // 2][:batch]
    x = cross_inputs(rng, spec, lengths)
    within(run(runtime, spec, x)["out"], *dec.cross(spec, x["q"], x["k"], x["v"], lengths))


@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("queries,dim", [(1, 64), (20, 128), (3, 30)])
def test_attention_cross_odd_lengths_and_what_lies_past_them(runtime, queries, dim, token_major):
    # Lengths zero, one, fractions, NaN, negative and past the end; keys and values past them are NaN and infinite.
    rng = np.random.default_rng(3)
    lengths = [0.0, 1.0, 63.0, 64.9, 65.0, np.nan, -4.0, 1e30, np.inf, 0.5]
    spec = cross_spec(len(lengths), 4, 2, queries, 130, dim, token_major)
    x = cross_inputs(rng, spec, lengths)
    for b, length in enumerate(lengths):
        n = dec.length_of(length, 130)
        dec.by_token(x["k"], token_major)[b, n:] = np.nan
        dec.by_token(x["v"], token_major)[b, n:] = np.inf
    clean = {n: np.where(np.isfinite(x[n]), x[n], 0) for n in ("k", "v")}
    want, off = dec.cross(spec, x["q"], clean["k"], clean["v"], lengths)
    got = run(runtime, spec, x)["out"]
    within(got, want, off)
    zero = dec.by_token(got.reshape(want.shape), token_major)[[0, 5, 6, 9]]
    assert (zero == 0).all()


def test_attention_cross_all_sequences_empty(runtime):
    rng = np.random.default_rng(4)
    spec = cross_spec(3, 2, 1, 2, 40, 16)
    x = cross_inputs(rng, spec, [0, 0, 0])
    kernel = runtime.compile(spec)
    bufs = [runtime.resident(x[n]) for n in ("q", "k", "v", "lengths")] + [runtime.resident(np.full(x["q"].size, 7.0))]
    runtime.execute([(kernel, bufs)], 1)
    assert (runtime.download(bufs[4]) == 0).all()


def test_attention_cross_many_sequences(runtime):
    # More sequences than a wave scans at once, most of them empty.
    rng = np.random.default_rng(6)
    lengths = [int(n) if rng.random() < 0.4 else 0 for n in rng.integers(1, 300, 200)]
    spec = cross_spec(200, 2, 2, 1, 300, 32)
    x = cross_inputs(rng, spec, lengths)
    within(run(runtime, spec, x)["out"], *dec.cross(spec, x["q"], x["k"], x["v"], lengths))


@pytest.mark.parametrize("scale", [30.0, 1e-3, 1e18])
def test_attention_cross_peaked_flat_and_huge(runtime, scale):
    rng = np.random.default_rng(9)
    spec = cross_spec(1, 2, 1, 9, 200, 64)
    x = cross_inputs(rng, spec, [200])
    x["q"] *= np.float32(scale)
    if scale > 1e9:  # scores of 1e18: one key takes all, and which one is beyond doubt
        want, _ = dec.cross(spec, x["q"], x["k"], x["v"], [200])
        off = 8 * dec.U * np.abs(want)
    else:
        want, off = dec.cross(spec, x["q"], x["k"], x["v"], [200])
    within(run(runtime, spec, x)["out"], want, off)


def test_attention_cross_keeps_non_finite_values_in_their_rows(runtime):
    rng = np.random.default_rng(10)
    spec = cross_spec(2, 1, 1, 3, 40, 16)
    x = cross_inputs(rng, spec, [40, 40])
    x["q"][0, 0, 1, 3] = np.nan
    x["v"][1, 0, 5, 2] = np.inf
    got = run(runtime, spec, x)["out"].reshape(x["q"].shape)
    assert np.isnan(got[0, 0, 1]).all() and np.isfinite(got[0, 0, [0, 2]]).all()
    assert np.isposinf(got[1, 0, :, 2]).all() and np.isfinite(np.delete(got[1, 0], 2, axis=1)).all()


# ---- the tree over a cache ---------------------------------------------------------------------------------

def tree_spec(batch, heads, kv_heads, nodes, capacity, dim, token_major=False):
    return {"op": "attention_tree", "batch": batch, "heads": heads, "kv_heads": kv_heads, "nodes": nodes,
            "capacity": capacity, "dim": dim, "token_major": token_major}


def tree_inputs(rng, spec, lengths, parents=None):
    tm, b, kv, d = spec["token_major"], spec["batch"], spec["kv_heads"], spec["dim"]
    if parents is None:
        parents = [[rng.integers(max(-1, n - 6), n) for n in range(spec["nodes"])] for _ in range(b)]
    cache, draft = shape_of(tm, b, kv, spec["capacity"], d), shape_of(tm, b, kv, spec["nodes"], d)
    return {"q": normal(rng, *shape_of(tm, b, spec["heads"], spec["nodes"], d)), "k_cache": normal(rng, *cache),
            "v_cache": normal(rng, *cache), "lengths": np.array(lengths, np.float32), "k_draft": normal(rng, *draft),
            "v_draft": normal(rng, *draft), "parents": np.array(parents, np.float32)}


def tree_want(spec, x):
    return dec.tree(spec, *(x[n] for n in ("q", "k_cache", "v_cache", "lengths", "k_draft", "v_draft", "parents")))


@pytest.mark.parametrize("batch,heads,kv_heads,nodes,capacity,dim", [
    (1, 1, 1, 1, 1, 4), (2, 8, 8, 1, 128, 64), (3, 8, 2, 5, 200, 128), (2, 4, 1, 13, 65, 80), (1, 2, 2, 64, 64, 64),
    (1, 4, 2, 65, 100, 128), (2, 2, 1, 37, 33, 33), (1, 1, 1, 256, 40, 32), (1, 8, 1, 17, 700, 96), (2, 3, 3, 129, 70, 10)])
@pytest.mark.parametrize("token_major", [False, True])
def test_attention_tree(runtime, batch, heads, kv_heads, nodes, capacity, dim, token_major):
    rng = np.random.default_rng(nodes + capacity)
    spec = tree_spec(batch, heads, kv_heads, nodes, capacity, dim, token_major)
    x = tree_inputs(rng, spec, [capacity, 0, capacity // 2][:batch])
    within(run(runtime, spec, x)["out"], *tree_want(spec, x))


@pytest.mark.parametrize("kind", ["chain", "star", "all absent", "holes"])
@pytest.mark.parametrize("nodes", [7, 100])
def test_attention_tree_shapes_of_trees(runtime, kind, nodes):
    rng = np.random.default_rng(nodes)
    parents = {"chain": [n - 1 for n in range(nodes)], "star": [-1] * nodes, "all absent": [-2] * nodes,
               # Forward, own, fractional, negative and non-finite parents hold no node; nobody sees those slots.
               "holes": [[-1, 1, 0, 0.5, -3, np.nan, np.inf][n % 7] if n < 14 else n - 2 for n in range(nodes)]}[kind]
    spec = tree_spec(2, 4, 2, nodes, 90, 64)
    x = tree_inputs(rng, spec, [90, 0], [parents, parents])
    got = run(runtime, spec, x)["out"]
    want, off = tree_want(spec, x)
    within(got, want, off)
    absent = [n for n, s in enumerate(dec.ancestors(parents)) if not s]
    assert (got.reshape(want.shape)[:, :, absent] == 0).all()


@pytest.mark.parametrize("nodes,dim", [(5, 64), (20, 128), (70, 36), (9, 30), (40, 80), (20, 91)])
def test_attention_tree_non_finite_values_stay_in_their_branch(runtime, nodes, dim):
    # Two chains; the first's last node is infinite and NaN in k, v and q, absent slots and the cache past its
    # length hold NaN. The second chain, and the first's earlier nodes, do not notice.
    rng = np.random.default_rng(nodes)
    half = nodes // 2
    parents = [n - 1 for n in range(half)] + [-1] + [n - 1 for n in range(half + 1, nodes - 1)] + [-2]
    spec = tree_spec(1, 2, 1, nodes, 100, dim)
    x = tree_inputs(rng, spec, [70], [parents])
    want, off = tree_want(spec, x)
    x["k_cache"][:, :, 70:] = np.nan
    x["v_cache"][:, :, 70:] = -np.inf
    for name in ("k_draft", "v_draft", "q"):
        x[name][:, :, -1] = np.nan
        x[name][:, :, half - 1] = np.inf
    x["v_draft"][:, :, half - 1, 1] = np.nan
    got = run(runtime, spec, x)["out"].reshape(want.shape)
    others = [n for n in range(nodes) if n != half - 1]
    within(got[:, :, others], want[:, :, others], off[:, :, others])
    assert not np.isfinite(got[:, :, half - 1]).any()


def test_attention_tree_infinite_draft_value_reaches_those_who_see_it(runtime):
    rng = np.random.default_rng(12)
    spec = tree_spec(1, 1, 1, 4, 70, 64)
    x = tree_inputs(rng, spec, [70], [[-1, 0, 0, 1]])
    x["v_draft"][0, 0, 1, 5] = np.inf
    got = run(runtime, spec, x)["out"].reshape(4, 64)
    assert np.isposinf(got[[1, 3], 5]).all()
    assert np.isfinite(got[[0, 2]]).all() and np.isfinite(np.delete(got, 5, axis=1)).all()


def test_attention_tree_long_cache_is_cut_and_joined(runtime):
    rng = np.random.default_rng(13)
    spec = tree_spec(2, 2, 1, 3, 40000, 32)
    x = tree_inputs(rng, spec, [40000, 77])
    within(run(runtime, spec, x, repeats=3)["out"], *tree_want(spec, x))


def test_attention_results_do_not_change_from_run_to_run(runtime):
    rng = np.random.default_rng(14)
    for spec, x in ((tree_spec(3, 8, 2, 9, 3001, 64), None), (cross_spec(2, 4, 2, 40, 900, 128), None)):
        x = tree_inputs(rng, spec, [3001, 5, 1000]) if "nodes" in spec else cross_inputs(rng, spec, [900, 333])
        first = run(runtime, spec, x)["out"]
        for repeats in (1, 3):
            assert (run(runtime, spec, x, repeats)["out"] == first).all()


def test_attention_tree_cache_past_four_gib(runtime):
    # A cache of 2^31 elements a tensor (8 GiB), one sequence: rows past 2^32 bytes are appended and read back.
    kv, dim, capacity = 8, 128, 1 << 21
    put = {"op": "cache_append", "batch": 1, "kv_heads": kv, "rows": 70, "picks": 70, "capacity": capacity, "dim": dim,
           "token_major": True}
    spec = tree_spec(1, kv, kv, 1, capacity, dim, True)
    rng = np.random.default_rng(15)
    n = capacity - 70
    k, v = normal(rng, 1, 70, kv, dim), normal(rng, 1, 70, kv, dim)
    q, kd, vd = (normal(rng, 1, 1, kv, dim) for _ in range(3))
    q *= 4  # the last rows' scores stand out of the zero keys' before them
    caches = [runtime.alloc(kv * capacity * dim) for _ in range(2)]
    lengths = runtime.alloc(1)
    append, attend = runtime.compile(put), runtime.compile(spec)
    out = runtime.alloc(kv * dim)
    bufs = [runtime.resident(x) for x in (k, v, np.arange(70), [n], q, kd, vd, [-1])]
    runtime.execute([(append, [*bufs[:4], *caches, lengths]),
                     (attend, [bufs[4], *caches, lengths, *bufs[5:], out])], 1)
    got = runtime.download(out).reshape(kv, dim).astype(np.float64)
    assert runtime.download(lengths)[0] == capacity
    for buffer in (*caches, lengths, out, *bufs):
        buffer.free()
    for h in range(kv):
        keys, values = (np.concatenate([a[0, :, h], b[0, :, h]]).astype(np.float64) for a, b in ((k, kd), (v, vd)))
        scores = keys @ q[0, 0, h].astype(np.float64) / np.sqrt(dim)
        weights = np.exp(scores)
        want = weights @ values / (weights.sum() + n)
        sizes = np.abs(keys) @ np.abs(q[0, 0, h]) / np.sqrt(dim)
        # As attend()'s bound; the zero keys' weights are a sum of at most capacity equal terms a lane, in 32 runs or
        # more (512 tiles a run at most), four keys a tile and lane: 2048 additions in a row.
        bound = dec.U * (2 * (2 * (dim + 2) * sizes.max() + 4) + 2 * 2048 + 16)
        assert (np.abs(got[h] - want) <= bound * (weights @ np.abs(values)) / (weights.sum() + n)).all()


# ---- the cache -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("batch,kv_heads,rows,picks,capacity,dim", [
    (1, 1, 1, 1, 1, 1), (3, 2, 7, 5, 40, 64), (2, 3, 20, 33, 50, 80), (4, 1, 100, 100, 150, 37), (2, 8, 64, 40, 60, 128),
    (2, 1, 17, 17000, 17100, 4), (1, 2, 5, 16385, 9000, 6), (5, 2, 9, 16, 16, 512)])
@pytest.mark.parametrize("token_major", [False, True])
def test_cache_append(runtime, batch, kv_heads, rows, picks, capacity, dim, token_major):
    rng = np.random.default_rng(picks)
    spec = {"op": "cache_append", "batch": batch, "kv_heads": kv_heads, "rows": rows, "picks": picks,
            "capacity": capacity, "dim": dim, "token_major": token_major}
    path = rng.integers(0, rows, (batch, picks)).astype(np.float32)  # rows may come twice
    ends = [-1.0, float(rows), np.nan, 0.5, np.inf]
    for b in range(1, batch):
        path[b, rng.integers(0, picks)] = ends[b % 5]
    lengths = np.array([0, capacity // 2, capacity, np.nan, capacity + 9][:batch], np.float32)
    x = {"k": normal(rng, *shape_of(token_major, batch, kv_heads, rows, dim)), "picks": path, "lengths": lengths,
         "v": normal(rng, *shape_of(token_major, batch, kv_heads, rows, dim)),
         "k_cache": normal(rng, *shape_of(token_major, batch, kv_heads, capacity, dim)),
         "v_cache": normal(rng, *shape_of(token_major, batch, kv_heads, capacity, dim))}
    want = dec.append(spec, x["k"], x["v"], path, lengths, x["k_cache"], x["v_cache"])
    got = run(runtime, spec, x, repeats=2)  # the lengths are not moved on: a replay writes the same rows
    for name, y in zip(("k_cache", "v_cache", "new_lengths"), want):
        assert (got[name].reshape(y.shape) == y).all(), name


# ---- together --------------------------------------------------------------------------------------------------

def test_a_decoder_steps_through_a_sequence(runtime):
    """Norm, rotation, attention over the cache and the append, token by token and draft by draft, against one causal
    pass of attention_online over the whole sequence."""
    heads, dim, seq = 3, 64, 23
    rng = np.random.default_rng(21)
    q, k, v = (normal(rng, 1, seq, heads, dim) for _ in range(3))
    weights = {n: 1 + 0.2 * normal(rng, dim) for n in ("q_weight", "k_weight")}
    whole = run(runtime, norm_spec(1, seq, heads, heads, dim, dim),
                {"q": q, "k": k, **weights, "positions": np.arange(seq)})
    qr, kr, vr = whole["q_out"], whole["k_out"], np.ascontiguousarray(np.swapaxes(v, 1, 2))
    want = run(runtime, {"op": "attention_online", "heads": heads, "seq": seq, "dim": dim, "causal": True},
               {"q": qr, "k": kr, "v": vr})["out"].reshape(heads, seq, dim)

    caches = [runtime.alloc(heads * seq * dim) for _ in range(2)]
    lengths = [runtime.resident([0.0]), runtime.alloc(1)]
    # Steps of one token, then a prompt's worth, then drafts with a rejected branch beside every accepted node.
    at, steps = 0, [1, 1, 9, 1, 4, 4, 3]
    assert sum(steps) == seq
    for count in steps:
        drafted = 2 * count if count > 1 else 1  # accepted tokens on even slots, wrong ones on odd
        rows = [at + n // 2 for n in range(drafted)] if count > 1 else [at]
        parents = [(n - 2 + n % 2 * 1 if n > 1 else -1) if n % 2 == 0 else n - 1 for n in range(drafted)]
        wrong = np.array([n % 2 for n in range(drafted)], bool)
        qs, ks, vs = (np.where(wrong[:, None, None], 5.0, x[0, rows]).astype(np.float32) for x in (q, k, v))
        positions = np.array([at + n // 2 + n % 2 for n in range(drafted)], np.float32)
        norm = runtime.compile(norm_spec(1, drafted, heads, heads, dim, dim))
        move = runtime.compile(rotary_spec(1, drafted, heads, dim, 2))  # position 0 everywhere: a change of layout
        tree = runtime.compile(tree_spec(1, heads, heads, drafted, seq, dim))
        append = runtime.compile({"op": "cache_append", "batch": 1, "kv_heads": heads, "rows": drafted,
                                  "picks": drafted, "capacity": seq, "dim": dim, "token_major": False})
        picks = np.full(drafted, -1.0)
        picks[:count] = np.arange(0, drafted, 2) if count > 1 else 0
        inputs = {n: runtime.resident(x) for n, x in (
            ("q", qs), ("k", ks), ("v", vs), ("positions", positions), ("zeros", np.zeros(drafted)),
            ("parents", parents), ("picks", picks), *weights.items())}
        made = {n: runtime.alloc(drafted * heads * dim) for n in ("q", "k", "v", "out")}
        runtime.execute([
            (norm, [inputs[n] for n in ("q", "k", "q_weight", "k_weight", "positions")] + [made["q"], made["k"]]),
            (move, [inputs["v"], inputs["zeros"], made["v"]]),
            (tree, [made["q"], *caches, lengths[0], made["k"], made["v"], inputs["parents"], made["out"]]),
            (append, [made["k"], made["v"], inputs["picks"], lengths[0], *caches, lengths[1]])], 2)
        out = runtime.download(made["out"]).reshape(heads, drafted, dim)
        right = [n for n in range(drafted) if not wrong[n]]
        # Both sides are FP32: 23 keys, dim 64, scores of normed vectors (|q| |k| / 8 <= 8 * 1.5^2): attend()'s bound
        # on each, 2 * 2 * 66 * 18 + 4 + 2 * 23 + 16 roundings of values of at most 4.
        assert np.abs(out[:, right] - want[:, at:at + count]).max() <= 2 * 4 * dec.U * (2 * (2 * 66 * 18 + 4) + 62)
        at += count
        assert runtime.download(lengths[1])[0] == at
        lengths.reverse()
        for x in (*inputs.values(), *made.values()):
            x.free()
        for kernel in (norm, move, tree, append):
            kernel.release()
    assert (runtime.download(caches[0]).reshape(heads, seq, dim) == kr.reshape(heads, seq, dim)).all()
    assert (runtime.download(caches[1]).reshape(heads, seq, dim) == vr.reshape(heads, seq, dim)).all()
    for x in (*caches, *lengths):
        x.free()


def test_two_kernels_of_one_shape_and_two_contexts(runtime):
    # One workspace a pipeline: dispatches of one kernel follow each other on the context's queue; another context
    # has a workspace of its own.
    rng = np.random.default_rng(30)
    spec = cross_spec(1, 2, 2, 1, 2000, 64)
    xs = [cross_inputs(rng, spec, [2000]) for _ in range(2)]
    kernel = runtime.compile(spec)
    bufs = [[runtime.resident(x[n]) for n in ("q", "k", "v", "lengths")] + [runtime.alloc(x["q"].size)] for x in xs]
    runtime.execute([(kernel, bufs[0]), (runtime.compile(spec), bufs[1])], 3)
    got = [runtime.download(b[4]) for b in bufs]
    with jade_hip.HipRuntime(0) as other:
        again = run(other, spec, xs[1])["out"]
    assert (again == got[1]).all()
    for x, y in zip(xs, got):
        within(y, *dec.cross(spec, x["q"], x["k"], x["v"], [2000]))


@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("heads", [16, 20, 40])
@pytest.mark.parametrize("q_scale,k_scale,v_scale", [(1.0, 1.0, 2.0 ** -120), (1.0, 1.0, 2.0 ** -60), (2.0 ** -120, 1.0, 1.0),
                                                    (1.0, 2.0 ** -120, 1.0), (2.0 ** -80, 2.0 ** 80, 2.0 ** 100),
                                                    (2.0 ** 70, 2.0 ** -70, 1.0), (1.0, 1.0, 0.0)])
def test_attention_cross_tiny_and_large_operands(runtime, dim, heads, q_scale, k_scale, v_scale):
    # Powers of two on the operands are exact: the outputs are those of N(0, 1) operands, scaled. V of 2^-120 has
    # outputs above 2^-126: nothing is subnormal but single values.
    rng = np.random.default_rng(31)
    spec = cross_spec(1, heads, 1, 1, 150, dim)
    x = cross_inputs(rng, spec, [150])
    for name, scale in (("q", q_scale), ("k", k_scale), ("v", v_scale)):
        x[name] = (x[name].astype(np.float64) * scale).astype(np.float32)
    want, off = dec.cross(spec, x["q"], x["k"], x["v"], [150])
    # Besides attend()'s bound, an FP32 output may be rounded to a multiple of 2^-149.
    within(run(runtime, spec, x)["out"], want, off + 2.0 ** -149)


@pytest.mark.parametrize("heads", [3, 20, 40])
@pytest.mark.parametrize("dim", [4, 12, 20, 36, 44, 60, 68, 76, 84, 100, 116, 124, 1, 2, 61, 67, 127])
@pytest.mark.parametrize("token_major", [False, True])
def test_attention_cross_head_dims(runtime, heads, dim, token_major):
    # Every remainder of the loads' 4, 8 and 16 dims, with one, two and three groups of rows.
    rng = np.random.default_rng(33)
    spec = cross_spec(1, 2 * heads, 2, 1, 140, dim, token_major)
    x = cross_inputs(rng, spec, [139])
    within(run(runtime, spec, x)["out"], *dec.cross(spec, x["q"], x["k"], x["v"], [139]))


# (batch, heads, kv_heads, queries, keys, dim) of each kernel, more sequences than a wave scans at once among them.
KERNELS = {"attention_ragged_d64": (70, 4, 2, 3, 90, 39), "attention_ragged_d128": (3, 2, 1, 8, 200, 101),
           "attention_ragged_parts_d64_r32": (3, 6, 2, 9, 150, 31), "attention_ragged_parts_d64_r64": (70, 1, 1, 40, 70, 63),
           "attention_ragged_parts_d96_r32": (3, 4, 1, 8, 390, 80), "attention_ragged_parts_d96_r64": (66, 1, 1, 50, 129, 95),
           "attention_ragged_parts_d128_r32": (3, 5, 1, 6, 400, 128), "attention_ragged_parts_d128_r64": (3, 2, 1, 35, 130, 127),
           "attention_flash_ragged_d32": (90, 8, 4, 20, 40, 24), "attention_flash_ragged_d64": (90, 4, 4, 33, 70, 60),
           "attention_flash_ragged_d96": (70, 10, 5, 17, 33, 84), "attention_flash_ragged_d128": (66, 8, 4, 50, 35, 116)}


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("token_major", [False, True])
def test_every_kernel_of_attention_cross(runtime, kernel, token_major):
    spec = cross_spec(*KERNELS[kernel], token_major)
    assert jade_hip.spec_describe(spec)["launch"]["kernel"] == kernel
    rng = np.random.default_rng(40)
    lengths = [spec["keys"], 0, 1, 32, 33][:spec["batch"]] + [int(n) for n in rng.integers(0, spec["keys"] + 1, spec["batch"])]
    lengths = lengths[:spec["batch"]]
    x = cross_inputs(rng, spec, lengths)
    clean = {n: x[n].copy() for n in "kv"}
    for b, n in enumerate(lengths):  # what lies past a length is never looked at
        dec.by_token(x["k"], token_major)[b, n:] = np.inf
        dec.by_token(x["v"], token_major)[b, n:] = np.nan
    # Some of the sequences against 64 bits; all of them against a launch of each alone would say the same.
    some = [0, 1, 2, spec["batch"] - 1]
    got = run(runtime, spec, x, repeats=2)["out"].reshape(x["q"].shape)
    part = dict(spec, batch=len(some))
    want, off = dec.cross(part, x["q"][some], clean["k"][some], clean["v"][some], [lengths[b] for b in some])
    within(got[some], want, off)
    assert np.isfinite(got).all()
    empty = [b for b in range(spec["batch"]) if lengths[b] == 0]
    assert (got[empty] == 0).all() and len(empty) >= 1


@pytest.mark.parametrize("kernel", [k for k in KERNELS if "flash" in k or "parts" in k])
def test_what_the_parts_do_not_carry(runtime, kernel):
    # Queries past 2^64, infinities and NaN among q, k and v: rows that do not meet them are as without them.
    spec = cross_spec(*KERNELS[kernel])
    rng = np.random.default_rng(41)
    lengths = [spec["keys"]] * spec["batch"]
    x = cross_inputs(rng, spec, lengths)
    x["q"][0, 0, 0] *= np.float32(2.0 ** 70)
    x["k"][0, 0] *= np.float32(2.0 ** -70)
    want, off = dec.cross(dict(spec, batch=3), x["q"][:3], x["k"][:3], x["v"][:3], lengths)
    x["q"][1, 0, 1, 2] = np.nan
    x["k"][2, 0, 7, 1] = np.nan  # seen by all rows of the group
    got = run(runtime, spec, x)["out"].reshape(x["q"].shape)
    within(got[0], want[0], off[0])
    assert np.isnan(got[1, 0, 1]).all()
    rows = [n for n in range(spec["queries"]) if n != 1]
    within(got[1, 0, rows], want[1, 0, rows], off[1, 0, rows])
    group = spec["heads"] // spec["kv_heads"]
    assert np.isnan(got[2, :group]).all()
    within(got[2, group:], want[2, group:], off[2, group:]) if group < spec["heads"] else None


@pytest.mark.parametrize("heads", [4, 20, 40])
@pytest.mark.parametrize("dim", [1, 30, 61, 67, 68, 80, 127])
@pytest.mark.parametrize("token_major", [False, True])
def test_what_lies_behind_a_row_that_is_not_whole_vectors(runtime, heads, dim, token_major):
    # Infinities and NaN in the other kv head, whose rows begin where a last vector of this one's ends, and (in
    # another sequence) in this head's next key, which is past the length.
    rng = np.random.default_rng(43)
    spec = cross_spec(2, 2 * heads, 2, 1, 140, dim, token_major)
    x = cross_inputs(rng, spec, [140, 77])
    want, off = dec.cross(spec, x["q"], x["k"], x["v"], [140, 77])
    for n, bad in (("k", np.nan), ("v", np.inf)):
        rows = dec.by_token(x[n], token_major)  # [batch, key, kv head, dim]
        rows[0, :, 1] = bad
        rows[1, 77:] = bad
    got = dec.by_token(run(runtime, spec, x)["out"].reshape(x["q"].shape), token_major)
    want, off = dec.by_token(want, token_major), dec.by_token(off, token_major)
    within(got[0, :, :heads], want[0, :, :heads], off[0, :, :heads])
    assert not np.isfinite(got[0, :, heads:]).any()
    within(got[1], want[1], off[1])


@pytest.mark.parametrize("nodes,dim", [(9, 64), (40, 128), (17, 30)])
def test_attention_tree_many_sequences(runtime, nodes, dim):
    rng = np.random.default_rng(42)
    spec = tree_spec(80, 2, 2, nodes, 50, dim)
    lengths = rng.integers(0, 51, 80)
    x = tree_inputs(rng, spec, lengths)
    got = run(runtime, spec, x)["out"].reshape(x["q"].shape)
    some = [0, 63, 64, 79]
    part = {n: v[some] for n, v in x.items()}
    want, off = tree_want(dict(spec, batch=4), part)
    within(got[some], want, off)


@pytest.mark.parametrize("heads,dim", [(16, 64), (20, 128), (40, 64), (40, 128), (20, 36), (20, 96), (40, 80), (40, 87)])
def test_attention_cross_not_finite_among_many_rows(runtime, heads, dim):
    # One row's query, one key's value: the others' outputs are as without them.
    rng = np.random.default_rng(32)
    spec = cross_spec(2, heads, 1, 1, 200, dim)
    x = cross_inputs(rng, spec, [200, 150])
    want, off = dec.cross(spec, x["q"], x["k"], x["v"], [200, 150])
    x["q"][0, 5] = np.nan
    x["q"][0, 7, 0, 1] = np.inf
    x["v"][1, 0, 149, 3] = -np.inf
    x["v"][1, 0, 150:] = np.nan
    got = run(runtime, spec, x)["out"].reshape(want.shape)
    others = [h for h in range(heads) if h not in (5, 7)]
    within(got[0, others], want[0, others], off[0, others])
    assert np.isnan(got[0, 5]).all()
    kept = [d for d in range(dim) if d != 3]
    within(got[1][..., kept], want[1][..., kept], off[1][..., kept])
    assert np.isneginf(got[1, :, 0, 3]).all()


@pytest.mark.parametrize("queries,dim", [(1, 8), (20, 8), (40, 12)])
def test_thousands_of_sequences(runtime, queries, dim):
    # Forty-seven scans of 64 sequences, most of them empty, so that runs begin far from each other.
    batch = 3000
    rng = np.random.default_rng(44)
    spec = cross_spec(batch, 1, 1, queries, 150, dim)
    lengths = np.where(rng.random(batch) < 0.7, 0, rng.integers(0, 151, batch))
    x = cross_inputs(rng, spec, lengths)
    got = run(runtime, spec, x)["out"].reshape(x["q"].shape)
    assert (got[lengths == 0] == 0).all() and np.isfinite(got).all()
    some = [0, 63, 64, 1500, 2999] + list(np.flatnonzero(lengths)[::90])
    want, off = dec.cross(dict(spec, batch=len(some)), *(x[n][some] for n in "qkv"), lengths[some])
    within(got[some], want, off)
