"""Paged attention over long caches and large values: sums of many weights, tables of many entries, means of values
whose sums no FP32 number holds. References in 64 bits for a few rows;
bounds count roundings (U is half an ulp), as paged_oracle.py's do."""
import numpy as np
import pytest

import paged_oracle as po
from decoder_oracle import U
from test_gpu_decoder import normal, run, within
from test_gpu_paged import paged_inputs, paged_spec

pytestmark = pytest.mark.gpu


def compile_paged(runtime, batch, heads, queries, page, tokens, dim, pages):
    return runtime.compile({"op": "attention_paged", "batch": batch, "heads": heads, "kv_heads": 1, "queries": queries,
                            "pages": pages, "page": page, "table": -(-tokens // page), "dim": dim,
                            "token_major": True, "pages_token_major": True})


def attend_on(runtime, kernel, *inputs):
    buffers = [runtime.resident(x) for x in inputs]
    out = runtime.alloc(inputs[0].size)
    runtime.execute([(kernel, buffers + [out])], 1)
    got = runtime.download(out).astype(np.float64)
    for b in (*buffers, out):
        b.free()
    kernel.release()
    return got


# Roundings of sums over keys, of terms alike: a running sum is half of its last value in the mean. A sum is put aside
# and begun anew after 64 tiles of a wave's 16 keys (FP32 MFMAs: an addition for each key, a lane's weights a quarter of
# them) or 128 tiles of 32 (parts: six products a key). The matrix cores do not round to nearest, 2 U for each addition.
# Then an addition for each such piece, and 512 for the runs that are joined. Numerator and denominator; last, both
# weights' and their scores' own roundings: 4 for exp2 and its argument, dim + 2 for the score.
def mean_bound(parts, tokens, dim):
    pieces = tokens / (4096 if parts else 1024) + 512
    products, weights = (128 * 32 * 6, 128 * 16) if parts else (64 * 16, 64 * 4)
    return U * ((2 * products + pieces) / 2 + (weights + pieces) / 2 + 2 * (4 + 2 * (dim + 2)) + 16)


@pytest.mark.parametrize("queries,dim,tokens", [(1, 8, 2 ** 21 + 777), (20, 8, 2 ** 20 + 1), (1, 80, 2 ** 18 + 99), (64, 8, 2 ** 22 + 33),
                                                (64, 128, 2 ** 19 + 5)])
@pytest.mark.parametrize("batch", [1, 300, 512])
def test_attention_paged_sums_of_a_million_equal_weights(runtime, queries, dim, tokens, batch):
    # The first token's score is the greatest; all others weigh 0.502 beside it, which takes two bf16 parts. Many
    # sequences over the same pages, so that one run has all of a sequence's tokens; and one, cut between all runs.
    rng = np.random.default_rng(60)
    page = 1024
    table = -(-tokens // page)
    q = np.zeros((batch, queries, 1, dim), np.float32)
    q[..., 0] = 1
    k, v = np.zeros((2, table * page, dim), np.float32)
    k[1:, 0] = np.log(0.501953125) * np.sqrt(dim)
    # Values: everywhere 1; the first half of the tokens; every other one; one wave's; random ones; far ones.
    at = np.arange(table * page)
    v[:, 0], v[:, 1], v[:, 2], v[:, 3] = 1, at < tokens // 2, at % 2, at % 64 < 16
    v[:, 4], v[:, 5], v[:, 6] = rng.random(at.size), at >= tokens - 5000, 1 + (at % 3 == 0)
    v[:, 7:] = v[:, :1]
    tables = np.tile(np.arange(table, dtype=np.float32), (batch, 1))
    kernel = compile_paged(runtime, batch, 1, queries, page, tokens, dim, table)
    parts = kernel.launch["kernel"].startswith("attention_paged_flash")
    assert parts == (queries == 64)
    got = attend_on(runtime, kernel, q, k, v, tables, np.full(batch, tokens, np.float32), np.full(batch, queries, np.float32))
    weights = np.ones(tokens)
    weights[1:] = np.exp(float(k[1, 0]) / np.sqrt(dim))
    sums = np.cumsum(weights[:, None] * v[:tokens, :8].astype(np.float64), axis=0)[-queries:]
    want = sums / np.cumsum(weights)[-queries:, None]
    error = np.abs(got.reshape(batch, queries, dim)[..., :8] - want) / want
    assert error.max() <= mean_bound(parts, tokens, dim), (error.max(axis=(0, 1)), mean_bound(parts, tokens, dim))


@pytest.mark.parametrize("page,queries,dim", [(16, 1, 32), (48, 1, 31), (1008, 1, 32), (1024, 1, 32), (16, 64, 32), (48, 64, 32),
                                              (1008, 64, 32), (1024, 64, 32), (48, 20, 32)])
def test_attention_paged_tables_of_many_entries(runtime, page, queries, dim):
    # Pages in no order; scores so far apart that a few dozen of the keys make up a row, wherever they lie.
    rng = np.random.default_rng(page + queries)
    tokens = 300000 + page // 2 + 5
    table = -(-tokens // page)
    q = 3 * normal(rng, 1, queries, 1, dim)
    k, v = normal(rng, 2, table * page, dim)
    tables = rng.permutation(table + 7)[:table].astype(np.float32)
    pools = np.full((2, table + 7, page, dim), np.nan, np.float32)
    for pool, x in zip(pools, (k, v)):
        pool[tables.astype(int)] = x.reshape(table, page, dim)
    kernel = compile_paged(runtime, 1, 1, queries, page, tokens, dim, table + 7)
    parts = kernel.launch["kernel"].startswith("attention_paged_flash")
    got = attend_on(runtime, kernel, q, *pools, tables, [tokens], [queries]).reshape(queries, dim)
    k, v = k.astype(np.float64), v.astype(np.float64)
    for i in sorted({0, queries // 2, queries - 1}):
        seen = tokens - queries + 1 + i
        row = q[0, i, 0].astype(np.float64) / np.sqrt(dim)
        scores, sizes = k[:seen] @ row, np.abs(k[:seen]) @ np.abs(row)
        p = np.exp(scores - scores.max())
        p /= p.sum()
        # Terms of any order: every addition's rounding in full, twice what mean_bound says; scores' by their sizes.
        off = 2 * mean_bound(parts, tokens, dim) + U * 4 * (dim + 2) * sizes.max()
        assert (np.abs(got[i] - p @ v[:seen]) <= off * (p @ np.abs(v[:seen]))).all()


@pytest.mark.parametrize("queries,dim", [(1, 64), (1, 37), (1, 128), (3, 80), (20, 64), (24, 128), (40, 64), (60, 96), (60, 128), (70, 30), (140, 128)])
@pytest.mark.parametrize("tokens", [96, 3840])
@pytest.mark.parametrize("scale", [0.0, 4.0])
def test_attention_paged_values_near_the_largest(runtime, queries, dim, tokens, scale):
    # Values whose weighted sum no FP32 number holds, though their mean is one: over equal keys, and where the maximum
    # grows from tile to tile; subnormal and ordinary values in the same rows. Whole, and cut between runs.
    rng = np.random.default_rng(61)
    spec = paged_spec(1, 2, 1, queries, 48, tokens // 48, dim)
    x = paged_inputs(rng, spec, [tokens], [queries])
    x["q"] *= np.float32(scale)
    v = po.pool_by_token(spec, x["v_pages"])
    v[..., 0::5] = np.abs(v[..., 0::5]) * 1e37 + 2e38
    v[..., 1::5] *= 5e37
    v[..., 2::5] *= 1e-38
    v[..., 4::5] *= 1e-43
    np.clip(v, -3.2e38, 3.2e38, out=v)
    want, off = po.paged(spec, x["q"], x["k_pages"], x["v_pages"], x["tables"], x["lengths"], x["counts"])
    assert (np.abs(want) + off).max() < np.finfo(np.float32).max
    got = po.rows_by_token(spec, run(runtime, spec, x)["out"], 2, queries)
    # Subnormal values: a smallest subnormal for each one summed.
    within(got, want, off + tokens * 2.0 ** -149)


@pytest.mark.parametrize("queries,dim", [(1, 64), (20, 128), (40, 64), (60, 128), (60, 64)])
def test_attention_paged_large_values_over_long_caches(runtime, queries, dim):
    # So many of them that sums are put aside; infinities beside them, which reach their dims' rows and no others.
    rng = np.random.default_rng(62)
    tokens, page = 70000, 1024
    table = -(-tokens // page)
    batch = 300
    q, k = np.zeros((batch, queries, 1, dim), np.float32), np.zeros((table * page, dim), np.float32)
    v = np.full((table * page, dim), 2.5e38, np.float32)
    v[:, 1], v[:, 2] = 1e-30, rng.random(table * page)
    v[tokens - queries // 2:tokens, 3] = np.inf
    v[::2, 4] = -2.5e38
    kernel = compile_paged(runtime, batch, 1, queries, page, tokens, dim, table)
    got = attend_on(runtime, kernel, q, k, v, np.tile(np.arange(table, dtype=np.float32), (batch, 1)),
                    np.full(batch, tokens), np.full(batch, queries)).reshape(batch, queries, dim)
    seen = tokens - queries + 1 + np.arange(queries)
    sizes, sums = (np.cumsum(f(v.astype(np.float64)), axis=0)[seen - 1] / seen[:, None] for f in (np.abs, np.asarray))
    reached = np.isinf(sums)
    assert reached[:, 3].sum() == queries // 2 and not reached[:, 4:].any()
    assert (got[:, reached] == np.inf).all()
    off = 2 * mean_bound(queries >= 40, tokens, dim) * sizes
    assert (np.abs(got[:, ~reached] - sums[~reached]) <= off[~reached]).all()


@pytest.mark.parametrize("queries,dim", [(1, 64), (3, 37), (20, 128), (40, 64), (70, 32), (60, 96), (60, 128)])
@pytest.mark.parametrize("tokens", [96, 3840])
def test_attention_paged_scores_of_minus_infinity(runtime, queries, dim, tokens):
    # They weigh nothing: rows that see no other score are zeros, those that see one other have its value.
    rng = np.random.default_rng(63)
    spec = paged_spec(1, 2, 1, queries, 48, tokens // 48, dim, spare=0)
    x = paged_inputs(rng, spec, [tokens], [queries])
    x["q"][:] = np.abs(x["q"])
    place = po.places(spec, x["tables"][0], [tokens - (queries + 1) // 2])[0]
    k = po.pool_by_token(spec, x["k_pages"])
    other = k[place].copy()
    k[..., dim // 2] = -np.inf
    k[place] = other
    got = po.rows_by_token(spec, run(runtime, spec, x)["out"], 2, queries)[0]
    first = queries - (queries + 1) // 2
    assert (got[:first] == 0).all()
    value = po.pool_by_token(spec, x["v_pages"])[place][0]
    assert (np.abs(got[first:] - value) <= 16 * U * np.abs(value)).all()
