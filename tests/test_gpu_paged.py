"""Decoding over a paged cache (attention_paged, pages_append, pages_fork, pages_copy, beam_select) on the GPU against
64-bit restatements (paged_oracle.py), with its derived bounds."""
import numpy as np
import pytest

import paged_oracle as po
from test_gpu_decoder import normal, run, within

pytestmark = pytest.mark.gpu

LAYOUTS = [(True, True), (True, False), (False, True), (False, False)]


def table_for(rng, spec, lengths):
    """Pages in no order for every sequence, -1 past its length; no page twice."""
    order = iter(rng.permutation(spec["pages"]))
    tables = np.full((spec["batch"], spec["table"]), -1, np.float32)
    for row, n in zip(tables, lengths):
        held = min(spec["table"], -(-int(n) // spec["page"]))
        row[:held] = [next(order) for _ in range(held)]
    return tables


def pools_for(rng, spec):
    n = spec["pages"] * spec["page"] * spec["kv_heads"] * spec["dim"]
    return {"k_pages": normal(rng, n), "v_pages": normal(rng, n)}


def same(got, want):
    np.testing.assert_array_equal(got.reshape(want.shape), want)


# ---- attention_paged -----------------------------------------------------------------------------------------

def paged_spec(batch, heads, kv_heads, queries, page, table, dim, layout=(True, True), spare=3):
    return {"op": "attention_paged", "batch": batch, "heads": heads, "kv_heads": kv_heads, "queries": queries,
            "pages": batch * table + spare, "page": page, "table": table, "dim": dim, "token_major": layout[0],
            "pages_token_major": layout[1]}


def paged_inputs(rng, spec, lengths, counts):
    cap = spec["table"] * spec["page"]
    return {"q": normal(rng, spec["batch"] * spec["heads"] * spec["queries"] * spec["dim"]), **pools_for(rng, spec),
            "tables": table_for(rng, spec, [po.length_of(n, cap) for n in lengths]),
            "lengths": np.array(lengths, np.float32), "counts": np.array(counts, np.float32)}


def check_paged(runtime, spec, x, clean=None):
    """`clean`: the pools that the oracle reads where those on the GPU hold what nobody may see."""
    y = dict(x, **(clean or {}))
    want, off = po.paged(spec, x["q"], y["k_pages"], y["v_pages"], x["tables"], x["lengths"], x["counts"])
    got = po.rows_by_token(spec, run(runtime, spec, x)["out"], spec["heads"], spec["queries"])
    within(got, want, off)
    return got, want


# One token of one sequence, groups, odd and scalar dims, pages of every step within a tile, tables past 64 tiles,
# blocks of rows that end inside a query's heads.
@pytest.mark.parametrize("batch,heads,kv_heads,queries,page,table,dim", [
    (1, 1, 1, 1, 16, 1, 1), (1, 8, 8, 1, 16, 9, 64), (2, 8, 2, 1, 16, 13, 128), (3, 6, 2, 2, 48, 3, 80), (2, 4, 4, 1, 256, 2, 96),
    (2, 3, 1, 5, 32, 5, 37), (1, 2, 1, 7, 1024, 1, 64), (2, 12, 4, 5, 16, 9, 3), (1, 5, 5, 3, 80, 4, 126), (2, 16, 1, 1, 112, 2, 32),
    (2, 2, 2, 16, 16, 6, 40)])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_attention_paged_few_rows(runtime, batch, heads, kv_heads, queries, page, table, dim, layout):
    rng = np.random.default_rng(page * table + dim)
    spec = paged_spec(batch, heads, kv_heads, queries, page, table, dim, layout)
    cap = page * table
    lengths = [cap, max(1, cap - 17), cap // 2][:batch]
    check_paged(runtime, spec, paged_inputs(rng, spec, lengths, [queries, max(1, queries - 1), 1][:batch]))


@pytest.mark.parametrize("batch,heads,kv_heads,queries,page,table,dim", [
    (2, 40, 1, 1, 16, 9, 64), (1, 40, 1, 2, 16, 9, 37), (1, 300, 1, 1, 16, 5, 128), (1, 300, 1, 3, 32, 3, 30), (2, 20, 1, 2, 48, 4, 32),
    (2, 20, 1, 1, 16, 9, 80), (1, 12, 1, 2, 16, 20, 96), (1, 20, 1, 1, 32, 5, 90), (2, 3, 1, 9, 16, 9, 67),
    (1, 2, 2, 17, 16, 4, 64), (2, 8, 2, 8, 16, 10, 128), (1, 6, 3, 40, 48, 4, 80), (2, 4, 1, 33, 32, 9, 96), (1, 1, 1, 200, 16, 15, 32),
    (2, 3, 3, 70, 80, 3, 37), (1, 5, 1, 61, 64, 7, 128), (2, 2, 1, 100, 256, 1, 30), (1, 7, 7, 129, 16, 9, 126), (2, 4, 2, 64, 16, 8, 64)])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_attention_paged_chunks(runtime, batch, heads, kv_heads, queries, page, table, dim, layout):
    rng = np.random.default_rng(queries + dim)
    spec = paged_spec(batch, heads, kv_heads, queries, page, table, dim, layout)
    cap = page * table
    lengths = [cap, max(1, cap - 19)][:batch]
    check_paged(runtime, spec, paged_inputs(rng, spec, lengths, [min(queries, cap), max(1, queries // 3)][:batch]))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("heads,kv_heads,queries,dim", [(4, 2, 1, 64), (4, 2, 3, 30), (4, 2, 20, 128), (4, 1, 70, 64)])
def test_attention_paged_odd_lengths_and_counts(runtime, heads, kv_heads, queries, dim, layout):
    # Lengths zero, one, fractions, NaN, past the table; counts zero, NaN, past the queries and past the length. Keys and
    # values past the lengths, and all of the pages that no table names, are NaN and infinite, and so are queries past the
    # counts; tables go on past the lengths with pages that are others', or with anything. Rows without a key are zeros.
    rng = np.random.default_rng(7)
    lengths = [0.0, 1.0, 16.0, 17.9, np.nan, -4.0, 1e30, 33.0, 5.0, 64.0, 40.0, np.inf]
    counts = [1.0, 1.0, 2.5, 1e9, 1.0, 1.0, 2.0, 0.0, 64.0, np.nan, 3.0, 1.0]
    spec = paged_spec(len(lengths), heads, kv_heads, queries, 16, 5, dim, layout)
    x = paged_inputs(rng, spec, lengths, counts)
    clean = {n: x[n].copy() for n in ("k_pages", "v_pages")}
    seen = np.zeros((spec["pages"], 16), bool)
    for b, n in enumerate(lengths):
        for place in po.places(spec, x["tables"][b], range(po.length_of(n, 80))):
            seen[place] = True
    for name, value in (("k_pages", np.nan), ("v_pages", np.inf)):
        po.pool_by_token(spec, x[name])[~seen] = value
        po.pool_by_token(spec, clean[name])[~seen] = 0
    q = po.rows_by_token(spec, x["q"], heads, queries)
    for b, (n, c) in enumerate(zip(lengths, counts)):
        held = -(-po.length_of(n, 80) // 16)
        x["tables"][b, held:] = rng.choice([0, 3, spec["pages"] - 1, np.nan, -1, 1e9, np.inf, 0.5], 5 - held)
        q[b, po.length_of(c, queries):] = np.nan
    got, want = check_paged(runtime, spec, x, clean)
    none = want == 0
    assert (got[none] == 0).all()


@pytest.mark.parametrize("queries,dim", [(1, 64), (5, 80), (24, 128), (48, 64), (48, 32), (48, 96), (48, 128), (48, 37)])
def test_attention_paged_entries_that_name_no_page(runtime, queries, dim):
    rng = np.random.default_rng(8)
    spec = paged_spec(4, 4, 2, queries, 48, 4, dim)
    x = paged_inputs(rng, spec, [192, 150, 97, 48], [queries] * 4)
    x["tables"][0, 1], x["tables"][0, 3] = np.nan, spec["pages"]
    x["tables"][1, 0], x["tables"][2, 2], x["tables"][3, 0] = -7, 0.5, np.inf  # the last has no page at all
    got, _ = check_paged(runtime, spec, x)
    assert (got[3] == 0).all()


@pytest.mark.parametrize("queries,dim", [(3, 64), (9, 128), (30, 64), (40, 128), (25, 80), (5, 37), (21, 30), (70, 64), (90, 128),
                                         (120, 32), (140, 80), (100, 37)])
def test_attention_paged_later_tokens_that_are_not_finite(runtime, queries, dim):
    # A chunk's own keys and values that are not finite reach the queries from that token on and no others.
    rng = np.random.default_rng(9)
    spec = paged_spec(1, 4, 2, queries, 16, 12, dim)
    length = 150
    x = paged_inputs(rng, spec, [length], [queries])
    clean = {n: x[n].copy() for n in ("k_pages", "v_pages")}
    bad = length - queries // 2
    places = po.places(spec, x["tables"][0], range(length))
    for name, values in (("k_pages", (np.nan, np.inf)), ("v_pages", (np.inf, np.nan))):
        pool = po.pool_by_token(spec, x[name])
        for t, value in zip((bad, bad + 1), values):
            if t < length:
                pool[places[t]] = value
    want, off = po.paged(spec, x["q"], clean["k_pages"], clean["v_pages"], x["tables"], x["lengths"], x["counts"])
    got = po.rows_by_token(spec, run(runtime, spec, x)["out"], 4, queries)
    first = bad - (length - queries)
    within(got[:, :first], want[:, :first], off[:, :first])
    assert not np.isfinite(got[:, first:]).any()


@pytest.mark.parametrize("queries,dim", [(1, 64), (1, 128), (3, 80), (20, 128), (40, 64), (60, 128), (200, 64), (70, 32), (90, 80)])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_attention_paged_long_contexts_are_cut_and_joined(runtime, queries, dim, layout):
    rng = np.random.default_rng(10)
    spec = paged_spec(2, 2, 1, queries, 64, 60, dim, layout)
    check_paged(runtime, spec, paged_inputs(rng, spec, [3840, 1777], [queries, 1]))


@pytest.mark.parametrize("queries,batch,table", [(1, 333, 4), (12, 333, 4), (24, 333, 4), (64, 333, 4), (1, 100, 13), (5, 70, 40), (24, 150, 9),
                                                 (64, 90, 21)])
def test_attention_paged_many_sequences_most_of_them_idle(runtime, queries, batch, table):
    # More than a wave's lanes of sequences, most of them without tokens or without new ones.
    rng = np.random.default_rng(11)
    spec = paged_spec(batch, 4, 2, queries, 16, table, 32)
    lengths = [int(rng.integers(1, 16 * table + 1)) if b % 3 == 0 else 0 for b in range(batch)]
    counts = [0 if b % 5 == 0 else min(max(n, 1), int(rng.integers(1, queries + 1))) for b, n in enumerate(lengths)]
    check_paged(runtime, spec, paged_inputs(rng, spec, lengths, counts))


# Whole prompts without a past, whose blocks of rows end at keys of their own; many short units a run.
@pytest.mark.parametrize("batch,heads,kv_heads,length,dim", [(1, 4, 1, 700, 64), (2, 2, 2, 600, 128), (3, 24, 24, 300, 32), (40, 8, 8, 150, 64)])
def test_attention_paged_whole_prompts(runtime, batch, heads, kv_heads, length, dim):
    rng = np.random.default_rng(16)
    spec = paged_spec(batch, heads, kv_heads, length, 32, -(-length // 32), dim)
    lengths = [length - 7 * b for b in range(batch)]
    x = paged_inputs(rng, spec, [max(1, n) for n in lengths], [max(1, n) for n in lengths])
    if batch * heads * length * length < 4e6:
        check_paged(runtime, spec, x)
        return
    # The same from a sequence's own prompt by itself, which the small cases check.
    got = po.rows_by_token(spec, run(runtime, spec, x)["out"], heads, length)
    for b in (0, batch // 2, batch - 1):
        one = dict(spec, batch=1)
        y = dict(x, tables=x["tables"][b:b + 1], lengths=x["lengths"][b:b + 1], counts=x["counts"][b:b + 1],
                 q=x["q"].reshape(batch, -1)[b])
        n = int(x["lengths"][b])
        rows = [0, n // 2, n - 1]
        pools = [po.pool_by_token(spec, x[name].astype(np.float64)) for name in ("k_pages", "v_pages")]
        places = po.places(spec, x["tables"][b], range(n))
        keys, values = ([pool[p] for p in places] for pool in pools)
        keys, values = np.array(keys), np.array(values)
        q = po.rows_by_token(one, y["q"].astype(np.float64), heads, length)[0]
        for i in rows:
            for h in (0, heads - 1):
                want, off = po.attend(q[i, h], keys[:, h * kv_heads // heads], values[:, h * kv_heads // heads], range(i + 1))
                assert (np.abs(got[b, i, h] - want) <= off).all()


@pytest.mark.parametrize("queries", [1, 24, 70])
def test_attention_paged_sequences_that_share_pages(runtime, queries):
    rng = np.random.default_rng(12)
    spec = paged_spec(3, 4, 4, queries, 16, 8, 64)
    x = paged_inputs(rng, spec, [100, 128, 77], [queries] * 3)
    x["tables"][1, :4] = x["tables"][2, :4] = x["tables"][0, :4]
    check_paged(runtime, spec, x)


@pytest.mark.parametrize("queries,dim", [(1, 64), (24, 128), (24, 80), (40, 64), (60, 128), (60, 96)])
def test_attention_paged_large_and_tiny_operands(runtime, queries, dim):
    rng = np.random.default_rng(13)
    spec = paged_spec(1, 2, 1, queries, 16, 6, dim)
    for q, k, v in ((1e-30, 1e30, 1e-40), (1e15, 1e-15, 1e30), (1e-20, 1.0, 1e-38), (2.0 ** 70, 2.0 ** -70, 1.0)):
        x = paged_inputs(rng, spec, [96], [queries])
        x["q"] = (x["q"] * np.float32(q)).astype(np.float32)
        x["k_pages"] = (x["k_pages"] * np.float32(k)).astype(np.float32)
        x["v_pages"] = (x["v_pages"].astype(np.float64) * v).astype(np.float32)
        want, off = po.paged(spec, x["q"], x["k_pages"], x["v_pages"], x["tables"], x["lengths"], x["counts"])
        # Results below FP32's normal range are off by the smallest subnormal, 2^-149, for each of the values summed.
        got = po.rows_by_token(spec, run(runtime, spec, x)["out"], 2, queries)
        within(got, want, off + 96 * 2.0 ** -149)


@pytest.mark.parametrize("queries,dim", [(1, 64), (6, 128), (10, 64), (40, 64), (40, 128), (9, 37)])
def test_attention_paged_queries_that_are_not_finite(runtime, queries, dim):
    # They spoil their own row and no other, whichever rows share their wave.
    rng = np.random.default_rng(17)
    spec = paged_spec(2, 8, 2, queries, 16, 8, dim)
    x = paged_inputs(rng, spec, [128, 100], [queries, queries])
    clean = x["q"].copy()
    q = po.rows_by_token(spec, x["q"], 8, queries)
    bad = [(0, 0, 1, 0, np.nan), (0, queries - 1, 6, dim - 1, np.inf), (1, queries // 2, 3, dim // 2, -np.inf)]
    for b, i, h, d, value in bad:
        q[b, i, h, d] = value
    want, off = po.paged(spec, clean, x["k_pages"], x["v_pages"], x["tables"], x["lengths"], x["counts"])
    got = po.rows_by_token(spec, run(runtime, spec, x)["out"], 8, queries)
    spoilt = np.zeros(got.shape[:3], bool)
    for b, i, h, *_ in bad:
        spoilt[b, i, h] = True
    assert np.isnan(got[spoilt]).any(axis=1).all()
    within(got[~spoilt], want[~spoilt], off[~spoilt])


@pytest.mark.parametrize("by_token", [True, False])
def test_pages_past_32_bits_of_elements(runtime, by_token):
    # Two pools of 20 GB, which only the kernels write: rows appended to their last pages, copied to the first, read by both
    # attention kernels. Without a copy on the host the first pages' content is what attention says it is.
    rng = np.random.default_rng(18)
    pool = dict(kv_heads=8, pages=300000, page=16, dim=128, pages_token_major=by_token)
    assert pool["pages"] * 16 * 8 * 128 > 2 ** 32
    k_pages, v_pages = (runtime.alloc(pool["pages"] * 16 * 8 * 128) for _ in range(2))
    append = runtime.compile({"op": "pages_append", "batch": 1, "rows": 100, **pool, "table": 7, "token_major": True})
    copy = runtime.compile({"op": "pages_copy", "copies": 7, **pool})
    far = np.array([299999, 262144, 262143, 299000, 280001, 299998, 270000], np.float32)
    near = np.array([0, 5, 1, 9, 2, 7, 3], np.float32)
    k, v = normal(rng, 1, 100, 8, 128), normal(rng, 1, 100, 8, 128)
    named = {n: runtime.resident(x) for n, x in dict(k=k, v=v, counts=[100], far=far, near=near, lengths=[0], ends=[100],
                                                     rows=[16] * 6 + [4]).items()}
    new_lengths = runtime.alloc(1)
    runtime.execute([(append, [named["k"], named["v"], named["counts"], named["far"], named["lengths"], k_pages, v_pages, new_lengths]),
                     (copy, [named["far"], named["near"], named["rows"], k_pages, v_pages])], 1)
    assert runtime.download(new_lengths) == [100]
    # The oracle's small pool: the pages in order.
    small = dict(pool, pages=7, pages_token_major=True)
    pools = [np.zeros((7, 16, 8, 128), np.float32) for _ in range(2)]
    for x, y in zip(pools, (k, v)):
        x.reshape(112, 8, 128)[:100] = y[0]
    for queries, count in ((1, 1), (40, 40)):
        spec = {"op": "attention_paged", "batch": 1, "heads": 16, "queries": queries, **pool, "table": 7, "token_major": True}
        attend = runtime.compile(spec)
        q = normal(rng, 1, queries, 16, 128)
        bq, bc, out = runtime.resident(q), runtime.resident([count]), runtime.alloc(q.size)
        want, off = po.paged(dict(spec, **small), q, *pools, np.arange(7.0)[None], [100], [count])
        for table in ("far", "near"):
            runtime.execute([(attend, [bq, k_pages, v_pages, named[table], named["ends"], bc, out])], 1)
            within(runtime.download(out), want, off)
        for x in (bq, bc, out):
            x.free()
        attend.release()
    for x in (*named.values(), k_pages, v_pages, new_lengths):
        x.free()


def test_attention_paged_runs_the_same_twice(runtime):
    rng = np.random.default_rng(14)
    for queries in (1, 24, 100):
        spec = paged_spec(3, 8, 2, queries, 16, 40, 128)
        x = paged_inputs(rng, spec, [640, 333, 500], [queries, 1, queries])
        first, again = (run(runtime, spec, x, repeats)["out"] for repeats in (1, 3))
        same(again, first)


def test_attention_paged_is_the_contiguous_caches_attention(runtime):
    # One new token a sequence: attention_tree of one node over the cache before it, to the bounds of both.
    rng = np.random.default_rng(15)
    batch, heads, kv, dim, cap = 3, 8, 2, 64, 160
    spec = paged_spec(batch, heads, kv, 1, 16, 10, dim, (False, False))
    lengths = [160, 97, 1]
    x = paged_inputs(rng, spec, lengths, [1] * 3)
    got = run(runtime, spec, x)["out"].reshape(batch, heads, dim)
    caches = {}
    drafts = {}
    for name in ("k", "v"):
        cache, draft = np.zeros((batch, kv, cap, dim), np.float32), np.zeros((batch, kv, 1, dim), np.float32)
        pool = po.pool_by_token(spec, x[name + "_pages"])
        for b, n in enumerate(lengths):
            rows = np.stack([pool[p] for p in po.places(spec, x["tables"][b], range(n))], axis=1)
            cache[b, :, :n - 1], draft[b, :, 0] = rows[:, :-1], rows[:, -1]
        caches[name + "_cache"], drafts[name + "_draft"] = cache, draft
    tree = {"op": "attention_tree", "batch": batch, "heads": heads, "kv_heads": kv, "nodes": 1, "capacity": cap, "dim": dim,
            "token_major": False}
    other = run(runtime, tree, {"q": x["q"], **caches, **drafts, "lengths": np.array(lengths, np.float32) - 1,
                                "parents": np.full((batch, 1), -1.0)})["out"].reshape(got.shape)
    _, off = po.paged(spec, x["q"], x["k_pages"], x["v_pages"], x["tables"], lengths, [1] * 3)
    assert (np.abs(got - other) <= 2 * off[:, 0]).all()


# ---- pages_append --------------------------------------------------------------------------------------------

def append_spec(batch, kv_heads, rows, page, table, dim, layout):
    return {"op": "pages_append", "batch": batch, "kv_heads": kv_heads, "rows": rows, "pages": batch * table + 2, "page": page,
            "table": table, "dim": dim, "token_major": layout[0], "pages_token_major": layout[1]}


def check_append(runtime, spec, x):
    want_k, want_v, want = po.append(spec, x["k"], x["v"], x["counts"], x["tables"], x["lengths"], x["k_pages"], x["v_pages"])
    got = run(runtime, spec, x, 2)  # the same rows in the same places again
    same(po.pool_by_token(spec, got["k_pages"]), want_k)
    same(po.pool_by_token(spec, got["v_pages"]), want_v)
    same(got["new_lengths"], want)


@pytest.mark.parametrize("batch,kv_heads,rows,page,table,dim", [
    (1, 1, 1, 16, 1, 1), (3, 8, 1, 16, 5, 128), (2, 3, 40, 16, 5, 40), (2, 2, 100, 48, 3, 7), (1, 5, 33, 64, 2, 512), (2, 1, 3, 1024, 1, 30)])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_pages_append(runtime, batch, kv_heads, rows, page, table, dim, layout):
    rng = np.random.default_rng(rows + dim)
    spec = append_spec(batch, kv_heads, rows, page, table, dim, layout)
    cap, n = page * table, batch * kv_heads * rows * dim
    lengths = [cap - rows, 3, cap // 2][:batch]
    check_append(runtime, spec, {"k": normal(rng, n), "v": normal(rng, n), "counts": np.array([rows, max(1, rows - 2), 1][:batch], np.float32),
                                 "tables": table_for(rng, spec, [cap] * batch), "lengths": np.array(lengths, np.float32),
                                 **pools_for(rng, spec)})


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dim", [8, 3])
def test_pages_append_odd_counts_lengths_and_tables(runtime, dim, layout):
    # Ends of tables, missing pages in the first place and later, rows at a page's edges, counts and lengths that are odd.
    rng = np.random.default_rng(20)
    lengths = [0.0, 15.0, 16.0, 17.0, 60.0, 64.0, 1e9, np.nan, -3.0, 31.5, 10.0, 10.0]
    counts = [0.0, 1.0, 20.0, 31.0, 20.0, 5.0, 5.0, 3.0, 2.9, 33.0, np.nan, 1e9]
    spec = append_spec(len(lengths), 2, 40, 16, 4, dim, layout)
    n = len(lengths) * 2 * 40 * dim
    x = {"k": normal(rng, n), "v": normal(rng, n), "counts": np.array(counts, np.float32),
         "tables": table_for(rng, spec, [64] * len(lengths)), "lengths": np.array(lengths, np.float32), **pools_for(rng, spec)}
    x["tables"][3, 2], x["tables"][7, 0], x["tables"][9, 3], x["tables"][11, 1] = -1, np.nan, spec["pages"], 1.5
    check_append(runtime, spec, x)


def test_pages_append_so_many_rows_that_they_are_counted_first(runtime):
    rng = np.random.default_rng(21)
    rows = 16 * 8200
    spec = append_spec(2, 1, rows, 16, 8300, 2, (True, True))
    assert runtime.compile(spec).launch["kernel"] == "pages_append_counted"
    x = {"k": normal(rng, 2 * rows * 2), "v": normal(rng, 2 * rows * 2), "counts": np.array([rows, rows], np.float32),
         "tables": table_for(rng, spec, [8300 * 16] * 2), "lengths": np.array([1000, 8300 * 16 - rows + 5], np.float32),
         **pools_for(rng, spec)}
    x["tables"][0, 5000] = -1
    got = run(runtime, spec, x)
    same(got["new_lengths"], np.array([80000, 8300 * 16], np.float32))
    for name in "kv":
        want = x[name + "_pages"].reshape(spec["pages"], 16, 2).copy()
        for b, (start, n) in enumerate(((1000, 79000), (8300 * 16 - rows + 5, rows - 5))):
            at = start + np.arange(n)
            want[x["tables"][b].astype(int)[at // 16], at % 16] = x[name].reshape(2, rows, 2)[b, :n]
        same(got[name + "_pages"], want)


# ---- pages_copy ----------------------------------------------------------------------------------------------

def copy_spec(copies, kv_heads, pages, page, dim, by_token):
    return {"op": "pages_copy", "copies": copies, "kv_heads": kv_heads, "pages": pages, "page": page, "dim": dim,
            "pages_token_major": by_token}


def check_copy(runtime, spec, sources, targets, rows, pools):
    x = {"sources": np.array(sources, np.float32), "targets": np.array(targets, np.float32), "copy_rows": np.array(rows, np.float32)}
    want = po.copy(spec, x["sources"], x["targets"], x["copy_rows"], pools["k_pages"], pools["v_pages"])
    got = run(runtime, spec, {**x, **pools}, 2)
    for name, y in zip(("k_pages", "v_pages"), want):
        same(po.pool_by_token(spec, got[name]), y)


@pytest.mark.parametrize("copies,kv_heads,page,dim", [(1, 1, 16, 1), (3, 8, 16, 128), (40, 3, 48, 40), (5, 2, 256, 7), (2, 1, 1024, 512),
                                                      (300, 2, 16, 64)])
@pytest.mark.parametrize("by_token", [True, False])
def test_pages_copy(runtime, copies, kv_heads, page, dim, by_token):
    rng = np.random.default_rng(copies)
    spec = copy_spec(copies, kv_heads, 2 * copies + 3, page, dim, by_token)
    order = rng.permutation(2 * copies + 3)
    rows = rng.integers(0, page + 1, copies)
    check_copy(runtime, spec, order[:copies], order[copies:2 * copies], rows, pools_for(rng, spec))


@pytest.mark.parametrize("by_token", [True, False])
def test_pages_copy_that_is_not_one_and_copies_that_meet(runtime, by_token):
    # Numbers that name no page, rows that are none or too many; a chain, a swap, a page copied to itself, one target twice,
    # a target that a copy without rows also names.
    rng = np.random.default_rng(30)
    copies = [(0, 1, 3), (-1, 2, 3), (3, np.nan, 3), (4, 40, 3), (5, 6, 0), (7, 8, 0.5), (9, 10, np.nan), (11, 12, 99), (13, 0.5, 1),
              (20, 21, 4), (21, 22, 4), (23, 24, 16), (24, 23, 16), (25, 25, 5), (26, 28, 2), (27, 28, 9), (29, 30, 0), (31, 30, 7),
              (32, 33, 2.7), (32, 34, 16), (32, 35, 1)]
    spec = copy_spec(len(copies), 2, 40, 16, 12, by_token)
    check_copy(runtime, spec, *zip(*copies), pools_for(rng, spec))


# ---- pages_fork ----------------------------------------------------------------------------------------------

def check_fork(runtime, spec, x, repeats=1):
    want = po.fork(spec, x["parents"], x["lengths"], x["tables"], x["reserve"], x["uses"])
    got = run(runtime, spec, {n: np.asarray(v, np.float32) for n, v in x.items()}, repeats)
    for name, y in want.items():
        np.testing.assert_array_equal(got[name].reshape(y.shape), y, err_msg=name)
    return want


def fork_state(rng, batch, page, table, pages, spare_pages=True):
    tables = np.full((batch, table), -1.0)
    order = list(rng.permutation(pages))
    lengths = rng.integers(0, table * page + 1, batch)
    uses = np.zeros(pages)
    for s in range(batch):
        held = min(table, -(-int(lengths[s]) // page) + (rng.random() < 0.4 if spare_pages else 0))
        share = 0
        if s and rng.random() < 0.5:  # the whole pages of the one before
            share = min(held, int(lengths[s - 1]) // page, int(lengths[s]) // page)
            tables[s, :share] = tables[s - 1, :share]
        for e in range(share, held):
            if not order:
                lengths[s] = min(lengths[s], e * page)
                break
            tables[s, e] = order.pop()
        for e in tables[s][tables[s] >= 0]:
            uses[int(e)] += 1
    return {"lengths": lengths, "tables": tables, "uses": uses}


@pytest.mark.parametrize("batch,page,table,pages", [(1, 16, 1, 1), (4, 16, 8, 40), (16, 48, 5, 60), (7, 16, 30, 150), (300, 16, 9, 3000),
                                                    (33, 1024, 3, 80), (5, 16, 300, 5000), (64, 32, 40, 1500),
                                                    (64, 16, 64, 8192), (64, 16, 65, 3000), (65, 16, 5, 300), (5, 16, 8, 8193), (3, 48, 2000, 5000)])
@pytest.mark.parametrize("reserve", [0, 1, 40])
def test_pages_fork(runtime, batch, page, table, pages, reserve):
    rng = np.random.default_rng(batch + pages + reserve)
    for _ in range(3):  # some of them run out of pages
        state = fork_state(rng, batch, page, table, pages)
        check_fork(runtime, {"op": "pages_fork", "batch": batch, "pages": pages, "page": page, "table": table},
                   {**state, "parents": rng.integers(-1, batch, batch), "reserve": np.full(batch, reserve)}, repeats=2)


@pytest.mark.parametrize("pages,kernel", [(64, "pages_fork_small"), (9000, "pages_fork")])
def test_pages_fork_odd_parents_lengths_tables_and_pinned_pages(runtime, pages, kernel):
    rng = np.random.default_rng(41)
    spec = {"op": "pages_fork", "batch": 8, "pages": pages, "page": 16, "table": 6}
    assert runtime.compile(spec).launch["kernel"] == kernel
    state = fork_state(rng, 8, 16, 6, pages)
    state["lengths"] = state["lengths"].astype(np.float32)
    state["uses"][:] += rng.integers(0, 2, pages)  # held by others too
    state["uses"][5] = np.nan
    for parents in ([0, 0, 0, 0, 0, 0, 0, 0], [-1, 8, np.nan, 0.5, np.inf, -0.0, 7, 1e9], [7, 6, 5, 4, 3, 2, 1, 0], [-1] * 8):
        check_fork(runtime, spec, {**state, "parents": np.array(parents, np.float32), "reserve": np.ones(8)})
    state["lengths"][:4] = [np.nan, 1e9, -1.0, 33.7]
    state["tables"][1, 1], state["tables"][2, 0], state["tables"][4, 2] = np.nan, pages, 1.5  # the pages after them are not held
    check_fork(runtime, spec, {**state, "parents": np.array([0, 1, 1, 2, 4, 4, 3, 3], np.float32),
                               "reserve": np.array([0, 1, np.nan, 1e9, 16, 17, -3, 2.5], np.float32)})


@pytest.mark.parametrize("pages", [4, 9000])
def test_pages_fork_without_free_pages(runtime, pages):
    # Three children of a sequence with a partial page, and one page to spare: the second child gets it, the third is cut
    # to its whole pages.
    spec = {"op": "pages_fork", "batch": 3, "pages": pages, "page": 16, "table": 4}
    want = check_fork(runtime, spec, {"parents": [0, 0, 0], "lengths": [40, 0, 0], "reserve": [1, 1, 1],
                                      "uses": [1, 1, 1, 0] + [1] * (pages - 4),
                                      "tables": [[2, 0, 1, -1], [-1] * 4, [-1] * 4]})
    assert want["new_lengths"].tolist() == [40, 40, 32] and want["missing"].tolist() == [0, 0, 1]
    assert want["targets"].tolist() == [-1, 3, -1] and want["sources"].tolist() == [-1, 1, -1]


def test_pages_fork_of_many_sequences_and_pages(runtime):
    rng = np.random.default_rng(42)
    batch, pages, table = 1000, 70000, 64
    state = fork_state(rng, batch, 16, table, pages)
    parents = np.where(rng.random(batch) < 0.1, -1, rng.integers(0, batch, batch))
    check_fork(runtime, {"op": "pages_fork", "batch": batch, "pages": pages, "page": 16, "table": table},
               {**state, "parents": parents, "reserve": rng.integers(0, 50, batch)})


# ---- beam_select ---------------------------------------------------------------------------------------------

def check_select(runtime, spec, logits, scores, finished):
    want, gap = po.select(spec, logits, scores, finished)
    # Beams are told apart by more than their scores may be off, before anything runs on the GPU.
    reach = np.abs(want["new_scores"][np.isfinite(want["new_scores"])]).max(initial=0)
    assert gap > 2 * po.score_bound(reach), gap
    got = run(runtime, spec, {"logits": logits, "scores": scores, "finished": finished}, 2)
    for name in ("parents", "tokens", "new_finished"):
        np.testing.assert_array_equal(got[name].reshape(want[name].shape), want[name], err_msg=name)
    there = want["new_scores"] > -np.inf
    new = got["new_scores"].reshape(there.shape).astype(np.float64)
    assert (new[~there] == -np.inf).all()
    finite = there & np.isfinite(want["new_scores"])
    assert (np.abs(new[finite] - want["new_scores"][finite]) <= po.score_bound(want["new_scores"][finite])).all()
    assert (new[there & ~finite] == want["new_scores"][there & ~finite]).all()


def select_spec(batch, beams, vocab, picks, end=2):
    return {"op": "beam_select", "batch": batch, "beams": beams, "vocab": vocab, "picks": picks, "end": end}


@pytest.mark.parametrize("batch,beams,vocab,picks", [
    (1, 1, 1, 1), (1, 1, 7, 5), (2, 3, 50, 6), (1, 4, 32000, 8), (3, 2, 1023, 64), (2, 5, 4097, 10), (1, 16, 8192, 32),
    (40, 4, 1000, 4), (1, 256, 300, 64), (5, 8, 50257, 16), (300, 2, 333, 3), (2, 2, 40000, 1), (70, 4, 9000, 8), (600, 1, 5000, 2)])
def test_beam_select(runtime, batch, beams, vocab, picks):
    rng = np.random.default_rng(vocab + picks)
    check_select(runtime, select_spec(batch, beams, vocab, picks), 3 * normal(rng, batch, beams, vocab),
                 (-10 * rng.random((batch, beams))).astype(np.float32), (rng.random((batch, beams)) < 0.2).astype(np.float32))


def test_beam_select_more_chunks_than_a_grid_has_blocks(runtime):
    rng = np.random.default_rng(54)
    batch, beams, picks = 65535, 17, 3
    logits, scores = normal(rng, batch, beams, 2), normal(rng, batch, beams)
    got = run(runtime, select_spec(batch, beams, 2, picks, 1), {"logits": logits, "scores": scores, "finished": np.zeros((batch, beams))})
    x = logits.astype(np.float64)
    every = (x - np.log(np.exp(x).sum(-1, keepdims=True)) + scores[..., None].astype(np.float64)).reshape(batch, -1)
    order = np.argsort(-every, axis=1, kind="stable")[:, :picks + 1]
    best = np.take_along_axis(every, order, 1)
    clear = (best[:, :-1] - best[:, 1:] > 2 * po.score_bound(10)).all(axis=1)
    assert clear.mean() > 0.99
    order = order[:, :picks]
    np.testing.assert_array_equal(got["parents"].reshape(batch, picks)[clear], (order // 2 + np.arange(batch)[:, None] * beams)[clear])
    np.testing.assert_array_equal(got["tokens"].reshape(batch, picks)[clear], (order % 2)[clear])
    assert (np.abs(got["new_scores"].reshape(batch, picks) - best[:, :picks]) <= po.score_bound(best[:, :picks])).all()


def test_beam_select_first_step_and_finished_beams(runtime):
    rng = np.random.default_rng(50)
    scores = np.array([[0, -np.inf, -np.inf, -np.inf], [-1, -2, -3, np.nan], [-np.inf] * 4, [-1.5, -0.25, -0.5, -7]], np.float32)
    finished = np.array([[0, 0, 0, 0], [0, 1, 0, 0], [0, 0, 1, 1], [2, 1, 0.5, 1]], np.float32)
    for end in (0, 99, 100, 2 ** 32 - 1):  # the last two end no beam, and a finished one does not go on
        check_select(runtime, select_spec(4, 4, 100, 8, end), normal(rng, 4, 4, 100), scores, finished)


@pytest.mark.parametrize("vocab", [500, 4099, 40000])
def test_beam_select_tokens_that_may_not_follow(runtime, vocab):
    # -inf, NaN and infinite logits; fewer tokens than picks; a beam without any.
    rng = np.random.default_rng(51)
    logits = normal(rng, 3, 3, vocab)
    logits[0][rng.random((3, vocab)) < 0.9] = -np.inf
    logits[1] = -np.inf
    logits[1, 0, [7, vocab - 1]], logits[1, 2, 3] = [1.0, 0.5], -2.0
    logits[2, 0, ::3], logits[2, 1, :] = np.nan, -np.inf
    logits[2, 2, [5, 400]] = np.inf  # they share what there is
    scores = np.array([[-1, -2, -3], [-1, -1, -5], [-4, -1, -2]], np.float32)
    check_select(runtime, select_spec(3, 3, vocab, 9), logits, scores, np.zeros((3, 3), np.float32))


@pytest.mark.parametrize("vocab,picks", [(100, 64), (5000, 7), (40000, 64)])
def test_beam_select_ties_go_to_the_lower_beam_then_token(runtime, vocab, picks):
    # Equal logits everywhere; few values, each of many tokens; the two beams' logits are the same.
    rng = np.random.default_rng(52)
    for rows in (np.zeros((2, 1, vocab)), rng.integers(0, 3, (2, 1, vocab)), -np.arange(vocab)[None, None].repeat(2, 0) / 64.0):
        logits = np.repeat(rows, 2, axis=1).astype(np.float32)
        spec = select_spec(2, 2, vocab, picks)
        scores = np.full((2, 2), -1.0, np.float32)
        want, _ = po.select(spec, logits, scores, np.zeros((2, 2)))
        got = run(runtime, spec, {"logits": logits, "scores": scores, "finished": np.zeros((2, 2))})
        for name in ("parents", "tokens"):
            same(got[name], want[name])


@pytest.mark.parametrize("scale", [1e-3, 30.0, 1e4])
def test_beam_select_flat_and_peaked_logits(runtime, scale):
    rng = np.random.default_rng(53)
    logits = (scale * rng.standard_normal((4, 3, 20000))).astype(np.float32)
    logits[3] += np.float32(1e4)
    check_select(runtime, select_spec(4, 3, 20000, 6), logits, (-5 * rng.random((4, 3))).astype(np.float32), np.zeros((4, 3), np.float32))


@pytest.mark.parametrize("batch,beams,vocab,picks", [(5, 4, 32000, 64), (2, 16, 20000, 32), (3, 16, 64, 64), (300, 2, 9100, 64), (1, 200, 4500, 64)])
def test_beam_select_one_beam_far_ahead(runtime, batch, beams, vocab, picks):
    # All that is chosen comes from one beam's lists, of fewer threads than are asked; sorted logits besides, where one
    # chunk has them all.
    rng = np.random.default_rng(55 + beams)
    logits = 3 * normal(rng, batch, beams, vocab)
    logits[0] = np.sort(logits[0], axis=-1)
    scores = np.full((batch, beams), -60.0, np.float32)
    scores[np.arange(batch), rng.integers(0, beams, batch)] = -1
    check_select(runtime, select_spec(batch, beams, vocab, picks), logits, scores, np.zeros((batch, beams), np.float32))


def test_beam_select_more_equal_lists_than_are_looked_at_at_once(runtime):
    spec = select_spec(1, 256, 5000, 64)
    logits, scores = np.zeros((1, 256, 5000), np.float32), np.full((1, 256), -2.0, np.float32)
    logits[0, 200:, 1::7] = 0.5
    want, _ = po.select(spec, logits, scores, np.zeros((1, 256)))
    got = run(runtime, spec, {"logits": logits, "scores": scores, "finished": np.zeros((1, 256))})
    for name in ("parents", "tokens"):
        same(got[name], want[name])
    logits[:] = 0
    want, _ = po.select(spec, logits, scores, np.zeros((1, 256)))
    got = run(runtime, spec, {"logits": logits, "scores": scores, "finished": np.zeros((1, 256))})
    for name in ("parents", "tokens"):
        same(got[name], want[name])


@pytest.mark.parametrize("vocab", [2048, 40000])
def test_beam_select_sums_of_tiny_terms_beside_large_ones(runtime, vocab):
    # Two beams of the same logits, 0 and -17, in another order, the second ahead by 1e-8. exp(0) is exact and exp(-17), off
    # by 4 U of its 4.1e-8, no matter; sums in 64 bits are good to 1e-12. Were neighbours added in 32 bits, the first beam's
    # sum would be short by 4.1e-8 of itself, and it ahead.
    logits = np.zeros((1, 2, vocab), np.float32)
    logits[0, 0, 1::2] = -17
    logits[0, 1, 2::4] = logits[0, 1, 3::4] = -17
    got = run(runtime, select_spec(1, 2, vocab, 3), {"logits": logits, "scores": np.array([0, 1e-8]), "finished": np.zeros(2)})
    same(got["parents"], np.array([1, 1, 1]))
    same(got["tokens"], np.array([0, 1, 4]))


@pytest.mark.parametrize("batch,page,table,pages", [(6, 16, 2100, 7000), (5, 1024, 4097, 9000), (2049, 16, 3, 4000), (2500, 48, 4, 6500),
                                                    (4097, 16, 2, 5500)])
def test_pages_fork_of_long_tables_and_large_batches(runtime, batch, page, table, pages):
    # Entries past those that a thread keeps in registers; needs past those that a block keeps in LDS.
    rng = np.random.default_rng(43)
    for reserve in (1, page * table):  # the second asks for whole tables
        state = fork_state(rng, batch, page, table, pages)
        check_fork(runtime, {"op": "pages_fork", "batch": batch, "pages": pages, "page": page, "table": table},
                   {**state, "parents": rng.integers(-1, batch, batch), "reserve": np.full(batch, reserve)}, repeats=2)


def test_pages_append_more_items_than_a_grid_has_blocks(runtime):
    # A row of each of 17 heads of 65535 sequences: blocks take a second item, of another sequence, after one whose table
    # has a page too few or none at all.
    rng = np.random.default_rng(22)
    spec = {"op": "pages_append", "batch": 65535, "kv_heads": 17, "rows": 1, "pages": 2 * 65535, "page": 16, "table": 2, "dim": 1,
            "token_major": False, "pages_token_major": True}
    assert 65535 * 17 > 2 ** 20
    n = 65535 * 17
    lengths = rng.integers(0, 33, 65535).astype(np.float32)
    tables = rng.permutation(2 * 65535).reshape(65535, 2).astype(np.float32)
    tables[::5, 0], tables[1::5, 1] = -1, np.nan
    counts = rng.integers(0, 3, 65535).astype(np.float32)
    x = {"k": normal(rng, n), "v": normal(rng, n), "counts": counts, "tables": tables, "lengths": lengths, **pools_for(rng, spec)}
    got = run(runtime, spec, x, 2)
    entry = np.take_along_axis(tables, np.minimum(lengths.astype(int)[:, None] // 16, 1), 1)[:, 0]
    made = (counts >= 1) & (lengths < 32) & (entry >= 0)
    same(got["new_lengths"], lengths + made)
    for name in "kv":
        want = x[name + "_pages"].reshape(-1, 16, 17).copy()
        want[entry[made].astype(int), lengths[made].astype(int) % 16] = x[name].reshape(65535, 17)[made]
        same(got[name + "_pages"], want)
