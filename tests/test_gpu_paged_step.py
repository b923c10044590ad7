"""A beam search over a paged cache as the documentation writes it: prompts in one chunk, forked to their beams, then steps of
append, attention, logits, selection, fork and copy, chained in one execute each, with every buffer taken into the next step.
Each stage against 64 bits of what the stage before it left, and the pages against plain lists of rows."""
import numpy as np
import pytest

import decoder_oracle as dec
import paged_oracle as po
import test_gpu_decoder as base

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", [(True, True), (True, False)])
@pytest.mark.parametrize("group,dim", [(2, 32), (1, 80)])
def test_the_documented_search(runtime, layout, group, dim):
    S, K, KV, page, table, vocab, end, steps = 3, 4, 2, 16, 5, 50, 7, 40
    B, H, pages = S * K, KV * group, 60
    rng = np.random.default_rng(90 + dim)
    rt = runtime
    pool = dict(kv_heads=KV, pages=pages, page=page, dim=dim, pages_token_major=layout[1])
    longest = 30
    first_append = rt.compile({"op": "pages_append", "batch": B, "rows": longest, **pool, "table": table, "token_major": layout[0]})
    first_attend = rt.compile({"op": "attention_paged", "batch": B, "heads": H, "queries": longest, **pool, "table": table,
                               "token_major": layout[0]})
    append = rt.compile({"op": "pages_append", "batch": B, "rows": 1, **pool, "table": table, "token_major": layout[0]})
    attend = rt.compile({"op": "attention_paged", "batch": B, "heads": H, "queries": 1, **pool, "table": table,
                         "token_major": layout[0]})
    project = rt.compile({"op": "gemm", "m": B, "n": vocab, "k": H * dim, "tiled": True})
    select = rt.compile({"op": "beam_select", "batch": S, "beams": K, "vocab": vocab, "picks": K, "end": end})
    fork = rt.compile({"op": "pages_fork", "batch": B, "pages": pages, "page": page, "table": table})
    copy = rt.compile({"op": "pages_copy", "copies": B, **pool})

    matrix = base.normal(rng, H * dim, vocab)
    weights = rt.resident(matrix)
    size = pages * page * KV * dim
    k_pages, v_pages = rt.alloc(size), rt.alloc(size)
    tables, new_tables, uses, new_uses = rt.alloc(B * table), rt.alloc(B * table), rt.alloc(pages), rt.alloc(pages)
    lengths, longer, ones = rt.alloc(B), rt.alloc(B), rt.resident(np.ones(B))
    parents, tokens, sources, targets, copy_rows, missing = (rt.alloc(B) for _ in range(6))
    scores, new_scores, finished, new_finished = rt.alloc(B), rt.alloc(B), rt.alloc(B), rt.alloc(B)
    logits, out = rt.alloc(B * vocab), rt.alloc(B * H * dim)

    def pages_of(b, n, get=None):
        """The keys and values of sequence b as its table names them."""
        get = get or rt.download(tables).reshape(B, table)[b]
        at = po.places(fork.spec, get, range(n))
        return [np.array([po.pool_by_token(copy.spec, rt.download(x))[p] for p in at]).reshape(n, KV, dim) for x in (k_pages, v_pages)]

    # Prompts of the first beam of every search: pages for them, then keys, values and attention in one chunk.
    prompt = [30, 16, 5]
    slots = [s * K for s in range(S)]
    count = np.zeros(B, np.float32)
    count[slots] = prompt
    rt.upload(tables, np.full(B * table, -1.0))
    rt.upload(parents, np.arange(B))
    reserve = rt.resident(count)
    chunk = {n: base.normal(rng, *base.shape_of(layout[0], B, h, longest, dim)) for n, h in (("q", H), ("k", KV), ("v", KV))}
    q, k, v = (rt.resident(chunk[n]) for n in "qkv")
    chunk_out = rt.alloc(B * H * longest * dim)
    rt.execute([(fork, [parents, lengths, tables, reserve, uses, new_tables, longer, new_uses, sources, targets, copy_rows, missing]),
                (first_append, [k, v, reserve, new_tables, longer, k_pages, v_pages, lengths]),
                (first_attend, [q, k_pages, v_pages, new_tables, lengths, reserve, chunk_out])], 1)
    tables, new_tables, uses, new_uses = new_tables, tables, new_uses, uses
    assert (rt.download(lengths) == count).all() and (rt.download(missing) == 0).all()
    want, off = po.paged(first_attend.spec, chunk["q"], rt.download(k_pages), rt.download(v_pages), rt.download(tables), count, count)
    base.within(po.rows_by_token(first_attend.spec, rt.download(chunk_out), H, longest), want, off)
    # Every sequence as plain rows, whoever holds them.
    rows = [[[], []] for _ in range(B)]
    for s, n in zip(slots, prompt):
        rows[s] = [list(dec.by_token(chunk[x], layout[0])[s, :n]) for x in "kv"]

    # Every beam goes on from its search's first; only that one has a score, so the first selection is among its tokens.
    rt.upload(parents, np.repeat(slots, K))
    rt.upload(reserve, np.ones(B))
    rt.execute([(fork, [parents, lengths, tables, reserve, uses, new_tables, longer, new_uses, sources, targets, copy_rows, missing]),
                (copy, [sources, targets, copy_rows, k_pages, v_pages])], 1)
    tables, new_tables, uses, new_uses, lengths, longer = new_tables, tables, new_uses, uses, longer, lengths
    rows = [[list(x) for x in rows[s]] for s in np.repeat(slots, K)]
    rt.upload(scores, np.where(np.arange(B) % K == 0, 0.0, -np.inf))

    chosen, copied = 0, 0
    for step in range(steps):
        new = {n: base.normal(rng, *base.shape_of(layout[0], B, h, 1, dim)) for n, h in (("q", H), ("k", KV), ("v", KV))}
        q1, k1, v1 = (rt.resident(new[n]) for n in "qkv")
        was = {n: rt.download(x) for n, x in (("tables", tables), ("lengths", lengths), ("uses", uses), ("scores", scores),
                                              ("finished", finished))}
        rt.execute([(append, [k1, v1, ones, tables, lengths, k_pages, v_pages, longer]),
                    (attend, [q1, k_pages, v_pages, tables, longer, ones, out]),
                    (project, [out, weights, logits]),
                    (select, [logits, scores, finished, parents, tokens, new_scores, new_finished])], 1)
        now = rt.download(longer)
        for b in range(B):
            if was["lengths"][b] < table * page and rows[b][0]:
                for x, y in zip(rows[b], (new["k"], new["v"])):
                    x.append(dec.by_token(y, layout[0])[b, 0])
            assert now[b] == len(rows[b][0])
        want, off = po.paged(attend.spec, new["q"], rt.download(k_pages), rt.download(v_pages), was["tables"], now, np.ones(B))
        got = rt.download(out)
        base.within(po.rows_by_token(attend.spec, got, H, 1), want, off)
        a, m = got.reshape(B, H * dim).astype(np.float64), matrix.astype(np.float64)
        got_logits = rt.download(logits)
        base.within(got_logits, a @ m, (H * dim + 2) * dec.U * (np.abs(a) @ np.abs(m)))
        want, gap = po.select(select.spec, got_logits, was["scores"], was["finished"])
        picked = {n: rt.download(x).reshape(S, K) for n, x in (("parents", parents), ("tokens", tokens), ("new_scores", new_scores),
                                                               ("new_finished", new_finished))}
        reach = np.abs(want["new_scores"][np.isfinite(want["new_scores"])]).max()
        there = want["new_scores"] > -np.inf
        assert (np.abs(picked["new_scores"][there] - want["new_scores"][there]) <= po.score_bound(reach)).all()
        if gap > 2 * po.score_bound(reach):
            chosen += 1
            for n in ("parents", "tokens", "new_finished"):
                assert (picked[n] == want[n]).all(), n

        rt.execute([(fork, [parents, longer, tables, reserve, uses, new_tables, lengths, new_uses, sources, targets, copy_rows, missing]),
                    (copy, [sources, targets, copy_rows, k_pages, v_pages])], 1)
        want = po.fork(fork.spec, picked["parents"].reshape(-1), now, was["tables"], np.ones(B), was["uses"])
        for n, x in (("new_tables", new_tables), ("new_lengths", lengths), ("new_uses", new_uses), ("sources", sources),
                     ("targets", targets), ("copy_rows", copy_rows), ("missing", missing)):
            assert (rt.download(x).reshape(want[n].shape) == want[n]).all(), n
        copied += int((want["copy_rows"] > 0).sum())
        tables, new_tables, uses, new_uses = new_tables, tables, new_uses, uses
        scores, new_scores, finished, new_finished = new_scores, scores, new_finished, finished
        rows = [[list(x) for x in rows[int(p)]] if p >= 0 else [[], []] for p in picked["parents"].reshape(-1)]
        if step % 5 == 4:
            for b in range(B):
                for got, want in zip(pages_of(b, len(rows[b][0])), rows[b]):
                    assert (got == np.array(want).reshape(got.shape)).all()
        for x in (q1, k1, v1):
            x.free()
    assert chosen > steps * 3 // 4 and copied > steps  # the search did branch
    for x in (weights, k_pages, v_pages, tables, new_tables, uses, new_uses, lengths, longer, ones, parents, tokens, sources, targets,
              copy_rows, missing, scores, new_scores, finished, new_finished, logits, out, q, k, v, chunk_out, reserve):
        x.free()
