"""Decoding over a paged cache in 64 bits, in numpy and plain lists, with bounds on what FP32 may be off (U is half an
ulp of it)."""
import numpy as np

from decoder_oracle import U, attend, by_token, length_of


def whole(x, most):
    """A whole number of 0 .. most - 1, or None."""
    x = np.float32(x)
    return int(x) if 0 <= x < most and x == np.trunc(x) else None


def pool_by_token(spec, pool):
    """[pages, page, kv heads, dim], whatever the layout."""
    shape = [spec["pages"], spec["page"], spec["kv_heads"], spec["dim"]]
    if not spec["pages_token_major"]:
        shape = [shape[0], shape[2], shape[1], shape[3]]
    return by_token(pool.reshape(shape), spec["pages_token_major"])


def rows_by_token(spec, x, heads, rows):
    shape = (spec["batch"], rows, heads, spec["dim"]) if spec["token_major"] else (spec["batch"], heads, rows, spec["dim"])
    return by_token(x.reshape(shape), spec["token_major"])


def places(spec, table, tokens):
    """(page, row) of each of `tokens`; None where the table has no page."""
    got = []
    for t in tokens:
        page = whole(table[t // spec["page"]], spec["pages"]) if t < spec["table"] * spec["page"] else None
        got.append(None if page is None else (page, t % spec["page"]))
    return got


def paged(spec, q, k_pages, v_pages, tables, lengths, counts):
    """attention_paged: outputs by token, and how far FP32 may be off."""
    q = rows_by_token(spec, q.astype(np.float64), spec["heads"], spec["queries"])
    k, v = (pool_by_token(spec, x.astype(np.float64)) for x in (k_pages, v_pages))
    out, off = np.zeros_like(q), np.zeros_like(q)
    group = spec["heads"] // spec["kv_heads"]
    tables = np.asarray(tables).reshape(spec["batch"], spec["table"])
    for b in range(spec["batch"]):
        length = length_of(lengths[b], spec["table"] * spec["page"])
        count = length_of(counts[b], spec["queries"])
        at = places(spec, tables[b], range(length))
        tokens = [t for t in range(length) if at[t] is not None]
        pages, rows = [at[t][0] for t in tokens], [at[t][1] for t in tokens]
        for h in range(spec["heads"]):
            keys, values = k[pages, rows, h // group], v[pages, rows, h // group]
            for i in range(count):
                sees = [n for n, t in enumerate(tokens) if t <= length - count + i]
                out[b, i, h], off[b, i, h] = attend(q[b, i, h], keys, values, sees)
    return out, off


def append(spec, k, v, counts, tables, lengths, k_pages, v_pages):
    """pages_append: both pools by token, and the new lengths."""
    pools = [pool_by_token(spec, x.copy()).copy() for x in (k_pages, v_pages)]
    new = np.zeros(spec["batch"], np.float32)
    tables = np.asarray(tables).reshape(spec["batch"], spec["table"])
    for b in range(spec["batch"]):
        at = length_of(lengths[b], spec["table"] * spec["page"])
        for i in range(length_of(counts[b], spec["rows"])):
            place = places(spec, tables[b], [at])[0]
            if place is None:
                break
            for pool, rows in zip(pools, (k, v)):
                pool[place] = rows_by_token(spec, rows, spec["kv_heads"], spec["rows"])[b, i]
            at += 1
        new[b] = at
    return pools[0], pools[1], new


def fork(spec, parents, lengths, tables, reserve, uses):
    """pages_fork, in plain lists."""
    batch, page, table, pages = (spec[n] for n in ("batch", "page", "table", "pages"))
    old, length = [], []
    for row, n in zip(np.asarray(tables).reshape(batch, table), lengths):
        held = []
        for e in row:
            p = whole(e, pages)
            if p is None:
                break
            held.append(p)
        old.append(held)
        length.append(min(length_of(n, table * page), len(held) * page))
    uses = [float(u) for u in uses]
    new, ends, copies = [[] for _ in range(batch)], [0] * batch, {}
    parents = [whole(p, batch) for p in parents]
    for s, p in enumerate(parents):
        if p is None:
            continue
        full = length[p] // page
        ends[s] = length[p]
        if s == parents.index(p):
            new[s] = list(old[p])
        else:
            new[s] = old[p][:full]
            if length[p] % page:
                copies[s] = old[p][full]
    for rows, sign in ((old, -1), (new, 1)):
        for row in rows:
            for e in row:
                uses[e] += sign
    free = [p for p, u in enumerate(uses) if u == 0]
    missing, moves = [0] * batch, [(-1, -1, 0)] * batch
    for s, p in enumerate(parents):
        if p is None:
            continue
        want = min(table, -(-(length[p] + length_of(reserve[s], table * page)) // page))
        kept = len(new[s])
        while len(new[s]) < want and free:
            uses[free[0]] = 1
            new[s].append(free.pop(0))
        missing[s] = max(0, want - len(new[s]))
        if s in copies:
            if len(new[s]) > kept:
                moves[s] = (copies[s], new[s][kept], length[p] % page)
            else:
                ends[s] = kept * page
    return {"new_tables": np.array([row + [-1] * (table - len(row)) for row in new], np.float32),
            "new_lengths": np.array(ends, np.float32), "new_uses": np.array(uses, np.float32),
            "sources": np.array([m[0] for m in moves], np.float32), "targets": np.array([m[1] for m in moves], np.float32),
            "copy_rows": np.array([m[2] for m in moves], np.float32), "missing": np.array(missing, np.float32)}


def copy(spec, sources, targets, copy_rows, k_pages, v_pages):
    """pages_copy: both pools by token."""
    was = [pool_by_token(spec, x) for x in (k_pages, v_pages)]
    pools = [x.copy() for x in was]
    made = [(whole(s, spec["pages"]), whole(t, spec["pages"]), length_of(n, spec["page"]))
            for s, t, n in zip(sources, targets, copy_rows)]
    named = [m for m in made if None not in m and m[2]]
    seen = set()
    for m in named:
        if all(m[1] != other[0] for other in named) and m[1] not in seen:
            for pool, old in zip(pools, was):
                pool[m[1], :m[2]] = old[m[0], :m[2]]
        seen.add(m[1])
    return pools[0], pools[1]


# Every term of a beam's sum of exponentials is off by an ulp of exp2 (2 U), a rounding where its argument's rest comes
# in and one of that rest: 4 U of the sum, and as much of its logarithm's value. The score is rounded once.
def score_bound(scores):
    return 4 * U + U * np.abs(scores)


def select(spec, logits, scores, finished):
    """beam_select: the outputs, and the least distance between two of the search's best that come of different beams
    (order and choice are theirs to the last bit only where that is more than the scores may be off)."""
    batch, beams, vocab, picks, end = (spec[n] for n in ("batch", "beams", "vocab", "picks", "end"))
    out = {"parents": np.full((batch, picks), -1.0), "tokens": np.full((batch, picks), -1.0),
           "new_scores": np.full((batch, picks), -np.inf), "new_finished": np.zeros((batch, picks))}
    gap = np.inf
    logits = logits.reshape(batch, beams, vocab).astype(np.float64)
    scores, finished = (x.reshape(batch, beams).astype(np.float64) for x in (scores, finished))
    for b in range(batch):
        every = np.full((beams, vocab), -np.inf)
        for n in range(beams):
            if not scores[b, n] > -np.inf:
                continue
            if finished[b, n] > 0:
                if end < vocab:
                    every[n, end] = scores[b, n]
                continue
            x = np.where(np.isnan(logits[b, n]), -np.inf, logits[b, n])
            top = x.max()
            if top == -np.inf:
                continue
            with np.errstate(invalid="ignore"):
                below = np.where(x == top, 0.0, x - top)
            every[n] = below - np.log(np.exp(below).sum()) + scores[b, n]
        flat = every.reshape(-1)
        order = np.lexsort((np.arange(flat.size), -flat))[:picks + 1]
        best = flat[order]
        for x, y, i, j in zip(best, best[1:], order, order[1:]):
            if i // vocab != j // vocab and y > -np.inf:
                gap = min(gap, x - y)
        for r, i in enumerate(order[:picks]):
            if flat[i] == -np.inf:
                break
            n, token = divmod(int(i), vocab)
            out["parents"][b, r], out["tokens"][b, r], out["new_scores"][b, r] = b * beams + n, token, flat[i]
            out["new_finished"][b, r] = token == end or finished[b, n] > 0
    return out, gap
