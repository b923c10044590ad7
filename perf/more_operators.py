"""The operators of decoding over a paged cache as cases that can be timed and compared.

Five operators, in the order in which a step uses them:
  beam_select     the best continuations of every beam: scores plus log-probabilities over beams and vocabulary
  pages_fork      the sequences that a selection leaves: tables of pages forked, freed and made longer
  pages_copy      the last page of a forked sequence, which its continuations fill differently
  pages_append    new keys and values into the pages of their sequences
  attention_paged attention of a chunk of new tokens of every sequence over its pages (one token: decoding)

With `own` false a pass computes the operator's plain form in torch; with `own` true it is one
`HipRuntime.execute` call over resident buffers, the way `tests/` and `bench.py` drive the library.
FP32 throughout; it is the only data type the framework takes. Lengths, counts, tables, parents and tokens are whole
numbers held as FP32 values.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

# No listed case costs more; a drawn one costs no more either.
MOST_FLOPS = 1.5e11
MOST_BYTES = 1.1e9
MOST_PAIRS = 6e8  # (query, key) pairs: the plain forms hold a score of each


def listed():
    return [
        # One token of one sequence of a small model: latency counts.
        {"name": "paged_single", "kind": "attention_paged", "batch": 1, "heads": 8, "kv_heads": 8, "queries": 1,
         "keys": 1000, "page": 16, "dim": 64, "token_major": False, "pages_token_major": False, "spread": 0.0,
         "counts": "all"},
        # A decode step of a server: sequences of unlike lengths.
        {"name": "paged_step", "kind": "attention_paged", "batch": 16, "heads": 32, "kv_heads": 8, "queries": 1,
         "keys": 8192, "page": 16, "dim": 128, "token_major": True, "pages_token_major": True, "spread": 0.5,
         "counts": "all"},
        # Continuous batching: prompts' chunks beside sequences that decode.
        {"name": "paged_mixed", "kind": "attention_paged", "batch": 8, "heads": 24, "kv_heads": 24, "queries": 200,
         "keys": 4096, "page": 48, "dim": 80, "token_major": True, "pages_token_major": False, "spread": 0.5,
         "counts": "mixed"},
        # A chunk of a long prompt, grouped heads.
        {"name": "paged_chunk", "kind": "attention_paged", "batch": 1, "heads": 32, "kv_heads": 8, "queries": 512,
         "keys": 16384, "page": 64, "dim": 128, "token_major": True, "pages_token_major": True, "spread": 0.0,
         "counts": "all"},
        # The new tokens of a decode step of 64 sequences: next to no work.
        {"name": "append_token", "kind": "pages_append", "batch": 64, "kv_heads": 8, "rows": 1, "keys": 4096, "page": 16,
         "dim": 128, "token_major": True, "pages_token_major": True, "spread": 0.75, "counts": "all"},
        # Four prompts of 4096 tokens, from the projection's layout to pages by head.
        {"name": "append_prompts", "kind": "pages_append", "batch": 4, "kv_heads": 8, "rows": 4096, "keys": 6000,
         "page": 64, "dim": 128, "token_major": True, "pages_token_major": False, "spread": 0.25, "counts": "all"},
        # One beam search of four beams.
        {"name": "fork_beams", "kind": "pages_fork", "batch": 4, "beams": 4, "page": 16, "table": 64, "reserve": 1,
         "spare": 64},
        # 64 searches of eight beams over long contexts.
        {"name": "fork_many", "kind": "pages_fork", "batch": 512, "beams": 8, "page": 16, "table": 2048, "reserve": 1,
         "spare": 65536},
        # The partial pages of a few forks.
        {"name": "copy_beams", "kind": "pages_copy", "batch": 4, "kv_heads": 8, "page": 16, "dim": 128,
         "pages_token_major": True, "spare": 250},
        # Those of many, of large pages.
        {"name": "copy_many", "kind": "pages_copy", "batch": 448, "kv_heads": 8, "page": 256, "dim": 128,
         "pages_token_major": False, "spare": 64},
        # One search of four beams.
        {"name": "beams_one", "kind": "beam_select", "batch": 1, "beams": 4, "vocab": 32000, "picks": 8, "end": 2},
        # 64 searches of eight beams over a large vocabulary of odd size.
        {"name": "beams_many", "kind": "beam_select", "batch": 64, "beams": 8, "vocab": 131071, "picks": 16, "end": 2},
    ]


def _size(rng, low, high):
    """A size spread over the logarithm of [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    while True:
        kind = rng.choice(["attention_paged"] * 4 + ["pages_append", "pages_fork", "pages_copy"] + ["beam_select"] * 2)
        page = 16 * rng.choice([1, 1, 1, 2, 3, 4, 4, 8, 16, rng.randint(1, 16)])
        kv_heads, group = _size(rng, 1, 32), rng.choice([1, 1, 2, 4, 8])
        dim = rng.choice([32, 40, 64, 64, 80, 96, 128, 128, 128, rng.randint(3, 128)])
        layout = {"token_major": rng.random() < 0.7, "pages_token_major": rng.random() < 0.5}
        if kind == "attention_paged":
            queries = 1 if rng.random() < 0.4 else _size(rng, 2, 2048)
            case = {"kind": kind, "batch": _size(rng, 1, 64), "heads": kv_heads * group, "kv_heads": kv_heads,
                    "queries": queries, "keys": queries + _size(rng, 1, 65536) - 1, "page": page, "dim": dim, **layout,
                    "spread": rng.choice([0.0, 0.5, 1.0]), "counts": rng.choice(["all", "mixed"])}
        elif kind == "pages_append":
            rows = 1 if rng.random() < 0.3 else _size(rng, 2, 8192)
            case = {"kind": kind, "batch": _size(rng, 1, 64), "kv_heads": kv_heads, "rows": rows,
                    "keys": rows + _size(rng, 1, 8192) - 1, "page": page, "dim": dim, **layout,
                    "spread": rng.choice([0.0, 0.5, 1.0]), "counts": rng.choice(["all", "mixed"])}
        elif kind == "pages_fork":
            beams = rng.choice([1, 2, 4, 5, 8, 16])
            case = {"kind": kind, "batch": beams * _size(rng, 1, 128), "beams": beams, "page": page,
                    "table": _size(rng, 2, 4096), "reserve": rng.choice([0, 1, 1, 1, 5, 64]),
                    "spare": rng.choice([0, _size(rng, 1, 100000)])}
        elif kind == "pages_copy":
            case = {"kind": kind, "batch": _size(rng, 1, 1024), "kv_heads": kv_heads, "page": page, "dim": dim,
                    "pages_token_major": layout["pages_token_major"], "spare": _size(rng, 1, 1024)}
        else:
            beams = rng.choice([1, 2, 3, 4, 5, 8, 8, 16])
            vocab = rng.choice([32000, 50257, 131072, _size(rng, 40, 200000)])
            case = {"kind": kind, "batch": _size(rng, 1, 64), "beams": beams, "vocab": vocab,
                    "picks": min(64, rng.choice([beams, 2 * beams, _size(rng, 1, 64)])),
                    "end": rng.choice([0, 2, vocab - 1, vocab])}
        cost = work(case)
        if (cost["flops"] <= MOST_FLOPS and cost["bytes"] <= MOST_BYTES and _footprint(case) <= 2 * MOST_BYTES
                and _pairs(case) <= MOST_PAIRS):
            return case


def _pairs(case):
    if case["kind"] != "attention_paged":
        return 0
    return case["batch"] * case["heads"] * case["queries"] * case["keys"]


def _table(case):
    """Entries of a sequence's table: enough for its longest."""
    return case["table"] if "table" in case else -(-case["keys"] // case["page"])


def _pages(case):
    """Pages of the pool: those in use and some to spare."""
    if case["kind"] == "pages_copy":
        return 2 * case["batch"] + case["spare"]
    if case["kind"] == "pages_fork":
        return case["batch"] * (case["table"] * 5 // 8 + 2) + case["spare"]
    return sum(-(-n // case["page"]) for n in _ends(case)) + 8


def _footprint(case):
    """Bytes of the tensors a case holds, the unused parts of its pools among them; the plain forms hold every key of
    the batch padded to the longest."""
    if case["kind"] in ("pages_fork", "beam_select"):
        return work(case)["bytes"] * (1 if case["kind"] == "pages_fork" else 3)
    pool = 8 * _pages(case) * case["page"] * case["kv_heads"] * case["dim"]
    if case["kind"] == "attention_paged":
        pool = max(pool, 8 * case["batch"] * case["kv_heads"] * case["keys"] * case["dim"])
    return pool + work(case)["bytes"]


# ---- whole-number inputs that the work depends on: they follow from the case alone ----------------------------------

def _new(case):
    """New tokens of each sequence: as many as fit, or prompts' chunks beside single tokens and parts of chunks; with
    the whole spread one sequence has none."""
    most = case["queries" if case["kind"] == "attention_paged" else "rows"]
    got = [most] * case["batch"]
    if case["counts"] == "mixed":
        got = [(most, 1, 1, max(1, most // 3))[b % 4] for b in range(case["batch"])]
    if case["spread"] == 1.0 and case["batch"] > 1:
        got[-1] = 0
    return got


def _ends(case):
    """Length of each sequence, its new tokens among them: from all the keys down to the share that `spread` leaves, in
    no order."""
    return [max(n, int(round(case["keys"] * (1.0 - case["spread"] * ((0.618034 * b) % 1.0)))))
            for b, n in enumerate(_new(case))]


def _copy_rows(case):
    """Rows of each copied page: all counts in turn, one copy in eight is not to be made."""
    return [0 if i % 8 == 5 else (i * 7) % case["page"] + 1 for i in range(case["batch"])]


def _rows_shape(case, heads, rows):
    if case["token_major"]:
        return (case["batch"], rows, heads, case["dim"])
    return (case["batch"], heads, rows, case["dim"])


def _pool_shape(case):
    if case["pages_token_major"]:
        return (_pages(case), case["page"], case["kv_heads"], case["dim"])
    return (_pages(case), case["kv_heads"], case["page"], case["dim"])


def _fork_inputs(case, g):
    """Searches of `beams` sequences that share the pages of a prompt and have later ones of their own, some of them
    with a page in hand; a selection of parents; the uses that follow."""
    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    batch, beams, page, table = case["batch"], case["beams"], case["page"], case["table"]
    lead = torch.arange(batch, device="cuda") // beams * beams
    most = max(1, table * page - case["reserve"])
    # A search's sequences are about as long as one another; the shared part ends with a whole page.
    base = (uniform(batch) * most / 2)[lead]
    lengths = (base + uniform(batch) * (most / 8)).long().clamp(1, most)
    held = (lengths + page - 1) // page + (uniform(batch) < 0.3).long()
    held = held.clamp(max=table)
    shared = (base * 0.75).long() // page
    shared = torch.minimum(shared, lengths // page)
    shared = torch.stack([shared.view(-1, beams).amin(dim=1)] * beams, dim=1).view(-1)
    own_pages = torch.where(lead == torch.arange(batch, device="cuda"), held, held - shared)
    start = own_pages.cumsum(0) - own_pages
    at = torch.arange(table, device="cuda").unsqueeze(0)
    first = lead == torch.arange(batch, device="cuda")
    place = torch.where(at < shared.unsqueeze(1), start[lead].unsqueeze(1) + at,
                        (start + torch.where(first, 0, -shared)).unsqueeze(1) + at)
    order = torch.randperm(_pages(case), generator=g, device="cuda")
    here = at < held.unsqueeze(1)
    tables = torch.where(here, order[torch.where(here, place, 0)], -1)
    uses = torch.zeros(_pages(case), device="cuda").index_add_(0, tables[here], torch.ones((), device="cuda").expand(int(here.sum())))
    parents = lead + (uniform(batch).square() * beams).long().clamp(max=beams - 1)
    parents = torch.where(uniform(batch) < 0.05, -1, parents)  # a search that has ended
    return {"parents": parents.float(), "lengths": lengths.float(), "tables": tables.float(),
            "reserve": torch.full((batch,), float(case["reserve"]), device="cuda"), "uses": uses}


def _inputs(case, seed):
    """The case's operands, made on the GPU from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, batch = case["kind"], case["batch"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def numbers(values):
        return torch.tensor(values, dtype=torch.float32, device="cuda")

    if kind == "beam_select":
        logits = 3 * normal(batch, case["beams"], case["vocab"])
        logits[torch.rand(logits.shape, generator=g, device="cuda") < 0.01] = -math.inf  # tokens that may not follow
        scores = -20 * torch.rand(batch, case["beams"], generator=g, device="cuda")
        finished = (torch.rand(batch, case["beams"], generator=g, device="cuda") < 0.1).float()
        return {"logits": logits, "scores": scores, "finished": finished}
    if kind == "pages_fork":
        return _fork_inputs(case, g)
    pool = _pool_shape(case)
    order = torch.randperm(_pages(case), generator=g, device="cuda")
    if kind == "pages_copy":
        rows = numbers(_copy_rows(case))
        targets = torch.where(rows > 0, order[batch:2 * batch], -1)
        return {"sources": order[:batch].float(), "targets": targets.float(), "copy_rows": rows,
                "k_pages": normal(*pool), "v_pages": normal(*pool)}
    ends, new = _ends(case), _new(case)
    tables = torch.full((batch, _table(case)), -1.0, device="cuda")
    start = 0
    for b, n in enumerate(ends):
        held = -(-n // case["page"])
        tables[b, :held] = order[start:start + held].float()
        start += held
    whole = {"tables": tables, "counts": numbers(new)}
    if kind == "pages_append":
        rows = _rows_shape(case, case["kv_heads"], case["rows"])
        return {"k": normal(*rows), "v": normal(*rows), **whole, "lengths": numbers([e - n for e, n in zip(ends, new)]),
                "k_pages": normal(*pool), "v_pages": normal(*pool)}
    return {"q": normal(*_rows_shape(case, case["heads"], case["queries"])), "k_pages": normal(*pool),
            "v_pages": normal(*pool), **whole, "lengths": numbers(ends)}


# ---- the framework's calls ---------------------------------------------------------------------------------

class _Memory:
    """A runtime buffer as torch sees it: a view, no copy."""

    def __init__(self, buffer, shape):
        self.buffer = buffer  # keeps the runtime alive with the view
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": "<f4", "data": (buffer.ptr, False),
                                         "version": 2}


def _view(buffer, shape):
    return torch.as_tensor(_Memory(buffer, shape), device="cuda")


def _spec(case):
    kind = case["kind"]
    names = {"attention_paged": ("batch", "heads", "kv_heads", "queries", "page", "dim", "token_major",
                                 "pages_token_major"),
             "pages_append": ("batch", "kv_heads", "rows", "page", "dim", "token_major", "pages_token_major"),
             "pages_fork": ("batch", "page"),
             "pages_copy": ("kv_heads", "page", "dim", "pages_token_major"),
             "beam_select": ("batch", "beams", "vocab", "picks", "end")}[kind]
    spec = {"op": kind, **{name: case[name] for name in names}}
    if kind == "pages_copy":
        spec["copies"] = case["batch"]
    elif kind != "beam_select":
        spec["table"] = _table(case)
    if kind != "beam_select":
        spec["pages"] = _pages(case)
    return spec


def _outputs(case):
    """Names and shapes of the outputs, in the order of the bindings."""
    kind, batch = case["kind"], case["batch"]
    if kind == "attention_paged":
        return {"out": _rows_shape(case, case["heads"], case["queries"])}
    if kind == "beam_select":
        return {name: (batch, case["picks"]) for name in ("parents", "tokens", "new_scores", "new_finished")}
    if kind == "pages_fork":
        return {"new_tables": (batch, case["table"]), "new_lengths": (batch,), "new_uses": (_pages(case),),
                "sources": (batch,), "targets": (batch,), "copy_rows": (batch,), "missing": (batch,)}
    pools = {"k_pages": _pool_shape(case), "v_pages": _pool_shape(case)}
    return pools if kind == "pages_copy" else {**pools, "new_lengths": (batch,)}


def prepare(case, seed):
    inputs = _inputs(case, seed)
    if not own:
        return {"case": case, "inputs": inputs}
    # The framework's kernels take buffers of its own runtime and a compiled kernel; a user's program keeps both.
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "jade-compute_amd"))
    import jade_hip

    runtime = jade_hip.HipRuntime(0)
    buffers, outputs = {}, {}
    for name, value in inputs.items():
        buffers[name] = runtime.alloc(value.numel())
        _view(buffers[name], value.shape).copy_(value)
    for name, shape in _outputs(case).items():
        if name not in buffers:  # the pools are read and written
            buffers[name] = runtime.alloc(math.prod(shape))
        outputs[name] = _view(buffers[name], shape)
    kernel = runtime.compile(_spec(case))
    torch.cuda.synchronize()  # the operands are in place before the runtime's own queue reads them
    return {"runtime": runtime, "jobs": [(kernel, [buffers[b["name"]] for b in kernel.bindings])], "outputs": outputs}


# ---- the plain forms -----------------------------------------------------------------------------------------

def _select(case, x):
    """Scores in 64 bits: beams are compared with one another by them."""
    batch, vocab, picks = case["batch"], case["vocab"], case["picks"]
    logits = x["logits"].double()
    top = logits.amax(dim=-1, keepdim=True)
    total = (logits - top).exp_().sum(dim=-1, keepdim=True).log_().add_(top)
    every = logits.sub_(total).add_(x["scores"].double().unsqueeze(-1))
    done = (x["finished"] > 0).unsqueeze(-1)
    every.masked_fill_(done, -math.inf)
    if case["end"] < vocab:
        every[..., case["end"]] = torch.where(done[..., 0], x["scores"].double(), every[..., case["end"]])
    values, at = every.view(batch, -1).topk(min(picks, case["beams"] * vocab), dim=-1)
    at, order = at.sort(dim=-1)
    values, order = values.gather(1, order).sort(dim=-1, descending=True, stable=True)
    at = at.gather(1, order)
    there = values > -math.inf
    beam, token = at // vocab, at % vocab
    first = torch.arange(batch, device=at.device).unsqueeze(1) * case["beams"]
    out = {"parents": torch.where(there, first + beam, -1).float(), "tokens": torch.where(there, token, -1).float(),
           "new_scores": values.float(),
           "new_finished": (there & ((token == case["end"]) | (x["finished"].gather(1, beam) > 0))).float()}
    short = picks - at.shape[1]
    if short:
        for name, value in (("parents", -1.0), ("tokens", -1.0), ("new_scores", -math.inf), ("new_finished", 0.0)):
            out[name] = torch.cat([out[name], torch.full((batch, short), value, device=at.device)], dim=1)
    return out


def _fork(case, x):
    batch, page, table = case["batch"], case["page"], case["table"]
    at = torch.arange(table, device="cuda").unsqueeze(0)
    tables, lengths = x["tables"].long(), x["lengths"].long()
    held = (tables >= 0).long().cumprod(dim=1).sum(dim=1)
    lengths = torch.minimum(lengths, held * page)
    full, part = lengths // page, lengths % page
    live = x["parents"] >= 0
    parent = x["parents"].long().clamp_min(0)
    # The first child of a parent keeps what it does not share.
    lowest = torch.full((batch,), batch, device="cuda").scatter_reduce_(
        0, parent, torch.where(live, torch.arange(batch, device="cuda"), batch), "amin")
    first = lowest[parent] == torch.arange(batch, device="cuda")
    keep = torch.where(live, torch.where(first, held[parent], full[parent]), 0)
    kept = at < keep.unsqueeze(1)
    new = torch.where(kept, tables[parent], -1)
    pool = x["uses"].numel()
    uses = (x["uses"] - torch.bincount(tables[at < held.unsqueeze(1)], minlength=pool)
            + torch.bincount(new[kept], minlength=pool))
    # Free pages in order of their number, given out in order of slots and places.
    want = ((lengths[parent] + x["reserve"].long() + page - 1) // page).clamp_max(table)
    need = torch.where(live, (want - keep).clamp_min(0), 0)
    before = need.cumsum(0) - need
    free = uses == 0
    rank = free.long().cumsum(0) - 1
    total = rank[-1] + 1
    pages = torch.full((pool + 1,), -1, device="cuda").scatter_(
        0, torch.where(free, rank, pool), torch.arange(pool, device="cuda"))
    pages[-1] = -1
    asked = before.unsqueeze(1) + at - keep.unsqueeze(1)
    given = (at >= keep.unsqueeze(1)) & (at < (keep + need).unsqueeze(1)) & (asked < total)
    new = torch.where(given, pages[torch.where(given, asked, 0)], new)
    uses = uses + torch.bincount(new[given], minlength=pool)
    missing = need - torch.minimum((total - before).clamp_min(0), need)
    # The copies of partial pages.
    f = full[parent].clamp_max(table - 1).unsqueeze(1)
    target = new.gather(1, f).squeeze(1)
    copy = live & ~first & (part[parent] > 0)
    made = copy & (target >= 0)
    out = torch.where(live, torch.where(copy & ~made, full[parent] * page, lengths[parent]), 0)
    return {"new_tables": new.float(), "new_lengths": out.float(), "new_uses": uses,
            "sources": torch.where(made, tables[parent].gather(1, f).squeeze(1), -1).float(),
            "targets": torch.where(made, target, -1).float(), "copy_rows": torch.where(made, part[parent], 0).float(),
            "missing": missing.float()}


def _copy(case, x):
    rows, targets, sources = x["copy_rows"].long(), x["targets"].long(), x["sources"].long()
    # A copy that is not made writes its source to itself.
    targets = torch.where(rows > 0, targets, sources)
    moved = torch.arange(case["page"], device="cuda") < rows.unsqueeze(1)
    moved = moved[:, :, None, None] if case["pages_token_major"] else moved[:, None, :, None]
    for pool in (x["k_pages"], x["v_pages"]):
        pool[targets] = torch.where(moved, pool[sources], pool[targets])
    return {"k_pages": x["k_pages"], "v_pages": x["v_pages"]}


def _append(case, x):
    batch, page, rows = case["batch"], case["page"], case["rows"]
    lengths, counts, tables = x["lengths"].long(), x["counts"].long(), x["tables"].long()
    # Places past the last row repeat it, so that every write has its row; a sequence without rows writes its first
    # row's old content to itself.
    at = torch.minimum(torch.arange(rows, device="cuda"), (counts - 1).clamp_min(0).unsqueeze(1))
    place = (lengths.unsqueeze(1) + at).clamp_max(tables.shape[1] * page - 1)
    pages = tables.gather(1, place // page).clamp_min(0)
    b = torch.arange(batch, device="cuda").unsqueeze(1)
    some = (counts > 0)[:, None, None, None]
    for pool, new in ((x["k_pages"], x["k"]), (x["v_pages"], x["v"])):
        by_token = pool if case["pages_token_major"] else pool.transpose(1, 2)
        values = new if case["token_major"] else new.transpose(1, 2)
        old = by_token[pages, place % page]
        by_token[pages, place % page] = torch.where(some, values[b, at], old)
    return {"k_pages": x["k_pages"], "v_pages": x["v_pages"], "new_lengths": (lengths + counts).float()}


def _keys(case, pool, tables):
    """The keys of every sequence, one after the other: [batch, kv heads, table * page, dim]."""
    rows = pool[tables.clamp_min(0)]
    axis = (0, 3, 1, 2, 4) if case["pages_token_major"] else (0, 2, 1, 3, 4)
    return rows.permute(axis).reshape(case["batch"], case["kv_heads"], -1, case["dim"])


def _attend(case, x):
    batch, queries, dim, kv_heads = case["batch"], case["queries"], case["dim"], case["kv_heads"]
    group = case["heads"] // kv_heads
    tables, lengths, counts = x["tables"].long(), x["lengths"].long(), x["counts"].long()
    q = x["q"].transpose(1, 2) if case["token_major"] else x["q"]
    q = q.reshape(batch, kv_heads, group * queries, dim) * dim ** -0.5
    k, v = _keys(case, x["k_pages"], tables), _keys(case, x["v_pages"], tables)
    i, j = torch.arange(queries, device="cuda"), torch.arange(k.shape[2], device="cuda")
    position = (lengths - counts).unsqueeze(1) + i
    sees = (j <= position.unsqueeze(-1)) & (i < counts.unsqueeze(1)).unsqueeze(-1)
    scores = q @ k.transpose(-1, -2).contiguous()
    scores.view(batch, kv_heads, group, queries, -1).masked_fill_(~sees[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    scores = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    scores = scores.div_(scores.sum(dim=-1, keepdim=True).clamp_min(1e-37))
    out = (scores @ v).view(batch, case["heads"], queries, dim)
    return {"out": out.transpose(1, 2).contiguous() if case["token_major"] else out}


def run(state):
    if own:
        state["runtime"].execute(state["jobs"], 1)
        return state["outputs"]
    form = {"beam_select": _select, "pages_fork": _fork, "pages_copy": _copy, "pages_append": _append,
            "attention_paged": _attend}[state["case"]["kind"]]
    return form(state["case"], state["inputs"])


def work(case):
    kind, batch = case["kind"], case["batch"]
    if kind == "beam_select":
        n = batch * case["beams"] * case["vocab"]
        return {"bytes": 4 * n + 8 * batch * case["beams"] + 16 * batch * case["picks"], "flops": 4 * n}
    if kind == "pages_fork":
        return {"bytes": 8 * (batch * case["table"] + _pages(case)) + 32 * batch, "flops": 0}
    row = case["kv_heads"] * case["dim"]
    if kind == "pages_copy":
        return {"bytes": 16 * row * sum(_copy_rows(case)) + 12 * batch, "flops": 0}
    new, ends = _new(case), _ends(case)
    if kind == "pages_append":
        return {"bytes": 16 * row * sum(new) + 12 * batch + 4 * sum(-(-n // case["page"]) for n in new), "flops": 0}
    pairs = sum(n * (e - n) + n * (n + 1) // 2 for n, e in zip(new, ends))
    return {"bytes": 8 * row * sum(e for n, e in zip(new, ends) if n) + 4 * case["heads"] * case["dim"] *
            (sum(new) + batch * case["queries"]) + 4 * sum(-(-e // case["page"]) for e in ends) + 8 * batch,
            "flops": 4 * case["heads"] * case["dim"] * pairs}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------

def _exact_select(case, x):
    batch, beams, vocab, picks = case["batch"], case["beams"], case["vocab"], case["picks"]
    out = {"parents": torch.full((batch, picks), -1.0, dtype=torch.float64, device="cuda"),
           "tokens": torch.full((batch, picks), -1.0, dtype=torch.float64, device="cuda"),
           "new_scores": torch.full((batch, picks), -math.inf, dtype=torch.float64, device="cuda"),
           "new_finished": torch.zeros(batch, picks, dtype=torch.float64, device="cuda")}
    for b in range(batch):
        logits = x["logits"][b].double()
        scores = torch.log_softmax(logits, dim=-1) + x["scores"][b].double().unsqueeze(1)
        for beam in torch.nonzero(x["finished"][b] > 0).flatten().tolist():
            scores[beam] = -math.inf
            if case["end"] < vocab:
                scores[beam, case["end"]] = x["scores"][b, beam].double()
        values, at = torch.sort(scores.flatten(), descending=True, stable=True)
        values, at = values[:picks], at[:picks]
        n = int((values > -math.inf).sum())
        values, at = values[:n], at[:n]
        out["parents"][b, :n] = (b * beams + at // vocab).double()
        out["tokens"][b, :n] = (at % vocab).double()
        out["new_scores"][b, :n] = values
        out["new_finished"][b, :n] = ((at % vocab == case["end"]) | (x["finished"][b][at // vocab] > 0)).double()
    return out


def _exact_fork(case, x):
    """Page by page on the host, in plain lists."""
    page, table, batch = case["page"], case["table"], case["batch"]
    parents, lengths, reserve = ([int(v) for v in x[n].tolist()] for n in ("parents", "lengths", "reserve"))
    old = [[int(p) for p in row if p >= 0] for row in x["tables"].tolist()]
    uses = [int(u) for u in x["uses"].tolist()]
    children = {}
    for s, p in enumerate(parents):
        if p >= 0:
            children.setdefault(p, []).append(s)
    new, copies = [[] for _ in range(batch)], {}
    for p, row in enumerate(old):
        full = lengths[p] // page
        for s in children.get(p, []):
            if s == children[p][0]:
                new[s] = list(row)
            else:
                new[s] = row[:full]
                if lengths[p] % page:
                    copies[s] = row[full]
    for row in old:
        for e in row:
            uses[e] -= 1
    for row in new:
        for e in row:
            uses[e] += 1
    free = iter([p for p, u in enumerate(uses) if u == 0])
    ends, missing = [0] * batch, [0] * batch
    moves = [(-1, -1, 0)] * batch
    for s, p in enumerate(parents):
        if p < 0:
            continue
        ends[s] = lengths[p]
        want = min(table, -(-(lengths[p] + reserve[s]) // page))
        while len(new[s]) < want:
            got = next(free, None)
            if got is None:
                missing[s] += want - len(new[s])
                break
            uses[got] += 1
            new[s].append(got)
        if s in copies:
            full = lengths[p] // page
            if len(new[s]) > full:
                moves[s] = (copies[s], new[s][full], lengths[p] % page)
            else:
                ends[s] = full * page
    rows = [row + [-1] * (table - len(row)) for row in new]
    values = {"new_tables": rows, "new_lengths": ends, "new_uses": uses, "sources": [m[0] for m in moves],
              "targets": [m[1] for m in moves], "copy_rows": [m[2] for m in moves], "missing": missing}
    return {name: torch.tensor(v, dtype=torch.float64, device="cuda") for name, v in values.items()}


def exact(case, seed):
    x = _inputs(case, seed)
    kind = case["kind"]
    if kind == "beam_select":
        return _exact_select(case, x)
    if kind == "pages_fork":
        return _exact_fork(case, x)
    by_token, page = case["pages_token_major"], case["page"]
    if kind == "pages_copy":
        pools = [x["k_pages"].double(), x["v_pages"].double()]
        for s, t, n in zip(x["sources"].long().tolist(), x["targets"].long().tolist(), _copy_rows(case)):
            for pool in pools:
                if n and by_token:
                    pool[t, :n] = pool[s, :n]
                elif n:
                    pool[t, :, :n] = pool[s, :, :n]
        return {"k_pages": pools[0], "v_pages": pools[1]}
    tables, ends, new = x["tables"].long().tolist(), _ends(case), _new(case)
    if kind == "pages_append":
        pools = [x["k_pages"].double(), x["v_pages"].double()]
        for b in range(case["batch"]):
            at = ends[b] - new[b]
            while at < ends[b]:
                n = min(ends[b] - at, page - at % page)
                i, p = at - (ends[b] - new[b]), tables[b][at // page]
                for pool, rows in zip(pools, (x["k"], x["v"])):
                    values = rows[b, i:i + n] if case["token_major"] else rows[b, :, i:i + n].transpose(0, 1)
                    if by_token:
                        pool[p, at % page:at % page + n] = values.double()
                    else:
                        pool[p, :, at % page:at % page + n] = values.double().transpose(0, 1)
                at += n
        return {"k_pages": pools[0], "v_pages": pools[1],
                "new_lengths": torch.tensor(ends, dtype=torch.float64, device="cuda")}
    q = x["q"].double() if case["token_major"] else x["q"].double().transpose(1, 2)
    out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    group = case["heads"] // case["kv_heads"]
    for b in range(case["batch"]):
        if not new[b]:
            continue
        entries = torch.tensor([e for e in tables[b] if e >= 0], device="cuda")
        hidden = torch.ones(new[b], ends[b], dtype=torch.bool, device="cuda").triu_(ends[b] - new[b] + 1)
        for kv in range(case["kv_heads"]):
            def rows_of(pool):
                rows = pool[entries, :, kv] if by_token else pool[entries, kv]
                return rows.reshape(-1, case["dim"])[:ends[b]].double()
            k, v = rows_of(x["k_pages"]).t().contiguous(), rows_of(x["v_pages"])
            for h in range(kv * group, (kv + 1) * group):
                scores = q[b, :new[b], h] @ k / math.sqrt(case["dim"])
                scores.masked_fill_(hidden, -math.inf)
                out[b, :new[b], h] = torch.softmax(scores, dim=-1) @ v
    return {"out": out if case["token_major"] else out.transpose(1, 2).contiguous()}
