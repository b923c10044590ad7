"""Specs, bindings, refusals and launches of decoding over a paged cache, on the CPU, and its oracle's own checks."""
import json

import numpy as np
import pytest

import jade_hip
import paged_oracle as po

POOL = {"kv_heads": 3, "pages": 20, "page": 16, "dim": 8, "pages_token_major": True}
PAGED = {"op": "attention_paged", "batch": 2, "heads": 6, "queries": 5, **POOL, "table": 4, "token_major": True}
APPEND = {"op": "pages_append", "batch": 2, "rows": 5, **POOL, "table": 4, "token_major": False}
FORK = {"op": "pages_fork", "batch": 4, "pages": 20, "page": 16, "table": 4}
COPY = {"op": "pages_copy", "copies": 3, **POOL}
SELECT = {"op": "beam_select", "batch": 2, "beams": 3, "vocab": 50, "picks": 6, "end": 2}
ALL = [PAGED, APPEND, FORK, COPY, SELECT]


def refused(spec):
    with pytest.raises(jade_hip.JadeError) as info:
        jade_hip.spec_describe(spec)
    assert info.value.code == 1
    return info.value.message


@pytest.mark.parametrize("spec", ALL, ids=lambda s: s["op"])
def test_descriptions(spec):
    d = jade_hip.spec_describe(spec)
    assert d["name"] == spec["op"] and d["hip_supported"] and d["launch"]["kernel"]
    assert not d["reference_valid"] and "reference" in d["reference_error"]
    for key, value in spec.items():
        assert d["spec"][key] == value
    assert jade_hip.spec_describe(json.dumps(d["spec"])) == d  # the canonical form round-trips


def test_bindings():
    def of(spec):
        return [(b["name"], b["elements"], b["write"]) for b in jade_hip.spec_describe(spec)["bindings"]]

    pool = 20 * 16 * 3 * 8
    assert of(PAGED) == [("q", 480, False), ("k_pages", pool, False), ("v_pages", pool, False), ("tables", 8, False),
                         ("lengths", 2, False), ("counts", 2, False), ("out", 480, True)]
    assert of(APPEND) == [("k", 240, False), ("v", 240, False), ("counts", 2, False), ("tables", 8, False),
                          ("lengths", 2, False), ("k_pages", pool, True), ("v_pages", pool, True),
                          ("new_lengths", 2, True)]
    assert of(FORK) == [("parents", 4, False), ("lengths", 4, False), ("tables", 16, False), ("reserve", 4, False),
                        ("uses", 20, False), ("new_tables", 16, True), ("new_lengths", 4, True), ("new_uses", 20, True),
                        ("sources", 4, True), ("targets", 4, True), ("copy_rows", 4, True), ("missing", 4, True)]
    assert of(COPY) == [("sources", 3, False), ("targets", 3, False), ("copy_rows", 3, False), ("k_pages", pool, True),
                        ("v_pages", pool, True)]
    assert of(SELECT) == [("logits", 300, False), ("scores", 6, False), ("finished", 6, False), ("parents", 12, True),
                          ("tokens", 12, True), ("new_scores", 12, True), ("new_finished", 12, True)]


@pytest.mark.parametrize("spec", ALL, ids=lambda s: s["op"])
def test_outputs_alias_nothing(spec):
    bindings = jade_hip.spec_describe(spec)["bindings"]
    lengths, ids = [b["elements"] for b in bindings], list(range(len(bindings)))
    jade_hip.spec_validate_bindings(spec, lengths, ids)
    for out, b in enumerate(bindings):
        for other in range(len(bindings)):
            if b["write"] and other != out:
                shared = list(ids)
                shared[out] = ids[other]
                with pytest.raises(jade_hip.JadeError):
                    jade_hip.spec_validate_bindings(spec, lengths, shared)
    with pytest.raises(jade_hip.JadeError):
        jade_hip.spec_validate_bindings(spec, [lengths[0] + 1] + lengths[1:], ids)


@pytest.mark.parametrize("spec", ALL, ids=lambda s: s["op"])
def test_every_field_is_needed_and_positive(spec):
    for key, value in spec.items():
        if key == "op":
            continue
        assert key in refused({k: v for k, v in spec.items() if k != key})
        if isinstance(value, int) and not isinstance(value, bool):
            if key != "end":  # token 0 may end a beam
                refused(dict(spec, **{key: 0}))
            refused(dict(spec, **{key: -1}))
        if isinstance(value, bool):
            assert "boolean" in refused(dict(spec, **{key: 1}))


@pytest.mark.parametrize("spec,why", [
    (dict(PAGED, page=8), "multiple of 16"), (dict(PAGED, page=24), "multiple of 16"), (dict(PAGED, page=1040), "1024"),
    (dict(PAGED, heads=7), "multiple"), (dict(PAGED, dim=129), "128"), (dict(PAGED, table=2 ** 20 + 1), "table"),
    (dict(PAGED, pages=2 ** 24 + 1), "pages"), (dict(PAGED, batch=65536), "batch"),
    (dict(PAGED, batch=65535, queries=100000), "31-bit"), (dict(PAGED, queries=2 ** 24 + 1), "queries"),
    (dict(PAGED, pages=2 ** 24, kv_heads=2 ** 10, heads=2 ** 10, dim=64), "2^40"),
    (dict(PAGED, batch=65535, table=2 ** 16), "31-bit"), (dict(PAGED, kv_heads=65536, heads=65536), "heads"),
    (dict(APPEND, dim=513), "512"), (dict(APPEND, rows=2 ** 24 + 1), "rows"), (dict(APPEND, page=17), "multiple of 16"),
    (dict(APPEND, batch=65535, rows=100000), "31-bit"), (dict(APPEND, table=2 ** 20 + 1), "table"),
    (dict(FORK, batch=65536), "batch"), (dict(FORK, page=2048), "1024"), (dict(FORK, pages=2 ** 24 + 1), "pages"),
    (dict(FORK, batch=65535, table=2 ** 16), "31-bit"),
    (dict(COPY, copies=65536), "copies"), (dict(COPY, dim=513), "512"), (dict(COPY, page=0), "multiple of 16"),
    (dict(COPY, pages=2 ** 24, kv_heads=2 ** 10, dim=64), "2^40"),
    (dict(SELECT, beams=257), "beams"), (dict(SELECT, picks=65), "picks"), (dict(SELECT, vocab=2 ** 24 + 1), "vocab"),
    (dict(SELECT, batch=65535, beams=256, vocab=200), "31-bit"), (dict(SELECT, batch=65536), "batch"),
    (dict(SELECT, end=2 ** 32), "u32")])
def test_refusals(spec, why):
    assert why in refused(spec)


def test_pools_pass_31_bits():
    d = jade_hip.spec_describe(dict(PAGED, kv_heads=8, heads=8, pages=2 ** 20, dim=128))
    assert d["bindings"][1]["elements"] == 2 ** 20 * 16 * 8 * 128 > 2 ** 33 and d["hip_supported"]


@pytest.mark.parametrize("spec", [
    dict(PAGED, batch=65535, heads=16, kv_heads=16, queries=8, table=64, dim=64),
    dict(PAGED, batch=1, heads=1, kv_heads=1, queries=2 ** 24, table=2, dim=4),
    dict(PAGED, batch=64, heads=128, kv_heads=8, queries=1000, table=1000, page=1024, dim=128),
    dict(APPEND, batch=4095, kv_heads=16, rows=32000, dim=1), dict(APPEND, batch=1, kv_heads=65535, rows=32000, dim=1),
    dict(APPEND, batch=127, kv_heads=1, rows=2 ** 24, dim=1, token_major=True),
    dict(FORK, batch=65535, pages=2 ** 24, table=2 ** 15, page=512),
    dict(COPY, copies=65535, kv_heads=65535, pages=4096, page=16, dim=4), dict(COPY, copies=1, kv_heads=4096, page=1024, dim=500),
    dict(SELECT, batch=65535, beams=256, vocab=100), dict(SELECT, batch=1, beams=1, vocab=2 ** 24, picks=64),
    dict(SELECT, batch=65535, beams=256, vocab=1), dict(SELECT, batch=1, beams=127, vocab=2 ** 24)],
    ids=lambda s: s["op"])
def test_the_largest_launches(spec):
    launch = jade_hip.spec_describe(spec)["launch"]
    if launch:
        for blocks, threads in zip(launch["grid"], launch["block"]):
            assert 1 <= blocks and blocks * threads < 2 ** 32, (spec, launch)
        assert launch["grid"][1] <= 65535 and launch["grid"][2] <= 65535


def test_work_past_32_bits_of_tiles_has_no_kernel():
    d = jade_hip.spec_describe(dict(PAGED, batch=16, heads=1, kv_heads=1, queries=2 ** 24, table=2 ** 20, dim=1))
    assert not d["hip_supported"] and d["launch"] is None


def test_pages_of_more_than_31_bits_are_not_copied():
    d = jade_hip.spec_describe(dict(COPY, pages=2, kv_heads=65535, page=1024, dim=512))
    assert not d["hip_supported"] and d["launch"] is None


# ---- the oracle ------------------------------------------------------------------------------------------

def test_oracle_pages_hold_what_a_contiguous_cache_does():
    import decoder_oracle as dec
    rng = np.random.default_rng(1)
    spec = dict(PAGED, batch=1, heads=3)
    order = rng.permutation(20)[:4]
    k, v = (rng.standard_normal((1, 64, 3, 8)).astype(np.float32) for _ in range(2))
    pools = [np.full((20, 16, 3, 8), np.nan, np.float32) for _ in range(2)]
    for pool, x in zip(pools, (k, v)):
        pool[order] = x.reshape(4, 16, 3, 8)
    q = rng.standard_normal((1, 5, 3, 8)).astype(np.float32)
    got, _ = po.paged(spec, q, *pools, order[None], [50], [5])
    for i in range(5):
        one, _ = dec.cross({"batch": 1, "heads": 3, "kv_heads": 3, "queries": 1, "keys": 64, "dim": 8, "token_major": True},
                           q[:, i:i + 1], k, v, [46 + i])
        assert np.abs(got[:, i] - one[:, 0]).max() < 1e-14


def test_oracle_forks_keep_every_use():
    rng = np.random.default_rng(2)
    for seed in range(20):
        tables = np.full((4, 4), -1.0)
        order = iter(rng.permutation(20))
        lengths = rng.integers(0, 60, 4)
        for row, n in zip(tables, lengths):
            held = -(-n // 16)
            row[:held] = [next(order) for _ in range(held)]
        uses = np.zeros(20)
        for e in tables[tables >= 0]:
            uses[int(e)] += 1
        got = po.fork(FORK, rng.integers(-1, 4, 4), lengths, tables, np.ones(4), uses)
        count = np.zeros(20)
        for e in got["new_tables"][got["new_tables"] >= 0]:
            count[int(e)] += 1
        assert (count == got["new_uses"]).all()


def test_oracle_mistakes_are_noticed():
    # A token too many, or one too few, is far outside the bound that the GPU's results are held to.
    rng = np.random.default_rng(3)
    spec = dict(PAGED, batch=1, heads=3, queries=1, dim=8)
    pools = [rng.standard_normal((20, 16, 3, 8)).astype(np.float32) for _ in range(2)]
    q, table = rng.standard_normal((1, 1, 3, 8)).astype(np.float32), np.arange(4.0)[None]
    want, off = po.paged(spec, q, *pools, table, [40], [1])
    for length in (39, 41):
        assert (np.abs(po.paged(spec, q, *pools, table, [length], [1])[0] - want) > off).mean() > 0.5
