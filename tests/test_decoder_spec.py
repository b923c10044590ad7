"""Specs, bindings and refusals of the operators of a decoder's step, on the CPU."""
import json

import numpy as np
import pytest

import decoder_oracle as dec
import jade_hip

ROTARY = {"op": "rotary", "batch": 2, "seq": 5, "heads": 3, "dim": 16, "rotary_dim": 8, "interleaved": False,
          "inverse": False, "token_major": True, "out_token_major": False, "base": 10000.0}
NORM = {"op": "qk_norm_rotary", "batch": 2, "seq": 5, "heads": 6, "kv_heads": 3, "dim": 16, "rotary_dim": 8,
        "interleaved": True, "token_major": True, "out_token_major": False, "epsilon": 1e-6, "base": 10000.0}
TREE = {"op": "attention_tree", "batch": 2, "heads": 6, "kv_heads": 3, "nodes": 7, "capacity": 100, "dim": 16,
        "token_major": False}
APPEND = {"op": "cache_append", "batch": 2, "kv_heads": 3, "rows": 7, "picks": 4, "capacity": 100, "dim": 16,
          "token_major": False}
CROSS = {"op": "attention_cross", "batch": 2, "heads": 6, "kv_heads": 3, "queries": 9, "keys": 50, "dim": 16,
         "token_major": True}
ALL = [ROTARY, NORM, TREE, APPEND, CROSS]


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
        assert d["spec"][key] == pytest.approx(value)
    assert jade_hip.spec_describe(json.dumps(d["spec"])) == d  # the canonical form round-trips


def test_bindings():
    def of(spec):
        return [(b["name"], b["elements"], b["write"]) for b in jade_hip.spec_describe(spec)["bindings"]]

    assert of(ROTARY) == [("x", 480, False), ("positions", 10, False), ("out", 480, True)]
    assert of(NORM) == [("q", 960, False), ("k", 480, False), ("q_weight", 16, False), ("k_weight", 16, False),
                        ("positions", 10, False), ("q_out", 960, True), ("k_out", 480, True)]
    assert of(TREE) == [("q", 1344, False), ("k_cache", 9600, False), ("v_cache", 9600, False), ("lengths", 2, False),
                        ("k_draft", 672, False), ("v_draft", 672, False), ("parents", 14, False), ("out", 1344, True)]
    assert of(APPEND) == [("k", 672, False), ("v", 672, False), ("picks", 8, False), ("lengths", 2, False),
                          ("k_cache", 9600, True), ("v_cache", 9600, True), ("new_lengths", 2, True)]
    assert of(CROSS) == [("q", 1728, False), ("k", 4800, False), ("v", 4800, False), ("lengths", 2, False),
                         ("out", 1728, True)]


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
        if isinstance(value, (int, float)) and not isinstance(value, bool):
            refused(dict(spec, **{key: 0}))
            refused(dict(spec, **{key: -1}))


@pytest.mark.parametrize("spec,why", [
    (dict(ROTARY, rotary_dim=7), "even"), (dict(ROTARY, rotary_dim=18), "even"), (dict(ROTARY, dim=514), "512"),
    (dict(ROTARY, base=1e39), "base"), (dict(ROTARY, factor=0.0), "factor"), (dict(ROTARY, magnitude=0.0), "magnitude"),
    (dict(ROTARY, context=-1.0), "context"), (dict(ROTARY, low_turns=1.0, high_turns=4.0), "context"),
    (dict(ROTARY, context=100.0), "turns"), (dict(ROTARY, context=100.0, low_turns=4.0, high_turns=4.0), "turns"),
    (dict(ROTARY, context=100.0, low_turns=-1.0, high_turns=4.0), "turns"), (dict(ROTARY, factor="4"), "number"),
    (dict(ROTARY, batch=65536), "batch"), (dict(ROTARY, batch=60000, seq=60000), "31-bit"),
    (dict(ROTARY, seq=4294967295), "dimension"), (dict(ROTARY, inverse=1), "boolean"),
    (dict(NORM, heads=65536), "heads"), (dict(NORM, kv_heads=60000, seq=60000), "31-bit"),
    (dict(TREE, nodes=257), "nodes"), (dict(TREE, dim=129), "128"), (dict(TREE, kv_heads=4), "multiple"),
    (dict(TREE, capacity=16777217), "capacity"), (dict(TREE, batch=65535, kv_heads=6, capacity=16777216), "2^40"),
    (dict(APPEND, rows=16777217), "rows"), (dict(APPEND, picks=16777217), "picks"), (dict(APPEND, dim=513), "512"),
    (dict(APPEND, batch=65535, picks=16777216), "31-bit"),
    (dict(CROSS, heads=7), "multiple"), (dict(CROSS, keys=16777217), "keys"), (dict(CROSS, dim=200), "128"),
    (dict(CROSS, batch=65535, queries=100000), "31-bit")])
def test_refusals(spec, why):
    assert why in refused(spec)


def test_work_past_32_bits_of_tiles_has_no_kernel():
    # 2^31 / 32 row blocks of one head, 2^18 tiles each.
    d = jade_hip.spec_describe(dict(CROSS, batch=1, heads=1, kv_heads=1, queries=2 ** 30, keys=2 ** 24, dim=1))
    assert not d["hip_supported"] and d["launch"] is None


def test_rows_too_far_apart_for_a_kernels_offsets_take_another():
    def kernel(**more):
        return jade_hip.spec_describe(dict(CROSS, batch=1, heads=65535, kv_heads=65535, queries=17, keys=5, **more))["launch"]["kernel"]

    # 128 keys, 65535 heads of 128 apart, span more than 2 GiB.
    assert kernel(dim=128, token_major=True) == "attention_ragged_d128"
    assert kernel(dim=128, token_major=False) == "attention_flash_ragged_d128"
    # 2^29 elements of one head's queries.
    far = jade_hip.spec_describe(dict(CROSS, batch=1, heads=1, kv_heads=1, queries=2 ** 23, keys=1000, dim=64))
    assert far["launch"]["kernel"] == "attention_ragged_parts_d64_r64"
    # More row blocks than a grid's second dimension.
    many = jade_hip.spec_describe(dict(CROSS, batch=1, heads=1, kv_heads=1, queries=2 ** 24, keys=1000, dim=4))
    assert many["launch"]["kernel"] == "attention_ragged_parts_d64_r64"


def test_caches_pass_31_bits():
    d = jade_hip.spec_describe(dict(TREE, batch=64, heads=8, kv_heads=8, capacity=131072, dim=128))
    assert d["bindings"][1]["elements"] == 64 * 8 * 131072 * 128 > 2 ** 31 and d["hip_supported"]


def test_scaling_is_part_of_the_kernels_identity():
    seen = {json.dumps(jade_hip.spec_describe(s)["spec"]) for s in (
        ROTARY, dict(ROTARY, factor=2.0), dict(ROTARY, magnitude=2.0), dict(ROTARY, inverse=True),
        dict(ROTARY, context=64.0, low_turns=1.0, high_turns=2.0), dict(ROTARY, factor=1.0, magnitude=1.0))}
    assert len(seen) == 5  # the last says what the first leaves out


def test_oracle_rotation_is_a_rotation():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((1, 4, 2, 16))
    y, _ = dec.rotate(ROTARY, x, np.arange(4.0)[None])
    z, _ = dec.rotate(ROTARY, y, np.arange(4.0)[None], inverse=True)
    assert np.abs(z - x).max() < 1e-14 and (y[:, 0] == x[:, 0]).all() and (y[..., 8:] == x[..., 8:]).all()
    # Scores of rotated vectors depend on the distance alone.
    same = np.broadcast_to(x[:, :1], x.shape)
    r, _ = dec.rotate(dict(ROTARY, rotary_dim=16), same, np.arange(4.0)[None])
    far, _ = dec.rotate(dict(ROTARY, rotary_dim=16), same, np.arange(100.0, 104.0)[None])
    assert np.abs((r[0, 0] * r[0, 3]).sum(-1) - (far[0, 0] * far[0, 3]).sum(-1)).max() < 1e-12


def test_oracle_mistakes_are_noticed():
    # A key left out, or one too many, is far outside the bound that the GPU's results are held to.
    rng = np.random.default_rng(2)
    q, k, v = rng.standard_normal(64), rng.standard_normal((300, 64)), rng.standard_normal((300, 64))
    want, off = dec.attend(q, k, v, np.arange(299))
    for sees in (np.arange(298), np.arange(300)):
        assert (np.abs(dec.attend(q, k, v, sees)[0] - want) > off).mean() > 0.5
