"""Launches that the specs of a decoder's step describe, on the CPU: what is called supported can be launched."""
import itertools

import pytest

import jade_hip
from test_decoder_spec import APPEND, CROSS, NORM, ROTARY, TREE


def launchable(spec):
    """Whether the spec has a kernel; then its grid has to be one that HIP takes: 2^32 - 1 threads a dimension."""
    launch = jade_hip.spec_describe(spec)["launch"]
    if launch is None:
        return False
    for blocks, threads in zip(launch["grid"], launch["block"]):
        assert 1 <= blocks and blocks * threads < 2 ** 32, (spec, launch)
    assert launch["grid"][1] <= 65535 and launch["grid"][2] <= 65535, (spec, launch)
    return True


@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("dim", [4, 8, 32, 64, 96, 128])
def test_cross_attention_of_very_many_short_heads(token_major, dim):
    seen = 0
    for batch, heads, queries, keys in itertools.product((1, 4096, 65535), (1, 256, 480, 512, 65535), (1, 17, 33, 257), (1, 33)):
        if batch * heads * max(queries, keys) * dim < 2 ** 31:
            seen += launchable(dict(CROSS, batch=batch, heads=heads, kv_heads=heads, queries=queries, keys=keys, dim=dim,
                                    token_major=token_major))
    assert seen > 10


def test_the_flash_form_is_left_where_its_grid_would_pass_32_bits():
    spec = dict(CROSS, batch=65535, heads=480, kv_heads=480, queries=17, keys=1, dim=4)
    assert jade_hip.spec_describe(spec)["launch"]["kernel"] == "attention_ragged_parts_d64_r32"
    # 2^24 - 1 blocks of 256 threads are taken.
    fewer = jade_hip.spec_describe(dict(spec, batch=65535, heads=256, kv_heads=256))["launch"]
    assert fewer["kernel"] == "attention_flash_ragged_d32" and fewer["grid"][0] == 65535 * 256


@pytest.mark.parametrize("spec", [
    dict(ROTARY, batch=65535, seq=16000, heads=1, dim=2, rotary_dim=2), dict(ROTARY, batch=1, seq=2 ** 30 - 1, heads=1, dim=2, rotary_dim=2),
    dict(NORM, batch=1, seq=2 ** 29 - 1, heads=1, kv_heads=2, dim=2, rotary_dim=2),
    dict(APPEND, batch=65535, kv_heads=16, rows=1, picks=32000, capacity=8, dim=1),
    dict(APPEND, batch=1, kv_heads=65535, rows=32000, picks=32000, capacity=16777216, dim=1),
    dict(APPEND, batch=127, kv_heads=1, rows=16777216, picks=16777216, capacity=16777216, dim=1, token_major=True),
    dict(TREE, batch=65535, heads=127, kv_heads=127, nodes=256, capacity=1, dim=1),
    dict(TREE, batch=65535, heads=8, kv_heads=8, nodes=32, capacity=16777216 // 128, dim=4)],
    ids=lambda s: s["op"])
def test_the_largest_of_the_others(spec):
    launchable(spec)
