"""A decoder's steps as the documentation writes them: projections, norm and rotation, attention of drafted tokens over the
caches and the append, chained in one execute with token-major tensors, grouped heads, several sequences of different
lengths, and the new lengths taken into the next step. Each stage against 64 bits of what the stage before it left."""
import numpy as np
import pytest

import decoder_oracle as dec
import test_gpu_decoder as base

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [1, 5, 20])
def test_the_documented_step(runtime, N):
    B, H, KV, D, C, width = 3, 6, 2, 64, 90, 96
    rng = np.random.default_rng(80 + N)
    rt = runtime
    projections = {n: rt.compile({"op": "gemm", "m": B * N, "n": heads * D, "k": width, "tiled": True})
                   for n, heads in (("q", H), ("k", KV), ("v", KV))}
    heads = dict(batch=B, kv_heads=KV, dim=D)
    turn = rt.compile({"op": "qk_norm_rotary", **heads, "seq": N, "heads": H, "rotary_dim": D, "interleaved": False,
                       "token_major": True, "out_token_major": True, "epsilon": 1e-6, "base": 1e6})
    attend = rt.compile({"op": "attention_tree", **heads, "heads": H, "nodes": N, "capacity": C, "token_major": True})
    append = rt.compile({"op": "cache_append", **heads, "rows": N, "picks": N, "capacity": C, "token_major": True})

    matrices = {n: base.normal(rng, width, h * D) / 8 for n, h in (("q", H), ("k", KV), ("v", KV))}
    fixed = {n: rt.resident(x) for n, x in matrices.items()}
    weights = {n: 1 + 0.2 * base.normal(rng, D) for n in ("q_weight", "k_weight")}
    q_weight, k_weight = (rt.resident(weights[n]) for n in ("q_weight", "k_weight"))
    caches = [rt.alloc(B * C * KV * D) for _ in range(2)]
    k_cache, v_cache = caches
    lengths, new_lengths = rt.resident(np.zeros(B)), rt.alloc(B)
    want_caches = [np.zeros((B, C, KV, D), np.float32) for _ in range(2)]
    at = np.zeros(B, int)
    made = {n: rt.alloc(B * N * h * D) for n, h in (("q", H), ("k", KV), ("v", KV), ("q_turned", H), ("k_turned", KV), ("out", H))}
    q, k, v, q_turned, k_turned, out = made.values()
    for step in range(4):
        x = base.normal(rng, B * N, width)
        depth, tree = np.zeros((B, N), int), np.zeros((B, N))
        for b in range(B):
            for n in range(N):
                tree[b, n] = n - 1 if n % 3 < 2 else rng.integers(-1, n)  # a chain with branches
                depth[b, n] = depth[b, int(tree[b, n])] + 1 if tree[b, n] >= 0 else 0
        position = at[:, None] + depth
        pick = np.full((B, N), -1.0)
        for b in range(B):  # a path to some node, in order
            path, n = [], int(rng.integers(0, N))
            while n >= 0:
                path.insert(0, n)
                n = int(tree[b, n])
            if b or step % 2:  # now and then a sequence accepts nothing
                pick[b, :len(path)] = path
        hidden, positions, parents, picks = (rt.resident(y) for y in (x, position, tree, pick))
        before = rt.download(lengths)
        assert (before == at).all()
        rt.execute([(projections["q"], [hidden, fixed["q"], q]), (projections["k"], [hidden, fixed["k"], k]),
                    (projections["v"], [hidden, fixed["v"], v]),
                    (turn, [q, k, q_weight, k_weight, positions, q_turned, k_turned]),
                    (attend, [q_turned, k_cache, v_cache, lengths, k_turned, v, parents, out]),
                    (append, [k_turned, v, picks, lengths, k_cache, v_cache, new_lengths])], 1)
        got = {n: rt.download(y) for n, y in made.items()}

        for n, h in (("q", H), ("k", KV), ("v", KV)):
            a, m = x.astype(np.float64), matrices[n].astype(np.float64)
            # A product and a sum for each of the `width` terms, each at most the sum of their sizes.
            base.within(got[n], a @ m, (width + 2) * dec.U * (np.abs(a) @ np.abs(m)))
            got[n] = got[n].reshape(B, N, h, D)
        for n in "qk":
            normed = dec.norm(got[n].astype(np.float64), weights[n + "_weight"].astype(np.float64), 1e-6)
            want, size = dec.rotate(turn.spec, normed, position.astype(np.float32))
            base.within(got[n + "_turned"], want, (dec.NORM_BOUND + dec.ROTARY_BOUND) * size)
            got[n + "_turned"] = got[n + "_turned"].reshape(want.shape)
        want, off = dec.tree(attend.spec, got["q_turned"], *want_caches, before, got["k_turned"], got["v"], tree)
        base.within(got["out"], want, off)
        *want_caches, want_lengths = dec.append(append.spec, got["k_turned"], got["v"], pick, before, *want_caches)
        for cache, want in zip(caches, want_caches):
            assert (rt.download(cache).reshape(want.shape) == want).all()
        assert (rt.download(new_lengths) == want_lengths).all()
        at = want_lengths.astype(int)
        lengths, new_lengths = new_lengths, lengths
        for y in (hidden, positions, parents, picks):
            y.free()
    assert len(set(at)) > 1  # the sequences went on at their own paces
    for y in (*made.values(), *fixed.values(), *caches, q_weight, k_weight, lengths, new_lengths):
        y.free()
