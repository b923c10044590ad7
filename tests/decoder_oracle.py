"""The operators of a decoder's step in 64 bits, in numpy, row by row, with bounds on what FP32 may be off.

U is half an ulp of FP32: every operation rounds by at most U of its result. The bounds count roundings, to first
order, and are written beside each operator.
"""
import numpy as np

U = 2.0 ** -24


def length_of(x, most):
    x = np.float32(x)
    return 0 if not x >= 1 else int(min(np.float32(most), x))


def node_of(x, n):
    """The parent of slot n: -1, an earlier slot, or None where the slot holds no node."""
    x = np.float32(x)
    if x == -1 or (0 <= x < n and x == np.trunc(x)):
        return int(x)
    return None


def ancestors(parents):
    seen = []
    for n, p in enumerate(parents):
        p = node_of(p, n)
        seen.append([] if p is None else ([] if p < 0 else seen[p]) + [n])
    return seen


def rates(spec):
    i = np.arange(spec["rotary_dim"] // 2)
    f = float(np.float32(spec["base"])) ** (-2.0 * i / spec["rotary_dim"])
    factor, context = spec.get("factor", 1.0), spec.get("context", 0.0)
    if not context:
        return f / factor
    turns = context * f / (2 * np.pi)
    keep = np.clip((turns - spec["low_turns"]) / (spec["high_turns"] - spec["low_turns"]), 0, 1)
    return f * (keep + (1 - keep) / factor)


def rotate(spec, x, positions, inverse=False):
    """x: [batch, seq, heads, dim] in 64 bits. Returns the outputs and, for each, m (|a| + |b|) of its pair (zero
    where the element is copied)."""
    r = spec["rotary_dim"]
    angle = positions.astype(np.float64).reshape(x.shape[0], x.shape[1], 1, 1) * rates(spec)
    m = float(np.float32(spec.get("magnitude", 1.0)))
    c, s = m * np.cos(angle), m * np.sin(angle) * (-1 if inverse else 1)
    ia = np.arange(0, r, 2) if spec["interleaved"] else np.arange(r // 2)
    ib = ia + 1 if spec["interleaved"] else ia + r // 2
    out, size = x.copy(), np.zeros_like(x)
    a, b = x[..., ia], x[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = m * (np.abs(a) + np.abs(b))
    return out, size


# cos and sin: 1 for the remainder's conversion, 2 for the series, 1 for the magnitude; the two products and their
# sum: 1 each. Times |a| + |b|.
ROTARY_BOUND = 6 * U
# The norm: at most 8 + 6 additions of squares in a row and the square itself, halved by the root: 7.5; the mean, the
# epsilon: 1; rsqrt: 2; x * inv * weight: 2. Then the rotation's, on values that are already off.
NORM_BOUND = 13 * U


def norm(x, weight, epsilon):
    return x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + float(np.float32(epsilon))) * weight


def attend(q, k, v, sees):
    """One query row over the keys `sees`: its output, and how far FP32 may be off.

    A score is a sum of dim products (dim + 2 roundings of at most the sum of their sizes, the scale among them),
    twice for its own and the maximum's; exp2 and its argument's subtraction: 4. A weight is off by that relatively,
    numerator and denominator each. The sums over the keys: one rounding a key at most, twice; 16 for rescaling and
    joining the parts."""
    if not len(sees):
        return np.zeros_like(q), np.zeros_like(q)
    k, v = k[sees], v[sees]
    scores = k @ q / np.sqrt(len(q))
    sizes = np.abs(k) @ np.abs(q) / np.sqrt(len(q))
    p = np.exp(scores - scores.max())
    p /= p.sum()
    bound = U * (2 * (2 * (len(q) + 2) * sizes.max() + 4) + 2 * len(sees) + 16)
    return p @ v, bound * (p @ np.abs(v))


def by_token(x, token_major):
    """[batch, rows, heads, dim] whatever the layout."""
    return x if token_major else np.swapaxes(x, 1, 2)


def cross(spec, q, k, v, lengths):
    tm = spec["token_major"]
    q, k, v = (by_token(x.astype(np.float64), tm) for x in (q, k, v))
    out, off = np.zeros_like(q), np.zeros_like(q)
    group = spec["heads"] // spec["kv_heads"]
    for b in range(spec["batch"]):
        sees = np.arange(length_of(lengths[b], spec["keys"]))
        for h in range(spec["heads"]):
            for n in range(spec["queries"]):
                out[b, n, h], off[b, n, h] = attend(q[b, n, h], k[b, :, h // group], v[b, :, h // group], sees)
    return by_token(out, tm), by_token(off, tm)


def tree(spec, q, kc, vc, lengths, kd, vd, parents):
    tm = spec["token_major"]
    q, kc, vc, kd, vd = (by_token(x.astype(np.float64), tm) for x in (q, kc, vc, kd, vd))
    out, off = np.zeros_like(q), np.zeros_like(q)
    group = spec["heads"] // spec["kv_heads"]
    for b in range(spec["batch"]):
        n_cached = length_of(lengths[b], spec["capacity"])
        seen = ancestors(parents[b])
        for h in range(spec["heads"]):
            k = np.concatenate([kc[b, :n_cached, h // group], kd[b, :, h // group]])
            v = np.concatenate([vc[b, :n_cached, h // group], vd[b, :, h // group]])
            for n in range(spec["nodes"]):
                if seen[n]:
                    sees = list(range(n_cached)) + [n_cached + x for x in seen[n]]
                    out[b, n, h], off[b, n, h] = attend(q[b, n, h], k, v, sees)
    return by_token(out, tm), by_token(off, tm)


def append(spec, k, v, picks, lengths, k_cache, v_cache):
    k_cache, v_cache = k_cache.copy(), v_cache.copy()
    new = np.zeros(spec["batch"], np.float32)
    for b in range(spec["batch"]):
        at = length_of(lengths[b], spec["capacity"])
        for p in picks[b]:
            if not (0 <= p < spec["rows"] and p == np.trunc(p)) or at >= spec["capacity"]:
                break
            for cache, rows in ((k_cache, k), (v_cache, v)):
                by_token(cache, spec["token_major"])[b, at] = by_token(rows, spec["token_major"])[b, int(p)]
            at += 1
        new[b] = at
    return k_cache, v_cache, new
