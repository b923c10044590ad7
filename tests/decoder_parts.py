"""Attention whose answer hangs on the last eight of an operand's 24 bits.

FP32 operands multiplied as bf16 parts need three parts each; with two, an operand is off by up to 2^-17 of itself, 128 U.
A case here makes one operand `deep`, which is that far off or nearly so, and leaves next to nothing else to round, so
that its bound lies far below. `simulate` computes a case with fewer parts of that operand.

  v  one key: the output is its value.
  p  two keys, scores 0 and x < 0, values 0 and 1: the output is p / (1 + p), p = exp(x).
  q  two keys of one element each, scores of about 48 and close to each other, values 1 and 0: the output is
  k  1 / (1 + exp(s1 - s0)), which takes 48 times what a score is off by.
"""
import numpy as np

from decoder_oracle import U

F = np.float32
CASES = ("v", "p", "q", "k")


def bf16(x):
    bits = np.asarray(x, F).view(np.uint32).astype(np.uint64)
    return ((bits + 0x7fff + (bits >> 16 & 1)) & 0xffff0000).astype(np.uint32).view(F)


def parts(x, count):
    """The first `count` bf16 parts of x."""
    out = []
    for _ in range(count):
        out.append(bf16(x))
        x = (x - out[-1]).astype(F)
    return out


def scale_of(dim):
    """log2(e) / sqrt(dim) as the kernels round it."""
    return F(1) / np.sqrt(F(dim)) * F(1.44269504088896340736)


def deep(rng, count, scale=F(1)):
    """Numbers in 1 .. 1.5 that two parts of them times `scale` miss by at least 0.7 of 2^-17."""
    found = []
    while len(found) < count:
        x = rng.uniform(1, 1.5, 4096).astype(F)
        y = (x * scale).astype(F)
        missed = np.abs(y.astype(np.float64) - sum(p.astype(np.float64) for p in parts(y, 2)))
        found += list(x[missed > 0.7 * 2.0 ** -17 * y])
    return np.array(found[:count], F)


def shallow(dim):
    """A number near 1 that is eight bits after the kernels' scaling."""
    scale = scale_of(dim)
    for bits in range(128, 256):
        want = F(bits) * F(2.0 ** np.floor(np.log2(scale))) / F(128)
        for q in (want / scale, np.nextafter(want / scale, F(0)), np.nextafter(want / scale, F(9))):
            if q * scale == want:
                return q
    raise AssertionError(dim)


def inputs(spec, case, rng):
    """q, k, v and lengths of [batch, heads, rows, dim] tensors."""
    b, h, kv, n, m, d = (spec[x] for x in ("batch", "heads", "kv_heads", "queries", "keys", "dim"))
    q, k, v = np.zeros((b, h, n, d), F), np.zeros((b, kv, m, d), F), np.zeros((b, kv, m, d), F)
    rows, i, j = b * h * n, 0, d - 1
    if case == "v":
        q[:], k[:] = rng.standard_normal(q.shape), rng.standard_normal(k.shape)
        v[:] = deep(rng, v.size).reshape(v.shape) * rng.choice([-1, 1], v.shape)
        return q, k, v, np.ones(b, F)
    if case == "p":
        q[..., i] = rng.uniform(-1.5, -0.05, (b, h, n)) * np.sqrt(d)
        k[:, :, 1, i] = 1
        v[:, :, 1] = 1
    else:
        near = 1 + rng.uniform(-0.02, 0.02, (b, h, n) if case == "q" else (b, kv))
        size = F(2.0 ** np.round(np.log2(38 * np.sqrt(d))))  # scores from 27 to 81
        if case == "q":
            q[..., i] = deep(rng, rows, scale_of(d)).reshape(b, h, n)
            q[..., j] = q[..., i] * near
            k[:, :, 0, i] = k[:, :, 1, j] = size
        else:
            q[..., i] = q[..., j] = shallow(d)
            k[:, :, 0, i] = deep(rng, b * kv).reshape(b, kv) * size
            k[:, :, 1, j] = k[:, :, 0, i] * near
        v[:, :, 0] = 1
    return q, k, v, np.full(b, 2, F)


def scores(spec, q, k):
    """[batch, heads, queries, 2] in 64 bits."""
    k = np.repeat(k[:, :, :2].astype(np.float64), spec["heads"] // spec["kv_heads"], axis=1)
    return q.astype(np.float64) @ np.swapaxes(k, 2, 3) / np.sqrt(spec["dim"])


def want(spec, case, q, k, v):
    """The outputs, all of a row alike but for case v, and how far FP32 may be off."""
    if case == "v":
        out = np.repeat(v[:, :, :1].astype(np.float64), spec["heads"] // spec["kv_heads"], axis=1)
        out = np.broadcast_to(out, q.shape)
        return out, 2 * U * np.abs(out)  # the sum's reciprocal and the product with it
    s = scores(spec, q, k)
    one = 0 if case in "qk" else 1  # the key whose value is 1
    gap = s[..., 1 - one] - s[..., one]
    out = 1 / (1 + np.exp(gap))
    # Scores: the query's scaling 1, the products left out 1, the last sum 2 (it may be cut off); the scale's own
    # roundings are common to both scores, 4 of their gap, and taking off the maximum is 1 of it. Two exponentials of
    # 2 each, their sum 1, its reciprocal 1 and the product with it 1.
    off = 4 * (np.abs(s[..., 0]) + np.abs(s[..., 1])) + 5 * np.abs(gap)
    off = U * out * ((1 - out) * (1.01 * off + 4) + 3)
    shape = q.shape
    return np.broadcast_to(out[..., None], shape), np.broadcast_to(off[..., None], shape)


def simulate(spec, case, q, k, v, count):
    """The case with `count` parts of its deep operand, the rest in 64 bits."""
    def cut(x):
        return sum(p.astype(np.float64) for p in parts(x, count))

    if case == "v":
        return np.broadcast_to(np.repeat(cut(v[:, :, :1]), spec["heads"] // spec["kv_heads"], axis=1), q.shape)
    if case == "q":
        q = cut((q * scale_of(spec["dim"])).astype(F)) / float(scale_of(spec["dim"]))
    if case == "k":
        k = cut(k)
    s = scores(spec, q, k)
    p = np.exp(s - s.max(axis=-1, keepdims=True))
    one = p[..., 0] if case in "qk" else cut(p[..., 1].astype(F)) if case == "p" else p[..., 1]
    return np.broadcast_to((one / p.sum(axis=-1))[..., None], q.shape)
