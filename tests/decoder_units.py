"""Attention of a decoder's step a (sequence, kv head) at a time in 64 bits, and how the ragged kernels cut their work.

The kernels cut all key tiles of all (sequence, kv head, row block)s, their units, into runs of equal length, one a
block; a cut goes to a unit's nearest end where a run has four or more of that sequence's units."""
import numpy as np

import decoder_oracle as dec
import jade_hip


def attend(q, k, v, sees=None):
    """Rows q over the keys, or of those the ones that `sees` [rows, keys] has: outputs and the bound of
    decoder_oracle.attend."""
    n, d = len(k), q.shape[1]
    if not n:
        return np.zeros_like(q), np.zeros_like(q)
    scores, sizes = q @ k.T / np.sqrt(d), np.abs(q) @ np.abs(k).T / np.sqrt(d)
    count = np.full(len(q), n)
    if sees is not None:
        scores[~sees], sizes[~sees], count = -np.inf, 0, sees.sum(axis=1)
    none = count == 0
    top = np.where(none, 0, scores.max(axis=1))
    p = np.exp(scores - top[:, None])
    p /= np.where(none, 1, p.sum(axis=1))[:, None]
    bound = dec.U * (2 * (2 * (d + 2) * sizes.max(axis=1) + 4) + 2 * count + 16)
    return p @ v, bound[:, None] * (p @ np.abs(v))


def unit(spec, x, b, kv):
    """Outputs and bounds [group, rows, dim] of sequence b's heads of one kv head."""
    tree = "nodes" in spec
    tm, group = spec["token_major"], spec["heads"] // spec["kv_heads"]
    rows, most = (spec["nodes"], spec["capacity"]) if tree else (spec["queries"], spec["keys"])

    def of(name, head):
        y = x[name][b]
        return (y[:, head] if tm else y[head]).astype(np.float64)

    n = dec.length_of(x["lengths"][b], most)
    q = np.concatenate([of("q", kv * group + g) for g in range(group)])
    k, v = (of(name, kv)[:n] for name in (("k_cache", "v_cache") if tree else ("k", "v")))
    sees = None
    if tree:
        k, v = np.concatenate([k, of("k_draft", kv)]), np.concatenate([v, of("v_draft", kv)])
        sees = np.zeros((rows, n + rows), bool)
        for m, seen in enumerate(dec.ancestors(x["parents"][b])):
            if seen:
                sees[m, :n] = True
                sees[m, n + np.array(seen)] = True
        sees = np.tile(sees, (group, 1))
    out, off = attend(q, k, v, sees)
    return out.reshape(group, rows, -1), off.reshape(group, rows, -1)


def check(spec, x, got, units):
    """`got` of the (sequence, kv head)s named, against 64 bits."""
    got, group = got.reshape(x["q"].shape), spec["heads"] // spec["kv_heads"]
    for b, kv in units:
        mine = got[b][:, kv * group:(kv + 1) * group].swapaxes(0, 1) if spec["token_major"] else got[b][kv * group:(kv + 1) * group]
        want, off = unit(spec, x, b, kv)
        over = np.abs(mine.astype(np.float64) - want) - off
        assert np.isfinite(mine).all() and over.max() <= 0, (b, kv, over.max(), off.max())


class Cuts:
    """How a launch is cut: `chunk` tiles a run, cuts that were `moved` to a unit's end, cuts `inside` a unit, `whole`
    units of two tiles or more that a run has to itself, and the most tiles of a unit in one run (`longest`)."""

    def __init__(self, spec, lengths):
        launch = jade_hip.spec_describe(spec)["launch"]
        self.kernel, runs = launch["kernel"], launch["grid"][0]
        tree, parts = "nodes" in spec, "parts" in self.kernel
        tile, block = (128, int(self.kernel.rsplit("_r", 1)[1])) if parts else (64, 16)
        rows = spec["heads"] // spec["kv_heads"] * (spec["nodes"] if tree else spec["queries"])
        units = spec["kv_heads"] * -(-rows // block)
        most, drafted = (spec["capacity"], -(-spec["nodes"] // tile)) if tree else (spec["keys"], 0)
        tiles = np.array([-(-dec.length_of(n, most) // tile) + drafted for n in lengths])
        before = np.concatenate([[0], np.cumsum(tiles)])
        total = int(before[-1]) * units
        self.chunk = -(-total // runs)
        starts = [0, total]
        self.moved = self.inside = 0
        for t in range(self.chunk, total, self.chunk):
            b = int(np.searchsorted(before, t // units, "right")) - 1
            mine = int(tiles[b])
            over = (t - int(before[b]) * units) % mine
            if 4 * mine <= self.chunk:
                self.moved += over != 0
                t += mine - over if 2 * over >= mine else -over
            else:
                self.inside += over != 0
            starts.append(t)
        starts = np.unique(starts)
        some = [b for b in range(len(tiles)) if tiles[b]]
        ends = np.concatenate([before[b] * units + tiles[b] * np.arange(1, units + 1) for b in some])
        begins = np.concatenate([before[b] * units + tiles[b] * np.arange(units) for b in some])
        self.longest = int(np.diff(np.union1d(ends, starts), prepend=0).max())
        own = np.searchsorted(starts, begins, "right") == np.searchsorted(starts, ends, "left")
        self.whole = int((own & (ends - begins > 1)).sum())
