"""The 4-bit KV cache in numpy: its layout, the quantizer's rule in f32 steps, attention over it in f64 and the eviction by weight
(not collected by pytest)."""
import numpy as np

LARGEST = 65504.0
SHIFTS = np.array([0, 16, 4, 20, 8, 24, 12, 28], np.uint32)


def quantize(x):
    """[.., 32 k] f32 -> (quants 0 .. 15, f16 scales [.., k]), every step one f32 operation."""
    b = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        high, low = b.max(-1, keepdims=True), b.min(-1, keepdims=True)
        d = np.where(high >= -low, high, low) * np.float32(-0.125)
        fits = np.all(np.abs(b) <= LARGEST, -1, keepdims=True)  # (false for NaN)
        held = np.where(fits, d, np.float32(np.nan)).astype(np.float16)
        held[held == 0] = 0  # (no sign)
        full = np.abs(held) > 0
        t = np.where(full, b * (np.float32(1) / np.where(full, d, np.float32(1))), np.float32(0))
        q = np.minimum((t + np.float32(8.5)).astype(np.int32), 15)
    return q.reshape(x.shape).astype(np.uint8), held[..., 0]


class Cache:
    """One cache of max_seq rows as the library lays it out."""

    def __init__(self, max_seq, n_kv, hd, fill=0xff):
        self.max_seq, self.n_kv, self.hd = max_seq, n_kv, hd
        self.raw = np.full(n_kv * max_seq * (hd // 2 + hd // 16), fill, np.uint8)  # (0xff: a row that is not written holds NaN)

    @property
    def words(self):
        return self.raw[:self.n_kv * self.max_seq * self.hd // 2].view(np.uint32).reshape(self.n_kv, self.max_seq, self.hd // 8)

    @property
    def scales(self):
        return self.raw[self.n_kv * self.max_seq * self.hd // 2:].view(np.float16).reshape(self.n_kv, self.max_seq, self.hd // 32)

    def append(self, row, x):
        """x: [n][n_kv][hd]; rows past the end are dropped."""
        x = x[:max(0, self.max_seq - row)]
        q, d = quantize(x)
        w = (q.reshape(*q.shape[:-1], -1, 8).astype(np.uint32) << SHIFTS).sum(-1, dtype=np.uint32)
        self.words[:, row:row + len(x)] = w.transpose(1, 0, 2)
        self.scales[:, row:row + len(x)] = d.transpose(1, 0, 2)

    def values(self, row, n):
        """[n_kv][n][hd] in f64."""
        q = (self.words[:, row:row + n, :, None] >> SHIFTS) & np.uint32(15)
        q = q.reshape(self.n_kv, n, self.hd // 32, 32).astype(np.float64) - 8
        with np.errstate(invalid="ignore"):
            return (q * self.scales[:, row:row + n].astype(np.float64)[..., None]).reshape(self.n_kv, n, self.hd)


def attention(q, k, v, pos0):
    """q [n][heads][hd] over Cache k, v at rows pos0 ..: (out [n][heads][hd], softmax weights [heads][n][pos0 + n]) in f64."""
    n, heads, hd = q.shape
    group = heads // k.n_kv
    kk, vv = k.values(0, pos0 + n), v.values(0, pos0 + n)
    out, weights = np.zeros((n, heads, hd)), np.zeros((heads, n, pos0 + n))
    with np.errstate(invalid="ignore"):
        for h in range(heads):
            s = q[:, h].astype(np.float64) @ kk[h // group].T / np.sqrt(hd)
            for j in range(n):  # every token over its own rows alone
                seen = pos0 + j + 1
                e = np.exp(s[j, :seen] - s[j, :seen].max())
                weights[h, j, :seen] = e / e.sum()
            out[:, h] = weights[h] @ vv[h // group] if np.isfinite(vv[h // group]).all() else np.stack(
                [weights[h, j, :pos0 + j + 1] @ vv[h // group][:pos0 + j + 1] for j in range(n)])
    return out, weights


def gathered(weights, n_kv):
    """[n_kv][rows] of attention()'s weights."""
    heads, _, rows = weights.shape
    return weights.reshape(n_kv, heads // n_kv, -1, rows).sum((1, 2))


def evicted(w, seq, keep, recent, drop):
    """The rows of one head that stay: of [keep, seq - recent) the `drop` of least weight leave, of equal ones the lower, NaN first."""
    order = sorted(range(keep, seq - recent), key=lambda r: (0, 0.0, r) if np.isnan(w[r]) else (1, w[r], r))
    gone = set(order[:drop])
    return np.array([r for r in range(seq) if r not in gone], np.uint32)
