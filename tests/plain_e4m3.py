"""Plain NumPy statement, in 64 bits, of the 8-bit cache: codes, the scale of a block, storing, attention, eviction.

Nothing is imported from the package.  A cache here is a list of rows per head kept with its block scales: `Rows` of one
(sequence, key/value head, plane) holds codes [rows, channels] (as the numbers they stand for) and one scale per 64 rows."""
import numpy as np

PAGE = 64


def nearest(x):
    """The nearest e4m3 number to each x, ties to the even mantissa: steps of 2^(e - 3) between 2^e and 2^(e + 1), of 2^-9
    below 2^-6.  What is not finite becomes NaN.  (No |x| here exceeds 448.)"""
    x = np.asarray(x, dtype=np.float64)
    ok = np.isfinite(x)
    y = np.where(ok, x, 0.0)
    _, e = np.frexp(y)                                    # |y| in [2^(e - 1), 2^e)
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    y = np.rint(y / step) * step
    return np.where(ok, y, np.nan)


def needed(values):
    """The least 2^k, k >= -126, with max |finite value| <= 448 * 2^k."""
    v = np.abs(np.asarray(values, dtype=np.float64))
    v = v[np.isfinite(v)]
    most = float(v.max()) if v.size else 0.0
    k = -126
    while most > 448.0 * 2.0 ** k:
        k += 1
    return 2.0 ** k


def rotate(x, cos, sin, pairing="half"):
    """x [..., channels] with the first 2 * len(cos) channels turned in pairs."""
    x = np.array(x, dtype=np.float64)
    half = len(cos)
    a, b = (x[..., :half], x[..., half:2 * half]) if pairing == "half" else (x[..., 0:2 * half:2], x[..., 1:2 * half:2])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    if pairing == "half":
        x[..., :half], x[..., half:2 * half] = ra, rb
    else:
        x[..., 0:2 * half:2], x[..., 1:2 * half:2] = ra, rb
    return x


class Rows:
    def __init__(self, channels):
        self.codes = np.zeros((0, channels))
        self.scales = []

    def append(self, x):
        """Store the rows x [n, channels]: one step's."""
        x = np.asarray(x, dtype=np.float64)
        at = 0
        while at < len(x):
            n_old = len(self.codes)
            inside = n_old % PAGE
            take = min(PAGE - inside, len(x) - at)
            s = needed(x[at: at + take])
            if inside:
                before = self.scales[-1]
                s = max(s, before)
                self.codes[n_old - inside:] = nearest(self.codes[n_old - inside:] * (before / s))
                self.scales[-1] = s
            else:
                self.scales.append(s)
            self.codes = np.concatenate([self.codes, nearest(x[at: at + take] / s)])
            at += take

    def values(self):
        return self.codes * np.repeat(np.asarray(self.scales), PAGE)[: len(self.codes), None]

    def keep(self, rows):
        """Only these rows (ascending) stay; blocks none of whose rows move are left as they are."""
        v = self.values()
        codes, scales = [], []
        for lo in range(0, len(rows), PAGE):
            part = list(rows[lo: lo + PAGE])
            if part == list(range(lo, lo + len(part))):
                codes.append(self.codes[part])
                scales.append(self.scales[lo // PAGE])
                continue
            s = needed(v[part])
            codes.append(nearest(v[part] / s))
            scales.append(s)
        self.codes, self.scales = np.concatenate(codes), scales


def attend(q, k, v, first_row, scale, window=0):
    """q [n, heads of one key head, channels] at rows first_row, ...; k, v [rows, channels].  Returns the outputs and the weight
    each row gathers."""
    q, k, v = (np.asarray(t, dtype=np.float64) for t in (q, k, v))
    out, gathered = np.zeros(q.shape), np.zeros(len(k))
    for i in range(q.shape[0]):
        row = first_row + i
        lo = max(0, row - window + 1) if window else 0
        for g in range(q.shape[1]):
            s = (k[lo: row + 1] @ q[i, g]) * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, g] = p @ v[lo: row + 1]
            gathered[lo: row + 1] += p
    return out, gathered


def chosen(weights, budget, recent):
    """Rows that stay of len(weights): the newest, and the heaviest of the others (the lower row on a tie)."""
    n = len(weights)
    if n <= budget:
        return list(range(n))
    order = sorted(range(n - recent), key=lambda i: (-weights[i], i))
    return sorted(order[: budget - recent]) + list(range(n - recent, n))
