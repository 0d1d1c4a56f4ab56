"""The 8-bit K/V pages and their attention in 64 bits, for the tests: codes and scales by the definition, a position at a
time, with the tolerance that the arithmetic of an f32 attention allows."""
import numpy as np

PAGE, BLOCK, LOW, HIGH = 64, 16, -48, 63


def step_of(top):
    """The least power of two 2^e, e >= LOW, with top <= 127 x 2^e; NaN where there is none up to HIGH."""
    if not np.isfinite(top):
        return np.nan
    e = LOW
    while top > 127.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e if e <= HIGH else np.nan


class Cache:
    """Values (in 64 bits) and steps of the slots' positions."""

    def __init__(self, kv, hd):
        self.kv, self.hd, self.slots = kv, hd, {}

    def _slot(self, slot):
        return self.slots.setdefault(slot, {"n": 0, "k": [], "v": []})   # k, v: [block] -> (codes [16, kv, hd], step [kv])

    def append(self, slot, pos, k, v):
        """k, v [rows, kv, hd] in 64 bits at positions pos.. (the positions from pos on are dropped first)."""
        s = self._slot(slot)
        assert pos <= s["n"]
        for name, x in (("k", k), ("v", v)):
            blocks = s[name]
            for b in range(pos // BLOCK, (pos + len(x) + BLOCK - 1) // BLOCK if len(x) else 0):
                old = max(0, pos - b * BLOCK)
                new = x[max(0, b * BLOCK - pos):max(0, (b + 1) * BLOCK - pos)]
                step = np.array([step_of(np.abs(new[:, h]).max()) for h in range(self.kv)])
                codes = np.zeros((BLOCK, self.kv, self.hd))
                if old:
                    was, was_step = blocks[b]
                    step = np.where(np.isnan(step) | np.isnan(was_step), np.nan, np.maximum(step, was_step))
                    codes[:old] = np.rint(was[:old] * (was_step / step)[:, None])
                with np.errstate(invalid="ignore", over="ignore"):
                    codes[old:old + len(new)] = np.rint(new / step[:, None])
                del blocks[b + 1:]
                blocks[b:] = [(codes, step)]
        if len(k):
            s["n"] = pos + len(k)

    def values(self, slot, name, first, count):
        blocks = self._slot(slot)[name]
        x = np.concatenate([c * s[:, None] for c, s in blocks]) if blocks else np.zeros((0, self.kv, self.hd))
        return x[first:first + count]

    def steps(self, slot, name):
        """[block, kv]"""
        return np.stack([s for _, s in self._slot(slot)[name]])


def normed(x, w, eps, form):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (w + 1.0 if form else w)


def turned(x, rope, pos):
    """x [rows, heads, hd] at positions pos..; rope [ctx, hd/2, 2] of (cos, sin)."""
    half = x.shape[-1] // 2
    cs = rope[pos:pos + len(x)].astype(np.float64)[:, None]
    a, b, c, s = x[..., :half], x[..., half:], cs[..., 0], cs[..., 1]
    return np.concatenate((a * c - b * s, a * s + b * c), -1)


def attention(q, k, v, pos, scale, window, steps):
    """q [rows, heads, hd] at positions pos.. over k, v [positions, kv, hd], `steps` [positions, kv] those of v's blocks:
    the output and how far the attention may be from it.

    With u = 2^-24: a score's products and sums round hd + 4 times at most, the halves of q leave 2^-22 of each value, so
    a score is off by at most d = scale x sum|q k| x ((hd + 4) u + 2^-22), and the exponent's argument (in base 2, after
    it is scaled and the block's exponent, at most 64 here, is added) rounds three times. A weight is then off by the
    relative d + 3 u x (|s| + 64) x 1.5 + 2^-21 (exp2, the halves of the weight, the scales); the sums over n positions
    round n times. Numerator and denominator both carry that.

    A weight times its block's step is held in two f16 halves, scaled so that the largest of the row lies in (2^13, 2^14]:
    where the halves reach f16's subnormals, which are 2^-24 apart, it is off by up to 2^-25, that is 2^-38 of the largest;
    each of the n positions' codes, 127 at most, may carry that."""
    rows, heads, hd = q.shape
    kv, u = k.shape[1], 2.0 ** -24
    out, tol = np.zeros((rows, heads, hd)), np.zeros((rows, heads, hd))
    for i in range(rows):
        lo = max(0, pos + i + 1 - window) if window else 0
        for h in range(heads):
            kk, vv = k[lo:pos + i + 1, h * kv // heads], v[lo:pos + i + 1, h * kv // heads]
            s = kk @ q[i, h] * scale
            big = (np.abs(kk) @ np.abs(q[i, h]) * abs(scale)).max()
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ vv
            rel = big * ((hd + 4) * u + 2.0 ** -22) + 4.5 * u * (np.abs(s).max() * 1.5 + 64) + 2.0 ** -21 + (len(kk) + 8) * u
            held = (p * steps[lo:pos + i + 1, h * kv // heads]).max()
            tol[i, h] = 2 * rel * (p @ np.abs(vv)) + len(kk) * 127 * 2.0 ** -38 * held + 1e-30
    return out, tol
