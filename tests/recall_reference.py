"""Rotary positions, room for tokens and the choice of blocks from their definitions, in 64 bits or whole numbers on the CPU."""
import numpy as np

MOST, POWER = 127, 40


def turned(x, positions, turn, amplitude, layout, back=False):
    """x (rows, heads, dim) with its pairs turned, as complex numbers."""
    x = np.array(x, np.float64)
    half = len(turn)
    one, two = (slice(0, half), slice(half, 2 * half)) if layout == 'half' else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    # the angle in extended precision: its own rounding is not to count
    angle = np.asarray(positions, np.longdouble)[:, None, None] * np.asarray(turn, np.longdouble) * (-1 if back else 1)
    angle = np.remainder(angle, 2 * np.arctan2(np.longdouble(0), np.longdouble(-1))).astype(np.float64)
    z = (x[..., one] + 1j * x[..., two]) * (amplitude * np.exp(1j * angle))
    x[..., one], x[..., two] = z.real, z.imag
    return x


def codes(x):
    """Whole numbers and exponents of x along its last axis, one vector at a time; NaN counts as 0."""
    x = np.where(np.isnan(x), 0.0, np.asarray(x, np.float64))
    most = np.abs(x).max(-1)
    e = np.full(most.shape, -POWER)
    for _ in range(2 * POWER):
        e += (most > MOST * 2.0 ** e) & (e < POWER)
    c = np.clip(np.rint(np.clip(x, -1e300, 1e300) * 2.0 ** -e[..., None]), -MOST, MOST)
    return c.astype(np.int64), e


def summary(keys):
    """Codes (dim,) and byte of a block's keys (tokens, dim)."""
    if not np.isfinite(keys).all():
        return np.zeros(keys.shape[1], np.int64), 255
    c, e = codes(keys.mean(0))
    return c, int(e) + 127


def blocks_of(q, k, position, length, block, top, near, first, causal, missing=()):
    """The blocks of one query (group, dim) with a world's keys of one head (length, dim), ascending; `missing`: blocks whose
    pages are not there."""
    if position < 0:
        return []
    high = min(position + 1, length) if causal else length
    blocks = -(-high // block)
    near_from = min(max(0, position // block - near + 1), blocks)
    always = set(range(min(first, near_from))) | set(range(near_from, blocks))
    rest = [b for b in range(blocks) if b not in always]
    if len(rest) > top:
        c, e = codes(q)
        scores = []
        for b in rest:
            s, byte = summary(k[b * block:(b + 1) * block])
            score = max(int(np.dot(c[h], s)) * 2.0 ** float(e[h] + byte - 127) for h in range(len(q)))
            scores.append(-np.inf if b in missing else np.inf if byte == 255 else score)
        order = sorted(range(len(rest)), key=lambda i: (-scores[i], i))
        rest = [rest[i] for i in order[:top]]
    return sorted(always | set(rest))


class Books:
    """What a room's tables, lengths and stack of free pages should be."""

    def __init__(self, table, length, free, tokens, page):
        self.table, self.length, self.free, self.tokens, self.page = table.copy(), length.astype(int).copy(), list(free), tokens, page
        self.why = 0

    def _give(self, w, keep):
        """Pages of world w from `keep` on, in their order."""
        held = -(-self.length[w] // self.page)
        pages = [int(x) for x in self.table[w, keep:held]]
        self.table[w, keep:held] = -1
        return pages

    def change(self, count, over=None, rows=2 ** 31 - 1):
        n, page = len(self.length), self.page
        over = np.zeros(n, bool) if over is None else over
        base = np.where(over, 0, self.length)
        after = base + count
        reach = min(self.tokens, self.table.shape[1] * page)
        why = 1 if np.any((after < 0) | ((count > 0) & (after > reach))) else 0
        fits = np.where((after < 0) | ((count > 0) & (after > reach)), base, after)
        held, kept, need = -(-self.length // page), -(-np.minimum(base, fits) // page), -(-fits // page)
        if (need - kept).sum() > len(self.free) + (held - kept).sum():
            why |= 2
        if np.maximum(count, 0).sum() > rows:
            why |= 4
        back = []
        for w in range(n):
            keep = (0 if over[w] else held[w]) if why else kept[w]
            back += self._give(w, keep)
            self.length[w] = base[w] if why else fits[w]
        self.free += back[::-1]
        self.why |= why
        if why:
            return np.zeros(n + 1, int)
        for w in range(n):
            for i in range(kept[w], need[w]):
                self.table[w, i] = self.free.pop()
        return np.concatenate([[0], np.cumsum(np.maximum(count, 0))])
