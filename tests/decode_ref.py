"""The decode operators' definitions in 64 bits, for tests: numpy, one value after another."""
import numpy as np

from ztensor_amd import _lib

F24 = 2.0 ** -24  # half a unit in the last place of 1, fp32


def padded(dim):
    return -(-dim // 64) * 64


def turn(x, positions, table, interleaved=False, inverse=False, dtype=np.float64):
    """x [T, H, D] turned; in float32 each product and sum is rounded by itself."""
    half = table.shape[2]
    y = x.astype(dtype).copy()
    c, s = table[positions, 0].astype(dtype)[:, None], table[positions, 1].astype(dtype)[:, None]
    s = -s if inverse else s
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = y[..., first].copy(), y[..., second].copy()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y


class Cache:
    """The cache on the host: codes [pages, heads, page, dim] of keys and values, and their scales, in float32."""

    def __init__(self, pages, heads, dim, page, rng=None):
        shape = (2, pages, heads, page, dim)
        self.dim, self.page = dim, page
        self.codes = np.zeros(shape, np.int8) if rng is None else rng.integers(-127, 128, shape).astype(np.int8)
        self.scales = (np.zeros(shape[:3], np.float32) if rng is None
                       else (0.02 * np.exp(0.5 * rng.standard_normal(shape[:3]))).astype(np.float32))

    def device(self, torch):
        k = np.zeros((*self.codes.shape[1:4], padded(self.dim)), np.int8)
        v = k.copy()
        k[..., :self.dim], v[..., :self.dim] = self.codes
        t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
        return t(k), t(v.transpose(0, 1, 3, 2)), t(self.scales[0]), t(self.scales[1])

    def append(self, x, slots):
        """x: keys and values [2][T, heads, dim] float32, in float32 arithmetic as the definition has it."""
        f = np.float32
        by_page = {}
        for t, s in enumerate(slots):
            if 0 <= s < self.codes.shape[1] * self.page:
                by_page.setdefault(s // self.page, []).append((t, s % self.page))
        for page, at in by_page.items():
            ts, places = [t for t, _ in at], [p for _, p in at]
            for kind in range(2):
                for h in range(self.codes.shape[2]):
                    new = x[kind][ts, h].astype(f)
                    had = f(0) if 0 in places else self.scales[kind, page, h]
                    peak = np.abs(new).max()
                    ok = np.isfinite(peak) and np.isfinite(had)
                    now = np.maximum(had, peak * f(1.0 / 127.0)) if ok else f(np.nan)
                    codes = self.codes[kind, page, h].astype(f)
                    if 0 in places:
                        codes[:] = 0
                    elif now > had:
                        codes = np.rint(codes * (had / now))
                    if ok:
                        codes[places] = np.clip(np.rint(new / (now if now > 0 else f(1))), -127, 127)
                        self.codes[kind, page, h] = codes.astype(np.int8)
                    self.scales[kind, page, h] = now

    def values(self):
        return self.codes.astype(np.float64) * self.scales.astype(np.float64)[..., None, None]


def attend(q, cache, table, lens, starts, window=0, scale=None):
    """(out, the largest of the rows' sums of |q k| times the scale, the values' largest) in 64 bits."""
    out = np.zeros(q.shape)
    kv = cache.values()
    scale = 1.0 / np.sqrt(q.shape[2]) if scale is None else scale
    group, most, big = q.shape[1] // cache.codes.shape[2], 0.0, 0.0
    for r, size in enumerate(lens):
        n = starts[r + 1] - starts[r]
        for i in range(n):
            hi = size - n + i + 1
            seen = [t for t in range(max(0, hi - window) if window else 0, hi)
                    if 0 <= table[r, t // cache.page] < cache.codes.shape[1]]
            if not seen:
                continue
            pages, places = [table[r, t // cache.page] for t in seen], [t % cache.page for t in seen]
            keys, values = kv[0][pages, :, places], kv[1][pages, :, places]  # [seen, heads, dim]
            row = q[starts[r] + i].astype(np.float64)
            with np.errstate(invalid="ignore"):
                for h in range(q.shape[1]):
                    s = keys[:, h // group] @ row[h] * scale
                    most = max(most, np.nan_to_num(np.abs(keys[:, h // group]) @ np.abs(row[h]) * scale).max())
                    p = np.exp(s - s.max())
                    out[starts[r] + i, h] = (p / p.sum()) @ values[:, h // group]
            big = max(big, np.nan_to_num(np.abs(values)).max())
    return out, most, big


def attend_bound(out, most, big, half):
    """How far a kernel's output may be: operands in 22 bits or more and fp32 sums in chains of at most 16 and 64 terms
    (each rounding of the scores shifts a weight by that times the score's terms, twice over numerator and sum), the
    weights' and the output's own rounding in 11 bits for fp16."""
    err = big * 2.0 ** -20 * (2 + most)
    return err + (big * 2.0 ** -11 + np.abs(out) * 2.0 ** -11 if half else 0)


def plan(lens, add, table, free, page):
    """The bookkeeping of a step, one request after another."""
    table, free = table.copy(), list(free)
    lens, add = [max(0, int(x)) for x in lens], [max(0, int(x)) for x in add]
    slots, positions, starts, out, short = [], [], [0], [], False
    for r, (held, n) in enumerate(zip(lens, add)):
        have, want = -(-held // page), -(-(held + n) // page)
        fits = held + n <= table.shape[1] * page
        if fits and want > have and (short or want - have > len(free)):
            short = True
        ok = fits and (want == have or not short)
        if ok:
            for j in range(have, want):
                table[r, j] = free.pop()
        for p in range(held, held + n):
            positions.append(p)
            slots.append(table[r, p // page] * page + p % page if ok and table[r, p // page] >= 0 else -1)
        starts.append(starts[-1] + n)
        out.append(held + n if ok else held)
    return table, slots, positions, starts, out, len(free)


def kept(z, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(the order of the tokens that stay, the weight of each token) in 64 bits."""
    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    order = np.argsort(-z, kind="stable")
    with np.errstate(invalid="ignore"):
        w = np.where(z == z.max(), 1.0, np.exp((z - z.max()) / (temperature if temperature > 0 else 1.0)))
    n = len(z) if top_k <= 0 or top_k > len(z) else top_k
    n = 1 if not temperature > 0 else min(n, int((w >= min(min_p, 1.0)).sum()))
    if top_p < 1:
        mass = np.cumsum(w[order[:n]])
        n = min(n, int((mass < top_p * mass[-1]).sum()) + 1)
    return order[:n], w


def rows(t, heads=None):
    return _lib.Rows(t.data_ptr(), t.stride(0), t.stride(1), heads or t.shape[1], 0)
