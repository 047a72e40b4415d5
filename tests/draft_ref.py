"""Definitions of the operators of drafted trees, shared pages and normed heads,
for tests: numpy, one value after another."""
import numpy as np


def normed(x, w, eps, dtype=np.float64):
    """Each head of x [T, H, D] over its root mean square, times w (None: ones); in float32 the factor (of a 64-bit sum)
    and both products are rounded by themselves."""
    y = x.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        r = 1.0 / np.sqrt(np.sum(y * y, -1, keepdims=True) / x.shape[-1] + eps)
        y = x.astype(dtype) * r.astype(dtype)
        return y if w is None else y * w.astype(dtype)


def ancestors(parents, n):
    """Of each row the rows above it, itself first; a parent that is no earlier row is none."""
    out = []
    for i in range(n):
        at, chain = i, []
        while at >= 0:
            chain.append(at)
            p = int(parents[at])
            at = p if 0 <= p < at else -1
        out.append(chain)
    return out


def tree(parents, lens, starts, tokens, words):
    positions, mask = np.zeros(tokens, np.int64), np.zeros((tokens, words), np.uint64)
    for r, size in enumerate(lens):
        lo, n = starts[r], starts[r + 1] - starts[r]
        for i, chain in enumerate(ancestors(parents[lo:lo + n], n)):
            positions[lo + i] = max(0, max(0, size) - n + len(chain) - 1)
            for j in chain:
                if j < 64 * words:
                    mask[lo + i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return positions, mask.view(np.int64)


def bits(mask, n):
    """[rows, n] of truth values; what is past the words is not set."""
    b = (mask.view(np.uint64)[:, :, None] >> np.arange(64, dtype=np.uint64)) & np.uint64(1)
    b = b.reshape(len(mask), -1) > 0
    return np.pad(b, ((0, 0), (0, max(0, n - b.shape[1]))))[:, :n]


def attend(q, cache, table, lens, starts, mask, window=0, scale=None):
    """decode_ref.attend's values for rows that see their context and what their masks say."""
    out = np.zeros(q.shape)
    kv = cache.values()
    scale = 1.0 / np.sqrt(q.shape[2]) if scale is None else scale
    group, most, big = q.shape[1] // cache.codes.shape[2], 0.0, 0.0
    for r, size in enumerate(lens):
        n = starts[r + 1] - starts[r]
        context = size - n
        own = bits(mask[starts[r]:starts[r] + n], n) if n else np.zeros((0, 0), bool)
        for i in range(n):
            lo = context + int(own[i].sum()) - window if window else 0
            seen = [t for t in range(max(0, size)) if (t >= lo if t < context else own[i, t - context])]
            seen = [t for t in seen if 0 <= table[r, t // cache.page] < cache.codes.shape[1]]
            if not seen:
                continue
            pages, places = [table[r, t // cache.page] for t in seen], [t % cache.page for t in seen]
            keys, values = kv[0][pages, :, places], kv[1][pages, :, places]  # [seen, heads, dim]
            row = q[starts[r] + i].astype(np.float64)
            for h in range(q.shape[1]):
                s = keys[:, h // group] @ row[h] * scale
                most = max(most, (np.abs(keys[:, h // group]) @ np.abs(row[h]) * abs(scale)).max())
                p = np.exp(s - s.max())
                out[starts[r] + i, h] = (p / p.sum()) @ values[:, h // group]
            big = max(big, np.abs(values).max())
    return out, most, big


def accept(drafted, drawn, parents, starts, slots=None):
    """(path, kept, last, token), one row after another."""
    path, kept, last, token = np.full(len(drafted), -1), [], [], []
    for lo, hi in zip(starts, starts[1:]):
        n, rows = hi - lo, []
        if n > 0 and (slots is None or slots[lo] >= 0):
            at = 0
            while at is not None:
                rows.append(at)
                parent = lambda i: i - 1 if parents is None else parents[lo + i]  # noqa: E731
                at = next((i for i in range(at + 1, n) if parent(i) == at and drawn[lo + at] >= 0
                           and drafted[lo + i] == drawn[lo + at]), None)
        path[lo:lo + len(rows)] = rows
        kept.append(len(rows))
        last.append(lo + rows[-1] if rows else -1)
        token.append(drawn[lo + rows[-1]] if rows else -1)
    return path, kept, last, token


def compact(cache, table, held, starts, path, kept):
    """Moves rows in a decode_ref.Cache in float32 arithmetic, page after page; returns the lengths."""
    f = np.float32
    pages, size = cache.codes.shape[1], cache.page
    out = []
    for r, base in enumerate(held):
        lo, n = starts[r], starts[r + 1] - starts[r]
        m = min(max(0, kept[r]), n)
        out.append(base + m)
        by_page = {}
        for j in range(m):
            p = int(path[lo + j])
            if j < p < n and base + p < table.shape[1] * size:
                by_page.setdefault((base + j) // size, []).append(((base + j) % size, int(table[r, (base + p) // size]), (base + p) % size))
        for index in sorted(by_page):
            page = int(table[r, index])
            moves = [(z, a, b) for z, a, b in by_page[index] if 0 <= a < pages and 0 <= page < pages]
            for kind in range(2):
                for h in range(cache.codes.shape[2]):
                    scale = cache.scales[kind, :, h]
                    had = scale[page]
                    far = [(z, cache.codes[kind, a, h, b].astype(f) * scale[a]) for z, a, b in moves if a != page]
                    near = [(z, cache.codes[kind, page, h, b].astype(f)) for z, a, b in moves if a == page]
                    now = had
                    if far:
                        now = np.maximum(had, np.abs([x for _, x in far]).max().astype(f) * f(1.0 / 127.0))
                    codes = cache.codes[kind, page, h].astype(f)
                    for z, x in near:
                        codes[z] = x
                    if now > had:
                        codes = np.rint(codes * (had / now))
                    for z, x in far:
                        codes[z] = np.clip(np.rint(x / (now if now > 0 else f(1))), -127, 127)
                    cache.codes[kind, page, h] = codes.astype(np.int8)
                    scale[page] = now
    return out


def trim(lens, keep, table, free, pages, page, refs=None):
    """(table, the free list, holders besides one)."""
    table, free, refs = table.copy(), list(free), None if refs is None else list(refs)
    given = {}
    for r, (n, k) in enumerate(zip(lens, keep)):
        for j in range(min(table.shape[1], -(-max(0, k) // page)), min(table.shape[1], -(-max(0, n) // page))):
            p = int(table[r, j])
            if 0 <= p < pages:
                given[p] = given.get(p, 0) + 1
                table[r, j] = -1
    for p in sorted(given):
        if refs is None or given[p] > refs[p]:
            free.append(p)
            if refs is not None:
                refs[p] = 0
        else:
            refs[p] -= given[p]
    return table, free[:pages], refs


def fork(source, target, lens, table, free, page, refs):
    """(table, lens, the free list, refs, pages to copy from and to)."""
    old, lens_old = table, list(lens)
    table, lens, free, refs = table.copy(), list(lens), list(free), list(refs)
    copies, short = [], False
    for s, t in zip(source, target):
        copies.append((-1, -1))
        if not 0 <= t < len(lens) or s == t:
            continue
        n = lens_old[s] if 0 <= s < len(lens) else 0
        n = n if 0 < n <= table.shape[1] * page else 0
        table[t], lens[t] = -1, 0
        if n == 0:
            continue
        part = n % page > 0
        if part and (short or not free):
            short = True
            continue
        full = n // page
        table[t, :full] = old[s, :full]
        for p in old[s, :full]:
            if 0 <= p < len(refs):
                refs[p] += 1
        if part:
            table[t, full] = free.pop()
            copies[-1] = (int(old[s, full]), int(table[t, full]))
        lens[t] = n
    return table, lens, free, refs, [a for a, _ in copies], [b for _, b in copies]
