"""Drafted trees, shared pages and normed heads on the 8-bit paged cache, as cases that can be timed.

  norm    RMS norms of q's and k's heads and their rotary positions in one pass
  append  the same on the way into the cache: a step's keys normed, turned and
          stored, q normed and turned beside them
  attend  attention of the rows of a drafted tree over the cache: each row
          sees its sequence's context and, of the step's rows, those whose bits
          its mask has
  settle  a step's bookkeeping: the tree's positions and masks from its
          parents, the path that the drawn tokens accept, its keys and values
          moved to the context's end in the caches of some layers, and the
          pages behind it given back
  fork    sequences that go on from others: full pages shared, the last one
          copied in the caches of some layers

A cache of H key/value heads of size D in pages of B tokens is a tuple
  k        int8 [pages, H, B, Dp]   Dp: D to the next multiple of 64, zeros past D
  v        int8 [pages, H, Dp, B]
  k_scale  float32 [pages, H]       a value is its code times the scale
  v_scale  float32 [pages, H]
"""
from __future__ import annotations

import itertools
import math
import random

import torch

own = False

_DEV = "cuda"
_EPS = 1e-6
_LARGEST = 1.6e11  # operations of an attention that no drawn case exceeds
_CACHE = 48 * 4096 * 8 * 128  # values of keys that no drawn case's lengths exceed


def listed():
    return [
        # one token's q and k in an 8B model whose heads are normed: what a call costs
        {"name": "norm_token", "op": "norm", "dtype": "f32", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "interleaved": False, "max_pos": 8192},
        # a long prompt of a larger one, half of each head turned
        {"name": "norm_prompt", "op": "norm", "dtype": "f16", "tokens": 4099, "heads": 64, "kv_heads": 4, "dim": 128,
         "rot": 64, "interleaved": True, "max_pos": 32768},
        # 48 sequences each add a token to their last page
        {"name": "append_norm_batch", "op": "append", "dtype": "f32", "requests": 48, "new": 1, "context": 2500,
         "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "page": 32, "max_pos": 8192},
        # prompts of odd lengths
        {"name": "append_norm_prompts", "op": "append", "dtype": "f16", "requests": 3, "new": 1300, "context": 400,
         "heads": 40, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "page": 64, "max_pos": 8192},
        # the first drafts of a chat
        {"name": "attend_tree_short", "op": "attend", "dtype": "f32", "requests": 1, "nodes": 8, "context": 60,
         "ragged": False, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0},
        # one sequence deep into a long document, a wide tree in a 70B layer
        {"name": "attend_tree_long", "op": "attend", "dtype": "f16", "requests": 1, "nodes": 61, "context": 30011,
         "ragged": False, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64, "window": 0},
        # continuous batching: small trees of sequences of very different lengths
        {"name": "attend_tree_batch", "op": "attend", "dtype": "f32", "requests": 32, "nodes": 13, "context": 6000,
         "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "window": 0},
        # wide trees of many sequences: the largest case
        {"name": "attend_tree_large", "op": "attend", "dtype": "f16", "requests": 24, "nodes": 64, "context": 12000,
         "ragged": True, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64, "window": 0},
        # a step of a small server, two layers
        {"name": "settle_8", "op": "settle", "requests": 8, "nodes": 12, "context": 900, "kv_heads": 8, "dim": 128,
         "page": 64, "layers": 2, "refused": 0, "spare": 200},
        # a step of a large one, small pages, some requests without pages for their drafts
        {"name": "settle_128", "op": "settle", "requests": 128, "nodes": 48, "context": 700, "kv_heads": 8, "dim": 128,
         "page": 16, "layers": 2, "refused": 5, "spare": 3000},
        # four continuations of one answer
        {"name": "fork_4", "op": "fork", "sources": 1, "forks": 4, "context": 500, "kv_heads": 8, "dim": 128, "page": 16,
         "layers": 2, "spare": 100},
        # ten of each of 16 prompts, and not enough free pages for all of them
        {"name": "fork_160", "op": "fork", "sources": 16, "forks": 160, "context": 1500, "kv_heads": 8, "dim": 128,
         "page": 64, "layers": 4, "spare": 150},
    ]


def _log(rng, a, b):
    return min(b, max(a, round(math.exp(rng.uniform(math.log(a), math.log(b))))))


def draw(rng):
    op = rng.choice(["norm", "append", "append", "attend", "attend", "attend", "attend", "settle", "settle", "fork"])
    dtype = rng.choice(["f32", "f16"])
    dim = rng.choice([64, 128, 128, 128, 80, 96, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 7, 8])
    page = rng.choice([16, 32, 64, 128])
    rot = rng.choice([dim, dim, dim // 2])
    if op == "norm":
        return {"op": op, "dtype": dtype, "tokens": _log(rng, 1, 4096), "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "rot": rng.choice([rot, rot, rot, 0]), "interleaved": rng.random() < 0.5,
                "max_pos": _log(rng, 5000, 65536)}
    if op == "append":
        new = rng.choice([1, 1, _log(rng, 2, 2000)])
        return {"op": op, "dtype": dtype, "requests": _log(rng, 1, 128 if new == 1 else max(1, 4000 // new)),
                "new": new, "context": _log(rng, 1, 4000), "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
                "interleaved": rng.random() < 0.5, "page": page, "max_pos": 8192}
    if op == "settle":
        nodes = _log(rng, 1, 130)
        requests = _log(rng, 1, max(1, min(160, 4000 // nodes)))
        return {"op": op, "requests": requests, "nodes": nodes, "context": _log(rng, 1, 900), "kv_heads": kv_heads,
                "dim": dim, "page": page, "layers": rng.randint(1, 3), "refused": rng.choice([0, 0, requests // 4]),
                "spare": _log(rng, 1, 5000)}
    if op == "fork":
        sources = _log(rng, 1, 24)
        forks = _log(rng, 1, 160)
        return {"op": op, "sources": sources, "forks": forks, "context": _log(rng, 1, 1500), "kv_heads": kv_heads,
                "dim": dim, "page": page, "layers": rng.randint(1, 3), "spare": _log(rng, 1, 2 * forks)}
    window = rng.choice([0, 0, 0, _log(rng, 10, 4096)])
    nodes = rng.choice([_log(rng, 1, 16), _log(rng, 8, 64), _log(rng, 60, 150)])
    context = _log(rng, 1, 30000)
    most = min(_CACHE / (context * kv_heads * dim), _LARGEST / (4.0 * heads * dim * nodes * (context + nodes)))
    return {"op": op, "dtype": dtype, "requests": _log(rng, 1, max(1, min(64, int(most)))), "nodes": nodes,
            "context": context, "ragged": rng.random() < 0.6, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "window": window}


# ------------------------------------------------------------------ inputs


def _type(case):
    return torch.float16 if case["dtype"] == "f16" else torch.float32


def _lengths(case):
    """(tokens in the cache before the step, tokens that the step adds) of each request: the case's, whatever the seed."""
    rng = random.Random(17)
    r, context = case["requests"], case["context"]
    new = case["nodes"] if "nodes" in case else case["new"]
    if not case.get("ragged", True):
        return [context] * r, [new] * r
    # between a few tokens and the whole; the first request has the whole
    held = [context if i == 0 else max(0, int(context * rng.random() ** 2)) for i in range(r)]
    fresh = [new if i == 0 or new == 1 else max(1, round(new * rng.uniform(0.3, 1.0))) for i in range(r)]
    return held, fresh


def _trees(case):
    """Parents of each request's rows (-1: its first row) and the path that the drawn tokens will accept."""
    rng = random.Random(23)
    parents, paths = [], []
    for n in _lengths(case)[1]:
        p = [-1] + [rng.randint(max(0, i - 1 - min(i, 6)), i - 1) for i in range(1, n)]
        at, path = rng.randrange(n), []
        while at >= 0:
            path.append(at)
            at = p[at]
        parents.append(p)
        paths.append(path[::-1])
    return parents, paths


def _table(case):
    """float32 [positions, 2, rot / 2]: the cosines and sines of a position."""
    rot = case["rot"]
    freq = 500000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64, device=_DEV) / rot)
    angle = torch.arange(case["max_pos"], dtype=torch.float64, device=_DEV)[:, None] * freq
    return torch.stack((angle.cos(), angle.sin()), 1).float()


def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(seed * 1000003 + 11)


def _heads(case, tokens, g):
    """q, k and v as a step's fused projection gives them: slices of its rows."""
    n, m, d = case["heads"], case["kv_heads"], case["dim"]
    x = torch.randn(tokens, (n + 2 * m) * d, device=_DEV, generator=g)
    x[:, ::37] *= 4  # a few channels are larger
    x = x.to(_type(case))
    q, k, v = x.split([n * d, m * d, m * d], 1)
    return q.view(tokens, n, d), k.view(tokens, m, d), v.view(tokens, m, d)


def _weights(case, g):
    """Weights of the norms: near 1, a few much larger."""
    w = 1 + 0.3 * torch.randn(2, case["dim"], device=_DEV, generator=g)
    w[:, ::29] *= 3
    return w[0].contiguous(), w[1].contiguous()


def _cache(case, pages, g):
    h, b, d = case["kv_heads"], case["page"], case["dim"]
    dp = -(-d // 64) * 64

    codes = lambda *n: torch.randn(n, device=_DEV, generator=g).mul_(36).clamp_(-127, 127).round_().to(torch.int8)  # noqa: E731
    k, v = codes(pages, h, b, dp), codes(pages, h, dp, b)
    k[..., d:] = 0
    v[:, :, d:] = 0
    scale = lambda: 0.028 * torch.exp(0.3 * torch.randn(pages, h, device=_DEV, generator=g))  # noqa: E731
    return k, v, scale(), scale()


def _paged(lengths, page, seed, spare=0):
    """A block table over pages in no order, the number of pages, and those that are left."""
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 3 + spare
    order = list(range(pages))
    random.Random(seed + 3).shuffle(order)
    width = max(need) + 1
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return table, pages, order[at:]


def _int(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=_DEV)


def _starts(fresh):
    return [0, *itertools.accumulate(fresh)]


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "norm":
        t = case["tokens"]
        q, k, _ = _heads(case, t, g)
        first = random.Random(seed).randrange(case["max_pos"] - t)
        wq, wk = _weights(case, g)
        state = {"case": case, "q": q, "k": k, "wq": wq, "wk": wk, "positions": None, "table": None}
        if case["rot"]:
            state.update(positions=_int(list(range(first, first + t))), table=_table(case))
        return state
    if op == "fork":
        return _prepare_fork(case, seed, g)
    held, fresh = _lengths(case)
    b = case["page"]
    if op == "settle":
        return _prepare_settle(case, seed, g, held, fresh)
    lens = [h + n for h, n in zip(held, fresh)]
    table, pages, _ = _paged(lens, b, seed)
    if op == "append":
        slots = [table[r][p // b] * b + p % b for r, (h, n) in enumerate(zip(held, fresh)) for p in range(h, h + n)]
        positions = [p for h, n in zip(held, fresh) for p in range(h, h + n)]
        q, k, v = _heads(case, len(slots), g)
        wq, wk = _weights(case, g)
        return {"case": case, "q": q, "k": k, "v": v, "wq": wq, "wk": wk, "cache": _cache(case, pages, g),
                "slots": _int(slots, torch.int64), "positions": _int(positions), "table": _table(case),
                "touched": _int(sorted({s // b for s in slots}))}
    q = torch.randn(sum(fresh), case["heads"], case["dim"], device=_DEV, generator=g)
    q *= 1.5 * torch.exp(0.4 * torch.randn(sum(fresh), case["heads"], 1, device=_DEV, generator=g))
    state = {"case": case, "q": q.to(_type(case)), "cache": _cache(case, pages, g), "blocks": _int(table),
             "kv_lens": _int(lens), "q_start": _int(_starts(fresh)), "max_q": max(fresh), "max_kv": max(lens)}
    parents = _int(sum(_trees(case)[0], []))
    state["mask"] = _plain_tree(parents, state["kv_lens"], state["q_start"], max(fresh))[1]
    return state


def _prepare_settle(case, seed, g, held, fresh):
    b, r = case["page"], case["requests"]
    rng = random.Random(seed)
    parents, paths = _trees(case)
    lens = [h + (n if i < r - case["refused"] else 0) for i, (h, n) in enumerate(zip(held, fresh))]
    table, pages, rest = _paged([max(1, x) for x in lens], b, seed, case["spare"])
    slots, drafted, drawn, touched = [], [], [], set()
    for i, (h, n) in enumerate(zip(held, fresh)):
        took = lens[i] == h + n
        places = [table[i][p // b] * b + p % b if took else -1 for p in range(h, h + n)]
        tokens = [rng.randrange(32000) for _ in range(n)]
        answer = [rng.randrange(32000) if rng.random() < 0.6 else tokens[rng.randrange(n)] for _ in range(n)]
        for at, then in zip(paths[i], paths[i][1:]):
            answer[at] = tokens[then]
        slots += places
        drafted += tokens
        drawn += answer
        touched |= {s // b for s in places if s >= 0}
    free = rest[:case["spare"]]
    room = pages - len(free)  # the list has room for all pages
    return {"case": case, "parents": _int(sum(parents, [])), "held": _int(held), "kv_lens": _int(lens),
            "q_start": _int(_starts(fresh)), "slots": _int(slots, torch.int64), "drafted": _int(drafted, torch.int64),
            "drawn": _int(drawn, torch.int64), "blocks": _int(table), "free_pages": _int(free + [0] * room),
            "free_count": _int([len(free)]), "caches": [_cache(case, pages, g) for _ in range(case["layers"])],
            "touched": _int(sorted(touched) or [0]), "max_q": max(fresh)}


def _fork_lengths(case):
    rng = random.Random(29)
    lens = [case["context"]] + [max(1, int(case["context"] * rng.uniform(0.2, 1.0))) for _ in range(case["sources"] - 1)]
    return lens, [i % case["sources"] for i in range(case["forks"])]


def _prepare_fork(case, seed, g):
    lens, sources = _fork_lengths(case)
    table, pages, rest = _paged(lens, case["page"], seed, case["spare"])
    n = case["forks"]
    rows = list(range(len(lens) + n))
    random.Random(seed + 1).shuffle(rows)  # the sequences' rows of the block table, in no order
    blocks, kv_lens = [[-1] * len(table[0]) for _ in rows], [0] * len(rows)
    for i, x in enumerate(lens):
        blocks[rows[i]], kv_lens[rows[i]] = table[i], x
    free = rest[:case["spare"]]
    return {"case": case, "source": _int([rows[s] for s in sources]), "target": _int(rows[len(lens):]),
            "kv_lens": _int(kv_lens), "blocks": _int(blocks), "refs": torch.zeros(pages, dtype=torch.int32, device=_DEV),
            "free_pages": _int(free + [0] * (pages - len(free))), "free_count": _int([len(free)]),
            "caches": [_cache(case, pages, g) for _ in range(case["layers"])]}


# ------------------------------------------------------------------ the plain forms


def _rotate(x, row, interleaved):
    """x [tokens, heads, size] in 32 bits by the table's rows [tokens, 2, rot / 2]."""
    half = row.shape[2]
    c, s = row[:, None, 0], row[:, None, 1]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _normed(x, w):
    """Each head over its root mean square (summed in 64 bits, rounded once), times the weights."""
    r = (1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + _EPS)).float()
    return x.float() * r * w


def _plain_norm(s):
    out = {}
    for name, w in (("q", s["wq"]), ("k", s["wk"])):
        x = _normed(s[name], w)
        if s["table"] is not None:
            x = _rotate(x, s["table"][s["positions"].long()], s["case"]["interleaved"])
        out[name] = x.to(s[name].dtype)
    return out


def _put(codes, scale, x, touched, unit, offset, tokens_last):
    """New values x [tokens, heads, size] at (unit, offset) of the touched pages, whose scale grows where they need it:
    the pages' values [n, heads, page, size] and scales [n, heads]; codes and scales go back into the cache too."""
    n, heads = touched.numel(), x.shape[1]
    peak = torch.zeros(n, heads, device=x.device)
    peak.scatter_reduce_(0, unit[:, None].expand(-1, heads), x.abs().amax(2), "amax")
    first = torch.full((n,), 1 << 30, dtype=torch.int64, device=x.device)
    first.scatter_reduce_(0, unit, offset, "amin")
    old = torch.where(first[:, None] == 0, 0.0, scale[touched])  # a page that starts here holds nothing
    now = torch.maximum(old, peak * (1.0 / 127.0))
    some = torch.where(now > 0, now, 1.0)
    page = codes[touched].float()
    page = page.transpose(2, 3) if tokens_last else page
    page = torch.where((now > old)[..., None, None], torch.round(page * (old / some)[..., None, None]), page).contiguous()
    page[unit, :, offset, :x.shape[2]] = torch.round(x / some[unit][..., None]).clamp(-127, 127)
    codes[touched] = (page.transpose(2, 3) if tokens_last else page).to(torch.int8)
    scale[touched] = now
    return page[..., :x.shape[2]] * now[..., None, None], now


def _plain_append(s):
    case = s["case"]
    k, v, k_scale, v_scale = s["cache"]
    row, touched = s["table"][s["positions"].long()], s["touched"].long()
    b = case["page"]
    unit, offset = torch.searchsorted(touched, s["slots"] // b), s["slots"] % b
    q = _rotate(_normed(s["q"], s["wq"]), row, case["interleaved"]).to(s["q"].dtype)
    key = _rotate(_normed(s["k"], s["wk"]), row, case["interleaved"])
    keys, ks = _put(k, k_scale, key, touched, unit, offset, False)
    values, vs = _put(v, v_scale, s["v"].float(), touched, unit, offset, True)
    return {"q": q, "keys": keys, "values": values, "k_scale": ks, "v_scale": vs}


def _of_request(q_start, tokens):
    """The request of each row, and the row's number in it."""
    t = torch.arange(tokens, device=q_start.device)
    of = torch.searchsorted(q_start[1:].contiguous().long(), t, right=True)
    return of, t - q_start.long()[of]


def _ancestors(parents, q_start, n):
    """[requests, n, n]: row i descends from row j, or is it.  Paths of length 1, 2, 4, ... are joined."""
    r = q_start.numel() - 1
    of, at = _of_request(q_start, parents.numel())
    up = torch.zeros(r, n, n, device=parents.device)
    up[of, at, at] = 1.0
    some = parents >= 0
    up[of[some], at[some], parents.long()[some]] = 1.0
    for _ in range(max(1, (n - 1).bit_length())):
        up = (torch.bmm(up, up) > 0).float()
    return up > 0, of, at


def _plain_tree(parents, kv_lens, q_start, n):
    """Positions int32 [tokens] and masks int64 [tokens, words]."""
    words = -(-n // 64)
    up, of, at = _ancestors(parents, q_start, n)
    rows = torch.nn.functional.pad(up[of, at], (0, 64 * words - n)).view(-1, words, 64)
    bit = torch.ones(64, dtype=torch.int64, device=parents.device) << torch.arange(64, device=parents.device)
    mask = (rows.long() * bit).sum(-1)
    count = (q_start[1:] - q_start[:-1]).long()
    position = ((kv_lens.long() - count)[of] + rows.sum((1, 2)) - 1).clamp(min=0)
    return position.int(), mask


def _plain_attend(s):
    case = s["case"]
    q, (k, v, k_scale, v_scale) = s["q"].float(), s["cache"]
    b, d, h = case["page"], case["dim"], case["kv_heads"]
    r, n = s["kv_lens"].numel(), s["max_q"]
    group = case["heads"] // h
    blocks = s["blocks"][:, :-(-s["max_kv"] // b)].long().clamp(min=0)
    size = blocks.shape[1] * b
    keys = (k[blocks].float() * k_scale[blocks][..., None, None]).transpose(1, 2).reshape(r, h, size, -1)[..., :d]
    values = (v[blocks].float() * v_scale[blocks][..., None, None]).permute(0, 2, 1, 4, 3).reshape(r, h, size, -1)[..., :d]
    start, count = s["q_start"][:-1].long(), (s["q_start"][1:] - s["q_start"][:-1]).long()
    i = torch.arange(n, device=q.device)
    at = (start[:, None] + i).clamp(max=q.shape[0] - 1)  # [r, n]
    rows = q[at].view(r, n, h, group, d).permute(0, 2, 3, 1, 4).reshape(r, h, group * n, d)
    score = torch.matmul(rows, keys.transpose(2, 3).contiguous()).mul_(d ** -0.5).view(r, h, group, n, size)
    context = s["kv_lens"].long() - count
    token = torch.arange(size, device=q.device)
    bits = (s["mask"][..., None] >> torch.arange(64, device=q.device)) & 1
    bits = bits.flatten(1)[at] > 0  # [r, n, 64 words]
    drafted = token - context[:, None]  # [r, size]: the row of the step that is there
    drafted_seen = bits.gather(2, drafted.clamp(0, bits.shape[2] - 1)[:, None].expand(-1, n, -1))
    before = (drafted < 0)[:, None].expand(-1, n, -1)
    if case["window"]:
        place = context[:, None] + bits.sum(2) - 1  # [r, n]
        before = before & (token > place[..., None] - case["window"])
    seen = torch.where((drafted < 0)[:, None], before, drafted_seen & (drafted < count[:, None])[:, None])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = weight.sum(-1)
    out = torch.matmul(weight.view(r, h, group * n, size), values).view(r, h, group, n, d)
    out = out / torch.where(total > 0, total, 1.0)[..., None]
    out = out.permute(0, 3, 1, 2, 4).reshape(r * n, h * group, d)
    of, row = _of_request(s["q_start"], q.shape[0])
    return out[of * n + row].to(s["q"].dtype)


def _plain_accept(s):
    """The rows whose tokens were drawn, each from its parent: a path from row 0."""
    n, t = s["max_q"], s["parents"].numel()
    up, of, at = _ancestors(s["parents"], s["q_start"], n)
    r = s["kv_lens"].numel()
    start = s["q_start"][:-1].long()
    parent = s["parents"].long()
    drawn = s["drawn"][(start[of] + parent).clamp(min=0)]
    match = (parent >= 0) & (s["drafted"] == drawn)
    # of siblings that match the first counts
    first = torch.full((r, n), n, dtype=torch.int64, device=of.device)
    first.view(-1).scatter_reduce_(0, of * n + parent.clamp(min=0), torch.where(match, at, n), "amin")
    good = torch.zeros(r, n, dtype=torch.bool, device=of.device)
    good[of, at] = ((parent < 0) & (at == 0)) | (match & (first[of, parent.clamp(min=0)] == at))
    kept = ((up & ~good[:, None]).sum(2) == 0)  # every row above it is good
    count = s["q_start"][1:] - s["q_start"][:-1]
    i = torch.arange(n, device=of.device)
    took = (count > 0) & (s["slots"][start.clamp(max=t - 1)] >= 0)
    kept &= (i < count[:, None]) & took[:, None]
    total = kept.sum(1)
    rank = kept.cumsum(1) - 1
    path = torch.full((r, n + 1), -1, dtype=torch.int64, device=of.device)
    path.scatter_(1, torch.where(kept, rank, n), i.expand(r, n).contiguous())
    path[:, n] = -1
    last = start + torch.where(kept, i, -1).amax(1)
    token = torch.where(total > 0, s["drawn"][last.clamp(0, t - 1)], -1)
    return path[of, at].int(), total.int(), torch.where(total > 0, last, -1).int(), token, path[:, :n]


def _moved(codes, scale, page, base, path, kept, table, tokens_last):
    """The tail of each request after its kept rows moved to its context's end: new codes [r, w, H, page, Dp], new
    scales [r, w, H], and which pages they are [r, w]."""
    r, n = path.shape
    w = -(-n // page) + 1  # pages that n tokens may lie on
    j0 = base // page
    col = j0[:, None] + torch.arange(w, device=base.device)
    pages = torch.where(col < table.shape[1], table.gather(1, col.clamp(max=table.shape[1] - 1)), -1)
    x = codes[pages.clamp(min=0)].float()
    x = x.transpose(3, 4) if tokens_last else x  # [r, w, H, page, Dp]
    h, dp = x.shape[2], x.shape[4]
    x = x.permute(0, 1, 3, 2, 4).reshape(r, w * page, h, dp)
    had = scale[pages.clamp(min=0)]  # [r, w, H]
    j = torch.arange(n, device=base.device)
    off = (base - j0 * page)[:, None]
    moves = (j < kept[:, None]) & (path != j)
    to = torch.where(moves, off + j, w * page)
    source = torch.arange(w * page + 1, device=base.device).expand(r, -1).clone()
    source.scatter_(1, to, torch.where(moves, off + path, w * page))
    source = source[:, :w * page]  # the place whose code comes here
    y = x.gather(1, source[..., None, None].expand(-1, -1, h, dp))
    place = torch.arange(w * page, device=base.device)
    other = (source // page) != (place // page)  # from another page: a value, not a code
    value = y * had.gather(1, (source // page)[..., None].expand(-1, -1, h))[..., None]
    peak = torch.where(other[..., None], value.abs().amax(3), 0.0).view(r, w, page, h).amax(2)
    now = torch.maximum(had, peak * (1.0 / 127.0))
    some = torch.where(now > 0, now, 1.0).repeat_interleave(page, 1)[..., None]  # [r, w page, H, 1]
    ratio = (had / torch.where(now > 0, now, 1.0)).repeat_interleave(page, 1)[..., None]
    grown = (now > had).repeat_interleave(page, 1)[..., None]
    own_code = torch.where(grown, torch.round(y * ratio), y)
    new = torch.where(other[..., None, None], torch.round(value / some).clamp(-127, 127), own_code)
    return new.view(r, w, page, h, dp).permute(0, 1, 3, 2, 4), now, pages, moves.any(1)


def _plain_compact(s, path, kept):
    b, r = s["case"]["page"], s["kv_lens"].numel()
    base, kept, table = s["held"].long(), kept.long(), s["blocks"].long()
    end = base + kept
    for k, v, k_scale, v_scale in s["caches"]:
        for codes, scale, last in ((k, k_scale, False), (v, v_scale, True)):
            new, now, pages, some = _moved(codes, scale, b, base, path, kept, table, last)
            j = (base // b)[:, None] + torch.arange(pages.shape[1], device=base.device)
            write = some[:, None] & (j * b < end[:, None]) & (pages >= 0)
            codes[pages[write]] = (new.transpose(3, 4) if last else new)[write].to(torch.int8)
            scale[pages[write]] = now[write]
    return end.int()


def _plain_trim(s, end):
    """Pages behind `end` of those that hold kv_lens tokens go to the list's end, in the order of their numbers."""
    b, table = s["case"]["page"], s["blocks"].long()
    j = torch.arange(table.shape[1], device=table.device)
    gone = (j >= ((end.long() + b - 1) // b)[:, None]) & (j < ((s["kv_lens"].long() + b - 1) // b)[:, None]) & (table >= 0)
    pages, count = s["free_pages"].numel(), s["free_count"].long()
    freed = torch.zeros(pages + 1, dtype=torch.bool, device=table.device)
    freed[torch.where(gone, table, pages)] = True
    freed = freed[:pages]
    to = count + freed.cumsum(0) - 1
    out = torch.cat((s["free_pages"], s["free_pages"][:1]))
    out[torch.where(freed, to, pages)] = torch.arange(pages, dtype=torch.int32, device=table.device)
    s["free_pages"].copy_(out[:pages])
    return torch.where(gone, -1, table).int(), (count + freed.sum()).int()


def _values(caches, pages, d):
    """The values of some pages of each cache, [n, H, page, d]; of no page: not a number."""
    out = {}
    at = pages.long().clamp(min=0)
    none = (pages < 0)[:, None]
    for i, (k, v, k_scale, v_scale) in enumerate(caches):
        for name, codes, scale in (("keys", k, k_scale), ("values", v.transpose(2, 3), v_scale)):
            factor = torch.where(none, math.nan, scale[at])
            out[f"{name}{i}"] = codes[at][..., :d].float() * factor[..., None, None]
    return out


def _plain_settle(s):
    position, mask = _plain_tree(s["parents"], s["kv_lens"], s["q_start"], s["max_q"])
    path, kept, last, token, rows = _plain_accept(s)
    end = _plain_compact(s, rows, kept)
    table, count = _plain_trim(s, end)
    return {"positions": position, "mask": mask, "path": path, "kept": kept, "last": last, "token": token,
            "kv_lens": end, "blocks": table, "free_pages": s["free_pages"], "free_count": count,
            **_values(s["caches"], s["touched"], s["case"]["dim"])}


def _plain_fork(s):
    b = s["case"]["page"]
    source, target, table = s["source"].long(), s["target"].long(), s["blocks"].long()
    held = s["kv_lens"].long()[source]
    full, part = held // b, held % b > 0
    upto, count = part.long().cumsum(0), s["free_count"].long()
    done = ~part | (upto <= count)
    rows = table[source]
    fresh = s["free_pages"].long()[(count - upto).clamp(min=0)]
    j = torch.arange(table.shape[1], device=table.device)
    shared = done[:, None] & (j < full[:, None])
    last = rows.gather(1, full[:, None])[:, 0]
    new = torch.where(shared, rows, -1)
    new.scatter_(1, full[:, None], torch.where(done & part, fresh, new.gather(1, full[:, None])[:, 0])[:, None])
    s["refs"].scatter_add_(0, rows.clamp(min=0).view(-1), shared.int().view(-1))
    blocks, lens = s["blocks"].clone(), s["kv_lens"].clone()
    blocks[target], lens[target] = new.int(), torch.where(done, held, 0).int()
    copied = done & part
    copy_from, copy_to = torch.where(copied, last, -1).int(), torch.where(copied, fresh, -1).int()
    a, z = last[copied], fresh[copied]
    for parts in s["caches"]:
        for x in parts:
            x[z] = x[a]
    return {"blocks": blocks, "kv_lens": lens, "free_count": (count - copied.sum()).int(), "copy_from": copy_from,
            "copy_to": copy_to, "refs": s["refs"], **_values(s["caches"], copy_to, s["case"]["dim"])}


# ------------------------------------------------------------------ one pass

_kept = {}


def _engine():
    if "engine" not in _kept:
        from ztensor_amd.engine import ROCmEngine

        _kept["engine"] = ROCmEngine()
    return _kept["engine"]


def _call(s):
    case, e = s["case"], _engine()
    op = case["op"]
    if op in ("norm", "append"):
        from ztensor_amd.decode import HeadNorm

        norm = HeadNorm(s["wq"], s["wk"], _EPS)
    if op == "norm":
        q, k = e.norm_rope(s["q"], s["k"], norm, s["positions"], s["table"], interleaved=case["interleaved"])
        return {"q": q, "k": k}
    if op == "append":
        q = e.kv8_append(s["k"], s["v"], s["cache"], s["slots"], positions=s["positions"], table=s["table"],
                         interleaved=case["interleaved"], q=s["q"], norm=norm)
        keys, values = e.kv8_dequant(s["cache"], s["touched"], case["dim"])
        return {"q": q, "keys": keys, "values": values, "k_scale": s["cache"][2][s["touched"]],
                "v_scale": s["cache"][3][s["touched"]]}
    if op == "attend":
        return e.kv8_tree_attention(s["q"], s["cache"], s["blocks"], s["kv_lens"], s["q_start"], s["mask"],
                                    max_q=s["max_q"], max_kv=s["max_kv"], window=case["window"])
    out = {}
    if op == "settle":
        tree = e.kv8_tree(s["parents"], s["kv_lens"], s["q_start"], s["max_q"])
        took = e.tree_accept(s["drafted"], s["drawn"], s["q_start"], parents=s["parents"], slots=s["slots"])
        end = e.kv8_compact(s["caches"], s["blocks"], s["held"], s["q_start"], took.path, took.kept)
        left = e.kv8_trim(s["kv_lens"], end, s["blocks"], s["free_pages"], s["free_count"], case["page"])
        out = {"positions": tree.positions, "mask": tree.mask, "path": took.path, "kept": took.kept, "last": took.last,
               "token": took.token, "kv_lens": end, "blocks": left.block_table, "free_pages": s["free_pages"],
               "free_count": left.free_count}
        pages = s["touched"]
    else:
        f = e.kv8_fork(s["source"], s["target"], s["kv_lens"], s["blocks"], s["refs"], s["free_pages"], s["free_count"],
                       case["page"])
        e.kv8_copy(s["caches"], f.copy_from, f.copy_to)
        out = {"blocks": f.block_table, "kv_lens": f.kv_lens, "free_count": f.free_count, "copy_from": f.copy_from,
               "copy_to": f.copy_to, "refs": s["refs"]}
        pages = f.copy_to
    for i, cache in enumerate(s["caches"]):
        out[f"keys{i}"], out[f"values{i}"] = e.kv8_dequant(cache, pages, case["dim"])
    return out


def run(state):
    if own:
        return _call(state)
    return {"norm": _plain_norm, "append": _plain_append, "attend": _plain_attend, "settle": _plain_settle,
            "fork": _plain_fork}[state["case"]["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    op, kv, d = case["op"], case["kv_heads"], case["dim"]
    size = 2 if case.get("dtype") == "f16" else 4
    if op == "norm":
        t, heads = case["tokens"], case["heads"] + kv
        return {"bytes": 2 * t * heads * d * size + t * 4 * (case["rot"] + bool(case["rot"])) + 8 * d,
                "flops": t * heads * (4 * d + 3 * case["rot"])}
    b = case["page"]
    if op == "fork":
        lens, sources = _fork_lengths(case)
        copied = min(case["spare"], sum(lens[s] % b > 0 for s in sources))
        held = sum(-(-lens[s] // b) for s in sources)
        page = kv * (2 * b * d + 8)
        # rows of the table read and written, pages in and out, and their values out in 32 bits
        return {"bytes": 12 * held + 20 * case["forks"] + copied * case["layers"] * (2 * page + 8 * kv * b * d), "flops": 0}
    held, fresh = _lengths(case)
    t = sum(fresh)
    if op == "append":
        pages = sum(-(-(h + n) // b) - h // b for h, n in zip(held, fresh))
        old = sum(h % b for h, n in zip(held, fresh))
        # q in and out, k and v in, the table's rows and slots; the pages' codes, in where they held some, and their
        # values out in 32 bits
        moved = t * ((2 * case["heads"] + 2 * kv) * d * size + 4 * case["rot"] + 12)
        moved += 2 * kv * d * (2 * old + t) + 2 * pages * kv * (4 * b * d + 12)
        return {"bytes": moved, "flops": t * (case["heads"] + kv) * (4 * d + 3 * case["rot"]) + 4 * t * kv * d}
    if op == "settle":
        _, paths = _trees(case)
        took = case["requests"] - case["refused"]
        moves = sum(sum(p != i for i, p in enumerate(path)) for path in paths[:took])
        pages = sum(-(-(h + n) // b) - h // b for h, n in zip(held[:took], fresh))
        words = -(-max(fresh) // 64)
        # parents, tokens, drawn ones and slots in, masks, positions and paths out; moved codes in and out; values out
        return {"bytes": t * (28 + 8 * words + 8) + 20 * case["requests"]
                + case["layers"] * (moves * 4 * kv * d + pages * kv * (10 * b * d + 8)), "flops": 0}
    tokens = pairs = 0
    for parents, h, n in zip(_trees(case)[0], held, fresh):
        depth = []
        for p in parents:
            depth.append(1 + (depth[p] if p >= 0 else 0))
        w = case["window"] or h + n
        tokens += min(h, w - 1) + n
        pairs += sum(min(h, max(0, w - x)) + x for x in depth)
    moved = 2 * t * case["heads"] * d * size + 2 * tokens * kv * d + (8 * kv + 4) * -(-tokens // b) + 8 * t * -(-max(fresh) // 64)
    return {"bytes": moved, "flops": 4 * pairs * case["heads"] * d}


# ------------------------------------------------------------------ the definitions in 64 bits


def _exact_normed(x, w, rounded):
    """Over the root of the mean square; rounded: each factor and product to 32 bits, as stored keys are defined."""
    x = x.double()
    r = (x.pow(2).sum(-1) / x.shape[-1] + _EPS).rsqrt().unsqueeze(-1)
    return ((x * r.float().double()).float().double() * w.double()).float().double() if rounded else x * r * w.double()


def _exact_turn(x, table, positions, interleaved, rounded):
    """Each pair (a, b) times cos + i sin."""
    half = table.shape[2]
    row = table.double()[positions.long()]
    c, s = row[:, None, 0], row[:, None, 1]
    out = x.clone()
    one = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    two = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., one], x[..., two]
    by = (lambda y: y.float().double()) if rounded else (lambda y: y)
    out[..., one] = by(by(a * c) - by(b * s))
    out[..., two] = by(by(b * c) + by(a * s))
    return out


def _exact_append(s):
    case = s["case"]
    b, d = case["page"], case["dim"]
    k, v, k_scale, v_scale = s["cache"]
    f = lambda y: y.float().double()  # noqa: E731
    q = _exact_turn(_exact_normed(s["q"], s["wq"], False), s["table"], s["positions"], case["interleaved"], False)
    key = _exact_turn(_exact_normed(s["k"], s["wk"], True), s["table"], s["positions"], case["interleaved"], True)
    slots, found = s["slots"].tolist(), {}
    for t, slot in enumerate(slots):
        found.setdefault(slot // b, []).append(t)
    out = {"keys": [], "values": [], "k_scale": [], "v_scale": []}
    for page in s["touched"].tolist():
        at = found[page]
        first, n = slots[at[0]] % b, len(at)
        for name, scale, codes, x in (("keys", k_scale, k[page], key), ("values", v_scale, v[page].transpose(1, 2), s["v"].double())):
            x = x[at[0]:at[0] + n].transpose(0, 1)  # [heads, n, d]
            had = scale[page].double() if first else torch.zeros(x.shape[0], dtype=torch.float64, device=_DEV)
            seventh = float(torch.tensor(1.0 / 127.0))  # of 32 bits
            step = torch.maximum(had, f(x.abs().amax((1, 2)) * seventh))
            grown = (step > had)[:, None, None]
            old = codes[..., :d].double()
            held = torch.where(grown, f(old * f(had / step)[:, None, None]).round(), old)
            held[:, first:first + n] = f(x / step[:, None, None]).round()
            out[name].append(held * step[:, None, None])
            out["k_scale" if name == "keys" else "v_scale"].append(step)
    return {"q": q, **{n: torch.stack(x) for n, x in out.items()}}


def _exact_attend(s):
    case = s["case"]
    b, d, group = case["page"], case["dim"], case["heads"] // case["kv_heads"]
    k, v, k_scale, v_scale = s["cache"]
    start, lens = s["q_start"].tolist(), s["kv_lens"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEV)
    for r, (size, parents) in enumerate(zip(lens, _trees(case)[0])):
        lo, hi = start[r], start[r + 1]
        n = hi - lo
        above = torch.zeros(n, n, dtype=torch.bool)
        for i, p in enumerate(parents):
            if p >= 0:
                above[i] = above[p]
            above[i, i] = True
        above = above.to(_DEV)
        pages = s["blocks"][r, :-(-size // b)].long()
        seen = torch.ones(n, size - n, dtype=torch.bool, device=_DEV)
        if case["window"]:
            place = size - n + above.sum(1) - 1
            seen = torch.arange(size - n, device=_DEV) > (place - case["window"])[:, None]
        hidden = ~torch.cat((seen, above), 1)
        for h in range(case["kv_heads"]):
            keys = (k[pages, h].double() * k_scale[pages, h].double()[:, None, None]).reshape(-1, k.shape[3])[:size, :d]
            values = v[pages, h].double() * v_scale[pages, h].double()[:, None, None]
            values = values.transpose(1, 2).reshape(-1, k.shape[3])[:size, :d]
            rows = s["q"][lo:hi, h * group:(h + 1) * group].double().reshape(n * group, d)
            score = (rows @ keys.t() / math.sqrt(d)).view(n, group, size).masked_fill(hidden[:, None], -math.inf)
            out[lo:hi, h * group:(h + 1) * group] = (torch.softmax(score, -1).view(n * group, size) @ values).view(n, group, d)
    return out


def _exact_settle(s):
    """One request, page and row after another."""
    case = s["case"]
    b, d = case["page"], case["dim"]
    f = lambda y: y.float().double()  # noqa: E731
    seventh = float(torch.tensor(1.0 / 127.0))
    start, held, lens, table = (s[x].tolist() for x in ("q_start", "held", "kv_lens", "blocks"))
    drafted, drawn, parents = (s[x].tolist() for x in ("drafted", "drawn", "parents"))
    lists = []  # (page, [(place, page it comes from, place there)]) of each request, in order
    for r, (lo, hi) in enumerate(zip(start, start[1:])):
        if lens[r] != held[r] + hi - lo:
            continue
        at, path = 0, [0]
        while at is not None:
            at = next((i for i in range(at + 1, hi - lo)
                       if parents[lo + i] == at and drafted[lo + i] == drawn[lo + at]), None)
            path += [] if at is None else [at]
        by = {}
        for j, p in enumerate(path):
            if j != p:
                z, a = held[r] + j, held[r] + p
                by.setdefault(table[r][z // b], []).append((z % b, table[r][a // b], a % b))
        lists += sorted(by.items(), key=lambda x: table[r].index(x[0]))
    out, touched = {}, s["touched"].long()
    for i, (k, v, k_scale, v_scale) in enumerate(s["caches"]):
        for name, codes, scale in (("keys", k, k_scale), ("values", v.transpose(2, 3), v_scale)):
            codes, scale = codes[..., :d].double(), scale.double()
            first, had = codes.clone(), scale.clone()
            for page, moves in lists:
                z, p, a = (torch.tensor(x, device=_DEV) for x in zip(*moves))
                far = p != page
                x = f(first[p, :, a] * had[p][..., None])  # [moves, heads, d]
                step = had[page]
                if bool(far.any()):
                    step = torch.maximum(step, f(x[far].abs().amax((0, 2)) * seventh))
                grown = (step > had[page])[:, None, None]
                ratio = f(had[page] / step)[:, None, None]
                new = first[page].clone()
                new[:, z] = first[p, :, a].transpose(0, 1)
                new = torch.where(grown, f(new * ratio).round(), new)
                new[:, z[far]] = f(x[far] / step[:, None]).round().transpose(0, 1)
                codes[page], scale[page] = new, step
            out[f"{name}{i}"] = codes[touched] * scale[touched][..., None, None]
    return {**dict.fromkeys(("positions", "mask", "path", "kept", "last", "token", "kv_lens", "blocks", "free_pages",
                             "free_count")), **out}


def _exact_fork(s):
    """What the pages that are copied to hold: their sources' values."""
    case = s["case"]
    b, d = case["page"], case["dim"]
    free, lens = s["free_pages"].tolist()[:int(s["free_count"])], s["kv_lens"].tolist()
    pages = []
    for r in s["source"].tolist():
        part = lens[r] % b > 0
        pages.append(int(s["blocks"][r, lens[r] // b]) if part and free else -1)
        if part and free:
            free.pop()
    at = torch.tensor(pages, device=_DEV)
    out = dict.fromkeys(("blocks", "kv_lens", "free_count", "copy_from", "copy_to", "refs"))
    for i, (k, v, k_scale, v_scale) in enumerate(s["caches"]):
        for name, codes, scale in (("keys", k, k_scale), ("values", v.transpose(2, 3), v_scale)):
            x = codes[at][..., :d].double() * scale[at].double()[..., None, None]
            out[f"{name}{i}"] = x.masked_fill((at < 0)[:, None, None, None], math.nan)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        out = {}
        for name, w in (("q", s["wq"]), ("k", s["wk"])):
            out[name] = _exact_normed(s[name], w, False)
            if case["rot"]:
                out[name] = _exact_turn(out[name], s["table"], s["positions"], case["interleaved"], False)
        return out
    return {"append": _exact_append, "attend": _exact_attend, "settle": _exact_settle, "fork": _exact_fork}[case["op"]](s)
