"""What a decode loop does between its linear layers, as cases that can be timed.

The framework's matmuls give q, k and v and take the attention's output; these
are the operators between them, and the ones around the layers:

  rope    rotary positions of q and k: the whole head or part of it, the
          pairs as halves or interleaved, tables scaled for long contexts
  append  a step's keys (rotated) and values into an 8-bit paged cache with
          one scale for each page and head, q rotated in the same call; the
          touched pages come back as the values that they stand for
  attend  attention of one token, a few tokens or prompts over that cache
  plan    block tables, slots and positions from the requests' lengths
  sample  temperature, top-k, top-p and min-p from given random numbers

The cache of H key/value heads of size D in pages of B tokens is a tuple
  k        int8 [pages, H, B, Dp]   Dp: D to the next multiple of 64, zeros past D
  v        int8 [pages, H, Dp, B]   token-minor, as the second product reads it
  k_scale  float32 [pages, H]       a value is its code times the scale
  v_scale  float32 [pages, H]
"""
from __future__ import annotations

import itertools
import math

import torch

own = False

_DEV = "cuda"
_FIX = float(2 ** 40)  # sampling weights are whole numbers of 2^-40
_LARGEST = 1.6e11  # operations of an attention that no drawn case exceeds
_CACHE = 64 * 4096 * 8 * 128  # values of keys that no drawn case's lengths exceed


def listed():
    return [
        # one token's q and k in an 8B model: what a single call costs
        {"name": "rope_token", "op": "rope", "dtype": "f32", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "interleaved": False, "scaling": "none", "max_pos": 8192},
        # a long prompt in a 70B model's layer, part of the head, pairs interleaved, positions past the trained range
        {"name": "rope_prompt", "op": "rope", "dtype": "f16", "tokens": 4099, "heads": 64, "kv_heads": 8, "dim": 128,
         "rot": 64, "interleaved": True, "scaling": "yarn", "max_pos": 32768},
        # 64 sequences each add a token to their last page
        {"name": "append_batch64", "op": "append", "dtype": "f32", "requests": 64, "new": 1, "context": 3000,
         "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "scaling": "llama3",
         "page": 64, "max_pos": 16384},
        # prompts of odd lengths go into small pages, one of them onto a page that holds tokens already
        {"name": "append_prompts", "op": "append", "dtype": "f16", "requests": 3, "new": 1400, "context": 500,
         "heads": 64, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "scaling": "none",
         "page": 16, "max_pos": 8192},
        # the first tokens of a chat: a single sequence with almost nothing in the cache
        {"name": "attend_short", "op": "attend", "dtype": "f32", "requests": 1, "new": 1, "context": 36,
         "ragged": False, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0},
        # one sequence deep into a long document, a 70B layer
        {"name": "attend_long", "op": "attend", "dtype": "f16", "requests": 1, "new": 1, "context": 40010,
         "ragged": False, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64, "window": 0},
        # continuous batching: 64 sequences of very different lengths
        {"name": "attend_batch64", "op": "attend", "dtype": "f32", "requests": 64, "new": 1, "context": 8000,
         "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "window": 0},
        # a prompt, a piece of another one and a decoding sequence in one call: the largest case
        {"name": "attend_prompts", "op": "attend", "dtype": "f16", "requests": 3, "new": 4096, "context": 2900,
         "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0},
        # a step of a small server
        {"name": "plan_8", "op": "plan", "requests": 8, "new": 1, "context": 2000, "page": 64, "width": 128,
         "spare": 1000},
        # a step of a large one: prompts among 512 sequences, and not enough free pages for all of them
        {"name": "plan_512", "op": "plan", "requests": 512, "new": 300, "context": 8000, "page": 16, "width": 1024,
         "spare": 600},
        # one sequence's next token
        {"name": "sample_1", "op": "sample", "dtype": "f32", "requests": 1, "vocab": 131072, "mix": "both"},
        # 128 sequences with settings of their own, an odd vocabulary
        {"name": "sample_128", "op": "sample", "dtype": "f32", "requests": 128, "vocab": 100003, "mix": "each"},
    ]


def _log(rng, a, b):
    return min(b, max(a, round(math.exp(rng.uniform(math.log(a), math.log(b))))))


def draw(rng):
    op = rng.choice(["rope", "append", "append", "attend", "attend", "attend", "attend", "plan", "sample", "sample"])
    dtype = rng.choice(["f32", "f16"])
    if op == "plan":
        page = rng.choice([16, 32, 64, 128])
        context = _log(rng, 16, 12000)
        new = rng.choice([1, 1, _log(rng, 2, 500)])
        requests = _log(rng, 1, 512)
        return {"op": op, "requests": requests, "new": new, "context": context, "page": page,
                "width": (context + new) // page + rng.randint(1, 40), "spare": _log(rng, 1, 4 * requests)}
    if op == "sample":
        requests = _log(rng, 1, 128)
        return {"op": op, "dtype": dtype, "requests": requests, "vocab": _log(rng, 300, 152000),
                "mix": rng.choice(["none", "top_k", "top_p", "min_p", "both", "each", "greedy"])}
    dim = rng.choice([64, 128, 128, 128, 80, 96, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 7, 8])
    page = rng.choice([16, 32, 64, 128])
    if op == "rope":
        return {"op": op, "dtype": dtype, "tokens": _log(rng, 1, 4096), "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "rot": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "ntk", "yarn", "llama3"]), "max_pos": _log(rng, 5000, 65536)}
    if op == "append":
        new = rng.choice([1, 1, _log(rng, 2, 2000)])
        return {"op": op, "dtype": dtype, "requests": _log(rng, 1, 128 if new == 1 else max(1, 4000 // new)),
                "new": new, "context": _log(rng, 1, 4000), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(["none", "yarn"]), "page": page, "max_pos": 8192}
    kind = rng.choice(["token", "token", "few", "prompt", "prompt"])
    window = rng.choice([0, 0, 0, _log(rng, 10, 4096)])
    width = kv_heads * dim
    if kind == "prompt":
        requests = rng.randint(1, 3)
        most = _LARGEST / (4.0 * heads * dim * requests)  # pairs of a query and a key that a request may have
        new = _log(rng, 20, min(4096, int(math.sqrt(most))))
        context = _log(rng, 1, max(2, min(4000, int(most / new) - new // 2)))
    else:
        new = 1 if kind == "token" else rng.randint(2, 8)
        context = _log(rng, 1, 40000)
        requests = _log(rng, 1, max(1, min(96, _CACHE // (context * width))))
    return {"op": op, "dtype": dtype, "requests": requests, "new": new, "context": context,
            "ragged": rng.random() < 0.6, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "window": window}


# ------------------------------------------------------------------ inputs


def _type(case):
    return torch.float16 if case["dtype"] == "f16" else torch.float32


def _lengths(case):
    """(tokens in the cache before the step, tokens that the step adds) of each request: the case's, whatever the seed."""
    g = torch.Generator().manual_seed(17)
    r, new, context = case["requests"], case["new"], case["context"]
    if not case.get("ragged", True):
        return [context] * r, [new] * r
    # between a few tokens and the whole; the first request has the whole
    part = torch.rand(r, generator=g, dtype=torch.float64)
    held = [max(0, int(context * p ** 2)) for p in part.tolist()]
    fresh = [new] * r
    if new > 8:  # prompts: a whole one, a piece of one, and single tokens among them
        part = torch.rand(r, generator=g, dtype=torch.float64).tolist()
        fresh = [new if i == 0 else 1 if i % 3 == 2 else max(1, int(new * p * 0.5)) for i, p in enumerate(part)]
        held[0] = 0
    else:
        held[0] = context
    return held, fresh


def _frequencies(case):
    """The angle per position of each pair, in 64 bits, and the factor on the table."""
    rot, base = case["rot"], 500000.0 if case["scaling"] == "llama3" else 10000.0
    i = torch.arange(rot // 2, dtype=torch.float64)
    kind, factor, trained = case["scaling"], 8.0, 4096.0
    if kind == "ntk":
        base *= factor ** (rot / (rot - 2.0))
    freq = base ** (-2.0 * i / rot)
    if kind == "linear":
        return freq / factor, 1.0
    if kind == "yarn":  # fast pairs stay, slow ones are stretched, a ramp between
        pair = lambda turns: rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return freq * (1 - ramp) + freq / factor * ramp, 0.1 * math.log(factor) + 1.0
    if kind == "llama3":
        wave = 2 * math.pi / freq
        mix = ((trained / wave - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return freq * mix + freq / factor * (1 - mix), 1.0
    return freq, 1.0


def _table(case):
    """float32 [positions, 2, rot / 2]: the cosines and sines of a position."""
    freq, factor = _frequencies(case)
    angle = torch.arange(case["max_pos"], dtype=torch.float64, device=_DEV)[:, None] * freq.to(_DEV)
    return (torch.stack((angle.cos(), angle.sin()), 1) * factor).float()


def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(seed * 1000003 + 5)


def _heads(case, tokens, g):
    """q, k and v as a step's fused projection gives them: slices of its rows."""
    n, m, d = case["heads"], case["kv_heads"], case["dim"]
    x = torch.randn(tokens, (n + 2 * m) * d, device=_DEV, generator=g)
    x[:, ::37] *= 4  # a few channels are larger
    x = x.to(_type(case))
    q, k, v = x.split([n * d, m * d, m * d], 1)
    return q.view(tokens, n, d), k.view(tokens, m, d), v.view(tokens, m, d)


def _cache(case, pages, g):
    h, b, d = case["kv_heads"], case["page"], case["dim"]
    dp = -(-d // 64) * 64

    codes = lambda *n: torch.randn(n, device=_DEV, generator=g).mul_(36).clamp_(-127, 127).round_().to(torch.int8)  # noqa: E731
    k, v = codes(pages, h, b, dp), codes(pages, h, dp, b)
    k[..., d:] = 0
    v[:, :, d:] = 0
    scale = lambda: 0.028 * torch.exp(0.3 * torch.randn(pages, h, device=_DEV, generator=g))  # noqa: E731
    return k, v, scale(), scale()


def _paged(case, seed, spare=0):
    """Lengths, a block table over pages in no order, and the number of pages."""
    held, fresh = _lengths(case)
    b = case["page"]
    need = [-(-(h + n) // b) for h, n in zip(held, fresh)]
    pages = sum(need) + 3 + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed + 3)).tolist()
    width = max(need) + 1
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return held, fresh, table, pages, order[at:]


def _int(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=_DEV)


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "rope":
        t = case["tokens"]
        q, k, _ = _heads(case, t, g)
        first = int(torch.randint(0, case["max_pos"] - t, (1,), generator=torch.Generator().manual_seed(seed)))
        return {"case": case, "q": q, "k": k, "positions": _int(range(first, first + t)), "table": _table(case)}
    if op == "append":
        held, fresh, table, pages, _ = _paged(case, seed)
        b = case["page"]
        slots = [table[r][p // b] * b + p % b for r, (h, n) in enumerate(zip(held, fresh)) for p in range(h, h + n)]
        positions = [p for h, n in zip(held, fresh) for p in range(h, h + n)]
        q, k, v = _heads(case, len(slots), g)
        touched = sorted({s // b for s in slots})
        return {"case": case, "q": q, "k": k, "v": v, "cache": _cache(case, pages, g),
                "slots": _int(slots, torch.int64), "positions": _int(positions), "table": _table(case),
                "touched": _int(touched)}
    if op == "attend":
        held, fresh, table, pages, _ = _paged(case, seed)
        lens = [h + n for h, n in zip(held, fresh)]
        q = torch.randn(sum(fresh), case["heads"], case["dim"], device=_DEV, generator=g)
        q *= 1.5 * torch.exp(0.4 * torch.randn(sum(fresh), case["heads"], 1, device=_DEV, generator=g))
        return {"case": case, "q": q.to(_type(case)), "cache": _cache(case, pages, g), "blocks": _int(table),
                "kv_lens": _int(lens), "q_start": _int([0, *itertools.accumulate(fresh)]), "max_q": max(fresh), "max_kv": max(lens)}
    if op == "plan":
        held, fresh, table, pages, rest = _paged(case, seed, case["spare"])
        width, b = case["width"], case["page"]
        # pages that the step has yet to take are not in the table
        blocks = [[p if j < -(-h // b) else -1 for j, p in enumerate(row[:width])] + [-1] * (width - len(row))
                  for h, row in zip(held, table)]
        free = (rest + [0] * case["spare"])[:case["spare"]]
        return {"case": case, "kv_lens": _int(held), "new": _int(fresh), "blocks": _int(blocks),
                "free_pages": _int(free), "free_count": _int([case["spare"]]), "tokens": sum(fresh)}
    r, v, mix = case["requests"], case["vocab"], case["mix"]
    # logits of a language model: a wide bulk, and for each row a few tokens that stand out
    logits = 2.0 * torch.randn(r, v, device=_DEV, generator=g)
    at = torch.randint(0, v, (r, 40), device=_DEV, generator=g)
    logits.scatter_(1, at, 9.0 + 2.5 * torch.randn(r, 40, device=_DEV, generator=g))
    one = lambda x: torch.full((r,), x, device=_DEV)  # noqa: E731
    rand = lambda: torch.rand(r, device=_DEV, generator=g)  # noqa: E731
    temperature, top_k, top_p, min_p = one(1.0), one(0), one(1.0), one(0.0)
    if mix == "each":
        temperature = (0.3 + 1.2 * rand()) * (rand() > 0.1)
        top_k = torch.randint(1, 200, (r,), device=_DEV, generator=g) * (rand() > 0.5)
        top_p = torch.where(rand() > 0.3, 0.5 + 0.5 * rand(), 1.0)
        min_p = 0.1 * rand() * (rand() > 0.5)
    elif mix == "greedy":
        temperature = one(0.0)
    else:
        temperature = one(0.8)
        top_k = one(50) if mix in ("top_k", "both") else top_k
        top_p = one(0.95) if mix in ("top_p", "both") else top_p
        min_p = one(0.05) if mix in ("min_p", "both") else min_p
    return {"case": case, "logits": logits.to(_type(case)), "u": rand(), "temperature": temperature.float(),
            "top_k": top_k.to(torch.int32), "top_p": top_p.float(), "min_p": min_p.float()}


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


def _put(codes, scale, x, touched, unit, offset, tokens_last):
    """New values x [tokens, heads, size] at (unit, offset) of the touched pages, whose scale grows where they need it:
    the pages' codes [n, heads, page, size] and scales [n, heads], which go back into the cache too."""
    n, heads = touched.numel(), x.shape[1]
    peak = torch.zeros(n, heads, device=x.device)
    peak.scatter_reduce_(0, unit[:, None].expand(-1, heads), x.abs().amax(2), "amax")
    first = torch.full((n,), 1 << 30, dtype=torch.int64, device=x.device)
    first.scatter_reduce_(0, unit, offset, "amin")
    old = torch.where(first[:, None] == 0, 0.0, scale[touched])  # a page that starts here holds nothing
    now = torch.maximum(old, peak / 127.0)
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
    q = _rotate(s["q"].float(), row, case["interleaved"]).to(s["q"].dtype)
    key = _rotate(s["k"].float(), row, case["interleaved"])
    keys, ks = _put(k, k_scale, key, touched, unit, offset, False)
    values, vs = _put(v, v_scale, s["v"].float(), touched, unit, offset, True)
    return {"q": q, "keys": keys, "values": values, "k_scale": ks, "v_scale": vs}


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
    place = (s["kv_lens"].long() - count)[:, None] + i  # position of each query
    token = torch.arange(size, device=q.device)
    seen = token <= place[..., None]
    if case["window"]:
        seen &= token > place[..., None] - case["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = weight.sum(-1)
    out = torch.matmul(weight.view(r, h, group * n, size), values).view(r, h, group, n, d)
    out = out / torch.where(total > 0, total, 1.0)[..., None]
    out = out.permute(0, 3, 1, 2, 4).reshape(r * n, h * group, d)
    of = torch.repeat_interleave(torch.arange(r, device=q.device), count, output_size=q.shape[0])
    return out[of * n + torch.arange(q.shape[0], device=q.device) - start[of]].to(s["q"].dtype)


def _plain_plan(s):
    b, width = s["case"]["page"], s["case"]["width"]
    held, new, blocks = s["kv_lens"].long(), s["new"].long(), s["blocks"].long()
    end = held + new
    fits = end <= width * b
    have = (held + b - 1) // b
    need = torch.where(fits, (end + b - 1) // b - have, 0)
    upto = need.cumsum(0)
    free = s["free_count"].long()
    done = fits & ((need == 0) | (upto <= free))
    j = torch.arange(width, device=held.device)
    nth = upto[:, None] - need[:, None] + j - have[:, None]  # of all the pages taken
    taken = done[:, None] & (j >= have[:, None]) & (j < (have + need)[:, None])
    page = s["free_pages"].long()[(free - 1 - nth).clamp(0, s["free_pages"].numel() - 1)]
    blocks = torch.where(taken, page, blocks)
    start = torch.cat((new.new_zeros(1), new.cumsum(0)))
    t = torch.arange(s["tokens"], device=held.device)
    of = torch.searchsorted(start[1:].contiguous(), t, right=True)
    position = held[of] + t - start[of]
    at = blocks[of, (position // b).clamp(max=width - 1)]
    slots = torch.where(done[of] & (at >= 0), at * b + position % b, -1)
    return {"blocks": blocks.int(), "slots": slots, "positions": position.int(), "q_start": start.int(),
            "kv_lens": torch.where(done, end, held).int(), "free_count": (free - torch.where(done, need, 0).sum()).int()}


def _plain_sample(s):
    z = s["logits"].float()
    z = torch.where(torch.isnan(z), -math.inf, z)
    vocab = z.shape[1]
    greedy = s["temperature"] <= 0
    top = z.amax(1, keepdim=True)
    weight = torch.exp((z - top) / torch.where(greedy, 1.0, s["temperature"])[:, None])
    weight = torch.where(z == top, 1.0, weight)
    fixed = (weight * _FIX).long()  # whole numbers: their sums are exact in any order
    order = torch.sort(z, dim=1, descending=True, stable=True).indices
    whole = fixed.gather(1, order).cumsum(1)
    k = torch.where((s["top_k"] <= 0) | (s["top_k"] > vocab), vocab, s["top_k"].long())
    k = torch.where(greedy, 1, k)
    kept = torch.minimum(k, (weight >= s["min_p"].clamp(max=1)[:, None]).sum(1))
    mass = whole.gather(1, kept[:, None] - 1)
    enough = torch.ceil(s["top_p"].double()[:, None] * mass.double()).long()
    nucleus = (whole < enough).sum(1) + 1
    kept = torch.where(s["top_p"] < 1, torch.minimum(kept, nucleus), kept)
    total = whole.gather(1, kept[:, None] - 1)
    rank = torch.empty_like(order).scatter_(1, order, torch.arange(vocab, device=z.device).expand_as(order))
    fixed = torch.where(rank < kept[:, None], fixed, 0)
    aim = torch.minimum((s["u"].double()[:, None] * total.double()).long(), total - 1)
    token = (fixed.cumsum(1) <= aim).sum(1)
    chosen = fixed.gather(1, token[:, None])
    return {"tokens": token, "logprobs": torch.log(chosen.double() / total.double())[:, 0].float()}


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
    if op == "rope":
        q, k = e.rope(s["q"], s["k"], s["positions"], s["table"], interleaved=case["interleaved"])
        return {"q": q, "k": k}
    if op == "append":
        q = e.kv8_append(s["k"], s["v"], s["cache"], s["slots"], positions=s["positions"], table=s["table"],
                         interleaved=case["interleaved"], q=s["q"])
        keys, values = e.kv8_dequant(s["cache"], s["touched"], case["dim"])
        return {"q": q, "keys": keys, "values": values, "k_scale": s["cache"][2][s["touched"]],
                "v_scale": s["cache"][3][s["touched"]]}
    if op == "attend":
        return e.kv8_attention(s["q"], s["cache"], s["blocks"], s["kv_lens"], s["q_start"], max_q=s["max_q"],
                               max_kv=s["max_kv"], window=case["window"])
    if op == "plan":
        p = e.kv8_plan(s["kv_lens"], s["new"], s["blocks"], s["free_pages"], s["free_count"], case["page"], s["tokens"])
        return {"blocks": p.block_table, "slots": p.slots, "positions": p.positions, "q_start": p.q_start,
                "kv_lens": p.kv_lens, "free_count": p.free_count}
    tokens, logprobs = e.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                min_p=s["min_p"])
    return {"tokens": tokens, "logprobs": logprobs}


def run(state):
    if own:
        return _call(state)
    op = state["case"]["op"]
    if op == "rope":
        row = state["table"][state["positions"].long()]
        return {n: _rotate(state[n].float(), row, state["case"]["interleaved"]).to(state[n].dtype) for n in ("q", "k")}
    return {"append": _plain_append, "attend": _plain_attend, "plan": _plain_plan, "sample": _plain_sample}[op](state)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    op = case["op"]
    size = 2 if case.get("dtype") == "f16" else 4
    if op == "plan":
        held, fresh = _lengths(case)
        r, t = case["requests"], sum(fresh)
        return {"bytes": 4 * (2 * r * case["width"] + 2 * r + case["spare"]) + 12 * t + 8 * r, "flops": 4 * t}
    if op == "sample":
        n = case["requests"] * case["vocab"]
        return {"bytes": n * size + 28 * case["requests"], "flops": 6 * n}
    heads, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if op == "rope":
        t = case["tokens"]
        return {"bytes": 2 * t * (heads + kv) * d * size + t * (4 * case["rot"] + 4),
                "flops": 3 * t * (heads + kv) * case["rot"]}
    held, fresh = _lengths(case)
    t, b = sum(fresh), case["page"]
    if op == "append":
        pages = sum(-(-(h + n) // b) - h // b for h, n in zip(held, fresh))
        old = sum(h % b for h, n in zip(held, fresh))
        # q in and out, k and v in, the table's rows and slots; the pages' codes, in where they held some, and their
        # values out in 32 bits
        moved = t * ((2 * heads + 2 * kv) * d * size + 4 * case["rot"] + 12)
        moved += 2 * kv * d * (2 * old + t) + 2 * pages * kv * (4 * b * d + 12)
        return {"bytes": moved, "flops": 3 * t * (heads + kv) * case["rot"] + 4 * t * kv * d}
    tokens = pairs = 0
    for h, n in zip(held, fresh):
        w = case["window"] or h + n
        tokens += min(h + n, w + n - 1)
        pairs += sum(min(h + i + 1, w) for i in range(n))
    moved = 2 * t * heads * d * size + 2 * tokens * kv * d + 8 * kv * -(-tokens // b) + 4 * -(-tokens // b)
    return {"bytes": moved, "flops": 4 * pairs * heads * d}


# ------------------------------------------------------------------ the definitions in 64 bits


def _exact_turn(x, table, positions, interleaved):
    """Each pair (a, b) as a complex number times cos + i sin."""
    half = table.shape[2]
    row = table.double()[positions.long()]
    unit = torch.complex(row[:, 0], row[:, 1])[:, None]
    out = x.double().clone()
    if interleaved:
        z = torch.view_as_complex(out[..., :2 * half].unflatten(-1, (half, 2)).contiguous()) * unit
        out[..., :2 * half] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(out[..., :half].contiguous(), out[..., half:2 * half].contiguous()) * unit
        out[..., :half], out[..., half:2 * half] = z.real, z.imag
    return out


def _exact_append(s):
    case = s["case"]
    b, d = case["page"], case["dim"]
    k, v, k_scale, v_scale = s["cache"]
    q = _exact_turn(s["q"], s["table"], s["positions"], case["interleaved"])
    key = _exact_turn(s["k"], s["table"], s["positions"], case["interleaved"])
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
            step = torch.maximum(had, x.abs().amax((1, 2)) / 127)
            grown = (step > had)[:, None, None]
            old = codes[..., :d].double()
            held = torch.where(grown, (old * (had / step)[:, None, None]).round(), old)
            held[:, first:first + n] = (x / step[:, None, None]).round()
            out[name].append(held * step[:, None, None])
            out["k_scale" if name == "keys" else "v_scale"].append(step)
    return {"q": q, **{n: torch.stack(x) for n, x in out.items()}}


def _exact_attend(s):
    case = s["case"]
    b, d, group = case["page"], case["dim"], case["heads"] // case["kv_heads"]
    k, v, k_scale, v_scale = s["cache"]
    start, lens = s["q_start"].tolist(), s["kv_lens"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEV)
    for r, size in enumerate(lens):
        lo, hi = start[r], start[r + 1]
        pages = s["blocks"][r, :-(-size // b)].long()
        place = torch.arange(size - (hi - lo), size, device=_DEV)[:, None]
        token = torch.arange(size, device=_DEV)
        hidden = token > place
        if case["window"]:
            hidden |= token <= place - case["window"]
        for h in range(case["kv_heads"]):
            keys = (k[pages, h].double() * k_scale[pages, h].double()[:, None, None]).reshape(-1, k.shape[3])[:size, :d]
            values = v[pages, h].double() * v_scale[pages, h].double()[:, None, None]
            values = values.transpose(1, 2).reshape(-1, k.shape[3])[:size, :d]
            for i in range(h * group, (h + 1) * group):
                score = s["q"][lo:hi, i].double() @ keys.t() / math.sqrt(d)
                p = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
                out[lo:hi, i] = p.masked_fill(hidden, 0.0) @ values
    return out


def _exact_sample(s):
    out = []
    for z, u, t, k, p, m in zip(s["logits"].double(), *(s[n].tolist() for n in ("u", "temperature", "top_k", "top_p", "min_p"))):
        if t <= 0:
            out.append(0.0)
            continue
        w = torch.exp((z - z.max()) / t)
        down, order = torch.sort(w, descending=True, stable=True)
        n = min(k if k > 0 else w.numel(), int((down >= m).sum()))
        if p < 1:
            part = down[:n].cumsum(0)
            n = min(n, int((part < p * part[-1]).sum()) + 1)
        keep = torch.zeros_like(w)
        keep[order[:n]] = down[:n]
        part = keep.cumsum(0)
        token = min(int((part <= u * part[-1]).sum()), w.numel() - 1)
        out.append(float(torch.log(keep[token] / part[-1])))
    return {"tokens": None, "logprobs": torch.tensor(out, dtype=torch.float64, device=_DEV)}


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "rope":
        return {n: _exact_turn(s[n], s["table"], s["positions"], case["interleaved"]) for n in ("q", "k")}
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](s)
