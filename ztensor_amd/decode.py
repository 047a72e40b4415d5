"""What a decode step does between its linear layers: rotary positions, an
int8 paged key/value cache and attention over it, the pages' bookkeeping, and
the choice of a token.

The kernels are zt_rope, zt_norm_rope, zt_kv8_* and zt_sample of libzt_hip.so; DecodeOps
holds the engine's methods for them.  A step of a batch of requests:

    p = engine.kv8_plan(kv_lens, new, block_table, free_pages, free_count, page_tokens, tokens)
    for each layer:  q, k, v from the engine's matmuls, as [tokens, heads, head_dim]
        q = engine.kv8_append(k, v, cache, p.slots, positions=p.positions, table=rope, q=q)
        a = engine.kv8_attention(q, cache, p.block_table, p.kv_lens, p.q_start, max_q=..., max_kv=...)
    tokens, logprobs = engine.sample(logits, u, temperature=..., top_p=...)

Lengths, tables and slots stay on the device, so a step can be captured in a
graph; what the host knows (the number of tokens, bounds on the lengths) is
passed as numbers.
"""
from __future__ import annotations

import math
import struct
from typing import NamedTuple

import torch

from . import _lib
from ._stream import _on_engine_stream

_TYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16}


class KV8Cache(NamedTuple):
    """An int8 paged cache of one layer: a value is its code times the scale
    of its page and head.  Any tuple of the four tensors does as well."""

    k: torch.Tensor  # int8 [pages, kv_heads, page_tokens, Dp]: Dp is head_dim to the next multiple of 64, zeros past it
    v: torch.Tensor  # int8 [pages, kv_heads, Dp, page_tokens]
    k_scale: torch.Tensor  # float32 [pages, kv_heads]
    v_scale: torch.Tensor

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, head_dim: int, page_tokens: int = 64,
                 device: torch.device | str = "cuda") -> "KV8Cache":
        dp = -(-head_dim // 64) * 64
        return cls(torch.zeros((pages, kv_heads, page_tokens, dp), dtype=torch.int8, device=device),
                   torch.zeros((pages, kv_heads, dp, page_tokens), dtype=torch.int8, device=device),
                   torch.zeros((pages, kv_heads), dtype=torch.float32, device=device),
                   torch.zeros((pages, kv_heads), dtype=torch.float32, device=device))


class HeadNorm(NamedTuple):
    """The norms of q's and k's heads: each over the root of the mean of its
    squares + eps, times weights (float32 [head_dim]; None: ones)."""

    q: torch.Tensor | None
    k: torch.Tensor | None
    eps: float = 1e-6


class KV8Plan(NamedTuple):
    """What kv8_plan gives for a step."""

    block_table: torch.Tensor  # int32 [requests, width], the step's pages included
    slots: torch.Tensor  # int64 [tokens], -1: none
    positions: torch.Tensor  # int32 [tokens]
    q_start: torch.Tensor  # int32 [requests + 1]
    kv_lens: torch.Tensor  # int32 [requests], the step's tokens included
    free_count: torch.Tensor  # int32 [1]


def rope_frequencies(rot_dim: int, base: float = 10000.0, scaling: dict | None = None) -> tuple[torch.Tensor, float]:
    """The angle per position of each of the rot_dim / 2 pairs (float64) and
    the factor on their cosines and sines.  scaling: {"type": ...} and

    linear  factor: positions are divided by it
    ntk     factor: the base grows, so that the slowest pair is stretched by it
    yarn    factor, original_max_position, beta_fast (32), beta_slow (1),
            attention_factor (0.1 ln factor + 1): pairs that turn more than
            beta_fast times over the trained positions stay, those below
            beta_slow are divided by the factor, a linear ramp between
    llama3  factor, original_max_position, low_freq_factor (1),
            high_freq_factor (4): by wavelength, in the same manner
    """
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rope: rot_dim is a positive even number, got {rot_dim}")
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    s = dict(scaling or {})
    kind, factor = s.pop("type", "none"), float(s.pop("factor", 1.0))
    if not factor >= 1.0:
        raise ValueError(f"rope: a scaling factor is at least 1, got {factor}")
    trained = float(s.pop("original_max_position", 0))
    if kind in ("yarn", "llama3") and trained <= 0:
        raise ValueError(f"rope: {kind} scaling needs original_max_position")
    mult = 1.0
    if kind == "ntk":
        if rot_dim == 2:
            raise ValueError("rope: ntk scaling needs more than one pair")
        base *= factor ** (rot_dim / (rot_dim - 2.0))
    freq = base ** (-2.0 * i / rot_dim)
    if kind == "linear":
        freq = freq / factor
    elif kind == "yarn":
        fast, slow = float(s.pop("beta_fast", 32.0)), float(s.pop("beta_slow", 1.0))
        mult = float(s.pop("attention_factor", 0.1 * math.log(factor) + 1.0))
        # the pair that turns so many times over the trained positions
        pair = lambda turns: rot_dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot_dim - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        freq = freq * (1.0 - ramp) + freq / factor * ramp
    elif kind == "llama3":
        lo, hi = float(s.pop("low_freq_factor", 1.0)), float(s.pop("high_freq_factor", 4.0))
        mix = ((trained * freq / (2 * math.pi) - lo) / (hi - lo)).clamp(0.0, 1.0)
        freq = freq * mix + freq / factor * (1.0 - mix)
    elif kind not in ("none", "ntk"):
        raise ValueError(f"rope: unknown scaling {kind!r}")
    if s:
        raise ValueError(f"rope: {kind} scaling does not take {sorted(s)}")
    return freq, mult


def rope_table(rot_dim: int, max_pos: int, base: float = 10000.0, scaling: dict | None = None,
               device: torch.device | str = "cuda") -> torch.Tensor:
    """float32 [max_pos, 2, rot_dim / 2], the cosines and sines that rope and
    kv8_append read, computed in 64 bits and rounded once.  Made once."""
    freq, mult = rope_frequencies(rot_dim, base, scaling)
    angle = torch.arange(max_pos, dtype=torch.float64)[:, None] * freq
    return (torch.stack((angle.cos(), angle.sin()), 1) * mult).float().to(device)


# The C structures (zt_rows, zt_kv8_cache, zt_kv8_attn) as bytes that a call takes for a pointer to them: packing one
# costs a third of building a ctypes.Structure (0.5 us of a call's 10 instead of 2).
_ROWS = struct.Struct("@Pqqii")
_ROWS2 = struct.Struct("@PqqiiPqqii")
_NORM = struct.Struct("@PPd")
_CACHE = struct.Struct("@PPPPiiii")
_ATTN = struct.Struct("@PPPPiiiiPqqiiPqqiiPPPPiiiiiiii")


def _like(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x, memory_format=torch.contiguous_format)


class DecodeOps:
    """ROCmEngine's methods for the operators between the linear layers."""

    def _rows(self, x: torch.Tensor, name: str) -> tuple:
        """zt_rows' fields of a [tokens, heads, head_dim] tensor."""
        st = x.stride()
        if len(st) != 3 or x.device != self.device or (st[2] != 1 and x.shape[2] > 1):
            raise ValueError(f"{name} is [tokens, heads, head_dim] on the engine's device, values of a head neighbours")
        return x.data_ptr(), st[0], st[1], x.shape[1], 0

    def _dense(self, x: torch.Tensor | None, name: str, dtype: torch.dtype, shape: tuple) -> int:
        """The address of a contiguous tensor of that type and shape (None: any size) on the engine's device."""
        if x is None:
            return 0
        if x.dtype is dtype and x.is_contiguous() and x.device == self.device:
            have = x.shape
            if have == shape or (len(have) == len(shape) and all(n is None or n == m for n, m in zip(shape, have))):
                return x.data_ptr()
        raise ValueError(f"{name} is a contiguous {dtype} tensor {list(shape)} on the engine's device")

    def _type(self, name: str, x: torch.Tensor, *more: torch.Tensor) -> int:
        dtype = x.dtype
        t = _TYPES.get(dtype)
        for y in more:
            if y.dtype is not dtype:
                t = None
        if t is None:
            raise TypeError(f"{name} takes float32 or float16 tensors of one type")
        return t

    def _norm(self, norm: HeadNorm, dim: int) -> bytes:
        """zt_head_norm."""
        dense, f32, one = self._dense, torch.float32, (dim,)
        return _NORM.pack(dense(norm[0], "norm.q", f32, one), dense(norm[1], "norm.k", f32, one), norm[2])

    def _kv8(self, cache, head_dim: int) -> tuple:
        """zt_kv8_cache's fields."""
        k, v, ks, vs = cache
        shape, i8, dev = k.shape, torch.int8, self.device
        if len(shape) != 4 or k.dtype is not i8 or v.dtype is not i8 or k.device != dev or v.device != dev:
            raise ValueError("a cache is int8 [pages, kv_heads, page_tokens, Dp] keys and [.., Dp, page_tokens] values")
        pages, heads, page, dp = shape
        if (v.shape != (pages, heads, dp, page) or not k.is_contiguous() or not v.is_contiguous()
                or dp != (head_dim + 63) // 64 * 64):
            raise ValueError(f"cache of {tuple(k.shape)} keys and {tuple(v.shape)} values for heads of {head_dim}")
        return (k.data_ptr(), v.data_ptr(), self._dense(ks, "k_scale", torch.float32, (pages, heads)),
                self._dense(vs, "v_scale", torch.float32, (pages, heads)), pages, heads, head_dim, page)

    @_on_engine_stream
    def rope(self, q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, table: torch.Tensor, *,
             interleaved: bool = False, inverse: bool = False, q_out: torch.Tensor | None = None,
             k_out: torch.Tensor | None = None):
        """q and k ([tokens, heads, head_dim], any strides of tokens and heads)
        turned by their tokens' positions (int32 [tokens]) in one launch, as
        new tensors or into q_out and k_out, which may be q and k themselves.
        Returns (q, k); with k None, (q, None).  table: rope_table's, of all
        of the head or its first part.  inverse: by the negative angle, which
        is how a gradient goes back."""
        if q_out is None:
            q_out = _like(q)
        rows = self._rows
        if k is None:
            t, n = self._type("rope", q, q_out), 1
            ins, outs = _ROWS.pack(*rows(q, "q")), _ROWS.pack(*rows(q_out, "q_out"))
        else:
            if k_out is None:
                k_out = _like(k)
            t, n = self._type("rope", q, k, q_out, k_out), 2
            ins = _ROWS2.pack(*rows(q, "q"), *rows(k, "k"))
            outs = _ROWS2.pack(*rows(q_out, "q_out"), *rows(k_out, "k_out"))
            if k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2] or k_out.shape != k.shape:
                raise ValueError("rope: q, k and their outputs have the same tokens and head size")
        if q_out.shape != q.shape:
            raise ValueError("rope: q, k and their outputs have the same tokens and head size")
        tokens, _, dim = q.shape
        tab = self._dense(table, "table", torch.float32, (None, 2, None))
        self.lib.call("zt_rope", ins, outs, n, self._dense(positions, "positions", torch.int32, (tokens,)), tab, tokens,
                      dim, 2 * table.shape[2], table.shape[0], t, (_lib.ROPE_INTERLEAVED if interleaved else 0)
                      | (_lib.ROPE_INVERSE if inverse else 0), self._s)
        return q_out, k_out if n == 2 else None

    @_on_engine_stream
    def norm_rope(self, q: torch.Tensor, k: torch.Tensor | None, norm: HeadNorm, positions: torch.Tensor | None = None,
                  table: torch.Tensor | None = None, *, interleaved: bool = False, q_out: torch.Tensor | None = None,
                  k_out: torch.Tensor | None = None):
        """rope of q and k whose heads (of an even size up to 256) are normed
        first, in the same pass; without a table normed only.  The norm's
        squares are summed in 64 bits, and its factor, the products and the
        rotation rounded to 32 one by one; the result is rounded once to the
        tensors' type.  q_out and k_out may be q and k themselves."""
        if q_out is None:
            q_out = _like(q)
        rows = self._rows
        if k is None:
            t, n = self._type("norm_rope", q, q_out), 1
            ins, outs = _ROWS.pack(*rows(q, "q")), _ROWS.pack(*rows(q_out, "q_out"))
        else:
            if k_out is None:
                k_out = _like(k)
            t, n = self._type("norm_rope", q, k, q_out, k_out), 2
            ins = _ROWS2.pack(*rows(q, "q"), *rows(k, "k"))
            outs = _ROWS2.pack(*rows(q_out, "q_out"), *rows(k_out, "k_out"))
            if k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2] or k_out.shape != k.shape:
                raise ValueError("norm_rope: q, k and their outputs have the same tokens and head size")
        if q_out.shape != q.shape:
            raise ValueError("norm_rope: q, k and their outputs have the same tokens and head size")
        tokens, _, dim = q.shape
        pos = tab = half = most = 0
        if table is not None:
            if positions is None:
                raise ValueError("norm_rope: a rope table needs positions")
            pos = self._dense(positions, "positions", torch.int32, (tokens,))
            tab = self._dense(table, "table", torch.float32, (None, 2, None))
            most, _, half = table.shape
        self.lib.call("zt_norm_rope", ins, outs, n, self._norm(norm, dim), pos, tab, tokens, dim, 2 * half, most, t,
                      _lib.ROPE_INTERLEAVED if interleaved else 0, self._s)
        return q_out, k_out if n == 2 else None

    @_on_engine_stream
    def kv8_append(self, k: torch.Tensor, v: torch.Tensor, cache, slots: torch.Tensor, *,
                   positions: torch.Tensor | None = None, table: torch.Tensor | None = None,
                   interleaved: bool = False, q: torch.Tensor | None = None,
                   q_out: torch.Tensor | None = None, norm: HeadNorm | None = None) -> torch.Tensor | None:
        """Puts a step's keys and values ([tokens, kv_heads, head_dim]) into
        the cache at their slots (int64 [tokens], kv8_plan's).  With a rope
        table the keys are turned by their positions first, and q, if given,
        into a new tensor or q_out, which is returned.  With norm the heads of
        keys and q are normed before that (norm_rope's rule); q may then go
        without a table.

        A page's scale grows where the new values need it, and the codes that
        it holds are rounded to the new scale; a page that starts anew (its
        first place is among the slots) forgets what it held.  Tokens whose
        slot is outside the cache (-1) are left out, wherever they stand: a
        step's rejected tokens for instance.  The others of one page stand
        next to each other but for those, each slot once."""
        rows, pack = self._rows, _ROWS.pack
        krows, vrows = rows(k, "k"), rows(v, "v")
        tokens, heads, dim = k.shape
        if v.shape != k.shape:
            raise ValueError("kv8_append: k and v have one shape")
        qr = qo = None
        if q is not None:
            if (table is None and norm is None) or q.dim() != 3 or q.shape[0] != tokens or q.shape[2] != dim:
                raise ValueError("kv8_append: q goes with a rope table or a norm, and has k's tokens and head size")
            if q_out is None:
                q_out = _like(q)
            elif q_out.shape != q.shape:
                raise ValueError("kv8_append: q_out has q's shape")
            t = self._type("kv8_append", k, v, q, q_out)
            qr, qo = pack(*rows(q, "q")), pack(*rows(q_out, "q_out"))
        elif q_out is not None:
            raise ValueError("kv8_append: q_out goes with q")
        else:
            t = self._type("kv8_append", k, v)
        c = self._kv8(cache, dim)
        if heads != c[5]:
            raise ValueError(f"kv8_append: {heads} heads for a cache of {c[5]}")
        pos = tab = half = most = 0
        if table is not None:
            if positions is None:
                raise ValueError("kv8_append: a rope table needs positions")
            pos = self._dense(positions, "positions", torch.int32, (tokens,))
            tab = self._dense(table, "table", torch.float32, (None, 2, None))
            most, _, half = table.shape
        name, norms = ("zt_kv8_append", ()) if norm is None else ("zt_kv8_append_norm", (self._norm(norm, dim),))
        self.lib.call(name, _CACHE.pack(*c), pack(*krows), pack(*vrows),
                      self._dense(slots, "slots", torch.int64, (tokens,)), qr, qo, *norms, pos, tab, tokens, 2 * half,
                      most, t, _lib.ROPE_INTERLEAVED if interleaved else 0, self._s)
        return q_out

    @_on_engine_stream
    def kv8_dequant(self, cache, pages: torch.Tensor, head_dim: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The keys and values of some pages (int32 [n]) as fp32
        [n, kv_heads, page_tokens, head_dim], code * scale."""
        c, n = self._kv8(cache, head_dim), pages.numel()
        p = self._dense(pages, "pages", torch.int32, (n,))
        keys, values = torch.empty((2, n, c[5], c[7], head_dim), dtype=torch.float32, device=self.device).unbind()
        self.lib.call("zt_kv8_dequant", _CACHE.pack(*c), p, n, keys.data_ptr(), values.data_ptr(), self._s)
        return keys, values

    @_on_engine_stream
    def kv8_plan(self, kv_lens: torch.Tensor, new: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                 free_count: torch.Tensor, page_tokens: int, tokens: int, *, in_place: bool = False) -> KV8Plan:
        """The pages, slots and positions of a step that adds new[r] tokens to
        each request of kv_lens[r] (int32 [requests] both), `tokens` of them in
        all (or more: the rest get slot -1).  New pages come off the end of the
        first free_count (int32 [1]) of free_pages; a request that finds too
        few, or whose row of block_table (int32 [requests, width]) is full,
        gets none, nor do those after it that want some: their slots are -1
        and their lengths stay (kv_lens[r] as it was, though new[r] > 0).
        Their rows in q_start are still theirs; what kv8_attention gives for
        them has no meaning, and no token is to be drawn from it.  in_place:
        the new pages are written into block_table itself, not a copy."""
        r, width = block_table.shape
        dense, i32, one = self._dense, torch.int32, (r,)
        args = (dense(kv_lens, "kv_lens", i32, one), dense(new, "new", i32, one),
                dense(block_table, "block_table", i32, (r, width)), r, width,
                dense(free_pages, "free_pages", i32, (None,)), dense(free_count, "free_count", i32, (1,)),
                free_pages.shape[0], page_tokens, tokens)
        table = block_table if in_place else torch.empty_like(block_table)
        slots = torch.empty(tokens, dtype=torch.int64, device=self.device)
        small = torch.empty(tokens + 2 * r + 2, dtype=i32, device=self.device)
        positions, q_start, lens, left = small.split_with_sizes((tokens, r + 1, r, 1))
        at = small.data_ptr()
        self.lib.call("zt_kv8_plan", *args, table.data_ptr(), slots.data_ptr(), at, at + 4 * tokens,
                      at + 4 * (tokens + r + 1), at + 4 * (tokens + 2 * r + 1), self._s)
        return KV8Plan(table, slots, positions, q_start, lens, left)

    @_on_engine_stream
    def kv8_attention(self, q: torch.Tensor, cache, block_table: torch.Tensor, kv_lens: torch.Tensor,
                      q_start: torch.Tensor, *, max_q: int | None = None, max_kv: int | None = None,
                      window: int = 0, scale: torch.Tensor | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of q [tokens, heads, head_dim] over the cache:
        request r's rows are q_start[r] to q_start[r + 1] - 1, the last of its
        kv_lens[r] tokens, whose keys and values are in the cache already.
        window > 0: a row sees the last `window` tokens only.  scale: float32
        [1] on the device, 1 / sqrt(head_dim) without.  max_q, max_kv: bounds
        of the rows and the length of one request (without, what q and
        block_table allow): they choose the launch, not the result's meaning.
        Rows that see nothing are zeros.  A request whose step kv8_plan
        refused has rows, but no tokens for them: values without a meaning."""
        if out is None:
            out = _like(q)
        elif out.shape != q.shape:
            raise ValueError("kv8_attention: out has q's shape")
        t = self._type("kv8_attention", q, out)
        rows, dense, i32 = self._rows, self._dense, torch.int32
        qrows, orows = rows(q, "q"), rows(out, "out")
        tokens, heads, dim = q.shape
        c = self._kv8(cache, dim)
        r, width = block_table.shape
        if heads % c[5]:
            raise ValueError(f"kv8_attention: {heads} heads over {c[5]} of the cache")
        a = _ATTN.pack(*c, *qrows, *orows, dense(block_table, "block_table", i32, (r, width)),
                       dense(kv_lens, "kv_lens", i32, (r,)), dense(q_start, "q_start", i32, (r + 1,)),
                       dense(scale, "scale", torch.float32, (1,)), r, width, tokens, tokens if max_q is None else max_q,
                       min(width * c[7], 0x7FFFFFFF) if max_kv is None else max_kv, window, t, 0)
        ws, wsb = self._workspace(self.lib.zt_kv8_attention_workspace_bytes(a))
        self.lib.call("zt_kv8_attention", a, ws, wsb, self._s)
        return out

    @_on_engine_stream
    def sample(self, logits: torch.Tensor, u: torch.Tensor, *, temperature: torch.Tensor | None = None,
               top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
               min_p: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """A token (int64 [rows]) of each row of logits [rows, vocab] from the
        uniforms u in [0, 1) (float32 [rows]), and the log of its share of the
        kept probability (float32 [rows]).  temperature, top_p, min_p: float32
        [rows], top_k: int32 [rows], None: off.  temperature <= 0: the largest
        logit.  A row with no logit above -inf gives token -1."""
        st = logits.stride()
        if len(st) != 2 or logits.device != self.device or (st[1] != 1 and logits.shape[1] > 1):
            raise ValueError("sample: logits are [rows, vocab] on the engine's device, a row's values neighbours")
        rows, vocab = logits.shape
        t, f32, dense, one = self._type("sample", logits), torch.float32, self._dense, (rows,)
        args = (dense(u, "u", f32, one), dense(temperature, "temperature", f32, one),
                dense(top_k, "top_k", torch.int32, one), dense(top_p, "top_p", f32, one),
                dense(min_p, "min_p", f32, one))
        token = torch.empty(rows, dtype=torch.int64, device=self.device)
        logprob = torch.empty_like(u)
        ws, wsb = self._workspace(self.lib.zt_sample_workspace_bytes(rows, vocab))
        self.lib.call("zt_sample", logits.data_ptr(), st[0], rows, vocab, t, *args, token.data_ptr(),
                      logprob.data_ptr(), ws, wsb, self._s)
        return token, logprob
