"""Drafted trees and shared pages on the int8 paged cache.

A step that checks drafted tokens instead of adding one: each request's first
row is the token that it stands at, the others are drafts that continue an
earlier row of it (its parent).  With `held` the lengths before the step:

    p = engine.kv8_plan(held, new, block_table, free_pages, free_count, page_tokens, tokens)
    t = engine.kv8_tree(parents, p.kv_lens, p.q_start, max_q)  # (window= for a model that has one, here and in the attention)
    for each layer:
        q = engine.kv8_append(k, v, cache, p.slots, positions=t.positions, table=rope, q=q)
        a = engine.kv8_tree_attention(q, cache, p.block_table, p.kv_lens, p.q_start, t.mask, max_q=..., max_kv=...)
    drawn, _ = engine.sample(logits of all rows, u, ...)
    took = engine.tree_accept(drafted, drawn, p.q_start, parents=parents, slots=p.slots)
    lens = engine.kv8_compact(caches, p.block_table, held, p.q_start, took.path, took.kept)
    left = engine.kv8_trim(p.kv_lens, lens, p.block_table, free_pages, p.free_count, page_tokens)

after which each request stands at took.token[r], and holds lens[r] tokens.

Sequences that go on from others (several answers to a prompt, beams) share
their full pages; refs counts for each page how many sequences hold it besides
one:

    f = engine.kv8_fork(source, target, kv_lens, block_table, refs, free_pages, free_count, page_tokens)
    engine.kv8_copy(caches, f.copy_from, f.copy_to)

and kv8_trim with refs gives a page back when its last holder does.  Beams, whose
targets held something else: the forks first, then what those rows held goes back
by the table from before (keep 0 for the targets, the others' lengths for them):

    left = engine.kv8_trim(kv_lens, keep, block_table, free_pages, f.free_count, page_tokens, refs=refs)
    # on with f.block_table, f.kv_lens and left.free_count

A step writes into the page that a sequence's last tokens are on, if it is not
full, so that page has to be its own: who is cut in the middle of a page that
others hold too goes on as a fork of itself, in another row.
"""
from __future__ import annotations

import struct
from typing import NamedTuple, Sequence

import torch

from . import _lib
from ._stream import _on_engine_stream
from .decode import _ATTN, _CACHE, DecodeOps, _like

_FORK = struct.Struct("@12P6i")


class KV8Tree(NamedTuple):
    """What kv8_tree gives for a step."""

    positions: torch.Tensor  # int32 [tokens]
    mask: torch.Tensor  # int64 [tokens, words]


class TreeAccept(NamedTuple):
    """What tree_accept gives for a step."""

    path: torch.Tensor  # int32 [tokens]: of each request the kept rows, counted from its first, then -1
    kept: torch.Tensor  # int32 [requests]
    last: torch.Tensor  # int32 [requests]: the last kept row, counted from the step's first; -1: none
    token: torch.Tensor  # int64 [requests]: drawn there; -1: none


class KV8Trim(NamedTuple):
    """What kv8_trim gives."""

    block_table: torch.Tensor  # int32 [requests, width]
    free_count: torch.Tensor  # int32 [1]


class KV8Fork(NamedTuple):
    """What kv8_fork gives."""

    block_table: torch.Tensor  # int32 [rows, width]
    kv_lens: torch.Tensor  # int32 [rows]
    free_count: torch.Tensor  # int32 [1]
    copy_from: torch.Tensor  # int32 [forks], -1: nothing to copy
    copy_to: torch.Tensor


class DraftOps(DecodeOps):
    """ROCmEngine's methods for drafted trees and shared pages."""

    def _caches(self, caches: Sequence) -> tuple[bytes, int]:
        """zt_kv8_cache of each."""
        packed = []
        for cache in caches:
            shape = cache[0].shape
            packed.append(_CACHE.pack(*self._kv8(cache, shape[3] if len(shape) == 4 else 0)))
        return b"".join(packed), len(packed)

    @_on_engine_stream
    def kv8_tree(self, parents: torch.Tensor, kv_lens: torch.Tensor, q_start: torch.Tensor, max_q: int, *,
                 window: int = 0) -> KV8Tree:
        """Positions and masks of a step's trees.  parents (int32 [tokens]): the
        row of its request that a row continues, counted from the request's
        first row and before it (else, -1 for instance, the context).  kv_lens
        and q_start: kv8_plan's, the step's tokens included.  max_q, at most
        1024: a bound of the rows of one request; a row that is past the mask's
        words (64 rows each) is seen by none.  window: the attention's; rows
        that many steps above a row, or more, are not in its mask."""
        tokens, r, i32 = parents.shape[0], kv_lens.shape[0], torch.int32
        words = max(1, -(-max_q // 64))
        dense = self._dense
        args = (dense(parents, "parents", i32, (tokens,)), dense(kv_lens, "kv_lens", i32, (r,)),
                dense(q_start, "q_start", i32, (r + 1,)), r, tokens, words)
        positions = torch.empty(tokens, dtype=i32, device=self.device)
        mask = torch.empty((tokens, words), dtype=torch.int64, device=self.device)
        self.lib.call("zt_kv8_tree_window", *args, window, positions.data_ptr(), mask.data_ptr(), self._s)
        return KV8Tree(positions, mask)

    @_on_engine_stream
    def kv8_tree_attention(self, q: torch.Tensor, cache, block_table: torch.Tensor, kv_lens: torch.Tensor,
                           q_start: torch.Tensor, mask: torch.Tensor, *, max_q: int | None = None,
                           max_kv: int | None = None, window: int = 0, scale: torch.Tensor | None = None,
                           out: torch.Tensor | None = None) -> torch.Tensor:
        """kv8_attention for rows that are not in a line: row i of a request
        sees its context (the tokens before the request's rows) and, of those
        rows, row j where bit j % 64 of mask[i, j // 64] is set (int64 [tokens,
        words]; kv8_tree's, or any other).  window > 0: of the context the
        tokens after position - window, its position being the context's length
        and the rows that it sees, less one; of the request's rows what the mask
        has (give kv8_tree the same window).  A row that sees nothing is zeros."""
        if out is None:
            out = _like(q)
        elif out.shape != q.shape:
            raise ValueError("kv8_tree_attention: out has q's shape")
        t = self._type("kv8_tree_attention", q, out)
        rows, dense, i32 = self._rows, self._dense, torch.int32
        qrows, orows = rows(q, "q"), rows(out, "out")
        tokens, heads, dim = q.shape
        c = self._kv8(cache, dim)
        r, width = block_table.shape
        if heads % c[5]:
            raise ValueError(f"kv8_tree_attention: {heads} heads over {c[5]} of the cache")
        bits = dense(mask, "mask", torch.int64, (tokens, None))
        a = _ATTN.pack(*c, *qrows, *orows, dense(block_table, "block_table", i32, (r, width)),
                       dense(kv_lens, "kv_lens", i32, (r,)), dense(q_start, "q_start", i32, (r + 1,)),
                       dense(scale, "scale", torch.float32, (1,)), r, width, tokens, tokens if max_q is None else max_q,
                       min(width * c[7], 0x7FFFFFFF) if max_kv is None else max_kv, window, t, 0)
        ws, wsb = self._workspace(self.lib.zt_kv8_tree_attention_workspace_bytes(a))
        self.lib.call("zt_kv8_tree_attention", a, bits, mask.shape[1], ws, wsb, self._s)
        return out

    @_on_engine_stream
    def tree_accept(self, drafted: torch.Tensor, drawn: torch.Tensor, q_start: torch.Tensor, *,
                    parents: torch.Tensor | None = None, slots: torch.Tensor | None = None) -> TreeAccept:
        """The path of each request's tree that the drawn tokens accept: its
        first row, then, again and again, the first row whose parent that is
        and whose token (drafted, int64 [tokens]) is the one drawn after it
        (drawn, int64 [tokens]: a sample of every row).  parents None: a chain.
        slots (kv8_plan's): a request without pages keeps nothing."""
        tokens, r, i32, i64 = drafted.shape[0], q_start.shape[0] - 1, torch.int32, torch.int64
        if r < 0:
            raise ValueError("tree_accept: q_start has an entry more than there are requests")
        dense, one = self._dense, (tokens,)
        args = (dense(drafted, "drafted", i64, one), dense(drawn, "drawn", i64, one), dense(parents, "parents", i32, one),
                dense(q_start, "q_start", i32, (None,)), dense(slots, "slots", i64, one), r, tokens)
        small = torch.empty(tokens + 2 * r, dtype=i32, device=self.device)
        token = torch.empty(r, dtype=i64, device=self.device)
        path, kept, last = small.split_with_sizes((tokens, r, r))
        at = small.data_ptr()
        self.lib.call("zt_tree_accept", *args, at, at + 4 * tokens, at + 4 * (tokens + r), token.data_ptr(), self._s)
        return TreeAccept(path, kept, last, token)

    @_on_engine_stream
    def kv8_compact(self, caches: Sequence, block_table: torch.Tensor, held: torch.Tensor, q_start: torch.Tensor,
                    path: torch.Tensor, kept: torch.Tensor) -> torch.Tensor:
        """Moves each request's kept rows (tree_accept's path and kept) to the
        end of the held[r] tokens that it had before the step (int32
        [requests]), in the caches of all layers, which have one shape; returns
        the lengths, held + kept.  A code that goes to another page is rounded
        to that page's scale, which grows where it has to."""
        packed, n = self._caches(caches)
        r, width = block_table.shape
        dense, i32, one = self._dense, torch.int32, (r,)
        args = (dense(block_table, "block_table", i32, (r, width)), r, width, dense(held, "held", i32, one),
                dense(q_start, "q_start", i32, (r + 1,)), dense(path, "path", i32, (None,)), dense(kept, "kept", i32, one),
                path.shape[0])
        lens = torch.empty(r, dtype=i32, device=self.device)
        self.lib.call("zt_kv8_compact", packed, n, *args, lens.data_ptr(), self._s)
        return lens

    @_on_engine_stream
    def kv8_copy(self, caches: Sequence, source: torch.Tensor, target: torch.Tensor) -> None:
        """Copies pages (int32 [n] both; -1: none) in the caches of all layers,
        which have one shape.  No page is a target twice, or source and target."""
        packed, layers = self._caches(caches)
        n, i32 = source.shape[0], torch.int32
        self.lib.call("zt_kv8_copy", packed, layers, self._dense(source, "source", i32, (n,)),
                      self._dense(target, "target", i32, (n,)), n, self._s)

    @_on_engine_stream
    def kv8_trim(self, kv_lens: torch.Tensor, keep: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                 free_count: torch.Tensor, page_tokens: int, *, refs: torch.Tensor | None = None,
                 in_place: bool = False) -> KV8Trim:
        """Cuts requests of kv_lens[r] tokens to the first keep[r] (int32
        [requests] both; 0 ends a request): pages that nothing is left on become
        -1 in the table and go to the end of the free list, whose first
        free_count (int32 [1]) entries are there.  free_pages (int32 [pages])
        has room for all pages and is written in place.  refs (int32 [pages],
        in place too): a page that others hold as well stays, with one holder
        fewer (one that keep[r] ends in is not to be written to then: a fork of
        the request has its own).  in_place: the -1 are written into block_table
        itself."""
        r, width = block_table.shape
        dense, i32, one = self._dense, torch.int32, (r,)
        pages = free_pages.shape[0]
        args = (dense(kv_lens, "kv_lens", i32, one), dense(keep, "keep", i32, one),
                dense(block_table, "block_table", i32, (r, width)), r, width,
                dense(free_pages, "free_pages", i32, (pages,)), dense(free_count, "free_count", i32, (1,)), pages,
                page_tokens, dense(refs, "refs", i32, (pages,)))
        table = block_table if in_place else torch.empty_like(block_table)
        left = torch.empty_like(free_count)
        self.lib.call("zt_kv8_trim", *args, table.data_ptr(), left.data_ptr(), self._s)
        return KV8Trim(table, left)

    @_on_engine_stream
    def kv8_fork(self, source: torch.Tensor, target: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor,
                 refs: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor, page_tokens: int) -> KV8Fork:
        """Row target[i] of block_table goes on from what row source[i] holds
        before the call (int32 [forks] both; of forks with one target the first
        is done, the others are nothing).  Full pages are
        shared (refs, int32 [pages], one more, in place); a last page that is
        not full gets a page of its own, and copy_from / copy_to are what
        kv8_copy is to do for it.  A fork that finds no free page gets length 0.
        What a target's row held is not given back: kv8_trim does that, before,
        or after with block_table as it was."""
        n, (r, width), i32, dense = source.shape[0], block_table.shape, torch.int32, self._dense
        pages = free_pages.shape[0]
        args = (dense(source, "source", i32, (n,)), dense(target, "target", i32, (n,)), dense(kv_lens, "kv_lens", i32, (r,)),
                dense(block_table, "block_table", i32, (r, width)), dense(free_pages, "free_pages", i32, (pages,)),
                dense(free_count, "free_count", i32, (1,)), dense(refs, "refs", i32, (pages,)))
        if refs is None:
            raise ValueError("kv8_fork: refs are needed")
        table = torch.empty_like(block_table)
        small = torch.empty(r + 1 + 2 * n, dtype=i32, device=self.device)
        lens, left, copy_from, copy_to = small.split_with_sizes((r, 1, n, n))
        at = small.data_ptr()
        self.lib.call("zt_kv8_fork", _FORK.pack(*args, table.data_ptr(), at, at + 4 * r, at + 4 * (r + 1),
                                                at + 4 * (r + 1 + n), n, r, width, pages, page_tokens, 0), self._s)
        return KV8Fork(table, lens, left, copy_from, copy_to)
