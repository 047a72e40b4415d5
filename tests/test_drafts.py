"""The operators of drafted trees and shared pages without a GPU: their refusals
(nothing is launched: the pointers are not real), and the tests' own definitions."""
import ctypes
import itertools

import numpy as np
import pytest

import draft_ref
from ztensor_amd import _lib

BAD = _lib.HIP_ERROR_INVALID_VALUE
R, W, T, PAGES, FORKS = 4, 8, 9, 16, 5
SIZE = {"parents": 4 * T, "kv_lens": 4 * R, "keep": 4 * R, "held": 4 * R, "kept": 4 * R, "last": 4 * R, "token": 8 * R, "q_start": 4 * R + 4,
        "positions": 4 * T, "mask": 16 * T, "drafted": 8 * T, "drawn": 8 * T, "slots": 8 * T, "path": 4 * T, "table": 4 * R * W,
        "table_out": 4 * R * W, "lens_out": 4 * R, "free_pages": 4 * PAGES, "free_count": 4, "count_out": 4, "refs": 4 * PAGES,
        "source": 4 * FORKS, "target": 4 * FORKS, "copy_from": 4 * FORKS, "copy_to": 4 * FORKS}
AT = {n: (1 << 20) + 4096 * i for i, n in enumerate(SIZE)}
EIGHT = ("token", "mask", "drafted", "drawn", "slots")
ref = ctypes.byref


def cache(**other):
    return _lib.KV8(**{**dict(k=1 << 24, v=1 << 25, k_scale=1 << 26, v_scale=1 << 27, pages=8, kv_heads=2, head_dim=64, page_tokens=16), **other})


def caches(*c):
    return (_lib.KV8 * len(c))(*c)


def tree(**o):
    a = {**AT, "requests": R, "tokens": T, "words": 2, **o}
    return _lib.load().zt_kv8_tree(*(a[n] for n in ("parents", "kv_lens", "q_start", "requests", "tokens", "words", "positions", "mask")), None)


def accept(**o):
    a = {**AT, "requests": R, "tokens": T, **o}
    return _lib.load().zt_tree_accept(*(a[n] for n in ("drafted", "drawn", "parents", "q_start", "slots", "requests", "tokens", "path",
                                                       "kept", "last", "token")), None)


def compact(**o):
    a = {**AT, "caches": caches(cache()), "layers": 1, "requests": R, "width": W, "tokens": T, **o}
    return _lib.load().zt_kv8_compact(*(a[n] for n in ("caches", "layers", "table", "requests", "width", "held", "q_start", "path", "kept",
                                                       "tokens", "lens_out")), None)


def trim(**o):
    a = {**AT, "requests": R, "width": W, "pages": PAGES, "page": 16, **o}
    return _lib.load().zt_kv8_trim(*(a[n] for n in ("kv_lens", "keep", "table", "requests", "width", "free_pages", "free_count", "pages",
                                                    "page", "refs", "table_out", "count_out")), None)


def fork(**o):
    a = {**AT, "n": FORKS, "rows": R, "width": W, "pages": PAGES, "page": 16, "reserved": 0, **o}
    if a.get("null"):
        return _lib.load().zt_kv8_fork(None, None)
    names = ("source", "target", "kv_lens", "table", "free_pages", "free_count", "refs", "table_out", "lens_out", "count_out", "copy_from",
             "copy_to", "n", "rows", "width", "pages", "page", "reserved")
    return _lib.load().zt_kv8_fork(ref(_lib.KV8Fork(*(a[n] for n in names))), None)


IO = {tree: (("parents", "kv_lens", "q_start"), ("positions", "mask")),
      accept: (("drafted", "drawn", "parents", "q_start", "slots"), ("path", "kept", "last", "token")),
      compact: (("table", "held", "q_start", "path", "kept"), ("lens_out",)),
      trim: (("kv_lens", "keep", "table", "free_count"), ("free_pages", "refs", "table_out", "count_out")),
      fork: (("source", "target", "kv_lens", "table", "free_pages", "free_count"),
             ("refs", "table_out", "lens_out", "count_out", "copy_from", "copy_to"))}
OPTIONAL = {(accept, "parents"), (accept, "slots"), (trim, "refs")}


@pytest.mark.parametrize("call", IO, ids=lambda c: c.__name__)
def test_buffers(call):
    ins, outs = IO[call]
    for name in ins + outs:
        if (call, name) not in OPTIONAL:
            assert call(**{name: 0}) == BAD, name
        assert call(**{name: AT[name] + (4 if name in EIGHT else 2)}) == BAD, name
    for out, other in itertools.product(outs, ins + outs):
        if out == other or (call is trim and {out, other} == {"table", "table_out"}):
            continue
        assert call(**{out: AT[other]}) == BAD, (out, other)
        step = 8 if out in EIGHT or other in EIGHT else 4
        if SIZE[other] > step:
            assert call(**{out: AT[other] + (SIZE[other] - 1) // step * step}) == BAD, (out, other)
    if call is trim:  # a table may be written in place, but not half
        assert call(table_out=AT["table"] + 4) == BAD


def test_sizes():
    for bad in (dict(requests=-1), dict(requests=1 << 24), dict(tokens=-1), dict(words=0), dict(words=17)):
        assert tree(**bad) == BAD, bad
    assert tree(tokens=0) == 0
    for bad in (dict(requests=-1), dict(requests=1 << 24), dict(tokens=-1)):
        assert accept(**bad) == BAD, bad
    assert accept(tokens=0, requests=0) == 0
    shapes = [caches(cache(), cache(**b)) for b in (dict(pages=9), dict(kv_heads=1), dict(head_dim=72), dict(page_tokens=32), dict(k=0), dict(v=(1 << 25) + 8))]
    for c in shapes:
        assert compact(caches=c, layers=2) == BAD and copy(caches=c, layers=2) == BAD
    for bad in (dict(caches=None), dict(layers=0), dict(layers=-1), dict(requests=-1), dict(width=0), dict(tokens=-1),
                dict(requests=1 << 16, width=1 << 15)):
        assert compact(**bad) == BAD, bad
    assert compact(requests=0) == 0 and compact(layers=(1 << 16) + 1) == BAD
    for bad in (dict(requests=-1), dict(width=0), dict(pages=-1), dict(pages=(1 << 20) + 1), dict(page=8), dict(page=48),
                dict(requests=1 << 16, width=1 << 15), dict(requests=1 << 24)):
        assert trim(**bad) == BAD, bad
    for bad in (dict(n=-1), dict(rows=-1), dict(width=0), dict(pages=-1), dict(page=24), dict(reserved=1), dict(null=True),
                dict(rows=1 << 16, width=1 << 15), dict(rows=1 << 24), dict(n=1 << 24)):
        assert fork(**bad) == BAD, bad


def copy(**o):
    a = {"caches": caches(cache()), "layers": 1, "source": 1 << 20, "target": 1 << 21, "n": 3, **o}
    return _lib.load().zt_kv8_copy(*(a[n] for n in ("caches", "layers", "source", "target", "n")), None)


def test_copy_refuses():
    assert copy(n=0) == 0
    for bad in (dict(caches=None), dict(layers=0), dict(source=0), dict(target=0), dict(source=(1 << 20) + 2), dict(n=-1),
                dict(caches=caches(cache(page_tokens=24))), dict(n=(1 << 31) - 1)):
        assert copy(**bad) == BAD, bad


def test_tree_attention_refuses():
    lib = _lib.load()
    rows = _lib.Rows(1 << 20, 256, 64, 4, 0)

    def call(mask=1 << 20, words=1, ws=1 << 20, wsb=1 << 40, **other):
        a = _lib.KV8Attn(**{**dict(cache=cache(), q=rows, out=rows, table=1 << 20, kv_lens=1 << 20, q_start=1 << 20, requests=2, width=4,
                                   tokens=3, max_q=2, max_kv=64), **other})
        return lib.zt_kv8_tree_attention(ref(a), mask, words, ws, wsb, None)

    assert call(tokens=0) == 0 and call(tokens=0, mask=0) == 0
    for bad in (dict(mask=0), dict(mask=(1 << 20) + 4), dict(words=0), dict(words=17), dict(words=-1), dict(ws=0), dict(ws=(1 << 20) + 8),
                dict(wsb=16), dict(table=0), dict(kv_lens=0), dict(q_start=0), dict(type=2), dict(window=-1), dict(width=0),
                dict(cache=cache(head_dim=60)), dict(tokens=-1), dict(reserved=1), dict(scale=2)):
        assert call(**bad) == BAD, bad
    assert lib.zt_kv8_tree_attention(None, 1 << 20, 1, 1 << 20, 1 << 40, None) == BAD


def test_packed_structure_is_the_c_one():
    drafts = pytest.importorskip("ztensor_amd.drafts")
    assert drafts._FORK.size == ctypes.sizeof(_lib.KV8Fork)
    f = _lib.KV8Fork.from_buffer_copy(drafts._FORK.pack(*range(1, 19)))
    assert (f.source, f.refs, f.copy_to, f.n, f.rows, f.width, f.pages, f.page_tokens, f.reserved) == (1, 7, 12, 13, 14, 15, 16, 17, 18)


def test_definitions_by_hand():
    positions, mask = draft_ref.tree(np.array([-1, 0, 0, 1, 9, -1, 0]), [10, 2], [0, 5, 7], 8, 1)
    assert positions.tolist() == [5, 6, 6, 7, 5, 0, 1, 0]
    assert mask[:, 0].tolist() == [0b1, 0b11, 0b101, 0b1011, 0b10000, 0b1, 0b11, 0]
    got = draft_ref.accept([5, 6, 7, 7, 8], [7, 1, 9, 8, 3], [-1, 0, 0, 0, 2], [0, 5])
    assert [x if isinstance(x, list) else x.tolist() for x in got] == [[0, 2, -1, -1, -1], [2], [2], [9]]
    table = np.array([[3, 1, 2], [3, 4, -1]])
    assert draft_ref.trim([40, 20], [3, 0], table, [0], 5, 16, [0, 0, 0, 1, 0])[1:] == ([0, 1, 2, 4], [0, 0, 0, 0, 0])
    t, lens, free, refs, a, b = draft_ref.fork([0, 0], [1, 2], [20, 0, 0], np.array([[3, 1], [-1, -1], [-1, -1]]), [0, 7], 16, [0] * 8)
    assert t.tolist() == [[3, 1], [3, 7], [3, 0]] and lens == [20, 20, 20] and free == [] and refs[3] == 2 and (a, b) == ([1, 1], [7, 0])
