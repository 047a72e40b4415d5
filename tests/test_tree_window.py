"""A tree's masks for attention with a window: refusals, without a GPU (nothing is launched: the pointers are not real)."""
from test_drafts import AT, BAD, R, T
from ztensor_amd import _lib


def call(**o):
    a = {**AT, "requests": R, "tokens": T, "words": 2, "window": 5, **o}
    names = ("parents", "kv_lens", "q_start", "requests", "tokens", "words", "window", "positions", "mask")
    return _lib.load().zt_kv8_tree_window(*(a[n] for n in names), None)


def test_refuses():
    assert call(tokens=0) == 0
    for bad in (dict(window=-1), dict(window=-2 ** 31), dict(requests=-1), dict(requests=1 << 24), dict(tokens=-1), dict(words=0), dict(words=17),
                dict(parents=0), dict(kv_lens=0), dict(q_start=0), dict(positions=0), dict(mask=0), dict(mask=AT["mask"] + 4),
                dict(positions=AT["parents"]), dict(mask=AT["positions"])):
        assert call(**bad) == BAD, bad
