"""The decode operators without a GPU: the entry points' refusals (nothing is
launched: the pointers are not real), and the rotary tables."""
import ctypes
import math

import numpy as np
import pytest

from ztensor_amd import _lib

torch = pytest.importorskip("torch")

from ztensor_amd.decode import rope_frequencies, rope_table  # noqa: E402

P, BAD = 1 << 20, _lib.HIP_ERROR_INVALID_VALUE


def rows(p=P, heads=4, reserved=0):
    return _lib.Rows(p, heads * 64, 64, heads, reserved)


def cache(**other):
    return _lib.KV8(**{**dict(k=P, v=P, k_scale=P, v_scale=P, pages=8, kv_heads=2, head_dim=64, page_tokens=16), **other})


BAD_CACHES = [dict(k=0), dict(v=P + 8), dict(k_scale=0), dict(v_scale=0), dict(pages=-1), dict(kv_heads=0), dict(head_dim=60),
              dict(head_dim=264), dict(head_dim=0), dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=256),
              dict(pages=1 << 28)]


def test_packed_structures_are_the_c_ones():
    from ztensor_amd import decode

    for packed, c in ((decode._ROWS, _lib.Rows), (decode._ROWS2, _lib.Rows * 2), (decode._CACHE, _lib.KV8),
                      (decode._ATTN, _lib.KV8Attn)):
        assert packed.size == ctypes.sizeof(c)
    fields = decode._ATTN.pack(*range(1, 31))
    a = _lib.KV8Attn.from_buffer_copy(fields)
    assert (a.cache.k, a.cache.page_tokens, a.q.p, a.q.heads, a.out.p, a.out.head_stride, a.table, a.scale, a.requests,
            a.type, a.reserved) == (1, 8, 9, 12, 14, 16, 19, 22, 23, 29, 30)


def test_rope_refuses():
    lib, two = _lib.load(), (_lib.Rows * 2)(rows(), rows())

    def call(ins=two, outs=two, n=2, pos=P, table=P, tokens=3, dim=64, rot=64, most=100, type=0, flags=0):
        return lib.zt_rope(ins, outs, n, pos, table, tokens, dim, rot, most, type, flags, None)

    arr = lambda a, b: (_lib.Rows * 2)(a, b)  # noqa: E731
    assert call(tokens=0) == 0
    for bad in (dict(n=0), dict(n=3), dict(ins=None), dict(outs=None), dict(tokens=-1), dict(dim=0), dict(dim=63, rot=62),
                dict(rot=0), dict(rot=63), dict(rot=66), dict(most=0), dict(type=2), dict(type=-1), dict(flags=4), dict(pos=0),
                dict(table=0), dict(pos=P + 2), dict(table=P + 1), dict(ins=arr(rows(0), rows())),
                dict(outs=arr(rows(), rows(P + 2))), dict(outs=arr(rows(heads=3), rows())),
                dict(ins=arr(rows(reserved=1), rows())), dict(ins=arr(rows(heads=0), rows()), outs=arr(rows(heads=0), rows()))):
        assert call(**bad) == BAD, bad


def test_append_and_dequant_refuse():
    lib, ref = _lib.load(), ctypes.byref

    def call(c=cache(), k=rows(heads=2), v=rows(heads=2), slots=P, q=None, q_out=None, pos=P, table=P, tokens=3, rot=64,
             most=100, type=0, flags=0):
        r = lambda x: None if x is None else ref(x)  # noqa: E731
        return lib.zt_kv8_append(r(c), r(k), r(v), slots, r(q), r(q_out), pos, table, tokens, rot, most, type, flags, None)

    assert call(tokens=0) == 0
    cases = [dict(c=cache(**b)) for b in BAD_CACHES]
    cases += [dict(c=None), dict(k=None), dict(v=None), dict(slots=0), dict(slots=P + 4), dict(q=rows()), dict(q_out=rows()),
              dict(q=rows(), q_out=rows(), table=0), dict(q=rows(), q_out=rows(heads=3)), dict(pos=0), dict(tokens=-1),
              dict(rot=3), dict(rot=66), dict(rot=0), dict(most=0), dict(type=5), dict(flags=2), dict(k=rows(heads=3)),
              dict(v=rows(heads=1)), dict(k=rows(0, 2)), dict(v=rows(P + 2, 2))]
    for bad in cases:
        assert call(**bad) == BAD, bad
    assert lib.zt_kv8_dequant(ref(cache()), P, 0, P, P, None) == 0
    for args in [(ref(cache()), P, -1, P, P), (ref(cache()), 0, 1, P, P), (ref(cache()), P, 1, 0, P), (None, P, 1, P, P),
                 (ref(cache()), P, 1, P, P + 2)] + [(ref(cache(**b)), P, 1, P, P) for b in BAD_CACHES]:
        assert lib.zt_kv8_dequant(*args, None) == BAD


def test_plan_refuses():
    lib = _lib.load()
    names = ("lens add table requests width free count capacity page tokens table_out slots positions q_start lens_out "
             "count_out").split()
    good = dict(zip(names, (P, P, P, 4, 8, P, P, 16, 16, 9, P, P, P, P, P + 64, P + 128)))
    for bad in [{n: 0} for n in ("lens", "add", "table", "free", "count", "table_out", "slots", "positions", "q_start",
                                 "lens_out", "count_out", "width", "page")] + [
            dict(requests=-1), dict(width=-1), dict(tokens=-1), dict(capacity=-1), dict(page=24), dict(page=256),
            dict(slots=P + 4), dict(positions=P + 2), dict(requests=1 << 20, width=1 << 12), dict(lens_out=P),
            dict(count_out=P)]:
        assert lib.zt_kv8_plan(*{**good, **bad}.values(), None) == BAD, bad


def test_attention_refuses():
    lib = _lib.load()

    def desc(**other):
        c = {k: other.pop(k) for k in list(other) if k in dict(_lib.KV8._fields_)}
        return _lib.KV8Attn(**{**dict(cache=cache(**c), q=rows(), out=rows(), table=P, kv_lens=P, q_start=P, scale=0, requests=2,
                                      width=4, tokens=3, max_q=2, max_kv=64, window=0, type=0, reserved=0), **other})

    big = 1 << 40
    assert lib.zt_kv8_attention(ctypes.byref(desc(tokens=0)), P, big, None) == 0
    shape = [dict(b) for b in BAD_CACHES] + [dict(requests=-1), dict(width=0), dict(tokens=-1), dict(max_q=-1), dict(max_kv=-1),
                                             dict(window=-1), dict(type=2), dict(reserved=1), dict(q=rows(heads=3)),
                                             dict(q=rows(heads=3), out=rows(heads=3)), dict(out=rows(heads=2))]
    for bad in shape:
        assert lib.zt_kv8_attention_workspace_bytes(ctypes.byref(desc(**bad))) == -1, bad
        assert lib.zt_kv8_attention(ctypes.byref(desc(**bad)), P, big, None) == BAD, bad
    for bad in (dict(table=0), dict(kv_lens=0), dict(q_start=0), dict(q_start=P + 2), dict(scale=P + 1), dict(q=rows(0)),
                dict(out=rows(P + 2)), dict(q=rows(reserved=1))):
        assert lib.zt_kv8_attention(ctypes.byref(desc(**bad)), P, big, None) == BAD, bad
    assert lib.zt_kv8_attention(None, P, big, None) == BAD and lib.zt_kv8_attention_workspace_bytes(None) == -1
    need = desc(max_kv=100000, width=7000, requests=1, max_q=1)
    bytes_ = lib.zt_kv8_attention_workspace_bytes(ctypes.byref(need))
    if bytes_ > 0:
        for ws, n in ((0, bytes_), (P, bytes_ - 1), (P + 8, bytes_)):
            assert lib.zt_kv8_attention(ctypes.byref(need), ws, n, None) == BAD


def test_sample_refuses():
    lib = _lib.load()

    def call(logits=P, stride=100, rows=2, vocab=100, type=0, u=P, t=0, k=0, p=0, m=0, token=P, logprob=P, ws=P, wsb=1 << 40):
        return lib.zt_sample(logits, stride, rows, vocab, type, u, t, k, p, m, token, logprob, ws, wsb, None)

    assert call(rows=0) == 0
    for bad in (dict(logits=0), dict(u=0), dict(token=0), dict(logprob=0), dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 20) + 1),
                dict(type=3), dict(token=P + 4), dict(t=P + 2), dict(k=P + 1), dict(p=P + 2), dict(m=P + 3), dict(logits=P + 2),
                dict(logprob=P + 2)):
        assert call(**bad) == BAD, bad
    assert lib.zt_sample_workspace_bytes(-1, 5) == -1 and lib.zt_sample_workspace_bytes(1, 0) == -1
    need = lib.zt_sample_workspace_bytes(2, 100)
    if need > 0:
        for ws, n in ((0, need), (P, need - 1), (P + 8, need)):
            assert call(ws=ws, wsb=n) == BAD


def test_rope_tables():
    """The tables against the formulas, value by value."""
    rot, base = 64, 10000.0
    plain = [base ** (-2 * i / rot) for i in range(rot // 2)]
    for scaling, mult in ((None, 1), ({"type": "linear", "factor": 4}, 1), ({"type": "ntk", "factor": 4}, 1),
                          ({"type": "yarn", "factor": 8, "original_max_position": 2048}, 0.1 * math.log(8) + 1),
                          ({"type": "llama3", "factor": 8, "original_max_position": 1024}, 1)):
        f, m = rope_frequencies(rot, base, scaling)
        assert m == pytest.approx(mult)
        kind = scaling and scaling["type"]
        for i, x in enumerate(plain):
            if kind == "linear":
                x /= 4
            elif kind == "ntk":
                x = (base * 4 ** (rot / (rot - 2))) ** (-2 * i / rot)
            elif kind == "yarn":
                turns = 2048 * x / (2 * math.pi)
                edge = lambda n: rot * math.log(2048 / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
                lo, hi = math.floor(edge(32)), math.ceil(edge(1))
                far = min(1.0, max(0.0, (i - lo) / (hi - lo)))
                assert (turns > 40) <= (far == 0) and (turns < 0.7) <= (far == 1)
                x = x * (1 - far) + x / 8 * far
            elif kind == "llama3":
                wave = 2 * math.pi / x
                if wave > 1024:
                    x /= 8
                elif wave > 256:
                    s = (1024 / wave - 1) / 3
                    x = (1 - s) * x / 8 + s * x
            assert f[i].item() == pytest.approx(x, rel=1e-12)
        t = rope_table(rot, 50, base, scaling, "cpu")
        assert t.shape == (50, 2, 32) and t.dtype == torch.float32
        want = np.stack([np.cos(49 * f.numpy()), np.sin(49 * f.numpy())]) * m
        assert np.array_equal(t[49].numpy(), want.astype(np.float32))
    # the slowest pair is stretched by the factor, the fastest stays
    f, _ = rope_frequencies(rot, base, {"type": "ntk", "factor": 4})
    assert f[0] == 1.0 and f[-1].item() == pytest.approx(plain[-1] / 4)
    for bad in (dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=8, scaling={"type": "other"}),
                dict(rot_dim=8, scaling={"type": "yarn", "factor": 2}), dict(rot_dim=8, scaling={"type": "linear", "factor": 0.5}),
                dict(rot_dim=8, scaling={"type": "linear", "factor": 2, "beta_fast": 1}),
                dict(rot_dim=2, scaling={"type": "ntk", "factor": 2})):
        with pytest.raises(ValueError):
            rope_frequencies(**bad)
