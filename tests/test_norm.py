"""zt_norm_rope and zt_kv8_append_norm without a GPU: their refusals (nothing is
launched: the pointers are not real)."""
import ctypes

import pytest

from ztensor_amd import _lib

P, BAD = 1 << 20, _lib.HIP_ERROR_INVALID_VALUE
ref = ctypes.byref


def rows(p=P, heads=4, reserved=0):
    return _lib.Rows(p, heads * 64, 64, heads, reserved)


def norm(q=P, k=P, eps=1e-6):
    return _lib.HeadNorm(q, k, eps)


BAD_NORMS = [dict(eps=0.0), dict(eps=-1e-6), dict(eps=float("nan")), dict(eps=float("inf")), dict(q=P + 2), dict(k=P + 1)]


def test_packed_structure_is_the_c_one():
    decode = pytest.importorskip("ztensor_amd.decode")
    assert decode._NORM.size == ctypes.sizeof(_lib.HeadNorm)
    n = _lib.HeadNorm.from_buffer_copy(decode._NORM.pack(1, 2, 0.5))
    assert (n.q, n.k, n.eps) == (1, 2, 0.5)


def test_norm_rope_refuses():
    lib, two = _lib.load(), (_lib.Rows * 2)(rows(), rows())

    def call(ins=two, outs=two, n=2, norm=ref(norm()), pos=P, table=P, tokens=3, dim=64, rot=64, most=100, type=0, flags=0):
        return lib.zt_norm_rope(ins, outs, n, norm, pos, table, tokens, dim, rot, most, type, flags, None)

    arr = lambda a, b: (_lib.Rows * 2)(a, b)  # noqa: E731
    assert call(tokens=0) == 0
    assert call(tokens=0, table=0, pos=0, rot=0, most=0) == 0 and call(tokens=0, norm=ref(norm(0, 0))) == 0
    bad = [dict(norm=ref(norm(**b))) for b in BAD_NORMS]
    bad += [dict(norm=None), dict(n=0), dict(n=3), dict(ins=None), dict(outs=None), dict(tokens=-1), dict(dim=0), dict(dim=63, rot=62),
            dict(dim=258), dict(rot=0), dict(rot=63), dict(rot=66), dict(most=0), dict(type=2), dict(type=-1), dict(flags=2),
            dict(flags=4), dict(pos=0), dict(pos=P + 2), dict(table=P + 1), dict(ins=arr(rows(0), rows())),
            dict(outs=arr(rows(), rows(P + 2))), dict(outs=arr(rows(heads=3), rows())),
            dict(ins=arr(rows(reserved=1), rows())), dict(ins=arr(rows(heads=0), rows()), outs=arr(rows(heads=0), rows()))]
    for b in bad:
        assert call(**b) == BAD, b
    # a grid that would pass 2^31 workgroups
    assert call(tokens=2 ** 31 - 1, dim=256, ins=arr(rows(heads=4096), rows(heads=4096)), outs=arr(rows(heads=4096), rows(heads=4096))) == BAD


def test_append_norm_refuses():
    lib = _lib.load()
    cache = _lib.KV8(k=P, v=P, k_scale=P, v_scale=P, pages=8, kv_heads=2, head_dim=64, page_tokens=16)

    def call(c=cache, k=rows(heads=2), v=rows(heads=2), slots=P, q=None, q_out=None, n=norm(), pos=P, table=P, tokens=3,
             rot=64, most=100, type=0, flags=0):
        r = lambda x: None if x is None else ref(x)  # noqa: E731
        return lib.zt_kv8_append_norm(r(c), r(k), r(v), slots, r(q), r(q_out), r(n), pos, table, tokens, rot, most, type, flags, None)

    assert call(tokens=0) == 0 and call(tokens=0, q=rows(), q_out=rows(), table=0) == 0
    for b in [dict(n=norm(**x)) for x in BAD_NORMS] + [
            dict(n=None), dict(c=None), dict(k=None), dict(v=None), dict(slots=0), dict(q=rows()), dict(q_out=rows()),
            dict(q=rows(), q_out=rows(heads=3)), dict(pos=0), dict(tokens=-1), dict(rot=3), dict(rot=66), dict(most=0), dict(type=5),
            dict(flags=2), dict(k=rows(heads=3)), dict(k=rows(0, 2)), dict(v=rows(P + 2, 2)), dict(tokens=1 << 30)]:
        assert call(**b) == BAD, b
