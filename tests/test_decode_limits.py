"""Sizes so near 2^31 that the kernels' 32-bit sums would pass it are refused
(nothing is launched: the pointers are not real)."""
import ctypes

from ztensor_amd import _lib

P, BAD = 1 << 20, _lib.HIP_ERROR_INVALID_VALUE


def test_plan_of_a_row_that_fills_31_bits():
    pointers = iter(range(1 << 40, 1 << 50, 1 << 36))
    p = lambda: next(pointers)  # noqa: E731
    for requests, width in ((1, 2 ** 31 - 1), (1, 2 ** 31 - 256), (2, 2 ** 30 - 1)):
        args = (p(), p(), p(), requests, width, p(), p(), 16, 16, 9, p(), p(), p(), p(), p(), p())
        assert _lib.load().zt_kv8_plan(*args, None) == BAD


def test_append_of_2_30_tokens():
    cache = _lib.KV8(P, P, P, P, 8, 1, 64, 16)
    rows = ctypes.byref(_lib.Rows(P, 64, 64, 1, 0))
    for tokens in (1 << 30, 2 ** 31 - 1):
        assert _lib.load().zt_kv8_append(ctypes.byref(cache), rows, rows, P, None, None, 0, 0, tokens, 0, 0, 0, 0, None) == BAD


def test_attention_of_rows_that_fill_31_bits():
    for tokens, heads in ((2 ** 31 - 1, 1), (2 ** 31 - 256, 1), (2 ** 27, 16)):
        rows = _lib.Rows(P, 64 * heads, 64, heads, 0)
        a = _lib.KV8Attn(cache=_lib.KV8(P, P, P, P, 8, 1, 64, 16), q=rows, out=rows, table=P, kv_lens=P, q_start=P, requests=1,
                         width=4, tokens=tokens, max_q=1, max_kv=64)
        assert _lib.load().zt_kv8_attention_workspace_bytes(ctypes.byref(a)) == -1
