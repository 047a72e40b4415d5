"""The workspace of a tree's attention: no more than its kernels have places for."""
import ctypes

import pytest

from ztensor_amd import _lib

P = 1 << 20


@pytest.mark.parametrize("dim,heads,kv,tokens,max_q,max_kv,requests,typ,rows,workgroups", [
    (128, 64, 8, 61, 61, 30011, 1, 1, 128, 512), (128, 32, 8, 400, 13, 6000, 32, 0, 64, 512), (256, 8, 1, 64, 64, 9000, 2, 0, 64, 256),
    (64, 8, 8, 40, 10, 500, 4, 0, 128, 0), (128, 8, 8, 34, 17, 9000, 2, 0, 64, 512)])
def test_tree_attention_places(dim, heads, kv, tokens, max_q, max_kv, requests, typ, rows, workgroups):
    """At most 1024 waves of 16 rows with two places each, and `workgroups` of so many rows; a place is a row's sums in fp32,
    their maximum and their weights; and 8 bytes for each token and head."""
    a = _lib.KV8Attn(cache=_lib.KV8(P, P, P, P, 8, kv, dim, 16), q=_lib.Rows(P, dim * heads, dim, heads, 0),
                     out=_lib.Rows(P, dim * heads, dim, heads, 0), table=P, kv_lens=P, q_start=P, requests=requests, width=4096,
                     tokens=tokens, max_q=max_q, max_kv=max_kv, type=typ)
    got = _lib.load().zt_kv8_tree_attention_workspace_bytes(ctypes.byref(a))
    places = 2 * 1024 * 16 + 2 * workgroups * rows
    assert 0 < got <= places * (4 * dim + 8) + 8 * tokens * heads + 32
