"""Attention of drafted trees where the calls are large: more requests than a
workgroup looks up at a time, one sequence dealt out to many workgroups (whose
parts eight waves join), rows of more than eight parts, more tiles than the card's
workgroups, and every head size the tiled kernel has.  Against the definition in
64 bits, within decode_ref.attend_bound and, of long contexts, what adding up
their tiles may add: each tile's sum is rounded into a row's, numerator and
denominator, 2^-24 of it each time."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import decode_ref as ref  # noqa: E402
import draft_ref  # noqa: E402
from test_gpu_tree import DT, eng, i32, paged, some_parents, starts_of  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def attend(q, cache, table, lens, starts, mask, window=0):
    """draft_ref.attend's values, the rows of a request at a time."""
    out, most, big = np.zeros(q.shape), 0.0, 0.0
    kv, scale, group = cache.values(), 1.0 / np.sqrt(q.shape[2]), q.shape[1] // cache.codes.shape[2]
    for r, size in enumerate(lens):
        n = starts[r + 1] - starts[r]
        if n == 0:
            continue
        context, t = size - n, np.arange(size)
        own = draft_ref.bits(mask[starts[r]:starts[r] + n], n)
        seen = np.concatenate([np.ones((n, context), bool), own], 1)
        if window:
            seen[:, :context] = t[None, :context] >= (context + own.sum(1) - window)[:, None]
        pages, places = table[r, t // cache.page], t % cache.page
        for h in range(q.shape[1]):
            keys, values = (kv[i][pages, h // group, places] for i in range(2))
            rows = q[starts[r]:starts[r] + n, h]
            s = np.where(seen, rows @ keys.T * scale, -np.inf)
            most = max(most, (np.abs(rows) @ np.abs(keys).T * scale)[seen].max())
            p = np.exp(s - s.max(1, keepdims=True))
            out[starts[r]:starts[r] + n, h] = p @ values / p.sum(1, keepdims=True)
            big = max(big, np.abs(values).max())
    return out, most, big


def check(eng, rng, counts, contexts, heads, kv, dim, page, dtype, window=0, **bounds):  # noqa: F811
    lens = [c + n for c, n in zip(contexts, counts)]
    starts = starts_of(counts, 1)
    tokens = starts[-1] + 2
    table, pages = paged(rng, lens, page)
    cache = ref.Cache(pages, kv, dim, page, rng)
    words = max(1, -(-max(counts) // 64))
    mask = draft_ref.tree(np.array([-1] + some_parents(rng, counts) + [0, 0]), lens, starts, tokens, words)[1]
    q = torch.from_numpy((1.5 * rng.standard_normal((tokens, heads, dim))).astype(np.float32)).cuda().to(DT[dtype])
    args = q, cache.device(torch), i32(table), i32(lens), i32(starts), torch.from_numpy(mask).cuda()
    got = eng.kv8_tree_attention(*args, window=window, max_q=max(counts), **bounds)
    assert torch.equal(got, eng.kv8_tree_attention(*args, window=window, max_q=max(counts), **bounds))
    got = got.double().cpu().numpy()
    assert (got[0] == 0).all() and (got[-2:] == 0).all()  # of no request
    want, most, big = attend(q.double().cpu().numpy(), cache, table, lens, starts, mask, window)
    tiles = -(-max(lens) // 64)
    bound = ref.attend_bound(want, most, big, dtype == "f16") + 2 * tiles * 2.0 ** -24 * big
    assert (np.abs(got - want) <= bound).all(), np.abs(got - want).max()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("requests", [70, 130])
@pytest.mark.parametrize("context", [150, 700])
def test_many_requests(eng, dtype, requests, context):  # noqa: F811
    """Empty ones, rows of up to 16 a kv head and of more; whole groups of rows (short contexts) and equal shares."""
    rng = np.random.default_rng(requests + context)
    counts = rng.choice([0, 1, 3, 8, 9, 21, 40], requests).tolist()
    counts[0], counts[64], counts[-1] = 40, 0, 13
    check(eng, rng, counts, rng.integers(0, context, requests).tolist(), 4, 2, 64, 16, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_many_requests_of_few_rows(eng, dtype):  # noqa: F811
    rng = np.random.default_rng(7)
    check(eng, rng, rng.integers(0, 5, 150).tolist(), rng.integers(0, 600, 150).tolist(), 6, 2, 64, 16, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("kv,dim,context,n", [(1, 64, 6000, 20), (1, 128, 9001, 20), (2, 64, 8999, 8), (1, 192, 7000, 33), (2, 256, 6100, 20),
                                              (1, 64, 7777, 100), (2, 128, 5000, 8)])
def test_one_long_sequence(eng, dtype, kv, dim, context, n):  # noqa: F811
    check(eng, np.random.default_rng(context), [n], [context], 2 * kv, kv, dim, 64, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("dim,counts,contexts", [(64, (30,), (3900,)), (128, (30, 4), (2700, 100)), (192, (40, 20), (3300, 3000)),
                                                 (256, (17, 64), (2900, 2000))])
def test_rows_of_many_parts(eng, dtype, dim, counts, contexts):  # noqa: F811
    """Nine to sixteen workgroups a row."""
    check(eng, np.random.default_rng(dim), counts, contexts, 4, 2, dim, 32, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("requests,kv,dim,context", [(24, 2, 64, 3500), (30, 3, 128, 1800), (10, 4, 136, 2000), (40, 1, 192, 2500), (9, 4, 256, 2500)])
def test_more_tiles_than_workgroups(eng, dtype, requests, kv, dim, context):  # noqa: F811
    """All that the card holds at a time; a workgroup's share spans segments."""
    rng = np.random.default_rng(requests)
    counts = rng.integers(9, 50, requests).tolist()
    counts[1] = 2
    check(eng, rng, counts, (context * rng.random(requests) ** 2).astype(int).tolist(), 2 * kv, kv, dim, 64, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("dim", [136, 160, 184, 192, 200, 256])
@pytest.mark.parametrize("counts,contexts,window", [((70, 5), (40, 130), 0), ((33, 64), (500, 900), 0), ((70, 20), (600, 100), 130)])
def test_head_sizes(eng, dtype, dim, counts, contexts, window):  # noqa: F811
    check(eng, np.random.default_rng(dim), counts, contexts, 4, 2, dim, 16, dtype, window=window)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("window", [300, 2000])
def test_windows(eng, dtype, window):  # noqa: F811
    rng = np.random.default_rng(window)
    check(eng, rng, (30, 64, 3, 0, 20), (5000, 900, 3000, 10, 40), 8, 2, 128, 64, dtype, window=window)
