"""Drafted trees under a sliding window: a row sees the last `window` tokens of
its context and the rows above it, itself among them, as it would if they were all
that there is (kv8_attention of its path)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import decode_ref as ref  # noqa: E402
import draft_ref  # noqa: E402
from test_gpu_tree import DT, eng, i32, paged, some_parents, starts_of  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def attend(q, cache, table, lens, starts, parents, window):
    """(out, most, big) as decode_ref.attend's, row after row: the last `window` of its context's tokens and its path's rows."""
    out, most, big = np.zeros(q.shape), 0.0, 0.0
    kv, scale, group = cache.values(), 1.0 / np.sqrt(q.shape[2]), q.shape[1] // cache.codes.shape[2]
    for r, size in enumerate(lens):
        n = starts[r + 1] - starts[r]
        for i, chain in enumerate(draft_ref.ancestors(parents[starts[r]:starts[r + 1]], n)):
            seen = (list(range(size - n)) + [size - n + j for j in sorted(chain)])[-window:]
            pages, places = [table[r, t // cache.page] for t in seen], [t % cache.page for t in seen]
            keys, values = kv[0][pages, :, places], kv[1][pages, :, places]
            row = q[starts[r] + i]
            for h in range(q.shape[1]):
                s = keys[:, h // group] @ row[h] * scale
                most = max(most, (np.abs(keys[:, h // group]) @ np.abs(row[h]) * scale).max())
                p = np.exp(s - s.max())
                out[starts[r] + i, h] = (p / p.sum()) @ values[:, h // group]
            big = max(big, np.abs(values).max())
    return out, most, big


@pytest.mark.parametrize("window", [1, 2, 7, 64, 70, 2 ** 31 - 1])
@pytest.mark.parametrize("counts,words", [((1,), 1), ((5, 0, 64, 1), 1), ((65, 128, 7), 2), ((300, 20), 3), ((1030, 2), 16)])
def test_masks(eng, window, counts, words):  # noqa: F811
    rng = np.random.default_rng(window % 1000 + sum(counts))
    starts = starts_of(counts)
    parents = np.array([int(rng.integers(max(-1, i - 3), i)) if i else -1 for n in counts for i in range(n)])
    lens = [n + 9 for n in counts]
    got = eng.kv8_tree(i32(parents), i32(lens), i32(starts), 64 * words, window=window)
    plain = eng.kv8_tree(i32(parents), i32(lens), i32(starts), 64 * words)
    assert torch.equal(got.positions, plain.positions)
    want = np.zeros((starts[-1], words), np.uint64)
    for lo, n in zip(starts, counts):
        for i, chain in enumerate(draft_ref.ancestors(parents[lo:lo + n], n)):
            for j in chain[:window]:  # (itself first)
                if j < 64 * words:
                    want[lo + i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    assert np.array_equal(got.mask.cpu().numpy(), want.view(np.int64))


def steps(eng, rng, counts, contexts, heads, kv, dim, page, dtype, window, parents):  # noqa: F811
    lens = [c + n for c, n in zip(contexts, counts)]
    starts = starts_of(counts)
    table, pages = paged(rng, lens, page)
    cache = ref.Cache(pages, kv, dim, page, rng)
    on = cache.device(torch)
    q = torch.from_numpy((1.5 * rng.standard_normal((starts[-1], heads, dim))).astype(np.float32)).cuda().to(DT[dtype])
    t = eng.kv8_tree(i32(parents), i32(lens), i32(starts), max(counts), window=window)
    got = eng.kv8_tree_attention(q, on, i32(table), i32(lens), i32(starts), t.mask, window=window, max_q=max(counts))
    qn = q.double().cpu().numpy()
    want, most, big = attend(qn, cache, table, lens, starts, np.array(parents), window)
    bound = ref.attend_bound(want, most, big, dtype == "f16")
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()
    line = eng.kv8_attention(q, on, i32(table), i32(lens), i32(starts), window=window)
    return got, line, bound


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("window", [1, 5, 8, 50, 100])
@pytest.mark.parametrize("counts,contexts,heads", [((1, 6, 3), (130, 2, 0), 8), ((40, 70), (130, 40), 4), ((90, 5, 20), (130, 130, 0), 8)])
def test_a_chain_is_the_causal_call(eng, dtype, window, counts, contexts, heads):  # noqa: F811
    """Chains shorter and longer than the window: kv8_attention's rows, within what both may be off."""
    parents = [i - 1 for n in counts for i in range(n)]
    a, b, bound = steps(eng, np.random.default_rng(window), counts, contexts, heads, 2, 128, 16, dtype, window, parents)
    assert ((a.double() - b.double()).abs().cpu().numpy() <= 2 * bound).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("window", [1, 3, 12, 60])
@pytest.mark.parametrize("counts,contexts,heads,dim", [((9, 2, 13), (150, 3, 0), 2, 64), ((70, 12), (90, 200), 4, 80), ((150,), (33,), 2, 128)])
def test_trees(eng, dtype, window, counts, contexts, heads, dim):  # noqa: F811
    rng = np.random.default_rng(window + dim)
    steps(eng, rng, counts, contexts, heads, 1, dim, 32, dtype, window, some_parents(rng, counts))


def test_refuses(eng):  # noqa: F811
    from ztensor_amd._lib import ZTError

    with pytest.raises(ZTError):
        eng.kv8_tree(i32([-1]), i32([1]), i32([0, 1]), 1, window=-1)
