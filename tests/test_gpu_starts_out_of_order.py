"""Starts that are in no order have no meaning, but stay inside the buffers: rows
outside the starts' bounds, pages of no row and guard rows are as they were, and
lengths and paths are those of the rows that a request can have."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import decode_ref as ref  # noqa: E402
from test_gpu_tree import eng, i32, paged  # noqa: E402, F401

pytestmark = pytest.mark.gpu

TOKENS = 60
STARTS = [[-9, 5, 2, 9, 60], [2 ** 31 - 1, -2 ** 31, 30, -2, 2 ** 31 - 1], [50, 40, 30, 20, 10], [-2 ** 31] * 5, [0, 70, 3, 66, 60],
          [0, 60, 0, 60, 0], [10, 20, 15, 15, 40]]


def span(starts, r):
    """A request's rows: its first, and how many."""
    lo = min(max(0, starts[r]), TOKENS)
    return lo, max(0, min(max(0, starts[r + 1]), TOKENS) - lo)


def guarded(n, dtype, width=1):
    whole = torch.full((n + 8, width), 77, dtype=dtype, device="cuda")
    return whole, whole[4:n + 4]


def intact(whole):
    return bool((whole[:4] == 77).all() and (whole[-4:] == 77).all())


@pytest.mark.parametrize("starts", STARTS, ids=str)
def test_tree_and_accept(eng, starts):  # noqa: F811
    rng = np.random.default_rng(1)
    requests, lib, s = len(starts) - 1, eng.lib, torch.cuda.current_stream().cuda_stream
    parents, lens = i32(rng.integers(-1, 20, TOKENS)), i32([100, 800, 40, 300])
    drafted, drawn = (torch.from_numpy(rng.integers(0, 3, TOKENS)).cuda() for _ in range(2))
    positions, mask, path, kept, last, token = (guarded(n, d, w) for n, d, w in (
        (TOKENS, torch.int32, 1), (TOKENS, torch.int64, 2), (TOKENS, torch.int32, 1), (requests, torch.int32, 1), (requests, torch.int32, 1),
        (requests, torch.int64, 1)))
    at = i32(starts)
    for window in (0, 3):
        lib.call("zt_kv8_tree_window", parents.data_ptr(), lens.data_ptr(), at.data_ptr(), requests, TOKENS, 2, window,
                 positions[1].data_ptr(), mask[1].data_ptr(), s)
    lib.call("zt_tree_accept", drafted.data_ptr(), drawn.data_ptr(), parents.data_ptr(), at.data_ptr(), 0, requests, TOKENS,
             path[1].data_ptr(), kept[1].data_ptr(), last[1].data_ptr(), token[1].data_ptr(), s)
    torch.cuda.synchronize()
    assert all(intact(x[0]) for x in (positions, mask, path, kept, last, token))
    for r in range(requests):
        lo, n = span(starts, r)
        k, z = kept[1][r].item(), last[1][r].item()
        assert (k == 0) == (n == 0) and 0 <= k <= n and (z == -1 if n == 0 else lo <= z < lo + n)
    for row, p in enumerate(path[1].flatten().tolist()):
        owners = [span(starts, r) for r in range(requests) if span(starts, r)[0] <= row < sum(span(starts, r))]
        assert p == 77 if not owners and p == 77 else -1 <= p < max([n for _, n in owners], default=0)


@pytest.mark.parametrize("starts", STARTS, ids=str)
def test_compact(eng, starts):  # noqa: F811
    rng = np.random.default_rng(2)
    lens, held = [100, 800, 40, 300], [90, 700, 0, 290]
    table, pages = paged(rng, lens, 16)
    cache = ref.Cache(pages, 2, 64, 16, rng)
    on = cache.device(torch)
    before = [x.clone() for x in on]
    path, kept = rng.integers(-2, 40, TOKENS), [9, -1, 2 ** 31 - 1, 7]
    got = eng.kv8_compact([on], i32(table), i32(held), i32(starts), i32(path), i32(kept))
    want = [h + min(max(0, k), span(starts, r)[1]) for r, (h, k) in enumerate(zip(held, kept))]
    assert got.tolist() == want
    mine = set()  # pages that a request's kept rows may go to
    for r in range(4):
        mine |= {int(table[r, p // 16]) for p in range(held[r], min(want[r], 16 * table.shape[1]))}
    others = torch.tensor([p for p in range(pages) if p not in mine], device="cuda")
    for x, y in zip(on, before):
        assert torch.equal(x[others], y[others])


@pytest.mark.parametrize("most,longest", [(40, 800), (1, 64), (40, 100)])
@pytest.mark.parametrize("starts", STARTS, ids=str)
def test_attention(eng, starts, most, longest):  # noqa: F811
    rng = np.random.default_rng(3)
    lens = [100, 800, 40, 300]
    table, pages = paged(rng, lens, 16)
    cache = ref.Cache(pages, 2, 128, 16, rng).device(torch)
    before = [x.clone() for x in cache]
    q = torch.from_numpy(rng.standard_normal((TOKENS, 4, 128)).astype(np.float32)).cuda()
    mask = torch.from_numpy(rng.integers(-2 ** 63, 2 ** 63 - 1, (TOKENS, 1))).cuda()
    whole = torch.full((TOKENS + 4, 4, 128), 7.0, device="cuda")
    out = eng.kv8_tree_attention(q, cache, i32(table), i32(lens), i32(starts), mask, max_q=most, max_kv=longest, out=whole[2:-2])
    torch.cuda.synchronize()
    assert out.shape == q.shape and (whole[:2] == 7).all() and (whole[-2:] == 7).all()
    assert all(torch.equal(x, y) for x, y in zip(cache, before))
