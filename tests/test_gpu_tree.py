"""Drafted trees on the GPU: their tables, attention over the cache under their
masks, and the accepted paths, against the definitions (draft_ref).  Tables and
paths equal; attention within decode_ref.attend_bound."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import decode_ref as ref  # noqa: E402
import draft_ref  # noqa: E402
from ztensor_amd.engine import ROCmEngine  # noqa: E402

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16}


@pytest.fixture(scope="module")
def eng():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return ROCmEngine()


def i32(x):
    return torch.tensor(np.asarray(x, dtype=np.int32).tolist(), dtype=torch.int32, device="cuda").reshape(np.shape(x))


def i64(x):
    return torch.tensor([int(v) for v in x], dtype=torch.int64, device="cuda")


def starts_of(counts, before=0):
    return [before, *(before + np.cumsum(counts)).tolist()]


def some_parents(rng, counts):
    out = []
    for n in counts:
        out += [-1] * (n > 0) + [int(rng.integers(max(0, i - 5), i)) for i in range(1, n)]
    return out


# ------------------------------------------------------------------- tables


@pytest.mark.parametrize("counts,words,before,after", [((1,), 1, 0, 0), ((5, 0, 64, 1), 1, 0, 3), ((65, 128, 7), 2, 2, 0),
                                                       ((300, 20), 3, 0, 1), ((1030, 2), 16, 0, 0), ((1300,), 16, 1, 1)])
def test_tree(eng, counts, words, before, after):
    rng = np.random.default_rng(sum(counts))
    starts = starts_of(counts, before)
    tokens = starts[-1] + after
    parents = np.array([-1] * before + some_parents(rng, counts) + [0] * after)
    parents[rng.integers(0, tokens, 3)] = [-7, tokens + 5, 2 ** 31 - 1]  # not earlier rows: none
    lens = [int(rng.integers(0, 50)) + (n if i % 3 != 1 else 0) for i, n in enumerate(counts)]
    want, mask = draft_ref.tree(parents, lens, starts, tokens, words)
    got = eng.kv8_tree(i32(parents), i32(lens), i32(starts), 64 * words)
    assert got.mask.shape == (tokens, words)
    assert got.positions.cpu().tolist() == want.tolist() and np.array_equal(got.mask.cpu().numpy(), mask)


def test_tree_of_a_chain_and_of_nothing(eng):
    n = 1024
    got = eng.kv8_tree(i32(range(-1, n - 1)), i32([n + 9]), i32([0, n]), n)
    assert got.positions.cpu().tolist() == list(range(9, 9 + n))
    assert all(bin(int(x) & (2 ** 64 - 1)).count("1") == min(64, max(0, i + 1 - 64 * w)) for w in (0, 15)
               for i, x in enumerate(got.mask[:, w].cpu().tolist()))
    none = eng.kv8_tree(i32([]), i32([4]), i32([0, 0]), 1)
    assert none.positions.numel() == 0 and none.mask.shape == (0, 1)
    alone = eng.kv8_tree(i32([0, 0]), i32([]), i32([0]), 1)
    assert alone.positions.tolist() == [0, 0] and alone.mask.tolist() == [[0], [0]]


# ---------------------------------------------------------------- attention


def paged(rng, lens, page, extra=3):
    need = [-(-max(1, n) // page) for n in lens]
    order = rng.permutation(sum(need) + extra)
    table, at = np.full((len(lens), max(need) + 1), -1), 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    return table, sum(need) + extra


def check(eng, rng, counts, contexts, heads, kv, dim, page, dtype, window=0, words=None, mask=None, before=0, after=0, scale=None,
          break_pages=False, **bounds):
    lens = [c + n for c, n in zip(contexts, counts)]
    starts = starts_of(counts, before)
    tokens = starts[-1] + after
    table, pages = paged(rng, lens, page)
    cache = ref.Cache(pages, kv, dim, page, rng)
    if break_pages:
        table[0, 0], table[-1, 0] = -1, pages + 4
    words = words or max(1, -(-max(counts) // 64))
    if mask is None:
        mask = draft_ref.tree(np.array([-1] * before + some_parents(rng, counts) + [0] * after), lens, starts, tokens, words)[1]
    q = torch.from_numpy((1.5 * rng.standard_normal((tokens, heads, dim))).astype(np.float32)).cuda().to(DT[dtype])
    got = eng.kv8_tree_attention(q, cache.device(torch), i32(table), i32(lens), i32(starts), torch.from_numpy(mask).cuda(), window=window,
                                 scale=None if scale is None else torch.tensor([scale], device="cuda"), **bounds).double().cpu().numpy()
    want, most, big = draft_ref.attend(q.double().cpu().numpy(), cache, table, lens, starts, mask, window, scale)
    assert (np.abs(got - want) <= ref.attend_bound(want, most, big, dtype == "f16")).all(), np.abs(got - want).max()
    return got


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 4])
@pytest.mark.parametrize("counts,contexts", [((12, 5), (-2, 6)), ((40,), (-9,)), ((90, 7), (-70, -3))])
def test_the_largest_window(eng, counts, contexts, window):
    """Requests that hold fewer tokens than they have rows: no first token, before or behind an int's end."""
    for dtype in DT:
        assert np.abs(check(eng, np.random.default_rng(3), counts, contexts, 2, 1, 64, 16, dtype, window=window)).max() > 0


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("counts,contexts,heads,kv,dim,page", [
    ((1,), (0,), 4, 2, 64, 16), ((1,), (37,), 8, 2, 128, 16), ((8,), (60,), 8, 2, 128, 32), ((7, 1, 13), (5, 200, 0), 4, 1, 64, 64),
    ((16,), (48,), 4, 1, 128, 16), ((33, 5), (70, 129), 2, 2, 80, 32), ((64,), (100,), 2, 1, 128, 128), ((64, 3, 40), (0, 65, 190), 8, 1, 64, 16),
    ((100,), (77,), 2, 2, 128, 64), ((130, 2), (31, 300), 7, 1, 96, 16), ((20, 64), (250, 3), 4, 2, 256, 64), ((9,), (15,), 3, 3, 192, 16)])
def test_attention(eng, dtype, counts, contexts, heads, kv, dim, page):
    rng = np.random.default_rng(sum(counts) + dim)
    check(eng, rng, counts, contexts, heads, kv, dim, page, dtype, before=sum(counts) % 3, after=2)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("window", [1, 2, 7, 64, 100])
@pytest.mark.parametrize("counts,contexts,heads", [((9, 2), (150, 3), 2), ((70, 12), (90, 200), 4)])
def test_windows(eng, dtype, window, counts, contexts, heads):
    check(eng, np.random.default_rng(window), counts, contexts, heads, 1, 64, 16, dtype, window=window)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("n,heads,words", [(5, 2, 1), (64, 2, 1), (90, 2, 2), (200, 1, 2), (150, 4, 4)])
def test_any_masks(eng, dtype, n, heads, words):
    """Rows that see later ones, or none; bits of rows that are not there; rows past the words."""
    rng = np.random.default_rng(n)
    mask = rng.integers(-2 ** 63, 2 ** 63, (n + 3, words), dtype=np.int64)
    mask[::3] &= rng.integers(-2 ** 63, 2 ** 63, (len(mask[::3]), words), dtype=np.int64)
    mask[1] = 0
    for context in (0, 21):
        got = check(eng, rng, (n, 3), (context, 0), heads, 1, 64, 16, dtype, words=words, mask=mask)
        assert context or (got[1] == 0).all()
    check(eng, rng, (n, 3), (40, 5), heads, 1, 64, 16, dtype, words=words, mask=mask, window=30)


@pytest.mark.parametrize("heads", [2, 40])
def test_rows_that_see_nothing(eng, heads):
    """No context and no bits; a context on no page; lengths below the rows; none at all."""
    rng = np.random.default_rng(1)
    mask = np.zeros((6, 1), np.int64)
    got = check(eng, rng, (3, 3), (0, 0), heads, 1, 64, 16, "f32", mask=mask)
    assert (got == 0).all()
    check(eng, rng, (4, 2), (40, 33), heads, 2, 64, 16, "f16", break_pages=True)
    for lens in ((2, 5), (0, 0), (-4, 1)):
        table, pages = paged(rng, (40, 40), 16)
        cache = ref.Cache(pages, 1, 64, 16, rng)
        q = torch.randn(6, heads, 64, device="cuda")
        mask = np.full((6, 1), -1, np.int64)
        got = eng.kv8_tree_attention(q, cache.device(torch), i32(table), i32(lens), i32([0, 4, 6]), torch.from_numpy(mask).cuda())
        want, most, big = draft_ref.attend(q.double().cpu().numpy(), cache, table, [max(0, x) for x in lens], [0, 4, 6], mask)
        assert (np.abs(got.double().cpu().numpy() - want) <= ref.attend_bound(want, most, big, False)).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_what_is_masked_may_be_anything(eng, dtype):
    """Pages of values that are not numbers change nothing for rows that do not see them."""
    rng = np.random.default_rng(5)
    table = np.array([[2, 0, 1, 4]])
    cache = ref.Cache(5, 2, 64, 16, rng)
    q = torch.randn(17, 4, 64, device="cuda").to(DT[dtype])
    mask = np.zeros((17, 1), np.int64)
    mask[:, 0] = 1  # all see row 0 only, which ends page 0 of the table's second; the others lie on the third
    args = i32(table), i32([48]), i32([0, 17])
    want = eng.kv8_tree_attention(q, cache.device(torch), *args, torch.from_numpy(mask).cuda())
    for bad in (np.nan, np.inf):
        cache.scales[:, 1] = bad
        got = eng.kv8_tree_attention(q, cache.device(torch), *args, torch.from_numpy(mask).cuda())
        assert torch.equal(got, want) and torch.isfinite(got).all()
    exact, most, big = draft_ref.attend(q.double().cpu().numpy(), ref_without(cache), table, [48], [0, 17], mask)
    assert (np.abs(got.double().cpu().numpy() - exact) <= ref.attend_bound(exact, most, big, dtype == "f16")).all()


def ref_without(cache):
    cache.scales[:, 1] = 1.0
    return cache


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("counts,heads", [((1, 6, 3), 4), ((40, 70), 2), ((90, 5), 4)])
@pytest.mark.parametrize("window", [0, 50])
def test_a_chain_is_the_causal_call(eng, dtype, counts, heads, window):
    """Masks of rows in a line: kv8_attention's rows, within what both may be off (its window is over all tokens)."""
    rng = np.random.default_rng(2)
    lens = [n + 130 for n in counts]
    table, pages = paged(rng, lens, 16)
    cache = ref.Cache(pages, 2, 128, 16, rng)
    starts = starts_of(counts)
    q = torch.randn(starts[-1], 2 * heads, 128, device="cuda").to(DT[dtype])
    mask = np.zeros((starts[-1], 2), np.int64)
    for lo, n in zip(starts, counts):
        for i in range(n):
            row = [j for j in range(i + 1) if not window or j > i - window]
            for j in row:
                mask[lo + i, j // 64] |= np.int64(np.uint64(1) << np.uint64(j % 64)) if j % 64 < 63 else np.int64(-2 ** 63)
    on = cache.device(torch)
    a = eng.kv8_attention(q, on, i32(table), i32(lens), i32(starts), window=window).double().cpu().numpy()
    if window and max(counts) > window:
        return  # positions by the mask's rows are then not those of a line
    b = eng.kv8_tree_attention(q, on, i32(table), i32(lens), i32(starts), torch.from_numpy(mask).cuda(), window=window).double().cpu().numpy()
    want, most, big = draft_ref.attend(q.double().cpu().numpy(), cache, table, lens, starts, mask, window)
    assert (np.abs(a - b) <= 2 * ref.attend_bound(want, most, big, dtype == "f16")).all()


def test_strides_scale_bounds_and_out(eng):
    rng = np.random.default_rng(9)
    check(eng, rng, (12, 3), (90, 20), 4, 2, 64, 16, "f32", scale=-0.3)
    check(eng, rng, (12, 70), (500, 20), 4, 2, 64, 16, "f16", scale=0.0)
    for bounds in (dict(max_q=1, max_kv=1), dict(max_q=12, max_kv=200), dict(max_q=4000, max_kv=100000)):
        check(eng, rng, (12, 5), (170, 20), 4, 2, 64, 16, "f32", **bounds)
    lens, starts = [41], [0, 9]
    table, pages = paged(rng, lens, 16)
    cache = ref.Cache(pages, 2, 64, 16, rng)
    mask = torch.full((9, 1), 511, device="cuda")
    wide = torch.randn(9, 3, 4 * 64 + 6, device="cuda")
    q = wide[:, 1, 3:3 + 256].unflatten(1, (4, 64))
    out = torch.full((4, 9, 64), 7.0, device="cuda")
    args = cache.device(torch), i32(table), i32(lens), i32(starts), mask
    got = eng.kv8_tree_attention(q, *args, out=out.transpose(0, 1))
    same = eng.kv8_tree_attention(q.contiguous(), *args)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, same)
    with pytest.raises(ValueError):
        eng.kv8_tree_attention(q, *args[:-1], mask[:8])
    with pytest.raises(ValueError):
        eng.kv8_tree_attention(q, *args[:-1], mask.int())
    from ztensor_amd._lib import ZTError

    with pytest.raises(ZTError):
        eng.kv8_tree_attention(q, *args[:-1], torch.zeros(9, 17, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("heads,most,longest", [(2, 40, 800), (8, 40, 800), (8, 1, 64), (8, 40, 100)])
def test_starts_out_of_order(eng, heads, most, longest):
    """No meaning, but nothing outside the buffers is read or written: finite values, and the guard rows untouched."""
    rng = np.random.default_rng(most)
    lens = [100, 800, 40, 300]
    table, pages = paged(rng, lens, 16)
    cache = ref.Cache(pages, 2, 128, 16, rng).device(torch)
    q = torch.from_numpy(rng.standard_normal((60, heads, 128)).astype(np.float32)).cuda()
    mask = torch.from_numpy(rng.integers(-2 ** 63, 2 ** 63 - 1, (60, 1)))
    tokens = torch.from_numpy(rng.integers(0, 3, (2, 60))).cuda()
    parents = i32(rng.integers(-1, 20, 60))
    whole = torch.full((64, heads, 128), 7.0, device="cuda")
    for starts in ([-9, 5, 2, 9, 60], [2 ** 31 - 1, -2 ** 31, 30, -2, 2 ** 31 - 1], [50, 40, 30, 20, 10], [-2 ** 31] * 5):
        print(starts, flush=True)
        out = eng.kv8_tree_attention(q, cache, i32(table), i32(lens), i32(starts), mask.cuda(), max_q=most, max_kv=longest, out=whole[2:62])
        assert torch.isfinite(out).all() and (whole[:2] == 7).all() and (whole[62:] == 7).all()
        eng.kv8_tree(parents, i32(lens), i32(starts), 60)
        took = eng.tree_accept(tokens[0], tokens[1], i32(starts), parents=parents)
        eng.kv8_compact([cache], i32(table), i32([2 ** 31 - 1, 700, 0, 5]), i32(starts), took.path, took.kept)
        torch.cuda.synchronize()


def test_attention_again_and_captured(eng):
    """The same bits every call, and in replays whose lengths, masks and starts change."""
    rng = np.random.default_rng(11)
    s = torch.cuda.Stream()
    e = ROCmEngine(stream=s)
    with torch.cuda.stream(s):
        lens = [400, 75, 20]
        table, pages = paged(rng, [500, 100, 100], 16)
        cache = ref.Cache(pages, 2, 128, 16, rng).device(torch)
        q = torch.randn(40, 8, 128, device="cuda")
        kv_lens, starts, parents = i32(lens), i32([0, 20, 21, 33]), i32(some_parents(rng, [20, 1, 12]) + [0] * 7)
        blocks = i32(table)

        def step():
            t = e.kv8_tree(parents, kv_lens, starts, 40)
            return e.kv8_tree_attention(q, cache, blocks, kv_lens, starts, t.mask, max_q=40, max_kv=500)

        first = step().clone()
        assert torch.equal(step(), first)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = step()
        for a, b, c in (([400, 75, 20], [0, 20, 21, 33], 1), ([333, 99, 64], [0, 40, 40, 40], 2), ([30, 31, 32], [5, 17, 30, 39], 3)):
            kv_lens.copy_(i32(a))
            starts.copy_(i32(b))
            q.normal_()
            g.replay()
            got = out.clone()
            assert torch.equal(got, step())
            torch.cuda.synchronize()


# ------------------------------------------------------------------- accept


@pytest.mark.parametrize("counts,before,after", [((1,), 0, 0), ((7, 0, 64, 2), 2, 3), ((65, 3), 0, 0), ((500, 1, 129), 0, 1)])
@pytest.mark.parametrize("chain", [False, True])
def test_accept(eng, counts, before, after, chain):
    rng = np.random.default_rng(sum(counts))
    starts = starts_of(counts, before)
    tokens = starts[-1] + after
    for vocab in (2, 3, 50):
        parents = np.array([-1] * before + some_parents(rng, counts) + [0] * after)
        drafted, drawn = rng.integers(0, vocab, (2, tokens))
        if chain or vocab == 3:
            drafted[:] = 1
            drawn = rng.choice([1] * 30 + [0, -1], tokens)
        slots = rng.integers(-1, 40, tokens)
        for use in (None, slots):
            want = draft_ref.accept(drafted, drawn, None if chain else parents, starts, use)
            got = eng.tree_accept(i64(drafted), i64(drawn), i32(starts), parents=None if chain else i32(parents),
                                  slots=None if use is None else i64(use))
            assert [x.cpu().tolist() for x in got] == [list(map(int, x)) for x in want]


def test_accept_of_tokens_that_are_nobodys(eng):
    got = eng.tree_accept(i64([-1, -1, -1]), i64([-1, -1, -1]), i32([0, 3]))
    assert [x.tolist() for x in got] == [[0, -1, -1], [1], [0], [-1]]
    got = eng.tree_accept(i64([2 ** 40, 2 ** 40 + 1, 1]), i64([2 ** 40 + 1, 1, 5]), i32([0, 3]))
    assert [x.tolist() for x in got] == [[0, 1, 2], [3], [2], [5]]
    none = eng.tree_accept(i64([]), i64([]), i32([0, 0]))
    assert [x.tolist() for x in none] == [[], [0], [-1], [-1]]


def test_accept_refuses(eng):
    one = i64([1, 2, 3])
    with pytest.raises(ValueError, match="q_start"):
        eng.tree_accept(one, one, i32([]))
    with pytest.raises(ValueError, match="drawn"):
        eng.tree_accept(one, one[:2].contiguous(), i32([0, 3]))
    with pytest.raises(ValueError, match="parents"):
        eng.tree_accept(one, one, i32([0, 3]), parents=one)
    none = eng.tree_accept(one[:0], one[:0], i32([0]))
    assert [x.numel() for x in none] == [0, 0, 0, 0]
