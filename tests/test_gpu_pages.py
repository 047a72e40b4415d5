"""Pages on the GPU: kept rows moved, pages copied, shared and given back, against
the definitions one value after another (draft_ref), to the bit; and a run of
steps over drafted trees that leaves what single tokens leave."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import decode_ref as ref  # noqa: E402
import draft_ref  # noqa: E402
from ztensor_amd.decode import KV8Cache, rope_table  # noqa: E402
from ztensor_amd.engine import ROCmEngine  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return ROCmEngine()


def i32(x):
    return torch.tensor(np.asarray(x, dtype=np.int32).tolist(), dtype=torch.int32, device="cuda").reshape(np.shape(x))


def paged(rng, lens, page, width=None, extra=3):
    need = [-(-n // page) for n in lens]
    order = rng.permutation(sum(need) + extra)
    table, at = np.full((len(lens), width or max(need) + 1), -1), 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    return table, sum(need) + extra, order[at:].tolist()


def some_path(rng, n, m):
    """m rows of n, rising, the first of them 0 mostly."""
    rest = np.sort(rng.choice(np.arange(1, n), m - 1, replace=False)) if m > 1 else []
    return ([0] if rng.random() < 0.8 or m > n - 1 else [int(rng.integers(0, min(n - m + 1, rest[0] if m > 1 else n)))]) + [int(x) for x in rest]


# ------------------------------------------------------------------ compact


@pytest.mark.parametrize("heads,dim,page,held,counts,layers", [
    (2, 64, 16, (5, 16, 0), (12, 30, 1), 1), (1, 128, 16, (30, 3), (64, 40), 2), (3, 80, 32, (31, 64, 7), (33, 20, 5), 1),
    (2, 256, 128, (120, 0), (20, 200), 1), (1, 72, 64, (60, 63), (5, 2), 3), (2, 128, 64, (1, 2, 3, 500), (70, 9, 0, 64), 1),
    (1, 64, 16, (7,), (9,), 40), (2, 192, 32, (3, 90), (100, 37), 1), (1, 136, 128, (200, 5), (150, 300), 2)])
def test_compact(eng, heads, dim, page, held, counts, layers):
    rng = np.random.default_rng(dim + page)
    lens = [h + n for h, n in zip(held, counts)]
    table, pages, _ = paged(rng, lens, page)
    starts = [0, *np.cumsum(counts).tolist()]
    for again in range(3):
        caches = [ref.Cache(pages, heads, dim, page, rng) for _ in range(layers)]
        if again == 1:  # pages of scale 0, and of very different ones
            caches[0].scales[:] *= rng.choice([0.0, 1e-3, 1.0, 40.0], caches[0].scales.shape).astype(np.float32)
        path, kept = np.full(starts[-1], -1), []
        for r, n in enumerate(counts):
            m = 0 if n == 0 else n if again == 2 and r == 0 else int(rng.integers(1, n + 1))
            rows = some_path(rng, n, m) if m else []
            path[starts[r]:starts[r] + m] = rows
            kept.append(m)
        on = [c.device(torch) for c in caches]
        got = eng.kv8_compact(on, i32(table), i32(held), i32(starts), i32(path), i32(kept))
        for c in caches:
            want = draft_ref.compact(c, table, held, starts, path, kept)
        assert got.tolist() == want
        for a, c in zip(on, caches):
            for x, y in zip(a, c.device(torch)):
                assert torch.equal(x, y)


def test_compact_of_what_is_not_a_path(eng):
    """Rows that do not rise, that come twice, that are not there; counts past the rows; pages outside the cache; rows past
    the table; a scale that is not a number goes on to the page that takes its codes."""
    rng = np.random.default_rng(4)
    held, counts = (10, 20, 30, 5), (20, 10, 8, 12)
    starts = [0, *np.cumsum(counts).tolist()]
    table, pages, _ = paged(rng, [h + n for h, n in zip(held, counts)], 16)
    table = table[:, :3]  # request 2's rows end past it
    table[1, 1] = -1
    cache = ref.Cache(pages, 2, 64, 16, rng)
    path = rng.integers(-3, 25, starts[-1])
    path[:6] = [3, 19, 9, 9, 2, 2 ** 31 - 1]
    kept = [99, 10, 8, -5]
    on = cache.device(torch)
    got = eng.kv8_compact([on], i32(table), i32(held), i32(starts), i32(path), i32(kept))
    assert got.tolist() == [30, 30, 38, 5]
    draft_ref.compact(cache, table, held, starts, path, kept)
    for x, y in zip(on, cache.device(torch)):
        assert torch.equal(x, y)
    cache = ref.Cache(4, 1, 64, 16, rng)
    cache.scales[1, 2] = np.nan
    on = cache.device(torch)
    got = eng.kv8_compact([on], i32([[0, 2, 1]]), i32([10]), i32([0, 20]), i32([0, 8] + [-1] * 18), i32([2]))
    assert got.tolist() == [12]
    assert torch.isnan(on[3][0, 0]) and torch.isfinite(on[2]).all() and torch.isfinite(on[3][1]).all()


def test_compact_refuses(eng):
    a, b = (KV8Cache.allocate(4, 2, 64, n) for n in (16, 32))
    z = i32([0])
    from ztensor_amd._lib import ZTError

    with pytest.raises(ZTError):
        eng.kv8_compact([a, b], i32([[0]]), z, i32([0, 1]), z, z)
    with pytest.raises(ZTError):
        eng.kv8_compact([], i32([[0]]), z, i32([0, 1]), z, z)
    for bad in ((z, i32([0, 1, 2]), z, z), (i32([0, 0]), i32([0, 1]), z, z), (z, i32([0, 1]), z.long(), z), (z, i32([0, 1]), z, z.cpu())):
        with pytest.raises(ValueError):
            eng.kv8_compact([a], i32([[0]]), *bad)


# --------------------------------------------------------------------- copy


@pytest.mark.parametrize("heads,dim,page,layers", [(2, 64, 16, 1), (8, 128, 64, 2), (3, 80, 32, 33), (1, 256, 128, 1)])
def test_copy(eng, heads, dim, page, layers):
    rng = np.random.default_rng(page)
    caches = [ref.Cache(9, heads, dim, page, rng) for _ in range(layers)]
    on = [c.device(torch) for c in caches]
    a, b = [3, -1, 3, 8, 2, 20], [0, 1, 7, 6, -1, 4]
    eng.kv8_copy(on, i32(a), i32(b))
    for c, parts in zip(caches, on):
        for x, y in ((3, 0), (3, 7), (8, 6)):
            c.codes[:, y], c.scales[:, y] = c.codes[:, x], c.scales[:, x]
        for x, y in zip(parts, c.device(torch)):
            assert torch.equal(x, y)
    eng.kv8_copy(on, i32([]), i32([]))


# --------------------------------------------------------------------- trim


@pytest.mark.parametrize("requests,width,page,pages", [(1, 3, 16, 8), (5, 9, 32, 60), (1500, 4, 64, 7000), (40, 300, 128, 20000),
                                                       (3, 5, 16, 500000), (2, 3, 16, 1 << 20)])
@pytest.mark.parametrize("shared", [False, True])
def test_trim(eng, requests, width, page, pages, shared):
    rng = np.random.default_rng(requests + pages)
    held = rng.integers(0, (width + 1) * page, requests)
    keep = np.minimum(held, rng.integers(-page, width * page, requests))
    table = np.full((requests, width), -1)
    if shared:  # few pages in many rows, each held as often as it stands there
        table[:] = rng.integers(0, max(2, requests * width // 3), (requests, width)) % pages
        for r, n in enumerate(held):
            table[r, -(-int(n) // page):] = -1
        count = np.bincount(table[table >= 0], minlength=pages)
        refs = np.maximum(count - 1, 0)
    else:
        order = rng.permutation(pages)[:requests * width] if requests * width <= pages else None
        assert order is not None
        table.reshape(-1)[:] = order
        refs = None
    table[rng.integers(0, requests), 0] = pages + 3  # nobody's
    free = rng.integers(0, pages, 4).tolist()
    want, listed, holders = draft_ref.trim(held, keep, table, free, pages, page, refs)
    for in_place in (False, True):
        blocks, pool = i32(table), i32(np.pad(free, (0, pages - len(free)), constant_values=-9))
        rest = None if refs is None else i32(refs)
        got = eng.kv8_trim(i32(held), i32(keep), blocks, pool, i32([len(free)]), page, refs=rest, in_place=in_place)
        assert (got.block_table is blocks) == in_place and np.array_equal(got.block_table.cpu().numpy(), want)
        assert got.free_count.tolist() == [len(listed)] and pool.cpu().tolist()[:len(listed)] == listed
        assert (pool[len(listed):] == -9).all()
        assert refs is None or rest.cpu().tolist() == holders
        assert in_place or np.array_equal(blocks.cpu().numpy(), table)


def test_trim_of_a_full_list(eng):
    pool = i32([5, 6, 7])
    got = eng.kv8_trim(i32([48]), i32([0]), i32([[0, 1, 2]]), pool, i32([2]), 16)
    assert got.free_count.tolist() == [3] and pool.tolist() == [5, 6, 0] and got.block_table.tolist() == [[-1, -1, -1]]
    got = eng.kv8_trim(i32([]), i32([]), torch.empty(0, 2, dtype=torch.int32, device="cuda"), pool, i32([-4]), 16)
    assert got.free_count.tolist() == [0]


# --------------------------------------------------------------------- fork


@pytest.mark.parametrize("rows,forks,spare", [(6, 3, 5), (40, 30, 9), (700, 300, 400), (5, 0, 2), (9, 8, 0)])
def test_fork(eng, rows, forks, spare):
    rng = np.random.default_rng(rows)
    page, width = 16, 7
    held = np.zeros(rows, int)
    order = rng.permutation(rows)
    target, sources = order[:forks], order[forks:]
    held[sources] = rng.integers(0, width * page + 1, len(sources))
    held[sources[0]] = 32  # full pages
    table, pages, rest = paged(rng, held, page, width, spare)
    source = rng.choice(sources, forks) if forks else np.zeros(0, int)
    free = rest[:spare]
    refs = rng.integers(0, 3, pages)
    if forks > 7:
        source[1], source[2], target[3], source[4] = -1, rows, rows + 5, target[4]  # nobody, nobody, nowhere, itself
        held[source[5]] = width * page + 1  # more than its row
    want = draft_ref.fork(source, target, held, table, free, page, refs)
    shared = i32(refs)
    got = eng.kv8_fork(i32(source), i32(target), i32(held), i32(table), shared, i32(free + [0] * (pages - len(free))), i32([len(free)]), page)
    assert np.array_equal(got.block_table.cpu().numpy(), want[0]) and got.kv_lens.tolist() == list(want[1])
    assert got.free_count.tolist() == [len(want[2])] and shared.cpu().tolist() == list(want[3])
    assert got.copy_from.tolist() == want[4] and got.copy_to.tolist() == want[5]


def test_fork_of_rows_that_are_forked_to(eng):
    """Rows change places: each takes what the other held before the call."""
    table = [[0, 1], [2, -1]]
    refs = i32([0] * 5)
    got = eng.kv8_fork(i32([0, 1]), i32([1, 0]), i32([32, 16]), i32(table), refs, i32([3, 4, 0, 0, 0]), i32([2]), 16)
    assert got.block_table.tolist() == [[2, -1], [0, 1]] and got.kv_lens.tolist() == [16, 32] and refs.tolist() == [1, 1, 1, 0, 0]
    with pytest.raises(ValueError):
        eng.kv8_fork(i32([0]), i32([1]), i32([32, 16]), i32(table), None, i32([3]), i32([1]), 16)


# ---------------------------------------------------------------- all of them


class Requests:
    """Requests whose token t at position p has keys and values of its own, in caches of two layers."""

    def __init__(self, e, n, pages=96, page=16, heads=2, dim=64):
        self.e, self.page, self.dim = e, page, dim
        g = torch.Generator(device="cuda").manual_seed(3)
        self.embed = torch.randn(50, 3, heads, dim, device="cuda", generator=g)
        self.caches = [KV8Cache.allocate(pages, heads, dim, page) for _ in range(2)]
        self.rope = rope_table(dim, 512)
        self.lens, self.table = i32([0] * n), i32(np.full((n, 12), -1))
        self.free, self.count, self.refs = i32(range(pages)), i32([pages]), i32([0] * pages)

    def step(self, tokens, new, parents=None):
        """Attention's output of the step's rows (in both layers), and its plan."""
        e = self.e
        p = e.kv8_plan(self.lens, i32(new), self.table, self.free, self.count, self.page, tokens.numel())
        tree = None if parents is None else e.kv8_tree(i32(parents), p.kv_lens, p.q_start, max(new))
        at = p.positions if tree is None else tree.positions
        out = []
        for i, cache in enumerate(self.caches):
            q, k, v = ((1 + i) * self.embed[tokens]).unbind(1)
            q = e.kv8_append(k, v, cache, p.slots, positions=at, table=self.rope, q=q)
            out.append(e.kv8_attention(q, cache, p.block_table, p.kv_lens, p.q_start) if tree is None else
                       e.kv8_tree_attention(q, cache, p.block_table, p.kv_lens, p.q_start, tree.mask))
        return torch.stack(out, 1), p


def test_steps_over_trees_are_steps_of_tokens(eng):
    """Three requests generate by drafts: trees that hold the right tokens among wrong ones.  What single steps of the same
    tokens leave: their lengths, pages in use, and keys and values within two roundings of the pages' steps."""
    rng = np.random.default_rng(7)
    prompts = [[1, 2, 3], list(range(20)), [9] * 16]
    a = Requests(eng, 3)
    _, p = a.step(torch.tensor(sum(prompts, []), device="cuda"), [len(x) for x in prompts])
    a.lens, a.table, a.count = p.kv_lens, p.block_table, p.free_count
    texts = [list(x) for x in prompts]
    stand = [int(rng.integers(50)) for _ in prompts]  # a token of each that stands, not yet in the cache
    for step in range(8):
        drafted, parents, new, truth = [], [], [], []
        for r in range(3):
            right = rng.integers(0, 50, 4).tolist()  # what the model will say after each
            n = int(rng.integers(1, 30))
            tokens, par = [stand[r]], [-1]
            spine, said = 0, 0
            for i in range(1, n):
                if said < 3 and rng.random() < 0.3:  # the next right token
                    tokens.append(right[said])
                    par.append(spine)
                    spine, said = i, said + 1
                else:
                    tokens.append(50 + i)  # a wrong one
                    par.append(int(rng.integers(0, i)))
            drafted += tokens
            parents += par
            new.append(n)
            truth.append((right, said))
        shown = torch.tensor([t % 50 for t in drafted], device="cuda")
        x, p = a.step(shown, new, parents)
        assert torch.isfinite(x).all()
        starts = p.q_start.tolist()
        drawn = torch.full((starts[-1],), 49 + 1000, device="cuda")
        for r in range(3):
            at, (right, _) = starts[r], truth[r]
            for said in range(4):  # after each right token the next one is drawn
                drawn[at] = right[said]
                child = [i for i in range(starts[r], starts[r + 1]) if parents[i] == at - starts[r] and drafted[i] == right[said]]
                if not child:
                    break
                at = child[0]
        held = a.lens
        took = eng.tree_accept(torch.tensor(drafted, device="cuda"), drawn, p.q_start, parents=i32(parents), slots=p.slots)
        lens = eng.kv8_compact(a.caches, p.block_table, held, p.q_start, took.path, took.kept)
        left = eng.kv8_trim(p.kv_lens, lens, p.block_table, a.free, p.free_count, a.page, refs=a.refs)
        a.lens, a.table, a.count = lens, left.block_table, left.free_count
        for r in range(3):
            k = took.kept[r].item()
            rows = took.path[starts[r]:starts[r] + k].tolist()
            assert k >= 1 and rows[0] == 0
            texts[r] += [drafted[starts[r] + i] for i in rows]
            stand[r] = int(took.token[r]) % 50
    assert a.lens.tolist() == [len(t) for t in texts]
    used = sum(-(-len(t) // a.page) for t in texts)
    assert a.count.item() == 96 - used and (a.table >= 0).sum().item() == used
    held = a.table[a.table >= 0].tolist() + a.free[:a.count.item()].tolist()
    assert sorted(held) == list(range(96))
    # the same tokens in one step each
    b = Requests(eng, 3)
    for i in range(max(map(len, texts))):
        new = [int(i < len(t)) for t in texts]
        _, p = b.step(torch.tensor([t[i] for t in texts if i < len(t)], device="cuda"), new)
        b.lens, b.table, b.count = p.kv_lens, p.block_table, p.free_count
    for ca, cb in zip(a.caches, b.caches):
        for r, t in enumerate(texts):
            pages = -(-len(t) // a.page)
            ka, va = eng.kv8_dequant(ca, a.table[r, :pages].contiguous(), a.dim)
            kb, vb = eng.kv8_dequant(cb, b.table[r, :pages].contiguous(), b.dim)
            for x, y, scale_a, scale_b in ((ka, kb, ca[2], cb[2]), (va, vb, ca[3], cb[3])):
                # a page's step is at most the largest value that was ever on it over 127 (drafts that went among them); a code
                # is rounded when it is stored, when the page grows and when it moves, each time by at most half a step of then:
                # ten steps are twenty roundings
                step = torch.maximum(scale_a[a.table[r, :pages].long()], scale_b[b.table[r, :pages].long()])
                by_token = lambda z: z.transpose(1, 2).flatten(0, 1)[:len(t)]  # noqa: E731 (behind the text: anything)
                assert (by_token((x - y).abs()) <= by_token((10 * step[:, :, None, None]).expand_as(x))).all()


def test_forks_are_copies(eng):
    """Forks of a sequence go on by themselves, and all pages come back."""
    a = Requests(eng, 5)
    text = torch.arange(23, device="cuda")
    _, p = a.step(text, [23, 0, 0, 0, 0])
    a.lens, a.table, a.count = p.kv_lens, p.block_table, p.free_count
    before = a.count.item()
    f = eng.kv8_fork(i32([0, 0, 0]), i32([3, 1, 4]), a.lens, a.table, a.refs, a.free, a.count, a.page)
    eng.kv8_copy(a.caches, f.copy_from, f.copy_to)
    a.lens, a.table, a.count = f.kv_lens, f.block_table, f.free_count
    assert a.lens.tolist() == [23, 23, 0, 23, 23] and a.count.item() == before - 3
    x, p = a.step(torch.tensor([7, 7, 7, 7], device="cuda"), [1, 1, 0, 1, 1])
    assert all(torch.equal(x[0], y) for y in x[1:])
    a.lens, a.table, a.count = p.kv_lens, p.block_table, p.free_count
    x, p = a.step(torch.tensor([8, 9, 8, 10], device="cuda"), [1, 1, 0, 1, 1])
    assert torch.equal(x[0], x[2]) and not torch.equal(x[0], x[1])
    a.lens, a.table, a.count = p.kv_lens, p.block_table, p.free_count
    keep = i32([25, 0, 0, 25, 0])
    left = eng.kv8_trim(a.lens, keep, a.table, a.free, a.count, a.page, refs=a.refs, in_place=True)
    assert left.free_count.item() == before - 1 and a.refs.sum().item() == 1
    left = eng.kv8_trim(keep, i32([0] * 5), a.table, a.free, left.free_count, a.page, refs=a.refs, in_place=True)
    assert left.free_count.item() == 96 and a.refs.sum().item() == 0 and (a.table == -1).all()
    assert sorted(a.free.tolist()) == list(range(96))


def test_beams(eng):
    """Rows that go on from others while they hold something themselves: forks first, then what they held by the old table."""
    a, b = Requests(eng, 4), Requests(eng, 4)
    for each in (a, b):
        _, p = each.step(torch.arange(21 * 4, device="cuda") % 50, [21] * 4)
        each.lens, each.table, each.count = p.kv_lens, p.block_table, p.free_count
    order = [0, 0, 3, 0]  # row 2 goes on from 3, 1 and 3 from 0
    for step in range(3):
        f = eng.kv8_fork(i32(order), i32(range(4)), a.lens, a.table, a.refs, a.free, a.count, a.page)
        eng.kv8_copy(a.caches, f.copy_from, f.copy_to)
        keep = i32([n if order[r] == r else 0 for r, n in enumerate(a.lens.tolist())])
        left = eng.kv8_trim(a.lens, keep, a.table, a.free, f.free_count, a.page, refs=a.refs)
        a.lens, a.table, a.count = f.kv_lens, f.block_table, left.free_count
        text = torch.tensor([7 + step, 8, 9, 10], device="cuda")
        x, p = a.step(text, [1] * 4)
        a.lens, a.table, a.count = p.kv_lens, p.block_table, p.free_count
        if step == 0:  # what rows of their own leave, which had the sources' tokens all along
            y, _ = b.step(torch.cat([text[:1], text[3:]]), [1, 0, 0, 1])
            assert torch.equal(x[0], y[0])
        held = a.table[a.table >= 0].tolist()
        assert len(a.free[:a.count.item()].unique()) == a.count.item()
        assert sorted(set(held) | set(a.free[:a.count.item()].tolist())) == list(range(96))
        assert sum(a.refs.tolist()) == len(held) - len(set(held)) and not set(held) & set(a.free[:a.count.item()].tolist())
    left = eng.kv8_trim(a.lens, i32([0] * 4), a.table, a.free, a.count, a.page, refs=a.refs)
    assert left.free_count.item() == 96 and a.refs.sum().item() == 0


def test_a_cut_into_a_shared_page_goes_on_as_a_fork(eng):
    a, b = Requests(eng, 3), Requests(eng, 1)
    text = torch.arange(40, device="cuda")
    for each, new in ((a, [40, 0, 0]), (b, [40])):
        _, p = each.step(text, new)
        each.lens, each.table, each.count = p.kv_lens, p.block_table, p.free_count
    def fork(source, target):
        f = eng.kv8_fork(i32([source]), i32([target]), a.lens, a.table, a.refs, a.free, a.count, a.page)
        eng.kv8_copy(a.caches, f.copy_from, f.copy_to)
        a.lens, a.table, a.count = f.kv_lens, f.block_table, f.free_count
    def cut(keep):
        left = eng.kv8_trim(a.lens, i32(keep), a.table, a.free, a.count, a.page, refs=a.refs)
        a.lens, a.table, a.count = i32(keep), left.block_table, left.free_count
    fork(0, 1)
    cut([40, 20, 0])  # on page 1, which row 0 holds too
    fork(1, 2)
    cut([40, 0, 20])
    assert a.table[0, 0] == a.table[2, 0] and a.table[0, 1] != a.table[2, 1]
    for i in range(14):  # over the end of the page
        x, p = a.step(torch.tensor([3, 44], device="cuda"), [1, 0, 1])
        a.lens, a.table, a.count = p.kv_lens, p.block_table, p.free_count
        y, p = b.step(torch.tensor([3], device="cuda"), [1])
        b.lens, b.table, b.count = p.kv_lens, p.block_table, p.free_count
        assert torch.equal(x[0], y[0])
    cut([0, 0, 0])
    assert a.count.item() == 96 and a.refs.sum().item() == 0


def test_past_32_bits(eng):
    """Pages that lie more than 2 GiB into the cache: copied, their rows moved, a tree over them."""
    rng = np.random.default_rng(8)
    page, dim, heads = 128, 128, 4
    pages = (1 << 31) // (page * dim) + 4
    host = ref.Cache(3, 1, dim, page, rng)
    cache = KV8Cache(*(torch.empty(x, dtype=torch.int8, device="cuda") for x in ((pages, 1, page, dim), (pages, 1, dim, page))),
                     *(torch.empty((pages, 1), device="cuda") for _ in range(2)))
    for t, d in zip(cache, host.device(torch)):
        t[1:4] = d
    far = [pages - 1, pages - 3, pages - 2]
    eng.kv8_copy([cache], i32([1, 2, 3]), i32(far))
    for t in cache:
        assert torch.equal(t[1:4], t[far])
    held, n, lens = 150, 130, 280
    starts, table = [0, n], np.array([[0, 1, 2]])
    parents = np.array([-1] + [int(rng.integers(max(0, i - 4), i)) for i in range(1, n)])
    mask = draft_ref.tree(parents, [lens], starts, n, 3)[1]
    q = rng.standard_normal((n, heads, dim)).astype(np.float32)
    want, most, big = draft_ref.attend(q, host, table, [lens], starts, mask)
    got = eng.kv8_tree_attention(torch.from_numpy(q).cuda(), cache, i32([far]), i32([lens]), i32(starts), torch.from_numpy(mask).cuda())
    assert (np.abs(got.cpu().numpy() - want) <= ref.attend_bound(want, most, big, False)).all()
    path = np.full(n, -1)
    path[:120] = some_path(rng, n, 120)
    assert eng.kv8_compact([cache], i32([far]), i32([held]), i32(starts), i32(path), i32([120])).tolist() == [270]
    draft_ref.compact(host, table, [held], starts, path, [120])
    for t, d in zip(cache, host.device(torch)):
        assert torch.equal(t[far], d)


def test_captured(eng):
    """The bookkeeping of a step in a graph, replayed over other lengths."""
    rng = np.random.default_rng(1)
    s = torch.cuda.Stream()
    e = ROCmEngine(stream=s)
    with torch.cuda.stream(s):
        held, counts = [10, 33], [12, 9]
        table, pages, rest = paged(rng, [70, 70], 16)
        caches = [ref.Cache(pages, 2, 64, 16, rng).device(torch)]
        lens, starts = i32([22, 42]), i32([0, 12, 21])
        at, blocks, pool, count = i32(held), i32(table), i32(list(rest) + [0] * (pages - len(rest))), i32([len(rest)])
        drafted, drawn = torch.ones(2, 21, dtype=torch.int64, device="cuda")
        parents = i32([-1, 0, 1, 1, 3, 2, 4, 0, 7, 6, 5, 9, -1, 0, 0, 2, 3, 1, 4, 6, 7])

        def step():
            took = e.tree_accept(drafted, drawn, starts, parents=parents)
            end = e.kv8_compact(caches, blocks, at, starts, took.path, took.kept)
            left = e.kv8_trim(lens, end, blocks, pool, count, 16)
            f = e.kv8_fork(i0, i1, at, blocks, refs, pool, count, 16)
            return [*took, end, *left, *f]

        i0, i1, refs = i32([0]), i32([1]), i32([0] * pages)
        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = step()
        for a, b in (([10, 33], 1), ([3, 60], 2), ([40, 16], 1)):
            at.copy_(i32(a))
            lens.copy_(i32([a[0] + 12, a[1] + 9]))
            drawn.copy_(torch.from_numpy(rng.integers(1, 1 + b, 21)))
            state = [x.clone() for x in (*caches[0], pool, refs)]
            g.replay()
            got = [x.clone() for x in (*out, *caches[0], pool, refs)]
            for x, y in zip((*caches[0], pool, refs), state):
                x.copy_(y)
            want = [*step(), *caches[0], pool, refs]
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want))
