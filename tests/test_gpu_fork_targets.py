"""Forks whose targets come twice: the first of them is done, the others take nothing, and no page is lost."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import draft_ref  # noqa: E402
from test_gpu_pages import eng, i32, paged  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def check(eng, source, target, held, table, free, pages, page):  # noqa: F811
    refs = np.zeros(pages, int)
    first = [i for i, t in enumerate(target) if t not in target[:i]]
    once = draft_ref.fork([source[i] for i in first], [target[i] for i in first], held, table, free, page, refs)
    copies = np.full((2, len(target)), -1)
    copies[:, first] = once[4:]
    shared = i32(refs)
    got = eng.kv8_fork(i32(source), i32(target), i32(held), i32(table), shared, i32(free + [0] * (pages - len(free))), i32([len(free)]), page)
    assert np.array_equal(got.block_table.cpu().numpy(), once[0]) and got.kv_lens.tolist() == list(once[1])
    assert got.free_count.tolist() == [len(once[2])] and shared.cpu().tolist() == list(once[3])
    assert got.copy_from.tolist() == copies[0].tolist() and got.copy_to.tolist() == copies[1].tolist()
    left = got.free_count.item()
    mine = [int(p) for r, n in zip(got.block_table.cpu().numpy(), got.kv_lens.tolist()) for p in r[:-(-n // page)]]
    assert len(set(mine)) + left == len(set(mine) | set(free)), "pages that nobody has"


@pytest.mark.parametrize("rows,forks,spare", [(3, 2, 2), (9, 8, 9), (40, 300, 15), (40, 60, 400), (600, 500, 120)])
def test_targets_that_come_twice(eng, rows, forks, spare):  # noqa: F811
    rng = np.random.default_rng(forks)
    page, width = 16, 7
    held = np.zeros(rows, int)
    to = max(1, rows // 3)
    held[to:] = rng.integers(0, width * page + 1, rows - to)
    held[to] = 40
    table, pages, rest = paged(rng, held, page, width, spare)
    source, target = rng.integers(to, rows, forks).tolist(), rng.integers(0, to, forks).tolist()
    source[0] = to
    if forks > 7:
        source[3], target[5], target[6] = target[3], rows + 2, -1  # itself, nowhere
    check(eng, source, target, held, table, rest[:spare], pages, page)


def test_many_rows(eng):  # noqa: F811
    """Rows that share a bit are no targets that come twice."""
    rows = 300000
    held, table = np.zeros(rows, int), np.full((rows, 1), -1)
    held[7], table[7, 0] = 9, 0
    for target in ([5, 5 + (1 << 18), 8], [5, 5 + (1 << 18), 5]):
        check(eng, [7, 7, 7], target, held, table, [1, 2, 3], 4, 16)
