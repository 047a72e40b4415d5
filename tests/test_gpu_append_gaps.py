"""The cache writer on steps in which a page's tokens do not follow each other
place by place: some left out (slot -1, or outside the cache), places passed
over, places in no order."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import decode_ref as ref  # noqa: E402
from test_gpu_decode import DT, check_cache, cuda, eng, i32  # noqa: E402, F401
from ztensor_amd.decode import rope_table  # noqa: E402

pytestmark = pytest.mark.gpu


def steps(page):
    """Slots of a step: no page's tokens stand in two places."""
    a, b, c = 2 * page, 5 * page, 7 * page
    yield "a place passed over", [a + 5, a + 7]
    yield "one left out", [a + 5, -1, a + 7, b]
    yield "rejected in the middle of each request", [a + 9, a + 10, -1, a + 12, b, -1, b + 2, c + 3, 1 << 40, -7, c + 6]
    yield "a page that starts anew, with gaps", [a, -1, a + 3, -1, -1, a + 8, b + 1, b + 3]
    yield "from the end of one to the next", [a + page - 3, -1, a + page - 1, -1, b, b + 1, -1, b + 4]
    yield "first place not first", [a + 7, a + 2, a, a + 5, b + 6, b + 4]
    yield "over a wave's tokens", [a + 1] + [-1] * 70 + [a + 4] + [-1] * 200 + [a + 6, b]
    yield "over a workgroup's", [-1] * 130 + [a + 1] + [-1] * 300 + [a + 4] + [-1] * 4000 + [a + 6, -1, b + 2] + [-1] * 2500
    yield "nothing", [-1] * 90
    full = [t for p in range(page) for t in ([a + p, -1] if p % 3 else [a + p])]
    yield "a whole page", full + [-1] + [b + p for p in range(1, page, 2)]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("page,dim,table_of", [(16, 128, 0), (32, 40, 0), (64, 64, 64), (128, 256, 100)])
def test_tokens_that_do_not_follow_each_other(eng, page, dim, table_of, dtype):  # noqa: F811
    rng = np.random.default_rng(page)
    host = ref.Cache(9, 2, dim, page, rng)  # codes of earlier tokens, scales that some of the new ones pass
    host.scales *= 0.3
    cache = host.device(torch)
    table = rope_table(table_of, 500) if table_of else None
    for name, slots in steps(page):
        k, v = (cuda(rng.standard_normal((len(slots), 2, dim)).astype(np.float32)).to(DT[dtype]) for _ in range(2))
        pos = rng.integers(0, 500, len(slots))
        s = torch.tensor(slots, device="cuda")
        eng.kv8_append(k, v, cache, s, **({"positions": i32(pos), "table": table} if table_of else {}))
        kn, vn = k.float().cpu().numpy(), v.float().cpu().numpy()
        if table_of:
            kn = ref.turn(kn, pos, table.cpu().numpy(), dtype=np.float32)
        host.append((kn, vn), slots)
        print(name, flush=True)
        check_cache(cache, host)


def test_random_steps(eng):  # noqa: F811
    rng = np.random.default_rng(11)
    for trial in range(40):
        page = int(rng.choice([16, 32, 64, 128]))
        host = ref.Cache(30, 1, 64, page, rng)
        cache = host.device(torch)
        slots = []
        for p in rng.permutation(30)[:rng.integers(1, 20)]:
            for place in np.sort(rng.permutation(page)[:rng.integers(1, page + 1)]):
                slots += [-1] * int(rng.choice([0, 0, 0, 0, 1, 3, 80])) + [int(p) * page + int(place)]
        k, v = rng.standard_normal((2, len(slots), 1, 64)).astype(np.float32)
        eng.kv8_append(cuda(k), cuda(v), cache, torch.tensor(slots, device="cuda"))
        host.append((k, v), slots)
        check_cache(cache, host)
