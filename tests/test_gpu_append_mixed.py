"""The cache writer on steps of very many pages, and of few pages beside very
many: single tokens of many sequences, runs of any lengths, prompts, tokens that
are left out.  So many heads that a window's pages go to workgroups of other
windows too; what is written has the bits of calls of one head each, whose
windows keep their pages, and the definition's."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import decode_ref as ref  # noqa: E402
from test_gpu_decode import DT, cuda, eng  # noqa: E402, F401
from ztensor_amd.decode import HeadNorm, KV8Cache  # noqa: E402

pytestmark = pytest.mark.gpu

HEADS, DIM = 64, 8


def runs(rng, name):
    """Lengths of the step's runs, each on pages of its own, and how many tokens are left out before each."""
    if name == "single":
        return [1] * 1500, None
    if name == "single, then a prompt":
        return [1] * 300 + [900], None
    if name == "a prompt, then single":
        return [1100] + [1] * 70, None
    if name == "three windows of many":
        return [1] * 100 + [500] + [1] * 90 + [700] + [1] * 64, None
    if name == "runs of any lengths":
        return rng.integers(1, 40, 120).tolist(), None
    if name == "many windows a group":
        return [1] * 2100 + [1500] + rng.integers(1, 9, 300).tolist(), None
    lens = rng.choice([1, 1, 1, 2, 5, 130], 250).tolist()  # some left out
    return lens, rng.choice([0, 0, 0, 1, 2, 70], 250).tolist()


def step(rng, name, page):
    lens, out = runs(rng, name)
    need = [-(-(n + 3) // page) for n in lens]  # (a run begins up to three places behind its page's first)
    order = rng.permutation(sum(need))
    slots, at = [], 0
    for i, (n, p) in enumerate(zip(lens, need)):
        own = order[at:at + p]
        at += p
        first = int(rng.integers(0, 4))
        slots += [-1] * (out[i] if out else 0) + [int(own[t // page]) * page + t % page for t in range(first, first + n)]
    return np.array(slots), sum(need)


@pytest.mark.parametrize("dtype,page,norm", [("f32", 16, False), ("f16", 64, False), ("f16", 128, True), ("f32", 32, True)])
@pytest.mark.parametrize("name", ["single", "single, then a prompt", "a prompt, then single", "three windows of many", "runs of any lengths",
                                  "many windows a group", "some left out"])
def test_pages_that_others_write(eng, name, dtype, page, norm):  # noqa: F811
    rng = np.random.default_rng(page + len(name))
    slots, pages = step(rng, name, page)
    tokens = len(slots)
    assert tokens > 256 and 2 * HEADS * (-(-tokens // 64)) > 512
    host = ref.Cache(pages, HEADS, DIM, page)
    host.codes[:] = rng.integers(-127, 128, host.codes.shape)
    host.scales[:] = (0.01 * rng.integers(1, 4, host.scales.shape)).astype(np.float32)
    cache = KV8Cache(*host.device(torch))
    k, v = (cuda(rng.standard_normal((tokens, HEADS, DIM)).astype(np.float32)).to(DT[dtype]) for _ in range(2))
    q = cuda(rng.standard_normal((tokens, 3, DIM)).astype(np.float32)).to(DT[dtype]) if norm else None
    s = torch.from_numpy(slots).cuda()
    weights = HeadNorm(cuda(rng.standard_normal(DIM).astype(np.float32)), cuda(rng.standard_normal(DIM).astype(np.float32))) if norm else None
    heads = sorted(rng.permutation(HEADS)[:4].tolist())
    alone = [KV8Cache(*(x[:, h:h + 1].contiguous() for x in cache)) for h in heads]
    got = eng.kv8_append(k, v, cache, s, q=q, norm=weights)
    if norm:
        assert torch.equal(got, eng.norm_rope(q, None, weights)[0])
    for h, one in zip(heads, alone):
        eng.kv8_append(k[:, h:h + 1], v[:, h:h + 1], one, s, norm=weights)
        for x, y in zip(cache, one):
            assert torch.equal(x[:, h:h + 1], y), h
    if norm:  # (its definition: normed keys that are not rounded to their type; test_gpu_norm)
        return
    one = ref.Cache(pages, 1, DIM, page)
    h = heads[0]
    one.codes[:, :, 0], one.scales[:, :, 0] = host.codes[:, :, h], host.scales[:, :, h]
    one.append([x[:, h:h + 1].float().cpu().numpy() for x in (k, v)], slots.tolist())
    for x, y in zip(cache, one.device(torch)):
        assert torch.equal(x[:, h:h + 1], y)


@pytest.mark.parametrize("heads", [1, 12, 64])
@pytest.mark.parametrize("lens", [[1] * 20, [1] * 64, [1] * 65, [1] * 100, [1] * 129, [1] * 200, [1] * 256, [1] * 300, [65], [130], [300], [60, 1, 1, 3, 70],
                                  [1] * 60 + [140], [7] * 31], ids=lambda x: f"{len(x)} of {sum(x)}")
def test_last_windows_of_few_tokens(eng, lens, heads):  # noqa: F811
    """A last window of fewer tokens than others has workgroups: all pages are somebody's."""
    rng = np.random.default_rng(heads + sum(lens))
    page, need = 16, [-(-n // 16) for n in lens]
    order, slots, at = rng.permutation(sum(need)), [], 0
    for n, p in zip(lens, need):
        slots += [int(order[at + t // page]) * page + t % page for t in range(n)]
        at += p
    host = ref.Cache(sum(need), heads, DIM, page)
    cache = host.device(torch)
    k, v = rng.standard_normal((2, sum(lens), heads, DIM)).astype(np.float32)
    eng.kv8_append(cuda(k), cuda(v), cache, torch.tensor(slots, device="cuda"))
    host.append((k, v), slots)
    for x, y in zip(cache, host.device(torch)):
        assert torch.equal(x, y)
