"""Attention calls of random shapes, lengths, windows, missing pages, scales
and padding, each row, head and dim within its own bound."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_attention_scales import attend, paged  # noqa: E402
from test_gpu_decode import DT, cuda, eng, i32  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def drawn(rng, dtype):
    """(q, host cache, table, lengths, rows of each request, starts, window)"""
    kv, page = int(rng.choice([1, 2, 4])), int(rng.choice([16, 32, 64, 128]))
    heads = kv * int(rng.choice([1, 1, 2, 4, 7, 33]))
    dim = int(rng.choice([8, 64, 80, 128, 192, 200, 256]))
    requests = int(rng.integers(1, 6))
    lens = [5] + [int(n) for n in rng.integers(0, 500, requests - 1)]
    new = [int(n) for n in (1,) + tuple(rng.choice(([1], [0, 2, 8], [20, 60], [0, 1, 3, 40, 90])[rng.integers(4)], requests - 1))]
    host, table = paged(rng, lens, page, kv, dim)
    shape = host.scales[1].shape
    change = rng.integers(4)
    if change == 1:
        host.scales[1] *= rng.random(shape) > 0.4
    elif change == 2:
        host.scales[1] = np.exp(rng.uniform(-50, 6, shape)).astype(np.float32)
    elif change == 3:
        host.scales[0] *= np.exp(rng.uniform(-8, 1.5, shape)).astype(np.float32)
    host.scales[:, 0] = rng.choice([0, 1e20, np.nan])
    if rng.random() < 0.3:
        table[rng.random(table.shape) < 0.1] = rng.choice([-1, 1 << 28])
    before, after = (int(rng.integers(0, 5)), int(rng.integers(0, 50))) if rng.random() < 0.3 else (0, 0)
    starts = before + np.concatenate([[0], np.cumsum(new)]).astype(int)
    rows = starts[-1] + after
    q = rng.standard_normal((rows, heads, dim)) * np.exp(rng.uniform(-3, 0.7, (rows, heads, 1)))
    return cuda(q.astype(np.float32)).to(DT[dtype]), host, table, lens, new, starts, int(rng.choice([0, 0, 1, 17, 64, 100, 1000]))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("seed", range(10))
def test_random_calls(eng, seed, dtype):  # noqa: F811
    rng = np.random.default_rng(seed)
    for trial in range(5):
        q, host, table, lens, new, starts, window = drawn(rng, dtype)
        want, bound = attend(q.float().cpu().numpy(), host, table, lens, starts, dtype == "f16", window)
        for bounds in ({}, {"max_q": max(new), "max_kv": max(lens)}, {"max_q": 1, "max_kv": 1}):
            out = eng.kv8_attention(q, host.device(torch), i32(table), i32(lens), i32(starts), window=window, **bounds)
            far = np.abs(out.double().cpu().numpy() - want)
            assert (far <= bound).all(), (trial, q.shape, lens, new, window, bounds, float((far / (bound + 1e-300)).max()))
