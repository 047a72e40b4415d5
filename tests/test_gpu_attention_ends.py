"""Attention at the ends of its numbers: lengths and windows up to 2^31 - 1."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import decode_ref as ref  # noqa: E402
from test_gpu_decode import DT, cuda, eng, i32, paged  # noqa: E402, F401

pytestmark = pytest.mark.gpu

WIDTH, PAGE, LAST = 2 ** 24, 128, 3  # a table of 2^31 tokens: pages outside the cache, but for the last ones


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("new", [1, 7, 40])
@pytest.mark.parametrize("size", [2 ** 31 - 1, 2 ** 31 - 64, 2 ** 31 - 65, 2 ** 31 - 200])
def test_lengths_to_31_bits(eng, size, new, dtype):  # noqa: F811
    rng = np.random.default_rng(new)
    short = size - (WIDTH - LAST) * PAGE
    host, few = paged(rng, [LAST * PAGE], PAGE, 2, 128)
    few = few[:, :LAST]
    table = torch.full((1, WIDTH), -1, dtype=torch.int32, device="cuda")
    table[0, -LAST:] = i32(few[0])
    q = cuda(rng.standard_normal((new, 8, 128)).astype(np.float32)).to(DT[dtype])
    for window in (100, 64) + ((0,) if new == 1 and dtype == "f32" else ()):
        want, most, big = ref.attend(q.float().cpu().numpy(), host, few, [short], [0, new], window)
        out = eng.kv8_attention(q, host.device(torch), table, i32([size]), i32([0, new]), window=window)
        assert (np.abs(out.double().cpu().numpy() - want) <= ref.attend_bound(want, most, big, dtype == "f16")).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_windows_to_31_bits(eng, dtype):  # noqa: F811
    """Also of requests with more rows than tokens, whose first rows see nothing."""
    rng = np.random.default_rng(1)
    lens, new = [5, 70, 300, 1], [10, 90, 7, 40]
    host, table = paged(rng, lens, 16, 2, 128)
    starts = np.concatenate([[0], np.cumsum(new)])
    q = cuda(rng.standard_normal((starts[-1], 8, 128)).astype(np.float32)).to(DT[dtype])
    want, most, big = ref.attend(q.float().cpu().numpy(), host, table, lens, starts)
    for most_q in (90, 1):
        args = {"max_q": most_q, "max_kv": 300}
        out = eng.kv8_attention(q, host.device(torch), i32(table), i32(lens), i32(starts), **args)
        assert (np.abs(out.double().cpu().numpy() - want) <= ref.attend_bound(want, most, big, dtype == "f16")).all()
        for window in (300, 2 ** 30, 2 ** 31 - 1):
            assert torch.equal(eng.kv8_attention(q, host.device(torch), i32(table), i32(lens), i32(starts), window=window,
                                                 **args), out)
