"""Copies of the largest pages that a cache may have."""
import pytest

torch = pytest.importorskip("torch")

from ztensor_amd.decode import KV8Cache  # noqa: E402
from ztensor_amd.engine import ROCmEngine  # noqa: E402

pytestmark = pytest.mark.gpu


def test_a_page_of_two_gib():
    """65536 heads of 256 dims, 128 tokens: 2^31 bytes of keys and as many of values."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("under 20 GiB free")
    eng = ROCmEngine()
    cache = KV8Cache.allocate(2, 1 << 16, 256, 128)
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes.view(-1)[: 1 << 31].random_(-127, 128)
        scale[0] = torch.rand(1 << 16, device="cuda")
    first = [codes.view(-1)[:4096].clone() for codes in (cache.k, cache.v)]
    eng.kv8_copy([cache], torch.tensor([0], dtype=torch.int32, device="cuda"), torch.tensor([1], dtype=torch.int32, device="cuda"))
    for codes, scale, was in zip(cache[:2], cache[2:], first):
        flat = codes.view(-1)
        assert torch.equal(flat[:4096], was) and torch.equal(flat[: 1 << 31], flat[1 << 31:])
        assert torch.equal(scale[0], scale[1])
