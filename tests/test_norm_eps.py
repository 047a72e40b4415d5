"""Normed heads: what is added to a mean of squares may be any positive number."""
import ctypes

import numpy as np
import pytest

from test_norm import P, norm, ref, rows
from ztensor_amd import _lib

EPS = [5e-324, 1e-300, 1e30, 1.0000001e30, 1e38, 1e300, 1.7976931348623157e308]


@pytest.mark.parametrize("eps", EPS)
def test_is_taken(eps):
    lib, two = _lib.load(), (_lib.Rows * 2)(rows(), rows())
    assert lib.zt_norm_rope(two, two, 2, ref(norm(eps=eps)), P, P, 0, 64, 64, 100, 0, 0, None) == 0
    cache = _lib.KV8(k=P, v=P, k_scale=P, v_scale=P, pages=8, kv_heads=2, head_dim=64, page_tokens=16)
    one = ref(rows(heads=2))
    assert lib.zt_kv8_append_norm(ctypes.byref(cache), one, one, P, None, None, ref(norm(eps=eps)), P, P, 0, 64, 100, 0, 0, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("eps", EPS)
def test_values(eps):
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from ztensor_amd.decode import HeadNorm
    from ztensor_amd.engine import ROCmEngine

    x = np.random.default_rng(1).standard_normal((5, 3, 64)).astype(np.float32) * np.float32(1e20)
    got, _ = ROCmEngine().norm_rope(torch.from_numpy(x).cuda(), None, HeadNorm(None, None, eps))
    y = x.astype(np.float64)
    r = (1 / np.sqrt((y * y).mean(-1, keepdims=True) + eps)).astype(np.float32)
    assert np.array_equal(got.cpu().numpy(), x * r)
