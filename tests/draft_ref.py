"""Definitions of the operators of drafted trees, shared pages and normed heads,
for tests: numpy, one value after another."""
import numpy as np


def normed(x, w, eps, dtype=np.float64):
    """Each head of x [T, H, D] over its root mean square, times w (None: ones); in float32 the factor (of a 64-bit sum)
    and both products are rounded by themselves."""
    y = x.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        r = 1.0 / np.sqrt(np.sum(y * y, -1, keepdims=True) / x.shape[-1] + eps)
        y = x.astype(dtype) * r.astype(dtype)
        return y if w is None else y * w.astype(dtype)
