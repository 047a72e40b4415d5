"""Normed heads with their rotary positions, alone and on the way into the cache,
on the GPU: the bits of a program that rounds each step to fp32 (decode_ref,
draft_ref), and within the roundings of the 64-bit formula."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import decode_ref as ref  # noqa: E402
import draft_ref  # noqa: E402
from ztensor_amd.decode import HeadNorm, rope_table  # noqa: E402

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16}
EPS = 1e-6


@pytest.fixture(scope="module")
def eng():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from ztensor_amd.engine import ROCmEngine

    return ROCmEngine()


def cuda(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(dtype)


def i32(x):
    return torch.tensor(np.asarray(x, dtype=np.int32).tolist(), dtype=torch.int32, device="cuda").reshape(np.shape(x))


def fused(rng, tokens, heads, kv, dim, dtype, extra=0):
    """q, k, v as slices of one projection's rows (of `extra` more values), on the device and as float32."""
    x = rng.standard_normal((tokens, (heads + 2 * kv) * dim + extra)).astype(np.float32)
    x[:, ::19] *= 6
    d = cuda(x).to(DT[dtype])[:, extra:]
    on = [p.unflatten(1, (-1, dim)) for p in d.split([heads * dim, kv * dim, kv * dim], 1)]
    return on, [p.float().cpu().numpy() for p in on]


def weights(rng, dim):
    w = (1 + 0.4 * rng.standard_normal((2, dim))).astype(np.float32)
    w[:, ::7] *= 3
    return w


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot,extra", [
    (1, 32, 8, 128, 128, 0), (37, 7, 1, 80, 40, 0), (5, 3, 3, 64, 2, 0), (300, 4, 2, 256, 128, 0), (2, 1, 1, 22, 22, 0),
    (9, 5, 5, 96, 52, 0), (3, 2, 1, 2, 2, 0), (65, 3, 2, 256, 256, 1), (17, 4, 4, 128, 64, 3), (33, 2, 2, 200, 0, 0), (4, 9, 1, 130, 130, 0)])
def test_norm_rope(eng, dtype, interleaved, tokens, heads, kv, dim, rot, extra):
    rng = np.random.default_rng(dim * 7 + tokens)
    (q, k, _), (qh, kh, _) = fused(rng, tokens, heads, kv, dim, dtype, extra)
    w = weights(rng, dim)
    positions = rng.integers(0, 500, tokens)
    norm = HeadNorm(cuda(w[0]), cuda(w[1]), EPS)
    table = rope_table(rot, 500) if rot else None
    got = eng.norm_rope(q, k, norm, i32(positions) if rot else None, table, interleaved=interleaved)
    for x, g, by in ((qh, got[0], w[0]), (kh, got[1], w[1])):
        step, exact = draft_ref.normed(x, by, EPS, np.float32), draft_ref.normed(x, by, EPS)
        size = np.abs(exact)
        if rot:
            t = table.cpu().numpy()
            both = np.abs(ref.turn(size, positions, np.stack((np.abs(t[:, 0]), -np.abs(t[:, 1])), 1), interleaved))
            step, exact = ref.turn(step, positions, t, interleaved, dtype=np.float32), ref.turn(exact, positions, t, interleaved)
            # |a c| + |b s| of both values of a pair: the larger one covers each
            size = np.maximum(both, np.abs(ref.turn(size, positions, np.abs(t), interleaved)))
        g = g.cpu()
        want = torch.from_numpy(step).to(DT[dtype])
        assert torch.equal(g, want)
        # the factor and two products, then a product and a sum of the rotation: five roundings, of the type one more
        bound = 5.01 * ref.F24 * size + (torch.finfo(DT[dtype]).eps / 2 * np.abs(exact) + 2.0 ** -25 if dtype == "f16" else 0)
        assert (np.abs(g.double().numpy() - exact) <= bound).all()


def test_one_tensor_no_weights_in_place(eng):
    rng = np.random.default_rng(3)
    (q, k, _), (qh, kh, _) = fused(rng, 11, 6, 2, 128, "f32")
    want = torch.from_numpy(draft_ref.normed(qh, None, 1e-3, np.float32))
    alone, none = eng.norm_rope(q, None, HeadNorm(None, None, 1e-3))
    assert none is None and torch.equal(alone.cpu(), want)
    w = weights(rng, 128)
    table, pos = rope_table(128, 64), i32(range(11))
    norm = HeadNorm(None, cuda(w[1]), 1e-3)
    want = [x.clone() for x in eng.norm_rope(q, k, norm, pos, table)]
    a, b = eng.norm_rope(q, k, norm, pos, table, q_out=q, k_out=k)
    assert a is q and b is k and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(want[0].cpu(), torch.from_numpy(ref.turn(draft_ref.normed(qh, None, 1e-3, np.float32), np.arange(11), table.cpu().numpy(), dtype=np.float32)))


def test_rows_of_zeros_and_of_what_is_not_finite(eng):
    x = np.random.default_rng(4).standard_normal((4, 3, 64)).astype(np.float32)
    x[0, 1] = 0
    x[1, 0, 5] = np.nan
    x[2, 2, 7] = np.inf
    x[3, 1] *= 1e-12  # far below eps
    got = eng.norm_rope(cuda(x), None, HeadNorm(None, None, EPS))[0].cpu().numpy()
    assert (got[0, 1] == 0).all() and np.isnan(got[1, 0]).all()
    assert np.isnan(got[2, 2, 7]) and (np.delete(got[2, 2], 7) == 0).all()
    assert np.array_equal(got, draft_ref.normed(x, None, EPS, np.float32), equal_nan=True)
    far = eng.norm_rope(cuda(x), None, HeadNorm(None, None, EPS), i32([0, 1, 99, -1]), rope_table(32, 50))[0].cpu()
    assert torch.isnan(far[2:, :, :32]).all() and torch.isfinite(far[3, :, 32:]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("dim,rot,page,interleaved,new", [(128, 128, 16, False, (1, 1, 1)), (80, 40, 32, True, (5, 33, 2)),
                                                          (64, 64, 128, False, (130, 3, 64)), (256, 256, 64, True, (70, 1, 2)),
                                                          (128, 0, 16, False, (17, 16, 1)), (72, 6, 16, False, (3, 20, 9))])
def test_append(eng, dtype, dim, rot, page, interleaved, new):
    rng = np.random.default_rng(dim + page)
    held, heads, kv = (5, 0, page + 3), 4, 2
    cache = ref.Cache(24, kv, dim, page, rng)
    cache.scales *= 0.02  # some pages grow
    table = rng.permutation(24)[:21].reshape(3, 7)
    places = [(r, p) for r, (h, n) in enumerate(zip(held, new)) for p in range(h, h + n)]
    slots = [int(table[r, p // page] * page + p % page) for r, p in places]
    slots[-1] = -1
    positions = np.array([p for _, p in places])
    (q, k, v), (qh, kh, vh) = fused(rng, len(slots), heads, kv, dim, dtype)
    w = weights(rng, dim)
    norm = HeadNorm(cuda(w[0]), cuda(w[1]), EPS)
    rope = rope_table(rot, 4096) if rot else None
    on = cache.device(torch)
    got = eng.kv8_append(k, v, on, torch.tensor(slots, device="cuda"), positions=i32(positions) if rot else None, table=rope,
                         interleaved=interleaved, q=q, norm=norm)
    want, key = draft_ref.normed(qh, w[0], EPS, np.float32), draft_ref.normed(kh, w[1], EPS, np.float32)
    if rot:
        t = rope.cpu().numpy()
        want, key = (ref.turn(x, positions, t, interleaved, dtype=np.float32) for x in (want, key))
    assert torch.equal(got.cpu(), torch.from_numpy(want).to(DT[dtype]))
    cache.append([key, vh], slots)
    for x, y in zip(on, cache.device(torch)):
        assert torch.equal(x, y)


def test_append_of_rows_apart_and_gaps(eng):
    """Misaligned rows (one value at a time), and a page's tokens with left-out ones between them."""
    rng = np.random.default_rng(8)
    (_, k, v), (_, kh, vh) = fused(rng, 9, 1, 2, 64, "f16", extra=3)
    slots = [16, 17, -1, 20, 31, 5, -1, 7, 8]
    cache = ref.Cache(3, 2, 64, 16, rng)
    w = weights(rng, 64)
    on = cache.device(torch)
    assert eng.kv8_append(k, v, on, torch.tensor(slots, device="cuda"), norm=HeadNorm(None, cuda(w[1]))) is None
    cache.append([draft_ref.normed(kh, w[1], 1e-6, np.float32), vh], slots)
    for x, y in zip(on, cache.device(torch)):
        assert torch.equal(x, y)


def test_refusals_of_the_methods(eng):
    x = torch.zeros(3, 2, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    for norm in (HeadNorm(w[:32], None), HeadNorm(w.half(), None), HeadNorm(w.cpu(), None), HeadNorm(None, w[::2])):
        with pytest.raises(ValueError):
            eng.norm_rope(x, x, norm)
    with pytest.raises(ValueError):
        eng.norm_rope(x, None, HeadNorm(w, w), None, rope_table(64, 8))
    with pytest.raises(TypeError):
        eng.norm_rope(x, x.half(), HeadNorm(w, w))
    with pytest.raises(ValueError):
        eng.norm_rope(x, x[:2], HeadNorm(w, w))
    from ztensor_amd._lib import ZTError

    with pytest.raises(ZTError):
        eng.norm_rope(x, x, HeadNorm(w, w, 0.0))


def test_captured(eng):
    rng = np.random.default_rng(6)
    from ztensor_amd.engine import ROCmEngine

    s = torch.cuda.Stream()
    e = ROCmEngine(stream=s)
    with torch.cuda.stream(s):
        x = cuda(rng.standard_normal((6, 4, 128)).astype(np.float32))
        w = cuda(weights(rng, 128))
        cache = ref.Cache(4, 4, 128, 16).device(torch)
        slots, pos, table = torch.arange(6, device="cuda"), i32(range(6)), rope_table(128, 16)
        out = torch.empty_like(x)

        def step():
            e.norm_rope(x, None, HeadNorm(w[0], None), pos, table, q_out=out)
            e.kv8_append(x, x, cache, slots, positions=pos, table=table, norm=HeadNorm(None, w[1]))

        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step()
        for _ in range(3):
            x.copy_(cuda(rng.standard_normal((6, 4, 128)).astype(np.float32)))
            g.replay()
            got = [t.clone() for t in (out, *cache)]
            step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, (out, *cache)))
