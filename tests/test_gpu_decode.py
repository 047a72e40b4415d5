"""Rotary positions, the int8 paged cache and its attention, block tables and
sampling on the GPU, against the definitions in 64 bits (decode_ref).

Bars: rotations, codes and scales to the bit of a program that rounds each
step to fp32 (and within the roundings of the 64-bit rotation); attention
within decode_ref.attend_bound; tables, slots and tokens equal."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import decode_ref as ref  # noqa: E402
from ztensor_amd import _lib  # noqa: E402
from ztensor_amd.decode import KV8Cache, rope_table  # noqa: E402

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16}


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


def fused(rng, tokens, heads, kv, dim, dtype):
    """q, k, v as slices of one projection's rows, on the device and as float32."""
    x = rng.standard_normal((tokens, (heads + 2 * kv) * dim)).astype(np.float32)
    x[:, ::19] *= 6
    d = cuda(x).to(DT[dtype])
    parts = d.split([heads * dim, kv * dim, kv * dim], 1)
    on = [p.view(tokens, -1, dim) for p in parts]
    return on, [p.float().cpu().numpy() for p in on]


# ------------------------------------------------------------------- rotary


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot", [(1, 32, 8, 128, 128), (37, 7, 1, 80, 40), (5, 3, 3, 64, 2),
                                                     (300, 4, 2, 256, 128), (2, 1, 1, 22, 22), (9, 5, 5, 96, 52)])
def test_rope(eng, tokens, heads, kv, dim, rot, interleaved, dtype):
    rng = np.random.default_rng(tokens * dim + rot)
    (q, k, _), (qn, kn, _) = fused(rng, tokens, heads, kv, dim, dtype)
    table = rope_table(rot, 700, scaling={"type": "yarn", "factor": 4, "original_max_position": 128})
    tn = table.cpu().numpy()
    pos = rng.integers(0, 700, tokens)
    for inverse in (False, True):
        got = eng.rope(q, k, i32(pos), table, interleaved=interleaved, inverse=inverse)
        for y, x in zip(got, (qn, kn)):
            want = ref.turn(x, pos, tn, interleaved, inverse)
            once = ref.turn(x, pos, tn, interleaved, inverse, np.float32)
            assert y.is_contiguous() and torch.equal(y, cuda(once).to(DT[dtype]))
            # three roundings of terms of at most |a| + |b|, and the output's
            size = ref.turn(np.abs(x), pos, np.abs(tn), interleaved, True)  # |a c| + |b s| in the first, at least
            bound = 4 * ref.F24 * (np.abs(size) + np.abs(want) + np.abs(x).max(-1, keepdims=True) * 2)
            bound = bound + (2.0 ** -11 * np.abs(want) if dtype == "f16" else 0)
            assert (np.abs(y.double().cpu().numpy() - want) <= bound).all()


def test_rope_in_place_alone_and_outside_the_table(eng):
    rng = np.random.default_rng(3)
    (q, k, _), (qn, _, _) = fused(rng, 6, 4, 2, 64, "f32")
    table = rope_table(32, 10)
    pos = [0, 9, 10, -1, 1 << 30, 3]
    y, none = eng.rope(q, None, i32(pos), table)
    assert none is None
    assert torch.isnan(y[2:5, :, :32]).all() and torch.equal(y[2:5, :, 32:], q[2:5, :, 32:])
    assert torch.equal(y[[0, 1, 5]], cuda(ref.turn(qn, [0, 9, 0, 0, 0, 3], table.cpu().numpy(), dtype=np.float32))[[0, 1, 5]])
    back = q.clone()
    eng.rope(back, None, i32([0, 9, 0, 0, 0, 3]), table, q_out=back)
    eng.rope(back, None, i32([0, 9, 0, 0, 0, 3]), table, q_out=back, inverse=True)
    assert torch.allclose(back, q, rtol=0, atol=float(q.abs().max()) * 8 * ref.F24)


def test_rope_gradient(eng):
    """The inverse rotation is the gradient: against the formula's transpose and against differences."""
    rng = np.random.default_rng(8)
    x, g = rng.standard_normal((2, 3, 2, 16)).astype(np.float32)
    table = rope_table(12, 50)
    pos = [4, 49, 17]
    dx = eng.rope(cuda(g), None, i32(pos), table, inverse=True)[0].double().cpu().numpy()
    f = lambda v: (ref.turn(v, pos, table.cpu().numpy()) * g).sum()  # noqa: E731
    for t, h, d in [(0, 0, 0), (1, 1, 11), (2, 0, 5), (2, 1, 14)]:
        e = np.zeros(x.shape)
        e[t, h, d] = 1e-3
        assert abs((f(x + e) - f(x - e)) / 2e-3 - dx[t, h, d]) <= 1e-6  # linear: only roundings differ


# -------------------------------------------------------------------- cache


def check_cache(cache, host):
    k, v, ks, vs = cache
    k2, v2, ks2, vs2 = host.device(torch)
    for codes, scale, codes2, scale2 in ((k, ks, k2, ks2), (v, vs, v2, vs2)):
        ok = ~torch.isnan(scale2)  # a page whose scale is NaN has no values
        assert torch.equal(~torch.isnan(scale), ok) and torch.equal(scale[ok], scale2[ok])
        assert torch.equal(codes[ok], codes2[ok])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv,dim,rot,interleaved", [(4, 2, 128, 128, False), (7, 1, 80, 40, True),
                                                          (2, 2, 256, 256, False), (3, 3, 24, 20, False)])
def test_append_over_steps(eng, heads, kv, dim, rot, interleaved, page, dtype):
    """Prompts, then single tokens, some larger than all before: scales grow, pages fill up and new ones start."""
    rng = np.random.default_rng(page + dim)
    host = ref.Cache(12, kv, dim, page, rng)  # codes of earlier owners
    cache = host.device(torch)
    table = rope_table(rot, 1000, base=500.0)
    order, lens = rng.permutation(12), [0, 0, 0]
    pages = [order[:5], order[5:8], order[8:]]
    for step, add in enumerate([(page + 3, 1, 0), (1, page - 1, 5), (1, 1, 1), (page, 0, 1), (2, 1, 2 * page)]):
        slots, pos = [], []
        for r, n in enumerate(add):
            slots += [pages[r][p // page] * page + p % page for p in range(lens[r], lens[r] + n)]
            pos += list(range(lens[r], lens[r] + n))
            lens[r] += n
        (q, k, v), (qn, kn, vn) = fused(rng, len(slots), heads, kv, dim, dtype)
        grow = 1.0 if step % 2 else 3.0
        k, v, kn, vn = k * grow, v * grow, (k * grow).float().cpu().numpy(), (v * grow).float().cpu().numpy()
        out = eng.kv8_append(k, v, cache, torch.tensor(np.array(slots).tolist(), device="cuda"), positions=i32(pos), table=table,
                             interleaved=interleaved, q=q)
        tn = table.cpu().numpy()
        assert torch.equal(out, cuda(ref.turn(qn, pos, tn, interleaved, dtype=np.float32)).to(DT[dtype]))
        key = ref.turn(kn, pos, tn, interleaved, dtype=np.float32)
        before = host.values()
        host.append((key, vn), slots)
        check_cache(cache, host)
        # and the meaning of it, in 64 bits: a new value is within half a step, one that was there by another half
        exact, now, scales = (ref.turn(kn, pos, tn, interleaved), vn.astype(np.float64)), host.values(), host.scales
        for kind in range(2):
            for t, s in enumerate(slots):
                far = np.abs(now[kind, s // page, :, s % page] - exact[kind][t])
                assert (far <= scales[kind, s // page, :, None] * (0.5 + 2e-5) + 1e-30).all()
        old = [(r, p) for r in range(3) for p in range(lens[r] - add[r])]
        for r, p in old:
            at = (slice(None), pages[r][p // page], slice(None), p % page)
            assert (np.abs(now[at] - before[at]) <= scales[:, pages[r][p // page], :, None] * (0.5 + 2e-5)).all()
    some = i32([order[0], 12, order[6], -1])
    keys, values = eng.kv8_dequant(cache, some, dim)
    f32 = host.codes.astype(np.float32) * host.scales[..., None, None]
    for got, w in zip((keys, values), f32):
        assert torch.equal(got[[0, 2]], cuda(w[[order[0], order[6]]])) and torch.isnan(got[[1, 3]]).all()


def test_append_without_rotation_and_with_odd_strides(eng):
    """Rows that 4 values at a time do not fit, tokens without a slot, slots outside the cache."""
    rng = np.random.default_rng(5)
    host = ref.Cache(3, 2, 40, 16, rng)
    cache = host.device(torch)
    x = cuda(rng.standard_normal((2, 9, 2, 43)).astype(np.float32))
    k, v = x[0, :, :, 1:41], x[1, :, :, 3:43]
    slots = [-1, 5, 6, 48, -7, 16, 17, 1 << 40, 47]
    assert eng.kv8_append(k, v, cache, torch.tensor(slots, device="cuda")) is None
    host.append((k.cpu().numpy(), v.cpu().numpy()), slots)
    check_cache(cache, host)


def test_append_special_values(eng):
    """A page of zeros; values that are not finite make their page's scale NaN, for good, and no other's."""
    host = ref.Cache(4, 1, 64, 16)
    cache = host.device(torch)
    x = np.random.default_rng(1).standard_normal((5, 1, 64)).astype(np.float32)
    k, v = x.copy(), x.copy()
    k[0], v[1, 0, 3], k[2, 0, 9], v[3] = 0, np.inf, np.nan, 1e-42
    slots = [0, 16, 32, 48, 49]
    for s, at in ((slots, slice(0, 5)), ([1, 17, 33, 50], slice(0, 4))):
        if s is not slots:
            k, v = x.copy(), x.copy()
        eng.kv8_append(cuda(k[at]), cuda(v[at]), cache, torch.tensor(s, device="cuda"))
        host.append((k[at], v[at]), s)
        check_cache(cache, host)
    assert np.isnan(host.scales[1, 1, 0]) and np.isnan(host.scales[0, 2, 0]) and np.isfinite(host.scales[0, 1, 0])


@pytest.mark.parametrize("tokens", [2049, 5000])
def test_append_of_many_tokens(eng, tokens):
    rng = np.random.default_rng(tokens)
    page = 32
    host = ref.Cache(-(-tokens // page) + 2, 2, 64, page, rng)
    cache = host.device(torch)
    order = rng.permutation(host.codes.shape[1])
    slots = [int(order[(7 + t) // page]) * page + (7 + t) % page for t in range(tokens)]
    k, v = rng.standard_normal((2, tokens, 2, 64)).astype(np.float32)
    eng.kv8_append(cuda(k), cuda(v), cache, torch.tensor(slots, device="cuda"))
    host.append((k, v), slots)
    check_cache(cache, host)


# --------------------------------------------------------------------- plan


@pytest.mark.parametrize("requests,page,width,spare,most", [(1, 16, 1, 1, 3), (5, 16, 4, 3, 9), (300, 32, 12, 400, 40),
                                                            (700, 64, 9, 5000, 2), (257, 128, 3, 0, 130), (4, 64, 80, 90, 3000)])
def test_plan(eng, requests, page, width, spare, most):
    rng = np.random.default_rng(requests + width)
    for trial in range(3):
        lens = rng.integers(-1, width * page + 1, requests)
        add = rng.integers(-1, most + 1, requests) * (rng.random(requests) < 0.8)
        table = rng.integers(0, 10 ** 6, (requests, width)).astype(np.int32)
        table[rng.random((requests, width)) < 0.02] = -1
        free = rng.permutation(spare).astype(np.int32)
        want = ref.plan(lens, add, table, free, page)
        t = len(want[1])
        for tokens in (t, t + 37, max(0, t - 5)):
            p = eng.kv8_plan(i32(lens), i32(add), i32(table), i32(np.append(free, [7, 7])), i32([spare]), page, tokens,
                             in_place=trial == 1)
            assert p.block_table.cpu().tolist() == want[0].tolist()
            assert p.slots.cpu().tolist() == (want[1] + [-1] * 37)[:tokens]
            assert p.positions.cpu().tolist() == (want[2] + [0] * 37)[:tokens]
            assert p.q_start.cpu().tolist() == want[3] and p.kv_lens.cpu().tolist() == want[4]
            assert p.free_count.cpu().tolist() == [want[5]]


def test_plan_of_nothing_and_of_lengths_that_do_not_fit(eng):
    p = eng.kv8_plan(i32([]), i32([]), torch.empty((0, 4), dtype=torch.int32, device="cuda"), i32([3]), i32([1]), 16, 2)
    assert p.q_start.tolist() == [0] and p.free_count.tolist() == [1] and p.slots.tolist() == [-1, -1]
    big = 2 ** 31 - 1
    p = eng.kv8_plan(i32([big, 3, 0]), i32([big, big, 2]), i32([[5, 6]] * 3), i32([9, 8]), i32([99]), 16, 4)
    assert p.kv_lens.tolist() == [big, 3, 2] and p.free_count.tolist() == [1] and p.slots.tolist() == [-1] * 4
    assert p.block_table.tolist() == [[5, 6], [5, 6], [8, 6]]


def test_plan_of_a_length_past_31_bits(eng):
    """A row that would have room for it: the request gets nothing, as one that does not fit its row."""
    width = 2 ** 24  # of pages of 128: 2^31 tokens
    p = eng.kv8_plan(i32([2 ** 31 - 1]), i32([1]), torch.zeros((1, width), dtype=torch.int32, device="cuda"), i32([7]),
                     i32([1]), 128, 1, in_place=True)
    assert p.kv_lens.tolist() == [2 ** 31 - 1] and p.slots.tolist() == [-1] and p.free_count.tolist() == [1]


# ---------------------------------------------------------------- attention


def paged(rng, lens, page, kv, dim, spare=2, unused=-1):
    """A cache with those requests' tokens on pages in no order, and their table."""
    need = [-(-n // page) for n in lens]
    host = ref.Cache(sum(need) + spare, kv, dim, page, rng)
    order = rng.permutation(sum(need) + spare)
    table = np.full((len(lens), max(need) + 1), unused, np.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    return host, table


def check_attention(eng, rng, lens, new, heads, kv, dim, page, dtype, window=0, scale=None, tail=0, strided=True):
    host, table = paged(rng, lens, page, kv, dim)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(int)
    (q, _, _), (qn, _, _) = fused(rng, starts[-1] + tail, heads, kv, dim, dtype)
    q = q if strided else q.contiguous()
    args = (q, host.device(torch), i32(table), i32(lens), i32(starts))
    dev = None if scale is None else torch.tensor([scale], dtype=torch.float32, device="cuda")
    want, most, big = ref.attend(qn, host, table, lens, starts, window, scale)
    bound = ref.attend_bound(want, most, big, dtype == "f16")
    for bounds in ({"max_q": max(new), "max_kv": max(lens)}, {}, {"max_q": 1, "max_kv": 1}):
        out = eng.kv8_attention(*args, window=window, scale=dev, **bounds)
        assert out.dtype == q.dtype and out.shape == q.shape
        far = np.abs(out.double().cpu().numpy() - want)
        assert (far <= bound).all(), (bounds, float((far / bound).max()), np.argwhere(~(far <= bound))[:4].tolist())
        assert torch.equal(out, eng.kv8_attention(*args, window=window, scale=dev, **bounds))


HEADS = [(4, 1, 128), (8, 8, 64), (7, 1, 80), (16, 2, 256), (20, 1, 96), (33, 1, 128), (6, 3, 24)]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv,dim", HEADS)
def test_attention_of_single_tokens(eng, heads, kv, dim, page, dtype):
    rng = np.random.default_rng(heads * dim + page)
    lens = [1, 15, 16, 17, 0, 63, 64, 65, 200, 511, 777]
    check_attention(eng, rng, lens, [1] * len(lens), heads, kv, dim, page, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("page,window", [(16, 0), (64, 0), (32, 5), (128, 70)])
@pytest.mark.parametrize("heads,kv,dim", HEADS)
def test_attention_of_a_few_tokens(eng, heads, kv, dim, page, window, dtype):
    """Also requests without tokens, with more tokens than their length, and rows of no request."""
    rng = np.random.default_rng(heads + dim + page)
    check_attention(eng, rng, [3, 90, 64, 2, 300, 40], [3, 2, 0, 5, 7, 1], heads, kv, dim, page, dtype, window, tail=3)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("page,window", [(16, 0), (64, 33), (128, 0)])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 128), (3, 1, 64), (2, 1, 80), (2, 2, 256)])
def test_attention_of_prompts(eng, heads, kv, dim, page, window, dtype):
    rng = np.random.default_rng(dim + page + window)
    check_attention(eng, rng, [150, 333, 70, 129, 65], [150, 70, 1, 129, 17], heads, kv, dim, page, dtype, window, 0.11,
                    tail=2, strided=window == 0)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("lens,heads,kv", [([5000], 4, 1), ([3000, 10], 8, 2), ([2100, 70, 900, 1], 4, 4)])
def test_attention_of_long_caches(eng, lens, heads, kv, dtype):
    rng = np.random.default_rng(sum(lens))
    check_attention(eng, rng, lens, [1] * len(lens), heads, kv, 128, 64, dtype)
    check_attention(eng, rng, lens, [1] * len(lens), heads, kv, 64, 16, dtype, window=1500)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("new", [1, 40])
def test_attention_of_uneven_scales_and_large_queries(eng, new, dtype):
    """Pages whose scales differ by 10^4, queries from tiny to large, scores that leave one token."""
    rng = np.random.default_rng(new)
    host, table = paged(rng, [190, 70], 16, 2, 128)
    host.scales *= np.exp(rng.uniform(-9, 0, host.scales.shape)).astype(np.float32)
    q = (rng.standard_normal((2 * new, 4, 128)) * np.exp(rng.uniform(-9, 4, (2 * new, 4, 1)))).astype(np.float32)
    qd = cuda(q).to(DT[dtype])
    qn, starts = qd.float().cpu().numpy(), [0, new, 2 * new]
    want, _, big = ref.attend(qn, host, table, [190, 70], starts)
    out = eng.kv8_attention(qd, host.device(torch), i32(table), i32([190, 70]), i32(starts)).double().cpu().numpy()
    kv = np.abs(host.values()[0])
    most = np.abs(qn).max(axis=(1, 2))[:, None, None] * kv.max() * 128 / np.sqrt(128)  # of each row
    bound = ref.attend_bound(want, most, big, dtype == "f16")
    assert (np.abs(out - want) <= bound).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("lens,new", [([40, 700, 3], [1, 2, 1]), ([2500], [2]), ([300, 190], [90, 33])])
def test_attention_of_rows_before_the_first_request(eng, lens, new, dtype):
    """q_start need not begin with 0: the rows before it are of no request, and zeros whatever the workspace held."""
    rng = np.random.default_rng(len(lens))
    host, table = paged(rng, lens, 16, 2, 128)
    starts = 5 + np.concatenate([[0], np.cumsum(new)])
    q = cuda(rng.standard_normal((starts[-1] + 3, 8, 128)).astype(np.float32)).to(DT[dtype])
    want, most, big = ref.attend(q.float().cpu().numpy(), host, table, lens, starts)
    bound = ref.attend_bound(want, most, big, dtype == "f16")
    for bounds in ({"max_q": max(new), "max_kv": max(lens)}, {}):
        out = eng.kv8_attention(q, host.device(torch), i32(table), i32(lens), i32(starts), **bounds)
        assert (out[:5] == 0).all() and (out[starts[-1]:] == 0).all()
        assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("lens,new,tokens", [([40, 700, 300], [1, 2, 8], 6), ([300, 190, 500], [90, 33, 70], 140)])
def test_attention_of_requests_that_pass_the_rows(eng, lens, new, tokens):
    """Rows past q's end are not there; those before them keep their positions."""
    rng = np.random.default_rng(tokens)
    host, table = paged(rng, lens, 16, 2, 128)
    starts = np.concatenate([[0], np.cumsum(new)])
    q = rng.standard_normal((starts[-1], 8, 128)).astype(np.float32)
    want, most, big = ref.attend(q, host, table, lens, starts)
    out = eng.kv8_attention(cuda(q)[:tokens], host.device(torch), i32(table), i32(lens), i32(starts))
    assert (np.abs(out.double().cpu().numpy() - want[:tokens]) <= ref.attend_bound(want, most, big, False)).all()


@pytest.mark.parametrize("most", [1, 40])
def test_attention_of_starts_out_of_order(eng, most):
    """No meaning, but nothing outside the buffers is read or written: finite values, and the guard rows untouched."""
    rng = np.random.default_rng(most)
    lens = [100, 800, 40, 300]
    host, table = paged(rng, lens, 16, 2, 128)
    q = cuda(rng.standard_normal((60, 8, 128)).astype(np.float32))
    whole = torch.full((64, 8, 128), 7.0, device="cuda")
    for starts in ([-9, 5, 2, 9, 60], [2 ** 31 - 1, -2 ** 31, 30, -2, 2 ** 31 - 1], [50, 40, 30, 20, 10], [-2 ** 31] * 5):
        out = eng.kv8_attention(q, host.device(torch), i32(table), i32(lens), i32(starts), max_q=most, max_kv=800,
                                out=whole[2:62])
        assert torch.isfinite(out).all() and (whole[:2] == 7).all() and (whole[62:] == 7).all()


def test_attention_with_pages_that_are_not_there(eng):
    """Tokens on pages outside the cache are not seen; a row all of whose pages are missing gives zeros; what lies
    behind a length (any codes, NaN scales, wild table entries) does not matter."""
    rng = np.random.default_rng(4)
    for new in (1, 30):
        host, table = paged(rng, [200, 90, 50], 16, 2, 64, unused=1 << 30)
        host.scales[:, table[0, 12]] = np.nan  # tokens 192 .. 207, cut off by the length below
        table[0, [0, 5]], table[1, :6], table[2, 1] = [-1, 1 << 29], -5, len(host.codes[0])
        lens, starts = [190, 90, 50], [0, new, 2 * new, 3 * new]
        q = rng.standard_normal((3 * new, 4, 64)).astype(np.float32)
        want, most, big = ref.attend(q, host, table, lens, starts)
        out = eng.kv8_attention(cuda(q), host.device(torch), i32(table), i32(lens), i32(starts)).cpu().numpy()
        assert (np.abs(out - want) <= ref.attend_bound(want, most, big, False)).all()
        assert (out[new:2 * new] == 0).all()


def test_attention_shows_a_page_that_is_not_sound(eng):
    """A page whose scale is NaN gives NaN to who sees it, and to nobody else."""
    rng = np.random.default_rng(6)
    host, table = paged(rng, [100, 100, 100], 16, 1, 128)
    host.scales[0, table[0, 2]], host.scales[1, table[1, 6]] = np.nan, np.nan
    for new in (1, 20):
        q = cuda(rng.standard_normal((3 * new, 2, 128)).astype(np.float32))
        out = eng.kv8_attention(q, host.device(torch), i32(table), i32([100] * 3), i32([0, new, 2 * new, 3 * new]))
        assert torch.isnan(out[:new]).all() and torch.isfinite(out[2 * new:]).all()
        assert torch.isnan(out[new:2 * new][-4:]).all()  # the rows that see page 6: tokens 96 to 99
        assert torch.isfinite(out[new:2 * new][:-4]).all()


def test_attention_past_32_bits(eng):
    """Pages that lie more than 2 GiB into the cache."""
    rng = np.random.default_rng(7)
    page, kv, dim = 128, 1, 128
    pages = (1 << 31) // (page * dim) + 3
    host, table = paged(rng, [200], page, kv, dim, spare=0)
    cache = KV8Cache(*(torch.empty(s, dtype=torch.int8, device="cuda") for s in
                       ((pages, kv, page, dim), (pages, kv, dim, page))),
                     *(torch.empty((pages, kv), device="cuda") for _ in range(2)))
    for t, d in zip(cache, host.device(torch)):
        t[-2:] = d
    q = rng.standard_normal((1, 4, dim)).astype(np.float32)
    want, most, big = ref.attend(q, host, table, [200], [0, 1])
    table[table >= 0] += pages - 2
    out = eng.kv8_attention(cuda(q), cache, i32(table), i32([200]), i32([0, 1])).cpu().numpy()
    assert (np.abs(out - want) <= ref.attend_bound(want, most, big, False)).all()
    x = rng.standard_normal((2, 1, 1, dim)).astype(np.float32)
    eng.kv8_append(cuda(x[0]), cuda(x[1]), cache, torch.tensor([(pages - 1) * page + 100], device="cuda"))
    host.append(x, [page + 100])
    for t, d in zip(cache, host.device(torch)):
        assert torch.equal(t[-2:], d)
    keys, _ = eng.kv8_dequant(cache, i32([pages - 1]), dim)
    assert torch.equal(keys[0], cuda((host.codes[0, 1].astype(np.float32) * host.scales[0, 1][:, None, None])))


# ------------------------------------------------------------------- sample


def every_token(eng, z, dtype, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The middle of each kept token's share gives that token, for every one of them at once."""
    zd = cuda(z.astype(np.float32)).to(DT[dtype])
    order, w = ref.kept(zd.double().cpu().numpy(), temperature, top_k, top_p, min_p)
    ids = np.sort(order)
    share = w[ids] / w[ids].sum()
    ids, mid, share = (x[share > 1e-5] for x in (ids, np.cumsum(share) - share / 2, share))
    n = len(ids)
    one = lambda x, t=torch.float32: torch.full((n,), x, dtype=t, device="cuda")  # noqa: E731
    logits = zd.expand(n, -1)
    for rows in (logits, logits.contiguous()):
        tok, lp = eng.sample(rows, cuda(mid.astype(np.float32)), temperature=one(temperature),
                             top_k=one(top_k, torch.int32), top_p=one(top_p), min_p=one(min_p))
        assert tok.dtype == torch.int64 and tok.cpu().numpy().tolist() == ids.tolist()
        # exp of scores up to 30 apart in fp32, sums exact
        assert np.abs(lp.cpu().numpy() - np.log(share)).max() <= 1e-5
    return order, w


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 5003])
def test_sample_gives_every_token_its_share(eng, vocab, dtype):
    rng = np.random.default_rng(vocab)
    z = 2.5 * rng.standard_normal(vocab)
    every_token(eng, z, dtype)
    every_token(eng, z, dtype, temperature=0.6, top_k=7)
    every_token(eng, z, dtype, temperature=1.7, min_p=0.03)
    every_token(eng, z, dtype, top_k=vocab * 2 // 3)
    # a threshold in the middle between two sums: no rounding moves it over one
    zd = cuda(z.astype(np.float32)).to(DT[dtype]).double().cpu().numpy()
    for k, n in ((0, 1), (0, vocab // 2), (40, 12), (40, 30)):
        order, w = ref.kept(zd, 0.9, k)
        if 0 < n < len(order):
            mass = np.cumsum(w[order])
            every_token(eng, z, dtype, 0.9, k, float((mass[n - 1] - w[order[n - 1]] / 2) / mass[-1]), 1e-6)
    order, w = ref.kept(zd, 1.1, vocab * 3 // 4, 1.0, 1e-3)
    mass = np.cumsum(w[order])
    for n in {1, len(order) // 3 + 1, len(order)}:
        every_token(eng, z, dtype, 1.1, vocab * 3 // 4, float((mass[n - 1] - w[order[n - 1]] / 2) / mass[-1]), 1e-3)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_sample_of_equal_logits(eng, dtype):
    """Ties go to the lowest index: top-k and top-p cut inside a run of equal values."""
    z = np.repeat([3.0, 1.0, 3.0, -2.0], 500)
    for k, p in ((1, 1.0), (700, 1.0), (0, 0.3), (900, 0.5001), (0, 0.0)):
        order, w = every_token(eng, z, dtype, 1.0, k, p)
        assert len(order) < 2000
    every_token(eng, np.zeros(4000), dtype, 1.0, 2500, 0.9999)
    every_token(eng, np.zeros(4000), dtype)


def test_sample_special_rows(eng):
    inf, nan = np.inf, np.nan
    z = np.zeros((9, 70), np.float32)
    z[0, 5], z[1], z[2, :69], z[3, [4, 9]] = 2, nan, -inf, inf  # greedy; nothing; one token; two infinities
    z[4, ::2], z[5], z[6, 7], z[7, 3], z[8, 0] = nan, -inf, 1e30, -1e30, 40
    temperature = [0.0, 1.0, 1.0, 1.0, 1.0, 0.0, 1e-30, 1e30, nan]
    u = [0.7, 0.2, 0.5, 0.6, 0.999999, 0.1, 0.3, 0.0, 0.9]
    f = lambda x: torch.tensor(x, dtype=torch.float32, device="cuda")  # noqa: E731
    tok, lp = eng.sample(cuda(z), f(u), temperature=f(temperature))
    assert tok.tolist() == [5, -1, 69, 9, 69, -1, 7, 0, 0]
    assert torch.isnan(lp[[1, 5]]).all()
    want = np.log([1, 1, 1 / 2, 1 / 35, 1, 1 / (69 + np.exp(-1)), 1])
    assert np.abs(lp[[0, 2, 3, 4, 6, 7, 8]].cpu().numpy() - want).max() <= 1e-6
    # u outside [0, 1), settings that are not numbers or out of range: off, or the nearest that is in it
    tok, _ = eng.sample(cuda(np.zeros((6, 8), np.float32)), f([1.0, -1.0, 5.0, nan, 0.5, 0.5]), top_p=f([nan, 2, 1, 1, -3, 1]),
                        min_p=f([nan, -1, 0, 0, 0, 7]), top_k=i32([-4, 9, 0, 0, 0, 3]))
    assert tok.tolist() == [7, 0, 7, 0, 0, 1]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,vocab", [(1, 131072), (3, 50001), (200, 8191), (2, 1 << 20)])
def test_sample_of_many(eng, rows, vocab, dtype):
    """Rows of a large vocabulary with settings of their own, rows apart in memory, against 64 bits."""
    rng = np.random.default_rng(vocab)
    wide = cuda((2 * rng.standard_normal((rows, vocab + 3))).astype(np.float32)).to(DT[dtype])
    wide[:, rng.integers(0, vocab, 30)] += 8
    z = wide[:, 1:vocab + 1]
    t, k = rng.uniform(0.5, 1.3, rows).astype(np.float32), rng.integers(0, 100, rows) * (rng.random(rows) < 0.5)
    p, m = rng.uniform(0.3, 1.2, rows).astype(np.float32), (0.05 * rng.random(rows)).astype(np.float32)
    u, want = np.zeros(rows, np.float32), []
    zn = z.double().cpu().numpy()
    for r in range(rows):
        order, w = ref.kept(zn[r], float(t[r]), int(k[r]), float(p[r]), float(m[r]))
        ids = np.sort(order)
        mass = np.cumsum(w[ids])
        i = int(np.argmax(w[ids] * rng.random(len(ids))))  # one of the likelier ones
        u[r] = (mass[i] - w[ids[i]] / 2) / mass[-1]
        want.append(int(ids[i]))
    args = {"temperature": cuda(t), "top_k": i32(k), "top_p": cuda(p), "min_p": cuda(m)}
    tok, lp = eng.sample(z, cuda(u), **args)
    assert tok.tolist() == want
    again, lp2 = eng.sample(z, cuda(u), **args)
    assert torch.equal(tok, again) and torch.equal(lp, lp2)


# ------------------------------------------------------- streams and graphs


def test_a_step_on_its_own_stream_and_in_a_graph(eng):
    """plan, append, attention and sampling captured together replay as they run, with lengths that change between
    the replays and other work of the engine in between."""
    from ztensor_amd.engine import ROCmEngine

    side = torch.cuda.Stream()
    e = ROCmEngine(stream=side)
    rng = np.random.default_rng(2)
    heads, kv, dim, page, r = 8, 2, 64, 16, 3
    table = rope_table(dim, 400)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        cache = KV8Cache.allocate(64, kv, dim, page)
        lens, new = i32([30, 0, 200]), i32([1, 1, 1])
        blocks = i32(np.where(np.arange(16) < 13, np.arange(48).reshape(3, 16), -1))
        free, count = i32(np.arange(48, 64)), i32([16])
        x = cuda(rng.standard_normal((r, (heads + 2 * kv) * dim)).astype(np.float32))
        logits = cuda(rng.standard_normal((r, 500)).astype(np.float32))
        u = cuda(rng.random(r).astype(np.float32))

        def step():
            q, k, v = (p.view(r, -1, dim) for p in x.split([heads * dim, kv * dim, kv * dim], 1))
            p = e.kv8_plan(lens, new, blocks, free, count, page, r)
            q = e.kv8_append(k, v, cache, p.slots, positions=p.positions, table=table, q=q)
            a = e.kv8_attention(q, cache, p.block_table, p.kv_lens, p.q_start, max_q=1, max_kv=256)
            t, lp = e.sample(logits + a.view(r, -1)[:, :500], u, top_k=i32_k)
            return p.kv_lens, a, t, lp

        i32_k = i32([40, 0, 5])
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
        for i in range(3):
            x.copy_(cuda(rng.standard_normal(x.shape).astype(np.float32)))
            lens += 7
            state = [t.clone() for t in cache]
            want = [t.clone() for t in step()]
            e.kv8_attention(torch.randn(40, heads, dim, device="cuda"), cache, blocks, i32([40, 0, 0]), i32([0, 40, 40, 40]))
            e.sample(torch.randn(300, 9000, device="cuda"), torch.rand(300, device="cuda"))
            torch.cuda.synchronize()
            for t, s in zip(cache, state):
                t.copy_(s)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_engine_arguments(eng):
    t = torch.zeros(4, 2, 64, device="cuda")
    cache = KV8Cache.allocate(3, 2, 64, 16)
    table, pos, slots = rope_table(64, 8), i32([0] * 4), torch.zeros(4, dtype=torch.int64, device="cuda")
    good = dict(positions=pos, table=table)
    for call in (lambda: eng.rope(t.double(), None, pos, table), lambda: eng.rope(t, t.half(), pos, table),
                 lambda: eng.sample(t[0].double(), t[0, :, 0]), lambda: eng.kv8_append(t, t.half(), cache, slots),
                 lambda: eng.kv8_attention(t, cache, i32([[0]]), i32([4]), i32([0, 4]), out=t.half())):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: eng.rope(t, None, pos[:3], table), lambda: eng.rope(t, None, pos.long(), table),
                 lambda: eng.rope(t.cpu(), None, pos, table), lambda: eng.rope(t[:, :, ::2], None, pos, table),
                 lambda: eng.rope(t, None, pos, table.double()), lambda: eng.rope(t, t[:2], pos, table),
                 lambda: eng.kv8_append(t, t, cache, slots.int()), lambda: eng.kv8_append(t, t, cache, slots, table=table),
                 lambda: eng.kv8_append(t[:, :1], t[:, :1], cache, slots, **good),
                 lambda: eng.kv8_append(t, t, cache, slots, q=t), lambda: eng.kv8_append(t, t, cache[:3] + (cache[3][:2],), slots),
                 lambda: eng.kv8_append(t, t[:3], cache, slots), lambda: eng.kv8_dequant(cache, pos.long(), 64),
                 lambda: eng.kv8_dequant(cache, pos, 128), lambda: eng.kv8_dequant((cache.v, cache.k) + cache[2:], pos, 64),
                 lambda: eng.kv8_attention(t, cache, i32([[0]]), i32([4, 4]), i32([0, 4])),
                 lambda: eng.kv8_attention(t[:, :1], cache, i32([[0]]), i32([4]), i32([0, 4])),
                 lambda: eng.kv8_attention(t, cache, i32([[0]]), i32([4]), i32([0, 4]), out=t[:3]),
                 lambda: eng.kv8_plan(pos, pos, pos, pos, pos[:1], 16, 4), lambda: eng.sample(t[0], t[0, :, 0].half()),
                 lambda: eng.sample(t, pos), lambda: eng.sample(t[0], t[0, :, 0].contiguous(), top_k=t[0, :, 0].contiguous())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(_lib.ZTError):
        eng.kv8_plan(pos, pos, i32([[0]] * 4), pos, pos[:1], 24, 4)
    with pytest.raises(_lib.ZTError):
        eng.rope(t, None, pos, rope_table(66, 8))
    with pytest.raises(_lib.ZTError):
        eng.kv8_attention(t, cache, i32([[0]]), i32([4]), i32([0, 4]), window=-1)
    empty = eng.kv8_attention(t[:0], cache, i32([[0]]), i32([0]), i32([0, 0]))
    assert empty.shape == (0, 2, 64) and eng.sample(t[:0, 0], t[:0, 0, 0])[0].shape == (0,)
    assert eng.rope(t[:0], t[:0], pos[:0], table)[1].shape == (0, 2, 64)
    assert eng.kv8_append(t[:0], t[:0], cache, slots[:0]) is None and eng.kv8_dequant(cache, pos[:0], 64)[0].shape == (0, 2, 16, 64)


@pytest.mark.parametrize("new", [1, 24])
def test_attention_of_fp32_rows_holds_22_bits_of_each_weight(eng, new):
    """Small scores, so that the weights' own rounding is all there is: two parts that do not belong together (one
    rounded from the product, the other from its fp32 value) would show as 2^-11 of one weight."""
    rng = np.random.default_rng(new)
    lens = list(rng.integers(new, new + 30, 60))
    host, table = paged(rng, lens, 16, 2, 64)
    starts = list(range(0, 60 * new + 1, new))
    q = (0.01 * rng.standard_normal((60 * new, 8, 64))).astype(np.float32)
    want, most, big = ref.attend(q, host, table, lens, starts)
    out = eng.kv8_attention(cuda(q), host.device(torch), i32(table), i32(lens), i32(starts)).cpu().numpy()
    assert most < 1.5
    assert np.abs(out - want).max() <= ref.attend_bound(0, most, big, False)
