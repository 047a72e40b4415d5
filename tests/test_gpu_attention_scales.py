"""Attention over pages whose scales are far apart, or are of no matter: zero
and tiny scales of values among others, large ones that a row does not see or
gives no weight, against the definition in 64 bits.  Each row, head and dim is
held to a bound of its own, so that small results beside large ones count."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import decode_ref as ref  # noqa: E402
from test_gpu_decode import DT, cuda, eng, i32  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def attend(q, host, table, lens, starts, half, window=0):
    """(result, how far a kernel's may be) in 64 bits.  With p the softmax's weights, v the values and a = sum p |v|:

    scores    operands in 22 bits or more and fp32 sums in chains of at most 16 and 64 terms: each weight's share of
              2^-20 (2 + the row's largest sum of |q k| times the scale), in a and once more in the result (the sum)
    weights   the second product takes them as fp16 (two parts for fp32 rows) times their page's scale, in units of which
              the row's largest, max p scale, is 2^8 or more: what lies below is rounded to steps of 2^-24, and a code is
              at most 127
    fp16      11 bits of each weight, in a and in their sum, and of the result; of the sum besides steps of 2^-24 where
              the unit is 2^4 or more"""
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    kv, group = host.values(), q.shape[1] // host.codes.shape[2]
    scales = host.scales[1].astype(np.float64)
    for r, size in enumerate(lens):
        n = starts[r + 1] - starts[r]
        t = np.arange(size)
        page = table[r, t // host.page]
        t = t[(page >= 0) & (page < host.codes.shape[1])]
        page = table[r, t // host.page]
        k, v, vs = kv[0][page, :, t % host.page], kv[1][page, :, t % host.page], scales[page]
        for i in range(n):
            hi = size - n + i + 1
            see = (t < hi) & (t >= (hi - window if window else 0))
            if not see.any():
                continue
            for h in range(q.shape[1]):
                row, x, y = q[starts[r] + i, h].astype(np.float64), k[see, h // group], v[see, h // group]
                s = x @ row / np.sqrt(q.shape[2])
                most = (np.abs(x) @ np.abs(row)).max() / np.sqrt(q.shape[2])
                p = np.exp(s - s.max())
                p /= p.sum()
                o, a, count = p @ y, p @ np.abs(y), len(p)
                b = 2.0 ** -20 * (2 + most) * (a + np.abs(o)) + count * 127 * 2.0 ** -33 * (p * vs[see, h // group]).max()
                if half:
                    b = b + 2.0 ** -11 * (a + 2 * np.abs(o)) + count * 2.0 ** -28 * np.abs(o) + 2.0 ** -25
                out[starts[r] + i, h], bound[starts[r] + i, h] = o, b
    return out, bound


def paged(rng, lens, page, kv, dim):
    """As the requests' pages in no order; page 0 is nobody's."""
    need = [-(-n // page) for n in lens]
    host = ref.Cache(sum(need) + 1, kv, dim, page, rng)
    order, table = 1 + rng.permutation(sum(need)), np.full((len(lens), max(need) + 1), -1, np.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    return host, table


def check(eng, q, host, table, lens, starts, dtype, **bounds):  # noqa: F811
    qd = cuda(q.astype(np.float32)).to(DT[dtype])
    want, bound = attend(qd.float().cpu().numpy(), host, table, lens, starts, dtype == "f16")
    args = (qd, host.device(torch), i32(table), i32(lens), i32(starts))
    out = eng.kv8_attention(*args, **bounds)
    far = np.abs(out.double().cpu().numpy() - want)
    worst = np.unravel_index(np.argmax(far / (bound + 1e-300)), far.shape)
    assert (far <= bound).all(), (worst, float(far[worst]), float(bound[worst]), float(want[worst]))
    return out


LENS = [190, 70, 333, 25]
SIZES = pytest.mark.parametrize("new", [1, 7, 40])  # one row of a group, a few, more than the first kernel takes
TYPES = pytest.mark.parametrize("dtype", ["f32", "f16"])


def queries(rng, new, heads, dim):
    n = [min(new, size) for size in LENS]
    return rng.standard_normal((sum(n), heads, dim)), np.concatenate([[0], np.cumsum(n)]).astype(int)


@TYPES
@SIZES
@pytest.mark.parametrize("ratio", [0.0, 2.0 ** -5, 2.0 ** -9, 1e-6, 1e-9, 1e-12, 1e-30])
def test_pages_of_small_values_keep_their_weight_in_the_sum(eng, ratio, new, dtype):  # noqa: F811
    """Half of the pages' values are nothing, or nearly, beside those of a request's first page: their tokens' weights
    still divide."""
    rng = np.random.default_rng(new)
    host, table = paged(rng, LENS, 16, 2, 128)
    small = rng.random(host.scales[1].shape) < 0.5
    small[table[:, 0]] = False
    host.scales[1] *= np.where(small, ratio, 1.0).astype(np.float32)
    q, starts = queries(rng, new, 8, 128)
    check(eng, q, host, table, LENS, starts, dtype)
    check(eng, q, host, table, LENS, starts, dtype, max_q=1, max_kv=1)


@TYPES
@SIZES
def test_many_small_weights_in_the_sum(eng, new, dtype):  # noqa: F811
    """One token, and 4000 of 2^-20 of its weight whose values are a hundredth of its page's."""
    rng = np.random.default_rng(3)
    host, table = paged(rng, [4000], 16, 1, 128)
    host.codes[0] = 0
    host.codes[0, table[0, 0], 0, 0] = 127
    host.scales[0] = 20 * np.log(2) * np.sqrt(128) / (127 * 128)
    host.scales[1] = 0.01
    host.scales[1, table[0, 0]] = 1.0
    q = np.ones((new, 4, 128))
    check(eng, q, host, table, [4000], [0, new], dtype)


@TYPES
@SIZES
@pytest.mark.parametrize("ratio", [0.0, 1e-6, 1e-12, 1e-30])
def test_rows_that_see_small_values_only(eng, ratio, new, dtype):  # noqa: F811
    """Half of the pages' values are nothing, or nearly, beside the others': rows beside those that see the others, and
    rows that see the others with little weight, keep the precision of their own."""
    rng = np.random.default_rng(new)
    host, table = paged(rng, LENS, 16, 2, 128)
    host.scales[1] *= np.where(rng.random(host.scales[1].shape) < 0.5, ratio, 1.0).astype(np.float32)
    q, starts = queries(rng, new, 8, 128)
    check(eng, q, host, table, LENS, starts, dtype)
    check(eng, q, host, table, LENS, starts, dtype, max_q=1, max_kv=1)


@TYPES
@SIZES
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 4, 64, 32), (6, 2, 80, 64), (2, 1, 192, 16), (4, 1, 256, 128)])
def test_pages_of_any_scale(eng, heads, kv, dim, page, new, dtype):  # noqa: F811
    """From 1e-18 to 1e3 (fp16 results stay finite), some zero."""
    rng = np.random.default_rng(dim + new)
    host, table = paged(rng, LENS, page, kv, dim)
    shape = host.scales[1].shape
    host.scales[1] = (np.exp(rng.uniform(-41, 5, shape)) * (rng.random(shape) > 0.2)).astype(np.float32)
    q, starts = queries(rng, new, heads, dim)
    check(eng, q, host, table, LENS, starts, dtype)


@TYPES
@SIZES
@pytest.mark.parametrize("large", [1e4, 1e12, 3e38])
def test_pages_of_nobody_do_not_matter(eng, large, new, dtype):  # noqa: F811
    """Lanes past a length, and on pages outside the cache, read page 0: any finite scale there leaves every bit."""
    rng = np.random.default_rng(new)
    host, table = paged(rng, LENS, 16, 2, 128)
    table[2, 3:6] = -1, 1 << 20, len(host.codes[0])
    q, starts = queries(rng, new, 8, 128)
    host.scales[:, 0] = 0
    want = check(eng, q, host, table, LENS, starts, dtype)
    host.scales[:, 0] = large
    assert torch.equal(check(eng, q, host, table, LENS, starts, dtype), want)


@TYPES
@SIZES
def test_tokens_that_a_row_does_not_see_do_not_matter(eng, new, dtype):  # noqa: F811
    """The last tokens' pages hold values 2^40 times the others' (for fp16 rows the others' are as much smaller, so that
    results stay finite): the rows before them are what they were.  With a window, tokens behind it likewise."""
    rng = np.random.default_rng(new)
    small = np.float32(2.0 ** -32) if dtype == "f16" else np.float32(1)
    for window in (0, 40):
        host, table = paged(rng, LENS, 16, 2, 128)
        host.scales[1] *= small
        for r, size in enumerate(LENS):
            host.scales[1, table[r, (size - 1) // 16 if not window else max(0, size - new - window) // 16]] *= np.float32(2.0 ** 40)
        q, starts = queries(rng, new, 8, 128)
        qd = cuda(q.astype(np.float32)).to(DT[dtype])
        want, bound = attend(qd.float().cpu().numpy(), host, table, LENS, starts, dtype == "f16", window)
        out = eng.kv8_attention(qd, host.device(torch), i32(table), i32(LENS), i32(starts), window=window)
        assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()


@TYPES
@SIZES
def test_large_values_of_no_weight(eng, new, dtype):  # noqa: F811
    """A page whose values are 2^40 times the others', and whose tokens weigh about 2^-65 of theirs."""
    rng = np.random.default_rng(new)
    host, table = paged(rng, LENS, 16, 2, 128)
    host.scales[0] *= 0.05
    for r in range(len(LENS)):
        host.codes[0, table[r, 1]] = -127
        host.scales[0, table[r, 1]] = 45 * np.sqrt(128) / (127 * 128)
        host.scales[1, table[r, 1]] = 2.0 ** 40
    q, starts = queries(rng, new, 8, 128)
    check(eng, 1 + 0.01 * q, host, table, LENS, starts, dtype)


@pytest.mark.parametrize("new", [1, 2, 5])
@pytest.mark.parametrize("before", [0, 63, 200])
def test_a_weight_that_is_all_is_one(eng, before, new):  # noqa: F811
    """fp16 rows that see one token, or give the others nothing: its values, rounded once (and fp32 sums), since the
    sum's weight is rounded as the product's is.  The columns beside them have no rows, or rows that see nothing."""
    rng = np.random.default_rng(before)
    host, table = paged(rng, [before + new], 16, 1, 128)
    host.codes[0], host.scales[0] = 0, 0.1
    for i in range(new):  # token before + i answers to value i of a query alone
        host.codes[0, table[0, (before + i) // 16], 0, (before + i) % 16, i] = 127
    q = np.zeros((new, 4, 128))
    for i in range(new):
        q[i, :, i] = 60
    qd = cuda(q.astype(np.float16))
    want, _ = attend(q, host, table, [before + new], [0, new], True)
    out = eng.kv8_attention(qd, host.device(torch), i32(table), i32([before + new]), i32([0, new]))
    far = np.abs(out.double().cpu().numpy() - want)
    assert (far <= np.abs(want) * (2.0 ** -11 + 2.0 ** -18) + 2.0 ** -25).all(), float((far / np.abs(want)).max())
