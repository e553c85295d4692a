"""rn_attend_shared against attention in 64 bits.

Tolerance of a row: with A = scale x the largest sum over d of |q_d k_d| of a key it
sees and B = sum_k p_k |v_k| of the column, the output is off by at most
B (2 ds + dw + dn):
  ds  a score's error: a query enters as two fp16 parts, each cut towards zero (2^-20
      of it together, or 2^-24 of the row's peak), 64 products are added in f32 (at
      most 130 roundings of 2^-24), the scale and the exponent's argument are rounded
      to 2^-24 of values up to A log2(e), 4 times: A (2^-20 + 134 x 1.5 x 2^-24) and
      64 x 2^-24 of scale x peak x the largest |k|; the logarithm L of the value's scale
      is rounded to 2^-23 and enters 4 rounded sums: 6 ln 2 |L| 2^-24;
      it enters a weight and the total: twice;
  dw  a weight's: the exponential (2^-22), the inverse of the value's scale (2^-23), two
      fp16 parts (2^-20);
  dn  f32 sums of n weights and of n products in some order, and the joining of the
      shares: 2 (n + 64) 2^-24.
And by the floor of the weights: weight x value scale, times 2^14 over the largest such
product, are fp16 pairs, whose low part is cut at the step 2^-24 of the smallest numbers,
so each may be off by 2^-38 of the largest one, which is at most the largest scale times
the largest weight; times |code| (fp16: |v|) up to 127, while a row of 64 random codes
holds one above 63, so at most 2 max |v|, over a total of at least the largest weight:
n 2^-36 max |v|.
"""
import numpy as np
import pytest
import torch

import rustyneedle_amd as rn

pytestmark = pytest.mark.gpu
DEV = "cuda"
LOG2E = 1.4426950408889634


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class Held:
    """Keys and values [sequences][kv][capacity][64] of a format, and as doubles."""

    def __init__(self, format, sequences, kv, capacity, rng, spread=1.0):
        shape = (sequences, kv, capacity, 64)
        self.format, self.shape = format, shape
        if format == rn.CACHE_I8:
            self.codes = [torch.from_numpy(rng.integers(-127, 128, shape, dtype=np.int8)).to(DEV) for _ in range(2)]
            self.scales = [torch.from_numpy((0.02 * rng.uniform(0.5, 1.5, shape[:3])
                                             * 2.0 ** rng.uniform(-spread, spread, shape[:3])).astype(np.float32)).to(DEV)
                           for _ in range(2)]
            if spread > 1:
                self.scales[0].fill_(0.02)
        else:
            self.codes = [torch.from_numpy(rng.standard_normal(shape).astype(np.float16)).to(DEV) for _ in range(2)]
            self.scales = [None, None]

    def cache(self):
        s = [None if t is None else t.data_ptr() for t in self.scales]
        return rn.Cache.view(self.format, *self.shape[:3], self.codes[0].data_ptr(), self.codes[1].data_ptr(), *s)

    def log_scale(self, b, h, length):
        """The largest |log2| of a value row's scale."""
        if self.scales[1] is None or not length:
            return 0.0
        return float(torch.log2(self.scales[1][b, h, :length].clamp(min=2.0 ** -100)).abs().max())

    def doubles(self, b, h, length):
        out = []
        for c, s in zip(self.codes, self.scales):
            x = c[b, h, :length].double()
            out.append(x if s is None else x * s[b, h, :length].double()[:, None])
        return out


def attend(q, prefix, prefix_length, own, lengths=None, counts=None, window=0, scale=0.125, out=None, error=None,
           stream=None, fill=7.0):
    n, t, heads, _ = q.shape
    if out is None:
        out = torch.full((n, t, heads, 64), fill, device=DEV)
    p, o = prefix and prefix.cache(), own and own.cache()
    size = rn.attend_shared_workspace(n, t, heads, p, prefix_length, o)
    work = torch.full((max(size, 1),), 0xff, dtype=torch.uint8, device=DEV)  # NaN: it need not be cleared
    torch.cuda.synchronize()
    rn.attend_shared(q.data_ptr(), out.data_ptr(), n, t, heads, p, prefix_length, o,
                     None if lengths is None else lengths.data_ptr(), None if counts is None else counts.data_ptr(),
                     scale, window, work.data_ptr(), size, q.stride(1), out.stride(1),
                     None if error is None else error.data_ptr(), stream)
    torch.cuda.synchronize()
    return out


def check(got, q, prefix, prefix_length, own, lengths=None, counts=None, window=0, scale=0.125, fill=7.0):
    n, t, heads, _ = q.shape
    kv = (prefix or own).shape[1]
    group = heads // kv
    lengths = [own.shape[2] if own else 0] * n if lengths is None else lengths.tolist()
    counts = [t] * n if counts is None else counts.tolist()
    worst = 0.0
    for b in range(n):
        assert (got[b, counts[b]:] == fill).all(), "rows behind the count"
        for h in range(kv):
            parts = []
            if prefix_length:
                parts.append(prefix.doubles(0, h, prefix_length))
            if own:
                parts.append(own.doubles(b, h, lengths[b]))
            k, v = (torch.cat([p[i] for p in parts]) for i in range(2))
            logs = max(prefix.log_scale(0, h, prefix_length) if prefix_length else 0.0,
                       own.log_scale(b, h, lengths[b]) if own else 0.0)
            for i in range(counts[b]):
                end = prefix_length + lengths[b] - counts[b] + i + 1
                first = max(0, end - window) if window else 0
                rows = got[b, i, h * group:(h + 1) * group].double()
                if end <= 0:
                    assert (rows == 0).all()
                    continue
                ks, vs = k[first:end], v[first:end]
                x = q[b, i, h * group:(h + 1) * group].double()
                p = torch.softmax(torch.matmul(x, ks.T) * scale, -1)
                want = torch.matmul(p, vs)
                a = scale * torch.matmul(x.abs(), ks.abs().T).amax(-1, keepdim=True)
                floor = 64 * 2.0 ** -24 * scale * x.abs().amax(-1, keepdim=True) * ks.abs().max()
                ds = a * (2.0 ** -20 + 134 * 1.5 * 2.0 ** -24) + floor + 6 * 0.7 * logs * 2.0 ** -24
                dw = 2.0 ** -22 + 2.0 ** -23 + 2.0 ** -20
                dn = 2 * (end - first + 64) * 2.0 ** -24
                bound = torch.matmul(p, vs.abs()) * (2 * ds + dw + dn) + (end - first) * 2.0 ** -36 * vs.abs().max()
                off = (rows - want).abs()
                assert torch.isfinite(rows).all()
                assert (off <= bound).all(), (b, i, h, float((off / bound).max()))
                worst = max(worst, float((off / bound).max()))
    return worst


def made(rng, n, t, heads, kv, prefix, capacity, formats):
    q = torch.from_numpy(rng.standard_normal((n, t, heads, 64)).astype(np.float32)).to(DEV)
    p = Held(formats[0], 1, kv, prefix + 3, rng) if prefix else None
    o = Held(formats[1], n, kv, capacity, rng) if capacity else None
    return q, p, o


I8, F16 = rn.CACHE_I8, rn.CACHE_F16


@pytest.mark.parametrize("formats", [(I8, I8), (F16, F16), (F16, I8), (I8, F16)])
@pytest.mark.parametrize("n,t,heads,kv,prefix,capacity", [
    (1, 1, 1, 1, 0, 1), (1, 1, 1, 1, 1, 1), (2, 1, 3, 1, 63, 64), (3, 1, 4, 2, 64, 65), (4, 1, 8, 8, 65, 63),
    (5, 1, 12, 4, 300, 130), (1, 1, 8, 8, 1000, 700), (17, 1, 4, 2, 257, 40), (40, 1, 2, 1, 513, 90),
    (70, 1, 4, 4, 200, 33), (140, 1, 2, 2, 129, 17), (33, 1, 4, 1, 64, 300), (2, 1, 64, 1, 190, 70),
    (600, 1, 1, 1, 70, 20), (3, 1, 6, 3, 0, 1500)])
def test_one_query(n, t, heads, kv, prefix, capacity, formats):
    rng = np.random.default_rng(n * 7 + prefix)
    q, p, o = made(rng, n, t, heads, kv, prefix, capacity, formats)
    lengths = rng.integers(1, capacity + 1, n)
    lengths[0] = capacity
    if n > 2:
        lengths[1], lengths[2] = 0, 1
    lengths = ints(lengths)
    got = attend(q, p, prefix, o, lengths)
    check(got, q, p, prefix, o, lengths)
    assert torch.equal(got, attend(q, p, prefix, o, lengths)), "the same call twice"


@pytest.mark.parametrize("format", [I8, F16])
@pytest.mark.parametrize("window", [0, 1, 5, 64, 100])
@pytest.mark.parametrize("n,t,heads,kv,prefix,capacity", [
    (3, 2, 2, 1, 100, 70), (4, 5, 12, 4, 200, 130), (2, 9, 8, 4, 0, 65), (6, 17, 2, 2, 65, 40), (2, 40, 4, 1, 130, 200),
    (30, 5, 3, 1, 64, 64)])
def test_drafted_queries(n, t, heads, kv, prefix, capacity, window, format):
    rng = np.random.default_rng(t + window)
    q, p, o = made(rng, n, t, heads, kv, prefix, capacity, (format, format))
    counts = rng.integers(0, t + 1, n)
    counts[0] = t
    lengths = np.minimum(capacity, counts + rng.integers(0, capacity, n))
    lengths[1] = 0  # the queries are the last positions of the prefix
    lengths, counts = ints(lengths), ints(counts)
    got = attend(q, p, prefix, o, lengths, counts, window)
    check(got, q, p, prefix, o, lengths, counts, window)


@pytest.mark.parametrize("formats", [(I8, I8), (F16, F16), (F16, I8), (I8, F16)])
@pytest.mark.parametrize("window", [0, 1100, 150])
@pytest.mark.parametrize("n,t,heads,kv", [
    (1, 1, 2, 2), (1, 3, 4, 4), (1, 7, 2, 2), (5, 1, 4, 2), (1, 12, 2, 2), (20, 1, 2, 2), (2, 10, 2, 2), (1, 30, 1, 1), (40, 1, 2, 2),
    (4, 12, 3, 3), (2, 30, 2, 2), (70, 1, 4, 4), (6, 12, 2, 2), (4, 33, 2, 2), (9, 1, 64, 1), (130, 1, 16, 8)])
def test_a_prefix_shared_by_few_and_many_rows(n, t, heads, kv, window, formats):
    """A prefix that is split over blocks, beside own caches: 1 to 576 rows of it a key head,
    1 to 64 of an own cache."""
    rng = np.random.default_rng(n + t)
    prefix, capacity = 1133, 150
    q, p, o = made(rng, n, t, heads, kv, prefix, capacity, formats)
    lengths = rng.integers(0, capacity + 1, n)
    lengths[0] = capacity
    if n > 2:
        lengths[1], lengths[2] = 0, 1
    lengths, counts = ints(lengths), ints(rng.integers(0, t + 1, n) if t > 1 and n > 1 else [t] * n)
    got = attend(q, p, prefix, o, lengths, counts, window)
    check(got, q, p, prefix, o, lengths, counts, window)
    assert torch.equal(got, attend(q, p, prefix, o, lengths, counts, window)), "the same call twice"


@pytest.mark.parametrize("format", [I8, F16])
def test_windows_wider_than_everything(format):
    rng = np.random.default_rng(21)
    for prefix in (40, 1200):
        q, p, o = made(rng, 3, 2, 4, 2, prefix, 90, (format, format))
        lengths = ints([90, 0, 31])
        want = attend(q, p, prefix, o, lengths)
        for window in (prefix + 90, 1 << 26, 2 ** 31 - 1):
            got = attend(q, p, prefix, o, lengths, None, window)
            check(got, q, p, prefix, o, lengths, None, window)
            if window > 1 << 26:
                assert torch.equal(got, want)


@pytest.mark.parametrize("format", [I8, F16])
def test_prefix_alone_and_own_alone(format):
    rng = np.random.default_rng(3)
    for n, t, prefix in ((1, 1, 1), (4, 1, 700), (2, 6, 4), (90, 1, 333)):
        q, p, _ = made(rng, n, t, 4, 2, prefix, 0, (format, format))
        check(attend(q, p, prefix, None), q, p, prefix, None)
    q, _, o = made(rng, 5, 2, 4, 2, 0, 77, (format, format))
    check(attend(q, None, 0, o), q, None, 0, o)  # every sequence full


def test_nothing_to_see_gives_zeros():
    """An empty prefix without own caches, and own caches of no rows."""
    rng = np.random.default_rng(23)
    q, p, o = made(rng, 3, 2, 4, 2, 20, 30, (I8, I8))
    assert (attend(q, p, 0, None) == 0).all()
    assert (attend(q, None, 0, o, ints([0, 0, 0])) == 0).all()
    assert (attend(q, p, 0, o, ints([0, 0, 0])) == 0).all()
    got = attend(q, p, 1, o, ints([0, 0, 0]))  # the first query stands before the first position
    assert (got[:, 0] == 0).all()
    check(got, q, p, 1, o, ints([0, 0, 0]))


@pytest.mark.parametrize("format", [I8, F16])
@pytest.mark.parametrize("prefix", [0, 100, 1500])
def test_a_prompt_in_one_call(prefix, format):
    """Hundreds of queries a sequence, each seeing up to its own position."""
    rng = np.random.default_rng(24)
    q, p, o = made(rng, 2, 333, 4, 2, prefix, 400, (format, format))
    lengths, counts = ints([400, 200]), ints([333, 200])
    got = attend(q, p, prefix, o, lengths, counts)
    check(got, q, p, prefix, o, lengths, counts)


@pytest.mark.parametrize("format", [I8, F16])
def test_long_prefix_and_a_long_own_cache(format):
    rng = np.random.default_rng(5)
    q, p, o = made(rng, 20, 1, 4, 2, 9001, 3000, (format, format))
    lengths = ints(rng.integers(0, 3001, 20))
    check(attend(q, p, 9001, o, lengths), q, p, 9001, o, lengths)


@pytest.mark.parametrize("format", [I8, F16])
@pytest.mark.parametrize("size", [1e-42, 1e-30, 1e-4, 30.0, 3000.0])
def test_queries_of_any_size(size, format):
    """Tiny ones weigh all positions alike, huge ones pick one; a row of zeros among them."""
    rng = np.random.default_rng(6)
    q, p, o = made(rng, 6, 1, 4, 2, 150, 90, (format, format))
    q *= size
    q[2] = 0
    q[3, 0, 1, 5] = size * 1000
    lengths = ints([90, 3, 50, 64, 65, 0])
    check(attend(q, p, 150, o, lengths), q, p, 150, o, lengths)


@pytest.mark.parametrize("format", [I8, F16])
@pytest.mark.parametrize("prefix", [100, 1400])
@pytest.mark.parametrize("n,t,heads", [(3, 1, 4), (20, 1, 12), (6, 3, 4)])
def test_a_query_that_is_not_finite_stays_alone(n, t, heads, prefix, format):
    rng = np.random.default_rng(25)
    q, p, o = made(rng, n, t, heads, 2, prefix, 60, (format, format))
    lengths = ints([60] * n)
    clean = attend(q, p, prefix, o, lengths)
    for value in (float("nan"), float("inf")):
        bad = q.clone()
        bad[1, 0, 1, 7] = value
        got = attend(bad, p, prefix, o, lengths)
        assert torch.isnan(got[1, 0, 1]).all()
        rest = torch.ones((n, t, heads), dtype=torch.bool, device=DEV)
        rest[1, 0, 1] = False
        assert torch.equal(got[rest], clean[rest])


@pytest.mark.parametrize("format", [I8, F16])
def test_offsets_past_32_bits(format):
    """Sequences that lie more than 2^32 bytes apart."""
    rng = np.random.default_rng(26)
    apart, n, kv, capacity = (1 << 26) + 3, 2, 2, 50
    q, p, o = made(rng, n, 1, 4, kv, 70, capacity, (format, format))
    rows = apart + kv * capacity
    codes = [torch.empty((rows, 64), dtype=o.codes[0].dtype, device=DEV) for _ in range(2)]
    scales = [None if x is None else torch.empty((rows,), device=DEV) for x in o.scales]
    for b in range(n):
        here = slice(b * apart, b * apart + kv * capacity)
        for i in range(2):
            codes[i][here] = o.codes[i][b].reshape(-1, 64)
            if scales[i] is not None:
                scales[i][here] = o.scales[i][b].reshape(-1)
    view = rn.Cache.view(format, n, kv, capacity, codes[0].data_ptr(), codes[1].data_ptr(),
                         *[None if x is None else x.data_ptr() for x in scales], apart, capacity)
    lengths = ints([50, 31])
    want = [attend(q, a, 70 if a else 0, o, lengths) for a in (p, None)]
    o.cache = lambda: view
    for a, w in zip((p, None), want):
        got = attend(q, a, 70 if a else 0, o, lengths)
        check(got, q, a, 70 if a else 0, o, lengths)
        assert torch.equal(got, w)


@pytest.mark.parametrize("prefix", [400, 1400])
def test_value_scales_of_any_size(prefix):
    """Value rows whose scales differ by many powers of two, growing and falling; zero rows."""
    rng = np.random.default_rng(7)
    for spread in (8.0, 40.0):
        q, _, _ = made(rng, 4, 1, 4, 2, 0, 0, (I8, I8))
        p, o = Held(I8, 1, 2, prefix, rng, spread), Held(I8, 4, 2, 300, rng, spread)
        p.scales[1][0, 0] = torch.sort(p.scales[1][0, 0]).values
        p.scales[1][0, 1] = torch.sort(p.scales[1][0, 1], descending=True).values
        o.scales[1][1] = 0.0
        lengths = ints([300, 130, 1, 257])
        check(attend(q, p, prefix, o, lengths), q, p, prefix, o, lengths)


@pytest.mark.parametrize("prefix", [100, 1400])
@pytest.mark.parametrize("n,t", [(3, 1), (3, 7), (12, 2)])
def test_value_scales_that_are_none(n, t, prefix):
    """Scales below 2^-100 are 0, whatever the codes; negative, infinite ones and NaN make
    their own rows' outputs NaN and no others, where they are not seen nothing."""
    rng = np.random.default_rng(22)
    q, p, o = made(rng, n, t, 4, 2, prefix, 80, (I8, I8))
    lengths = ints([80] + [50] * (n - 1))
    p.scales[1][0, 0, 5:70] = 0.0
    p.scales[1][0, 1, 7] = 2.0 ** -101
    o.scales[1][0, 0, 3:9] = 2.0 ** -120
    o.scales[1][1, 1, :] = 0.0
    got = attend(q, p, prefix, o, lengths)
    for held in (p, o):
        held.scales[1][held.scales[1] < 2.0 ** -100] = 0.0
    assert torch.equal(got, attend(q, p, prefix, o, lengths))
    check(got, q, p, prefix, o, lengths)
    for value in (-0.02, float("inf"), -float("inf"), float("nan")):
        o.scales[1][0, 1, 79] = value   # the last position of sequence 0: its last query's alone
        o.scales[1][1, 0, 50:] = value  # behind the length
        p.scales[1][0, 1, prefix] = value
        bad = attend(q, p, prefix, o, lengths)
        assert torch.isnan(bad[0, t - 1, 2:]).all()
        rest = torch.ones((n, t, 4), dtype=torch.bool, device=DEV)
        rest[0, t - 1, 2:] = False
        assert torch.equal(bad[rest], got[rest])


@pytest.mark.parametrize("format", [I8, F16])
@pytest.mark.parametrize("prefix", [200, 1300])
@pytest.mark.parametrize("heads", [4, 12, 44])
def test_what_is_not_seen_does_not_matter(heads, prefix, format):
    """NaN and infinities behind a sequence's length, before a window and in drafted
    positions after a query: the rows that do not see them are as without them, and
    those that do are NaN or infinite."""
    rng = np.random.default_rng(8)
    n, t, kv, capacity = 3, 3, 2, 100
    q, p, o = made(rng, n, t, heads, kv, prefix, capacity, (format, format))
    lengths, counts, window = ints([60, 80, 3]), ints([3, 3, 2]), 90
    clean = attend(q, p, prefix, o, lengths, counts, window)
    check(clean, q, p, prefix, o, lengths, counts, window)

    def spoil(held, b, h, at, value):
        for c, s in zip(held.codes, held.scales):
            if s is None:
                c[b, h, at] = value
            else:
                s[b, h, at] = value

    for value in (float("nan"), float("inf"), -float("inf")):
        pp, oo = Held(format, 1, kv, prefix + 3, rng), Held(format, n, kv, capacity, rng)
        for a, b in ((pp, p), (oo, o)):
            a.codes = [x.clone() for x in b.codes]
            a.scales = [x if x is None else x.clone() for x in b.scales]
        spoil(pp, 0, 0, prefix, value)          # behind the prefix
        spoil(pp, 0, 1, 10, value)              # before every window
        spoil(oo, 0, 0, slice(60, 100), value)  # behind the length
        spoil(oo, 1, 1, 79, value)              # the last drafted token: only the last query sees it
        spoil(oo, 2, 0, 2, value)
        got = attend(q, pp, prefix, oo, lengths, counts, window)
        sees = torch.zeros((n, t, heads), dtype=torch.bool, device=DEV)
        sees[1, 2, heads // 2:] = True
        sees[2, 1, :heads // 2] = True
        assert torch.equal(got[~sees], clean[~sees])
        assert (~torch.isfinite(got[sees])).any(-1).all()


def test_values_alone_that_are_not_finite():
    """An infinite fp16 value with a weight: its column is infinite, the others are not touched;
    in tiles that some rows do not see, too."""
    rng = np.random.default_rng(9)
    for lengths in ([64, 64], [70, 40]):
        q, _, o = made(rng, 2, 2, 2, 1, 0, 70, (F16, F16))
        o.codes[1][0, 0, lengths[0] - 1, 5] = float("inf")
        o.codes[1][1, 0, 3, 9] = float("-inf")
        got = attend(q, None, 0, o, ints(lengths))
        finite = torch.isfinite(got)
        want = torch.ones_like(finite)
        want[0, 1, :, 5] = False
        want[1, :, :, 9] = False
        assert torch.equal(finite, want)
        assert (got[0, 1, :, 5] == float("inf")).all() and (got[1, :, :, 9] == float("-inf")).all()


def test_bad_numbers_give_nan_in_their_sequence_alone():
    rng = np.random.default_rng(10)
    for prefix in (0, 50, 1000):
        for capacity in (40, 0):
            if not prefix and not capacity:
                continue
            q, p, o = made(rng, 5, 2, 4, 2, prefix, capacity, (I8, I8))
            lengths = ints([10, -1, 41, 40, 5]) if capacity else None
            counts = ints([2, 2, 1, 3, -1])
            error = ints([0])
            got = attend(q, p, prefix, o, lengths, counts, error=error)
            assert error.item() == rn.RN_ERR_ARGUMENT
            bad = [False, capacity > 0, capacity > 0, True, True]
            for b in range(5):
                if bad[b]:
                    assert torch.isnan(got[b]).all(), b
                else:
                    one = lengths[b:b + 1] if capacity else None
                    mine = Held(I8, 1, 2, max(capacity, 1), rng)
                    if capacity:
                        mine.codes = [x[b:b + 1] for x in o.codes]
                        mine.scales = [x[b:b + 1] for x in o.scales]
                    check(got[b:b + 1], q[b:b + 1], p, prefix, mine if capacity else None, one, counts[b:b + 1])
            error.zero_()
            attend(q, p, prefix, o, ints([2] * 5) if capacity else None, None, error=error)
            assert error.item() == 0


def test_strides_of_rows_and_caches():
    """Queries inside the fused q/k/v rows of a product, outputs with a gap, caches of
    one layer inside a batch's arena."""
    rng = np.random.default_rng(11)
    n, t, heads, kv = 4, 2, 4, 2
    fused = torch.from_numpy(rng.standard_normal((n, t, heads + 2 * kv, 64)).astype(np.float32)).to(DEV)
    q = fused[:, :, :heads]
    out = torch.full((n, t, heads + 1, 64), 3.0, device=DEV)
    arena = Held(F16, n, 3 * kv, 80, rng)  # [sequence][layer][head]
    layer = Held(F16, n, kv, 80, rng)
    layer.codes = [x[:, kv:2 * kv] for x in arena.codes]
    view = rn.Cache.view(F16, n, kv, 80, layer.codes[0].data_ptr(), layer.codes[1].data_ptr(), None, None,
                         3 * kv * 80, 80)
    layer.cache = lambda: view
    lengths = ints([80, 2, 33, 64])
    attend(q, None, 0, layer, lengths, out=out)
    check(out[:, :, :heads], q, None, 0, layer, lengths)
    assert (out[:, :, heads] == 3.0).all()


def test_own_stream_two_graphs_and_changed_lengths():
    """Two captured graphs with a workspace each, replayed on two streams at once with
    other lengths and queries every time, against eager calls."""
    rng = np.random.default_rng(12)
    calls = []
    for n, t, heads, kv, prefix, capacity in ((6, 1, 8, 8, 300, 90), (3, 4, 12, 4, 70, 200), (6, 1, 8, 8, 2000, 90),
                                             (5, 4, 12, 4, 1500, 200)):
        q, p, o = made(rng, n, t, heads, kv, prefix, capacity, (I8, I8))
        lengths, out = ints([t] * n), torch.zeros_like(q)
        size = rn.attend_shared_workspace(n, t, heads, p.cache(), prefix, o.cache())
        work = torch.zeros((size,), dtype=torch.uint8, device=DEV)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        pc, oc = p.cache(), o.cache()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            rn.attend_shared(q.data_ptr(), out.data_ptr(), n, t, heads, pc, prefix, oc, lengths.data_ptr(), None,
                             0.125, 0, work.data_ptr(), size, stream=stream.cuda_stream)
        calls.append((q, p, o, prefix, capacity, lengths, out, work, stream, graph))
    for step in range(5):
        for q, p, o, prefix, capacity, lengths, out, work, stream, graph in calls:
            q.copy_(torch.from_numpy(rng.standard_normal(q.shape).astype(np.float32)))
            lengths.copy_(ints(rng.integers(q.shape[1], capacity + 1, q.shape[0])))
            out.zero_()
        torch.cuda.synchronize()
        for call in calls:
            with torch.cuda.stream(call[8]):
                call[9].replay()
        torch.cuda.synchronize()
        for q, p, o, prefix, capacity, lengths, out, work, stream, graph in calls:
            assert torch.equal(out, attend(q, p, prefix, o, lengths)), step


def test_pointers_that_are_no_device_memory_are_refused():
    rng = np.random.default_rng(13)
    q, p, o = made(rng, 2, 1, 4, 2, 20, 10, (I8, I8))
    out, lengths = torch.zeros_like(q), ints([1, 2])
    size = rn.attend_shared_workspace(2, 1, 4, p.cache(), 20, o.cache())
    work = torch.zeros((size + 256,), dtype=torch.uint8, device=DEV)
    host = np.zeros((1024,), np.float32)
    at = (host.ctypes.data + 255) & ~255
    good = dict(q=q.data_ptr(), out=out.data_ptr(), workspace=work.data_ptr(), lengths=lengths.data_ptr())

    def call(**wrong):
        a = dict(good, **wrong)
        rn.attend_shared(a["q"], a["out"], 2, 1, 4, p.cache(), 20, o.cache(), a["lengths"], None, 0.125, 0,
                         a["workspace"], size)

    call()
    torch.cuda.synchronize()
    for wrong in (dict(q=at), dict(out=at), dict(workspace=at), dict(lengths=at), dict(q=q.data_ptr() + 4),
                  dict(workspace=work.data_ptr() + 16)):
        with pytest.raises(rn.RnError) as e:
            call(**wrong)
        assert e.value.code == rn.RN_ERR_ARGUMENT, wrong


def test_a_sessions_cache_is_the_prefix(tiny_config, tiny_weights):
    """Sessions' and batches' own caches in place: one query a head over a session's
    layer equals rn_attend_heads over the downloaded cache, within the tolerance of
    both; a Needle 3 session's int8 cache likewise against its codes."""
    from rustyneedle_amd import needle3
    rng = np.random.default_rng(14)
    session = rn.Model(tiny_config, tiny_weights).session(96)
    session.feed(rng.integers(0, tiny_config["vocab"], 70))
    keys, values = session.get_cache(70)
    heads = tiny_config["heads"]
    q = torch.from_numpy(rng.standard_normal((3, 1, heads, 64)).astype(np.float32)).to(DEV)
    for layer in range(tiny_config["layers"]):
        held = Held(F16, 1, heads, 70, rng)
        held.codes = [torch.from_numpy(x[layer].copy()).to(DEV).reshape(1, heads, 70, 64) for x in (keys, values)]
        want = held.cache
        view = session.layer_cache(layer)
        held.cache = lambda: view
        got = attend(q, held, 70, None)
        check(got, q, held, 70, None)
        held.cache = want
        assert torch.equal(got, attend(q, held, 70, None))
    model = needle3.Model(needle3.synthetic_archive(needle3.NEEDLE3_SMALL))
    s3 = model.session(64)
    s3.feed(rng.integers(0, 512, 50).astype(np.uint32))
    k, ks, v, vs = s3.cache(1)
    kv = k.shape[1]
    held = Held(I8, 1, kv, 50, rng)
    held.codes = [torch.from_numpy(np.ascontiguousarray(x.transpose(1, 0, 2))[None]).to(DEV) for x in (k, v)]
    held.scales = [torch.from_numpy(x[None].copy()).to(DEV) for x in (ks, vs)]
    view = s3.layer_cache(1)
    want = held.cache
    held.cache = lambda: view
    q = torch.from_numpy(rng.standard_normal((2, 1, 2 * kv, 64)).astype(np.float32)).to(DEV)
    got = attend(q, held, 50, None)
    check(got, q, held, 50, None)


def test_a_batchs_caches_are_the_own_ones(tiny_config, tiny_weights):
    rng = np.random.default_rng(15)
    model = rn.Model(tiny_config, tiny_weights)
    layers, heads = tiny_config["layers"], tiny_config["heads"]
    batch = rn.Batch(model, 3, 40)
    lengths = [5, 40, 17]
    filled = [[rng.standard_normal((layers, heads, n, 64)).astype(np.float16) for _ in range(2)] for n in lengths]
    for b, (k, v) in enumerate(filled):
        batch.set_cache(b, k, v)
    q = torch.from_numpy(rng.standard_normal((3, 1, heads, 64)).astype(np.float32)).to(DEV)
    view = batch.layer_cache(1)
    held = Held(F16, 3, heads, 40, rng)
    for b, pair in enumerate(filled):
        for c, x in zip(held.codes, pair):
            c[b, :, :lengths[b]] = torch.from_numpy(x[1]).to(DEV)
    held.cache = lambda: view
    check(attend(q, None, 0, held, ints(lengths)), q, None, 0, held, ints(lengths))
