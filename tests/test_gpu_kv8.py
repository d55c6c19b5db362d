"""The 8-bit cache's operators on the device against their plain 64-bit forms."""
import numpy as np
import pytest

import lowbits as L

pytestmark = pytest.mark.gpu


class Device:
    """A host cache's pages on the device."""

    def __init__(self, hip, c):
        self.hip, self.c = hip, c
        self.bufs = [hip.DeviceBuffer.from_numpy(a) for a in (c.k, c.v, c.ks, c.vs)]
        self.cache = hip.KV8Cache(*self.bufs, c.pages, c.heads, c.page, c.dim)

    def batch(self, table, lens, starts, max_new=None, max_len=None):
        width = max([len(r) for r in table] + [1])
        t = np.full((len(table), width), -1, np.int32)
        for i, r in enumerate(table):
            t[i, :len(r)] = r
        self.idx = [self.hip.DeviceBuffer.from_numpy(np.asarray(a, np.int32)) for a in (t, lens, starts)]
        n = max([b - a for a, b in zip(starts, starts[1:])] + [0])
        return self.hip.KV8Batch(self.idx[0], width, self.idx[1], self.idx[2], len(lens),
                                 n if max_new is None else max_new, max(lens) if max_len is None else max_len)

    def pull(self):
        c = self.c
        return [b.download(np.uint8, a.shape) for b, a in zip(self.bufs, (c.k, c.v, c.ks, c.vs))]

    def free(self):
        for b in self.bufs + getattr(self, "idx", []):
            b.free()


def cast(x, dtype):
    return L.bf16_bits(x) if dtype == "bf16" else np.ascontiguousarray(x, np.float32)


def value(x, dtype):
    return L.bf16_value(x) if dtype == "bf16" else x


def layout(rng, page, lens, pages=None):
    """Page ids of each sequence, shuffled, and the number of pages."""
    need = [-(-max(n, 0) // page) for n in lens]
    total = sum(need) + 2 if pages is None else pages
    ids = rng.permutation(total)
    out, at = [], 0
    for n in need:
        out.append([int(i) for i in ids[at:at + n]])
        at += n
    return out, total


def put(hip, d, table, lens, starts, k, v, dtype, ld=0):
    b = d.batch(table, lens, starts)
    with hip.DeviceBuffer.from_numpy(k) as dk, hip.DeviceBuffer.from_numpy(v) as dv:
        hip.kv8_append(d.cache, b, dk, dv, dtype=dtype, k_ld=ld, v_ld=ld)
        hip.synchronize()


def same(got, c):
    for name, g, w in zip(("k", "v", "ks", "vs"), got, (c.k, c.v, c.ks, c.vs)):
        if name in ("k", "v"):  # a NaN's sign is not held
            g, w = np.where(g & 127 == 127, 127, g), np.where(w & 127 == 127, 127, w)
        np.testing.assert_array_equal(g, w, err_msg=name)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page,dim,heads", [(16, 64, 1), (32, 96, 3), (64, 128, 8), (128, 256, 2), (256, 64, 5)])
def test_append_in_steps(hip, page, dim, heads, dtype):
    """A prompt, single tokens, a chunk: every code and scale as the plain form has it, other bytes untouched."""
    rng = np.random.default_rng(page + dim)
    total = [page * 2 + 5, 1, 3 * page, page + 1]
    table, pages = layout(rng, page, [t + 2 * page for t in total])
    c = L.Cache(pages, heads, page, dim, rng)
    d = Device(hip, c)
    lens = [0] * 4
    for step, news in enumerate([total, [1, 1, 1, 1], [1, 0, 1, 1], [page - 2, 5, page + 3, 1], [1, 1, 1, 1]]):
        lens = [a + n for a, n in zip(lens, news)]
        starts = [0] + list(np.cumsum(news))
        size = np.exp2(rng.integers(-4 + step, 4 + 2 * step, (starts[-1], heads, 1)))  # scales grow on the way
        k, v = (cast(rng.standard_normal((starts[-1], heads, dim)) * size, dtype) for _ in range(2))
        put(hip, d, table, lens, starts, k, v, dtype)
        c.append(table, lens, starts, value(k, dtype), value(v, dtype))
        same(d.pull(), c)
    d.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_special_values_and_ties(hip, dtype):
    """Infs and NaNs (stored as NaN, out of the scale), zeros, subnormals, exact ties, the largest finite values."""
    rng = np.random.default_rng(3)
    c = L.Cache(3, 2, 16, 64, rng)
    d = Device(hip, c)
    k = rng.standard_normal((40, 2, 64)).astype(np.float32)
    k[0, 0, 3], k[1, 1, 5], k[20, 0, 7] = np.inf, -np.inf, np.nan
    k[2:10] = rng.choice([1.0625, 1.1875, 17, 19, 448, -464, 2.0 ** -10, 3 * 2.0 ** -10, 0, -0.0], (8, 2, 64))
    v = np.zeros((40, 2, 64), np.float32)
    v[16:32] = rng.standard_normal((16, 2, 64)) * 3e38 / 6
    v[32:] = 1e-40
    k, v = cast(k, dtype), cast(v, dtype)
    put(hip, d, [[2, 0, 1]], [40], [0, 40], k, v, dtype)
    c.append([[2, 0, 1]], [40], [0, 40], value(k, dtype), value(v, dtype))
    same(d.pull(), c)
    # one large token: the last page's earlier codes are rounded again, its NaN stays
    k1 = cast(np.full((1, 2, 64), 1e4), dtype)
    put(hip, d, [[2, 0, 1]], [41], [0, 1], k1, k1, dtype)
    c.append([[2, 0, 1]], [41], [0, 1], value(k1, dtype), value(k1, dtype))
    same(d.pull(), c)
    d.free()


def test_append_skips_absent_pages_and_short_sequences(hip):
    rng = np.random.default_rng(4)
    c = L.Cache(4, 1, 16, 64, rng)
    d = Device(hip, c)
    table, lens, starts = [[3, -1, 1], [99, 0], [2]], [40, 20, 3], [0, 40, 60, 68]  # the last: 8 rows, 3 tokens
    k, v = (rng.standard_normal((68, 1, 64)).astype(np.float32) for _ in range(2))
    put(hip, d, table, lens, starts, k, v, "f32")
    c.append(table, lens, starts, k, v)
    same(d.pull(), c)
    d.free()


def test_append_again_changes_nothing_and_strides(hip):
    rng = np.random.default_rng(5)
    c = L.Cache(4, 2, 32, 64, rng)
    d = Device(hip, c)
    wide = rng.standard_normal((70, 3 * 128 + 1)).astype(np.float32)  # rows of a stacked projection, odd stride
    flat = wide[:, :128].reshape(70, 2, 64)
    b = d.batch([[3, 0, 2]], [70], [0, 70])
    with hip.DeviceBuffer.from_numpy(wide) as w:
        for _ in range(2):
            hip.kv8_append(d.cache, b, w, w, k_ld=385, v_ld=385)
    hip.synchronize()
    c.append([[3, 0, 2]], [70], [0, 70], flat, flat)
    same(d.pull(), c)
    d.free()


# ---- attention -----------------------------------------------------------------------------

def attend(hip, d, table, lens, starts, q, dtype, scale, window, max_len=None, ld=0):
    b = d.batch(table, lens, starts, max_len=max_len)
    with hip.DeviceBuffer.from_numpy(q) as dq, hip.DeviceBuffer.from_numpy(np.full(q.size + 16, 7, q.dtype)) as do:
        hip.kv8_attend(d.cache, b, dq, do, q.shape[1], dtype=dtype, scale=scale, window=window, q_ld=ld)
        hip.synchronize()
        out = do.download(q.dtype, (q.size + 16,))
    assert (out[q.size:] == 7).all()
    return value(out[:q.size].reshape(q.shape), dtype)


def check_attend(got, want, vmax, cond, dtype):
    """Scores are off by at most 16 roundings (2^-24) of the sum of their products' magnitudes, the exponential by 2
    units and its argument's rounding, each weight therefore by a factor within 1 + e, e = 2^-20 (1 + cond); an output
    is a weighted mean of V, off by at most 2 e of the largest.  bf16: weights and output are rounded to 8 bits."""
    e = 2.0 ** -20 * (1 + cond)
    bound = (2 * e + (2.0 ** -7 if dtype == "bf16" else 2.0 ** -19)) * vmax
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    off = np.abs(np.where(np.isnan(want), 0, got) - np.where(np.isnan(want), 0, want))
    assert (off <= bound[..., None]).all(), float((off / np.maximum(bound[..., None], 1e-300)).max())


def filled(hip, rng, page, heads, dim, lens, size=1.0):
    table, pages = layout(rng, page, lens)
    c = L.Cache(pages, heads, page, dim, rng)
    n = [max(x, 0) for x in lens]
    starts = [0] + list(np.cumsum(n))
    k, v = ((rng.standard_normal((starts[-1], heads, dim)) * size).astype(np.float32) for _ in range(2))
    c.append(table, n, starts, k, v)
    return table, c


CASES = [  # heads, q_heads, dim, page, lens, news, window
    (1, 1, 64, 16, [1], [1], 0),
    (2, 2, 64, 16, [17, 1, 64], [1, 1, 1], 0),
    (8, 32, 128, 64, [100, 1, 257], [1, 1, 1], 0),
    (2, 14, 128, 32, [65, 129], [1, 1], 0),
    (1, 8, 256, 128, [200, 5], [1, 1], 0),
    (4, 4, 96, 16, [333], [1], 0),
    (2, 8, 128, 64, [2000, 300], [1, 1], 0),
    (1, 4, 64, 256, [700], [1], 100),
    (2, 8, 128, 64, [70, 33, 5], [70, 3, 5], 0),
    (1, 7, 64, 16, [130, 64], [41, 64], 0),
    (2, 4, 96, 32, [150], [37], 0),
    (1, 2, 256, 16, [90, 91], [33, 90], 0),
    (2, 2, 128, 16, [300, 20], [64, 20], 17),
    (1, 16, 64, 64, [200], [130], 64),
    (3, 3, 128, 128, [129, 128, 127], [2, 128, 100], 1),
    (1, 32, 128, 64, [260], [65], 0),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_attend(hip, case, dtype):
    heads, q_heads, dim, page, lens, news, window = case
    rng = np.random.default_rng(len(lens) * 100 + dim + page)
    table, c = filled(hip, rng, page, heads, dim, lens)
    starts = [0] + list(np.cumsum(news))
    q = cast(rng.standard_normal((starts[-1], q_heads, dim)), dtype)
    d = Device(hip, c)
    got = attend(hip, d, table, lens, starts, q, dtype, dim ** -0.5, window)
    check_attend(got, *c.attend(table, lens, starts, value(q, dtype), dim ** -0.5, window), dtype)
    d.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 3])
def test_attend_splits_a_long_sequence(hip, n, dtype):
    """max_len decides the split; lengths below, at and above it give the same values."""
    rng = np.random.default_rng(9)
    lens = [5000, 1, 2049]
    news = [n, 1, n]
    table, c = filled(hip, rng, 64, 1, 64, lens)
    starts = [0] + list(np.cumsum(news))
    q = cast(rng.standard_normal((starts[-1], 4, 64)), dtype)
    d = Device(hip, c)
    ref = c.attend(table, lens, starts, value(q, dtype), 0.125, 0)
    for most in (5000, 1 << 20, 4096, 256, 0):
        check_attend(attend(hip, d, table, lens, starts, q, dtype, 0.125, 0, max_len=most), *ref, dtype)
    d.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("news", [[1, 1, 1, 1], [40, 30, 20, 9]])
def test_attend_rows_that_see_nothing(hip, news, dtype):
    """Absent pages, sequences of length 0 and shorter than their rows: such rows are 0, the others unharmed."""
    rng = np.random.default_rng(11)
    lens = [50, 40, 0, 5]
    table, c = filled(hip, rng, 16, 2, 64, lens)
    table[0][0], table[0][2] = -1, c.pages + 5
    table[1] = [-1] * len(table[1])
    starts = [0] + list(np.cumsum(news))
    q = cast(rng.standard_normal((starts[-1], 4, 64)), dtype)
    d = Device(hip, c)
    got = attend(hip, d, table, lens, starts, q, dtype, 0.125, 0)
    want, vmax, cond = c.attend(table, lens, starts, value(q, dtype), 0.125, 0)
    check_attend(got, want, vmax, cond, dtype)
    assert (got[starts[1]:starts[3]] == 0).all()
    d.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,window", [(1, 0), (20, 0), (20, 8), (90, 0), (90, 33)])
def test_attend_nan_in_masked_places(hip, n, window, dtype):
    """NaN codes past the end, before the window and ahead of some rows reach only the rows that see them."""
    rng = np.random.default_rng(13)
    lens = [150]
    table, c = filled(hip, rng, 64, 1, 64, lens)
    last = table[0][2]
    c.v[last, 0, :, 150 - 128:] = 0x7f          # past the end
    c.k[last, 0, 150 - 128:] = 0xff
    c.v[last, 0, 3, 149 - 128] = 0x7f           # the last token: its dim 3
    c.k[table[0][2], 0, 146 - 128, 5] = 0x7f    # a key: the whole row from there on
    c.v[table[0][0], 0, 7, 2] = 0xff            # an early token's dim 7
    starts = [0, n]
    q = cast(rng.standard_normal((n, 4, 64)), dtype)
    d = Device(hip, c)
    got = attend(hip, d, table, lens, starts, q, dtype, 0.125, window)
    want, vmax, cond = c.attend(table, lens, starts, value(q, dtype), 0.125, window)
    check_attend(got, want, vmax, np.where(np.isnan(cond), 0, cond), dtype)
    d.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_large_scores_and_uneven_scales(hip, dtype):
    """Scores of hundreds, pages whose scales differ by 2^20, one q row of zeros and one with a NaN."""
    rng = np.random.default_rng(17)
    table, c = filled(hip, rng, 16, 1, 64, [80])
    c.ks[table[0], 0] = 127 - rng.integers(0, 4, 5) - 5
    c.vs[table[0], 0] = 127 - rng.integers(0, 20, 5)
    q = rng.standard_normal((6, 2, 64)).astype(np.float32) * 3
    q[2, 0] = 0
    q[3, 1, 4] = np.nan
    q = cast(q, dtype)
    d = Device(hip, c)
    got = attend(hip, d, table, [80], [0, 6], q, dtype, 0.125, 0)
    want, vmax, cond = c.attend(table, [80], [0, 6], value(q, dtype), 0.125, 0)
    check_attend(got, want, vmax, np.where(np.isnan(cond), 0, cond), dtype)
    d.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 70])
def test_attend_strided_rows_and_replays(hip, n, dtype):
    """q as part of wider rows; the same bits again, eager and on every replay of a recorded call."""
    rng = np.random.default_rng(19)
    table, c = filled(hip, rng, 64, 2, 64, [300, 200])
    starts, lens = [0, n, 2 * n], [300, 200]
    wide = cast(rng.standard_normal((2 * n, 5 * 64 + 3)), dtype)
    q = np.ascontiguousarray(wide[:, :256]).reshape(2 * n, 4, 64)
    d = Device(hip, c)
    b = d.batch(table, lens, starts)
    with hip.DeviceBuffer.from_numpy(wide) as dq, hip.DeviceBuffer(q.nbytes) as do:
        def call():
            hip.kv8_attend(d.cache, b, dq, do, 4, dtype=dtype, q_ld=323)
        call()
        hip.synchronize()
        first = do.download(q.dtype, q.shape)
        with hip.Graph() as g:
            call()
        for i in range(4):
            do.upload(np.full(q.shape, i, q.dtype))
            g.launch()
            hip.synchronize()
            np.testing.assert_array_equal(do.download(q.dtype, q.shape), first)
            call()
            hip.synchronize()
            np.testing.assert_array_equal(do.download(q.dtype, q.shape), first)
        g.destroy()
    check_attend(value(first, dtype), *c.attend(table, lens, starts, value(q, dtype), 0.125, 0), dtype)
    d.free()
