"""The MXFP4 operators on the device against their plain 64-bit forms."""
import numpy as np
import pytest

import lowbits as L

pytestmark = pytest.mark.gpu


def dev(hip, a):
    return hip.DeviceBuffer.from_numpy(a)


def quantize(hip, x, dtype="f32", ld=0, rows=None, k=None):
    rows, k = x.shape[0] if rows is None else rows, x.shape[1] if k is None else k
    qb, sb = hip.mxfp4_row(k)
    with dev(hip, x) as dx, hip.DeviceBuffer(rows * qb + 64) as dq, hip.DeviceBuffer(rows * sb + 64) as ds:
        dq.upload(np.full(rows * qb + 64, 0xA5, np.uint8))
        ds.upload(np.full(rows * sb + 64, 0xA5, np.uint8))
        hip.mxfp4_quantize(dx, dq, ds, rows, k, dtype=dtype, ld=ld)
        hip.synchronize()
        q, s = dq.download(np.uint8, (rows * qb + 64,)), ds.download(np.uint8, (rows * sb + 64,))
    assert (q[rows * qb:] == 0xA5).all() and (s[rows * sb:] == 0xA5).all()
    return q[:rows * qb].reshape(rows, qb), s[:rows * sb].reshape(rows, sb)


def rows_of(rng, rows, k, spread=True):
    x = rng.standard_normal((rows, k)).astype(np.float32)
    if spread:  # blocks of very different sizes, exact ties among them
        x *= np.exp2(rng.integers(-30, 30, (rows, 1))).astype(np.float32)
        tie = rng.random((rows, k)) < 0.2
        x = np.where(tie, rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -2.5, 0.0, -0.0], (rows, k)), x)
    return x.astype(np.float32)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 31), (3, 32), (2, 33), (5, 127), (4, 128), (7, 129), (33, 4097),
                                    (1, 16384), (300, 515), (65537, 40)])
def test_quantize_bits(hip, rows, k, dtype):
    x = rows_of(np.random.default_rng(rows * 7919 + k), rows, k)
    src = L.bf16_bits(x) if dtype == "bf16" else x
    q, s = quantize(hip, src, dtype)
    wq, ws = L.mx_quantize(L.bf16_value(src) if dtype == "bf16" else x)
    np.testing.assert_array_equal(s, ws)
    np.testing.assert_array_equal(q, wq)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_special_blocks(hip, dtype):
    """Infs and NaNs, all-zero blocks, subnormals, and the ends of the scale's range."""
    x = np.random.default_rng(1).standard_normal((16, 96)).astype(np.float32)
    x[0, 3] = np.inf
    x[1, 40] = -np.inf
    x[2, 95] = np.nan
    x[3, :32] = 0.0
    x[4, :32] = -0.0
    x[5, :32] = 1e-45
    x[6, :32] *= np.float32(1e-38)
    x[7, :32] *= np.float32(2.0) ** -126
    x[8, :32] = np.float32(3.3e38)
    x[9, :32] = np.float32(2.0) ** -125 * np.arange(32, dtype=np.float32) / 8
    x[10, :32] = np.float32(2.0) ** 127
    src = L.bf16_bits(x) if dtype == "bf16" else x
    q, s = quantize(hip, src, dtype)
    wq, ws = L.mx_quantize(L.bf16_value(src) if dtype == "bf16" else x)
    np.testing.assert_array_equal(s, ws)
    np.testing.assert_array_equal(q, wq)
    assert s[0, 0] == 255 and s[1, 1] == 255 and s[2, 2] == 255 and s[0, 1] != 255


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("k,ld,off", [(100, 101, 0), (257, 300, 1), (64, 64, 3)])
def test_quantize_strided_and_unaligned_rows(hip, k, ld, off, dtype):
    rng = np.random.default_rng(k)
    x = rng.standard_normal((9, ld)).astype(np.float32)
    src = L.bf16_bits(x) if dtype == "bf16" else x
    flat = np.concatenate([np.zeros(off, src.dtype), src.reshape(-1)])
    qb, sb = hip.mxfp4_row(k)
    with dev(hip, flat) as dx, hip.DeviceBuffer(9 * qb) as dq, hip.DeviceBuffer(9 * sb) as ds:
        hip.mxfp4_quantize(dx.addr + off * src.itemsize, dq, ds, 9, k, dtype=dtype, ld=ld)
        hip.synchronize()
        q, s = dq.download(np.uint8, (9, qb)), ds.download(np.uint8, (9, sb))
    wq, ws = L.mx_quantize((L.bf16_value(src) if dtype == "bf16" else x)[:, :k])
    np.testing.assert_array_equal(q, wq)
    np.testing.assert_array_equal(s, ws)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k,ld", [(1, 1, 0), (3, 130, 0), (2, 4097, 4099), (256, 32, 0)])
def test_dequantize_values(hip, rows, k, ld, dtype):
    """Every code under every scale byte (255 is NaN), exactly; nothing written past a row."""
    rng = np.random.default_rng(k)
    qb, sb = hip.mxfp4_row(k)
    q = rng.integers(0, 256, (rows, qb), dtype=np.uint8)
    s = (np.arange(rows * sb) % 256).astype(np.uint8).reshape(rows, sb)
    if k > 4000:
        s = rng.integers(0, 256, (rows, sb), dtype=np.uint8)
    want = L.mx_values(q, s, k)
    step, ty = ld or k, np.float32 if dtype == "f32" else np.uint16
    with dev(hip, q) as dq, dev(hip, s) as ds, dev(hip, np.full(rows * step + 8, 7, ty)) as dy:
        hip.mxfp4_dequantize(dq, ds, dy, rows, k, dtype=dtype, ld=ld)
        hip.synchronize()
        raw = dy.download(ty, (rows * step + 8,))
    assert (raw[rows * step:] == 7).all()
    got = raw[:rows * step].reshape(rows, step)
    assert (got[:, k:] == 7).all()
    got = (got if dtype == "f32" else L.bf16_value(got))[:, :k].astype(np.float64)
    with np.errstate(over="ignore"):
        want = np.where(np.isnan(want), want, want.astype(np.float32).astype(np.float64))
        if dtype == "bf16":  # 6 * 2^127 and the like pass the type's range: cut like f32's
            want = L.bf16_value((want.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)).astype(np.float64)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(got[~np.isnan(want)], want[~np.isnan(want)])


# ---- products ---------------------------------------------------------------------------

def weights(rng, n, k, scale=0.02):
    x = (rng.standard_normal((n, k)) * scale).astype(np.float32)
    return L.mx_quantize(x)


def run_product(hip, x, wq, ws, n, k, xs=None):
    m = x.shape[0]
    with dev(hip, x) as dx, dev(hip, wq) as dq, dev(hip, ws) as ds, dev(hip, np.full((m * n + 16,), 7.0, np.float32)) as dy:
        if xs is None:
            hip.gemv_mxfp4_rd(dx, dq, ds, dy, m, k, n)
        else:
            with dev(hip, xs) as dxs:
                hip.gemm_mxfp4(dx, dxs, dq, ds, dy, m, k, n)
                hip.synchronize()
        hip.synchronize()
        y = dy.download(np.float32, (m * n + 16,))
    assert (y[m * n:] == 7.0).all()
    return y[:m * n].reshape(m, n)


def check_product(y, x, w):
    """x [m, k], w [n, k] in f64.  Each output is a chain of f32 sums, at most 5 per 128 k and 40 more where waves
    and terms meet, each off by at most a unit (2^-23) of the sum of magnitudes; x's digits are cut at 2^-24 of its
    block's largest value.  Gaussian sums are far inside: their norm is held to 1e-6."""
    m, k = x.shape
    g = -(-k // 128)
    xb = np.zeros((m, -(-k // 32) * 32))
    xb[:, :k] = np.abs(x)
    xb = np.repeat(xb.reshape(m, -1, 32).max(2), 32, 1)[:, :k]
    want = x @ w.T
    bound = (5 * g + 40) * 2.0 ** -23 * (xb @ np.abs(w).T) + 1e-44
    np.testing.assert_array_less(np.abs(y - want), bound + 1e-300)
    assert np.linalg.norm(y - want) <= 1e-6 * max(np.linalg.norm(want), 1e-30) * (1 if k > 64 else 4)


SHAPES = [(1, 1, 1), (1, 16, 128), (1, 17, 129), (1, 1792, 4096), (1, 300, 14336), (2, 130, 4097), (3, 64, 8192), (4, 33, 640),
          (5, 257, 300), (5, 40, 5000), (6, 100, 96), (7, 33, 4097), (16, 515, 1031), (17, 128, 256), (33, 200, 4097),
          (64, 96, 512), (65, 129, 130), (130, 270, 1000), (257, 513, 384)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_f32(hip, m, n, k):
    rng = np.random.default_rng(m * 31 + n * 17 + k)
    x = rng.standard_normal((m, k)).astype(np.float32)
    wq, ws = weights(rng, n, k)
    check_product(run_product(hip, x, wq, ws, n, k), x.astype(np.float64), L.mx_values(wq, ws, k))


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_mxfp4(hip, m, n, k):
    rng = np.random.default_rng(m * 37 + n * 13 + k)
    xq, xs = weights(rng, m, k, 1.0)
    wq, ws = weights(rng, n, k)
    check_product(run_product(hip, xq, wq, ws, n, k, xs), L.mx_values(xq, xs, k), L.mx_values(wq, ws, k))


@pytest.mark.parametrize("m", [1, 3, 5, 6, 20])
def test_product_blocks_of_very_different_sizes(hip, m):
    """Scales spread over 2^-40 .. 2^40, zero blocks and x spread over 2^-20 .. 2^20 within a row."""
    rng = np.random.default_rng(m)
    n, k = 70, 700
    x = (rng.standard_normal((m, k)) * np.exp2(rng.integers(-20, 20, (m, k)))).astype(np.float32)
    w = (rng.standard_normal((n, k)) * np.repeat(np.exp2(rng.integers(-40, 40, (n, 22))), 32, 1)[:, :k]).astype(np.float32)
    w[:, 64:96] = 0
    x[:, 128:160] = 0
    wq, ws = L.mx_quantize(w)
    y = run_product(hip, x, wq, ws, n, k)
    wv = L.mx_values(wq, ws, k)
    x64 = x.astype(np.float64)
    xb = np.zeros((m, 704))
    xb[:, :k] = np.abs(x)
    xb = np.repeat(xb.reshape(m, -1, 32).max(2), 32, 1)[:, :k]
    assert (np.abs(y - x64 @ wv.T) <= (5 * 6 + 40) * 2.0 ** -23 * (xb @ np.abs(wv).T)).all()


@pytest.mark.parametrize("m", [1, 4, 5, 6, 18, 70])
def test_product_inf_and_nan_classes(hip, m):
    """inf, -inf and NaN activations and NaN blocks give the formula's classes; other rows and outputs keep values."""
    rng = np.random.default_rng(m)
    n, k = 50, 300
    x = rng.standard_normal((m, k)).astype(np.float32)
    wq, ws = weights(rng, n, k)
    ws[7, 1] = 255
    x[m - 1, 5] = np.inf
    if m > 1:
        x[0, 299] = -np.inf
        x[0, 17] = np.inf
    if m > 4:
        x[2, 100] = np.uint32(0x7f800001).view(np.float32)  # a NaN whose high half alone would be an inf
    y = run_product(hip, x, wq, ws, n, k)
    w = L.mx_values(wq, ws, k)
    with np.errstate(invalid="ignore"):
        want = np.stack([[(x[i].astype(np.float64) * w[j]).sum() for j in range(n)] for i in range(m)])
    np.testing.assert_array_equal(np.isnan(y), np.isnan(want))
    np.testing.assert_array_equal(np.isposinf(y), np.isposinf(want))
    np.testing.assert_array_equal(np.isneginf(y), np.isneginf(want))
    ok = np.isfinite(want)
    assert np.abs(y[ok] - want[ok]).max(initial=0.0) < 1e-5 * 0.02 * 300


@pytest.mark.parametrize("m", [2, 33])
def test_product_mxfp4_nan_blocks(hip, m):
    rng = np.random.default_rng(m)
    xq, xs = weights(rng, m, 260, 1.0)
    wq, ws = weights(rng, 40, 260)
    xs[1, 2], ws[3, 0] = 255, 255
    y = run_product(hip, xq, wq, ws, 40, 260, xs)
    want = np.zeros((m, 40), bool)
    want[1], want[:, 3] = True, True
    np.testing.assert_array_equal(np.isnan(y), want)


@pytest.mark.parametrize("m", [1, 40])
def test_product_of_no_length_is_zero(hip, m):
    z = np.zeros((1, 64), np.uint8)
    np.testing.assert_array_equal(run_product(hip, np.zeros((m, 1), np.float32), z, z, 33, 0), np.zeros((m, 33)))
    np.testing.assert_array_equal(run_product(hip, np.zeros((m, 64), np.uint8), z, z, 33, 0, z), np.zeros((m, 33)))


@pytest.mark.parametrize("m,n,k", [(1, 500, 4096), (9, 300, 1000), (48, 512, 2048)])
def test_product_repeats_and_replays_bit_for_bit(hip, m, n, k):
    """Eager calls and every replay of a recorded one give the same bits, with other work between."""
    rng = np.random.default_rng(k)
    x = rng.standard_normal((m, k)).astype(np.float32)
    wq, ws = weights(rng, n, k)
    first = run_product(hip, x, wq, ws, n, k)
    with dev(hip, x) as dx, dev(hip, wq) as dq, dev(hip, ws) as ds, hip.DeviceBuffer(4 * m * n) as dy, \
            hip.DeviceBuffer(m * hip.mxfp4_row(k)[0]) as xq, hip.DeviceBuffer(m * hip.mxfp4_row(k)[1]) as xs, \
            hip.DeviceBuffer(4 * m * n) as dz:
        with hip.Graph() as g:
            hip.gemv_mxfp4_rd(dx, dq, ds, dy, m, k, n)
            hip.mxfp4_quantize(dx, xq, xs, m, k)
            hip.gemm_mxfp4(xq, xs, dq, ds, dz, m, k, n)
        hip.mxfp4_quantize(dx, xq, xs, m, k)
        hip.gemm_mxfp4(xq, xs, dq, ds, dz, m, k, n)
        hip.synchronize()
        z = dz.download(np.float32, (m, n))
        for i in range(4):
            dy.upload(np.full((m, n), i, np.float32))
            dz.upload(np.full((m, n), i, np.float32))
            g.launch()
            hip.synchronize()
            np.testing.assert_array_equal(dy.download(np.float32, (m, n)), first)
            np.testing.assert_array_equal(dz.download(np.float32, (m, n)), z)
            np.testing.assert_array_equal(run_product(hip, x, wq, ws, n, k), first)
        g.destroy()
