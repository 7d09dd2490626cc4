"""Layer norm and its backward pass against the formulas in float64.

Bounds, with u = 2^-24 the unit roundoff of fp32 (half a step relative to the value): a sum of n terms of which no chain
of dependent additions is longer than d is within d u sum|terms| of the exact one, to first order. Rows are summed by at
least 64 partial sums once they are longer than 64 elements, so d = n / 64 + 24 covers a lane's own chain, the 12 additions
across a group and what the formula rounds before and after; columns are summed over the rows in any order: d = rows + 8.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24

# Columns around everything a kernel could switch on: single elements, whole vectors and not, one to many elements a lane,
# a wave and a group per row, rows that do not fit the registers of a group.
SHAPES = [(1, 1), (7, 1), (300, 2), (5, 3), (1000, 4), (33, 5), (70, 8), (4097, 12), (65, 63), (64, 64), (63, 65), (513, 128), (3, 129), (1, 255), (2049, 256), (16, 257), (37, 772), (64, 1001),
          (8, 1024), (301, 1028), (2, 1500), (11, 2048), (130, 2052), (9, 3001), (257, 4096), (6, 4100), (5, 5003), (4, 8192), (260, 8196), (3, 16384), (2, 16388), (2, 20001), (1, 32768), (3, 32772), (1, 70000), (2, 70001),
          (1, 1 << 20), (20000, 36), (100003, 16), (5000, 200)]


def chain(cols):
    return cols / 64 + 24


def forward64(x, w, b, eps):
    x = x.astype(np.float64)
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1.0 / np.sqrt((d * d).mean(1) + eps)
    return d * rstd[:, None] * w + b, mean, rstd


def forward_bounds(x, w, b, eps):
    y, mean, rstd = forward64(x, w, b, eps)
    k = chain(x.shape[1]) * U
    x = x.astype(np.float64)
    d_mean = k * np.abs(x).mean(1)
    var_rel = k + 4 * U + (d_mean * rstd) ** 2  # sums of squares about a mean that is off by d_mean
    rstd_rel = 0.5 * var_rel + 3 * U
    xhat = np.abs(x - mean[:, None]) * rstd[:, None]
    d_y = np.abs(w) * ((d_mean * rstd)[:, None] + xhat * (rstd_rel[:, None] + 4 * U)) + 2 * U * (np.abs(y) + np.abs(b) + np.abs(w) * xhat)
    return d_y * 1.01 + 1e-37, d_mean * 1.01 + U * np.abs(mean), rstd * rstd_rel * 1.01


def make(rows, cols, seed=0, shift=1.0):
    rng = np.random.default_rng([rows, cols, seed])
    x = (rng.normal(size=(rows, cols)) * rng.uniform(0.3, 2.0, (rows, 1)) + shift * rng.normal(size=(rows, 1))).astype(np.float32)
    return x, (1 + 0.3 * rng.normal(size=cols)).astype(np.float32), (0.2 * rng.normal(size=cols)).astype(np.float32), rng.normal(size=(rows, cols)).astype(np.float32)


def offset_buffer(rt, arr, words):
    """The array in a buffer of its own, `words` words behind the start: addresses that are not 16-byte aligned."""
    arr = np.ascontiguousarray(arr, dtype=np.float32).reshape(-1)
    whole = rt.DeviceBuffer(arr.size + words + 8)
    whole.fill(0x7FC00000)
    whole.write(arr, offset_words=words)
    view = rt.DeviceBuffer.view(whole.ptr + 4 * words, arr.size)
    view.whole = whole
    return view


def guarded(rt, n):
    """An output of n words with 64 words of a known pattern before and behind it."""
    whole = rt.DeviceBuffer(n + 128)
    whole.fill(0xABCDEF01)
    view = rt.DeviceBuffer.view(whole.ptr + 256, n)
    view.whole = whole
    return view


def untouched(view):
    w = view.whole.numpy(np.uint32)
    return (w[:64] == 0xABCDEF01).all() and (w[-64:] == 0xABCDEF01).all()


@pytest.mark.parametrize("shape", SHAPES)
def test_forward_against_float64(rt, shape):
    rows, cols = shape
    x, w, b, _ = make(rows, cols)
    xb, wb, bb = (rt.DeviceBuffer.from_numpy(a) for a in (x, w, b))
    y, mean, rstd = guarded(rt, x.size), guarded(rt, rows), guarded(rt, rows)
    rt.layer_norm_rows(xb, wb, bb, y, rows, cols, eps=1e-5, mean=mean, rstd=rstd)
    want = forward64(x, w.astype(np.float64), b.astype(np.float64), 1e-5)
    bounds = forward_bounds(x, w.astype(np.float64), b.astype(np.float64), 1e-5)
    for got, ref, bound in zip((y.numpy(np.float32, shape), mean.numpy(), rstd.numpy()), want, bounds):
        assert (np.abs(got - ref) <= bound).all(), float(np.max(np.abs(got - ref) / bound))
    assert untouched(y) and untouched(mean) and untouched(rstd)
    # without weight, bias and statistics, in place
    rt.layer_norm_rows(xb, None, None, xb, rows, cols)
    one, zero = np.ones(cols), np.zeros(cols)
    assert (np.abs(xb.numpy(np.float32, shape) - forward64(x, one, zero, 1e-5)[0]) <= forward_bounds(x, one, zero, 1e-5)[0]).all()


@pytest.mark.parametrize("shape", SHAPES)
def test_backward_against_float64(rt, shape):
    rows, cols = shape
    x, w, _, dy = make(rows, cols, seed=1)
    xb, wb, dyb = (rt.DeviceBuffer.from_numpy(a) for a in (x, w, dy))
    y, mean, rstd = rt.DeviceBuffer(x.size), rt.DeviceBuffer(rows), rt.DeviceBuffer(rows)
    rt.layer_norm_rows(xb, wb, None, y, rows, cols, mean=mean, rstd=rstd)
    m, s = mean.numpy().astype(np.float64)[:, None], rstd.numpy().astype(np.float64)[:, None]  # the call's own inputs
    dx, dw, db = guarded(rt, x.size), guarded(rt, cols), guarded(rt, cols)
    rt.layer_norm_rows_backward(xb, dyb, wb, mean, rstd, rows, cols, dx=dx, dweight=dw, dbias=db)

    k = chain(cols) * U
    xhat = (x - m) * s
    g = dy.astype(np.float64) * w
    mg, mgx = g.mean(1, keepdims=True), (g * xhat).mean(1, keepdims=True)
    want_dx = s * (g - mg - xhat * mgx)
    bound_dx = s * (k * np.abs(g).mean(1, keepdims=True) + np.abs(xhat) * (k + 4 * U) * np.abs(g * xhat).mean(1, keepdims=True) + 6 * U * (np.abs(g) + np.abs(mg) + np.abs(xhat * mgx))) * 1.01 + 1e-37
    got = dx.numpy(np.float32, shape)
    assert (np.abs(got - want_dx) <= bound_dx).all(), float(np.max(np.abs(got - want_dx) / bound_dx))
    terms = dy * xhat
    assert (np.abs(dw.numpy() - terms.sum(0)) <= (rows + 8) * U * np.abs(terms).sum(0) + 1e-37).all()
    assert (np.abs(db.numpy() - dy.astype(np.float64).sum(0)) <= (rows + 8) * U * np.abs(dy.astype(np.float64)).sum(0) + 1e-37).all()
    assert untouched(dx) and untouched(dw) and untouched(db)

    # each output on its own gives the same words; dx over dy, then dx over x
    one_w, one_b, one_x = rt.DeviceBuffer(cols), rt.DeviceBuffer(cols), rt.DeviceBuffer(x.size)
    rt.layer_norm_rows_backward(xb, dyb, wb, mean, rstd, rows, cols, dweight=one_w)
    rt.layer_norm_rows_backward(xb, dyb, wb, mean, rstd, rows, cols, dbias=one_b)
    rt.layer_norm_rows_backward(xb, dyb, wb, mean, rstd, rows, cols, dx=one_x)
    assert np.array_equal(one_w.numpy(), dw.numpy()) and np.array_equal(one_b.numpy(), db.numpy()) and np.array_equal(one_x.numpy(np.float32, shape), got)
    over = rt.DeviceBuffer.from_numpy(dy)
    rt.layer_norm_rows_backward(xb, over, wb, mean, rstd, rows, cols, dx=over, dweight=one_w, dbias=one_b)
    assert np.array_equal(over.numpy(np.float32, shape), got) and np.array_equal(one_w.numpy(), dw.numpy()) and np.array_equal(one_b.numpy(), db.numpy())
    rt.layer_norm_rows_backward(xb, dyb, wb, mean, rstd, rows, cols, dx=xb, dweight=one_w, dbias=one_b)
    assert np.array_equal(xb.numpy(np.float32, shape), got) and np.array_equal(one_w.numpy(), dw.numpy()) and np.array_equal(one_b.numpy(), db.numpy())


# on both sides of the number of rows up to which one launch does everything, unless dx takes the place of an input
@pytest.mark.parametrize("rows", [1, 15, 128, 129, 511, 512, 513, 1024, 1025])
@pytest.mark.parametrize("cols", [1, 17, 250, 256, 257, 1024, 1030, 9000])
def test_few_rows_backward_in_place_and_not(rt, rows, cols):
    x, w, _, dy = make(rows, cols, seed=3)
    xb, wb = rt.DeviceBuffer.from_numpy(x), rt.DeviceBuffer.from_numpy(w)
    mean, rstd = rt.DeviceBuffer(rows), rt.DeviceBuffer(rows)
    rt.layer_norm_rows(xb, wb, None, rt.DeviceBuffer(x.size), rows, cols, mean=mean, rstd=rstd)
    m, s = mean.numpy().astype(np.float64)[:, None], rstd.numpy().astype(np.float64)[:, None]
    terms = dy * ((x - m) * s)
    chain = (rows + 8) * U  # a sum of `rows` terms in any order, each off by a few roundings
    results = []
    for place in ("own", "dy", "x"):
        xb, dyb = rt.DeviceBuffer.from_numpy(x), rt.DeviceBuffer.from_numpy(dy)
        dx = {"own": guarded(rt, x.size), "dy": dyb, "x": xb}[place]
        dw, db = guarded(rt, cols), guarded(rt, cols)
        rt.layer_norm_rows_backward(xb, dyb, wb, mean, rstd, rows, cols, dx=dx, dweight=dw, dbias=db)
        assert (np.abs(dw.numpy() - terms.sum(0)) <= chain * np.abs(terms).sum(0) + 4 * U * (np.abs(dy) * s * (np.abs(x) + np.abs(m))).sum(0)).all()
        assert (np.abs(db.numpy() - dy.astype(np.float64).sum(0)) <= chain * np.abs(dy).sum(0)).all()
        assert untouched(dw) and untouched(db) and (place != "own" or untouched(dx))
        results.append(dx.numpy(np.float32, x.shape))
    assert np.array_equal(results[0], results[1]) and np.array_equal(results[0], results[2])
    # each gradient by itself: the same words as together
    for name in ("dx", "dweight", "dbias"):
        n = x.size if name == "dx" else cols
        alone, together = guarded(rt, n), {k: rt.DeviceBuffer(x.size if k == "dx" else cols) for k in ("dx", "dweight", "dbias")}
        xb, dyb = rt.DeviceBuffer.from_numpy(x), rt.DeviceBuffer.from_numpy(dy)
        rt.layer_norm_rows_backward(xb, dyb, wb, mean, rstd, rows, cols, **{name: alone})
        rt.layer_norm_rows_backward(xb, dyb, wb, mean, rstd, rows, cols, **together)
        assert untouched(alone) and np.array_equal(alone.numpy(np.uint32), together[name].numpy(np.uint32))


# rows that end one, two and three elements into a vector, on both sides of the widths at which another kernel takes over
@pytest.mark.parametrize("cols", [1023, 1025, 2047, 2049, 4093, 4095, 4097, 4098, 4099, 8190, 8193, 8195, 16381, 16382, 16383, 16385, 16386, 24577, 24579])
@pytest.mark.parametrize("rows", [1, 7])
def test_rows_that_end_inside_a_vector(rt, rows, cols):
    test_forward_against_float64(rt, (rows, cols))
    test_backward_against_float64(rt, (rows, cols))
    x, w, _, dy = make(rows, cols, seed=2)
    xb, wb, dyb, dx = (rt.DeviceBuffer.from_numpy(a) for a in (x, w, dy, np.zeros_like(x)))
    mean, rstd = rt.DeviceBuffer(rows), rt.DeviceBuffer(rows)
    rt.layer_norm_rows(xb, wb, None, dx, rows, cols, mean=mean, rstd=rstd)
    rt.layer_norm_rows_backward(xb, dyb, wb, mean, rstd, rows, cols, dx=dx)
    want = dx.numpy(np.float32, x.shape)
    rt.layer_norm_rows_backward(xb, dyb, wb, mean, rstd, rows, cols, dx=dyb)  # the gradient in dy's place: the same words
    assert np.array_equal(dyb.numpy(np.float32, x.shape), want)


@pytest.mark.parametrize("shape", [(9, 64), (130, 256), (33, 1024), (5, 4096), (3, 20000)])
@pytest.mark.parametrize("odd", ["x", "weight", "out", "dy"])
def test_addresses_that_are_only_word_aligned(rt, shape, odd):
    rows, cols = shape
    x, w, b, dy = make(rows, cols, seed=2)
    place = lambda a, name: offset_buffer(rt, a, 1 if name == odd else 4)  # noqa: E731
    xb, wb, bb, dyb = place(x, "x"), place(w, "weight"), place(b, "weight"), place(dy, "dy")
    y, dx, dw, db = (place(np.zeros(n, np.float32), "out") for n in (x.size, x.size, cols, cols))
    mean, rstd = place(np.zeros(rows), "out"), place(np.zeros(rows), "out")
    rt.layer_norm_rows(xb, wb, bb, y, rows, cols, mean=mean, rstd=rstd)
    want, bounds = forward64(x, w.astype(np.float64), b.astype(np.float64), 1e-5), forward_bounds(x, w.astype(np.float64), b.astype(np.float64), 1e-5)
    assert (np.abs(y.numpy(np.float32, shape) - want[0]) <= bounds[0]).all()
    rt.layer_norm_rows_backward(xb, dyb, wb, mean, rstd, rows, cols, dx=dx, dweight=dw, dbias=db)
    plain = [rt.DeviceBuffer(n) for n in (x.size, cols, cols)]
    rt.layer_norm_rows_backward(rt.DeviceBuffer.from_numpy(x), rt.DeviceBuffer.from_numpy(dy), rt.DeviceBuffer.from_numpy(w), mean, rstd, rows, cols, dx=plain[0], dweight=plain[1], dbias=plain[2])
    xhat = (x - mean.numpy().astype(np.float64)[:, None]) * rstd.numpy().astype(np.float64)[:, None]
    scale = np.abs(dy * xhat).sum(0)
    # the two may take different kernels: each is within the bound of the exact sum
    assert (np.abs(dw.numpy() - (dy * xhat).sum(0)) <= (rows + 8) * U * scale).all()
    assert (np.abs(plain[1].numpy() - (dy * xhat).sum(0)) <= (rows + 8) * U * scale).all()
    assert (np.abs(db.numpy().astype(np.float64) - plain[2].numpy()) <= 2 * (rows + 8) * U * np.abs(dy).sum(0)).all()
    size = np.abs(dx.numpy(np.float32, shape)).max(1, keepdims=True)
    assert (np.abs(dx.numpy(np.float32, shape).astype(np.float64) - plain[0].numpy(np.float32, shape)) <= 2 * (chain(cols) + 10) * U * 4 * size).all()


@pytest.mark.parametrize("cols", [4, 63, 256, 1024, 5000, 40000])
def test_rows_with_a_large_mean_keep_their_digits(rt, cols):
    """Values 1000 + k / 8 with small k: sums of integers over 8 far below 2^24 steps, so the mean is exact when it is a
    step itself, and so is every difference."""
    rng = np.random.default_rng(cols)
    k = rng.integers(-4, 5, (5, cols))
    k[:, 1:] = np.where(np.arange(1, cols) % 2, -k[:, : cols - 1], k[:, 1:]) if cols > 1 else k[:, 1:]
    x = (1000.0 + k / 8.0).astype(np.float32)
    y = rt.DeviceBuffer(x.size)
    rt.layer_norm_rows(rt.DeviceBuffer.from_numpy(x), None, None, y, 5, cols)
    want = forward64(x, np.ones(cols), np.zeros(cols), 1e-5)[0]
    bound = forward_bounds(x, np.ones(cols), np.zeros(cols), 1e-5)[0]
    assert (np.abs(y.numpy(np.float32, x.shape) - want) <= bound).all()


def test_constant_rows_are_zero_plus_bias(rt):
    for cols in (1, 4, 100, 1024, 5000, 40000):
        x = np.repeat(np.array([[0.0], [3.0], [-1.5]], np.float32), cols, 1)
        b = np.linspace(-1, 1, cols, dtype=np.float32)
        y = rt.DeviceBuffer(x.size)
        rt.layer_norm_rows(rt.DeviceBuffer.from_numpy(x), None, rt.DeviceBuffer.from_numpy(b), y, 3, cols)
        # sums of up to 40000 equal small halves are exact while they stay below 2^23: the difference to the mean is 0
        assert np.array_equal(y.numpy(np.float32, x.shape), np.repeat(b[None], 3, 0)), cols


@pytest.mark.parametrize("cols", [3, 64, 1024, 4100, 40000])
def test_nan_and_infinity_stay_in_their_rows(rt, cols):
    x, w, b, dy = make(6, cols, seed=3)
    clean = x.copy()
    x[1, 0], x[3, cols - 1], x[4, cols // 2] = np.nan, np.inf, -np.inf
    y, mean, rstd, dx = rt.DeviceBuffer(x.size), rt.DeviceBuffer(6), rt.DeviceBuffer(6), rt.DeviceBuffer(x.size)
    wb, bb = rt.DeviceBuffer.from_numpy(w), rt.DeviceBuffer.from_numpy(b)
    rt.layer_norm_rows(rt.DeviceBuffer.from_numpy(x), wb, bb, y, 6, cols, mean=mean, rstd=rstd)
    got = y.numpy(np.float32, x.shape)
    assert np.isnan(got[[1, 3, 4]]).any(1).all() and np.isfinite(got[[0, 2, 5]]).all()
    rt.layer_norm_rows(rt.DeviceBuffer.from_numpy(clean), wb, bb, y, 6, cols)
    assert np.array_equal(got[[0, 2, 5]], y.numpy(np.float32, x.shape)[[0, 2, 5]])
    rt.layer_norm_rows_backward(rt.DeviceBuffer.from_numpy(x), rt.DeviceBuffer.from_numpy(dy), wb, mean, rstd, 6, cols, dx=dx)
    back = dx.numpy(np.float32, x.shape)
    assert np.isnan(back[[1, 3, 4]]).any(1).all() and np.isfinite(back[[0, 2, 5]]).all()


def test_no_rows(rt):
    one = rt.DeviceBuffer.from_numpy(np.ones(8, np.float32))
    dw, db = rt.DeviceBuffer.from_numpy(np.ones(8, np.float32)), rt.DeviceBuffer.from_numpy(np.ones(8, np.float32))
    rt.layer_norm_rows(one, None, None, one, 0, 8)
    rt.layer_norm_rows_backward(one, one, None, one, one, 0, 8, dx=None, dweight=dw, dbias=db)
    assert np.array_equal(one.numpy(), np.ones(8)) and not dw.numpy().any() and not db.numpy().any()


def test_backward_against_differences(rt):
    """dx, dweight and dbias of L = sum(y * dy) against central differences of the forward call itself. With x, dy of order
    one and C = 48 the third derivative of L along one element is of order 1, so a step h costs h^2 / 6 and the rounding of L
    (48 terms of order 1, computed in float64 from y, each y off by at most 40 u) 48 * 40 u / h: 3e-3 and 4e-3 at h = 0.03."""
    rows, cols, h = 3, 48, 0.03
    x, w, b, dy = make(rows, cols, seed=4, shift=0.2)

    def loss(x, w, b):
        y = rt.DeviceBuffer(x.size)
        rt.layer_norm_rows(rt.DeviceBuffer.from_numpy(x), rt.DeviceBuffer.from_numpy(w), rt.DeviceBuffer.from_numpy(b), y, rows, cols)
        return float((y.numpy(np.float32, x.shape).astype(np.float64) * dy).sum())

    y, mean, rstd = rt.DeviceBuffer(x.size), rt.DeviceBuffer(rows), rt.DeviceBuffer(rows)
    xb, wb = rt.DeviceBuffer.from_numpy(x), rt.DeviceBuffer.from_numpy(w)
    rt.layer_norm_rows(xb, wb, rt.DeviceBuffer.from_numpy(b), y, rows, cols, mean=mean, rstd=rstd)
    dx, dw, db = rt.DeviceBuffer(x.size), rt.DeviceBuffer(cols), rt.DeviceBuffer(cols)
    rt.layer_norm_rows_backward(xb, rt.DeviceBuffer.from_numpy(dy), wb, mean, rstd, rows, cols, dx=dx, dweight=dw, dbias=db)
    for array, grad in ((x, dx.numpy(np.float32, x.shape)), (w, dw.numpy()), (b, db.numpy())):
        for at in ((0, 0), (1, 17), (2, 47)) if array.ndim == 2 else ((0,), (17,), (47,)):
            keep = array[at]
            array[at] = keep + np.float32(h)
            up, step_up = loss(x, w, b), float(array[at])
            array[at] = keep - np.float32(h)
            down, step_down = loss(x, w, b), float(array[at])
            array[at] = keep
            assert abs((up - down) / (step_up - step_down) - grad[at]) < 2e-2


def test_a_row_of_many_columns(rt):
    """140 000 001 columns: more than a launch of one group per 64 columns of the two gradients covers. x = +-1 in turn and one 0: mean 0
    (whole numbers below 2^24 in every partial sum of 8192), variance 1 up to 1e-8 and the rounding of sums."""
    cols = 140_000_001
    x = np.ones(cols, np.float32)
    x[1::2] = -1
    x[-1] = 0
    dy = (np.arange(cols) % 5 - 2).astype(np.float32)
    xb, dyb = rt.DeviceBuffer.from_numpy(x), rt.DeviceBuffer.from_numpy(dy)
    y, mean, rstd, dw, db = rt.DeviceBuffer(cols), rt.DeviceBuffer(1), rt.DeviceBuffer(1), rt.DeviceBuffer(cols), rt.DeviceBuffer(cols)
    rt.layer_norm_rows(xb, None, None, y, 1, cols, eps=0.0, mean=mean, rstd=rstd)
    assert mean.numpy()[0] == 0 and abs(rstd.numpy()[0] - 1) < 1e-5
    s = rstd.numpy()[0]
    assert np.array_equal(y.numpy(), x * s)
    rt.layer_norm_rows_backward(xb, dyb, None, mean, rstd, 1, cols, dweight=dw, dbias=db)
    assert np.array_equal(db.numpy(), dy) and np.array_equal(dw.numpy(), dy * (x * s))
    for b in (xb, dyb, y, dw, db):
        b.free()


def test_many_rows_of_one_column_in_place(rt):
    """2^30 + 3 rows of one element: each is its own mean, so y = bias everywhere; two launches."""
    rows = (1 << 30) + 3
    x, mean = rt.DeviceBuffer(rows), rt.DeviceBuffer(rows)
    x.fill(0x40400000)
    rt.layer_norm_rows(x, None, rt.DeviceBuffer.from_numpy(np.array([0.25], np.float32)), x, rows, 1, mean=mean)
    for b, want in ((x, 0.25), (mean, 3.0)):
        for at in (0, rows // 2, (1 << 29) - 2, rows - 5):
            assert (b.numpy(np.float32, (5,), offset_words=at) == want).all()
        out = rt.DeviceBuffer(1)
        rt.reduce_rows("min", b, out, 1, rows)
        assert out.numpy()[0] == want
        rt.reduce_rows("max", b, out, 1, rows)
        assert out.numpy()[0] == want
        b.free()
