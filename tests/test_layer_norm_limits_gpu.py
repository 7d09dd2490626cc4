"""Rows of layer norm at the ends of fp32, as the header states them; the rows beside them are untouched."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [8, 100, 1024, 1025, 5000, 16384, 20000])
def test_rows_beyond_the_range_of_the_sums(rt, cols):
    rows = 9
    rng = np.random.default_rng(cols)
    x = rng.normal(size=(rows, cols)).astype(np.float32)
    weight, bias = (1 + 0.2 * rng.normal(size=cols)).astype(np.float32), rng.normal(size=cols).astype(np.float32)
    bufs = [rt.DeviceBuffer.from_numpy(weight), rt.DeviceBuffer.from_numpy(bias), rt.DeviceBuffer(rows * cols), rt.DeviceBuffer(rows), rt.DeviceBuffer(rows)]

    def run(x, eps):
        w, b, y, mean, rstd = bufs
        rt.layer_norm_rows(rt.DeviceBuffer.from_numpy(x), w, b, y, rows, cols, eps=eps, mean=mean, rstd=rstd)
        return y.numpy(np.float32, x.shape), rstd.numpy()

    clean = run(x, 1e-5)[0]
    x[2] = np.where(np.arange(cols) % 2, 1e20, -1e20)  # squares of 1e40
    x[4] = 3e38                                          # a sum of 2.4e39 and more
    x[6] = -2.0                                          # all equal
    y, rstd = run(x, 1e-5)
    assert rstd[2] == 0 and np.array_equal(y[2], bias)
    assert np.isnan(y[4]).all()
    assert np.array_equal(y[6], bias) and abs(rstd[6] - 1e5 ** 0.5) < 1e-3
    y0, rstd0 = run(x, 0.0)
    assert np.isinf(rstd0[6]) and np.isnan(y0[6]).all()
    others = [0, 1, 3, 5, 7, 8]
    assert np.array_equal(y[others], clean[others]) and np.isfinite(y0[others]).all()
