"""The embedding gradient of few positions: in one launch where the table has rows enough to spread them, else by ordered positions. The
number of launches is read from a recorded graph; the sums are of whole numbers, so the result is exact either way."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ONE = [(1, 1, 5), (384, 1, 20), (384, 8, 64), (385, 17, 64), (1000, 42, 33), (2016, 84, 40), (2048, 86, 130), (2048, 5000, 16)]
ORDERED = [(385, 1, 20), (385, 16, 64), (1009, 42, 33), (1024, 8, 256), (2017, 84, 40), (2048, 50, 64), (2048, 1, 1024), (2048, 85, 130), (2049, 5000, 16)]


@pytest.mark.parametrize("shape, one", [(s, True) for s in ONE] + [(s, False) for s in ORDERED])
@pytest.mark.parametrize("kind", ["even", "skewed", "one token"])
def test_few_rows_of_a_table_are_not_left_to_one_launch(rt, shape, one, kind):
    n, vocab, cols = shape
    rng = np.random.default_rng([n, vocab, cols])
    t = {"even": lambda: rng.integers(-1, vocab, n), "skewed": lambda: np.minimum(rng.geometric(0.1, n) - 1, vocab), "one token": lambda: np.full(n, vocab - 1)}[kind]().astype(np.int32)
    dy = rng.integers(-4, 5, (n, cols)).astype(np.float32)
    want = np.zeros((vocab, cols))
    known = (t >= 0) & (t < vocab)
    np.add.at(want, t[known], 2.0 * dy[known])
    tb, dyb, d = rt.DeviceBuffer.from_numpy(t), rt.DeviceBuffer.from_numpy(dy), rt.DeviceBuffer(vocab * cols)
    call = lambda: rt.embedding_rows_backward(tb, dyb, d, n, vocab, cols, scale=2.0)  # noqa: E731
    call()  # sizes the scratch buffer
    assert np.array_equal(d.numpy(np.float32, (vocab, cols)), want.astype(np.float32))
    graph = rt.Graph()
    with graph:
        call()
    assert (graph.nodes == 1) == one, graph.nodes
    for _ in range(2):
        d.fill(0x7FC00000)
        graph.launch()
        assert np.array_equal(d.numpy(np.float32, (vocab, cols)), want.astype(np.float32))
    graph.destroy()
