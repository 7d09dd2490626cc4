"""Embedding lookup and the gradient of its table.

The lookup is one product rounded once: exact against numpy's float32 product. The gradient is tested with small integers,
whose sums are exact in fp32 in any order, and a power of two as the scale: bit-exact; and with reals, where a sum of n
terms in any order is within n u sum|terms| of the exact one (u = 2^-24), plus u for the scaling.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24

# (n, vocab, cols): single tokens, sizes around tiles of 32, 128, 2048, 8192 and 16384 positions, tables of one row, of less and more than
# 2^8 and 2^16 rows, odd widths
SHAPES = [(1, 1, 1), (1, 10, 3), (2, 1, 64), (33, 5, 4), (64, 300, 250), (77, 1009, 250), (127, 3, 65), (128, 256, 128), (129, 255, 100), (500, 1009, 250), (1000, 2, 1000), (2047, 70, 36), (2048, 70000, 8),
          (2049, 65536, 12), (4097, 65535, 16), (8191, 100, 20), (8192, 5000, 4), (8193, 5000, 5), (16384, 300, 64), (16385, 70000, 7), (20000, 1, 24), (40000, 31, 256), (60000, 50000, 33), (131073, 1000, 8), (300000, 100003, 3),
          (5, 40, 5000), (300, 20, 4100), (4, 3, 70000)]


def tokens_for(n, vocab, seed, pad=0.0):
    rng = np.random.default_rng([n, vocab, seed])
    ranks = np.minimum((np.exp(rng.random(n) * np.log(vocab + 1.0)) - 1).astype(np.int64), vocab - 1)  # few frequent, many rare
    t = rng.permutation(vocab)[ranks].astype(np.int32)
    if pad:
        t[rng.random(n) < pad] = -1
    return t


def gradient(tokens, dy, vocab):
    """Sums by token in float64: differences of running sums over the rows in token order."""
    known = (tokens >= 0) & (tokens < vocab)
    order = np.flatnonzero(known)[np.argsort(tokens[known], kind="stable")]
    out = np.zeros((vocab, dy.shape[1]))
    if len(order):
        values, starts = np.unique(tokens[order], return_index=True)
        out[values] = np.add.reduceat(dy[order].astype(np.float64), starts, axis=0)
    return out


@pytest.mark.parametrize("shape", SHAPES)
def test_lookup_is_exact(rt, shape):
    n, vocab, cols = shape
    t = tokens_for(n, vocab, 0, pad=0.2)
    t[-1:] = vocab  # one past the table
    t[: n // 50] = np.iinfo(np.int32).min
    table = np.random.default_rng(vocab).normal(size=(vocab, cols)).astype(np.float32)
    out = rt.DeviceBuffer(n * cols + 64)
    out.fill(0xABCDEF01)
    scale = np.float32(np.sqrt(cols))
    rt.embedding_rows(rt.DeviceBuffer.from_numpy(t), rt.DeviceBuffer.from_numpy(table), out, n, vocab, cols, scale=float(scale))
    known = (t >= 0) & (t < vocab)
    want = np.where(known[:, None], scale * table[np.clip(t, 0, vocab - 1)], np.float32(0))
    got = out.numpy(np.float32)
    assert np.array_equal(got[: n * cols].reshape(n, cols), want)
    assert (out.numpy(np.uint32)[n * cols:] == 0xABCDEF01).all()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", ["skewed", "padded", "one token", "distinct", "none"])
def test_gradient_of_integers_is_exact(rt, shape, kind):
    n, vocab, cols = shape
    rng = np.random.default_rng([n, vocab, cols])
    t = {"skewed": lambda: tokens_for(n, vocab, 1), "padded": lambda: tokens_for(n, vocab, 2, pad=0.5), "one token": lambda: np.full(n, vocab - 1, np.int32),
         "distinct": lambda: rng.permutation(max(n, vocab))[:n].astype(np.int32), "none": lambda: np.where(np.arange(n) % 2, -1, vocab).astype(np.int32)}[kind]()
    dy = rng.integers(-4, 5, (n, cols)).astype(np.float32)
    d = rt.DeviceBuffer(vocab * cols + 64)
    d.fill(0x7FC00000)  # NaN wherever nothing is written
    rt.embedding_rows_backward(rt.DeviceBuffer.from_numpy(t), rt.DeviceBuffer.from_numpy(dy), d, n, vocab, cols, scale=0.25)
    got = d.numpy(np.float32)
    assert np.array_equal(got[: vocab * cols].reshape(vocab, cols), (0.25 * gradient(t, dy, vocab)).astype(np.float32))
    assert np.isnan(got[vocab * cols:]).all()


@pytest.mark.parametrize("shape", [(77, 1009, 250), (500, 20, 64), (3000, 50, 100), (8193, 5000, 5), (20000, 300, 36), (60000, 7, 16), (131073, 70000, 4)])
def test_gradient_of_reals_and_the_same_again(rt, shape):
    n, vocab, cols = shape
    t = tokens_for(n, vocab, 3, pad=0.1)
    dy = np.random.default_rng(n).normal(size=(n, cols)).astype(np.float32)
    tb, dyb = rt.DeviceBuffer.from_numpy(t), rt.DeviceBuffer.from_numpy(dy)
    d = rt.DeviceBuffer(vocab * cols)
    scale = np.float32(np.sqrt(cols))
    rt.embedding_rows_backward(tb, dyb, d, n, vocab, cols, scale=float(scale))
    got = d.numpy(np.float32, (vocab, cols))
    counts = np.bincount(t[(t >= 0) & (t < vocab)], minlength=vocab)[:, None]
    want, size = scale * gradient(t, dy, vocab), scale * gradient(t, np.abs(dy), vocab)
    assert (np.abs(got - want) <= (counts + 2) * U * size).all()
    for _ in range(3):  # atomics would change the last bits
        d.fill(0)
        rt.embedding_rows_backward(tb, dyb, d, n, vocab, cols, scale=float(scale))
        assert np.array_equal(d.numpy(np.float32, (vocab, cols)), got)


@pytest.mark.parametrize("words", [1, 2, 3])
def test_addresses_that_are_only_word_aligned(rt, words):
    n, vocab, cols = 300, 57, 64
    t = tokens_for(n, vocab, 4, pad=0.1)
    rng = np.random.default_rng(6)
    table, dy = rng.normal(size=(vocab, cols)).astype(np.float32), rng.integers(-4, 5, (n, cols)).astype(np.float32)

    def shifted(arr):
        whole = rt.DeviceBuffer(arr.size + 8)
        whole.write(arr.reshape(-1), offset_words=words)
        view = rt.DeviceBuffer.view(whole.ptr + 4 * words, arr.size)
        view.whole = whole
        return view

    tb, out, d = shifted(t), shifted(np.zeros(n * cols, np.float32)), shifted(np.zeros(vocab * cols, np.float32))
    rt.embedding_rows(tb, shifted(table), out, n, vocab, cols)
    assert np.array_equal(out.numpy(np.float32, (n, cols)), np.where((t >= 0)[:, None], table[np.clip(t, 0, vocab - 1)], np.float32(0)))
    rt.embedding_rows_backward(tb, shifted(dy), d, n, vocab, cols)
    assert np.array_equal(d.numpy(np.float32, (vocab, cols)), gradient(t, dy, vocab).astype(np.float32))


def test_nan_and_infinity_reach_only_the_rows_that_hold_them(rt):
    n, vocab, cols = 400, 30, 20
    t = tokens_for(n, vocab, 5, pad=0.2)
    dy = np.random.default_rng(7).integers(-4, 5, (n, cols)).astype(np.float32)
    hit, pad = int(np.flatnonzero(t >= 0)[0]), int(np.flatnonzero(t < 0)[0])
    dy[hit, 3], dy[pad] = np.inf, np.nan  # a padded position may hold anything
    d = rt.DeviceBuffer(vocab * cols)
    rt.embedding_rows_backward(rt.DeviceBuffer.from_numpy(t), rt.DeviceBuffer.from_numpy(dy), d, n, vocab, cols)
    got = d.numpy(np.float32, (vocab, cols))
    assert np.array_equal(got, gradient(t, dy, vocab).astype(np.float32))
    assert (~np.isfinite(got)).sum() == 1


@pytest.mark.parametrize("shape", [(2047, 300, 20), (2048, 8193, 257), (2048, 7, 1030), (2049, 8193, 64), (2048, 70001, 3), (1, 300000, 5), (40, 1100000, 2), (2000, 1025, 65), (33, 1, 600), (1024, 257, 256)])
@pytest.mark.parametrize("kind", ["skewed", "one token", "runs of 32 and 33", "the last rows", "none"])
def test_gradient_of_few_positions(rt, shape, kind):
    """One launch up to 2048 positions: groups of 8 to 256 rows, rows with up to 32 positions and with more."""
    n, vocab, cols = shape
    rng = np.random.default_rng([n, vocab, cols, 2])
    t = {"skewed": lambda: tokens_for(n, vocab, 7, pad=0.1), "one token": lambda: np.full(n, vocab - 1, np.int32), "runs of 32 and 33": lambda: (np.repeat(np.arange(n), 1 + 31 + np.arange(n) % 2)[:n] % vocab).astype(np.int32),
         "the last rows": lambda: (vocab - 1 - rng.integers(0, min(vocab, 40), n)).astype(np.int32), "none": lambda: np.where(np.arange(n) % 2, np.iinfo(np.int32).min, np.iinfo(np.int32).max).astype(np.int32)}[kind]()
    dy = rng.integers(-4, 5, (n, cols)).astype(np.float32)
    dy[(t < 0) | (t >= vocab)] = np.nan  # nobody's
    d = rt.DeviceBuffer(vocab * cols + 64)
    d.fill(0x7FC00000)
    rt.embedding_rows_backward(rt.DeviceBuffer.from_numpy(t), rt.DeviceBuffer.from_numpy(dy), d, n, vocab, cols, scale=2.0)
    got = d.numpy(np.float32)
    assert np.array_equal(got[: vocab * cols].reshape(vocab, cols), (2.0 * gradient(t, dy, vocab)).astype(np.float32))
    assert np.isnan(got[vocab * cols:]).all()


# on both sides of the sizes at which another kernel takes over: 512 positions, 8192 rows, 512 columns, 4096 and 131072 positions
@pytest.mark.parametrize("shape", [(511, 8191, 511), (512, 8192, 512), (512, 8193, 512), (513, 8192, 64), (512, 9, 513), (512, 7, 512), (65, 8, 130), (4095, 300, 20), (4096, 300, 20), (4097, 300, 20),
                                   (131072, 300, 4), (131073, 300, 4)])
@pytest.mark.parametrize("kind", ["skewed", "one token", "a long run and a short one", "none"])
def test_gradient_beside_the_sizes_where_the_kernel_changes(rt, shape, kind):
    n, vocab, cols = shape
    rng = np.random.default_rng([n, vocab, cols, 1])
    t = {"skewed": lambda: tokens_for(n, vocab, 6, pad=0.1), "one token": lambda: np.full(n, vocab // 2, np.int32),
         "a long run and a short one": lambda: np.where(np.arange(n) % 9 == 4, 0, vocab - 1).astype(np.int32), "none": lambda: np.full(n, vocab, np.int32)}[kind]()
    dy = rng.integers(-4, 5, (n, cols)).astype(np.float32)
    dy[(t < 0) | (t >= vocab)] = np.nan  # nobody's
    d = rt.DeviceBuffer(vocab * cols + 64)
    d.fill(0x7FC00000)
    rt.embedding_rows_backward(rt.DeviceBuffer.from_numpy(t), rt.DeviceBuffer.from_numpy(dy), d, n, vocab, cols, scale=0.5)
    got = d.numpy(np.float32)
    assert np.array_equal(got[: vocab * cols].reshape(vocab, cols), (0.5 * gradient(t, dy, vocab)).astype(np.float32))
    assert np.isnan(got[vocab * cols:]).all()


def test_no_tokens(rt):
    d = rt.DeviceBuffer.from_numpy(np.ones(12, np.float32))
    rt.embedding_rows(d, d, rt.DeviceBuffer(4), 0, 3, 4)
    rt.embedding_rows_backward(d, d, d, 0, 3, 4)
    assert not d.numpy().any()


def test_offsets_past_32_bits(rt):
    """A table of more than 2^32 bytes: the last rows are looked up and get their gradient."""
    vocab, cols, n = 1 << 20, 1100, 5
    t = np.array([vocab - 1, 0, vocab - 1, 1 << 19, -1], np.int32)
    table = rt.DeviceBuffer(vocab * cols)
    table.fill(0)
    rows = {v: np.random.default_rng(v).integers(-8, 9, cols).astype(np.float32) for v in (0, 1 << 19, vocab - 1)}
    for v, r in rows.items():
        table.write(r, offset_words=v * cols)
    tb, out = rt.DeviceBuffer.from_numpy(t), rt.DeviceBuffer(n * cols)
    rt.embedding_rows(tb, table, out, n, vocab, cols, scale=2.0)
    want = np.stack([2 * rows[int(v)] if v >= 0 else np.zeros(cols, np.float32) for v in t])
    assert np.array_equal(out.numpy(np.float32, (n, cols)), want)
    table.fill(0x7FC00000)
    rt.embedding_rows_backward(tb, out, table, n, vocab, cols)
    for v in (0, 1 << 19, vocab - 1):
        assert np.array_equal(table.numpy(np.float32, (cols,), offset_words=v * cols), want[t == v].sum(0)), v
    for v in (1, (1 << 19) - 1, (1 << 19) + 1, vocab - 2):
        assert not table.numpy(np.float32, (cols,), offset_words=v * cols).any(), v
    table.free()


def test_many_rows_of_one_column(rt):
    """A table of 2^29 + 7 rows, more than a launch has waves for: every row is written."""
    vocab = (1 << 29) + 7
    d = rt.DeviceBuffer(vocab)
    d.fill(0x7FC00000)
    t = np.array([0, vocab - 1, 1 << 28, vocab - 1, -1], np.int32)
    rt.embedding_rows_backward(rt.DeviceBuffer.from_numpy(t), rt.DeviceBuffer.from_numpy(np.array([1, 2, 3, 4, 5], np.float32)), d, 5, vocab, 1)
    got = d.numpy()
    assert got[0] == 1 and got[vocab - 1] == 6 and got[1 << 28] == 3
    got[[0, vocab - 1, 1 << 28]] = 0
    assert not got.any()
    d.free()


def test_many_positions_of_one_token(rt):
    """2^28 positions, more parts than a launch has groups of eight waves for. Sums of ones over 64 and more positions are multiples
    of 64 below 2^29: exact."""
    n = 1 << 28
    t, dy, d = rt.DeviceBuffer(n), rt.DeviceBuffer(n), rt.DeviceBuffer(10)
    t.fill(7)
    dy.fill(0x3F800000)
    rt.embedding_rows_backward(t, dy, d, n, 10, 1, scale=0.5)
    assert np.array_equal(d.numpy(), np.where(np.arange(10) == 7, n / 2, 0).astype(np.float32))
    for b in (t, dy):
        b.free()
