"""Orthogonalisation by Newton-Schulz products against the same recurrence in float64.

Bounds: the products may hold each operand as a pair of 16-bit halves, which keeps at least 22 bits of a value: an operand
is off by at most 2^-22 of its magnitude (half a last step of the low half, and the dropped product of two low halves
counts as one more), and the fp32 accumulation of k-blocks adds a chain of K / 8 + 16 additions. With
e(K) = 4 * 2^-22 + (K / 8 + 16) * 2^-24, one product P Q is within e(K) |P| |Q| element by element. Carried through one
step: |A| gets e |X||X|^T, and so on; the test evaluates that recurrence with absolute values. Values below 2^-24 of the bound on X
may round on a fixed grid: an absolute 2^-24 * 2^-11 per element of X covers it.
Over several steps the map s -> a s + b s^3 + c s^5 multiplies a perturbation of X by at most max |p'| per step: with the
common coefficients 3.4445 at s = 0, so an error of the first step can grow by 3.4445^4 = 141 and all five together by
less than 200. Relative to |X|_F the five-step results are held to 200 e(K).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
QUINTIC = (3.4445, -4.7750, 2.0315)
SHAPES = [(1, 1), (1, 5), (5, 1), (2, 3), (3, 256), (16, 40), (31, 33), (32, 32), (33, 31), (64, 64), (63, 65), (65, 200), (128, 128), (129, 127), (100, 1000), (1000, 100), (256, 256), (255, 300), (256, 64), (257, 129),
          (384, 400), (512, 512), (700, 513), (1, 4096), (2048, 3)]


def e(k):
    return 4 * 2.0 ** -22 + (k / 8 + 16) * 2.0 ** -24


def step64(x, abc):
    a, b, c = (float(np.float32(v)) for v in abc)
    gram = x @ x.T
    return a * x + (b * gram + c * gram @ gram) @ x


def newton_schulz64(g, steps, abc=QUINTIC, eps=1e-7):
    x = g.astype(np.float64)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (np.linalg.norm(x) + float(np.float32(eps)))
    for k in range(steps):
        x = step64(x, abc[k] if np.ndim(abc) == 2 else abc)
    return x.T if tall else x


def make(rows, cols, seed=0):
    rng = np.random.default_rng([rows, cols, seed])
    r = min(4, rows, cols)
    return (0.02 * (rng.normal(size=(rows, cols)) + rng.normal(size=(rows, r)) @ rng.normal(size=(r, cols)))).astype(np.float32)


def run(rt, g, batch=1, **kw):
    rows, cols = g.shape[-2:]
    gb, out = rt.DeviceBuffer.from_numpy(g), rt.DeviceBuffer(g.size + 64)
    out.fill(0xABCDEF01)
    rt.newton_schulz(gb, out, rows, cols, batch=batch, **kw)
    assert (out.numpy(np.uint32)[g.size:] == 0xABCDEF01).all()
    assert np.array_equal(gb.numpy(np.float32, g.shape), g, equal_nan=True)
    return out.numpy(np.float32, g.shape)


@pytest.mark.parametrize("shape", SHAPES)
def test_one_step_element_by_element(rt, shape):
    g = make(*shape)
    x = g.astype(np.float64)
    x = np.abs(x.T if shape[0] > shape[1] else x) / (np.linalg.norm(x) + 1e-7)
    m, n = x.shape
    a, b, c = (abs(v) for v in QUINTIC)
    # |error| of A = X X^T, of B = a I + b A + c A^2, of B X; x itself is off by 2^-22 |x| and the grid
    dx = 2.0 ** -22 * x + 2.0 ** -35
    gram = x @ x.T
    d_gram = e(n) * gram + dx @ x.T + x @ dx.T
    poly = a * np.eye(m) + b * gram + c * gram @ gram
    d_poly = b * d_gram + c * (e(m) * gram @ gram + 2 * gram @ d_gram) + 2.0 ** -22 * poly + 2.0 ** -35
    bound = e(m) * poly @ x + d_poly @ x + poly @ dx
    bound = bound.T if shape[0] > shape[1] else bound
    got = run(rt, g, steps=1)
    assert (np.abs(got - newton_schulz64(g, 1)) <= bound).all(), float(np.max(np.abs(got - newton_schulz64(g, 1)) / bound))


@pytest.mark.parametrize("shape", SHAPES)
def test_five_steps(rt, shape):
    g = make(*shape, seed=1)
    want, got = newton_schulz64(g, 5), run(rt, g)
    assert np.linalg.norm(got - want) <= 200 * e(max(shape)) * np.linalg.norm(want)
    s = np.linalg.svd(got.astype(np.float64), compute_uv=False)
    assert s[0] < 1.3  # the quintic's largest value over [0, 1.2] is below 1.2
    if max(shape) >= 2 * min(shape):  # well conditioned: every direction arrives
        assert s[-1] > 0.5


@pytest.mark.parametrize("batch, shape", [(2, (256, 256)), (3, (64, 256)), (5, (256, 3)), (7, (33, 31)), (17, (16, 48)), (130, (5, 9))])
def test_a_batch_is_its_matrices_one_by_one(rt, batch, shape):
    g = np.stack([make(*shape, seed=10 + k) * 10.0 ** ((k % 5) - 2) for k in range(batch)]).astype(np.float32)
    got = run(rt, g, batch=batch)
    for k in range(0, batch, max(1, batch // 7)):
        assert np.array_equal(got[k], run(rt, g[k])), k
        want = newton_schulz64(g[k], 5)
        assert np.linalg.norm(got[k] - want) <= 200 * e(max(shape)) * np.linalg.norm(want)


# on both sides of the sizes at which another kernel takes over, in both orientations
@pytest.mark.parametrize("shape", [(64, 65), (64, 128), (64, 129), (64, 256), (64, 257), (65, 65), (65, 256), (1, 256), (1, 257), (17, 31), (48, 250)])
@pytest.mark.parametrize("tall", [False, True])
def test_beside_the_sizes_where_the_kernel_changes(rt, shape, tall):
    batch = 3
    g = np.stack([make(*shape, seed=20 + k) for k in range(batch)])
    g = np.ascontiguousarray(np.swapaxes(g, 1, 2)) if tall else g
    rows, cols = g.shape[1:]
    triples = ((3.9, -8.1, 4.9), QUINTIC, (1.875, -1.25, 0.375))
    got = run(rt, g, batch=batch, steps=3, coefficients=triples)
    b = rt.DeviceBuffer.from_numpy(g)
    rt.newton_schulz(b, b, rows, cols, steps=3, batch=batch, coefficients=triples)
    assert np.array_equal(b.numpy(np.float32, g.shape), got)  # in place
    for k in range(batch):
        want = newton_schulz64(g[k], 3, triples)
        # at most 3.9 * 3.4445 * 1.875 times an error of the first step, three steps' worth of them
        assert np.linalg.norm(got[k] - want) <= 3 * 25.2 * e(max(shape)) * np.linalg.norm(want)


@pytest.mark.parametrize("shape", [(40, 40), (64, 200), (300, 128)])
def test_other_coefficients_and_step_counts(rt, shape):
    g = make(*shape, seed=3)
    # the classical cubic, once and twelve times: p' <= 1.5, so an early error grows by 1.5^k
    cubic = (1.5, -0.5, 0.0)
    for steps in (1, 3, 12):
        want = newton_schulz64(g, steps, cubic)
        assert np.linalg.norm(run(rt, g, steps=steps, coefficients=cubic) - want) <= 3 * 1.5 ** steps * e(max(shape)) * np.linalg.norm(want)
    # a triple of its own for every step, the first with large coefficients: p' <= 8.3 and 4 and 2
    triples = ((8.28721, -23.5959, 17.3004), (4.10706, -2.94785, 0.54484), (1.875, -1.25, 0.375))
    want = newton_schulz64(g, 3, triples)
    assert np.linalg.norm(run(rt, g, steps=3, coefficients=triples) - want) <= 8.3 * 4.2 * 2 * 2 * e(max(shape)) * np.linalg.norm(want)


def test_coefficients_that_blow_up_stay_finite_as_long_as_the_result_is(rt):
    """X <- 100 X, four times: the halves' common scale has to follow."""
    g = make(48, 64, seed=4)
    want = newton_schulz64(g, 4, (100.0, 0.0, 0.0))
    got = run(rt, g, steps=4, coefficients=(100.0, 0.0, 0.0))
    assert np.linalg.norm(got - want) <= 8 * e(64) * np.linalg.norm(want)


@pytest.mark.parametrize("factor", [1e-18, 1e-6, 1.0, 1e8, 1e30])
def test_the_size_of_the_matrix_does_not_matter(rt, factor):
    """Squares that leave the range of fp32 on either side: the norm is summed in 64 bits. eps = 0, so X is the same."""
    g = make(40, 90, seed=5).astype(np.float64) * factor
    g = g.astype(np.float32)
    want = newton_schulz64(g, 5, eps=0.0)
    assert np.linalg.norm(run(rt, g, eps=0.0) - want) <= 200 * e(90) * np.linalg.norm(want)


def test_a_norm_far_below_eps(rt):
    """|G| = 1e-3 eps: X is 1e-3 of a normalised matrix, still far above the halves' grid."""
    g = make(32, 48, seed=6)
    g = (g / np.linalg.norm(g) * 1e-10).astype(np.float32)
    want = newton_schulz64(g, 5)
    got = run(rt, g)
    assert np.linalg.norm(got - want) <= (200 * e(48) + 500 * 2.0 ** -35 * 1e3 * np.sqrt(32 * 48)) * np.linalg.norm(want)


def test_zeros_nan_and_infinity(rt):
    assert not run(rt, np.zeros((40, 50), np.float32)).any()
    assert not run(rt, np.zeros((40, 50), np.float32), eps=0.0).any()
    for bad in (np.nan, np.inf, -np.inf):
        g = np.stack([make(40, 50, seed=7), make(40, 50, seed=8), make(40, 50, seed=9)])
        clean = run(rt, g, batch=3)
        g[1, 7, 9] = bad
        got = run(rt, g, batch=3)
        assert np.isnan(got[1]).all() and np.array_equal(got[0], clean[0]) and np.array_equal(got[2], clean[2])


@pytest.mark.parametrize("shape", [(48, 70), (200, 64), (300, 300)])
def test_in_place_and_rank_deficient(rt, shape):
    rows, cols = shape
    rng = np.random.default_rng(11)
    g = (rng.normal(size=(rows, 2)) @ rng.normal(size=(2, cols))).astype(np.float32)  # rank 2 up to its own rounding
    want = run(rt, g)
    b = rt.DeviceBuffer.from_numpy(g)
    rt.newton_schulz(b, b, rows, cols)
    assert np.array_equal(b.numpy(np.float32, shape), want)
    assert np.linalg.norm(want - newton_schulz64(g, 5)) <= 200 * e(max(shape)) * np.linalg.norm(want)


def test_word_aligned_addresses(rt):
    g = make(70, 90, seed=12)
    whole, out = rt.DeviceBuffer(g.size + 4), rt.DeviceBuffer(g.size + 4)
    whole.write(g.reshape(-1), offset_words=1)
    rt.newton_schulz(rt.DeviceBuffer.view(whole.ptr + 4, g.size), rt.DeviceBuffer.view(out.ptr + 12, g.size), 70, 90)
    assert np.array_equal(out.numpy(np.float32, g.shape, offset_words=3), run(rt, g))


@pytest.mark.parametrize("batch, shape", [(4, (1000, 1020)), (16, (1020, 1000)), (16, (1000, 1020)), (25, (1000, 1020)), (1, (2100, 2051)), (1, (3600, 65))])
def test_many_tiles(rt, batch, shape):
    """Enough work for the large tiles (128 and 256 rows and columns), with ragged edges, against float64 for the first and the
    last matrix of the batch; and the same words when it runs again."""
    rng = np.random.default_rng([batch, *shape])
    g = (rng.standard_normal((batch, *shape), dtype=np.float32) + rng.standard_normal((batch, shape[0], 4), dtype=np.float32) @ rng.standard_normal((batch, 4, shape[1]), dtype=np.float32))
    steps = 2
    got = run(rt, g, batch=batch, steps=steps)
    for k in {0, batch - 1}:
        want = newton_schulz64(g[k], steps)
        # two steps: the first's error grows by at most 3.4445
        assert np.linalg.norm(got[k] - want) <= 3 * 3.5 * e(max(shape)) * np.linalg.norm(want)
    assert np.array_equal(run(rt, g, batch=batch, steps=steps), got)


@pytest.mark.parametrize("shape", [(1300, 3400), (3400, 1300), (2000, 4100), (2990, 3000), (3500, 3500), (2040, 2010), (1500, 2960)])
def test_products_whose_last_tiles_are_cut_along_k(rt, shape):
    """More tiles of 64 or 128 than compute units: those left over are worked on in parts, whose sums meet in a fixed order."""
    rng = np.random.default_rng(shape)
    g = rng.standard_normal(shape, dtype=np.float32) + rng.standard_normal((shape[0], 4), dtype=np.float32) @ rng.standard_normal((4, shape[1]), dtype=np.float32)
    got = run(rt, g, steps=2)
    want = newton_schulz64(g, 2)
    # two steps: the first's error grows by at most 3.4445
    assert np.linalg.norm(got - want) <= 3 * 3.5 * e(max(shape)) * np.linalg.norm(want)
    # no tile is off: every block of 32 x 32 by itself, against the size of a row and column of blocks
    off = np.abs(got - want)
    bound = 3 * 3.5 * e(max(shape)) * np.linalg.norm(want) / np.sqrt(want.size) * 64
    assert off.max() <= bound
    assert np.array_equal(run(rt, g, steps=2), got)
