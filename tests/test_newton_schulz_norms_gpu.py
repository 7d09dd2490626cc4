"""Orthogonalisation of matrices whose norm is far below eps, a layer that hardly gets a gradient: X = G / (|G| + eps) is small then, and
so is the result, with as many correct digits as that of any other matrix.

The scales of the halves follow a power of two that |X| does not exceed and is above half of. Elements below 2^-16 of the bound on their matrix are
held to 2^-39 of it. On the matrices of rank one below, the smallest element is 2^-14.4 of the norm at the largest size; the bound may be
twice |X|, eight times |A| and |B| and sixteen times the next |X| (its power, and the next power of two): elements down to 2^-18.4 of
it, which are held to 2^-20.6 of themselves. So r = 2^-20 takes the place of 2^-22 in the bounds that are derived beside the imported ones.
"""
import numpy as np
import pytest

from test_newton_schulz_halves import CASES, bound, e, rank_one

pytestmark = pytest.mark.gpu
EPS = float(np.float32(1e-7))
QUINTIC = (3.4445, -4.7750, 2.0315)


def run(rt, g, batch=1, **kw):
    gb, out = rt.DeviceBuffer.from_numpy(g), rt.DeviceBuffer(g.size)
    out.fill(0x7FC00000)
    rt.newton_schulz(gb, out, *g.shape[-2:], batch=batch, **kw)
    return out.numpy(np.float32, g.shape)


def powers_of_two(v):
    """fp32 words of powers of two down to 2^-149, by their bits: libraries built for fast math make the host's own conversion flush what is
    below 2^-126 to zero."""
    k = np.round(np.log2(np.abs(v))).astype(np.int64)
    words = np.where(k >= -126, (np.maximum(k, -126) + 127) << 23, 1 << np.clip(k + 149, 0, 22)) | np.where(v < 0, 1 << 31, 0)
    return words.astype(np.uint32).view(np.float32)


@pytest.mark.parametrize("case", [c for c in CASES if c[1] != (4100, 2000)], ids=str)
def test_every_kernel_keeps_the_digits_of_a_small_matrix(rt, case):
    """Down to results of about 2^-100: (0, 0, 1) gives the fifth power of |X|."""
    batch, shape = case[:2]
    p, q = rank_one(shape, 0)
    norm = np.linalg.norm(p) * np.linalg.norm(q)
    for program, smallest in ((((1, 0, 0),), 90), (((0, 1, 0),), 30), (((0, 0, 1),), 18), (((1, 0, 0), (0, 0, 1)), 18), (((0, 1, 0), (1, 0, 0)), 30), (((2, 1, 0), (3, 0, 1)), 60)):
        for below in (1, 3, 9, smallest):
            t = 2.0 ** (np.round(np.log2(EPS / norm)) - below)
            g = np.broadcast_to(powers_of_two(np.outer(p, q) * t), (batch, *shape)).copy()
            s = norm * t / (norm * t + EPS)
            want = np.outer(p, q) * t / (norm * t + EPS)
            for a, b, c in program:
                by = a + b * s ** 2 + c * s ** 4
                want, s = want * by, s * by
            got = run(rt, g, batch=batch, steps=len(program), coefficients=program)
            for k in {0, batch - 1}:
                worst = np.max(np.abs(got[k] - want) / np.abs(want))
                assert worst <= bound(program, *sorted(shape), r=2.0 ** -20), (program, below, worst)


@pytest.mark.parametrize("shape", [(64, 64), (256, 40), (300, 300), (129, 400), (1000, 1020), (2100, 2051)])
@pytest.mark.parametrize("size", [1e-12, 1e-13, 1e-14, 1e-18, 1e-25, 1e-32])
def test_five_steps_of_a_gradient_far_below_eps(rt, shape, size):
    """|X| <= 1e-5: five steps multiply it by 3.4445 each but for 4e-5 of it, whose own error does not count. Each step stores X, to 2^-23, and
    rounds its halves' sum, their factor and the sum with B X by 2^-24: 5 * 2.5 * 2^-23, and the first X: 8 * 2^-22 together. Small
    elements' 2^-39 of the bound add sqrt(mn) 2^-38 = 2^-27 of the norm."""
    rng = np.random.default_rng(shape)
    g = rng.standard_normal(shape)
    g = (g / np.linalg.norm(g) * size).astype(np.float32)
    x = g.astype(np.float64)
    x = x / (np.linalg.norm(x) + EPS)
    a, b, c = (float(np.float32(v)) for v in QUINTIC)
    for _ in range(5):
        gram = x @ x.T
        x = a * x + (b * gram + c * gram @ gram) @ x
    got = run(rt, g)
    assert np.linalg.norm(got - x) <= 8 * 2.0 ** -22 * np.linalg.norm(x)


@pytest.mark.parametrize("shape", [(30, 50), (64, 256), (100, 120)])
def test_a_matrix_is_scaled_by_its_own_norm(rt, shape):
    """A batch of large, small, zero and undefined matrices: each comes out as it does alone."""
    rng = np.random.default_rng(shape)
    g = rng.standard_normal((7, *shape)).astype(np.float32)
    for k, size in enumerate((1.0, 1e-12, 1e-9, 0.0, 1e-20, 1e8, 1.0)):
        g[k] *= np.float32(size)
    g[6, 1, 2] = np.nan
    got = run(rt, g, batch=7)
    assert not got[3].any() and np.isnan(got[6]).all()
    for k in range(7):
        assert np.array_equal(got[k], run(rt, g[k]), equal_nan=True), k
    assert np.array_equal(run(rt, g, batch=7), got, equal_nan=True)


@pytest.mark.parametrize("shape", [(64, 64), (200, 300)])
def test_a_recorded_call_follows_the_norm(rt, shape):
    """The scale is found by the device: a graph recorded with an ordinary gradient is replayed with smaller and larger ones."""
    rng = np.random.default_rng(shape)
    g = rng.standard_normal(shape).astype(np.float32)
    gb, out = rt.DeviceBuffer.from_numpy(g), rt.DeviceBuffer(g.size)
    rt.newton_schulz(gb, out, *shape)
    graph = rt.Graph()
    with graph:
        rt.newton_schulz(gb, out, *shape)
    for size in (1.0, 1e-12, 1e-16, 1e3, 1e-9):
        h = g * np.float32(size)
        gb.write(h)
        want = run(rt, h)
        graph.launch()
        assert np.array_equal(out.numpy(np.float32, shape), want), size
    graph.destroy()


@pytest.mark.parametrize("shape", [(20, 50), (150, 70)])
def test_sixty_four_steps_from_far_below_eps_to_orthogonal(rt, shape):
    """The cubic from |X| = 1e-5 on: it grows by 1.5 a step until the singular values are 1, where an error no longer grows. Each of the
    64 steps adds at most 8 * 2^-22, as above, and e(K) of the products that bend the growth."""
    rng = np.random.default_rng(shape)
    g = rng.standard_normal(shape)
    g = (g / np.linalg.norm(g) * 1e-12).astype(np.float32)
    x = g.astype(np.float64)
    x = x / (np.linalg.norm(x) + EPS)
    for _ in range(64):
        x = 1.5 * x - 0.5 * x @ x.T @ x
    got = run(rt, g, steps=64, coefficients=(1.5, -0.5, 0.0))
    assert np.linalg.norm(got - x) <= 64 * (8 * 2.0 ** -22 + 2 * e(max(shape))) * np.linalg.norm(x)
    assert abs(np.linalg.svd(got.astype(np.float64), compute_uv=False) - 1).max() < 1e-4
