"""Many Newton-Schulz steps. X and X^T are both kept between steps; a step multiplies a difference between the two copies by its first
coefficient whatever X is, while it brings X itself back to a s + b s^3 + c s^5 of its singular values. So a difference of one last bit
would be all of the result after some twenty steps: the copies have to be equal to the bit.

Bounds. The cubic and the quintic with p(1) = 1, p'(1) = 0 grow X to orthogonal, where an error of its singular values dies out; a step adds at
most 8 * 2^-22 for what it stores and rounds and 2 e(K) for its products, none of which grows relative to X: 64 of those. The common quintic
has no fixed point but an interval, [0.68, 1.14] once there: its singular values are looked at.
"""
import numpy as np
import pytest

from test_newton_schulz_halves import e

pytestmark = pytest.mark.gpu
SHAPES = [(20, 50), (50, 20), (64, 64), (64, 256), (200, 60), (1, 200), (256, 3), (33, 129), (100, 120), (300, 300), (257, 600)]


def run(rt, g, **kw):
    gb, out = rt.DeviceBuffer.from_numpy(g), rt.DeviceBuffer(g.size)
    rt.newton_schulz(gb, out, *g.shape, **kw)
    return out.numpy(np.float32, g.shape).astype(np.float64)


def recurrence(g, steps, abc):
    a, b, c = (float(np.float32(v)) for v in abc)
    x = g.astype(np.float64)
    x = x / (np.linalg.norm(x) + float(np.float32(1e-7)))
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    for _ in range(steps):
        gram = x @ x.T
        x = a * x + (b * gram + c * gram @ gram) @ x
    return x.T if tall else x


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("abc", [(1.5, -0.5, 0.0), (1.875, -1.25, 0.375)])
@pytest.mark.parametrize("steps", [20, 40, 64])
def test_orthogonal_stays_orthogonal(rt, shape, abc, steps):
    g = np.random.default_rng(shape).standard_normal(shape).astype(np.float32)
    want = recurrence(g, steps, abc)
    assert np.linalg.norm(run(rt, g, steps=steps, coefficients=abc) - want) <= steps * (8 * 2.0 ** -22 + 2 * e(max(shape))) * np.linalg.norm(want)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("steps", [20, 33, 64])
def test_the_common_quintic_keeps_its_interval(rt, shape, steps):
    g = np.random.default_rng(shape).standard_normal(shape).astype(np.float32)
    values = np.linalg.svd(recurrence(g, steps, (3.4445, -4.7750, 2.0315)), compute_uv=False)
    assert 0.68 < values.min() and values.max() < 1.14
    values = np.linalg.svd(run(rt, g, steps=steps), compute_uv=False)
    assert 0.67 < values.min() and values.max() < 1.15
