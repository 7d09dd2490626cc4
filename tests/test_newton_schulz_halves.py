"""Every product of the orthogonalisation takes both halves of both its operands: matrices on which the loss of one low half, or
of its product with the other operand's high half, shows in every element.

On matrices of random numbers it does not: the low halves' signs are random, and what is lost averages out over a long product. So
G = p q^T here, p and q powers of two times random signs. Then X = p q^T / (|p| |q|) has one mantissa in all elements, X X^T =
p p^T / |p|^2 another, all singular values but one are 0 and that one is 1: a step gives (a + b + c) X. All terms of an
element of a product have one sign, and a dropped low half makes each of them, and so the element, wrong by the same part. p and q are
drawn until that part is at least FRACTION for both mantissas (at most 2^-11 = 4.9e-4 is possible).

Bounds, element by element and relative, since nothing cancels: with e(K) of one product (its operands' halves, 4 * 2^-22, and a chain of
K / 8 + 16 additions in fp32), r = 2^-22 for storing a value, A is within e(n) + 3 r, A^2 within e(m) + 2 that, B within what its terms are
and r, B X within e(m) + r and that of B. One step's coefficients at a time: (0, 0, 1) is bounded by 1.04e-4 at the largest size here.
The CPU part shows that each loss breaks the bounds; the GPU part that each kernel keeps them.
"""
import numpy as np
import pytest

FRACTION = 2.4e-4
R = 2.0 ** -22
# steps whose coefficients make the parts of a step visible: all three products; B's addend; X's addend; X as it is stored between steps
PROGRAMS = [((0, 0, 1),), ((0, 1, 0),), ((1, 0, 0),), ((1, 0, 0), (0, 0, 1)), ((0, 1, 0), (1, 0, 0))]

# batch, shape, the tiles and which of the three products is cut: every kernel and both orientations
ONE_GROUP, UNCUT = (0, 0), (False, False, False)
CASES = [
    (1, (64, 64), ONE_GROUP, UNCUT), (3, (64, 256), ONE_GROUP, UNCUT), (2, (128, 40), ONE_GROUP, UNCUT),
    (1, (300, 300), (32, 32), UNCUT), (2, (129, 260), (32, 32), UNCUT),
    (1, (1000, 1020), (64, 64), UNCUT), (4, (1020, 1000), (64, 128), UNCUT), (16, (1000, 1020), (128, 256), UNCUT), (25, (1000, 1020), (256, 128), UNCUT), (16, (1020, 1000), (128, 256), UNCUT),
    (1, (1400, 1530), (64, 64), (False, False, True)), (1, (1300, 3400), (64, 128), (False, False, True)), (1, (2000, 4100), (64, 128), (True, True, True)), (1, (4100, 2000), (64, 128), (True, True, True)),
    (1, (3000, 3000), (128, 128), (True, True, True)),
]


def e(k):
    return 4 * 2.0 ** -22 + (k / 8 + 16) * 2.0 ** -24


def bound(program, m, n, r=R):
    x = 2 * r  # what X is off by, relative: the norm, the split
    for a, b, c in program:
        gram = e(n) + 2 * x + r
        square = e(m) + 2 * gram + r
        poly = b * gram + c * square + (b + c) * r
        x = a * x + (b + c) * (e(m) + x) + poly + r
    return x + 2 * r


def fraction(v):
    """How much of v its low half holds."""
    v = v * 2.0 ** (14 - np.floor(np.log2(v)))
    return abs(v - float(np.float16(v))) / v


def rank_one(shape, seed):
    """p, q for a matrix of this shape, drawn until both mantissas have large low halves."""
    for attempt in range(2000):
        rng = np.random.default_rng([*shape, seed, attempt])
        p, q = (2.0 ** -rng.integers(0, 3, k) * rng.choice([-1.0, 1.0], k) for k in shape)
        short = np.linalg.norm(p if shape[0] <= shape[1] else q)
        if fraction(1 / (np.linalg.norm(p) * np.linalg.norm(q))) >= FRACTION and fraction(1 / short ** 2) >= FRACTION:
            return p, q
    raise AssertionError("no such p and q")


def expected(p, q, eps=1e-7):
    norm = np.linalg.norm(p) * np.linalg.norm(q)
    return np.outer(p, q) / (norm + eps)  # s = norm / (norm + eps): within 1e-8 of 1 here, and so are its powers


def model(p, q, program, lost):
    """The recurrence with operands in halves and sums in 64 bits. lost: (what, which) that is left out: a product's high times low ('hl')
    or low times high, or the low half of an addend."""
    def scale(top):
        return 2.0 ** (15 - np.frexp(top)[1])

    def split(v):
        hi = v.astype(np.float16)
        return hi.astype(np.float64), (v - hi).astype(np.float16).astype(np.float64)

    def product(what, P, Q):
        t = P[0] @ Q[0].T
        return t + (0 if (what, "hl") == lost else P[0] @ Q[1].T) + (0 if (what, "lh") == lost else P[1] @ Q[0].T)

    def added(what, V):
        return V[0] if (what, "lo") == lost else V[0] + V[1]

    x = expected(p, q)
    x = x if x.shape[0] <= x.shape[1] else x.T
    at = 2.0 ** 14
    x = split(x * at)
    for k, (a, b, c) in enumerate(program):
        to = scale(1.0001)
        A = split((product("gram", x, x) * (to / at ** 2)).astype(np.float32))
        B = split((product("poly", A, A) * (c / to)).astype(np.float32) + b * added("addend of B", A))
        last = k + 1 == len(program)
        y = product("update", B, (x[0].T, x[1].T)) / (to * at) + added("addend of X", x) * (a / at)
        x = split(y * at) if not last else y
    return x


def worst(got, want):
    return float(np.max(np.abs(got - want) / np.abs(want)))


@pytest.mark.parametrize("case", CASES, ids=str)
def test_a_lost_half_is_more_than_the_bounds(case):
    m, n = sorted(case[1])
    for program in PROGRAMS:
        assert bound(program, m, n) < 0.8 * FRACTION, program


@pytest.mark.parametrize("shape", [(300, 320), (1000, 1020)])
def test_the_bounds_see_every_lost_half(shape):
    p, q = rank_one(shape, 0)
    want = expected(p, q)
    for program in PROGRAMS:
        assert worst(model(p, q, program, None), want) <= bound(program, *shape)
    for what, which, program in (("gram", "hl", 0), ("gram", "lh", 0), ("poly", "hl", 0), ("poly", "lh", 0), ("update", "hl", 0), ("update", "lh", 0),
                                 ("addend of B", "lo", 1), ("addend of X", "lo", 2), ("addend of X", "lo", 3), ("update", "hl", 4), ("update", "lh", 4)):
        assert worst(model(p, q, PROGRAMS[program], (what, which)), want) > bound(PROGRAMS[program], *shape), (what, which, program)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_every_kernel_keeps_both_halves(rt, case):
    import ctypes as C

    from tensorfrost_amd._lib import call

    batch, shape, tiles, cut = case
    t, c = (C.c_int * 2)(), (C.c_uint * 3)()
    call("tfhip_test_newton_schulz_tiles", batch, *shape, t, c)
    assert tuple(t) == tiles and tuple(v > 1 for v in c) == cut, (tuple(t), tuple(c))
    pairs = [rank_one(shape, k) for k in range(min(batch, 3))]
    g = np.stack([np.outer(*pairs[k % len(pairs)]) for k in range(batch)]).astype(np.float32)
    gb, out = rt.DeviceBuffer.from_numpy(g), rt.DeviceBuffer(g.size)
    for program in PROGRAMS:
        out.fill(0x7FC00000)
        rt.newton_schulz(gb, out, *shape, steps=len(program), batch=batch, coefficients=program)
        got = out.numpy(np.float32, g.shape)
        for k in {0, batch // 2, batch - 1}:
            want = expected(*pairs[k % len(pairs)])
            assert worst(got[k], want) <= bound(program, *sorted(shape)), (program, k)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 200), (200, 1), (40, 60), (1, 300), (300, 300), (1000, 1020)])
def test_how_well_small_elements_are_held(rt, shape):
    """X <- X. One row holds elements from 1 to 2^-45 of the norm, so that X has norm 1: each is held to 2^-23 of itself or, where that is more,
    to 2^-39; the norm, the factor and the sum of the halves round by 2^-24 each."""
    rng = np.random.default_rng(shape)
    g = np.zeros(shape, np.float32)
    line = g[:, 0] if shape[1] == 1 else g[shape[0] // 2]
    line[:] = 2.0 ** -rng.uniform(0, 45, line.size) * rng.choice([-1.0, 1.0], line.size)
    line[line.size // 3] = 3.0
    gb, out = rt.DeviceBuffer.from_numpy(g), rt.DeviceBuffer(g.size)
    rt.newton_schulz(gb, out, *shape, steps=1, coefficients=(1, 0, 0), eps=0.0)
    want = g.astype(np.float64) / np.linalg.norm(g.astype(np.float64))
    off = np.abs(out.numpy(np.float32, shape) - want)
    assert (off <= np.maximum(2.0 ** -23 * np.abs(want), 2.0 ** -39) + 3 * 2.0 ** -24 * np.abs(want)).all()
    assert off.max() > 0  # and not all of them better than that
