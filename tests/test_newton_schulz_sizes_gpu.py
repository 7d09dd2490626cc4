"""Orthogonalisation at the ends of its sizes: matrices of more than 2^32 bytes, batches that take several work spaces, as many matrices as
a call may have. Matrices of rank one, so that the result is known in closed form on the device: (a + b + c) p q^T / (|p| |q|).

The bounds are those derived in the module that is imported, element by element and relative."""
import pytest

from test_newton_schulz_halves import bound

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def check(rt, batch, m, n, program, several_norms=False):
    gen = torch.Generator("cuda").manual_seed(m + n + batch)
    sign = lambda *s: torch.randint(0, 2, s, generator=gen, device="cuda") * 2 - 1  # noqa: E731
    power = lambda *s: 2.0 ** -torch.randint(0, 3, s, generator=gen, device="cuda").double()  # noqa: E731
    p, q = power(batch, m) * sign(batch, m), power(batch, n) * sign(batch, n)
    if several_norms:
        p *= 2.0 ** torch.randint(-30, 30, (batch, 1), generator=gen, device="cuda").double()
    g = torch.empty(batch, m, n, device="cuda")
    for k in range(0, batch, 4096):
        g[k:k + 4096] = p[k:k + 4096, :, None].float() * q[k:k + 4096, None, :].float()  # powers of two: exact
    out = torch.full_like(g, float("nan"))
    torch.cuda.synchronize()
    rt.newton_schulz(rt.DeviceBuffer.view(g.data_ptr(), g.numel()), rt.DeviceBuffer.view(out.data_ptr(), out.numel()), m, n, steps=len(program), batch=batch, coefficients=program, eps=0.0)
    rt.synchronize()
    factor = 1.0
    for a, b, c in program:
        factor = factor * (a + b * factor ** 2 + c * factor ** 4)
    want = p * (factor / (p.norm(dim=1, keepdim=True) * q.norm(dim=1, keepdim=True)))
    worst = 0.0
    step = max(1, (1 << 27) // n)
    for k in range(batch) if m * n >= 1 << 20 else [None]:
        if k is None:
            w = want[:, :, None] * q[:, None, :]
            worst = max(worst, float(((out.double() - w) / w).abs().nan_to_num(nan=1e9).max()))
            continue
        for r in range(0, m, step):
            w = want[k, r:r + step, None] * q[k, None, :]
            worst = max(worst, float(((out[k, r:r + step].double() - w) / w).abs().nan_to_num(nan=1e9).max()))
    assert worst <= bound(program, *sorted((m, n))), worst


@pytest.mark.parametrize("shape", [(18000, 62000), (62000, 18000)])
def test_matrices_of_more_than_four_gibibytes(rt, shape):
    check(rt, 1, *shape, ((0, 0, 1),))
    torch.cuda.empty_cache()


@pytest.mark.parametrize("batch, shape", [(700, (500, 512)), (30000, (1, 300)), (25000, (300, 1))])
def test_batches_that_take_several_work_spaces(rt, batch, shape):
    """4 GiB hold 682 matrices of 512 x 512 and 24966 of 32 x 320."""
    check(rt, batch, *shape, ((0, 0, 1), (1, 0, 0)), several_norms=True)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("shape", [(3, 5), (64, 7), (1, 1)])
def test_as_many_matrices_as_a_call_takes(rt, shape):
    check(rt, 65535, *shape, ((0, 1, 0), (0, 0, 1)), several_norms=True)
    torch.cuda.empty_cache()
