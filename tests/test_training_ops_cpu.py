"""What the training operators refuse, checked before any device is needed: the C entry points look at their arguments
first and at the library's state last, so on a machine without a GPU a call that passes every check ends with
TFHIP_ERR_STATE and a call that does not with TFHIP_ERR_ARG."""
import ctypes as C
import math

import numpy as np
import pytest

from tensorfrost_amd import _lib, runtime

ARG, STATE = -3, -4
BASE = 0x10000000  # addresses that are never touched: every call here ends before a kernel


def status(func, *args):
    return getattr(_lib.load(), func)(*args)


def message():
    return _lib.load().tfhip_last_error().decode()


@pytest.fixture(autouse=True)
def _without_a_device():
    if status("tfhip_sync") != STATE:  # bound to a device: the allowed calls would run
        pytest.skip("the library is bound to a device in this process")


def at(k):
    return BASE + k * (1 << 24)


def norm(x=at(0), w=at(1), b=at(2), y=at(3), mean=at(4), rstd=at(5), rows=8, cols=16, eps=1e-5):
    return status("tfhip_layer_norm_rows_f32", x, w, b, y, mean, rstd, rows, cols, eps)


def norm_back(x=at(0), dy=at(1), w=at(2), mean=at(3), rstd=at(4), dx=at(5), dw=at(6), db=at(7), rows=8, cols=16):
    return status("tfhip_layer_norm_rows_backward_f32", x, dy, w, mean, rstd, dx, dw, db, rows, cols)


def embed(tokens=at(0), table=at(1), out=at(2), n=8, vocab=10, cols=16, scale=1.0):
    return status("tfhip_embedding_rows_f32", tokens, table, out, n, vocab, cols, scale)


def embed_back(tokens=at(0), dy=at(1), dtable=at(2), n=8, vocab=10, cols=16, scale=1.0):
    return status("tfhip_embedding_rows_backward_f32", tokens, dy, dtable, n, vocab, cols, scale)


MUON = (C.c_float * 3)(3.4445, -4.7750, 2.0315)


def schulz(g=at(0), out=at(1), batch=1, rows=8, cols=16, steps=1, coefficients=MUON, eps=1e-7):
    return status("tfhip_newton_schulz_f32", g, out, batch, rows, cols, steps, coefficients, eps)


@pytest.mark.parametrize("call", [
    lambda: norm(), lambda: norm(w=None, b=None, mean=None, rstd=None), lambda: norm(y=at(0)), lambda: norm(eps=0.0),
    lambda: norm_back(), lambda: norm_back(w=None), lambda: norm_back(dx=at(0)), lambda: norm_back(dx=at(1)), lambda: norm_back(dx=None), lambda: norm_back(dw=None, db=None),
    lambda: norm_back(rows=0, x=None, dy=None, mean=None, rstd=None),
    lambda: embed(), lambda: embed_back(), lambda: embed_back(n=0, tokens=None, dy=None),
    lambda: schulz(), lambda: schulz(out=at(0)), lambda: schulz(rows=32768, cols=65535, out=at(0)), lambda: schulz(rows=65535, cols=32768, out=at(0)), lambda: schulz(eps=0.0),
])
def test_allowed_calls_get_as_far_as_the_device(call):
    assert call() == STATE, message()
    assert "tfhip_init" in message()


@pytest.mark.parametrize("call", [lambda: norm(rows=0), lambda: norm(rows=0, x=None, y=None), lambda: embed(n=0), lambda: embed(n=0, tokens=None, out=None), lambda: schulz(batch=0)])
def test_empty_calls_are_no_ops(call):
    assert call() == 0, message()


@pytest.mark.parametrize("call, text", [
    (lambda: norm(x=None), "null"), (lambda: norm(y=None), "null"), (lambda: norm(cols=0), "without columns"), (lambda: norm(rows=1 << 31), "beyond"), (lambda: norm(cols=1 << 31), "beyond"),
    (lambda: norm(eps=-1e-5), "eps"), (lambda: norm(eps=math.nan), "eps"), (lambda: norm(eps=math.inf), "eps"),
    (lambda: norm(y=at(0) + 4), "x and y overlap"), (lambda: norm(y=at(0) - 4), "x and y overlap"), (lambda: norm(y=at(1)), "overlap"), (lambda: norm(mean=at(0)), "x and mean overlap"),
    (lambda: norm(mean=at(5)), "mean and rstd overlap"), (lambda: norm(rstd=at(3) + 4 * (8 * 16 - 1)), "y and rstd overlap"), (lambda: norm(mean=at(2)), "bias and mean overlap"),
    (lambda: norm_back(x=None), "null"), (lambda: norm_back(dy=None), "null"), (lambda: norm_back(mean=None), "null"), (lambda: norm_back(rstd=None), "null"),
    (lambda: norm_back(dx=None, dw=None, db=None), "none of"), (lambda: norm_back(cols=0), "without columns"),
    (lambda: norm_back(dx=at(0) + 4), "x and dx overlap"), (lambda: norm_back(dx=at(1) + 4), "dy and dx overlap"), (lambda: norm_back(dw=at(7)), "dweight and dbias overlap"),
    (lambda: norm_back(dw=at(2)), "weight and dweight overlap"), (lambda: norm_back(db=at(5)), "dx and dbias overlap"), (lambda: norm_back(dx=at(3)), "mean and dx overlap"),
    (lambda: norm_back(dx=at(0), dy=at(0) + 64), "overlap"),
    (lambda: embed(tokens=None), "null"), (lambda: embed(table=None), "null"), (lambda: embed(out=None), "null"), (lambda: embed(vocab=0), "empty"), (lambda: embed(cols=0), "empty"),
    (lambda: embed(n=1 << 30), "2^30"), (lambda: embed(vocab=1 << 31), "beyond"), (lambda: embed(out=at(1)), "overlaps"), (lambda: embed(out=at(0)), "overlaps"),
    (lambda: embed(out=at(1) + 4 * 159), "overlaps"), (lambda: embed_back(tokens=None), "null"), (lambda: embed_back(dy=None), "null"), (lambda: embed_back(dtable=None), "null"),
    (lambda: embed_back(n=0, dtable=None), "null"), (lambda: embed_back(dtable=at(1)), "overlaps"), (lambda: embed_back(dtable=at(0)), "overlaps"), (lambda: embed_back(vocab=0), "empty"),
    (lambda: schulz(g=None), "null"), (lambda: schulz(out=None), "null"), (lambda: schulz(coefficients=None), "null"), (lambda: schulz(rows=0), "empty"), (lambda: schulz(cols=0), "empty"),
    (lambda: schulz(steps=0), "steps"), (lambda: schulz(steps=65, coefficients=(C.c_float * 195)()), "steps"), (lambda: schulz(steps=-1), "steps"), (lambda: schulz(out=at(0) + 4), "overlap"),
    (lambda: schulz(rows=32769, cols=32769), "32768"), (lambda: schulz(rows=32768, cols=65536), "32768"), (lambda: schulz(rows=1 << 60, cols=1 << 60), "32768"),
    (lambda: schulz(rows=1 << 24, cols=1), "32768"), (lambda: schulz(batch=65536), "65535"),
    (lambda: schulz(eps=-1.0), "eps"), (lambda: schulz(eps=math.nan), "eps"), (lambda: schulz(coefficients=(C.c_float * 3)(1.0, math.nan, 0.0)), "coefficient 1"),
    (lambda: schulz(steps=2, coefficients=(C.c_float * 6)(1, 0, 0, 1, 0, math.inf)), "coefficient 5"),
])
def test_refused_calls_say_why(call, text):
    assert call() == ARG, message()
    assert text in message()


def buf(words):
    return runtime.DeviceBuffer.view(BASE, words)


def test_buffers_that_are_too_small_are_refused_by_the_python_calls():
    small, big = buf(10), buf(1000)
    for f in (lambda: runtime.layer_norm_rows(small, big, big, big, 8, 16), lambda: runtime.layer_norm_rows(big, small, big, big, 8, 16), lambda: runtime.layer_norm_rows(big, big, big, big, 8, 16, mean=buf(7)),
              lambda: runtime.layer_norm_rows_backward(big, big, big, big, big, 8, 16, dx=small), lambda: runtime.layer_norm_rows_backward(big, big, big, big, big, 8, 16, dweight=small),
              lambda: runtime.embedding_rows(small, big, big, 11, 5, 16), lambda: runtime.embedding_rows(big, small, big, 11, 5, 16), lambda: runtime.embedding_rows_backward(big, big, small, 5, 10, 16),
              lambda: runtime.newton_schulz(small, big, 8, 16), lambda: runtime.newton_schulz(big, buf(8 * 16 * 3 - 1), 8, 16, batch=3)):
        with pytest.raises(ValueError, match="are needed"):
            f()


@pytest.mark.parametrize("steps, coefficients", [(5, (1.0, 2.0)), (5, np.zeros((4, 3))), (3, np.zeros((3, 4))), (-1, (1.0, 2.0, 3.0))])
def test_coefficients_that_do_not_fit_the_steps(steps, coefficients):
    with pytest.raises((ValueError, _lib.TFHipError)):
        runtime.newton_schulz(buf(1000), buf(1000), 8, 16, steps=steps, coefficients=coefficients)


def test_views_own_nothing():
    v = runtime.DeviceBuffer.view(BASE, 4)
    v.free()
    assert v.ptr is None
    for bad in (0, None, BASE + 2):
        with pytest.raises(ValueError):
            runtime.DeviceBuffer.view(bad, 4)
    with pytest.raises(ValueError):
        runtime.DeviceBuffer.view(BASE, 0)


def test_freed_buffers_are_refused_not_taken_as_left_out():
    """A null pointer means "not given" to the library: no weight, no bias, an output that is not wanted."""
    def gone():
        v = buf(1000)
        v.free()
        return v

    big = buf(1000)
    forward = lambda **kw: runtime.layer_norm_rows(**{**dict(x=big, weight=big, bias=big, y=big, rows=8, cols=16), **kw})  # noqa: E731
    backward = lambda **kw: runtime.layer_norm_rows_backward(**{**dict(x=big, dy=big, weight=big, mean=big, rstd=big, rows=8, cols=16, dx=big), **kw})  # noqa: E731
    lookup = lambda **kw: runtime.embedding_rows(**{**dict(tokens=big, table=big, out=big, n=8, vocab=5, cols=16), **kw})  # noqa: E731
    gradient = lambda **kw: runtime.embedding_rows_backward(**{**dict(tokens=big, dy=big, dtable=big, n=8, vocab=5, cols=16), **kw})  # noqa: E731
    schulz = lambda **kw: runtime.newton_schulz(**{**dict(g=big, out=big, rows=8, cols=16), **kw})  # noqa: E731
    for f, names in ((forward, ("x", "weight", "bias", "y", "mean", "rstd")), (backward, ("x", "dy", "weight", "mean", "rstd", "dx", "dweight", "dbias")),
                     (lookup, ("tokens", "table", "out")), (gradient, ("tokens", "dy", "dtable")), (schulz, ("g", "out"))):
        for name in names:
            with pytest.raises(ValueError, match=f"{name} has been freed"):
                f(**{name: gone()})


@pytest.mark.parametrize("steps", [0, 65, 1 << 28, (1 << 32) + 5])
def test_step_counts_are_looked_at_before_coefficients_are_laid_out(steps):
    """One triple for each of 2^28 steps would take 3 GiB; 2^32 + 5 is 5 in the library's 32 bits."""
    import tracemalloc

    tracemalloc.start()
    with pytest.raises(ValueError, match="1 to 64"):
        runtime.newton_schulz(buf(1000), buf(1000), 8, 16, steps=steps)
    assert tracemalloc.get_traced_memory()[1] < 1 << 20
    tracemalloc.stop()


@pytest.mark.parametrize("call", [
    lambda high, most: embed(table=high, out=high + 64, vocab=most, cols=most, n=1), lambda high, most: embed_back(dtable=high, dy=high + 64, vocab=most, cols=most, n=1),
    lambda high, most: norm(x=high, mean=high + 64, y=high, rows=most, cols=most), lambda high, most: norm_back(x=high, dw=high + 64, dx=None, rows=most, cols=most),
])
def test_overlaps_with_matrices_that_reach_past_the_last_address(call):
    """(2^31 - 1)^2 words of 4 bytes from a usual device address on end beyond 2^64."""
    assert call(0x7F0000000000, (1 << 31) - 1) == ARG and "overlap" in message()


def test_arrays_without_elements_overlap_nothing():
    assert norm_back(rows=0, x=at(6) + 4, dy=at(7) + 4, mean=at(6) + 8, rstd=at(7)) == STATE, message()
