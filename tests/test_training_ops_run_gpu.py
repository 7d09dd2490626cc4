"""The operators of a training step together, as a program would use them: embedding -> layer norm -> dense layer, back
through all three, the dense layer's gradient orthogonalised; as one host program, as calls recorded into graphs, from two
threads, on memory of another library.

Bounds: u = 2^-24. A chain of sums, each off by at most its number of terms times u relative to the sum of magnitudes, is
carried through the step in magnitudes (the linear parts), as the test states at each output.
"""
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
QUINTIC = (3.4445, -4.7750, 2.0315)


def bits(x):
    return int(np.float32(x).view(np.int32))


def make(n, vocab, cols, k, seed=0):
    rng = np.random.default_rng([n, vocab, cols, k, seed])
    tokens = rng.integers(0, vocab, n).astype(np.int32)
    tokens[:: max(1, n // 4)] = rng.integers(0, vocab)  # one token several times
    tokens[n - n // 10:] = -1                           # the padded end
    f = lambda *s: rng.normal(size=s).astype(np.float32)  # noqa: E731
    dy = f(n, k)
    dy[n - n // 10:] = 0.0
    return tokens, f(vocab, cols), (1 + 0.2 * f(cols)).astype(np.float32), 0.1 * f(cols), f(cols, k) / np.float32(np.sqrt(cols)), dy


def step64(tokens, table, weight, bias, W, dy, eps, scale):
    table, weight, bias, W, dy = (a.astype(np.float64) for a in (table, weight, bias, W, dy))
    known = tokens >= 0
    e = np.where(known[:, None], scale * table[np.clip(tokens, 0, None)], 0.0)
    d = e - e.mean(1, keepdims=True)
    rstd = 1 / np.sqrt((d * d).mean(1, keepdims=True) + eps)
    xhat = d * rstd
    h = xhat * weight + bias
    dW = h.T @ dy
    dh = dy @ W.T
    g = dh * weight
    de = rstd * (g - g.mean(1, keepdims=True) - xhat * (g * xhat).mean(1, keepdims=True))
    dtable = np.zeros_like(table)
    np.add.at(dtable, tokens[known], scale * de[known])
    x = dW if dW.shape[0] <= dW.shape[1] else dW.T
    x = x / (np.linalg.norm(x) + 1e-7)
    for _ in range(5):
        a = x @ x.T
        x = QUINTIC[0] * x + (QUINTIC[1] * a + QUINTIC[2] * a @ a) @ x
    update = x if dW.shape[0] <= dW.shape[1] else x.T
    return h @ W, dtable, (dh * xhat).sum(0), dh.sum(0), update, dict(h=h, xhat=xhat, dh=dh, rstd=rstd, g=g, de=de, dW=dW)


def check_step(got, inputs, eps, scale):
    tokens, table, weight, bias, W, dy = inputs
    n, cols = len(tokens), table.shape[1]
    y, dtable, dweight, dbias, update, s = step64(*inputs, eps, scale)
    aw, ady = np.abs(W.astype(np.float64)), np.abs(dy.astype(np.float64))
    # xhat: mean, centring, sum of squares, reciprocal root: (cols / 64 + 24) u twice, relative to its row's largest
    k_row = 2 * (cols / 64 + 24) * U
    d_xhat = k_row * (1 + np.abs(s["xhat"]).max(1, keepdims=True)) * np.ones_like(s["xhat"])
    d_h = d_xhat * np.abs(weight) + 4 * U * np.abs(s["h"]) + 2 * U * np.abs(bias)
    assert (np.abs(got[0] - y) <= d_h @ aw + (cols + 8) * U * (np.abs(s["h"]) @ aw)).all()
    d_dh = (W.shape[1] + 8) * U * (ady @ aw.T)
    adh, axhat = np.abs(s["dh"]), np.abs(s["xhat"])
    assert (np.abs(got[2] - dweight) <= (d_dh * axhat + adh * d_xhat).sum(0) + (n + 8) * U * (adh * axhat).sum(0) + 1e-30).all()
    assert (np.abs(got[3] - dbias) <= d_dh.sum(0) + (n + 8) * U * adh.sum(0) + 1e-30).all()
    ag, d_g = np.abs(s["g"]), d_dh * np.abs(weight) + 2 * U * np.abs(s["g"])
    m = lambda a: a.mean(1, keepdims=True)  # noqa: E731
    d_de = s["rstd"] * (d_g + m(d_g) + axhat * m(d_g * axhat + ag * d_xhat) + d_xhat * m(ag * axhat) + k_row * (m(ag) + axhat * m(ag * axhat)) + 8 * U * (ag + m(ag) + axhat * m(ag * axhat))) \
        + 2 * k_row * np.abs(s["de"])
    bound = np.zeros_like(dtable)
    known = tokens >= 0
    np.add.at(bound, tokens[known], scale * (d_de + (n + 4) * U * np.abs(s["de"]))[known])
    assert (np.abs(got[1] - dtable) <= bound + 1e-30).all()
    # the update: what X is off by grows by at most 3.4445^5 = 485 on its way, and the products add 200 e(K) (derived with their own test)
    d_dW = d_h.T @ ady + (n + 8) * U * (np.abs(s["h"]).T @ ady)
    e = 4 * 2.0 ** -22 + (max(W.shape) / 8 + 16) * U
    assert np.linalg.norm(got[4] - update) <= 485 * 2 * np.linalg.norm(d_dW) / np.linalg.norm(s["dW"]) + 200 * e * np.linalg.norm(update)


SIZES = [(40, 17, 32, 8), (500, 101, 96, 24), (5000, 300, 256, 64), (9000, 2000, 64, 130)]


@pytest.fixture(scope="module")
def tf(rt):
    from tensorfrost_amd import host

    host.initialize(host.hip)
    return host


@pytest.mark.parametrize("size", SIZES)
def test_the_step_as_one_program(tf, size):
    inputs = make(*size)
    eps, scale = 1e-5, float(np.float32(np.sqrt(size[2])))
    program = tf.compile("embed_norm_dense", [bits(eps), bits(scale)])
    first = [t.numpy for t in program(*inputs)]
    check_step(first, inputs, eps, scale)
    again = [t.numpy for t in program(*inputs)]
    assert all(np.array_equal(a, b) for a, b in zip(first, again))  # the same words every time
    program.destroy()


def test_the_step_recorded_and_replayed(tf):
    size, eps, scale = SIZES[1], 1e-5, 2.0
    program = tf.compile("embed_norm_dense", [bits(eps), bits(scale)])
    inputs = make(*size)
    tensors = [tf.tensor(a) for a in inputs]
    program(*tensors)  # sizes the scratch buffer
    graph = program.record(*tensors)
    other = tf.compile("newton_schulz")
    for k in range(4):
        graph.replay()
        check_step([t.numpy for t in graph.outputs], inputs, eps, scale)
        other(np.random.default_rng(k).normal(size=(2, 60 + 40 * k, 90)).astype(np.float32))  # eager work with its own scratch between replays
        tf.synchronize()
        inputs = make(*size, seed=k + 1)
        for t, a in zip(tensors, inputs):
            t.write(a)
    graph.destroy()
    program.destroy()


def test_each_operator_as_a_program(tf, rt):
    tokens, table, weight, bias, _, _ = make(300, 57, 100, 4)
    rng = np.random.default_rng(0)
    b = {k: rt.DeviceBuffer.from_numpy(v) for k, v in dict(tokens=tokens, table=table, w=weight, b=bias).items()}
    e, y, mean, rstd = rt.DeviceBuffer(300 * 100), rt.DeviceBuffer(300 * 100), rt.DeviceBuffer(300), rt.DeviceBuffer(300)
    rt.embedding_rows(b["tokens"], b["table"], e, 300, 57, 100, scale=3.0)
    got = tf.compile("embedding", [bits(3.0)])(tokens, table).numpy
    assert np.array_equal(got, e.numpy(np.float32, (300, 100)))
    rt.layer_norm_rows(e, b["w"], b["b"], y, 300, 100, eps=1e-3, mean=mean, rstd=rstd)
    norm = [t.numpy for t in tf.compile("layer_norm", [bits(1e-3)])(got, weight, bias)]
    assert np.array_equal(norm[0], y.numpy(np.float32, (300, 100))) and np.array_equal(norm[1], mean.numpy()) and np.array_equal(norm[2], rstd.numpy())
    dy = rng.normal(size=(300, 100)).astype(np.float32)
    dyb, dx, dw, db = rt.DeviceBuffer.from_numpy(dy), rt.DeviceBuffer(300 * 100), rt.DeviceBuffer(100), rt.DeviceBuffer(100)
    rt.layer_norm_rows_backward(e, dyb, b["w"], mean, rstd, 300, 100, dx=dx, dweight=dw, dbias=db)
    back = [t.numpy for t in tf.compile("layer_norm_backward")(got, dy, weight, norm[1], norm[2])]
    assert np.array_equal(back[0], dx.numpy(np.float32, (300, 100))) and np.array_equal(back[1], dw.numpy()) and np.array_equal(back[2], db.numpy())
    d = rt.DeviceBuffer(57 * 100)
    rt.embedding_rows_backward(b["tokens"], dx, d, 300, 57, 100, scale=3.0)
    assert np.array_equal(tf.compile("embedding_backward", [57, bits(3.0)])(tokens, back[0]).numpy, d.numpy(np.float32, (57, 100)))
    g = rng.normal(size=(3, 40, 70)).astype(np.float32)
    gb = rt.DeviceBuffer.from_numpy(g)
    rt.newton_schulz(gb, gb, 40, 70, steps=3, batch=3, coefficients=(1.5, -0.5, 0.0), eps=1e-6)
    assert np.array_equal(tf.compile("newton_schulz", [3, bits(1e-6), bits(1.5), bits(-0.5), bits(0.0)])(g).numpy, gb.numpy(np.float32, g.shape))
    with pytest.raises(tf.TFHostError, match="Newton-Schulz steps"):
        tf.compile("newton_schulz", [0])(g)
    with pytest.raises(tf.TFHostError, match="number of rows"):
        tf.compile("embedding_backward")


class Calls:
    """The five calls on buffers of their own, of one size."""

    def __init__(self, rt, n, vocab, cols, seed=0):
        self.rt, self.n, self.vocab, self.cols = rt, n, vocab, cols
        self.tokens, self.table, self.weight, self.bias, _, _ = make(n, vocab, cols, 4, seed)
        self.b = {k: rt.DeviceBuffer.from_numpy(v) for k, v in dict(tokens=self.tokens, table=self.table, weight=self.weight, bias=self.bias).items()}
        self.e, self.y, self.de = (rt.DeviceBuffer(n * cols) for _ in range(3))
        self.mean, self.rstd = rt.DeviceBuffer(n), rt.DeviceBuffer(n)
        self.dw, self.db = rt.DeviceBuffer(cols), rt.DeviceBuffer(cols)
        self.dtable, self.update = rt.DeviceBuffer(vocab * cols), rt.DeviceBuffer(vocab * cols)

    def run(self):
        rt, b, n, vocab, cols = self.rt, self.b, self.n, self.vocab, self.cols
        rt.embedding_rows(b["tokens"], b["table"], self.e, n, vocab, cols)
        rt.layer_norm_rows(self.e, b["weight"], b["bias"], self.y, n, cols, mean=self.mean, rstd=self.rstd)
        rt.layer_norm_rows_backward(self.e, self.y, b["weight"], self.mean, self.rstd, n, cols, dx=self.de, dweight=self.dw, dbias=self.db)
        rt.embedding_rows_backward(b["tokens"], self.de, self.dtable, n, vocab, cols)
        rt.newton_schulz(self.dtable, self.update, vocab, cols)

    def results(self):
        return [x.numpy() for x in (self.y, self.mean, self.rstd, self.de, self.dw, self.db, self.dtable, self.update)]

    def clear(self):
        for x in (self.e, self.y, self.de, self.mean, self.rstd, self.dw, self.db, self.dtable, self.update):
            x.fill(0x7FC00000)


def same(a, b):
    return all(np.array_equal(x, y) for x, y in zip(a, b))


def test_two_recorded_graphs_and_eager_calls_share_the_scratch_buffer(rt):
    a, b = Calls(rt, 700, 90, 120, seed=1), Calls(rt, 6000, 150, 300, seed=2)
    wants = []
    for c in (a, b):
        c.run()
        wants.append(c.results())
    graphs = []
    for c in (a, b):
        g = rt.Graph()
        with g:
            c.run()
        graphs.append(g)
    big = Calls(rt, 20000, 400, 512, seed=3)
    for k in range(4):
        a.clear()
        b.clear()
        graphs[k % 2].launch()
        graphs[1 - k % 2].launch()
        if k == 1:
            big.run()  # makes the scratch buffer grow while the graphs are alive
        rt.synchronize()
        assert same(a.results(), wants[0]) and same(b.results(), wants[1]), k
    big_want = big.results()
    big.clear()
    big.run()
    assert same(big.results(), big_want)
    for g in graphs:
        g.destroy()


def test_a_recording_that_would_need_a_larger_scratch_buffer_is_refused(rt):
    import ctypes as C
    from tensorfrost_amd._lib import TFHipError, call

    size = C.c_size_t()
    call("tfhip_scratch_info", C.byref(size), C.byref(C.c_size_t()), C.byref(C.c_size_t()))
    side = 256
    while 24 * side * side <= size.value and side < 32768:
        side *= 2
    if 24 * side * side <= size.value:
        pytest.skip("the scratch buffer already holds the largest matrix")
    g, out = rt.DeviceBuffer(side * side), rt.DeviceBuffer(side * side)
    graph = rt.Graph()
    with pytest.raises(TFHipError, match="run the same work once before recording"):
        with graph:
            rt.newton_schulz(g, out, side, side)
    rt.synchronize()
    small = rt.DeviceBuffer.from_numpy(np.eye(8, dtype=np.float32))
    rt.newton_schulz(small, small, 8, 8)  # the library goes on working
    assert np.isfinite(small.numpy()).all()


def test_two_threads_at_once(rt):
    """Every call with several launches keeps the scratch buffer to itself until they are on the stream."""
    calls = [Calls(rt, 6000, 150, 300, seed=4), Calls(rt, 900, 400, 64, seed=5)]
    wants = []
    for c in calls:
        c.run()
        wants.append(c.results())
        c.clear()
    errors = []

    def work(c):
        try:
            for _ in range(30):
                c.run()
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    rt.synchronize()
    assert not errors
    assert same(calls[0].results(), wants[0]) and same(calls[1].results(), wants[1])


def test_a_graph_launched_beside_another_threads_calls(rt):
    """The graph's work and the other thread's calls use the same scratch buffer: neither may begin inside the other."""
    recorded, eager = Calls(rt, 6000, 150, 300, seed=6), Calls(rt, 7000, 300, 90, seed=7)
    wants = []
    for c in (recorded, eager):
        c.run()
        wants.append(c.results())
    graph = rt.Graph()
    with graph:
        recorded.run()
    for c in (recorded, eager):
        c.clear()
    errors = []

    def work(step):
        try:
            for _ in range(30):
                step()
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(step,)) for step in (graph.launch, eager.run)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    rt.synchronize()
    assert not errors
    assert same(recorded.results(), wants[0]) and same(eager.results(), wants[1])
    graph.destroy()


def test_memory_of_another_library_and_its_stream(rt):
    torch = pytest.importorskip("torch")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        x = torch.randn(300, 500, device="cuda")
        y = torch.empty_like(x)
    stream.synchronize()  # the library works on a stream of its own
    rt.layer_norm_rows(rt.DeviceBuffer.view(x.data_ptr(), x.numel()), None, None, rt.DeviceBuffer.view(y.data_ptr(), y.numel()), 300, 500)
    rt.synchronize()
    with torch.cuda.stream(stream):
        want = (x.double() - x.double().mean(1, keepdim=True)) / torch.sqrt(x.double().var(1, correction=0, keepdim=True) + 1e-5)
        off = (y.double() - want).abs().max()
    stream.synchronize()
    assert off.item() < 60 * U * 8  # |xhat| < 8 here; (500 / 64 + 24) u and the rest twice


def test_the_step_against_differences(rt):
    """d loss / d table of loss = sum(y dy) by central differences of the calls themselves. h = 0.02: the third derivative along one
    element of the table is of the order of cols^0 here, so the difference is off by some h^2 = 4e-4 times a few, and by the rounding of
    y: 60 u per element of order 1, 48 elements, over 2 h: 5e-3."""
    n, vocab, cols = 6, 4, 8
    tokens = np.array([0, 1, 1, 3, 0, -1], np.int32)
    rng = np.random.default_rng(5)
    table = rng.normal(size=(vocab, cols)).astype(np.float32)
    weight, dy = (1 + 0.2 * rng.normal(size=cols)).astype(np.float32), rng.normal(size=(n, cols)).astype(np.float32)
    tb, wb, dyb = rt.DeviceBuffer.from_numpy(tokens), rt.DeviceBuffer.from_numpy(weight), rt.DeviceBuffer.from_numpy(dy)
    e, y, mean, rstd = rt.DeviceBuffer(n * cols), rt.DeviceBuffer(n * cols), rt.DeviceBuffer(n), rt.DeviceBuffer(n)

    def loss(table):
        rt.embedding_rows(tb, rt.DeviceBuffer.from_numpy(table), e, n, vocab, cols, scale=1.5)
        rt.layer_norm_rows(e, wb, None, y, n, cols, mean=mean, rstd=rstd)
        return float((y.numpy().astype(np.float64) * dy.reshape(-1)).sum())

    loss(table)
    de, dtable = rt.DeviceBuffer(n * cols), rt.DeviceBuffer(vocab * cols)
    rt.layer_norm_rows_backward(e, dyb, wb, mean, rstd, n, cols, dx=de)
    rt.embedding_rows_backward(tb, de, dtable, n, vocab, cols, scale=1.5)
    got = dtable.numpy(np.float32, (vocab, cols))
    assert not got[2].any()
    for v, c in ((0, 0), (1, 3), (1, 7), (3, 5), (2, 1)):
        h = np.float32(0.02)
        up, down = table.copy(), table.copy()
        up[v, c] += h
        down[v, c] -= h
        assert abs((loss(up) - loss(down)) / (float(up[v, c]) - float(down[v, c])) - got[v, c]) < 2e-2
