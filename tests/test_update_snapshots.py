"""Updates whose gradients are read from variables that the same step writes: every gradient is the
value before the step, however many updates the step has, fused or one by one, on either device.

Tolerance: the orthogonalised update is off by at most 2e-3 in the spectral norm (see
``test_newton_schulz``), times rate and scale, for each update of a variable."""
import numpy as np
import pytest

import distributed_tensorflow_amd as tf

COEF = (3.4445, -4.7750, 2.0315)
DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def _ns64(g, steps=5, coef=COEF, eps=1e-7):
    x = np.asarray(g, np.float64)
    x = x / (np.sqrt((x * x).sum()) + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    for _ in range(steps):
        s = x @ x.T
        x = coef[0] * x + (coef[1] * s + coef[2] * s @ s) @ x
    return x.T if tall else x


def _rule(w, grads, lr=0.05, mu=0.95):
    """The updates of one variable, one after the other."""
    w, v = np.asarray(w, np.float64), 0.0
    for g in grads:
        g = np.asarray(g, np.float64)
        v = mu * v + g
        w = w - lr * max(1.0, w.shape[1] / w.shape[0]) ** 0.5 * _ns64(g + mu * v)
    return w


def _step(device, fusion, values, pairs):
    """One step of ``pairs(variables)`` -> [(gradient, variable)]; the variables afterwards."""
    with tf.Graph().as_default():
        ws = [tf.Variable(tf.constant(v), name="w%d" % i) for i, v in enumerate(values)]
        train = tf.train.MuonOptimizer(0.05).apply_gradients(pairs(ws))
        with tf.Session(config=tf.ConfigProto(device=device, graph_fusion=fusion)) as sess:
            sess.run(tf.global_variables_initializer())
            sess.run(train)
            got = sess.run(ws)
            assert sess.stats["torch_fallbacks"] == 0 or device == "cpu"
            return got


def _near(got, want, updates):
    s = max(1.0, want.shape[1] / want.shape[0]) ** 0.5
    assert np.abs(got - want).max() <= updates * 0.05 * s * 2e-3


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fusion", [True, False])
@pytest.mark.parametrize("read", ["loss", "identity", "itself", "turned"])
def test_a_variable_updated_twice(device, fusion, read):
    rng = np.random.RandomState(5)
    values = [rng.randn(*s).astype(np.float32) for s in ((70, 90), (12, 10), (33, 33))]

    def pairs(ws):
        if read == "loss":
            g = [tf.gradients(tf.nn.l2_loss(w), [w._variable])[0] for w in ws]
        elif read == "identity":
            g = [tf.identity(w) for w in ws]
        elif read == "itself":
            g = [w._variable for w in ws]
        else:
            g = [tf.reshape(tf.identity(w), [w.shape[0], w.shape[1]]) for w in ws]
        return [*zip(g, ws), *zip([tf.identity(x) for x in g], ws)]
    for w, got in zip(values, _step(device, fusion, values, pairs)):
        _near(got, _rule(w, [w, w]), 2)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fusion", [True, False])
@pytest.mark.parametrize("computed", [False, True])
def test_variables_that_are_each_other_s_gradients(device, fusion, computed):
    rng = np.random.RandomState(6)
    values = [rng.randn(*s).astype(np.float32) for s in ((66, 70), (66, 70), (66, 70))]

    def pairs(ws):
        g = [tf.identity(ws[(i + 1) % 3]) for i in range(3)]
        if computed:
            g = [tf.multiply(x, 2.0) for x in g]
        return list(zip(g, ws))
    out = _step(device, fusion, values, pairs)
    for i, w in enumerate(values):
        _near(out[i], _rule(w, [values[(i + 1) % 3]]), 1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fusion", [True, False])
def test_a_momentum_as_gradient(device, fusion):
    """The second step's gradient is the momentum that the update advances."""
    rng = np.random.RandomState(7)
    w0, g0 = (rng.randn(40, 72).astype(np.float32) for _ in range(2))
    with tf.Graph().as_default():
        w = tf.Variable(tf.constant(w0), name="w")
        opt = tf.train.MuonOptimizer(0.05)
        first = opt.apply_gradients([(tf.constant(g0), w)])
        m = opt.get_slot(w, "momentum")
        second = opt.apply_gradients([(tf.identity(m), w)])
        with tf.Session(config=tf.ConfigProto(device=device, graph_fusion=fusion)) as sess:
            sess.run(tf.global_variables_initializer())
            sess.run(first)
            sess.run(second)
            got, gm = sess.run([w, m])
    _near(got, _rule(w0, [g0, g0]), 2)
    np.testing.assert_allclose(gm, 1.95 * g0, rtol=1e-6)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fusion", [True, False])
@pytest.mark.parametrize("vectors", ["sgd", "momentum"])
@pytest.mark.parametrize("order", ["vectors first", "matrix first"])
def test_vectors_and_matrices_of_one_step(device, fusion, vectors, order):
    """Matrices and vectors are updated by different nodes; a gradient that only one of them needs
    and that passes through what the other writes (gamma's through the matrix behind the layer
    norm, the matrix's through the vector it is scaled by) is taken before either is written. The
    rates are large, so that updated variables would give other gradients. (Tolerances: fp32 sums
    of up to 40 terms; the orthogonalised update as above.)"""
    rng = np.random.RandomState(9)
    bx, by = rng.randn(8, 40).astype(np.float32), rng.randn(8, 30).astype(np.float32)
    with tf.Graph().as_default():
        tf.set_random_seed(3)
        x, y = tf.placeholder(tf.float32, [8, 40]), tf.placeholder(tf.float32, [8, 30])
        s = tf.Variable(tf.constant(rng.randn(30).astype(np.float32)), name="s")
        h = tf.layers.layer_norm(x, name="norm")
        w = tf.Variable(tf.random_normal([40, 30]), name="w")
        loss = tf.reduce_sum(tf.square(tf.subtract(tf.multiply(tf.matmul(h, w), s), y)))
        vector = tf.train.GradientDescentOptimizer(0.5) if vectors == "sgd" else \
            tf.train.MomentumOptimizer(0.5, 0.9)
        opt = tf.train.MuonOptimizer(5.0, vector_optimizer=vector)
        gv = sorted(opt.compute_gradients(loss),
                    key=lambda p: len(p[1].shape) * (1 if order == "vectors first" else -1))
        train = opt.apply_gradients(gv)
        with tf.Session(config=tf.ConfigProto(device=device, graph_fusion=fusion)) as sess:
            sess.run(tf.global_variables_initializer())
            feed = {x: bx, y: by}
            before = sess.run([v for _, v in gv])
            grads = sess.run([g for g, _ in gv], feed)
            sess.run(train, feed)
            after = sess.run([v for _, v in gv])
    for v, g, got in zip(before, grads, after):
        if v.ndim == 1:
            np.testing.assert_allclose(got, v - 0.5 * g, rtol=1e-4, atol=1e-4)
        else:
            assert np.abs(got - _rule(v, [g], lr=5.0)).max() <= 5.0 * 2e-3


@pytest.mark.parametrize("fusion", [True, False])
def test_a_read_behind_an_assignment_is_the_new_value(fusion):
    """A gradient that is read behind another write of the step is that write's value."""
    rng = np.random.RandomState(8)
    w0, w1 = (rng.randn(20, 30).astype(np.float32) for _ in range(2))
    with tf.Graph().as_default():
        w = tf.Variable(tf.constant(w0), name="w")
        with tf.control_dependencies([w.assign(tf.constant(w1))]):
            g = tf.identity(w)
        train = tf.train.MuonOptimizer(0.05).apply_gradients([(g, w), (tf.identity(g), w)])
        with tf.Session(config=tf.ConfigProto(device="cpu", graph_fusion=fusion)) as sess:
            sess.run(tf.global_variables_initializer())
            sess.run(train)
            _near(sess.run(w), _rule(w1, [w1, w1]), 2)


@pytest.mark.gpu
@pytest.mark.parametrize("fusion", [True, False])
def test_captured_steps_copy_what_they_overwrite(fusion):
    """Replays read the variables as each step finds them: the same bits as eager steps."""
    rng = np.random.RandomState(10)
    values = [rng.randn(*s).astype(np.float32) for s in ((70, 90), (70, 90), (24, 10))]
    bx = rng.randn(8, 24).astype(np.float32)
    runs = []
    for graphs in (True, False):
        with tf.Graph().as_default():
            ws = [tf.Variable(tf.constant(v), name="w%d" % i) for i, v in enumerate(values)]
            b = tf.Variable(tf.zeros([10]), name="b")
            x = tf.placeholder(tf.float32, [8, 24])
            loss = tf.reduce_sum(tf.square(tf.add(tf.matmul(x, ws[2]), b)))
            g2, gb = tf.gradients(loss, [ws[2]._variable, b._variable])
            opt = tf.train.MuonOptimizer(0.05, vector_optimizer=tf.train.MomentumOptimizer(0.01, 0.9))
            train = opt.apply_gradients([(tf.identity(ws[1]), ws[0]), (tf.identity(ws[0]), ws[1]),
                                         (g2, ws[2]), (gb, b), (tf.identity(ws[0]), ws[0])])
            with tf.Session(config=tf.ConfigProto(device="cuda:0", graph_fusion=fusion,
                                                  hip_graphs=graphs)) as sess:
                sess.run(tf.global_variables_initializer())
                got = []
                for _ in range(6):
                    sess.run([train, loss], {x: bx})
                    got.append(sess.run(ws + [b]))
                runs.append((got, dict(sess.stats)))
    assert runs[0][1]["graph_replays"] >= 2 and runs[1][1]["graph_replays"] == 0
    assert runs[0][1]["torch_fallbacks"] == 0
    for a, b in zip(runs[0][0], runs[1][0]):
        for u, v in zip(a, b):
            assert np.array_equal(u, v)
    _near(runs[0][0][0][0], _rule(values[0], [values[1], values[0]]), 2)
    _near(runs[0][0][0][1], _rule(values[1], [values[0]]), 1)
