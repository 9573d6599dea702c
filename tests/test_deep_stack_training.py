"""Layer normalisation and the Muon rule together, as a user trains a stack of dense layers with
them: through sessions on the CPU and the GPU, captured steps, checkpoints, parameter servers and
collective jobs."""
import threading

import numpy as np
import pytest
import torch

import distributed_tensorflow_amd as tf
from distributed_tensorflow_amd.ops import ref_kernels
from distributed_tensorflow_amd.parallel.comm import LoopbackComm

from test_optimizers import _free_port, _mlp_job

COEF = (3.4445, -4.7750, 2.0315)


def _ns64(g, steps=5, coef=COEF, eps=1e-7):
    x = np.asarray(g, np.float64)
    x = x / (np.sqrt((x * x).sum()) + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    for _ in range(steps):
        s = x @ x.T
        x = coef[0] * x + (coef[1] * s + coef[2] * s @ s) @ x
    return x.T if tall else x


def _build(make_opt, hidden=(24, 16), inputs=12, classes=5, seed=3):
    tf.set_random_seed(seed)
    x = tf.placeholder(tf.float32, [None, inputs], name="x")
    y = tf.placeholder(tf.int64, [None], name="y")
    h = x
    for i, n in enumerate(hidden):
        h = tf.layers.dense(h, n, name="dense%d" % i)
        h = tf.layers.layer_norm(h, activation=tf.nn.relu, name="norm%d" % i)
    logits = tf.layers.dense(h, classes, name="out")
    loss = tf.losses.sparse_softmax_cross_entropy(labels=y, logits=logits)
    step = tf.train.get_or_create_global_step()
    # (behind the layers: an op's random stream goes by its place in the graph, so a schedule's
    # ops in front of them would give the same program other weights)
    optimizer = make_opt()
    grads_and_vars = optimizer.compute_gradients(loss)
    train = optimizer.apply_gradients(grads_and_vars, global_step=step)
    return x, y, loss, train, grads_and_vars, step


def _batch(seed, inputs=12, classes=5, n=32):
    rng = np.random.RandomState(seed)
    return rng.randn(n, inputs).astype(np.float32), rng.randint(0, classes, n).astype(np.int64)


def _run(device, make_opt, steps=4, fusion=True, graphs=True, **kw):
    with tf.Graph().as_default():
        x, y, loss, train, gv, step = _build(make_opt, **kw)
        names = [v.op.name for v in tf.trainable_variables()]
        with tf.Session(config=tf.ConfigProto(device=device, graph_fusion=fusion,
                                              hip_graphs=graphs)) as sess:
            sess.run(tf.global_variables_initializer())
            start = sess.run(tf.trainable_variables())
            out, first = [], None
            for k in range(steps):
                bx, by = _batch(k, kw.get("inputs", 12), kw.get("classes", 5))
                if k == 0:
                    first = sess.run([g for g, _ in gv], {x: bx, y: by})
                out.append(float(sess.run([train, loss], {x: bx, y: by})[1]))
            types = {s.node.type for p in sess._plans.values() for s in p.steps}
            return dict(start=dict(zip(names, start)), first=dict(zip(names, first)), losses=out,
                        end=dict(zip(names, sess.run(tf.trainable_variables()))), types=types,
                        step=float(sess.run(step)), stats=dict(sess.stats),
                        fallbacks=list(getattr(sess, "fallback_log", [])))


def _muon(lr=0.05, **kw):
    return tf.train.MuonOptimizer(lr, vector_optimizer=tf.train.AdamOptimizer(0.01), **kw)


@pytest.mark.parametrize("nesterov,decay,rms", [(True, 0.0, 0.0), (False, 0.1, 0.0),
                                                (True, 0.05, 0.2)])
def test_first_step_is_the_published_rule(nesterov, decay, rms):
    run = _run("cpu", lambda: _muon(use_nesterov=nesterov, weight_decay=decay, rms_scale=rms,
                                    momentum=0.9), steps=1)
    assert "MultiApplyOptimizer" in run["types"] and run["step"] == 1
    for n, w in run["start"].items():
        g = run["first"][n].astype(np.float64)
        if w.ndim == 1:                       # adam's first step: sign(g) * rate
            big = np.abs(g) > 1e-5
            np.testing.assert_allclose(run["end"][n][big], (w - 0.01 * np.sign(g))[big],
                                       rtol=1e-3, atol=1e-5)
            continue
        u = 1.9 * g if nesterov else g
        s = rms * np.sqrt(max(w.shape)) if rms else np.sqrt(max(1.0, w.shape[1] / w.shape[0]))
        want = (1 - 0.05 * decay) * w - 0.05 * s * _ns64(u)
        np.testing.assert_allclose(run["end"][n], want, rtol=1e-4, atol=2e-5)


def test_fused_and_unfused_updates_agree_and_schedules_drive_the_rate():
    a = _run("cpu", _muon)
    b = _run("cpu", _muon, fusion=False)
    assert "ApplyOptimizer" in b["types"] and "ApplyOptimizer" not in a["types"]
    c = _run("cpu", lambda: _muon(tf.train.exponential_decay(
        0.05, tf.train.get_or_create_global_step(), 1, 1.0)))
    for n in a["end"]:
        np.testing.assert_allclose(a["end"][n], b["end"][n], rtol=1e-5, atol=1e-6)
        np.testing.assert_allclose(a["end"][n], c["end"][n], rtol=1e-5, atol=1e-6)


def test_vectors_need_an_optimizer_of_their_own_and_slots_are_named():
    w = tf.Variable(tf.zeros([4, 3]), name="W")
    b = tf.Variable(tf.zeros([3]), name="b")
    x = tf.placeholder(tf.float32, [None, 4])
    loss = tf.reduce_sum(tf.square(tf.add(tf.matmul(x, w), b)))
    with pytest.raises(ValueError, match="vector_optimizer.*b"):
        tf.train.MuonOptimizer(0.1).minimize(loss)
    only = tf.train.MuonOptimizer(0.1, name="Matrices")
    only.minimize(loss, var_list=[w])
    assert only.get_slot(w, "momentum").op.name == "W/Matrices"
    assert "slot_of" not in only.get_slot(w, "momentum").op.attrs
    both = _muon()
    both.minimize(loss)
    assert both.get_slot_names() == ["momentum", "m", "v"]
    assert both.get_slot(b, "m") is not None and both.get_slot(w, "m") is None
    for bad in (dict(steps=0), dict(epsilon=-1.0), dict(coefficients=(1.0, 2.0)),
                dict(rms_scale=-0.1)):
        with pytest.raises(ValueError):
            tf.train.MuonOptimizer(0.1, **bad)


def test_newton_schulz_op_between_compute_and_apply():
    x = tf.placeholder(tf.float32, [6, 4])
    o = tf.newton_schulz(x)
    st = tf.newton_schulz(tf.expand_dims(x, 0), steps=2, coefficients=[COEF, (1.5, -0.5, 0.0)])
    v = np.random.RandomState(0).randn(6, 4).astype(np.float32)
    with tf.Session(config=tf.ConfigProto(device="cpu")) as sess:
        a, b = sess.run([o, st], {x: v})
    np.testing.assert_allclose(a, _ns64(v), rtol=1e-4, atol=1e-5)
    assert b.shape == (1, 6, 4)
    with pytest.raises(LookupError):
        tf.gradients(tf.reduce_sum(o), [x])
    for bad in (lambda: tf.newton_schulz(tf.placeholder(tf.float32, [3])),
                lambda: tf.newton_schulz(tf.placeholder(tf.int32, [3, 3])),
                lambda: tf.newton_schulz(x, steps=0),
                lambda: tf.newton_schulz(x, epsilon=-1.0),
                lambda: tf.newton_schulz(x, coefficients=[COEF] * 4)):
        with pytest.raises((TypeError, ValueError)):
            bad()


def test_momentum_is_checkpointed(tmp_path):
    def build():
        opt = tf.train.MuonOptimizer(0.05)
        tf.set_random_seed(3)
        w = tf.Variable(tf.random_normal([4, 2]), name="W")
        x = tf.placeholder(tf.float32, [None, 4])
        return w, x, opt, opt.minimize(tf.reduce_mean(tf.square(tf.matmul(x, w)))), \
            tf.train.Saver()
    bx = np.random.RandomState(1).randn(8, 4).astype(np.float32)
    with tf.Graph().as_default():
        w, x, opt, train, saver = build()
        with tf.Session(config=tf.ConfigProto(device="cpu")) as sess:
            sess.run(tf.global_variables_initializer())
            for _ in range(3):
                sess.run(train, {x: bx})
            path = saver.save(sess, str(tmp_path / "model"))
            sess.run(train, {x: bx})
            want = sess.run(w)
    with tf.Graph().as_default():
        w, x, opt, train, saver = build()
        with tf.Session(config=tf.ConfigProto(device="cpu")) as sess:
            saver.restore(sess, path)
            sess.run(train, {x: bx})
            np.testing.assert_array_equal(sess.run(w), want)


@pytest.mark.parametrize("strategy", ["allreduce_sync", "reduce_scatter_sync"])
def test_collective_replicas_stay_identical(strategy):
    """Two ranks, other batches on each: the orthogonalised update is taken from the reduced
    gradient of the whole matrix on both, whatever part of it a rank would own."""
    cluster = tf.train.ClusterSpec({"worker": ["localhost:1", "localhost:2"]})
    results = {}
    comms = LoopbackComm.create_world(2)
    threads = [threading.Thread(target=_mlp_job,
                                args=(cluster, i, 5, results, lambda: _muon(0.01), "rccl",
                                      comms[i], strategy)) for i in range(2)]
    [t.start() for t in threads]
    [t.join(120) for t in threads]
    assert set(results) == {0, 1}
    a, b = (results[i]["final"] for i in range(2))
    assert np.array_equal(a["w1"], b["w1"]) and a["step"] == b["step"] == 5
    assert np.isfinite(a["w1"]).all()


def test_momentum_lives_on_the_parameter_server():
    port = _free_port()
    cluster = tf.train.ClusterSpec({"ps": ["127.0.0.1:%d" % port], "worker": ["127.0.0.1:0"]})
    server = tf.train.Server(cluster, job_name="ps", task_index=0,
                             config=tf.ConfigProto(device="cpu"))
    results = {}
    t = threading.Thread(target=_mlp_job, args=(cluster, 0, 4, results, lambda: _muon(0.01)))
    t.start()
    t.join(120)
    assert 0 in results and results[0]["slot_device"] == "/job:ps/task:0"
    assert np.isfinite(results[0]["costs"]).all() and results[0]["final"]["step"] == 4
    server.stop()


def test_rule_step_matches_the_oracle_for_stacks():
    gen = torch.Generator().manual_seed(0)
    w, g, v = (torch.randn(3, 5, 7, generator=gen) for _ in range(3))
    hyper = (0.1, 0.9, 1.0, 0.0, 0.0, 1e-7, 2.0, *COEF, *COEF)
    nw, nv, _ = ref_kernels.optimizer_rule_step("muon", hyper, w, g, v)
    for i in range(3):
        a, b, _ = ref_kernels.optimizer_rule_step("muon", hyper, w[i], g[i], v[i])
        assert torch.equal(a, nw[i]) and torch.equal(b, nv[i])


# ---------------------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_gpu_session_trains_the_stack_with_native_kernels_and_captures_it():
    """The whole step -- dense layers, layer norms, their gradients, Muon and Adam -- runs on
    native kernels, is captured, and its replays follow the eager steps of the same program."""
    captured = _run("cuda:0", _muon, steps=6)
    eager = _run("cuda:0", _muon, steps=6, graphs=False)
    unfused = _run("cuda:0", _muon, steps=6, fusion=False)
    assert captured["stats"]["torch_fallbacks"] == 0, captured["fallbacks"]
    assert captured["stats"]["graph_replays"] >= 2 and eager["stats"]["graph_replays"] == 0
    for n in captured["end"]:
        assert np.array_equal(captured["end"][n], eager["end"][n]), n
        np.testing.assert_allclose(captured["end"][n], unfused["end"][n], rtol=1e-4, atol=1e-5)


@pytest.mark.gpu
def test_gpu_first_step_matches_the_cpu():
    """One step from the same weights: gradients agree to fp32 chains of a few hundred terms, and
    the update is the rule on each side's own gradient."""
    gpu, cpu = _run("cuda:0", _muon, steps=1), _run("cpu", _muon, steps=1)
    for n, w in gpu["start"].items():
        np.testing.assert_allclose(w, cpu["start"][n], rtol=1e-6, atol=1e-6)
        np.testing.assert_allclose(gpu["first"][n], cpu["first"][n], rtol=1e-3, atol=1e-5)
        if w.ndim == 2:
            s = np.sqrt(max(1.0, w.shape[1] / w.shape[0]))
            want = w - 0.05 * s * _ns64(1.95 * gpu["first"][n].astype(np.float64))
            np.testing.assert_allclose(gpu["end"][n], want, rtol=1e-4, atol=2e-5)


@pytest.mark.gpu
def test_gpu_schedule_is_read_on_the_device():
    def make():
        step = tf.train.get_or_create_global_step()
        return _muon(tf.train.exponential_decay(0.05, step, 1, 0.5))
    sched = _run("cuda:0", make, steps=5)
    assert sched["stats"]["torch_fallbacks"] == 0, sched["fallbacks"]
    cpu = _run("cpu", make, steps=1)
    one = _run("cuda:0", make, steps=1)
    flat = _run("cuda:0", _muon, steps=1)
    for n in flat["end"]:
        np.testing.assert_allclose(one["end"][n], flat["end"][n], rtol=1e-5, atol=1e-6)
        assert one["end"][n].shape == cpu["end"][n].shape
    frozen = _run("cuda:0", lambda: _muon(tf.train.exponential_decay(
        0.05, tf.train.get_or_create_global_step(), 1, 1e-9)), steps=5)
    # from the second step on the rate is nothing: the matrices stay where the first step left them
    for n, w in one["end"].items():
        if w.ndim == 2:
            np.testing.assert_allclose(frozen["end"][n], w, rtol=0, atol=1e-6)


@pytest.mark.gpu
def test_gpu_newton_schulz_op():
    x = tf.placeholder(tf.float32, [60, 40])
    v = np.random.RandomState(0).randn(60, 40).astype(np.float32)
    with tf.Session(config=tf.ConfigProto(device="cuda:0")) as sess:
        got = sess.run(tf.newton_schulz(x), {x: v})
    np.testing.assert_allclose(got, _ns64(v), rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("fusion", [True, False])
def test_gradients_that_are_the_weights_and_weights_updated_twice(device, fusion):
    """The gradient of w w / 2 is w itself: it is read before w is written. A matrix given twice
    is updated twice. (Tolerance: the rule's result is off by at most 2e-3 in the spectral norm,
    times the rate; the momentum of the second update adds its own.)"""
    rng = np.random.RandomState(5)
    values = [rng.randn(*s).astype(np.float32) for s in ((70, 90), (12, 10), (90, 33), (20, 24))]
    for twice in (False, True):
        with tf.Graph().as_default():
            ws = [tf.Variable(tf.constant(v), name="w%d" % i) for i, v in enumerate(values)]
            loss = tf.add(tf.add(tf.nn.l2_loss(ws[0]), tf.nn.l2_loss(ws[1])),
                          tf.add(tf.nn.l2_loss(ws[2]), tf.nn.l2_loss(ws[3])))
            opt = tf.train.MuonOptimizer(0.05)
            gv = opt.compute_gradients(loss)
            train = opt.apply_gradients(gv + [(tf.identity(g), v) for g, v in gv[:2]]
                                        if twice else gv)
            with tf.Session(config=tf.ConfigProto(device=device, graph_fusion=fusion)) as sess:
                sess.run(tf.global_variables_initializer())
                sess.run(train)
                got = sess.run(ws)
        for i, (w, g) in enumerate(zip(values, got)):
            s = max(1.0, w.shape[1] / w.shape[0]) ** 0.5
            if not (twice and i < 2):
                assert np.abs(g - (w - 0.05 * s * _ns64(w))).max() <= 0.05 * s * 2e-3
            elif fusion or device == "cpu":
                # both gradients are the weight's value before the step
                assert np.abs(g - (w - 0.1 * s * _ns64(w))).max() <= 0.1 * s * 2e-3
