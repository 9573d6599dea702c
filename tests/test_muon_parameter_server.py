"""Muon with variables and momenta on a parameter server: the update is the rule, and a GPU worker
computes it with the framework's kernels.

Tolerances: gradients are fp32 sums over 16 rows. The update is within 2e-3 of the rule in the
spectral norm, times the rate (see ``test_newton_schulz``); the momentum adds two products."""
import threading

import numpy as np
import pytest

import distributed_tensorflow_amd as tf
from distributed_tensorflow_amd.ops import ref_kernels

from test_optimizers import _free_port
from test_update_snapshots import _ns64

SHAPES = ((30, 70), (70, 96), (96, 10))


def _job(cluster, device, fusion, schedule, results, steps=2):
    rng = np.random.RandomState(0)
    xs, ys = rng.randn(16, 30).astype(np.float32), rng.randn(16, 10).astype(np.float32)
    with tf.Graph().as_default():
        tf.set_random_seed(4)
        config = tf.ConfigProto(device=device, graph_fusion=fusion)
        server = tf.train.Server(cluster, job_name="worker", task_index=0, config=config)
        with tf.device(tf.train.replica_device_setter(worker_device="/job:worker/task:0",
                                                      cluster=cluster)):
            x, y = tf.placeholder(tf.float32, [16, 30]), tf.placeholder(tf.float32, [16, 10])
            ws = [tf.Variable(tf.random_normal(list(s)), name="w%d" % i)
                  for i, s in enumerate(SHAPES)]
            b = tf.Variable(tf.zeros([10]), name="b")
            h = tf.nn.tanh(tf.matmul(tf.nn.tanh(tf.matmul(x, ws[0])), ws[1]))
            loss = tf.reduce_sum(tf.square(tf.subtract(tf.add(tf.matmul(h, ws[2]), b), y)))
            step = tf.train.get_or_create_global_step()
            rate = tf.train.exponential_decay(0.05, step, 1, 0.5) if schedule else 0.05
            opt = tf.train.MuonOptimizer(rate, momentum=0.9, weight_decay=0.1,
                                         vector_optimizer=tf.train.GradientDescentOptimizer(0.01))
            gv = opt.compute_gradients(loss)
            train = opt.apply_gradients(gv, global_step=step)
            init = tf.global_variables_initializer()
        with tf.Session(server.target, config=config) as sess:
            sess.run(init)
            slots = [opt.get_slot(w, "momentum") for w in ws]
            got = []
            for _ in range(steps):
                before = sess.run(ws + slots)
                grads = sess.run([g for g, v in gv][:len(ws)], {x: xs, y: ys})
                sess.run(train, {x: xs, y: ys})
                got.append((before, grads, sess.run(ws + slots)))
            results.update(got=got, stats=dict(sess.stats), device=slots[0].device)
        server.stop()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("fusion", [True, False])
@pytest.mark.parametrize("schedule", [False, True])
def test_updates_are_the_rule(device, fusion, schedule, monkeypatch):
    if device != "cpu":
        def refuse(*args):
            raise AssertionError("the rule ran in torch")
        monkeypatch.setattr(ref_kernels, "newton_schulz", refuse)
    port = _free_port()
    cluster = tf.train.ClusterSpec({"ps": ["127.0.0.1:%d" % port], "worker": ["127.0.0.1:0"]})
    ps = tf.train.Server(cluster, job_name="ps", task_index=0, config=tf.ConfigProto(device="cpu"))
    results = {}
    t = threading.Thread(target=_job, args=(cluster, device, fusion, schedule, results))
    t.start()
    t.join(100)
    ps.stop()
    assert results and results["device"] == "/job:ps/task:0"
    assert results["stats"]["torch_fallbacks"] == 0
    n = len(SHAPES)
    for k, (before, grads, after) in enumerate(results["got"]):
        lr = 0.05 * (0.5 ** k if schedule else 1.0)
        for i in range(n):
            w, v, g = (np.asarray(a[j], np.float64) for a, j in ((before, i), (before, n + i),
                                                                  (grads, i)))
            v = 0.9 * v + g
            s = lr * max(1.0, w.shape[1] / w.shape[0]) ** 0.5
            want = (1 - lr * 0.1) * w - s * _ns64(g + 0.9 * v)
            assert np.abs(after[i] - want).max() <= s * 2e-3 + 2.0 ** -20 * np.abs(w).max()
            assert np.abs(after[n + i] - v).max() <= 2.0 ** -20 * np.abs(v).max()
        assert np.abs(after[0] - before[0]).max() > 0.2 * lr / 8


def test_a_counter_on_the_parameter_server_is_shipped_by_a_gpu_worker():
    """Muon's step counter is an ``AssignAdd`` of its own (matrices and vectors are two nodes): the
    GPU kernel of the op hands variables of another process to their store."""
    import types

    import torch

    from distributed_tensorflow_amd.framework.op_registry import get_opdef
    from distributed_tensorflow_amd.ops import hip_kernels  # noqa: F401
    from distributed_tensorflow_amd.parallel.ps_transport import RemoteVariableStore
    store = object.__new__(RemoteVariableStore)        # (no connection: nothing is sent here)
    shipped = []
    ctx = types.SimpleNamespace(
        session=types.SimpleNamespace(_store_for=lambda op: store),
        var_assign_add=lambda op, delta: shipped.append((op.name, float(delta))),
        note_fallback=lambda op, why: pytest.fail("refused: %s" % why))
    var = types.SimpleNamespace(name="global_step")
    for kind, sign in (("AssignAdd", 1.0), ("AssignSub", -1.0)):
        op = types.SimpleNamespace(name="add", type=kind, inputs=[types.SimpleNamespace(op=var)])
        get_opdef(kind).hip_kernel(op, [None, torch.tensor(3.0)], ctx)
        assert shipped.pop() == ("global_step", 3.0 * sign)
