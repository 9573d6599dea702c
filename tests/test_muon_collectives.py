"""Muon and layer norm on two collective ranks against one process that sees both batches: the mean
of the ranks' gradients (``SyncReplicasOptimizer``) is the gradient of the joint batch, their sum
(without it) twice that. Every variable and momentum has to follow the one process's values, not
only the other rank's.

Tolerances. Gradients of the two differ by fp32 sums in another order, 2^-20 of their size. Five
Newton-Schulz steps grow what lies in nearly empty directions up to 485-fold, so an update (of
spectral norm about one, times rate and scale) may differ by 485 * 2^-20 = 5e-4 in a step; weights
that differ by that change the next gradients by as much relatively, so the sum of steps is allowed
four times their number. A rank that used its own gradient alone would be off by the update's size."""
import threading

import numpy as np
import pytest

import distributed_tensorflow_amd as tf
from distributed_tensorflow_amd.parallel.comm import LoopbackComm

STEPS, RATE, ROWS = 3, 0.02, 24


def _batches(k):
    rng = np.random.RandomState(100 + k)
    return rng.randn(2 * ROWS, 12).astype(np.float32), rng.randn(2 * ROWS, 10).astype(np.float32)


def _job(rank, results, mean, cluster=None, comm=None, strategy=None):
    with tf.Graph().as_default():
        config = tf.ConfigProto(device="cpu", strategy=strategy)
        target, server = "", None
        if comm is not None:
            server = tf.train.Server(cluster, job_name="worker", task_index=rank, protocol="rccl",
                                     config=config, comm=comm)
            target = server.target
        tf.set_random_seed(11)
        x = tf.placeholder(tf.float32, [None, 12])
        y = tf.placeholder(tf.float32, [None, 10])
        h = tf.layers.dense(x, 16, name="first")
        h = tf.layers.layer_norm(h, activation=tf.nn.tanh, name="norm")
        out = tf.layers.dense(h, 10, name="last")
        loss = tf.reduce_mean(tf.square(tf.subtract(out, y)))
        if comm is None and not mean:
            loss = tf.multiply(loss, 2.0)
        step = tf.train.get_or_create_global_step()
        opt = tf.train.MuonOptimizer(RATE, vector_optimizer=tf.train.MomentumOptimizer(0.1, 0.9))
        sync = tf.train.SyncReplicasOptimizer(opt, 2) if comm is not None and mean else opt
        train = sync.minimize(loss, global_step=step)
        variables = tf.trainable_variables()
        slots = [opt.get_slot(v, "momentum") for v in variables if len(v.shape) == 2]
        sv = tf.train.Supervisor(is_chief=rank == 0, global_step=step, logdir=None,
                                 init_op=tf.global_variables_initializer(),
                                 recovery_wait_secs=0.05, summary_op=None)
        with sv.prepare_or_wait_for_session(target, config=config) as sess:
            if sync is not opt:
                sync.configure_session(sess)
            start = sess.run(variables)
            for k in range(STEPS):
                bx, by = _batches(k)
                if comm is not None:
                    bx, by = (b[rank * ROWS:(rank + 1) * ROWS] for b in (bx, by))
                sess.run(train, {x: bx, y: by})
            results[rank] = dict(start=start, end=sess.run(variables), slots=sess.run(slots),
                                 step=float(sess.run(step)))
        sv.stop()
        if server is not None:
            server.stop()


@pytest.mark.parametrize("strategy", ["allreduce_sync", "reduce_scatter_sync"])
@pytest.mark.parametrize("mean", [True, False])
def test_two_ranks_follow_one_process_on_both_batches(strategy, mean):
    alone, results = {}, {}
    _job(0, alone, mean)
    cluster = tf.train.ClusterSpec({"worker": ["localhost:1", "localhost:2"]})
    comms = LoopbackComm.create_world(2)
    threads = [threading.Thread(target=_job, args=(i, results, mean, cluster, comms[i], strategy))
               for i in range(2)]
    [t.start() for t in threads]
    [t.join(100) for t in threads]
    assert set(results) == {0, 1}
    one = alone[0]
    for got in results.values():
        assert got["step"] == one["step"] == STEPS
        for s, a, b in zip(one["start"], got["end"], one["end"]):
            if s.ndim == 2:
                scale = RATE * max(1.0, s.shape[1] / s.shape[0]) ** 0.5
                assert np.abs(a - b).max() <= 4 * STEPS * scale * 5e-4
                # (the update is far larger than that, so a wrong one would show)
                assert np.abs(b - s).max() >= 20 * 4 * scale * 5e-4
            else:
                np.testing.assert_allclose(a, b, rtol=0, atol=4 * STEPS * 5e-4 * 0.1 * RATE
                                           + 2.0 ** -18 * np.abs(b).max())
        for a, b in zip(got["slots"], one["slots"]):
            assert np.abs(a - b).max() <= 4 * STEPS * 5e-4 * np.abs(b).max()
