"""What the Newton-Schulz products and the Muon update refuse, and that a refused call changed
nothing: the same on the CPU, where the graph is built, and on the GPU."""
import ctypes

import numpy as np
import pytest
import torch

import distributed_tensorflow_amd as tf

COEF = (3.4445, -4.7750, 2.0315)


def test_shapes_beyond_the_kernels_range_are_refused_on_the_host():
    """(Sizes that do not fit a C int would otherwise arrive as their low 32 bits.)"""
    from distributed_tensorflow_amd.ops import hip
    if not hip.library_present():
        pytest.skip("native library not built")
    for shape in ((2 ** 32 + 5, 1), (7, 2 ** 32 + 9), (4000001, 3), (3, 4000001), (300000, 300000)):
        with pytest.raises(hip.HipKernelError, match="matrices of up to"):
            hip._ns_groups([(4, 5), shape], "cpu", "newton_schulz")
    groups, (ws, base, size) = hip._ns_groups([(4, 5)] * 16 + [(96, 80)] * 2, "cpu", "newton_schulz")
    assert [g[:2] for g in groups] == [(0, 16), (16, 18)] and base % 256 == 0
    ints = ctypes.c_int * 2
    assert size >= hip.lib().dtf_newton_schulz_workspace(2, ints(96, 96), ints(80, 80)) - 256


@pytest.mark.parametrize("rows", [(9.0, 0.0, 0.0), (float("nan"), 0.0, 0.0), (20.0, -40.0, 20.0),
                                  (1.0, float("inf"), 0.0), [COEF, (4.0, 0.0, 0.0)]])
def test_coefficients_are_refused_where_the_graph_is_built(rows):
    steps = 2 if hasattr(rows[0], "__len__") else 5
    with pytest.raises(ValueError, match="grow beyond"):
        tf.newton_schulz(tf.placeholder(tf.float32, [6, 4]), steps=steps, coefficients=rows)
    with pytest.raises(ValueError, match="grow beyond"):
        tf.train.MuonOptimizer(0.1, steps=steps, coefficients=rows)


def test_matrices_beyond_the_kernels_range_are_refused_where_the_graph_is_built():
    for shape in ([4000001, 3], [2, 3, 4000001], [300000, 300000], [None, 4000001]):
        with pytest.raises(ValueError, match="matrices of up to"):
            tf.newton_schulz(tf.placeholder(tf.float32, shape))
    tf.newton_schulz(tf.placeholder(tf.float32, [None, 40]))
    w = tf.Variable(tf.zeros([4000001, 1]), name="long")
    with pytest.raises(ValueError, match="matrices of up to"):
        tf.train.MuonOptimizer(0.1).apply_gradients([(tf.identity(w), w)])


@pytest.mark.parametrize("shape", [(0, 4, 5), (3, 0, 5), (0, 4), (4, 0)])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def test_empty_variables_are_updated_to_themselves(shape, device):
    with tf.Graph().as_default():
        w = tf.Variable(tf.zeros(list(shape)), name="none")
        full = tf.Variable(tf.ones([2, 3]), name="some")
        train = tf.train.MuonOptimizer(0.1).apply_gradients(
            [(tf.zeros(list(shape)), w), (tf.ones([2, 3]), full)])
        with tf.Session(config=tf.ConfigProto(device=device)) as sess:
            sess.run(tf.global_variables_initializer())
            sess.run(train)
            a, b = sess.run([w, full])
    assert a.shape == shape and np.abs(b - 1.0).max() > 0


def test_graph_and_library_refuse_the_same_coefficients():
    from distributed_tensorflow_amd.framework.ops import newton_schulz_steps
    from distributed_tensorflow_amd.ops import hip
    if not hip.library_present():
        pytest.skip("native library not built")
    rng = np.random.RandomState(0)
    lib, ints, ptrs = hip.lib(), ctypes.c_int * 1, ctypes.c_void_p * 1
    taken = 0
    for trial in range(400):
        steps = int(rng.randint(1, 6))
        rows = [tuple(np.array(COEF) * (1 + 0.3 * rng.randn(3)) * rng.choice([1.0, 0.0, 1.0, 1.0], 3))
                for _ in range(steps)]
        if trial % 10 == 0:
            rows = [(1.5, -0.5, 0.0)] * steps
        # (no workspace: -1 once the coefficients are taken, -2 before)
        code = lib.dtf_newton_schulz(1, ptrs(4096), ptrs(4096), ints(96), ints(80), 0, steps,
                                     (ctypes.c_float * (3 * steps))(*[v for r in rows for v in r]),
                                     1e-7, 4096, 0, None)
        try:
            newton_schulz_steps(steps, rows)
            assert code == -1, rows
            taken += 1
        except ValueError:
            assert code == -2, rows
    assert 60 < taken < 340


@pytest.fixture(scope="module")
def hip():
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    from distributed_tensorflow_amd.ops import hip as h
    h.lib()
    return h


@pytest.mark.gpu
def test_a_refused_update_of_many_matrices_changed_nothing(hip):
    """The 17th matrix, in the second group of launches, is too long."""
    shapes = [(20, 30)] * 16 + [(4000001, 1)]
    ws = [torch.ones(s, device="cuda") for s in shapes]
    vs = [torch.ones(s, device="cuda") for s in shapes]
    gs = [torch.full(s, 0.5, device="cuda") for s in shapes]
    with pytest.raises(hip.HipKernelError, match="matrices of up to"):
        hip.multi_muon(ws, gs, vs, 0.1)
    for t in ws + vs:
        assert torch.equal(t, torch.ones_like(t))
    hip.multi_muon(ws[:16], gs[:16], vs[:16], 0.1)
    assert not torch.equal(ws[0], torch.ones_like(ws[0]))


@pytest.mark.gpu
def test_groups_of_launches_share_a_workspace(hip):
    """33 matrices in three groups, of other forms and sizes in each: what each is alone."""
    shapes = ([(20, 30)] * 8 + [(100, 90)] * 8) + [(100, 784), (784, 100)] * 8 + [(9, 300)]
    gen = torch.Generator().manual_seed(0)
    mats = [torch.randn(s, generator=gen).cuda() for s in shapes]
    alone = [hip.newton_schulz(m) for m in mats]
    for _ in range(2):
        for a, b in zip(hip.newton_schulz(mats), alone):
            # (mid matrices beside thin ones keep their kernels, so the bits are the same)
            assert torch.equal(a, b)
