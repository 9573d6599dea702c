"""Layer normalisation: the graph op, its gradient and the layer on the CPU; the gfx950 kernels
against a 64-bit computation of the same formulas on the GPU.

Tolerances count roundings. u = 2^-24 is half a step of fp32. A sum over a row adds at most
K = 40 + cols / 1024 terms one after the other on its way (16 or fewer in a lane, or cols / 8192
vectors of 8 in the kernels for long rows, then 4-10 levels of a tree), so it is off by at most
K u times the sum of magnitudes. A 16-bit result adds one rounding of its own, eps / 2."""
import numpy as np
import pytest
import torch

import distributed_tensorflow_amd as tf

U = 2.0 ** -24
EPS = 1e-5
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


# ---------------------------------------------------------------------------------------
# the formulas in 64 bits, with bounds of the fp32 kernels' error
# ---------------------------------------------------------------------------------------
def _final(exact, dtype):
    """Half a step of the result's type; fp16 adds half its subnormal step."""
    return exact.abs() * (torch.finfo(dtype).eps / 2) + (2.0 ** -25 if dtype == F16 else 0.0)


def forward_exact(x, gamma, beta, eps=EPS):
    xd = x.double().cpu()
    n = xd.shape[-1]
    g = gamma.double().cpu() if gamma is not None else torch.ones(n, dtype=torch.float64)
    b = beta.double().cpu() if beta is not None else torch.zeros(n, dtype=torch.float64)
    mean = xd.mean(-1, keepdim=True)
    var = (xd - mean).square().mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    h = (xd - mean) * rstd
    y = h * g + b
    k = 40 + n / 1024
    # the differences from the mean carry 2u of themselves and K u of their mean magnitude (<= 1
    # in units of the deviation); rstd carries (K / 2 + 4) u
    tol = U * g.abs() * (h.abs() * (k / 2 + 8) + k) + 2 * U * y.abs() + _final(y, x.dtype)
    return (y, tol, mean.squeeze(-1), rstd.squeeze(-1),
            U * (mean.abs() + k * torch.sqrt(var)).squeeze(-1), U * (k / 2 + 4) * rstd.squeeze(-1))


def backward_exact(dy, x, mean, rstd, gamma, rows_per_sum):
    d, xd = dy.double().cpu(), x.double().cpu()
    n = xd.shape[-1]
    d, xd = d.reshape(-1, n), xd.reshape(-1, n)
    r = rstd.double().cpu().reshape(-1, 1)
    g = gamma.double().cpu() if gamma is not None else torch.ones(n, dtype=torch.float64)
    h = (xd - mean.double().cpu().reshape(-1, 1)) * r
    gg = d * g
    s, q = gg.mean(-1, keepdim=True), (gg * h).mean(-1, keepdim=True)
    dx = r * (gg - s - h * q)
    k = 40 + n / 1024
    # h carries 3u, the two means K u of their magnitudes, the three terms 4u each
    tol = r * U * (8 * (gg.abs() + s.abs() + (h * q).abs())
                   + k * (gg.abs().mean(-1, keepdim=True)
                          + h.abs() * (gg * h).abs().mean(-1, keepdim=True)))
    k2 = 100 + rows_per_sum          # a lane's rows, its row group's and its workgroup's fold
    p_t = gamma.dtype if gamma is not None else F32
    dgamma, dbeta = (d * h).sum(0), d.sum(0)
    t_g = U * (k2 + 4) * (d * h).abs().sum(0) + _final(dgamma, p_t)
    t_b = U * k2 * d.abs().sum(0) + _final(dbeta, p_t)
    return (dx, tol + _final(dx, x.dtype)), (dgamma, t_g), (dbeta, t_b)


def _check(got, want, tol, what):
    err = (got.double().cpu().reshape(want.shape) - want).abs()
    worst = (err - tol).max().item() if err.numel() else 0.0
    assert not torch.isnan(err).any() and worst <= 0.0, (what, worst, err.max().item())


def _data(rows, cols, dtype, p_dtype, seed=0):
    gen = torch.Generator().manual_seed(seed * 7919 + rows * 31 + cols)
    x = torch.randn(rows, cols, generator=gen) * torch.exp(torch.randn(rows, 1, generator=gen)) \
        + 3.0 * torch.randn(rows, 1, generator=gen)
    dy = torch.randn(rows, cols, generator=gen)
    gamma = 1.0 + 0.3 * torch.randn(cols, generator=gen)
    beta = torch.randn(cols, generator=gen)
    return x.to(dtype), dy.to(dtype), gamma.to(p_dtype), beta.to(p_dtype)


# ---------------------------------------------------------------------------------------
# graph level
# ---------------------------------------------------------------------------------------
def _graph_run(device, x, dy, gamma, beta, fusion=True):
    """y and the gradients of sum(y * dy) through a session."""
    g = tf.Graph()
    with g.as_default():
        xp = tf.placeholder(tf.float32, [None, x.shape[1]])
        gv = tf.Variable(tf.constant(gamma), name="gamma") if gamma is not None else None
        bv = tf.Variable(tf.constant(beta), name="beta") if beta is not None else None
        y = tf.nn.layer_norm(xp, gv, bv, epsilon=EPS)
        loss = tf.reduce_sum(tf.multiply(y, tf.placeholder(tf.float32, [None, x.shape[1]],
                                                           name="dy")))
        dyp = g.get_operation_by_name("dy").outputs[0]
        wrt = [xp] + [v for v in (gv, bv) if v is not None]
        grads = tf.gradients(loss, wrt)
        with tf.Session(config=tf.ConfigProto(device=device, graph_fusion=fusion)) as sess:
            sess.run(tf.global_variables_initializer())
            return sess.run([y] + grads, {xp: x, dyp: dy})


@pytest.mark.parametrize("params", ["both", "gamma", "beta", "none"])
def test_graph_op_and_gradient_on_the_cpu(params):
    x, dy, gamma, beta = (t.numpy() for t in _data(7, 13, F32, F32))
    gamma = gamma if params in ("both", "gamma") else None
    beta = beta if params in ("both", "beta") else None
    got = _graph_run("cpu", x, dy, gamma, beta)

    def value(xv, gv, bv):
        mean = xv.mean(1, keepdims=True)
        h = (xv - mean) / np.sqrt(((xv - mean) ** 2).mean(1, keepdims=True) + EPS)
        return h * (1.0 if gv is None else gv) + (0.0 if bv is None else bv)
    x64, d64 = x.astype(np.float64), dy.astype(np.float64)
    np.testing.assert_allclose(got[0], value(x64, gamma, beta), rtol=2e-6, atol=2e-6)
    # central differences of sum(y * dy)
    step = 1e-5
    args = [x64] + [p.astype(np.float64) for p in (gamma, beta) if p is not None]
    for i, arg in enumerate(args):
        num = np.zeros_like(arg)
        for idx in np.ndindex(*arg.shape):
            vals = []
            for sgn in (1, -1):
                moved = [a.copy() for a in args]
                moved[i][idx] += sgn * step
                rest = moved[1:]
                gv = rest.pop(0) if gamma is not None else None
                bv = rest.pop(0) if beta is not None else None
                vals.append((value(moved[0], gv, bv) * d64).sum())
            num[idx] = (vals[0] - vals[1]) / (2 * step)
        np.testing.assert_allclose(got[1 + i], num, rtol=1e-4, atol=1e-4)


def test_layer_creates_its_variables_and_trains_them():
    x = tf.placeholder(tf.float32, [None, 6])
    h = tf.layers.layer_norm(tf.layers.dense(x, 5, name="hidden"), activation=tf.nn.relu,
                             name="norm")
    bare = tf.layers.layer_norm(h, center=False, scale=False, name="bare")
    names = [v.op.name for v in tf.trainable_variables()]
    assert names == ["hidden/kernel", "hidden/bias", "norm/gamma", "norm/beta"]
    loss = tf.reduce_sum(tf.square(bare))
    train = tf.train.GradientDescentOptimizer(0.1).minimize(
        tf.add(loss, tf.reduce_sum(tf.square(h))))
    with tf.Session(config=tf.ConfigProto(device="cpu")) as sess:
        sess.run(tf.global_variables_initializer())
        before = sess.run(tf.trainable_variables())
        sess.run(train, {x: np.random.RandomState(0).randn(9, 6).astype(np.float32)})
        after = sess.run(tf.trainable_variables())
    np.testing.assert_array_equal(before[2], np.ones(5, np.float32))
    for b, a, n in zip(before[2:], after[2:], names[2:]):
        assert not np.array_equal(a, b), n


def test_graph_op_refuses_what_it_does_not_cover():
    x = tf.placeholder(tf.float32, [None, 8])
    with pytest.raises(ValueError, match="last dimension"):
        tf.nn.layer_norm(tf.placeholder(tf.float32, [4, None]))
    with pytest.raises(ValueError, match="last dimension"):
        tf.nn.layer_norm(tf.placeholder(tf.float32, [4, 0]))
    with pytest.raises(TypeError, match="int32"):
        tf.nn.layer_norm(tf.placeholder(tf.int32, [4, 8]))
    with pytest.raises(ValueError, match="scale has shape"):
        tf.nn.layer_norm(x, tf.ones([7]))
    with pytest.raises(ValueError, match="epsilon"):
        tf.nn.layer_norm(x, epsilon=-1.0)
    with pytest.raises(ValueError, match="epsilon"):
        tf.nn.layer_norm(x, epsilon=float("nan"))
    with pytest.raises(TypeError, match="offset"):
        tf.nn.layer_norm(x, tf.ones([8]), tf.placeholder(tf.bfloat16, [8]))


def test_entry_points_reject_bad_arguments_without_a_gpu():
    from distributed_tensorflow_amd.ops import hip
    if not hip.library_present():
        pytest.skip("native library not built")
    lib = hip.lib()
    z = 0

    def fwd(ldx=8, xt=0, pt=0, mean=None, rstd=None, rows=4, cols=8, eps=1e-5, x=None):
        return lib.dtf_layer_norm(x, ldx, xt, None, None, pt, x, mean, rstd, rows, cols, eps, z)
    assert fwd() == -1                            # no tensors
    assert fwd(rows=0) == 0                       # nothing to do
    for bad in (dict(cols=0), dict(rows=-1), dict(ldx=7), dict(xt=3), dict(xt=1, pt=2),
                dict(eps=-1.0), dict(eps=float("nan")), dict(mean=64), dict(cols=1 << 31)):
        assert fwd(**dict(dict(x=4096), **bad)) == -1, bad
    assert lib.dtf_layer_norm_grad_workspace(4, 0, 0) == 0
    assert lib.dtf_layer_norm_grad_workspace(4, 8, 0) >= 16
    assert lib.dtf_layer_norm_grad(4096, 8, 4096, 8, 0, 4096, 4096, None, 0, 4096, None, 4096,
                                   None, 4, 8, z) == -1     # sums without a workspace
    with pytest.raises(hip.HipKernelError, match="GPU tensor"):
        hip.layer_norm(torch.zeros(2, 3))
    with pytest.raises(hip.HipKernelError, match="GPU tensor"):
        hip.layer_norm_grad(torch.zeros(2, 3), torch.zeros(2, 3), torch.zeros(2), torch.zeros(2))


# ---------------------------------------------------------------------------------------
# kernels
# ---------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def hip():
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    from distributed_tensorflow_amd.ops import hip as h
    h.lib()
    return h


# every plan of the launcher from both sides of its borders, then widths off every grid
COLS = [1, 2, 3, 7, 64, 65, 100, 128, 129, 256, 257, 500, 512, 513, 784, 1000, 1024, 1025, 1537,
        2048, 2049, 4096, 4097, 8191, 8192, 8193, 16384, 16385, 40001]
TYPES = [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,p_dtype", TYPES)
@pytest.mark.parametrize("cols", COLS)
def test_forward_and_backward_match_64_bits(hip, cols, dtype, p_dtype):
    for rows in (1, 3, 70):
        x, dy, gamma, beta = (t.cuda() for t in _data(rows, cols, dtype, p_dtype))
        y, mean, rstd = hip.layer_norm(x, gamma, beta, EPS, want_stats=True)
        ey, ty, em, er, tm, tr = forward_exact(x, gamma, beta)
        assert y.dtype == dtype and y.shape == x.shape
        _check(y, ey, ty, "y")
        _check(mean, em, tm, "mean")
        _check(rstd, er, tr, "rstd")
        got = hip.layer_norm_grad(dy, x, mean, rstd, gamma)
        for what, t, (want, tol) in zip(("dx", "dgamma", "dbeta"), got,
                                        backward_exact(dy, x, mean, rstd, gamma, rows / 256)):
            _check(t, want, tol, (what, rows))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,dtype", [(10000, 784, F32), (4099, 100, F32),
                                             (20011, 17, BF16), (2053, 1537, BF16),
                                             (3001, 2048, F16), (1100, 9000, F32),
                                             (70003, 1, F32)])
def test_many_rows(hip, rows, cols, dtype):
    x, dy, gamma, beta = (t.cuda() for t in _data(rows, cols, dtype, F32))
    y, mean, rstd = hip.layer_norm(x, gamma, beta, EPS, want_stats=True)
    ey, ty, em, er, tm, tr = forward_exact(x, gamma, beta)
    _check(y, ey, ty, "y")
    _check(rstd, er, tr, "rstd")
    first = hip.layer_norm_grad(dy, x, mean, rstd, gamma)
    for what, t, (want, tol) in zip(("dx", "dgamma", "dbeta"), first,
                                    backward_exact(dy, x, mean, rstd, gamma, rows / 256)):
        _check(t, want, tol, what)
    again = hip.layer_norm_grad(dy, x, mean, rstd, gamma)       # fixed order: the same bits
    for a, b in zip(first, again):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_absent_parameters_and_unwanted_sums(hip, dtype):
    x, dy, gamma, beta = (t.cuda() for t in _data(33, 130, dtype, F32))
    for g, b in ((None, None), (gamma, None), (None, beta)):
        y, mean, rstd = hip.layer_norm(x, g, b, EPS, want_stats=True)
        assert torch.equal(y, hip.layer_norm(x, g, b, EPS))
        ey, ty = forward_exact(x, g, b)[:2]
        _check(y, ey, ty, "y")
        full = hip.layer_norm_grad(dy, x, mean, rstd, g)
        for what, t, (want, tol) in zip(("dx", "dgamma", "dbeta"), full,
                                        backward_exact(dy, x, mean, rstd, g, 1)):
            _check(t, want, tol, what)
        for wg, wb in ((True, False), (False, True), (False, False)):
            part = hip.layer_norm_grad(dy, x, mean, rstd, g, wg, wb)
            assert torch.equal(part[0], full[0])
            for want, t, f in zip((wg, wb), part[1:], full[1:]):
                assert (t is None) if not want else torch.equal(t, f)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [64, 100, 301])
def test_pitches_offsets_and_ranks(hip, cols, dtype):
    """Rows inside a wider matrix, at every alignment of their first element; inputs of rank 1
    and 3; transposed inputs; results that do not depend on where the rows lie."""
    x, dy, gamma, beta = (t.cuda() for t in _data(40, cols, dtype, F32))
    y, mean, rstd = hip.layer_norm(x, gamma, beta, EPS, want_stats=True)
    grads = hip.layer_norm_grad(dy, x, mean, rstd, gamma)
    for offset in range(0, 9):
        wide = torch.full((40, cols + 13), float("nan"), dtype=dtype, device="cuda")
        wide_d = wide.clone()
        xs, ds = wide[:, offset:offset + cols], wide_d[:, offset:offset + cols]
        xs.copy_(x)
        ds.copy_(dy)
        assert torch.equal(hip.layer_norm(xs, gamma, beta, EPS), y)
        for a, b in zip(hip.layer_norm_grad(ds, xs, mean, rstd, gamma), grads):
            assert torch.equal(a, b)
    shifted = torch.empty(cols + 1, device="cuda")[1:]
    shifted.copy_(gamma)
    assert torch.equal(hip.layer_norm(x, shifted, beta, EPS), y)
    y3, m3, _ = hip.layer_norm(x.view(4, 10, cols), gamma, beta, EPS, want_stats=True)
    assert y3.shape == (4, 10, cols) and m3.shape == (4, 10)
    assert torch.equal(y3.view(40, cols), y)
    y1, m1, r1 = hip.layer_norm(x[3], gamma, beta, EPS, want_stats=True)
    assert y1.shape == (cols,) and m1.shape == () and torch.equal(y1, y[3])
    d1 = hip.layer_norm_grad(dy[3], x[3], m1, r1, gamma)
    assert d1[0].shape == (cols,) and torch.equal(d1[0], grads[0][3])
    assert torch.equal(hip.layer_norm(x.t().contiguous().t(), gamma, beta, EPS), y)
    same = x[:1].expand(5, cols)
    assert torch.equal(hip.layer_norm(same, gamma, beta, EPS), y[:1].expand(5, cols))


@pytest.mark.gpu
def test_no_rows_and_one_column(hip):
    x = torch.empty(0, 37, device="cuda")
    y, mean, rstd = hip.layer_norm(x, want_stats=True)
    assert y.shape == (0, 37) and mean.shape == (0,)
    for cols in (37, 50000):
        x = torch.empty(0, cols, device="cuda")
        dx, dg, db = hip.layer_norm_grad(x, x, mean, rstd)
        assert dx.shape == (0, cols)
        assert torch.equal(dg, torch.zeros(cols, device="cuda")) and torch.equal(dg, db)
    # one column: the row is its own mean
    x = torch.tensor([[3.0], [-1e30]], device="cuda")
    beta = torch.tensor([0.25], device="cuda")
    assert torch.equal(hip.layer_norm(x, None, beta), torch.full((2, 1), 0.25, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [100, 1000, 5000, 20000])
def test_special_values_stay_in_their_row(hip, cols):
    x, dy, gamma, beta = (t.cuda() for t in _data(9, cols, F32, F32))
    y = hip.layer_norm(x, gamma, beta, EPS)
    bad = x.clone()
    bad[2, cols // 2] = float("nan")
    bad[5, cols - 1] = float("inf")
    got = hip.layer_norm(bad, gamma, beta, EPS)
    keep = [0, 1, 3, 4, 6, 7, 8]
    assert torch.equal(got[keep], y[keep])
    assert torch.isnan(got[2]).all() and torch.isnan(got[5]).all()
    # constant rows: no variance, so y is beta exactly
    const = torch.full((2, cols), 7.5, device="cuda")
    assert torch.equal(hip.layer_norm(const, gamma, beta, EPS), beta.expand(2, cols))
    # a row far from zero keeps its digits: the offset is a power of two, so x is exact
    far = torch.round(x * 64) / 64 + 4096.0
    ey, ty = forward_exact(far, gamma, beta)[:2]
    _check(hip.layer_norm(far, gamma, beta, EPS), ey, ty, "far")


@pytest.mark.gpu
def test_offsets_beyond_31_bits(hip):
    rows, pitch, cols = 70000, 40000, 70
    big = torch.empty(rows, pitch, dtype=BF16, device="cuda")
    x = big[:, 11:11 + cols]
    x.normal_()
    xc = x.contiguous()
    y, mean, rstd = hip.layer_norm(x, want_stats=True)
    yc = hip.layer_norm(xc)
    assert torch.equal(y, yc)
    a = hip.layer_norm_grad(x, x, mean, rstd)
    b = hip.layer_norm_grad(xc, xc, mean, rstd)
    for s, t in zip(a, b):
        assert torch.equal(s, t)


@pytest.mark.gpu
def test_other_streams_and_captured_replays(hip):
    x, dy, gamma, beta = (t.cuda() for t in _data(300, 784, F32, F32))
    y, mean, rstd = hip.layer_norm(x, gamma, beta, EPS, want_stats=True)
    grads = hip.layer_norm_grad(dy, x, mean, rstd, gamma)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y2 = hip.layer_norm(x, gamma, beta, EPS)
        g2 = hip.layer_norm_grad(dy, x, mean, rstd, gamma)
    side.synchronize()
    assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(grads, g2))
    xin, din = x.clone(), dy.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hip.layer_norm(xin, gamma, beta, EPS, want_stats=True)
        gout = hip.layer_norm_grad(din, xin, out[1], out[2], gamma)
    for seed in (1, 2, 3):
        xn, dn, _, _ = (t.cuda() for t in _data(300, 784, F32, F32, seed))
        xin.copy_(xn)
        din.copy_(dn)
        graph.replay()
        want = hip.layer_norm(xn, gamma, beta, EPS, want_stats=True)
        gwant = hip.layer_norm_grad(dn, xn, want[1], want[2], gamma)
        torch.cuda.synchronize()
        for a, b in zip(list(out) + list(gout), list(want) + list(gwant)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_wrapper_refusals(hip):
    x = torch.zeros(4, 8, device="cuda")
    ok = torch.zeros(8, device="cuda")
    s = torch.zeros(4, device="cuda")
    E = hip.HipKernelError
    for call in (lambda: hip.layer_norm(x.double()),
                 lambda: hip.layer_norm(torch.zeros(4, 0, device="cuda")),
                 lambda: hip.layer_norm(torch.zeros((), device="cuda")),
                 lambda: hip.layer_norm(x, ok[:7]),
                 lambda: hip.layer_norm(x, ok.cpu()),
                 lambda: hip.layer_norm(x, ok.bfloat16()),
                 lambda: hip.layer_norm(x.bfloat16(), ok, ok.bfloat16()),
                 lambda: hip.layer_norm(x, epsilon=-1e-5),
                 lambda: hip.layer_norm_grad(x[:3], x, s, s),
                 lambda: hip.layer_norm_grad(x.bfloat16(), x, s, s),
                 lambda: hip.layer_norm_grad(x, x, s[:3], s),
                 lambda: hip.layer_norm_grad(x, x, s, s.double()),
                 lambda: hip.layer_norm_grad(x, x, s, s, ok[:5]),
                 lambda: hip.layer_norm_grad(x, x, s, s, param_dtype=torch.float16),
                 lambda: hip.layer_norm_grad(x, x, s, s, dgamma_out=ok[:5])):
        with pytest.raises(E):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("params", ["both", "gamma", "none"])
def test_session_runs_the_kernels(params):
    x, dy, gamma, beta = (t.numpy() for t in _data(50, 97, F32, F32))
    gamma = gamma if params != "none" else None
    beta = beta if params == "both" else None
    want = _graph_run("cpu", x, dy, gamma, beta)
    for fusion in (True, False):
        got = _graph_run("cuda:0", x, dy, gamma, beta, fusion)
        for g, w in zip(got, want):
            # both sides are fp32; the column sums over 50 rows are the longest chains
            np.testing.assert_allclose(g, w, rtol=2e-5, atol=2e-5)
