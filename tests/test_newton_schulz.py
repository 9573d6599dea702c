"""Newton-Schulz orthogonalisation and the Muon update: graph op, optimizer and refusals on the
CPU; the gfx950 kernels against a 64-bit computation on the GPU.

Tolerances. The kernels keep every operand of a product as two fp16 numbers (at most 2^-23 of it
lost), drop the product of the two small parts (2^-22 of a term) and add in fp32. Relative to the
largest singular value of its operand each of a step's three products is therefore off by no more
than d = 2^-20 in the spectral norm (a few terms of 2^-22, and the fp32 accumulation, whose error
grows with the root of the number of 32-term sums). An error made before step k passes through
the remaining steps' polynomials: a singular value's own change by p' <= a, and the rotation of a
pair (s_i, s_j) by (p(s_i) + p(s_j)) / (s_i + s_j) <= a. Over five steps of a = 3.4445 the first
step's errors grow 485-fold, so the result, of norm about one, is off by at most
3 d (a^5 + a^4 + ... + 1) < 700 * 3 * 2^-20 = 2e-3 in the spectral norm when the largest singular
value of the normalised input is one (rank one), and by that value times as much when it is
smaller: ``_spectral_bound``. Those are worst cases of aligned errors; the root mean square of an
element's error is held to the same bound times the root mean square of the result.
Long matrices take two steps as one, X = B'(A') B X with A' = B A B: seven products. An error of d
on A' changes B' by (|b| + 2 |c|) d < 9 d and one of d on A changes A' by a^2 d < 12 d, both times
the square of the largest singular value; aligned worst cases may so reach a few times the bound
of single steps when that value is near one, which errors of random sign do not: the same bound is
asked of them.
A 16-bit result adds its own rounding, eps / 2 per element."""
import numpy as np
import pytest
import torch

import distributed_tensorflow_amd as tf

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
COEF = (3.4445, -4.7750, 2.0315)


def exact(g, steps=5, coef=COEF, eps=1e-7):
    x = g.double().cpu()
    x = x / (torch.linalg.norm(x) + eps)
    rows = [coef] * steps if not hasattr(coef[0], "__len__") else coef
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    for a, b, c in rows:
        s = x @ x.t()
        x = a * x + (b * s + c * s @ s) @ x
    return x.t() if tall else x


def _spectral_bound(g, steps=5, growth=3.4445):
    x = g.double().cpu()
    norm = torch.linalg.norm(x)
    top = (torch.linalg.matrix_norm(x, 2) / norm).item() if norm > 0 else 1.0
    total, err = 0.0, 0.0
    for k in range(steps):
        # this step's own error, relative to the largest singular value on entry
        own = 3 * 2.0 ** -20 * max(min(1.3, top * growth ** k), 2.0 ** -10) * growth
        err = err * growth + own
    return err


def _check(got, g, dtype, **kw):
    want = exact(g, **kw)
    bound = _spectral_bound(g, kw.get("steps", 5))
    diff = got.double().cpu() - want
    assert got.shape == g.shape and got.dtype == dtype
    round_off = want.abs() * (torch.finfo(dtype).eps / 2) * 1.001
    if dtype == F32:
        round_off = round_off * 4
    elif dtype == F16:
        round_off = round_off + 2.0 ** -25
    excess = (diff.abs() - round_off).clamp(min=0)
    assert not torch.isnan(diff).any()
    # the spectral norm is at least the Frobenius norm over the root of the rank, and at least
    # every element
    fro = torch.linalg.norm(excess).item() / max(1, min(g.shape)) ** 0.5
    assert fro <= bound and excess.max().item() <= bound, (fro, excess.max().item(), bound)


def _matrix(rows, cols, kind="gauss", seed=0):
    gen = torch.Generator().manual_seed(seed * 1009 + rows * 17 + cols)
    if kind == "gauss":
        return torch.randn(rows, cols, generator=gen)
    if kind == "rank_one":
        return torch.outer(torch.randn(rows, generator=gen), torch.randn(cols, generator=gen))
    rank = max(1, min(rows, cols) // 4)
    return torch.randn(rows, rank, generator=gen) @ torch.randn(rank, cols, generator=gen) * 1e-3


def muon_exact(w, g, v, lr, mu=0.95, nesterov=True, decay=0.0, scale=None, **kw):
    w, g, v = (t.double().cpu() for t in (w, g, v))
    v = mu * v + g
    u = g + mu * v if nesterov else v
    s = max(1.0, w.shape[1] / w.shape[0]) ** 0.5 if scale is None else scale
    return (1 - lr * decay) * w - lr * s * exact(u, **kw), v, u


# ---------------------------------------------------------------------------------------
# without a GPU
# ---------------------------------------------------------------------------------------
def test_entry_points_reject_bad_arguments_without_a_gpu():
    import ctypes
    from distributed_tensorflow_amd.ops import hip
    if not hip.library_present():
        pytest.skip("native library not built")
    lib = hip.lib()
    ints = lambda *v: (ctypes.c_int * len(v))(*v)                       # noqa: E731
    ptrs = lambda *v: (ctypes.c_void_p * len(v))(*v)                    # noqa: E731
    coef = lambda *v: (ctypes.c_float * len(v))(*v)                     # noqa: E731
    need = lib.dtf_newton_schulz_workspace(1, ints(96), ints(80))
    assert need > 4 * (96 * 80 * 3 + 80 * 80 * 2)
    for bad in ((0, 5), (5, 0), (-1, 5), (1 << 23, 5)):
        assert lib.dtf_newton_schulz_workspace(1, ints(bad[0]), ints(bad[1])) == 0
    assert lib.dtf_newton_schulz_workspace(17, ints(*[4] * 17), ints(*[4] * 17)) == 0

    def call(count=1, g=4096, out=4096, rows=96, cols=80, type_=0, steps=1, c=COEF, eps=1e-7,
             ws=4096, size=need):
        return lib.dtf_newton_schulz(count, ptrs(g), ptrs(out), ints(rows), ints(cols), type_,
                                     steps, coef(*c), eps, ws, size, None)
    assert call(count=0) == 0
    for bad in (dict(count=-1), dict(g=None), dict(out=None), dict(rows=0), dict(cols=-3),
                dict(type_=3), dict(steps=0), dict(steps=33), dict(eps=-1.0),
                dict(eps=float("nan")), dict(ws=None), dict(ws=4097), dict(size=need // 2)):
        assert call(**bad) == -1, bad
    for c in ((9.0, 0.0, 0.0), (float("nan"), 0.0, 0.0), (20.0, -40.0, 20.0)):
        assert call(c=c) == -2, c
    one = ctypes.c_float * 1
    assert lib.dtf_multi_muon_f32(1, ptrs(4096), ptrs(4096), ptrs(None), one(1.0), ints(96),
                                  ints(80), 1, coef(*COEF), 1e-7, 0.1, None, 0.9, 1, 0.0, 4096,
                                  need, None) == -1
    for call in (lambda: hip.newton_schulz(torch.zeros(3, 4)),
                 lambda: hip.newton_schulz([torch.zeros(3, 4)]),
                 lambda: hip.newton_schulz(torch.zeros(3)),
                 lambda: hip.newton_schulz(torch.zeros(3, 4), steps=0),
                 lambda: hip.multi_muon([torch.zeros(3, 4)], [torch.zeros(3, 4)],
                                        [torch.zeros(3, 4)], 0.1)):
        with pytest.raises(hip.HipKernelError):
            call()


def test_product_kernels_use_no_scratch(tmp_path):
    """The products wait for their LDS-DMA requests with counted ``s_waitcnt vmcnt(N)``: a spilled
    register's loads and stores would be counted with them."""
    import os
    import re
    import shutil
    import subprocess
    from distributed_tensorflow_amd.ops import hip
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not installed")
    kernels = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(hip.__file__))), "csrc",
                           "kernels")
    asm = str(tmp_path / "k.s")
    subprocess.run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-S", "--cuda-device-only",
                    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-I" + kernels,
                    "-o", asm, os.path.join(kernels, "newton_schulz.hip")], check=True, timeout=600)
    sizes = [int(m.group(2)) for m in re.finditer(r"^(_Z\w+):.*?; ScratchSize: (\d+)",
                                                  open(asm).read(), re.S | re.M)
             if "ns_product_kernel" in m.group(1)]
    assert len(sizes) >= 10 and not any(sizes), sizes


# ---------------------------------------------------------------------------------------
# kernels
# ---------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def hip():
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    from distributed_tensorflow_amd.ops import hip as h
    h.lib()
    return h


# both sides of the 32-element chunks and the 64-wide tiles; thin ones; vectors; wide and tall
SHAPES = [(1, 1), (1, 2), (2, 1), (3, 3), (1, 300), (300, 1), (7, 31), (32, 32), (33, 32), (31, 65),
          (63, 64), (64, 65), (65, 129), (100, 10), (784, 100), (100, 784), (127, 128), (129, 500),
          (300, 301), (515, 1030)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("kind", ["gauss", "low_rank"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_newton_schulz_matches_64_bits(hip, rows, cols, kind, dtype):
    g = _matrix(rows, cols, kind).to(dtype).cuda()
    _check(hip.newton_schulz(g), g, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,dtype", [(2048, 2560, F32), (4100, 1900, BF16),
                                             (70, 60000, F32), (60001, 33, F32)])
def test_large_matrices(hip, rows, cols, dtype):
    g = _matrix(rows, cols, "low_rank").to(dtype).cuda()
    _check(hip.newton_schulz(g, steps=3), g, dtype, steps=3)


# (as many as it takes for the 256 x 128 tiles; odd edges on each side of them, wide and tall)
MANY = [(1001, 1003), (1003, 1001), (1009, 1011), (1024, 1021), (997, 1020), (1020, 999),
        (1018, 1023), (1010, 1009)]
MANY += [(c, r) for r, c in MANY[:7]] + [(70, 900)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
def test_many_large_matrices(hip, dtype):
    mats = [_matrix(r, c, ("low_rank", "gauss")[i % 2]).to(dtype).cuda()
            for i, (r, c) in enumerate(MANY)]
    outs = hip.newton_schulz(mats, steps=3)
    for g, out, again in zip(mats, outs, hip.newton_schulz(mats, steps=3)):
        assert torch.equal(out, again)
        _check(out, g, dtype, steps=3)


# up to 128 x 2048, which take one or two steps in a launch, and the sizes next to them
MID = [[(65, 65)], [(128, 128)], [(129, 128)], [(96, 97)], [(97, 96)], [(128, 2048)], [(2048, 128)],
       [(2049, 128)], [(66, 2047)], [(2000, 65)], [(100, 784), (784, 100), (10, 100), (128, 1000),
                                                   (65, 2048), (333, 81), (120, 120)] * 2]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("kind", ["gauss", "low_rank", "rank_one"])
@pytest.mark.parametrize("shapes", MID)
def test_mid_matrices(hip, shapes, kind, dtype):
    mats = [_matrix(r, c, kind, seed=i).to(dtype).cuda() for i, (r, c) in enumerate(shapes)]
    outs = hip.newton_schulz(mats)
    for g, out, again in zip(mats, outs, hip.newton_schulz(mats)):
        assert torch.equal(out, again)
        _check(out, g, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6])
def test_step_counts_of_mid_matrices(hip, steps):
    for g in (_matrix(100, 300).cuda(), _matrix(300, 90).cuda()):
        _check(hip.newton_schulz(g, steps=steps), g, F32, steps=steps)
    # factors whose product the images cannot hold: 4.2 and 4 stay single steps
    rows = [(4.2, -6.0, 2.4), (4.0, -2.85, 0.59), (2.0, -0.4, 0.035), (1.5, -0.1, 0.0)][:steps]
    _check(hip.newton_schulz(g, steps=len(rows), coefficients=rows), g, F32, steps=len(rows),
           coef=rows)


@pytest.mark.gpu
def test_special_values_of_mid_matrices(hip):
    mats = [torch.zeros(100, 200), _matrix(100, 200), _matrix(200, 100) * 1e-25, torch.zeros(70, 70),
            _matrix(90, 90) * 1e25]
    mats = [m.cuda() for m in mats]
    clean = hip.newton_schulz(mats, epsilon=0.0)
    for i in (0, 3):
        assert torch.isnan(clean[i]).all()                    # 0 / 0, in its own matrix alone
    for i in (1, 2, 4):
        _check(clean[i], mats[i], F32, eps=0.0)
    zeros = hip.newton_schulz(mats)
    assert torch.equal(zeros[0], mats[0]) and torch.equal(zeros[3], mats[3])
    for bad in (float("nan"), float("inf")):
        mats[1][7, 9] = bad
        out = hip.newton_schulz(mats, epsilon=0.0)
        assert torch.isnan(out[1]).any()
        for i in (2, 4):
            assert torch.equal(out[i], clean[i])


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_of_mid_matrices_on_a_stream_and_replayed(hip, nesterov):
    shapes = [(784, 100), (100, 10), (66, 70), (128, 2048), (1500, 97)]
    gs = [_matrix(*s).cuda() for s in shapes]
    ws, vs = ([_matrix(*s, seed=k).cuda() for s in shapes] for k in (1, 2))
    w0, v0 = [w.clone() for w in ws], [v.clone() for v in vs]
    want = [muon_exact(w, g, v, 0.05, nesterov=nesterov, decay=0.1) for w, g, v in zip(ws, gs, vs)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        hip.multi_muon(ws, gs, vs, 0.05, nesterov=nesterov, weight_decay=0.1)
    side.synchronize()
    for w, v, old, (ew, ev, u) in zip(ws, vs, w0, want):
        s = max(1.0, w.shape[1] / w.shape[0]) ** 0.5
        tol = 0.05 * s * _spectral_bound(u) + 4 * 2.0 ** -24 * (old.abs().max().item() + 0.05 * s)
        assert (w.double().cpu() - ew).abs().max().item() <= tol
        # the product, the sum and 0.95 itself round
        assert (v.double().cpu() - ev).abs().max().item() <= 4 * 2.0 ** -24 * ev.abs().max().item() * 2
    a, b = [w.clone() for w in w0], [v.clone() for v in v0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hip.multi_muon(a, gs, b, 0.05, nesterov=nesterov, weight_decay=0.1)
    for x, y in zip(a + b, w0 + v0):
        x.copy_(y)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(a + b, ws + vs):
            assert torch.equal(x, y)
        hip.multi_muon(ws, gs, vs, 0.05, nesterov=nesterov, weight_decay=0.1)


# long matrices, which take steps in pairs: alone, beside others, with products on either tile
LONG = [[(301, 7001)], [(7001, 129)], [(500, 8000), (40, 50), (333, 350), (8001, 300)],
        [(1300, 1701), (1701, 1300), (1299, 1699)]]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["gauss", "low_rank", "rank_one"])
@pytest.mark.parametrize("shapes", LONG)
def test_long_matrices(hip, shapes, kind):
    mats = [_matrix(r, c, kind).cuda() for r, c in shapes]
    for g, out in zip(mats, hip.newton_schulz(mats)):
        _check(out, g, F32)


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7])
def test_step_counts_of_long_matrices(hip, steps):
    g = _matrix(129, 6000).cuda()
    _check(hip.newton_schulz(g, steps=steps), g, F32, steps=steps)
    h = g.t().contiguous().bfloat16()
    _check(hip.newton_schulz(h, steps=steps), h, BF16, steps=steps)
    # factors whose product the images cannot hold: 4.2 and 4 stay single steps
    rows = [(4.2, -6.0, 2.4), (4.0, -2.85, 0.59), (2.0, -0.4, 0.035), (1.5, -0.1, 0.0)][:steps]
    _check(hip.newton_schulz(g, steps=len(rows), coefficients=rows), g, F32, steps=len(rows),
           coef=rows)


@pytest.mark.gpu
def test_wide_tiles_for_every_product(hip):
    shapes = [(2047, 2049), (2001, 1999), (1999, 5000), (5001, 1987)]
    mats = [_matrix(r, c).cuda() for r, c in shapes]
    for g, out in zip(mats, hip.newton_schulz(mats, steps=2)):
        _check(out, g, F32, steps=2)


@pytest.mark.gpu
def test_muon_of_many_large_matrices(hip):
    gs = [_matrix(r, c).cuda() for r, c in MANY]
    ws = [_matrix(r, c, seed=1).cuda() for r, c in MANY]
    vs = [_matrix(r, c, seed=2).cuda() for r, c in MANY]
    want = [muon_exact(w, g, v, 0.05, steps=3, decay=0.1) for w, g, v in zip(ws, gs, vs)]
    tops = [w.abs().max().item() for w in ws]
    hip.multi_muon(ws, gs, vs, 0.05, steps=3, weight_decay=0.1)
    for w, (ew, _, u), top in zip(ws, want, tops):
        s = max(1.0, w.shape[1] / w.shape[0]) ** 0.5
        tol = 0.05 * s * _spectral_bound(u, 3) + 4 * 2.0 ** -24 * (top + 0.05 * s)
        assert (w.double().cpu() - ew).abs().max().item() <= tol


@pytest.mark.gpu
def test_two_streams_at_once(hip):
    """Calls that run side by side have workspaces and arrival counts of their own."""
    sets = [[_matrix(300, 8000, seed=i).cuda()] if i % 2 else
            [_matrix(1024, 1024, seed=i).cuda(), _matrix(50, 70, seed=i).cuda()] for i in range(4)]
    want = [hip.newton_schulz(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[] for _ in sets]
    for _ in range(5):
        for s, stream, out in zip(sets, streams, got):
            with torch.cuda.stream(stream):
                out.append(hip.newton_schulz(s))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(w, out))


@pytest.mark.gpu
def test_singular_values_move_to_one(hip):
    """Against the definition on singular values: U p(p(...(S / |S|))) V^T."""
    g = _matrix(96, 160).cuda()
    u, s, vt = torch.linalg.svd(g.double().cpu(), full_matrices=False)
    s = s / (torch.linalg.norm(s) + 1e-7)
    for _ in range(5):
        s = COEF[0] * s + COEF[1] * s ** 3 + COEF[2] * s ** 5
    want = u @ torch.diag(s) @ vt
    got = hip.newton_schulz(g).double().cpu()
    assert (got - want).abs().max().item() <= _spectral_bound(g)


@pytest.mark.gpu
def test_steps_coefficients_and_epsilon(hip):
    g = _matrix(50, 90).cuda()
    for steps in (1, 2, 8):
        _check(hip.newton_schulz(g, steps=steps), g, F32, steps=steps)
    cubic = (1.5, -0.5, 0.0)
    _check(hip.newton_schulz(g, steps=4, coefficients=cubic), g, F32, steps=4, coef=cubic)
    rows = [(3.4445, -4.7750, 2.0315), (2.0, -1.5, 0.5), (1.5, -0.5, 0.0)]
    _check(hip.newton_schulz(g, steps=3, coefficients=rows), g, F32, steps=3, coef=rows)
    _check(hip.newton_schulz(g, epsilon=3.0), g, F32, eps=3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-30, 1e-18, 1e-6, 1e20, 3e37])
def test_inputs_of_any_size(hip, size):
    """The norm is taken in 64 bits: squares that fp32 does not hold do not matter."""
    g = (_matrix(40, 70) * 0.3 * size).cuda()
    eps = 0.0 if size < 1e-6 else 1e-7
    _check(hip.newton_schulz(g, epsilon=eps), g, F32, eps=eps)


@pytest.mark.gpu
def test_zero_and_non_finite_inputs(hip):
    zero = torch.zeros(30, 50, device="cuda")
    assert torch.equal(hip.newton_schulz(zero), zero)
    for bad in (float("nan"), float("inf")):
        g = _matrix(30, 50).cuda()
        g[3, 4] = bad
        clean = _matrix(70, 20).cuda()
        got = hip.newton_schulz([g, clean])
        assert torch.isnan(got[0]).all()
        assert torch.equal(got[1], hip.newton_schulz(clean))
    for shape in ((0, 5), (5, 0), (3, 0, 4)):
        e = torch.empty(shape, device="cuda")
        assert hip.newton_schulz(e).shape == shape
    assert hip.newton_schulz([]) == []


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_lists_stacks_and_views(hip, dtype):
    """Each matrix's result does not depend on what else is in the call, on where it lies or on
    the orientation it comes in."""
    shapes = [(100, 10), (33, 200), (1, 7), (64, 64), (90, 90)] * 4
    mats = [_matrix(r, c, seed=i).to(dtype).cuda() for i, (r, c) in enumerate(shapes)]
    alone = [hip.newton_schulz(m) for m in mats]
    for a, b in zip(hip.newton_schulz(mats), alone):
        assert torch.equal(a, b)
    stack = torch.stack(mats[3::5])
    out = hip.newton_schulz(stack)
    assert out.shape == stack.shape
    for i in range(len(stack)):
        assert torch.equal(out[i], alone[3::5][i])
    wide = torch.zeros(120, 40, dtype=dtype, device="cuda")
    wide[7:107, 3:13] = mats[0]
    assert torch.equal(hip.newton_schulz(wide[7:107, 3:13]), alone[0])
    flipped = mats[1].t().contiguous()
    a, b = hip.newton_schulz(flipped).float(), alone[1].float().t()
    assert torch.equal(hip.newton_schulz(flipped.t()), alone[1])
    assert (a - b).abs().max().item() <= _spectral_bound(mats[1]) + 2 * torch.finfo(dtype).eps


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov,decay", [(True, 0.0), (True, 0.1), (False, 0.01)])
def test_multi_muon_matches_64_bits(hip, nesterov, decay):
    shapes = [(784, 100), (100, 10), (1, 33), (64, 256), (130, 130)]
    gen = torch.Generator().manual_seed(5)
    ws = [torch.randn(s, generator=gen).cuda() for s in shapes]
    vs = [torch.randn(s, generator=gen).cuda() for s in shapes]
    lr = 0.05
    for step in range(2):
        gs = [torch.randn(s, generator=gen).cuda() for s in shapes]
        want = [muon_exact(w, g, v, lr, nesterov=nesterov, decay=decay)
                for w, g, v in zip(ws, gs, vs)]
        old = [(w.clone(), v.clone()) for w, v in zip(ws, vs)]
        hip.multi_muon(ws, gs, vs, lr if step else torch.tensor(lr, device="cuda"),
                       nesterov=nesterov, weight_decay=decay)
        for w, v, g, (ew, ev, u), (w0, v0) in zip(ws, vs, gs, want, old):
            s = max(1.0, w.shape[1] / w.shape[0]) ** 0.5
            # lr and the two factors are fp32; the sum rounds once more
            tol = lr * s * _spectral_bound(u) + 4 * 2.0 ** -24 * (w0.abs().max().item() + lr * s)
            assert (w.double().cpu() - ew).abs().max().item() <= tol
            # 0.95 in fp32 is off by half a step of itself, the product and the sum round once
            tol = 2.0 ** -24 * (2 * v0.abs() + g.abs() + 1.0).max().item() * 2
            assert (v.double().cpu() - ev).abs().max().item() <= tol


@pytest.mark.gpu
def test_multi_muon_stacks_scales_and_refusals(hip):
    gen = torch.Generator().manual_seed(6)
    w = torch.randn(3, 40, 60, generator=gen).cuda()
    g, v = torch.randn(3, 40, 60, generator=gen).cuda(), torch.zeros(3, 40, 60, device="cuda")
    w1, v1 = [t.clone() for t in w], [t.clone() for t in v]
    hip.multi_muon([w], [g], [v], 0.1, scales=[0.5])
    hip.multi_muon(w1, list(g), v1, 0.1, scales=[0.5] * 3)
    for i in range(3):
        assert torch.equal(w[i], w1[i]) and torch.equal(v[i], v1[i])
    m = torch.zeros(4, 5, device="cuda")
    a, b, c = m.clone(), m.clone(), m.clone()
    hip.multi_muon([torch.empty(0, 4, device="cuda")], [torch.empty(0, 4, device="cuda")],
                   [torch.empty(0, 4, device="cuda")], 0.1)
    # gradients that are, or lie in, a weight or a momentum: read before either is written
    buf = torch.randn(20, 40, 60, generator=gen).cuda()
    ps, gs, vs = list(buf[:17]), [*buf[1:17], buf[18]], [*buf[17:20], *torch.zeros(14, 40, 60).cuda()]
    want = [t.clone() for t in ps], [t.clone() for t in vs]
    hip.multi_muon(want[0], [g.clone() for g in gs], want[1], 0.1)
    hip.multi_muon(ps, gs, vs, 0.1)
    assert all(torch.equal(a, b) for a, b in zip(ps + vs, want[0] + want[1]))
    # (one gradient of two weights is fine)
    p, q, r = torch.zeros_like(m), torch.zeros_like(m), torch.randn(4, 5, generator=gen).cuda()
    hip.multi_muon([p, q], [r, r], [torch.zeros_like(m), torch.zeros_like(m)], 0.1)
    assert torch.equal(p, q) and p.abs().max() > 0
    for call in (lambda: hip.multi_muon([a], [b], [], 0.1),
                 lambda: hip.multi_muon([a], [b], [c], 0.1, scales=[]),
                 lambda: hip.multi_muon([a], [b], [a], 0.1),
                 lambda: hip.multi_muon([a, a], [b, b], [c, m], 0.1),
                 lambda: hip.multi_muon([a.t()], [b.t()], [c.t()], 0.1),
                 lambda: hip.multi_muon([a], [b.t()], [c], 0.1),
                 lambda: hip.multi_muon([a[0]], [b[0]], [c[0]], 0.1),
                 lambda: hip.multi_muon([a.bfloat16()], [b.bfloat16()], [c.bfloat16()], 0.1),
                 lambda: hip.multi_muon([a], [b], [c], torch.tensor(0.1)),
                 lambda: hip.multi_muon([a], [b], [c], 0.1, coefficients=(9.0, 0.0, 0.0)),
                 lambda: hip.newton_schulz(a, coefficients=(1.0, 2.0)),
                 lambda: hip.newton_schulz(a, steps=3, coefficients=[COEF] * 2),
                 lambda: hip.newton_schulz(a, epsilon=-1.0),
                 lambda: hip.newton_schulz(a.double()),
                 lambda: hip.newton_schulz([a, b.bfloat16()])):
        with pytest.raises(hip.HipKernelError):
            call()


@pytest.mark.gpu
def test_other_streams_and_captured_replays(hip):
    shapes = [(200, 150), (64, 64)]
    mats = [_matrix(r, c).cuda() for r, c in shapes]
    ref = hip.newton_schulz(mats)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = hip.newton_schulz(mats)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, out))
    ws = [torch.randn(s, generator=torch.Generator().manual_seed(1)).cuda() for s in shapes]
    vs = [torch.zeros(s, device="cuda") for s in shapes]
    gin = [m.clone() for m in mats]
    w2, v2 = [w.clone() for w in ws], [v.clone() for v in vs]
    graphs = []
    for _ in range(2):                        # two graphs, each with its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            hip.multi_muon(ws, gin, vs, 0.1)
        graphs.append(graph)
    for w, v, a, b in zip(ws, vs, w2, v2):
        w.copy_(a)
        v.copy_(b)
    for step in range(4):
        new = [_matrix(r, c, seed=step + 1).cuda() for r, c in shapes]
        for a, b in zip(gin, new):
            a.copy_(b)
        graphs[step % 2].replay()
        hip.multi_muon(w2, new, v2, 0.1)
        torch.cuda.synchronize()
        for a, b in zip(ws + vs, w2 + v2):
            assert torch.equal(a, b)
