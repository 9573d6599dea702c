"""How exact the Newton-Schulz kernels are, form by form, beside the same formula in plain fp32.

Yardstick. Both computations round their operands (fp32: 2^-24 of an element; pairs of fp16
numbers: 2^-23, and 2^-22 of a product left out) and carry these errors through the same
polynomials; their sums are fp32. The pairs lose up to four times as much on an operand in the worst
case, a third of that in the root mean square (three terms of random sign), and gain it back in
the sums, which hold at most 128 elements before they are emptied. So the kernels are held to twice
the fp32 form's relative error on the same input, and 16 steps of 2^-24 where that is tiny. A
product that is left without its small halves is off by 2^-11 of itself: a thousand times as much.

Rows (or columns) of very different size are compared row by row: a small row passes through the
products beside large ones and must keep its own digits. What is smaller than fp16's normal numbers
is absolute: an entry of X is off by at most 2^-50 and one of A or B by 2^-48 (X has norm one at the
start). The first is 2^-50 sqrt(n) on a row of n elements, taken again in every step while the row
grows 3.4-fold: 1.4 times that in all. The second meets rows of X of norm about one, m of them with
errors of random sign: 2^-48 sqrt(m). Both, relative to the row of X: ``floor``, under 2^-48
(sqrt(m) + sqrt(n)) over the smallest row's norm (300 x 1000, six decades: 7e-7; eight: 6e-5).

The thin form (up to 64 rows or columns) computes in 64 bits and rounds once: half a step of the
result, plus what the steps make of the 64-bit sums' rounding. A sum of 64 products of size one is
off by 10 * 2^-53. An error of the first A, between a direction that is nearly empty and one that is
not, grows by B on either side (3.4 and 1.3) in each of four steps, 400-fold; it is in the last B
nine-fold (|b| + 2 |c|) and meets a Q that has grown to 3.4445^4 = 141: 10 * 2^-53 * 400 * 9 * 141 =
6e-10 of a result of norm one, ``THIN`` = 2^-30."""
import numpy as np
import pytest
import torch

F32 = torch.float32
COEF = tuple(float(np.float32(c)) for c in (3.4445, -4.7750, 2.0315))
EPS = float(np.float32(1e-7))
THIN = 2.0 ** -30


def formula(g, dtype, steps=5):
    """The rule in ``dtype``; the norm, as everywhere, in 64 bits."""
    x = g.double()
    x = (x / (torch.linalg.norm(x) + EPS)).to(dtype)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    a, b, c = COEF
    for _ in range(steps):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return (x.t() if tall else x).double()


def whole(x, want):
    return (torch.linalg.norm(x.double() - want) / torch.linalg.norm(want)).item()


def by_lines(x, want, dim):
    """The worst row's (dim 1) or column's (dim 0) error, relative to itself."""
    off, size = (torch.linalg.norm(t, dim=dim) for t in (x.double() - want, want))
    return (off / size).max().item()


def bound(fp32_error):
    return 2.0 * fp32_error + 16 * 2.0 ** -24


def matrix(rows, cols, kind, seed=0, device="cpu"):
    gen = torch.Generator().manual_seed(seed * 1009 + rows * 17 + cols)

    def normal(*shape):
        return torch.randn(*shape, generator=gen)
    if kind == "gauss":
        g = normal(rows, cols)
    elif kind == "low_rank":
        rank = max(1, min(rows, cols) // 4)
        g = normal(rows, rank) @ normal(rank, cols) * 1e-3
    elif kind == "batch":                   # a dense layer's gradient over a batch of 64
        n = max(1, min(64, rows, cols))
        g = normal(n, rows).t() @ normal(n, cols) * (1e-2 / n) + 1e-4 * normal(rows, cols)
    elif kind.startswith("rows"):           # spread over so many decades
        g = normal(rows, cols) * 10.0 ** (-float(kind[4:]) * torch.rand(rows, 1, generator=gen))
    else:
        g = normal(rows, cols) * 10.0 ** (-float(kind[4:]) * torch.rand(1, cols, generator=gen))
    return g.to(device)


def floor(g, dim):
    x = g.double()
    x = x / torch.linalg.norm(x)
    smallest = torch.linalg.norm(x, dim=dim).min().item()
    return 2.0 ** -48 * (min(g.shape) ** 0.5 + g.shape[dim] ** 0.5) / smallest


# ---------------------------------------------------------------------------------------
# without a GPU: the scheme in torch, and what it is without one of its parts
# ---------------------------------------------------------------------------------------
X_SCALE, AB_SCALE, LO_SCALE = 2.0 ** 14, 2.0 ** 12, 2.0 ** 11


def scheme(g, steps=5, lo_scale=LO_SCALE, cross=(True, True), last=(True, True)):
    """The kernels' arithmetic with exact sums, rounded to fp32 behind every product. ``cross``:
    which of hi lo and lo hi are added (``last``: in the last product); ``lo_scale``: of the small
    halves."""
    def image(x, scale):
        s = x.double() * scale
        hi = s.to(torch.float16).double()
        return hi, ((s - hi) * lo_scale).to(torch.float16).double() / lo_scale

    def product(p, q, scale, terms=cross):
        r = p[0] @ q[0].t()
        if terms[0]:
            r = r + p[0] @ q[1].t()
        if terms[1]:
            r = r + p[1] @ q[0].t()
        return (r / scale).float().double()
    x = g.double()
    x = x / (torch.linalg.norm(x) + EPS)
    a, b, c = COEF
    for k in range(steps):
        xi, ti = image(x, X_SCALE), image(x.t(), X_SCALE)
        s = image(product(xi, xi, X_SCALE ** 2), AB_SCALE)
        poly = c * product(s, s, AB_SCALE ** 2) + b * (s[0] + s[1]) / AB_SCALE
        poly = poly + a * torch.eye(len(poly), dtype=torch.float64)
        x = product(image(poly.float(), AB_SCALE), ti, AB_SCALE * X_SCALE,
                    last if k + 1 == steps else cross)
    return x


@pytest.mark.parametrize("kind", ["gauss", "low_rank", "batch"])
def test_the_bound_notices_a_missing_half(kind):
    g = matrix(130, 300, kind)
    want = formula(g, torch.float64)
    limit = bound(whole(formula(g, F32), want))
    assert whole(scheme(g), want) <= limit
    for broken in (dict(cross=(True, False)), dict(cross=(False, True)), dict(last=(False, True)),
                   dict(last=(False, False)), dict(cross=(False, False))):
        assert whole(scheme(g, **broken), want) > 4 * limit, broken


@pytest.mark.parametrize("decades", [6, 8])
def test_the_bound_notices_small_halves_without_their_scale(decades):
    g = matrix(130, 300, "rows%d" % decades)
    want = formula(g, torch.float64)
    limit = bound(by_lines(formula(g, F32), want, 1)) + floor(g, 1)
    assert by_lines(scheme(g), want, 1) <= limit
    assert by_lines(scheme(g, lo_scale=1.0), want, 1) > 2 * limit


def test_the_thin_bound_notices_fp32():
    g = matrix(40, 70, "gauss")
    want = formula(g, torch.float64)
    off = (formula(g, F32) - want).abs()
    assert (off > 8 * (want.abs() * 2.0 ** -24 + THIN)).any()


# ---------------------------------------------------------------------------------------
# kernels
# ---------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def hip():
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    from distributed_tensorflow_amd.ops import hip as h
    h.lib()
    return h


# one list of shapes per form: up to 128 x 2048 (three and four K-tiles); 64 x 64 tiles; those in
# pairs of steps; K ranges that are shared; 256 x 128 tiles in single steps and in pairs
FORMS = {"mid96": [(96, 97), (70, 1500)], "mid128": [(784, 100), (128, 2048), (100, 784)],
         "small": [(1024, 1024), (257, 300)], "pairs": [(515, 1030), (1030, 515)],
         "shared": [(300, 8000)], "wide": [(2048, 2049), (2001, 1999), (2000, 2050)],
         "wide_pairs": [(1999, 5000), (5001, 1987)]}


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["gauss", "low_rank", "batch"])
@pytest.mark.parametrize("form", sorted(FORMS))
def test_errors_beside_plain_fp32(hip, form, kind):
    mats = [matrix(r, c, kind, i, "cuda") for i, (r, c) in enumerate(FORMS[form])]
    for g, got in zip(mats, hip.newton_schulz(mats)):
        want = formula(g, torch.float64)
        limit = bound(whole(formula(g, F32), want))
        assert whole(got, want) <= limit, (tuple(g.shape), whole(got, want), limit)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["rows4", "rows6", "rows8", "cols6", "cols8"])
@pytest.mark.parametrize("form", sorted(FORMS))
def test_rows_and_columns_of_different_size(hip, form, kind):
    """Each keeps its own digits, as it does in fp32."""
    mats = [matrix(r, c, kind, i, "cuda") for i, (r, c) in enumerate(FORMS[form])]
    dim = 1 if kind.startswith("rows") else 0
    for g, got in zip(mats, hip.newton_schulz(mats)):
        want = formula(g, torch.float64)
        limit = bound(by_lines(formula(g, F32), want, dim)) + floor(g, dim)
        assert by_lines(got, want, dim) <= limit, (tuple(g.shape), by_lines(got, want, dim), limit)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["gauss", "low_rank", "batch", "rows8", "cols8"])
@pytest.mark.parametrize("rows,cols", [(1, 9), (40, 70), (64, 64), (64, 256), (63, 2000), (5000, 17)])
def test_thin_results_are_rounded_once(hip, rows, cols, kind):
    g = matrix(rows, cols, kind, device="cuda")
    want = formula(g, torch.float64)
    off = (hip.newton_schulz(g).double() - want).abs()
    limit = want.abs() * 2.0 ** -24 + THIN
    assert (off <= limit).all(), (off / limit).max().item()
