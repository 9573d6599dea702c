"""What the operators for training stacks of dense layers are measured on: layer normalisation
(forward, backward), the orthogonalisation of a matrix by Newton-Schulz products, and the update
of a model's matrices by the Muon rule, each in plain elementary torch operations (``own`` false)
and as a user calls the framework's kernels (``own`` true).

Layer normalisation of the rows of x [rows, cols], every row on its own:

    mean = sum(x) / cols;  rstd = 1 / sqrt(sum((x - mean)^2) / cols + epsilon)
    y    = (x - mean) rstd gamma + beta

and its gradient for dy, from the stored mean and rstd, with h = (x - mean) rstd, g = dy gamma:

    dx = rstd (g - sum(g) / cols - h sum(g h) / cols);  dgamma = sum_rows(dy h);  dbeta = sum_rows(dy)

Orthogonalisation of G with rows <= cols (of its transpose otherwise):

    X = G / (|G|_F + epsilon);   ``steps`` times:  A = X X^T;  X = a X + (b A + c A A) X

The Muon update of a weight W [inputs, outputs] with momentum V:

    V = mu V + G;  W = (1 - lr decay) W - lr sqrt(max(1, outputs / inputs)) orthogonalise(G + mu V)
"""
import math

import torch

own = False

EPSILON = 1e-5            # of the layer norm
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NORM_EPSILON = 1e-7       # of the orthogonalisation
STEPS = 5
MOMENTUM, LEARNING_RATE, DECAY = 0.95, 0.02, 0.01

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------
def listed():
    return [
        # the hidden layer of the MNIST classifier at its batch of 100: latency is all there is
        {"name": "norm_hidden_100", "op": "norm", "rows": 100, "cols": 100, "dtype": "float32",
         "params": "float32"},
        # off the grid: odd row count, odd width
        {"name": "norm_odd", "op": "norm", "rows": 2053, "cols": 1537, "dtype": "float32",
         "params": "float32"},
        # a large batch of wide rows in 16 bits, parameters kept in 32
        {"name": "norm_wide", "op": "norm", "rows": 16384, "cols": 4096, "dtype": "bfloat16",
         "params": "float32"},
        # the gradients of the same layers
        {"name": "norm_grad_hidden_100", "op": "norm_grad", "rows": 100, "cols": 100,
         "dtype": "float32", "params": "float32"},
        {"name": "norm_grad_images", "op": "norm_grad", "rows": 10000, "cols": 784,
         "dtype": "float32", "params": "float32"},
        {"name": "norm_grad_wide", "op": "norm_grad", "rows": 16384, "cols": 4096,
         "dtype": "bfloat16", "params": "float32"},
        # the gradient of one hidden layer's matrix
        {"name": "orthogonalise_1024", "op": "orthogonalise", "batch": 1, "rows": 1024,
         "cols": 1024, "dtype": "float32"},
        # a stack of equal layers off the grid, gradients in 16 bits
        {"name": "orthogonalise_stack", "op": "orthogonalise", "batch": 3, "rows": 515,
         "cols": 1030, "dtype": "bfloat16"},
        # a large tall matrix
        {"name": "orthogonalise_large", "op": "orthogonalise", "batch": 1, "rows": 8192,
         "cols": 4096, "dtype": "float32"},
        # the two weights of the MNIST classifier
        {"name": "muon_classifier", "op": "muon", "shapes": "784x100,100x10"},
        # a classifier with three hidden layers
        {"name": "muon_hidden", "op": "muon", "shapes": "784x1024,1024x1024,1024x1024,1024x1000"},
        # square, wide and tall weights of a large model's blocks
        {"name": "muon_blocks", "op": "muon",
         "shapes": "2048x2048,2048x2048,2048x8192,8192x2048"},
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "orthogonalise", "muon"])
    if op in ("norm", "norm_grad"):
        cols = _log_uniform(rng, 1, 16384)
        rows = _log_uniform(rng, 1, min(65536, 16384 * 4096 // cols))
        dtype = rng.choice(["float32", "bfloat16", "float16"])
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype,
                "params": rng.choice(["float32", dtype])}
    if op == "orthogonalise":
        batch = rng.choice([1, 1, 2, 5])
        rows, cols = _log_uniform(rng, 1, 8192), _log_uniform(rng, 1, 8192)
        while batch * _orthogonalise_flops(rows, cols) > _orthogonalise_flops(8192, 4096):
            rows, cols = rows * 4 // 5, cols * 5 // 6
        return {"op": op, "batch": batch, "rows": rows, "cols": cols,
                "dtype": rng.choice(["float32", "bfloat16", "float16"])}
    shapes = ["%dx%d" % (_log_uniform(rng, 1, 2500), _log_uniform(rng, 1, 2500))
              for _ in range(rng.randint(1, 6))]
    return {"op": op, "shapes": ",".join(shapes)}


def _shapes(case):
    return [tuple(int(d) for d in s.split("x")) for s in case["shapes"].split(",")]


# ---------------------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------------------
def _gradient(rows, cols, gen):
    """The gradient of a dense layer's matrix: activations^T times deltas over a batch, so its
    rank is bounded by the batch and its singular values are far apart."""
    batch = max(1, min(128, rows, cols))
    x = torch.randn(batch, rows, device="cuda", generator=gen)
    d = torch.randn(batch, cols, device="cuda", generator=gen) * (1e-2 / batch)
    return x.t() @ d + 1e-4 * torch.randn(rows, cols, device="cuda", generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)
    op = case["op"]
    state = dict(case)
    if op in ("norm", "norm_grad"):
        rows, cols = case["rows"], case["cols"]
        x_t, p_t = DTYPES[case["dtype"]], DTYPES[case["params"]]
        # rows of their own size and offset, as they come out of a dense layer
        x = normal(rows, cols) * torch.exp(0.5 * normal(rows, 1)) + 0.5 * normal(rows, 1)
        state["x"] = x.to(x_t)
        state["gamma"] = (1.0 + 0.2 * normal(cols)).to(p_t)
        if op == "norm":
            state["beta"] = (0.2 * normal(cols)).to(p_t)
        else:
            state["dy"] = (0.1 * normal(rows, cols)).to(x_t)
            wide = state["x"].double()
            mean = wide.mean(dim=1)
            var = (wide - mean.unsqueeze(1)).square().mean(dim=1)
            state["mean"] = mean.float()
            state["rstd"] = (1.0 / torch.sqrt(var + EPSILON)).float()
    elif op == "orthogonalise":
        gs = [_gradient(case["rows"], case["cols"], gen) for _ in range(case["batch"])]
        g = gs[0] if case["batch"] == 1 else torch.stack(gs)
        state["g"] = g.to(DTYPES[case["dtype"]])
    else:
        shapes = _shapes(case)
        # one buffer holds all weights and momenta, as the training runtime keeps them
        sizes = [r * c for r, c in shapes]
        state["shapes"] = shapes
        state["sizes"] = [(n + 63) // 64 * 64 for n in sizes]
        flat = torch.zeros(2 * sum(state["sizes"]), device="cuda")
        params, moments = _views(flat, shapes, state["sizes"])
        for (r, c), p, m in zip(shapes, params, moments):
            p.copy_(normal(r, c) / math.sqrt(r))
            m.copy_(4.0 * _gradient(r, c, gen))
        state["flat"] = flat
        state["grads"] = [_gradient(r, c, gen) for r, c in shapes]
    return state


def _views(flat, shapes, sizes):
    """The weights and the momenta that lie in ``flat``."""
    views, at = [], 0
    for (r, c), n in list(zip(shapes, sizes)) * 2:
        views.append(flat[at:at + r * c].view(r, c))
        at += n
    return views[:len(shapes)], views[len(shapes):]


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def _plain_orthogonalise(g):
    a, b, c = COEFFICIENTS
    x = g.float()
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t()
    x = x / (torch.sqrt((x * x).sum()) + NORM_EPSILON)
    for _ in range(STEPS):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t().contiguous() if tall else x


def _plain(state):
    op = state["op"]
    if op == "norm":
        x = state["x"].float()
        mean = x.mean(dim=1, keepdim=True)
        d = x - mean
        rstd = 1.0 / torch.sqrt((d * d).mean(dim=1, keepdim=True) + EPSILON)
        y = d * rstd * state["gamma"].float() + state["beta"].float()
        return [y.to(state["x"].dtype), mean.squeeze(1), rstd.squeeze(1)]
    if op == "norm_grad":
        x, dy, gamma = state["x"].float(), state["dy"].float(), state["gamma"].float()
        rstd = state["rstd"].unsqueeze(1)
        h = (x - state["mean"].unsqueeze(1)) * rstd
        g = dy * gamma
        dx = rstd * (g - g.mean(dim=1, keepdim=True) - h * (g * h).mean(dim=1, keepdim=True))
        p_t = state["gamma"].dtype
        return [dx.to(state["x"].dtype), (dy * h).sum(dim=0).to(p_t), dy.sum(dim=0).to(p_t)]
    if op == "orthogonalise":
        g = state["g"]
        if g.dim() == 2:
            return _plain_orthogonalise(g).to(g.dtype)
        return torch.stack([_plain_orthogonalise(m) for m in g]).to(g.dtype)
    params, moments = _views(state["flat"], state["shapes"], state["sizes"])
    new_p, new_m = [], []
    for p, m, g in zip(params, moments, state["grads"]):
        m = MOMENTUM * m + g
        o = _plain_orthogonalise(g + MOMENTUM * m)
        scale = math.sqrt(max(1.0, p.shape[1] / p.shape[0]))
        new_p.append((1.0 - LEARNING_RATE * DECAY) * p - (LEARNING_RATE * scale) * o)
        new_m.append(m)
    return new_p + new_m


def run(state):
    if not own:
        return _plain(state)
    from distributed_tensorflow_amd.ops import hip
    op = state["op"]
    if op == "norm":
        return list(hip.layer_norm(state["x"], state["gamma"], state["beta"], epsilon=EPSILON,
                                   want_stats=True))
    if op == "norm_grad":
        return list(hip.layer_norm_grad(state["dy"], state["x"], state["mean"], state["rstd"],
                                        state["gamma"]))
    if op == "orthogonalise":
        return hip.newton_schulz(state["g"], steps=STEPS, coefficients=COEFFICIENTS,
                                 epsilon=NORM_EPSILON)
    flat = state["flat"].clone()          # the update is in place: each pass updates a copy
    params, moments = _views(flat, state["shapes"], state["sizes"])
    hip.multi_muon(params, state["grads"], moments, LEARNING_RATE, momentum=MOMENTUM,
                   nesterov=True, weight_decay=DECAY, steps=STEPS, coefficients=COEFFICIENTS,
                   epsilon=NORM_EPSILON)
    return params + moments


# ---------------------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------------------
def _exact_orthogonalise(g):
    a, b, c = COEFFICIENTS
    g = g.double()
    # row side or column side: the polynomial is applied on the shorter one
    x = g / (g.norm() + NORM_EPSILON)
    eye = torch.eye(min(g.shape), dtype=torch.float64, device=g.device)
    for _ in range(STEPS):
        if g.shape[0] <= g.shape[1]:
            s = x @ x.t()
            x = (a * eye + s @ (b * eye + c * s)) @ x
        else:
            s = x.t() @ x
            x = x @ (a * eye + s @ (b * eye + c * s))
    return x


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        x = state["x"].double()
        var, mean = torch.var_mean(x, dim=1, unbiased=False)
        rstd = (var + EPSILON).rsqrt()
        h = (x - mean[:, None]) * rstd[:, None]
        return [state["beta"].double() + h * state["gamma"].double(), mean, rstd]
    if op == "norm_grad":
        n = case["cols"]
        dy, r = state["dy"].double(), state["rstd"].double()[:, None]
        h = (state["x"].double() - state["mean"].double()[:, None]) * r
        g = dy * state["gamma"].double()
        dx = (r / n) * (n * g - g.sum(1, keepdim=True) - h * (g * h).sum(1, keepdim=True))
        return [dx, (dy * h).sum(0), dy.sum(0)]
    if op == "orthogonalise":
        g = state["g"]
        if g.dim() == 2:
            return _exact_orthogonalise(g)
        return torch.stack([_exact_orthogonalise(m) for m in g])
    params, moments = _views(state["flat"].double(), state["shapes"], state["sizes"])
    new_p, new_m = [], []
    for p, m, g in zip(params, moments, state["grads"]):
        g = g.double()
        v = MOMENTUM * m + g
        o = _exact_orthogonalise(g + MOMENTUM * v)
        step = LEARNING_RATE * max(1.0, p.shape[1] / p.shape[0]) ** 0.5
        new_p.append(p - LEARNING_RATE * DECAY * p - step * o)
        new_m.append(v)
    return new_p + new_m


# ---------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------
def _orthogonalise_flops(rows, cols):
    """Both symmetric products count half: X X^T and A A have one triangle to compute."""
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (m * m * n + m * m * m + 2 * m * m * n)


def work(case):
    op = case["op"]
    size = {"float32": 4, "bfloat16": 2, "float16": 2}
    if op in ("norm", "norm_grad"):
        rows, cols = case["rows"], case["cols"]
        e, p = size[case["dtype"]], size[case["params"]]
        if op == "norm":
            return {"bytes": rows * cols * 2 * e + 2 * cols * p + 8 * rows,
                    "flops": 8 * rows * cols}
        return {"bytes": rows * cols * 3 * e + 3 * cols * p + 8 * rows, "flops": 14 * rows * cols}
    if op == "orthogonalise":
        n = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": 2 * n * size[case["dtype"]],
                "flops": case["batch"] * _orthogonalise_flops(case["rows"], case["cols"])}
    shapes = _shapes(case)
    return {"bytes": 4 * 5 * sum(r * c for r, c in shapes),
            "flops": sum(_orthogonalise_flops(r, c) + 7 * r * c for r, c in shapes)}
