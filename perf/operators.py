"""Layer normalisation and the orthogonalised update, measured: cases, inputs, plain forms and 64-bit values.

Four kinds of pass (`case["op"]`):

  norm         y = layer_norm(x, w, b)                       the forward pass alone (encoding, serving)
  norm_train   y and the gradients dx, dw, db for a given dy (a training step's two passes); with "block" the
               normalisation of u = keep * keep_scale * leaky_relu(x): what follows a linear layer in a block
  orthogonal   O = orthogonalize(G): steps of X <- a X + (b A + c A^2) X with A = X X^T, from X = G / |G|_F
  muon         muon_step(params, grads, momenta): momentum, orthogonalisation and update of a list of weights

With `own` false `run` computes them from elementary torch operations in 32 bits, rounded once; with `own`
true it makes the calls of lrbinner_amd.train_ops."""
import functools
import math

import torch

own = False

EPS = 1e-5                             # layer norm
COEFFS = (3.4445, -4.7750, 2.0315)     # of the odd quintic that the orthogonalisation iterates
NORM_EPS = 1e-7                        # least Frobenius norm that a matrix is divided by
STEPS = 5
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
SLOPE, DROP = 0.01, 0.1                # LeakyReLU and dropout of this repository's blocks
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
#: the weights of this repository's default network (composition width 136, 32 coverage bins, hidden layers
#: 128 and 128, 8 latent dimensions), one a "RxC"
NETWORK = "128x168,128x128,8x128,8x128,128x8,128x128,168x128"


def listed():
    return [
        # one sample through one hidden layer of the default network: latency
        {"name": "norm 1x128 f32", "op": "norm", "rows": 1, "cols": 128, "type": "f32", "wtype": "f32"},
        # a chunk of the samples that are encoded together, 2^18 rows of the hidden width
        {"name": "norm 262144x128 f32", "op": "norm", "rows": 262144, "cols": 128, "type": "f32", "wtype": "f32"},
        # a packed batch of tokens in 16 bits, no size a multiple of anything
        {"name": "norm 8191x4095 bf16", "op": "norm", "rows": 8191, "cols": 4095, "type": "bf16", "wtype": "f32"},
        # one block of the default network in training, at its first batch size
        {"name": "block train 1024x128 f32", "op": "norm_train", "rows": 1024, "cols": 128, "type": "f32", "wtype": "f32", "block": True},
        # a training batch of a wide model in 16 bits with weights in 16 bits
        {"name": "train 32768x4096 bf16", "op": "norm_train", "rows": 32768, "cols": 4096, "type": "bf16", "wtype": "bf16", "block": False},
        # few long rows of an odd length
        {"name": "train 1000x10007 f16", "op": "norm_train", "rows": 1000, "cols": 10007, "type": "f16", "wtype": "f32", "block": False},
        # the widest weight of the default network
        {"name": "orthogonal 128x168 f32", "op": "orthogonal", "count": 1, "rows": 128, "cols": 168, "type": "f32"},
        # a tall weight of odd sizes
        {"name": "orthogonal 1025x511 f32", "op": "orthogonal", "count": 1, "rows": 1025, "cols": 511, "type": "f32"},
        # a stack of heads' or experts' weights in 16 bits
        {"name": "orthogonal 8x1024x2048 bf16", "op": "orthogonal", "count": 8, "rows": 1024, "cols": 2048, "type": "bf16"},
        # a step on all weights of the default network
        {"name": "muon network f32", "op": "muon", "shapes": NETWORK, "type": "f32"},
        # a step on the weights of one layer of a mid-sized model in 16 bits
        {"name": "muon layer bf16", "op": "muon", "shapes": "2048x2048,2048x2048,5461x2048,2048x5461", "type": "bf16"},
        # the largest single weight
        {"name": "muon 4096x4096 f32", "op": "muon", "shapes": "4096x4096", "type": "f32"},
    ]


MOST_VALUES = 32768 * 4096             # of a drawn normalisation
MOST_FLOPS = 1.0e12                    # of a drawn orthogonalisation


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _shape(rng, most):
    while True:
        r, c = _log(rng, 1, 6000), _log(rng, 1, 6000)
        if _products(r, c, STEPS) <= most:
            return r, c


def draw(rng):
    op = rng.choice(["norm", "norm_train", "orthogonal", "muon"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op in ("norm", "norm_train"):
        cols = _log(rng, 1, 16384)
        case = {"op": op, "rows": _log(rng, 1, max(1, min(1 << 18, MOST_VALUES // cols))), "cols": cols, "type": kind,
                "wtype": rng.choice(["f32", kind])}
        if op == "norm_train":
            case["block"] = rng.random() < 0.4
        return case
    if op == "orthogonal":
        count = _log(rng, 1, 16)
        r, c = _shape(rng, MOST_FLOPS / count)
        return {"op": op, "count": count, "rows": r, "cols": c, "type": kind}
    n = rng.randint(1, 6)
    return {"op": op, "shapes": ",".join("%dx%d" % _shape(rng, MOST_FLOPS / n) for _ in range(n)), "type": kind}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


# ---- inputs -----------------------------------------------------------------------------------

def _gradient(rows, cols, gen, count=()):
    """A weight's gradient as a batch leaves it: a sum of outer products whose strengths fall off over
    e^4, and a floor of noise."""
    r = max(1, min(rows, cols) // 2)
    fall = torch.exp(torch.linspace(0.0, -4.0, r, device="cuda"))
    d = torch.randn(*count, rows, r, device="cuda", generator=gen) * fall
    x = torch.randn(*count, r, cols, device="cuda", generator=gen)
    return torch.matmul(d, x) / r + 1e-3 * torch.randn(*count, rows, cols, device="cuda", generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["type"]]
    s = {"case": case}
    if case["op"] in ("norm", "norm_train"):
        n, d, wt = case["rows"], case["cols"], DTYPES[case["wtype"]]

        def rand(*shape):
            return torch.randn(*shape, device="cuda", generator=gen)

        # columns of unlike spread, rows off zero, as activations are
        s["x"] = (rand(n, d).mul_(0.5 + rand(d).abs_()).add_(0.5 * rand(n, 1))).to(t)
        s["w"] = (1 + 0.2 * rand(d)).to(wt)
        s["b"] = (0.2 * rand(d)).to(wt)
        if case["op"] == "norm_train":
            s["dy"] = rand(n, d).to(t)
            if case["block"]:
                s["keep"] = torch.rand(n, d, device="cuda", generator=gen) >= DROP
            for v in ("x", "w", "b"):
                s[v].requires_grad_()
    elif case["op"] == "orthogonal":
        s["g"] = _gradient(case["rows"], case["cols"], gen, (case["count"],) if case["count"] > 1 else ()).to(t)
    else:
        s["params"], s["grads"], s["momenta"] = [], [], []
        for r, c in _shapes(case):
            s["params"].append((torch.randn(r, c, device="cuda", generator=gen) / math.sqrt(c)).to(t))
            s["grads"].append(_gradient(r, c, gen).to(t))
            s["momenta"].append(_gradient(r, c, gen))    # held in 32 bits
    return s


# ---- the plain forms --------------------------------------------------------------------------

def _norm(u, w, b):
    """(y, the normalised rows, 1 / deviation), all in 32 bits."""
    centred = u - u.mean(-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    hat = centred * rstd
    return hat * w + b, hat, rstd


@torch.no_grad()
def _norm_train(s, block):
    x, dy, w, b = s["x"].float(), s["dy"].float(), s["w"].float(), s["b"].float()
    if block:
        slope = torch.where(x > 0, 1.0, SLOPE) * (s["keep"].float() * (1.0 / (1.0 - DROP)))
        y, hat, rstd = _norm(x * slope, w, b)
    else:
        y, hat, rstd = _norm(x, w, b)
    g = dy * w
    dx = (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True)) * rstd
    if block:
        dx = dx * slope
    return {"y": y.to(s["x"].dtype), "dx": dx.to(s["x"].dtype), "dw": (dy * hat).sum(0).to(s["w"].dtype), "db": dy.sum(0).to(s["b"].dtype)}


def _iterate(x, _):
    a, b, c = COEFFS
    gram = torch.matmul(x, x.transpose(-1, -2).contiguous())
    return a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)


def _orthogonal(g):
    x = g.transpose(-1, -2).contiguous() if g.shape[-2] > g.shape[-1] else g
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp_min(NORM_EPS)
    x = functools.reduce(_iterate, range(STEPS), x)
    return x.transpose(-1, -2) if g.shape[-2] > g.shape[-1] else x


def _muon(p, g, m, orthogonal=_orthogonal):
    """p and m after a step, in the type of m."""
    g = g.to(m.dtype)
    m = MOMENTUM * m + (1 - MOMENTUM) * g
    o = orthogonal((1 - MOMENTUM) * g + MOMENTUM * m)
    return p.to(m.dtype) * (1 - LR * DECAY) - LR * math.sqrt(max(1.0, p.shape[0] / p.shape[1])) * o, m


def _muon_in_place(p, g, m):
    new, momentum = _muon(p, g, m)
    m.copy_(momentum)
    p.copy_(new)


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from lrbinner_amd import train_ops
    if op == "norm":
        if own:
            return train_ops.layer_norm(state["x"], state["w"], state["b"], EPS)
        return _norm(state["x"].float(), state["w"].float(), state["b"].float())[0].to(state["x"].dtype)
    if op == "norm_train":
        if own:
            more = {"slope": SLOPE, "keep": state["keep"], "keep_scale": 1.0 / (1.0 - DROP)} if case["block"] else {}
            leaves = (state["x"], state["w"], state["b"])
            y = train_ops.layer_norm(*leaves, EPS, **more)
            dx, dw, db = torch.autograd.grad(y, leaves, state["dy"])
            return {"y": y, "dx": dx, "dw": dw, "db": db}
        return _norm_train(state, case["block"])
    if op == "orthogonal":
        if own:
            return train_ops.orthogonalize(state["g"], steps=STEPS, coefficients=COEFFS, eps=NORM_EPS)
        return _orthogonal(state["g"].float()).to(state["g"].dtype)
    if own:
        train_ops.muon_step(state["params"], state["grads"], state["momenta"], lr=LR, momentum=MOMENTUM, nesterov=True,
                            weight_decay=DECAY, steps=STEPS, coefficients=COEFFS, eps=NORM_EPS)
    else:
        [_muon_in_place(*t) for t in zip(state["params"], state["grads"], state["momenta"])]
    return {"params": state["params"], "momenta": state["momenta"]}


# ---- what a pass cannot do without --------------------------------------------------------------

def _products(rows, cols, steps):
    """Multiplications and additions of the steps' three products; of the two symmetric ones, half."""
    n, m = min(rows, cols), max(rows, cols)
    return steps * float(n * n * m + n * n * n + 2 * n * n * m)


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    t = size[case["type"]]
    if case["op"] in ("norm", "norm_train"):
        n, d, w = case["rows"], case["cols"], size[case["wtype"]]
        if case["op"] == "norm":
            return {"bytes": 2 * n * d * t + 2 * d * w, "flops": 8 * n * d}
        return {"bytes": n * d * (4 * t + (1 if case["block"] else 0)) + 3 * d * w, "flops": 22 * n * d}
    if case["op"] == "orthogonal":
        n, r, c = case["count"], case["rows"], case["cols"]
        return {"bytes": 2 * n * r * c * t, "flops": n * _products(r, c, STEPS)}
    return {"bytes": sum(r * c * (3 * t + 8) for r, c in _shapes(case)), "flops": sum(_products(r, c, STEPS) for r, c in _shapes(case))}


# ---- the definition in 64 bits ------------------------------------------------------------------

def _exact_norm(s, case):
    x = s["x"].detach().double()
    factor = torch.ones_like(x)
    if case.get("block"):
        factor[x <= 0] = SLOPE
        factor *= s["keep"].double() / (1.0 - DROP)
    u = (x * factor).requires_grad_()
    w, b = s["w"].detach().double().requires_grad_(), s["b"].detach().double().requires_grad_()
    var, mean = torch.var_mean(u, dim=1, unbiased=False, keepdim=True)
    y = (u - mean) / torch.sqrt(var + EPS) * w + b
    if case["op"] == "norm":
        return y.detach()
    du, dw, db = torch.autograd.grad(y, (u, w, b), s["dy"].double())
    return {"y": y.detach(), "dx": du * factor, "dw": dw, "db": db}


def _exact_orthogonal(g):
    """By the singular values where that is quick (the quintic acts on them alone), by products in 64 bits else."""
    a, b, c = COEFFS
    g = g.double()
    norm = torch.linalg.vector_norm(g, dim=(-2, -1), keepdim=True).clamp_min(NORM_EPS)
    if g.shape[-1] * g.shape[-2] <= 256 * 256 and g.dim() == 2:
        u, sv, vt = torch.linalg.svd((g / norm).cpu(), full_matrices=False)
        for _ in range(STEPS):
            sv = sv * (a + sv * sv * (b + c * sv * sv))
        return ((u * sv) @ vt).to(g.device)
    x = g / norm
    for _ in range(STEPS):
        if x.shape[-2] <= x.shape[-1]:
            gram = x @ x.mT
            x = a * x + (b * gram @ x + c * gram @ (gram @ x))
        else:
            gram = x.mT @ x
            x = a * x + (b * x @ gram + c * (x @ gram) @ gram)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "norm_train"):
        return _exact_norm(s, case)
    if case["op"] == "orthogonal":
        return _exact_orthogonal(s["g"])
    steps = [_muon(p, g, m.double(), _exact_orthogonal) for p, g, m in zip(s["params"], s["grads"], s["momenta"])]
    return {"params": [p for p, _ in steps], "momenta": [m for _, m in steps]}
