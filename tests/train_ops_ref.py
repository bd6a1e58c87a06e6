"""Plain 64-bit forms of lrbinner_amd.train_ops and the tolerances that its float32 arithmetic is held to."""
import math

import torch

# a rounding to nearest is off by at most half a step
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
U = 2.0 ** -24


def norm_ref(x, w, b, eps, dy=None, slope=1.0, keep=None, keep_scale=1.0):
    """(y, dx, dw, db) in float64 by the formulas, and the tolerance of each.

    Tolerances: a sum of float32 over a row is made of at most 16 + cols / 1024 sequential additions in a thread and 26 in
    the trees over threads and waves, so it is off by at most gamma = (48 + cols / 1024) U of the sum of the magnitudes; a
    sum over rows has at most rows / 64 + 64 (fewest workgroups: 64).  Every other operation is off by U of its result.
    First order throughout, with 10 % for the second."""
    cols = x.shape[-1]
    x2, dy2 = x.detach().double().reshape(-1, cols), None if dy is None else dy.double().reshape(-1, cols)
    f = torch.ones_like(x2)
    if slope != 1.0 or keep is not None:
        f = torch.where(x2 > 0, 1.0, slope).double()
        if keep is not None:
            kept = keep.reshape(-1, cols).bool()
            f = torch.where(kept, f * keep_scale, torch.zeros_like(f))
            x2 = torch.where(kept, x2, torch.zeros_like(x2))
    u = x2 * f
    mean = u.mean(1, keepdim=True)
    var = (u - mean).square().mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    hat = (u - mean) * rstd
    wd = torch.ones(cols, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    bd = torch.zeros(cols, dtype=torch.float64, device=x.device) if b is None else b.detach().double()
    y = hat * wd + bd
    gamma = (48 + cols / 1024) * U
    d_mean = gamma * u.abs().mean(1, keepdim=True) + U * mean.abs()
    # the variance also takes in the error of the mean it is made with, squared
    d_rstd = rstd * (0.5 * gamma + 4 * U) + 0.5 * rstd ** 3 * d_mean ** 2
    d_hat = rstd * (d_mean + 3 * U * u.abs()) + (u - mean).abs() * d_rstd + 2 * U * hat.abs()
    step = HALF_STEP[x.dtype]
    tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps  # the smallest number of the type
    tol_y = 1.1 * (wd.abs() * d_hat + 3 * U * (hat * wd).abs() + U * y.abs()) + 1.1 * step * y.abs() + tiny
    if dy is None:
        return (y.reshape(x.shape),), (tol_y.reshape(x.shape),)
    g = dy2 * wd
    m1, m2 = g.mean(1, keepdim=True), (g * hat).mean(1, keepdim=True)
    du = (g - m1 - hat * m2) * rstd
    dx = du * f
    d_m1 = (gamma + 2 * U) * g.abs().mean(1, keepdim=True)
    d_m2 = (gamma + 3 * U) * (g * hat).abs().mean(1, keepdim=True) + (g.abs() * d_hat).mean(1, keepdim=True)
    d_in = 3 * U * (g.abs() + m1.abs() + (hat * m2).abs()) + d_m1 + d_hat * m2.abs() + hat.abs() * d_m2
    tol_dx = 1.1 * f.abs() * (rstd * d_in + du.abs() * (d_rstd / rstd + 3 * U)) + 1.1 * step * dx.abs() + tiny
    rows_g = (u.shape[0] / 64 + 64) * U
    wt = w.dtype if w is not None else b.dtype if b is not None else torch.float32
    dw, db = (dy2 * hat).sum(0), dy2.sum(0)
    tol_dw = 1.1 * (rows_g * (dy2 * hat).abs().sum(0) + (dy2.abs() * d_hat).sum(0)) + 1.1 * HALF_STEP[wt] * dw.abs() + tiny
    tol_db = 1.1 * rows_g * dy2.abs().sum(0) + 1.1 * HALF_STEP[wt] * db.abs() + tiny
    return (y.reshape(x.shape), dx.reshape(x.shape), dw, db), (tol_y.reshape(x.shape), tol_dx.reshape(x.shape), tol_dw, tol_db)


def orthogonal_ref(g, steps, coefficients, eps, dtype=torch.float64):
    """The iteration in `dtype`, from a norm in float64."""
    a, b, c = coefficients
    x = g.to(dtype)
    turned = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2).contiguous() if turned else x
    norm = torch.sqrt(g.double().square().sum((-2, -1), keepdim=True)).clamp_min(eps)
    x = (x.double() / norm).to(dtype)
    for _ in range(steps):
        xt = x.transpose(-1, -2).contiguous()
        gram = torch.matmul(x, xt)
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.transpose(-1, -2) if turned else x


def orthogonal_tolerance(exact, g, steps, coefficients, eps):
    """Frobenius norm that the kernel's float32 result may be off by, for each matrix.

    The kernel's factors are off by 2^-23 of their entries (float32: 2^-24), its sums are float32 sums: what float32
    products are off by on the same matrix, twice, and once more for another order of the sums; and 2^-20 for where that
    happens to be exact.

    With few entries the float32 run may be exact by chance (of 5000 matrices of 2 x 3, several hundred), so for a short side
    up to 16 the matrix's sensitivity is counted too.  The iteration is g = U S V^T -> U F(S) V^T with F the composed odd
    polynomial, whose derivative at g has the operator norm D = max |F(s) -+ F(t)| / |s -+ t| over pairs of singular values
    (F' where they coincide).  A step rounds three factors, each by at most 2 U of its entries; the first X is g itself, and what
    is rounded further on is passed on by fewer steps.  3 `steps` independent roundings of 2 U add up to 2 U sqrt(3 steps)."""
    off = orthogonal_ref(g, steps, coefficients, eps, torch.float32).double() - exact
    tol = 3 * torch.linalg.vector_norm(off, dim=(-2, -1)) + 2.0 ** -20 * torch.linalg.vector_norm(exact, dim=(-2, -1))
    if min(g.shape[-2:]) > 16:
        return tol
    norm = torch.sqrt(g.double().square().sum((-2, -1)))
    x0 = norm / norm.clamp_min(eps)
    s = torch.linalg.svdvals(g.double().cpu()).to(g.device) / norm.clamp_min(eps).unsqueeze(-1)
    f, d = s, torch.ones_like(s)
    a, b, c = coefficients
    for _ in range(steps):
        d = d * (a + 3 * b * f ** 2 + 5 * c * f ** 4)
        f = f * (a + b * f ** 2 + c * f ** 4)
    lean = lambda v: (v.unsqueeze(-1) - v.unsqueeze(-2)).abs(), lambda v: (v.unsqueeze(-1) + v.unsqueeze(-2)).abs()
    most = d.abs().amax(-1)
    for pair in lean:
        q = pair(f) / pair(s)
        most = torch.maximum(most, torch.where(torch.isfinite(q), q, torch.zeros_like(q)).amax((-2, -1)))
    return tol + 2 * math.sqrt(3 * steps) * U * x0 * most


def gradient_like(rows, cols, gen, device="cpu", count=()):
    """A sum of outer products whose strengths fall off over e^4, and a floor of noise."""
    r = max(1, min(rows, cols) // 2)
    fall = torch.exp(torch.linspace(0.0, -4.0, r))
    d = torch.randn(*count, rows, r, generator=gen) * fall
    x = torch.randn(*count, r, cols, generator=gen)
    return (torch.matmul(d, x) / r + 1e-3 * torch.randn(*count, rows, cols, generator=gen)).to(device)


def within(got, want, tol, what=""):
    off = (got.double() - want.double()).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, by up to {float((off / tol).max()):.3g} times the tolerance"


def matrices_within(got, want, tol, half_step=0.0, what=""):
    """Every matrix of a stack within its Frobenius tolerance (and half a step of a 16-bit result's entries)."""
    off = torch.linalg.vector_norm(got.double() - want, dim=(-2, -1))
    most = tol + 1.1 * half_step * torch.linalg.vector_norm(want, dim=(-2, -1)) + math.sqrt(want.shape[-1] * want.shape[-2]) * 6e-8 * (half_step > 2.0 ** -20)
    assert bool((off <= most).all()), f"{what}: off by {float((off / most).max()):.3g} times the tolerance"


def far_row_tolerance(x, w, eps):
    """Of y for float32 rows whose mean may lie far above their deviation, up to 20,001 columns.

    The mean of the first pass is off by at most gamma |u| on average (48 + cols / 1024 roundings, as above), which every
    difference from it carries.  The mean of these differences, gamma of their own size off, is added, and the mean rounded: it is
    then off by U |mean| + gamma mean |u - first mean|.  The differences of the second pass are float32 numbers, off by U of
    themselves; the variance is (3 + cols / 1024) gamma-like roundings of the mean square of the first pass's differences, of which
    the square of the first mean's error is taken off again."""
    x = x.detach().double()
    gamma = (48 + x.shape[-1] / 1024) * U
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    first = gamma * x.abs().mean(-1, keepdim=True)        # error of the first mean
    d_mean = U * (mean.abs() + first) + gamma * (c.abs().mean(-1, keepdim=True) + first)
    var = c.square().mean(-1, keepdim=True)
    d_var = 3 * gamma * (var + first ** 2) + d_mean ** 2
    rstd = 1 / torch.sqrt(var + eps)
    # 1 / sqrt falls the fastest at its lower end
    low = torch.rsqrt((var - d_var).clamp_min(0) + eps)
    d_rstd = low - rstd + 4 * U * low
    d_hat = low * d_mean + (c.abs() + d_mean) * d_rstd + 4 * U * (c.abs() + d_mean) * low
    return 1.1 * (w.detach().double().abs() * d_hat) + 4 * U * (c * rstd * w.double()).abs() + 1e-30
