"""lrbinner_amd.train_ops on the GPU (csrc/lrb_norm.hip, csrc/lrb_muon.hip) against plain 64-bit forms."""
import math

import pytest
import torch

from lrbinner_amd import ae_utils, train_ops
from train_ops_ref import HALF_STEP, far_row_tolerance, gradient_like, matrices_within, norm_ref, orthogonal_ref, orthogonal_tolerance, within

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
COEF = train_ops.COEFFICIENTS


def inputs(rows, cols, dtype, wtype=torch.float32, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    x = (r(rows, cols) * (0.5 + r(cols).abs()) + 0.5 * r(rows, 1)).to(dtype)
    return x, (1 + 0.2 * r(cols)).to(wtype), (0.2 * r(cols)).to(wtype), r(rows, cols).to(dtype), \
        torch.rand(rows, cols, device="cuda", generator=gen) >= 0.2


def both_passes(x, w, b, dy, eps=1e-5, **more):
    leaves = [t.detach().requires_grad_() if t.layout == torch.strided and not t.requires_grad else t for t in (x, w, b)]
    y = train_ops.layer_norm(*leaves, eps, **more)
    return (y.detach(), *torch.autograd.grad(y, leaves, dy))


def check(x, w, b, dy, eps=1e-5, **more):
    got = both_passes(x, w, b, dy, eps, **more)
    want, tol = norm_ref(x, w, b, eps, dy, **more)
    for name, g, e, t in zip(("y", "dx", "dw", "db"), got, want, tol):
        within(g, e, t, name)
    with torch.no_grad():
        assert torch.equal(train_ops.layer_norm(x, w, b, eps, **more), got[0])
    return got


# every layout of a row over threads, its ends and their neighbours
COLS = [1, 2, 3, 7, 16, 63, 64, 65, 128, 129, 255, 256, 257, 511, 513, 1000, 1024, 1025, 2047, 2049, 4095, 4096, 4097, 8191, 8192,
        8193, 16383, 16384, 16385, 20001]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("cols", COLS)
def test_layer_norm(cols, kind):
    for rows in (1, 5, 67):
        for block in (False, True):
            x, w, b, dy, keep = inputs(rows, cols, TYPES[kind], torch.float32 if rows != 5 else TYPES[kind], seed=rows)
            check(x, w, b, dy, **(dict(slope=0.01, keep=keep, keep_scale=1.25) if block else {}))


@pytest.mark.parametrize("rows,cols", [(70001, 3), (33333, 128), (9001, 1000), (2500, 5000), (1500, 17000)])
def test_layer_norm_of_more_rows_than_workgroups(rows, cols):
    x, w, b, dy, keep = inputs(rows, cols, torch.float32)
    check(x, w, b, dy)
    check(x.bfloat16(), w, b, dy.bfloat16(), slope=0.3)
    check(x, w, b, dy, keep=keep, keep_scale=1.0)


@pytest.mark.parametrize("kind", list(TYPES))
def test_layer_norm_strides(kind):
    t = TYPES[kind]
    x, w, b, dy, keep = inputs(40, 301, t)
    wide = torch.zeros(40, 700, dtype=t, device="cuda")
    wide[:, 13:314] = x
    want = check(x, w, b, dy)
    for other in (wide[:, 13:314], x.t().contiguous().t(), torch.stack([x, x], 2)[:, :, 1]):
        assert not other.is_contiguous()
        for got, e in zip(both_passes(other, w, b, dy), want):
            assert torch.equal(got, e)
    for got, e in zip(both_passes(x, torch.stack([w, w], 1)[:, 0], b, wide.new_zeros(40, 302)[:, 1:].copy_(dy)), want):
        assert torch.equal(got, e)
    # one row of gradients for all, as a sum's backward pass gives
    check(x, w, b, dy[:1].expand(40, 301))
    check(x[3:4].expand(40, 301), w, b, dy)
    check(x, w, b, dy[:1, :1].expand(40, 301))
    # leading axes
    x3, dy3 = x.reshape(4, 10, 301), dy.reshape(4, 10, 301)
    for got, e in zip(both_passes(x3, w, b, dy3), want):
        assert torch.equal(got.reshape(e.shape), e)
    check(x3.transpose(0, 1), w, b, dy3.transpose(0, 1), keep=keep.reshape(4, 10, 301).transpose(0, 1), keep_scale=2.0)
    v = x[0].clone()
    assert torch.equal(train_ops.layer_norm(v, w, b), want[0][0])


def test_layer_norm_far_rows():
    big = torch.empty(2 ** 32 + 4096, dtype=torch.bfloat16, device="cuda")
    x, w, b, dy, _ = inputs(3, 1000, torch.bfloat16)
    far, far_dy = (big.as_strided((3, 1000), (2 ** 31 + 7, 1), at) for at in (0, 1500))
    far.copy_(x), far_dy.copy_(dy)
    for got, e in zip(both_passes(far, w, b, far_dy), both_passes(x, w, b, dy)):
        assert torch.equal(got, e)


def test_layer_norm_of_more_than_2_31_elements():
    rows, cols = 2 ** 23 + 3, 257
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    tail, w, b, dy, _ = inputs(50, cols, torch.bfloat16)
    x[-50:] = tail
    y = train_ops.layer_norm(x, w, b)
    assert torch.equal(y[-50:], train_ops.layer_norm(tail, w, b))
    assert torch.equal(y[:5], b.bfloat16().expand(5, cols))
    x.requires_grad_()
    full = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    full[-50:] = dy
    dx, = torch.autograd.grad(train_ops.layer_norm(x, w, b), x, full)
    assert torch.equal(dx[-50:], both_passes(tail, w, b, dy)[1]) and not bool(dx[:-50].any())


def test_layer_norm_parts():
    x, w, b, dy, keep = inputs(30, 200, torch.float32)
    want, tol = norm_ref(x, w, None, 1e-5, dy)
    xg, wg, bg = (t.clone().requires_grad_() for t in (x, w, b))
    got = torch.autograd.grad(train_ops.layer_norm(xg, wg), (xg, wg), dy)
    within(got[0], want[1], tol[1]), within(got[1], want[2], tol[2])
    want, tol = norm_ref(x, None, b, 1e-5, dy)
    got = torch.autograd.grad(train_ops.layer_norm(xg, None, bg), (xg, bg), dy)
    within(got[0], want[1], tol[1]), within(got[1], want[3], tol[3])
    want, tol = norm_ref(x, None, None, 1e-5, dy)
    within(torch.autograd.grad(train_ops.layer_norm(xg), xg, dy)[0], want[1], tol[1])
    want, tol = norm_ref(x, w, b, 1e-5, dy)
    within(torch.autograd.grad(train_ops.layer_norm(x, wg, b), wg, dy)[0], want[2], tol[2])
    within(torch.autograd.grad(train_ops.layer_norm(x, w, bg), bg, dy)[0], want[3], tol[3])
    within(torch.autograd.grad(train_ops.layer_norm(xg, w, b), xg, dy)[0], want[1], tol[1])
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(train_ops.layer_norm(xg, wg, bg), xg, dy.requires_grad_(), create_graph=True)
        g.sum().backward()


def test_layer_norm_no_rows():
    x, w = torch.zeros(0, 9, device="cuda", requires_grad=True), torch.ones(9, device="cuda", requires_grad=True)
    y = train_ops.layer_norm(x, w, w)
    y.sum().backward()
    assert y.shape == (0, 9) and x.grad.shape == (0, 9) and torch.equal(w.grad, torch.zeros_like(w))
    x = torch.zeros(0, 20000, device="cuda", requires_grad=True)
    w = torch.ones(20000, device="cuda", requires_grad=True)
    train_ops.layer_norm(x, w).sum().backward()
    assert not bool(w.grad.any())


@pytest.mark.parametrize("cols", [40, 700, 3000, 9000, 18000])
def test_layer_norm_not_a_number_stays_in_its_row(cols):
    x, w, b, dy, keep = inputs(9, cols, torch.float32)
    clean = both_passes(x, w, b, dy)
    x[3, 7], x[5, 20] = float("nan"), float("inf")
    y, dx, _, _ = both_passes(x, w, b, dy)
    for r in range(9):
        if r in (3, 5):
            assert bool(y[r].isnan().all()) and bool(dx[r].isnan().all())
        else:
            assert torch.equal(y[r], clean[0][r]) and torch.equal(dx[r], clean[1][r])
    # what is dropped does not count, whatever it holds; a row of which nothing is left is the bias
    x, w, b, dy, keep = inputs(9, cols, torch.float32)
    keep[4] = False
    clean = check(x, w, b, dy, slope=0.01, keep=keep, keep_scale=1.25)
    dirty = torch.where(keep, x, torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda")[torch.arange(cols, device="cuda") % 3])
    for got, e in zip(both_passes(dirty, w, b, dy, slope=0.01, keep=keep, keep_scale=1.25), clean):
        assert torch.equal(got, e)
    assert torch.equal(clean[0][4], b) and not bool(clean[1][:][~keep].any())


def test_layer_norm_constant_and_far_rows():
    x, w, b, dy, _ = inputs(6, 300, torch.float32)
    x[0] = 0
    x[1] = 1e4                       # no variance
    x[2] += 1e4                      # a mean far above the deviation
    x[3] *= 1e-20
    x[4] *= 1e15
    check(x, w, b, dy)
    check(x, w, b, dy, eps=1.0)


def test_layer_norm_same_bits_twice_and_on_another_stream():
    x, w, b, dy, keep = inputs(5000, 768, torch.bfloat16)
    first = both_passes(x, w, b, dy, slope=0.01, keep=keep, keep_scale=1.25)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = both_passes(x, w, b, dy, slope=0.01, keep=keep, keep_scale=1.25)
    torch.cuda.current_stream().wait_stream(side)
    for f, s in zip(first, second):
        assert torch.equal(f, s)


def test_layer_norm_gradient_against_differences():
    x, w, b, dy, keep = inputs(8, 1000, torch.float32)
    more = dict(slope=0.2, keep=keep, keep_scale=1.25)
    _, dx, dw, db = both_passes(x, w, b, dy, **more)
    gen = torch.Generator(device="cuda").manual_seed(4)
    for k, grad in enumerate((dx, dw, db)):
        v = torch.randn(grad.shape, device="cuda", generator=gen, dtype=torch.float64) * ((x, w, b)[k].abs() > 1e-3)

        def loss(s):
            a = [t.double() + (s * v if i == k else 0) for i, t in enumerate((x, w, b))]
            u = torch.where(keep, torch.where(a[0] > 0, a[0], 0.2 * a[0]) * 1.25, 0.0)
            c = u - u.mean(1, keepdim=True)
            return ((c / torch.sqrt(c.square().mean(1, keepdim=True) + 1e-5) * a[1] + a[2]) * dy.double()).sum()

        diff = float((loss(1e-6) - loss(-1e-6)) / 2e-6)
        # 8000 products of float32 gradients, each off by some 1e-6 of its size: a random sum
        assert abs(diff - float((grad.double() * v).sum())) < 1e-5 * float((grad.double() * v).norm()) + 1e-5 * (1 + abs(diff))


def capture(fn, warm=2):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(warm):
            fn()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def test_layer_norm_captured():
    cases = []
    for seed, (rows, cols) in enumerate([(300, 128), (100, 3000)]):  # two graphs that live side by side
        x, w, b, dy, keep = inputs(rows, cols, torch.float32, seed=seed)

        def passes(x=x, w=w, b=b, dy=dy, keep=keep):
            # gradients by formula of detached leaves: no eager graph of them lives when the capture begins
            leaves = [t.detach().requires_grad_() for t in (x, w, b)]
            y = train_ops.layer_norm(*leaves, slope=0.01, keep=keep, keep_scale=1.25)
            return (y.detach(), *torch.autograd.grad(y, leaves, dy))

        cases.append((*capture(passes), passes, x))
    for turn in range(4):
        for graph, out, passes, x in cases:
            x.copy_(torch.randn(x.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(turn)))
            graph.replay()
        noise = torch.randn(1000, 1000, device="cuda").sum()
        torch.cuda.synchronize()
        for graph, out, passes, x in cases:
            for got, e in zip(out, passes()):
                assert torch.equal(got, e)
        del noise


# ---- the orthogonalised update ------------------------------------------------------------------

def check_orthogonal(g, steps=5, coefficients=COEF, eps=1e-7, **more):
    got = train_ops.orthogonalize(g, steps=steps, coefficients=coefficients, eps=eps, **more)
    assert got.shape == g.shape
    exact = orthogonal_ref(g, steps, coefficients, eps)
    matrices_within(got, exact, orthogonal_tolerance(exact, g, steps, coefficients, eps), HALF_STEP[got.dtype], str(tuple(g.shape)))
    return got


SHAPES = [(1, 1), (1, 7), (5, 1), (2, 2), (8, 128), (128, 8), (31, 33), (63, 64), (64, 64), (65, 63), (64, 200), (100, 100), (127, 129),
          (128, 128), (128, 168), (168, 128), (129, 130), (200, 72), (128, 257), (130, 700), (256, 256), (257, 300), (511, 1025),
          (1000, 1), (1, 5000), (3, 4097), (700, 2100)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(shape, kind):
    g = gradient_like(*shape, torch.Generator().manual_seed(2), "cuda").to(TYPES[kind])
    got = check_orthogonal(g)
    assert got.dtype == g.dtype and got.is_contiguous()


# stacks that take the larger tiles, whole and cut
@pytest.mark.parametrize("count,rows,cols", [(3, 33, 70), (2, 70, 33), (70, 300, 330), (70, 200, 330), (210, 250, 256), (5000, 2, 3), (40, 129, 513)])
def test_orthogonalize_stacks(count, rows, cols):
    g = gradient_like(rows, cols, torch.Generator().manual_seed(5), "cuda", (count,))
    check_orthogonal(g)
    check_orthogonal(g.transpose(1, 2))
    check_orthogonal(g.bfloat16())


# long enough that several steps share one formation of X
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(700, 2100), (1500, 600), (513, 4000)])
def test_orthogonalize_in_blocks_of_steps(rows, cols, kind):
    gen = torch.Generator().manual_seed(8)
    g = gradient_like(rows, cols, gen, "cuda").to(TYPES[kind])
    n = min(rows, cols)
    for steps in (1, 2, 3, 4, 5, 6, 7, 12):
        check_orthogonal(g, steps=steps)
        check_orthogonal(g, steps=steps, coefficients=(15 / 8, -10 / 8, 3 / 8))
    check_orthogonal(g * 1e-12)
    check_orthogonal(torch.randn(rows, cols, generator=gen).cuda().to(TYPES[kind]))
    check_orthogonal((torch.randn(rows, 7, generator=gen) @ torch.randn(7, cols, generator=gen)).cuda().to(TYPES[kind]))
    u, _, vt = torch.linalg.svd(torch.randn(rows, cols, generator=gen).cuda(), full_matrices=False)
    check_orthogonal(((u * torch.logspace(0, -5, n, device="cuda")) @ vt).to(TYPES[kind]))
    three = torch.stack([g, g, g])
    three[1] = 0
    got = check_orthogonal(three)
    # (not the same bits in 0 and 2: which tiles of a launch are cut along k goes by their place in it)
    assert not bool(got[1].any()) and torch.equal(got, train_ops.orthogonalize(three))


@pytest.mark.parametrize("rows,cols", [(37, 90), (90, 37), (128, 168), (300, 200)])
def test_orthogonalize_strides(rows, cols):
    g = gradient_like(rows, cols, torch.Generator().manual_seed(6), "cuda")
    want = train_ops.orthogonalize(g)
    wide = torch.zeros(rows + 3, cols + 9, device="cuda")
    wide[1:rows + 1, 5:cols + 5] = g
    every = torch.zeros(2 * rows, 3 * cols, device="cuda")
    every[::2, ::3] = g
    for other in (wide[1:rows + 1, 5:cols + 5], g.t().contiguous().t(), every[::2, ::3]):
        assert torch.equal(train_ops.orthogonalize(other), want)
    assert torch.equal(train_ops.orthogonalize(g.t()), want.t())
    around = torch.full_like(wide, 7.0)
    out = around[1:rows + 1, 5:cols + 5]
    assert train_ops.orthogonalize(g, out=out) is out and torch.equal(out, want)
    out.fill_(7.0)
    assert bool((around == 7.0).all())  # nothing beside it was written
    turned = torch.empty(cols, rows, device="cuda").t()
    assert torch.equal(train_ops.orthogonalize(g, out=turned), want)
    here = g.clone()
    assert torch.equal(train_ops.orthogonalize(here, out=here), want)
    half = torch.empty(rows, cols, device="cuda", dtype=torch.float16)
    assert torch.equal(train_ops.orthogonalize(g, out=half), want.half())
    four = torch.stack([g, 2 * g, g.flip(0), g.flip(1)]).reshape(2, 2, rows, cols)
    got = train_ops.orthogonalize(four.transpose(0, 1))
    assert torch.equal(got[0, 0], want) and torch.equal(got[1, 0], train_ops.orthogonalize(four[0, 1]))
    same = train_ops.orthogonalize(g.expand(3, rows, cols))
    assert all(torch.equal(s, want) for s in same)


@pytest.mark.parametrize("shape", [(24, 40), (128, 168), (300, 260)])
def test_orthogonalize_values(shape):
    gen = torch.Generator().manual_seed(7)
    g = gradient_like(*shape, gen, "cuda")
    n = min(shape)
    u, _, vt = torch.linalg.svd(torch.randn(*shape, generator=gen, dtype=torch.float64), full_matrices=False)
    check_orthogonal(((u * torch.logspace(0, -6, n, dtype=torch.float64)) @ vt).float().cuda())   # ill conditioned
    check_orthogonal(torch.outer(torch.randn(shape[0], generator=gen), torch.randn(shape[1], generator=gen)).cuda())  # of rank one
    check_orthogonal(torch.randn(*shape, generator=gen).cuda())
    for scale in (1e-30, 1e-6, 1e6, 1e30):
        check_orthogonal(g * scale, eps=0.0)
        check_orthogonal(g * scale)  # below eps: scaled up by less
    for coefficients in ((1.5, -0.5, 0.0), (15 / 8, -10 / 8, 3 / 8), (2.0, -1.5, 0.5), (1.0, 0.0, 0.0), (6.0, -9.0, 4.0), (-3.0, 4.0, -2.0)):
        for steps in (1, 2, 7):
            if (coefficients[0], steps) in ((6.0, 2), (6.0, 7), (-3.0, 7)):  # singular values may grow without bound: refused
                with pytest.raises(ValueError, match="grow beyond"):
                    train_ops.orthogonalize(g, steps=steps, coefficients=coefficients)
                continue
            check_orthogonal(g, steps=steps, coefficients=coefficients)
    assert not bool(train_ops.orthogonalize(torch.zeros(*shape, device="cuda")).any())
    assert not bool(train_ops.orthogonalize(torch.zeros(*shape, device="cuda"), eps=0.0).any())
    assert not bool(train_ops.orthogonalize(g, coefficients=(0.0, 0.0, 0.0)).any())
    three = torch.stack([g, g, g])
    three[1, 3, 5] = float("nan")
    got = train_ops.orthogonalize(three)
    assert bool(got[1].isnan().all()) and torch.equal(got[0], train_ops.orthogonalize(g)) and torch.equal(got[2], got[0])
    three[1, 3, 5] = -float("inf")
    got = train_ops.orthogonalize(three)
    assert bool(got[1].isnan().all()) and torch.equal(got[2], got[0])


def weights(shapes, kinds, seed=0):
    gen = torch.Generator().manual_seed(seed)
    p = [torch.randn(s, generator=gen).cuda().to(k) for s, k in zip(shapes, kinds)]
    g = [gradient_like(s[-2], s[-1], gen, "cuda", s[:-2]).to(k) for s, k in zip(shapes, kinds)]
    m = [gradient_like(s[-2], s[-1], gen, "cuda", s[:-2]) for s in shapes]
    return p, g, m


def muon_ref(p, g, kept, lr, momentum, nesterov, decay, scale=None, steps=5):
    """p after a step in 64 bits, and its Frobenius tolerance.  u is made of the momentum that is `kept`: of the buffer as the call
    left it (whose own rounding to 16 bits may fall either way where it lies next to a border between two numbers)."""
    u = g.double()
    if kept is not None:
        u = (1 - momentum) * u + momentum * kept.double() if nesterov else kept.double()
    o = orthogonal_ref(u, steps, COEF, 1e-7)
    tol = orthogonal_tolerance(o, u.float(), steps, COEF, 1e-7)
    # u itself is float32 in the kernel: off by 3 roundings, which the iteration passes on as it does those of its factors
    off = orthogonal_ref((u.float() * (1 + 2.0 ** -22)).float(), steps, COEF, 1e-7) - o
    tol = 2 * tol + torch.linalg.vector_norm(off, dim=(-2, -1))
    by = math.sqrt(max(1, p.shape[-2] / p.shape[-1])) if scale is None else scale
    new = p.double() * (1 - lr * decay) - lr * by * o
    return new, lr * by * tol + 4 * 2.0 ** -24 * torch.linalg.vector_norm(new, dim=(-2, -1))


def check_muon(p, g, m, lr=0.1, momentum=0.9, nesterov=True, weight_decay=0.3, **more):
    ms = [None] * len(p) if m is None else m
    was, moved = [t.clone() for t in p], [None if c is None else momentum * c.double() + (1 - momentum) * b.double() for b, c in zip(g, ms)]
    train_ops.muon_step(p, g, m, lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, **more)
    for a, before, b, c, wc in zip(p, was, g, ms, moved):
        wa, tol = muon_ref(before, b, c, lr, momentum, nesterov, weight_decay, **more)
        matrices_within(a, wa, tol, HALF_STEP[a.dtype], str(tuple(a.shape)))
        if c is not None:
            # two products and a sum in float32, which may cancel
            within(c, wc, 3 * 2.0 ** -24 * (wc.abs() + (1 - momentum) * b.double().abs()) + 1.01 * HALF_STEP[c.dtype] * wc.abs() + 1e-7 * (wc.abs().max() + 1e-30), "momentum")


NETWORK = [(128, 168), (128, 128), (8, 128), (8, 128), (128, 8), (128, 128), (168, 128)]


@pytest.mark.parametrize("nesterov", [False, True])
def test_muon_step_on_the_default_network(nesterov):
    p, g, m = weights(NETWORK, [torch.float32] * 7)
    for _ in range(3):
        check_muon(p, g, m, nesterov=nesterov)


def test_muon_step_mixed():
    f, b, h = torch.float32, torch.bfloat16, torch.float16
    shapes = [(40, 60), (60, 40), (1, 9), (300, 500), (3, 20, 30), (2, 2, 50, 20), (700, 130), (128, 300), (5, 5)]
    p, g, m = weights(shapes, [f, b, h, b, f, h, f, b, f])
    check_muon(p, [x.float() for x in g], m)                  # gradients of another type
    check_muon(p, g, [x.bfloat16() for x in m])                # momentum in 16 bits
    check_muon(p, g, None, weight_decay=0.0)
    check_muon(p, g, m, scale=0.2, steps=3)
    turned = [x.transpose(-1, -2).contiguous().transpose(-1, -2) for x in p]
    check_muon(turned, g, m)
    check_muon(p, [x.transpose(-1, -2).contiguous().transpose(-1, -2) for x in g], m)
    wide = torch.randn(60, 300, device="cuda")                 # three weights side by side in one
    check_muon([wide[:, :100], wide[:, 100:200], wide[:, 200:]], [torch.randn(60, 100, device="cuda") for _ in range(3)], None)


def test_muon_step_long_list_and_empty_weights():
    shapes = [(10 + k, 50 - k) for k in range(37)] + [(0, 5), (4, 0), (20, 300)]
    p, g, m = weights([s for s in shapes if 0 not in s], [torch.float32] * 38)
    p.insert(7, torch.zeros(0, 5, device="cuda")), g.insert(7, torch.zeros(0, 5, device="cuda")), m.insert(7, torch.zeros(0, 5, device="cuda"))
    keep = [(q.clone(), n.clone()) for q, n in zip(p, m)]
    train_ops.muon_step(p, g, m, lr=0.1)
    for k in (0, 16, 20, 38):  # alone: the same bits as in company
        q, n = keep[k]
        train_ops.muon_step([q], [g[k]], [n], lr=0.1)
        assert torch.equal(q, p[k]) and torch.equal(n, m[k])


def test_muon_optimizer_captured():
    torch.manual_seed(0)

    def build():
        torch.manual_seed(1)
        layers = [torch.nn.Linear(40, 64, device="cuda"), torch.nn.Linear(64, 130, device="cuda")]
        return layers, train_ops.Muon([x.weight for x in layers], lr=0.05, weight_decay=0.1)

    data = torch.randn(6, 32, 40, device="cuda")
    target = torch.randn(32, 130, device="cuda")
    eager, opt_e = build()
    graphed, opt_g = build()
    static = data[0].clone()

    def step(layers, opt, x):
        opt.zero_grad(set_to_none=True)
        y = layers[1](train_ops.layer_norm(layers[0](x), slope=0.01))
        ((y - target) ** 2).mean(1).mean(0).backward()
        opt.step()

    fresh, opt_f = build()
    with pytest.raises(RuntimeError, match="before the capture"):
        # the refusal itself, without a capture that it would have to abandon
        saved, torch.cuda.is_current_stream_capturing = torch.cuda.is_current_stream_capturing, lambda: True
        try:
            step(fresh, opt_f, static)
        finally:
            torch.cuda.is_current_stream_capturing = saved
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for k in range(2):
            step(graphed, opt_g, static)
    torch.cuda.current_stream().wait_stream(side)
    for k in range(2):
        step(eager, opt_e, static)
    graph = torch.cuda.CUDAGraph()
    opt_g.zero_grad(set_to_none=True)
    with torch.cuda.graph(graph):
        step(graphed, opt_g, static)
    for k in range(1, 6):
        static.copy_(data[k])
        graph.replay()
        step(eager, opt_e, data[k])
        torch.cuda.synchronize()
        for a, b in zip(eager, graphed):
            # the linear layers' products are a library's, whose order of sums may differ between the two
            assert float((a.weight - b.weight).detach().abs().max()) < 1e-4


def test_muon_two_graphs_and_streams():
    p, g, m = weights([(128, 168), (300, 200)], [torch.float32] * 2)
    q, h, n = ([t.clone() for t in x] for x in (p, g, m))
    for t in h:
        t.mul_(-2.0).add_(0.001)
    first = capture(lambda: train_ops.muon_step(p, g, m, lr=0.1))[0]
    second = capture(lambda: train_ops.muon_step(q, h, n, lr=0.1))[0]
    copies = [[t.clone() for t in x] for x in (p, m, q, n)]
    side = torch.cuda.Stream()
    for _ in range(4):
        side.wait_stream(torch.cuda.current_stream())
        first.replay()
        with torch.cuda.stream(side):
            second.replay()
        torch.cuda.current_stream().wait_stream(side)
        train_ops.muon_step(copies[0], g, copies[1], lr=0.1)
        train_ops.muon_step(copies[2], h, copies[3], lr=0.1)
        torch.cuda.synchronize()
        for a, b in zip((p, m, q, n), copies):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_versions_are_counted():
    p, g, m = weights([(20, 30)], [torch.float32])
    p[0].requires_grad_()
    loss = (p[0] * p[0]).sum()
    train_ops.muon_step(p, g, m, lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


# ---- the network that uses them -------------------------------------------------------------------

def test_vae_with_layer_norm_runs_as_its_formula():
    torch.manual_seed(0)
    vae = ae_utils.VAE(32, 136, norm="layer", device="cuda")
    twin = ae_utils.VAE(32, 136, norm="layer").double()
    twin.load_state_dict({k: v.cpu() for k, v in vae.state_dict().items()})
    x = torch.rand(300, 168, device="cuda")
    mu = vae.encode(x)
    z = x.cpu().double()
    for lin, norm in zip(twin.encoderlayers, twin.encodernorms):
        z = torch.nn.functional.leaky_relu(lin(z), 0.01)
        z = (z - z.mean(1, keepdim=True)) / torch.sqrt(z.var(1, unbiased=False, keepdim=True) + 1e-5) * norm.weight + norm.bias
    assert float((twin.mu(z).detach() - torch.from_numpy(mu)).abs().max()) < 1e-4
    # a training step's gradients, dropout included: the draws of the same seed, once by the operator, once by formulas
    vae.train()

    def loss_and_grads(model, block):
        torch.manual_seed(5)
        model._block = block
        recon, m, s = model(x)
        loss = model.calc_loss(x, recon, m, s)[0]
        grads = torch.autograd.grad(loss, list(model.parameters()))
        del model._block
        return float(loss.detach()), grads

    def by_formulas(layer, norm, v):
        v = layer(v)
        keep = torch.empty(v.shape, dtype=torch.bool, device=v.device).bernoulli_(1 - vae.dropout)
        v = torch.nn.functional.leaky_relu(v, 0.01) * keep / (1 - vae.dropout)
        c = v - v.mean(1, keepdim=True)
        return c / torch.sqrt(c.square().mean(1, keepdim=True) + 1e-5) * norm.weight + norm.bias

    own, own_grads = loss_and_grads(vae, vae._block)
    ref, ref_grads = loss_and_grads(vae, by_formulas)
    assert abs(own - ref) < 1e-5 * abs(ref)
    for a, b in zip(own_grads, ref_grads):
        assert float((a - b).norm()) < 1e-4 * float(b.norm()) + 1e-7


@pytest.mark.parametrize("norm,optimizer", [("layer", "muon"), ("layer", "adam"), ("batch", "muon")])
@pytest.mark.parametrize("use_graph", [None, False])
def test_vae_trains(norm, optimizer, use_graph):
    torch.manual_seed(0)
    data = torch.rand(3000, 168, device="cuda")
    vae = ae_utils.VAE(32, 136, norm=norm, device="cuda")
    before = {k: v.clone() for k, v in vae.state_dict().items()}
    vae.trainmodel(data, nepochs=4, batchsteps=[2], batch_size=256, optimizer=optimizer, use_graph=use_graph)
    for k, v in vae.state_dict().items():
        assert bool(torch.isfinite(v).all()) and not torch.equal(v, before[k]), k
    assert getattr(vae, "_native", None) is None
    mu = vae.encode(data, chunk=1000)
    assert mu.shape == (3000, 8) and bool(torch.isfinite(torch.from_numpy(mu)).all())
    vae.trainmodel(data, nepochs=1, batchsteps=[], batch_size=256, optimizer=optimizer, use_graph=use_graph)


def test_a_run_after_a_fused_one_encodes_with_its_own_weights():
    torch.manual_seed(0)
    data = torch.rand(600, 168, device="cuda")
    vae = ae_utils.VAE(32, 136, device="cuda")
    vae.trainmodel(data, nepochs=1, batchsteps=[], batch_size=256)
    assert vae._native is not None
    vae.trainmodel(data, nepochs=2, batchsteps=[], batch_size=256, optimizer="muon")
    mu = vae.encode(data)
    vae.eval()
    with torch.no_grad():
        assert float((vae._encode(data)[0].cpu() - torch.from_numpy(mu)).abs().max()) < 1e-5


@pytest.mark.parametrize("shape", [(9, 32, 48), (5, 300, 200)])
def test_out_that_lies_over_other_matrices(shape):
    gen = torch.Generator(device="cuda").manual_seed(4)
    for take in (lambda b: (b[:-1], b[1:]), lambda b: (b[1:], b[:-1]), lambda b: (b, b.flip(0)), lambda b: (b, b)):
        buf = torch.randn(*shape, device="cuda", generator=gen)
        g, out = take(buf)
        want = train_ops.orthogonalize(g.clone())
        assert torch.equal(train_ops.orthogonalize(g, out=out), want)
    buf = torch.randn(shape[0], shape[0], 40, 24, device="cuda", generator=gen)  # a view that takes the stacks' axes in turn
    want = train_ops.orthogonalize(buf[0].clone())
    assert torch.equal(train_ops.orthogonalize(buf[0], out=buf[:, 0]), want)


def test_views_with_their_sign_turned():
    x, w, b, dy, _ = inputs(20, 33, torch.float32)
    turned = torch._neg_view(x.t().contiguous()).t()
    assert torch.equal(train_ops.layer_norm(turned, w, b), train_ops.layer_norm(-x, w, b))
    assert torch.equal(train_ops.layer_norm(torch._neg_view(x), w, b), train_ops.layer_norm(-x, w, b))
    assert torch.equal(train_ops.orthogonalize(torch._neg_view(x)), train_ops.orthogonalize(-x))


def test_inside_inference_mode():
    x, w, b, _, _ = inputs(20, 33, torch.float32)
    want, moved = train_ops.layer_norm(x, w, b), x.clone()
    turned = train_ops.orthogonalize(x)
    train_ops.muon_step([moved], [x], lr=0.1)
    with torch.inference_mode():
        assert torch.equal(train_ops.layer_norm(x, w, b), want) and torch.equal(train_ops.orthogonalize(x), turned)
        again = x.clone()
        train_ops.muon_step([again], [x], lr=0.1)
        assert torch.equal(again, moved)


def test_threads_on_streams_of_their_own():
    import threading

    gen = torch.Generator(device="cuda").manual_seed(5)
    gs = [torch.randn(*s, device="cuda", generator=gen) for s in ((100, 150), (300, 200), (64, 64), (700, 520))]
    want = [train_ops.orthogonalize(g) for g in gs]
    got, failed = [None] * len(gs), []
    torch.cuda.synchronize()

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    out = train_ops.orthogonalize(gs[k])
                torch.cuda.current_stream().synchronize()
                got[k] = out
        except Exception as e:  # an assertion of a thread is not seen
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(gs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def test_second_derivatives_are_refused():
    x, w, b, dy, _ = inputs(6, 20, torch.float32)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    plain = torch.autograd.grad(train_ops.layer_norm(*leaves), leaves, dy)
    graph = torch.autograd.grad(train_ops.layer_norm(*leaves), leaves, dy, create_graph=True)
    for g, e in zip(graph, plain):
        assert torch.equal(g, e)
    with pytest.raises(RuntimeError):  # (of gradients that hang on dy: by autograd itself, these do not)
        graph[0].sum().backward()


# 128-tiles, and 256-tiles, of which two products of a block share a launch; of an uneven number of steps
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("count,rows,cols", [(7, 1000, 2100), (4, 2048, 2700), (5, 1901, 900)])
def test_orthogonalize_stacks_in_blocks_of_steps(count, rows, cols, kind):
    g = gradient_like(rows, cols, torch.Generator().manual_seed(9), "cuda", (count,)).to(TYPES[kind])
    g[1] *= 1e-12  # below eps: factors of its own
    for steps in (3, 5, 8):
        got = check_orthogonal(g, steps=steps)
        assert torch.equal(got, train_ops.orthogonalize(g, steps=steps))


def test_muon_step_in_blocks_of_steps_on_weights_of_two_types():
    shapes = [(700, 2100), (1500, 600), (2, 640, 1500), (100, 90)]
    for kinds in (("bf16", "bf16", "f16", "bf16"), ("bf16", "f32", "f16", "f32")):
        p, g, m = weights(shapes, [TYPES[k] for k in kinds])
        check_muon(p, g, m)
        check_muon(p, g, None)


# long enough that A could be carried over several steps: it is formed anew for each, whatever the result's type
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("shape", [(700, 2100), (1500, 600), (7, 1000, 2100), (90, 130), (300, 200)])
def test_a_16_bit_result_is_the_float32_result_rounded(shape, kind):
    t = TYPES[kind]
    g = gradient_like(*shape[-2:], torch.Generator().manual_seed(3), "cuda", shape[:-2]).to(t)
    for steps in (2, 5):
        assert torch.equal(train_ops.orthogonalize(g, steps=steps), train_ops.orthogonalize(g.float(), steps=steps).to(t))
    p, m = torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).to(t), g.float()
    q, n = p.float(), m.clone()
    train_ops.muon_step([p], [g], [m], lr=0.1)
    train_ops.muon_step([q], [g.float()], [n], lr=0.1)
    assert torch.equal(p, q.to(t)) and torch.equal(m, n)


def test_muon_step_on_gradients_that_are_copied():
    gen = torch.Generator().manual_seed(6)
    grads = [gradient_like(20, 30, gen, "cuda", (3, 4)).transpose(0, 1) for _ in range(4)]
    grads += [gradient_like(200, 300, gen, "cuda", (4, 1)).expand(4, 3, 200, 300) for _ in range(3)]
    params = [torch.randn(g.shape, generator=gen).cuda() for g in grads]
    momenta = [torch.zeros(g.shape, device="cuda") for g in grads]
    others = [[t.clone() for t in x] for x in (params, momenta)]
    train_ops.muon_step(params, grads, momenta, lr=0.1)
    train_ops.muon_step(others[0], [g.contiguous() for g in grads], others[1], lr=0.1)
    for got, want in zip((params, momenta), others):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# rows in every layout over threads
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("cols", [7, 41, 61, 700, 1000, 4095, 10007, 16385, 20001])
def test_layer_norm_rows_of_equal_elements(cols, kind):
    t = TYPES[kind]
    x, w, b, dy, keep = inputs(9, cols, t)
    values = [1.0, 0.1, 1e3, 1e5 if kind != "f16" else 6e4, -7.7]
    for r, v in enumerate(values):
        x[r + 2] = v
    y = train_ops.layer_norm(x, w, b)
    for r in range(len(values)):  # no variance: what is left is the bias
        assert torch.equal(y[r + 2], b.to(t)), values[r]
    if kind != "f16":
        x[4] = 3e34
        assert torch.equal(train_ops.layer_norm(x, w, b)[4], b.to(t))
    # ... and of the activation's rows
    y = train_ops.layer_norm(x[2:4], w, b, slope=0.01, keep=keep[2:4] | True, keep_scale=1.25)
    assert torch.equal(y, b.to(t).expand(2, cols))


@pytest.mark.parametrize("cols", [61, 700, 4095, 10007, 16385, 20001])
def test_layer_norm_rows_far_from_zero(cols):
    x, w, b, dy, _ = inputs(6, cols, torch.float32)
    x += torch.tensor([[0.0], [1e3], [-1e4], [1e5], [3e6], [-1e7]], device="cuda")
    c = x.double() - x.double().mean(1, keepdim=True)
    want = c / torch.sqrt(c.square().mean(1, keepdim=True) + 1e-5) * w.double() + b.double()
    within(train_ops.layer_norm(x, w, b), want, far_row_tolerance(x, w, 1e-5) + 2.0 ** -24 * want.abs())


def test_what_torch_would_not_see_is_refused():
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, b, _, _ = inputs(6, 20, torch.float32)
    m = train_ops.LayerNorm(20, device="cuda")

    def step(v):
        p = torch.zeros_like(v)
        train_ops.muon_step([p], [v], lr=0.1)
        return p

    calls = (lambda v: train_ops.layer_norm(v, w, b), m, lambda v: train_ops.orthogonalize(v), step)
    for call in calls:
        for grad in (False, True):
            with torch.set_grad_enabled(grad):
                with pytest.raises(RuntimeError, match="traced"):
                    torch.jit.trace(call, (x,))
                for more in ({}, dict(pre_dispatch=True)):
                    with pytest.raises(RuntimeError, match="traced"):
                        make_fx(call, **more)(x)
                with forward_ad.dual_level():
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        call(forward_ad.make_dual(x, torch.ones_like(x)))
                with pytest.raises(RuntimeError):
                    torch.func.vmap(call)(x.unsqueeze(0))
                with pytest.raises(RuntimeError):
                    torch.func.jvp(call, (x,), (x,))
                call(x)
    with torch.no_grad(), forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            train_ops.layer_norm(x, forward_ad.make_dual(w, torch.ones_like(w)), b)
        assert torch.equal(train_ops.layer_norm(x, w, b), calls[0](x))


@pytest.mark.parametrize("grad", [False, True])
def test_layer_norm_in_a_compiled_function(grad):
    x, w, b, dy, _ = inputs(6, 20, torch.float32)
    leaves = [t.requires_grad_(grad) for t in (x, w, b)]
    compiled = torch.compile(lambda *a: train_ops.layer_norm(*a) * 2, backend="eager")
    want = train_ops.layer_norm(*leaves) * 2
    for _ in range(2):
        got = compiled(*leaves)
        assert torch.equal(got, want)
        if grad:
            for g, e in zip(torch.autograd.grad(got, leaves, dy), torch.autograd.grad(want, leaves, dy, retain_graph=True)):
                assert torch.equal(g, e)
    turned = torch.compile(lambda v: train_ops.orthogonalize(v) * 2, backend="eager")
    for _ in range(2):
        assert torch.equal(turned(x), train_ops.orthogonalize(x) * 2)


def test_a_penalty_on_the_gradient_is_refused():
    x, w, b, dy, _ = inputs(6, 20, torch.float32)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    plain = torch.autograd.grad(train_ops.layer_norm(*leaves).square().sum(), leaves)
    for of in ((x,), (w,), leaves):
        y = train_ops.layer_norm(*leaves)
        grads = torch.autograd.grad(y.sum(), of, create_graph=True)  # (the gradient of a sum depends on no leaf)
        with pytest.raises(RuntimeError, match="second derivatives"):
            (y.sum() + sum(g.square().sum() for g in grads)).backward()
    # a graph of the backward pass that nobody differentiates costs nothing but itself
    y = train_ops.layer_norm(*leaves)
    grads = torch.autograd.grad(y.square().sum(), leaves, create_graph=True)
    for g, e in zip(grads, plain):
        assert torch.equal(g, e)
    only = torch.autograd.grad(train_ops.layer_norm(x.detach(), w.detach(), b).sum(), b, create_graph=True)[0]
    assert torch.equal(only, torch.full_like(b, 6.0)) and not only.requires_grad


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("cols", [3, 40, 700, 9000, 18000])
def test_slope_0_is_a_relu(cols, kind):
    x, w, b, dy, keep = inputs(5, cols, TYPES[kind])
    x[1, 1], x[2, 2], x[3, 0] = -math.inf, math.nan, -0.0
    live = [0, 1, 3, 4]
    for more in ({}, dict(keep=keep, keep_scale=1.25)):
        y, dx = both_passes(x, w, b, dy, slope=0.0, **more)[:2]
        # (not the bits of a call on relu(x) without slope: another instance of the kernel, whose float32 operations may be
        # fused otherwise.  The tolerances hold for both.)
        part = {k: v[live] if k == "keep" else v for k, v in more.items()}
        want, tol = norm_ref(torch.relu(x[live]), w, b, 1e-5, dy[live], **part)
        within(y[live], want[0], tol[0], "y")
        above = (x[live] > 0).double()
        within(dx[live], want[1] * above, tol[1] * above, "dx")
        assert "keep" in more or bool(y[2].isnan().all())


@pytest.mark.parametrize("shape", [(40, 60), (300, 500)])
@pytest.mark.parametrize("momentum", [0.95, 0.999, 0.9999, 0.0])
def test_the_share_of_the_gradient_is_exact(shape, momentum):
    g = gradient_like(*shape, torch.Generator().manual_seed(2), "cuda")
    p, m = torch.zeros(*shape, device="cuda"), torch.zeros(*shape, device="cuda")
    train_ops.muon_step([p], [g], [m], lr=0.1, momentum=momentum)
    # 1 - momentum rounded to float32, and the product; float32's smallest number
    within(m, (1.0 - momentum) * g.double(), 2.02 * 2.0 ** -24 * (1.0 - momentum) * g.double().abs() + 2.0 ** -149)


# (short sides up to 16: there the tolerance counts how the iteration passes a rounding on)
@pytest.mark.parametrize("shape", [(12, 40), (12, 3000), (3000, 16)])
def test_coefficients_that_keep_a_singular_value_at_its_border(shape):
    g = torch.outer(torch.randn(shape[0], generator=torch.Generator().manual_seed(1)), torch.linspace(-1, 1, shape[1])).cuda()
    for steps, c in ((2, (0.0, 0.0, 1.0)), (3, (0.0, 0.0, 1.0)), (4, (0.5, 0.0, 0.5)), (32, (1.0, 0.0, 0.0)), (32, (1.5, -0.5, 0.0))):
        check_orthogonal(g, steps=steps, coefficients=c)
    with pytest.raises(ValueError, match="grow beyond"):
        train_ops.orthogonalize(g, steps=8, coefficients=(0.0, 0.0, 1.0))


class _Counted(torch.cuda.CUDAGraph):
    replays = 0

    def replay(self):
        _Counted.replays += 1
        super().replay()


@pytest.mark.parametrize("norm,optimizer", [("layer", "muon"), ("layer", "adam"), ("batch", "muon")])
@pytest.mark.parametrize("held", [False, True])
def test_the_vae_s_step_is_captured(norm, optimizer, held, monkeypatch):
    """Also where the caller holds a graph of the same weights."""
    torch.manual_seed(0)
    data = torch.rand(3000, 168, device="cuda")
    vae = ae_utils.VAE(32, 136, norm=norm, device="cuda")
    before = [p.detach().clone() for p in vae.parameters()]
    outputs = vae(data[:100]) if held else None
    mine = list(vae.parameters())
    monkeypatch.setattr(torch.cuda, "CUDAGraph", _Counted)
    _Counted.replays = 0
    vae.trainmodel(data, nepochs=4, batchsteps=[2], batch_size=256, optimizer=optimizer)
    # 11 batches of 256 and 5 of 512 an epoch, of which the first epoch of each size gives three to the warm-up
    assert _Counted.replays == 2 * 11 + 2 * 5 - 2 * 3
    for p, q, was in zip(vae.parameters(), mine, before):
        assert p is q and bool(torch.isfinite(p).all()) and not torch.equal(p, was)
    del outputs


def test_a_refused_step_leaves_no_state(monkeypatch):
    w = torch.nn.Parameter(torch.ones(3, 4, device="cuda"))
    w.grad = torch.ones_like(w)
    opt = train_ops.Muon([w])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before the capture"):
        opt.step()
    assert not opt.state_dict()["state"]


def test_a_failed_capture_is_said(monkeypatch, caplog):
    def refuses(graph):
        raise RuntimeError("no capture today")

    torch.manual_seed(0)
    data = torch.rand(1000, 168, device="cuda")
    vae = ae_utils.VAE(32, 136, norm="layer", device="cuda")
    before = [p.detach().clone() for p in vae.parameters()]
    monkeypatch.setattr(torch.cuda, "graph", refuses)
    with caplog.at_level("WARNING", logger="LRBinner"):
        vae.trainmodel(data, nepochs=2, batchsteps=[], batch_size=100)
    assert sum("no capture today" in r.message for r in caplog.records) == 1
    assert all(bool(torch.isfinite(p).all()) and not torch.equal(p, q) for p, q in zip(vae.parameters(), before))
