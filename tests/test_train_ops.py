"""lrbinner_amd.train_ops on the CPU: the definitions against 64 bits and against differences, the refusals, and what the
C entry points refuse without a GPU."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from lrbinner_amd import _lib, ae_utils, train_ops
from train_ops_ref import far_row_tolerance, gradient_like, matrices_within, norm_ref, orthogonal_ref, orthogonal_tolerance, within


def make(rows, cols, seed=0, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=gen) * 2 + 0.5).to(dtype)
    w, b = 1 + 0.3 * torch.randn(cols, generator=gen), torch.randn(cols, generator=gen)
    return x, w, b, torch.randn(rows, cols, generator=gen).to(dtype), torch.rand(rows, cols, generator=gen) >= 0.3


@pytest.mark.parametrize("block", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (17, 128), (5, 1001)])
def test_layer_norm_and_gradients(rows, cols, block):
    x, w, b, dy, keep = make(rows, cols)
    more = dict(slope=0.01, keep=keep, keep_scale=1 / 0.7) if block else {}
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = train_ops.layer_norm(*leaves, 1e-5, **more)
    got = (y, *torch.autograd.grad(y, leaves, dy))
    want, tol = norm_ref(x, w, b, 1e-5, dy, **more)
    for name, g, e, t in zip(("y", "dx", "dw", "db"), got, want, tol):
        # torch's own backward is made of other float32 operations than the formula's: four times as many
        within(g.detach(), e, 4 * t + 1e-6 * float(e.abs().max()), name)


def test_layer_norm_formula_against_differences():
    x, w, b, dy, keep = make(4, 33)
    more = dict(slope=0.2, keep=keep, keep_scale=1.5)
    (_, dx, dw, db), _ = norm_ref(x, w, b, 1e-5, dy, **more)
    gen = torch.Generator().manual_seed(9)
    for k, (t, grad) in enumerate(((x, dx), (w, dw), (b, db))):
        v, h = torch.randn(t.shape, generator=gen, dtype=torch.float64), 1e-6
        v = v * (t.abs() > 1e-3)  # not across the activation's kink
        at = [t.double() for t in (x, w, b)]

        def loss(s):
            moved = [a + s * v if i == k else a for i, a in enumerate(at)]
            u = torch.where(keep, torch.where(moved[0] > 0, moved[0], 0.2 * moved[0]) * 1.5, torch.zeros_like(moved[0]))
            c = u - u.mean(1, keepdim=True)
            return ((c / torch.sqrt(c.square().mean(1, keepdim=True) + 1e-5) * moved[1] + moved[2]) * dy.double()).sum()

        diff = (loss(h) - loss(-h)) / (2 * h)
        assert abs(float(diff - (grad * v).sum())) < 1e-6 * (1 + abs(float(diff)))


def test_what_is_dropped_does_not_count():
    x, w, b, _, keep = make(6, 40)
    keep[2] = False  # nothing is left of a row
    clean = train_ops.layer_norm(x, w, b, slope=0.01, keep=keep, keep_scale=2.0)
    x[~keep] = float("nan")
    assert torch.equal(train_ops.layer_norm(x, w, b, slope=0.01, keep=keep, keep_scale=2.0), clean)
    assert torch.equal(clean[2], b)


def test_layer_norm_module():
    m = train_ops.LayerNorm(8, slope=0.1)
    assert sorted(m.state_dict()) == ["bias", "weight"]
    x = torch.randn(3, 8)
    assert torch.equal(m(x), train_ops.layer_norm(x, m.weight, m.bias, slope=0.1))


@pytest.mark.parametrize("bad,error", [
    (dict(x=torch.zeros(2, 4, dtype=torch.float64)), TypeError),
    (dict(x=torch.zeros(2, 4, dtype=torch.long)), TypeError),
    (dict(x=torch.zeros(2, 0)), ValueError),
    (dict(x=torch.zeros(())), ValueError),
    (dict(weight=torch.ones(3)), ValueError),
    (dict(weight=torch.ones(1, 4)), ValueError),
    (dict(weight=torch.ones(4, dtype=torch.bfloat16)), TypeError),
    (dict(x=torch.zeros(2, 4, dtype=torch.bfloat16), weight=torch.ones(4, dtype=torch.bfloat16), bias=torch.ones(4)), TypeError),
    (dict(x=torch.zeros(2, 4, dtype=torch.bfloat16), weight=torch.ones(4, dtype=torch.float16)), TypeError),
    (dict(bias=torch.ones(5)), ValueError),
    (dict(keep=torch.ones(2, 3, dtype=torch.bool)), ValueError),
    (dict(keep=torch.ones(2, 4)), TypeError),
    (dict(eps=-1.0), ValueError),
    (dict(eps=float("nan")), ValueError),
    (dict(slope=float("inf")), ValueError),
    (dict(keep=torch.ones(2, 4, dtype=torch.bool), keep_scale=float("nan")), ValueError),
    (dict(weight=torch.ones(4, device="meta")), ValueError),
])
def test_layer_norm_refuses(bad, error):
    args = dict(x=torch.zeros(2, 4)) | bad
    with pytest.raises(error):
        train_ops.layer_norm(args.pop("x"), **args)


@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (7, 1), (12, 31), (40, 25), (3, 20, 33)])
def test_orthogonalize(shape):
    g = gradient_like(*shape[-2:], torch.Generator().manual_seed(1), count=shape[:-2])
    want = orthogonal_ref(g, 5, train_ops.COEFFICIENTS, 1e-7)
    matrices_within(train_ops.orthogonalize(g), want, orthogonal_tolerance(want, g, 5, train_ops.COEFFICIENTS, 1e-7))
    if min(shape[-2:]) > 1:
        # the singular vectors stay: the polynomial acts on the singular values
        u, s, vt = torch.linalg.svd((g.double() / torch.linalg.vector_norm(g.double(), dim=(-2, -1), keepdim=True)), full_matrices=False)
        a, b, c = train_ops.COEFFICIENTS
        for _ in range(5):
            s = a * s + b * s ** 3 + c * s ** 5
        assert float((u * s.unsqueeze(-2) @ vt - want).abs().max()) < 1e-9


def test_orthogonalize_edges():
    assert torch.equal(train_ops.orthogonalize(torch.zeros(4, 6)), torch.zeros(4, 6))
    assert train_ops.orthogonalize(torch.zeros(0, 6)).shape == (0, 6)
    g = torch.randn(4, 6)
    assert train_ops.orthogonalize(g, out=g) is g


@pytest.mark.parametrize("call,error", [
    (lambda: train_ops.orthogonalize(torch.zeros(4)), ValueError),
    (lambda: train_ops.orthogonalize(torch.zeros(4, 4, dtype=torch.float64)), TypeError),
    (lambda: train_ops.orthogonalize(torch.zeros(4, 4), steps=0), ValueError),
    (lambda: train_ops.orthogonalize(torch.zeros(4, 4), steps=33), ValueError),
    (lambda: train_ops.orthogonalize(torch.zeros(4, 4), steps=2.5), ValueError),
    (lambda: train_ops.orthogonalize(torch.zeros(4, 4), coefficients=(1.0, 2.0)), ValueError),
    (lambda: train_ops.orthogonalize(torch.zeros(4, 4), coefficients=(1.0, float("nan"), 0.0)), ValueError),
    (lambda: train_ops.orthogonalize(torch.zeros(4, 4), eps=-1.0), ValueError),
    (lambda: train_ops.orthogonalize(torch.zeros(4, 4), steps=2, coefficients=(6.0, -9.0, 4.0)), ValueError),
    (lambda: train_ops.orthogonalize(torch.zeros(4, 4), out=torch.zeros(4, 5)), ValueError),
    (lambda: train_ops.orthogonalize(torch.zeros(4, 4), out=torch.zeros(4, 4, dtype=torch.int32)), TypeError),
    (lambda: train_ops.orthogonalize(torch.zeros(4, 4), out=torch.zeros(4, 1).expand(4, 4)), ValueError),
    (lambda: train_ops.orthogonalize(torch.zeros(2, 3, 4, 4), out=torch.zeros(3, 2, 4, 4).transpose(0, 1)), ValueError),
])
def test_orthogonalize_refuses(call, error):
    with pytest.raises(error):
        call()


@pytest.mark.parametrize("nesterov", [False, True])
def test_muon_step(nesterov):
    gen = torch.Generator().manual_seed(3)
    shapes = [(6, 9), (9, 6), (2, 4, 5)]
    p, g, m = ([torch.randn(s, generator=gen) for s in shapes] for _ in range(3))
    want = []
    for a, b, c in zip(p, g, m):
        c = 0.9 * c.double() + 0.1 * b.double()
        u = 0.1 * b.double() + 0.9 * c if nesterov else c
        o = orthogonal_ref(u, 5, train_ops.COEFFICIENTS, 1e-7)
        want.append((a.double() * (1 - 0.1 * 0.5) - 0.1 * math.sqrt(max(1, a.shape[-2] / a.shape[-1])) * o, c))
    versions = [t._version for t in p + m]
    train_ops.muon_step(p, g, m, lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.5)
    for a, c, (wa, wc) in zip(p, m, want):
        assert float((a - wa).abs().max()) < 1e-5 and float((c - wc).abs().max()) < 1e-6
    assert all(t._version > v for t, v in zip(p + m, versions))


def test_muon_step_refuses():
    p, q = torch.zeros(4, 4), torch.zeros(4, 4)
    for args, error in [(([p], [], None), ValueError), (([p], [torch.zeros(4, 3)], None), ValueError),
                        (([p, p], [q, q], None), ValueError), (([p], [q], [p]), ValueError), (([p], [p], None), ValueError),
                        (([p], [q], [q]), ValueError), (([torch.zeros(4)], [torch.zeros(4)], None), ValueError),
                        (([p], [q.double()], None), TypeError), (([torch.zeros(1, 4).expand(4, 4)], [q], None), ValueError),
                        (([p], [torch.zeros(4, 4, device="meta")], None), ValueError)]:
        with pytest.raises(error):
            train_ops.muon_step(*args, lr=0.1)
    with pytest.raises(ValueError):
        train_ops.muon_step([p], [q], lr=float("nan"))
    with pytest.raises(ValueError):
        train_ops.muon_step([p], [q], lr=0.1, momentum=float("inf"))
    train_ops.muon_step([], [], lr=0.1)


def test_muon_optimizer(tmp_path):
    torch.manual_seed(0)
    w = torch.nn.Parameter(torch.randn(6, 4, dtype=torch.bfloat16))
    opt = train_ops.Muon([w], lr=0.1, weight_decay=0.1)
    w.grad = torch.randn(6, 4, dtype=torch.bfloat16)
    opt.step()
    kept = opt.state[w]["momentum"].clone()
    assert kept.dtype == torch.float32
    again = train_ops.Muon([w], lr=0.5)
    again.load_state_dict(opt.state_dict())
    assert torch.equal(again.state[w]["momentum"], kept) and again.state[w]["momentum"].dtype == torch.float32
    assert again.param_groups[0]["lr"] == 0.1
    with pytest.raises(ValueError):
        train_ops.Muon([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(ValueError):
        train_ops.Muon([w], momentum=1.0)
    with pytest.raises(TypeError):
        train_ops.Muon([torch.nn.Parameter(torch.zeros(4, 4, dtype=torch.float64))])
    live = train_ops.Muon([w])
    with pytest.raises(ValueError):
        live.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4))]})
    assert len(live.param_groups) == 1


def test_c_entry_points_refuse_before_they_touch_a_device():
    L = _lib.lib()
    buf = C.create_string_buffer(64)
    p = C.addressof(buf)
    fwd = lambda x_type=0, w_type=0, rows=1, cols=4, x=p, y=p, mean=None, rstd=None: L.lrb_layer_norm_fwd_dev(
        0, None, x_type, w_type, rows, cols, x, cols, None, None, 1e-5, 1.0, None, 1.0, y, mean, rstd)
    assert fwd(rows=0) == 0
    for bad in (dict(x_type=3), dict(x_type=-1), dict(w_type=1), dict(x_type=1, w_type=2), dict(cols=0), dict(cols=1 << 40),
                dict(rows=1 << 50), dict(x=None), dict(y=None), dict(mean=p)):
        assert fwd(**bad) == 1, bad
    assert L.lrb_layer_norm_bwd_ws_bytes(7, 4, 4) == 0
    assert L.lrb_layer_norm_bwd_dev(0, None, 0, 0, 1, 4, p, 4, p, 4, None, p, p, 1.0, None, 1.0, p, p, None, p, 0) == 1  # no room
    assert L.lrb_layer_norm_bwd_dev(0, None, 0, 0, 1, 4, None, 4, p, 4, None, p, p, 1.0, None, 1.0, p, None, None, None, 0) == 1

    def item(rows=300, cols=300, count=1, p_ptr=p, p_type=0, g_type=0, m=0, m_type=0):
        return C.create_string_buffer(train_ops._ITEM.pack(p_ptr, p, m, 90000, 300, 1, 90000, 300, 1, 0, 0, 0, count, rows, cols, p_type, g_type, m_type, 1.0, 0.0, 0))

    step = lambda it, n=1, steps=5, eps=0.0, ws=p, ws_bytes=64: L.lrb_muon_dev(0, None, it, n, 0.9, 1, steps, 1.5, -0.5, 0.0, eps, ws, ws_bytes)
    assert step(None, 0) == 0 and step(item(rows=0)) == 0 and step(item(count=0)) == 0
    for it, more in ((item(rows=-1), {}), (item(cols=1 << 25), {}), (item(rows=1 << 20, cols=1 << 20), {}), (item(p_ptr=0), {}),
                     (item(p_type=3), {}), (item(g_type=-1), {}), (item(m=p, m_type=9), {}), (item(), dict(steps=0)),
                     (item(), dict(steps=33)), (item(), dict(eps=-1.0)), (item(), dict(n=-1)), (None, {}), (item(), dict(ws=None)),
                     (item(), dict(ws_bytes=64))):
        assert step(it, **more) == 1, more
    assert L.lrb_muon_ws_bytes(item(), 1) >= 16 * 300 * 300 and L.lrb_muon_ws_bytes(item(rows=4, cols=4), 1) == 0  # (in LDS)
    assert L.lrb_muon_dev(0, None, item(), 1, 0.9, 1, 2, 6.0, -9.0, 4.0, 0.0, p, 1 << 30) == 1       # diverges
    assert L.lrb_muon_dev(0, None, item(), 1, 0.9, 1, 2, float("nan"), 1.0, 1.0, 0.0, p, 1 << 30) == 1


def test_muon_bound():
    bound = lambda steps, c: _lib.lib().lrb_muon_bound(steps, *c)
    for c in (train_ops.COEFFICIENTS, (1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (0.0, 0.0, 0.0), (-1.2, 0.3, 0.1), (1.0, 1.0, 0.0)):
        s = torch.linspace(0, 1, 100001, dtype=torch.float64)
        most = 1.0
        for _ in range(4):
            # of the interval up to the largest value so far, as the bound is made
            s = torch.linspace(0, float((c[0] * s + c[1] * s ** 3 + c[2] * s ** 5).abs().max()), 100001, dtype=torch.float64)
            most = max(most, float(s[-1]))
        assert abs(bound(4, c) - most) < 1e-6 * most, c


# ---- the network that uses them -------------------------------------------------------------------

def test_vae_with_layer_norm_and_muon(tmp_path):
    torch.manual_seed(0)
    data = torch.rand(600, 42)
    vae = ae_utils.VAE(10, 32, latent_dims=4, hidden_layers=[24, 16], norm="layer")
    assert [k for k in vae.state_dict() if "norms.0" in k] == ["encodernorms.0.weight", "encodernorms.0.bias",
                                                                "decodernorms.0.weight", "decodernorms.0.bias"]
    before = {k: v.clone() for k, v in vae.state_dict().items()}
    vae.trainmodel(data, nepochs=3, batchsteps=[1], batch_size=64, optimizer="muon", save_path=str(tmp_path / "m.pt"))
    after = vae.state_dict()
    assert all(bool(torch.isfinite(v).all()) and not torch.equal(v, before[k]) for k, v in after.items())
    assert torch.load(str(tmp_path / "m.pt"), weights_only=True)["norm"] == "layer"
    mu = vae.encode(data, chunk=100)
    # rows do not depend on each other
    assert mu.shape == (600, 4) and abs(mu[17:18] - vae.encode(data[17:18])).max() < 1e-5
    # what the eval pass computes is the module's formula
    x = data.double()
    for lin, norm in zip(vae.encoderlayers, vae.encodernorms):
        x = torch.nn.functional.leaky_relu(x @ lin.weight.double().T + lin.bias.double(), 0.01)
        x = (x - x.mean(1, keepdim=True)) / torch.sqrt(x.var(1, unbiased=False, keepdim=True) + 1e-5) * norm.weight.double() + norm.bias.double()
    assert float((x @ vae.mu.weight.double().T + vae.mu.bias.double() - torch.from_numpy(mu)).detach().abs().max()) < 1e-4


def test_vae_choices():
    with pytest.raises(ValueError, match="norm"):
        ae_utils.VAE(10, 32, norm="group")
    vae = ae_utils.VAE(10, 32, latent_dims=2, hidden_layers=[8])
    with pytest.raises(ValueError, match="optimizer"):
        vae.trainmodel(torch.rand(10, 42), nepochs=1, optimizer="sgd")


def test_vae_encode_takes_the_choices_from_the_environment(tmp_path, monkeypatch):
    (tmp_path / "profiles").mkdir()
    rng = np.random.default_rng(0)
    np.save(tmp_path / "profiles" / "com_profs.npy", rng.random((1100, 32)))
    np.save(tmp_path / "profiles" / "cov_profs.npy", rng.random((1100, 10)))
    monkeypatch.setenv("LRB_VAE_NORM", "layer")
    monkeypatch.setenv("LRB_VAE_OPTIMIZER", "muon")
    ae_utils.vae_encode(str(tmp_path), 3, [8, 8], 2, None, False)
    assert np.load(tmp_path / "latent.npy").shape == (1100, 3)
    assert torch.load(str(tmp_path / "model.pt"), weights_only=True)["norm"] == "layer"
    monkeypatch.setenv("LRB_VAE_OPTIMIZER", "none")
    with pytest.raises(ValueError, match="optimizer"):
        ae_utils.vae_encode(str(tmp_path), 3, [8, 8], 2, None, False)


def test_orthogonalize_at_the_ends_of_the_range():
    g = gradient_like(8, 12, torch.Generator().manual_seed(1))
    huge = g / g.abs().max() * 3e38  # its norm is beyond float32
    exact = orthogonal_ref(huge, 3, (1.5, -0.5, 0.0), 1e-7)
    matrices_within(train_ops.orthogonalize(huge, 3, (1.5, -0.5, 0.0)), exact, orthogonal_tolerance(exact, huge, 3, (1.5, -0.5, 0.0), 1e-7))
    assert not train_ops.orthogonalize(torch.zeros(3, 4), eps=0.0).any()
    with pytest.raises(ValueError):
        train_ops.orthogonalize(g, coefficients=(1e39, 0.0, 0.0))  # finite, but not in float32


def test_views_with_their_sign_turned():
    g = gradient_like(6, 9, torch.Generator().manual_seed(2))
    turned = torch._neg_view(g)
    assert turned.is_neg() and torch.equal(train_ops.orthogonalize(turned), train_ops.orthogonalize(-g))
    with pytest.raises(ValueError):
        train_ops.orthogonalize(g, out=torch._neg_view(torch.zeros(6, 9)))
    with pytest.raises(ValueError):
        train_ops.muon_step([torch._neg_view(torch.zeros(6, 9))], [g], lr=0.1)


def _four_axes(device):
    """Gradients of one shape whose leading axes cannot be flattened without a copy, and the same ones packed."""
    gen = torch.Generator().manual_seed(6)
    grads = [gradient_like(20, 30, gen, device, (3, 4)).transpose(0, 1) for _ in range(4)]
    grads += [gradient_like(20, 30, gen, device, (4, 1)).expand(4, 3, 20, 30) for _ in range(2)]
    return grads, [g.contiguous() for g in grads]


def test_muon_items_point_at_memory_that_lives():
    grads, packed = _four_axes("cpu")
    params = [torch.zeros(4, 3, 20, 30) for _ in grads]
    items, held = train_ops._muon_items(params, grads, [None] * len(grads), 0.1, 1.0, None)
    noise = [torch.full((12, 20, 30), 7.0) for _ in range(12)]  # takes what was given back
    for item, g in zip(items, packed):
        _, at, _, *strides = train_ops._ITEM.unpack(item)[:9]
        assert strides[3:6] == [600, 30, 1]
        there = np.ctypeslib.as_array((C.c_float * g.numel()).from_address(at))
        assert np.array_equal(there, g.numpy().ravel())
    del noise, held


def test_rows_far_from_zero():
    for cols in (41, 61, 1000, 4095):
        for value in (1.0, 0.1, 1e3, 1e5, -3e34, 3e38):
            x, w, b, _, _ = make(3, cols)
            x[1] = value  # no variance: what is left is the bias
            assert torch.equal(train_ops.layer_norm(x, w, b)[1], b)
    x, w, b, _, _ = make(5, 700)
    x += torch.tensor([[0.0], [1e3], [-1e4], [1e5], [3e6]])
    y = train_ops.layer_norm(x, w, b)
    c = x.double() - x.double().mean(1, keepdim=True)
    want = c / torch.sqrt(c.square().mean(1, keepdim=True) + 1e-5) * w.double() + b.double()
    within(y, want, far_row_tolerance(x, w, 1e-5) + 2.0 ** -24 * want.abs())


def test_what_torch_would_not_see_is_refused():
    """(What a call on the GPU asks before its launch; on the CPU torch sees everything.)"""
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.randn(3, 4)

    def asks(v):
        train_ops._refuse_unseen("layer_norm", v, None)
        return v + 1

    asks(x)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(asks, (x,))
    for more in ({}, dict(tracing_mode="fake"), dict(tracing_mode="symbolic"), dict(pre_dispatch=True)):
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(asks, **more)(x)
    with forward_ad.dual_level():
        asks(x)
        with pytest.raises(RuntimeError, match="forward-mode"):
            asks(forward_ad.make_dual(x, torch.ones_like(x)))
    asks(x)
    # the CPU's forms can be traced, and have forward-mode gradients
    m = train_ops.LayerNorm(4, slope=0.1)
    with torch.no_grad():
        traced, other = torch.jit.trace(m, (x,)), torch.randn(3, 4)
        assert torch.allclose(traced(other), m(other)) and torch.allclose(make_fx(m)(x)(other), m(other))
    with forward_ad.dual_level():
        assert forward_ad.unpack_dual(m(forward_ad.make_dual(x, torch.ones_like(x)))).tangent is not None


def test_slope_0_is_a_relu():
    x, w, b, dy, keep = make(5, 40)
    x[1, 3], x[2, 7], x[3, 9] = -math.inf, math.nan, -0.0
    y = train_ops.layer_norm(x, w, b, slope=0.0)
    want = train_ops.layer_norm(torch.relu(x), w, b)
    assert torch.equal(y.nan_to_num(77.0), want.nan_to_num(77.0))
    assert bool(y[2].isnan().all()) and bool(torch.isfinite(y[[0, 1, 3, 4]]).all())


def test_coefficients_under_which_roundings_grow_are_refused():
    g = torch.outer(torch.arange(1.0, 5.0), torch.arange(1.0, 7.0))
    unit = g / g.norm()  # of rank one: its singular value is 1, which x^5 keeps
    assert float((train_ops.orthogonalize(g, steps=3, coefficients=(0.0, 0.0, 1.0)) - unit).abs().max()) < 2e-5
    assert _lib.lib().lrb_muon_bound(3, 0.0, 0.0, 1.0) == 1.0
    for steps, c in ((8, (0.0, 0.0, 1.0)), (32, (0.0, 0.0, -1.0)), (12, (0.5, 0.0, 0.5)), (20, (0.0, 1.0, 0.0))):
        assert _lib.lib().lrb_muon_bound(steps, *c) > 64.0
        with pytest.raises(ValueError, match="grow beyond"):
            train_ops.orthogonalize(g, steps=steps, coefficients=c)
    for steps, c in ((32, train_ops.COEFFICIENTS), (32, (1.5, -0.5, 0.0)), (32, (15 / 8, -10 / 8, 3 / 8)), (32, (2.0, -1.5, 0.5)),
                     (32, (1.0, 0.0, 0.0))):
        assert _lib.lib().lrb_muon_bound(steps, *c) < 1.5


def test_the_largest_sizes():
    L = _lib.lib()
    for rows, cols, fits in ((46336, 46336, True), (46340, 46340, False), (448, 1 << 22, True), (500, 1 << 22, False), (1, 1 << 22, True),
                             (1, (1 << 22) + 1, False), ((1 << 22) + 1, 1, False), (1 << 22, 511, False), (1 << 22, 448, True),
                             (65536, 32704, True), (65536, 32705, False)):
        item = C.create_string_buffer(train_ops._ITEM.pack(64, 64, 0, 0, cols, 1, 0, cols, 1, 0, 0, 0, 1, rows, cols, 0, 0, 0, 1.0, 0.0, 0))
        assert (L.lrb_muon_ws_bytes(item, 1) > 0) == fits, (rows, cols)
        t = torch.empty(rows, cols, device="meta")
        if fits:
            train_ops._check_size(t, "g")
        else:
            assert L.lrb_muon_dev(0, None, item, 1, 0.0, 0, 5, 1.5, -0.5, 0.0, 0.0, 256, 1 << 60) == 1
            with pytest.raises(ValueError, match="2.31"):
                train_ops._check_size(t, "g")


def test_the_workspace_is_what_is_said():
    L = _lib.lib()

    def asks(*shapes):
        items = b"".join(train_ops._ITEM.pack(64, 64, 0, r * c, c, 1, r * c, c, 1, 0, 0, 0, n, r, c, 0, 0, 0, 1.0, 0.0, 0) for n, r, c in shapes)
        return L.lrb_muon_ws_bytes(C.create_string_buffer(items, len(items)), len(shapes))

    def said(n, rows, cols):
        s, l = sorted(((rows + 63) // 64 * 64, (cols + 63) // 64 * 64))
        return 4 * n * s * (5 * l + 3 * s)

    for shapes in ([(1, 4096, 4096)], [(1, 511, 1025)], [(8, 1024, 2048)], [(1, 16384, 16384)], [(1, 2048, 2048), (1, 5461, 2048), (2, 300, 70)]):
        most = sum(said(*s) for s in shapes)
        assert most <= asks(*shapes) <= most + (64 << 20) + (1 << 20) + most // 64, shapes
    assert (2 << 30) < asks((1000, 1024, 1024)) <= (4 << 30) + (128 << 20)
    for shape in ((128, 208), (320, 96), (64, 512), (1024, 32), (1, 1)):
        assert asks((3, *shape)) == 0


def test_a_captured_training_has_leaves_of_its_own():
    vae = ae_utils.VAE(10, 32, latent_dims=3, hidden_layers=[8], norm="layer")
    held = list(vae.parameters())
    x = torch.rand(5, 42)
    recon, mu, sigma = vae(x)  # a graph of the caller's, alive
    node = lambda p: torch.autograd.graph.get_gradient_edge(p).node
    before = [node(p) for p in held]
    with pytest.raises(KeyError), vae._fresh_leaves():
        fresh = list(vae.parameters())
        assert len(fresh) == len(held) and not any(a is b for a, b in zip(fresh, held))
        assert all(a.data_ptr() == b.data_ptr() and a.requires_grad for a, b in zip(fresh, held))
        assert not any(node(p) in before for p in fresh)
        vae.calc_loss(x, *vae(x))[0].backward()
        assert all(p.grad is not None for p in fresh) and all(p.grad is None for p in held)
        with torch.no_grad():
            vae.outputlayer.weight.zero_()
        raise KeyError
    assert all(a is b for a, b in zip(vae.parameters(), held)) and not bool(vae.outputlayer.weight.any())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        recon.sum().backward()  # the caller's graph knows that its weights have changed


def test_a_state_without_a_momentum_is_loaded():
    """As a refused first step left it."""
    w = torch.nn.Parameter(torch.ones(3, 4))
    opt = train_ops.Muon([w])
    opt.state[w]
    saved = opt.state_dict()
    again = train_ops.Muon([w])
    again.load_state_dict(saved)
    w.grad = torch.randn(3, 4)
    again.step()
    assert again.state[w]["momentum"].shape == (3, 4)


def test_a_list_with_a_weight_that_is_too_large_is_refused():
    small, wide = torch.zeros(3, 4), torch.empty(1, (1 << 22) + 1)
    with pytest.raises(ValueError, match="params: sides up to"):
        train_ops._muon_items([small, wide], [small, wide], [None, None], 0.1, 1.0, None)
