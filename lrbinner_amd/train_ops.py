"""Operators of a network's training on torch tensors: layer normalisation (K9) and the orthogonalised update (K10).

``layer_norm`` / ``LayerNorm`` normalise the rows of a tensor, with the LeakyReLU and the dropout that stand before a norm
in this package's blocks folded in, and give the gradients of input, weight and bias.  ``orthogonalize`` moves the
singular values of a matrix towards 1 by a polynomial iteration, ``muon_step`` takes an optimiser's step with it for a list
of weights (momentum, iteration and update in shared launches), and ``Muon`` is that as a ``torch.optim.Optimizer``.

On the GPU the arithmetic is csrc/lrb_norm.hip and csrc/lrb_muon.hip behind the C ABI of include/lrb_hip.h; calls go to
torch's current stream of the tensors' device, their workspace comes from torch's allocator (so calls may be captured in a
HIP graph; a captured backward pass, as any of torch's, wants leaves that no living eager graph holds), and there is no
fallback where the library is missing.  Launches on addresses are nothing that torch.jit.trace, make_fx or forward-mode
gradients could follow: under these a call raises RuntimeError.  On CPU tensors the same definitions run as torch
operations, as the network itself does without ``--cuda``.

Float32, bfloat16 and float16; what is summed is summed in float32 or more, and results are rounded once."""
import ctypes as C
import math
import struct

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import call, check

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # LRB_F32, LRB_BF16, LRB_F16
#: of the odd quintic a x + b x^3 + c x^5 that ``orthogonalize`` iterates on the singular values
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


# hipStream_t of torch's current stream on a device, by its index (a call of torch.cuda.current_stream costs a small
# operator as much as its launch)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


_tracing_state, _dispatch_modes = torch._C._get_tracing_state, torch._C._len_torch_dispatch_stack
_key_included, _PRE_DISPATCH = torch._C._dispatch_tls_is_dispatch_key_included, torch._C.DispatchKey.PreDispatch


def _has_proxy_mode():
    """Whether make_fx or torch.export is at work.  (Asked only where some mode is: its module takes long to import.)"""
    from torch.fx.experimental.proxy_tensor import get_proxy_mode
    return get_proxy_mode() is not None


def _refuse_unseen(name, *tensors):
    """Raises where torch records or differentiates, by the operations it sees, what is about to be launched unseen."""
    if torch.compiler.is_dynamo_compiling():  # torch.compile steps aside for the launch by itself
        return
    if _tracing_state() is not None or (_dispatch_modes() or _key_included(_PRE_DISPATCH)) and _has_proxy_mode():
        raise RuntimeError(f"{name}: a call on the GPU cannot be traced (its kernels would not be in the trace)")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{name}: forward-mode gradients are not given on the GPU")


def _known_type(t, name):
    if t.dtype not in _TYPES:
        raise TypeError(f"{name}: float32, bfloat16 or float16 is wanted, not {t.dtype}")


# ---- layer normalisation ----------------------------------------------------------------------

def _rows(t, cols):
    """t as rows x cols with the elements of a row side by side (a copy only where its strides allow no such view)."""
    t = t.resolve_neg().reshape(-1, cols)
    return t if cols == 1 or t.stride(1) == 1 else t.contiguous()


def _address(t):
    return None if t is None else t.data_ptr()


def _packed(t):
    return t if t is None or t.is_contiguous() and not t.is_neg() else t.resolve_neg().contiguous()


def _ln_forward(x, weight, bias, keep, eps, slope, keep_scale, stats):
    """y, and with `stats` the float32 [2, rows] of means and 1 / deviations that the backward pass takes."""
    cols = x.shape[-1]
    rows = x.numel() // cols
    dense = x.is_contiguous() and not x.is_neg()
    y = torch.empty_like(x) if dense else torch.empty_like(x, memory_format=torch.contiguous_format)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if stats else None
    if rows:
        stride = cols
        if not dense:
            x = _rows(x, cols)
            stride = x.stride(0)
        weight, bias, keep = _packed(weight), _packed(bias), _packed(keep)
        ref = weight if weight is not None else bias
        at = _address(stats)
        index = x.device.index
        rc = _lib.lib().lrb_layer_norm_fwd_dev(
            index, _stream(index), _TYPES[x.dtype], 0 if ref is None else _TYPES[ref.dtype], rows, cols, x.data_ptr(), stride,
            _address(weight), _address(bias), eps, slope, _address(keep), keep_scale, y.data_ptr(), at, at and at + 4 * rows)
        if rc:
            check("lrb_layer_norm_fwd_dev", rc)
    return y, stats


def _ln_backward(ctx, dy):
    x, weight, keep, stats = ctx.saved_tensors
    bias_type, slope, keep_scale = ctx.more
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    cols = x.shape[-1]
    rows = x.numel() // cols
    device = x.device
    w_type, dx, dw, db = bias_type, None, None, None
    weight, keep = _packed(weight), _packed(keep)
    dense = x.is_contiguous() and not x.is_neg()
    if need_x:
        dx = torch.empty_like(x) if dense else torch.empty_like(x, memory_format=torch.contiguous_format)
    if weight is not None:
        w_type = weight.dtype
        dw = torch.empty_like(weight) if need_w else None
        db = torch.empty_like(weight) if need_b else None
    elif need_b:
        db = torch.empty(cols, dtype=w_type, device=device)
    lib = _lib.lib()
    x_type = _TYPES[x.dtype]
    ws, ws_bytes = None, 0
    if need_w or need_b:
        ws_bytes = lib.lrb_layer_norm_bwd_ws_bytes(x_type, rows, cols)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    x_stride = dy_stride = cols
    if not dense:
        x = _rows(x, cols)
        x_stride = x.stride(0)
    if not dy.is_contiguous() or dy.is_neg():
        dy = _rows(dy, cols)
        dy_stride = dy.stride(0)
    index, at = device.index, stats.data_ptr() or None
    rc = lib.lrb_layer_norm_bwd_dev(
        index, _stream(index), x_type, 0 if w_type is None else _TYPES[w_type], rows, cols, x.data_ptr() or None, x_stride,
        dy.data_ptr() or None, dy_stride, _address(weight), at, at and at + 4 * rows, slope, _address(keep) or None, keep_scale,
        _address(dx) or None, _address(dw), _address(db), _address(ws), ws_bytes)
    if rc:
        check("lrb_layer_norm_bwd_dev", rc)
    return dx, dw, db, None, None, None, None


class _Once(torch.autograd.Function):
    """The first `count` tensors, as functions of all of them that cannot be differentiated."""

    @staticmethod
    def forward(ctx, count, *tensors):
        return tensors[:count]

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("layer_norm: second derivatives are not given on the GPU")


def _ln_backward_of_a_graph(ctx, dy):
    # (torch's once_differentiable looks at dy alone: the gradient of a sum, say, would pass for a constant)
    with torch.no_grad():
        grads = _ln_backward(ctx, dy)
    given = [g for g in grads if g is not None]
    given = iter(_Once.apply(len(given), *given, dy, *ctx.saved_tensors[:2]))
    return tuple(None if g is None else next(given) for g in grads)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, keep, eps, slope, keep_scale):
        y, stats = _ln_forward(x, weight, bias, keep, eps, slope, keep_scale, True)
        ctx.save_for_backward(x, weight, keep, stats)
        ctx.more = None if bias is None else bias.dtype, slope, keep_scale
        return y

    @staticmethod
    def backward(ctx, dy):
        # gradients are enabled here only where a graph of the backward pass is asked for
        return _ln_backward_of_a_graph(ctx, dy) if torch.is_grad_enabled() else _ln_backward(ctx, dy)


def _ln_plain(x, weight, bias, keep, eps, slope, keep_scale):
    u = x.float()
    if keep is not None or slope != 1.0:
        u = torch.relu(u) if slope == 0.0 else torch.where(u > 0, u, slope * u)  # (0 times -inf is no 0)
        if keep is not None:
            u = torch.where(keep.bool(), u * keep_scale, torch.zeros_like(u))
    centred = u - (u / u.shape[-1]).sum(-1, keepdim=True)  # (the sum of u may be beyond float32)
    centred = centred - centred.mean(-1, keepdim=True)  # what rounding has left out of the mean
    y = centred / torch.sqrt((centred * centred).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.float()
    if bias is not None:
        y = y + bias.float()
    return y.to(x.dtype)


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, slope=1.0, keep=None, keep_scale=1.0):
    """(u - mean(u)) / sqrt(var(u) + eps) * weight + bias over the last axis, in x's type, with gradients of x, weight and bias.

    u is x, or with ``slope`` (of a LeakyReLU; 0 a ReLU) or ``keep`` (bool or uint8, of x's shape, a dropout's draw)
    keep * keep_scale * leaky_relu(x); what is dropped counts as 0 whatever it holds.  ``weight`` and ``bias``: one element a
    column, float32 or of x's type (both alike), or None.  x may have any leading axes and strides; a copy is made only
    where the elements of a row are not side by side, or the rows not evenly spaced.  The statistics are float32.  On the GPU the
    gradients may be asked for with ``create_graph``, but not differentiated: that raises RuntimeError."""
    dtype, shape, device = x.dtype, x.shape, x.device
    if dtype not in _TYPES:
        _known_type(x, "x")
    if not shape or shape[-1] < 1:
        raise ValueError(f"x: at least one column is wanted, not shape {tuple(shape)}")
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps: {eps}")
    if not (math.isfinite(slope) and math.isfinite(keep_scale)):
        raise ValueError(f"slope {slope}, keep_scale {keep_scale}: finite numbers are wanted")
    cols = shape[-1]
    grad = x.requires_grad
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if t.shape != (cols,):
            raise ValueError(f"{name}: shape ({cols},) is wanted, not {tuple(t.shape)}")
        if t.dtype is not torch.float32 and t.dtype is not dtype:
            raise TypeError(f"{name}: float32 or {dtype} is wanted, not {t.dtype}")
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, x on {device}")
        grad = grad or t.requires_grad
    if weight is not None and bias is not None and weight.dtype is not bias.dtype:
        raise TypeError(f"weight and bias: one type is wanted, not {weight.dtype} and {bias.dtype}")
    if keep is not None:
        if keep.shape != shape:
            raise ValueError(f"keep: shape {tuple(shape)} is wanted, not {tuple(keep.shape)}")
        if keep.dtype is not torch.bool and keep.dtype is not torch.uint8:
            raise TypeError(f"keep: bool or uint8 is wanted, not {keep.dtype}")
        if keep.device != device:
            raise ValueError(f"keep is on {keep.device}, x on {device}")
    else:
        keep_scale = 1.0
    if not x.is_cuda:
        return _ln_plain(x, weight, bias, keep, eps, slope, keep_scale)
    _refuse_unseen("layer_norm", x, weight, bias)
    if grad and torch.is_grad_enabled():
        return _LayerNorm.apply(x, weight, bias, keep, eps, slope, keep_scale)
    return _ln_forward(x, weight, bias, keep, eps, slope, keep_scale, False)[0]


class LayerNorm(torch.nn.Module):
    """``layer_norm`` with a weight (ones) and a bias (zeros) of its own; ``slope``: of the LeakyReLU that stands before it."""

    def __init__(self, cols, eps=1e-5, *, slope=1.0, device=None, dtype=None):
        super().__init__()
        self.eps, self.slope = eps, slope
        self.weight = torch.nn.Parameter(torch.ones(cols, device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(cols, device=device, dtype=dtype))

    def forward(self, x, keep=None, keep_scale=1.0):
        return layer_norm(x, self.weight, self.bias, self.eps, slope=self.slope, keep=keep, keep_scale=keep_scale)

    def extra_repr(self):
        return f"{self.weight.numel()}, eps={self.eps}, slope={self.slope}"


# ---- the orthogonalised update ------------------------------------------------------------------

_ITEM = struct.Struct("=3Q9q3q3i2fi")  # lrb_muon_item
_DIVERGED = 64.0                       # LRB_MUON_DIVERGED


def _check_size(t, name):
    """What lrb_muon_dev takes (the lengths of its kernels' indices)."""
    rows, cols = t.shape[-2:]
    if rows > 1 << 22 or cols > 1 << 22 or (rows + 63) // 64 * 64 * ((cols + 63) // 64 * 64) >= 1 << 31:
        raise ValueError(f"{name}: sides up to 2^22, and fewer than 2^31 elements with both rounded up to multiples of 64 are wanted "
                         f"on the GPU, not {rows} x {cols}")


def _stack(t, name):
    """t as matrices x rows x columns, without a copy."""
    if t.dim() == 2:
        return t.unsqueeze(0)
    if t.dim() == 3:
        return t
    try:
        return t.view(-1, t.shape[-2], t.shape[-1])
    except RuntimeError:
        raise ValueError(f"{name}: the leading axes of shape {tuple(t.shape)}, strides {t.stride()} are not evenly spaced") from None


def _extent(t):
    """The bytes from the first to behind the last element of t, which has some."""
    return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _written(t, name):
    if t.is_neg():
        raise ValueError(f"{name} is written, but it is a view with its sign turned")
    if any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
        raise ValueError(f"{name} is written, but several of its elements share their memory (strides {t.stride()})")


def _check_iteration(steps, coefficients, eps):
    if int(steps) != steps or not 1 <= steps <= 32:
        raise ValueError(f"steps: 1 to 32 is wanted, not {steps}")
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise ValueError(f"coefficients: three finite numbers are wanted, not {coefficients}")
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps: {eps}")
    if not _lib.lib().lrb_muon_bound(int(steps), *coefficients) <= _DIVERGED:
        raise ValueError(f"coefficients {tuple(coefficients)}: a singular value may grow beyond {_DIVERGED:g} in {steps} steps")


def _muon_call(device, items, momentum, nesterov, steps, coefficients, eps):
    lib = _lib.lib()
    raw = C.create_string_buffer(b"".join(items), _ITEM.size * len(items))
    ws_bytes = lib.lrb_muon_ws_bytes(raw, len(items))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    a, b, c = coefficients
    check("lrb_muon_dev", lib.lrb_muon_dev(device.index, _stream(device.index), raw, len(items), momentum, 1 if nesterov else 0, int(steps),
                                           a, b, c, eps, ws.data_ptr() if ws_bytes else None, ws_bytes))


def _muon_items(params, grads, momenta, lr, decay, scale):
    """The C ABI's items, and the tensors whose memory they point at: these have to live until the launches are made."""
    items, held = [], []
    for p, g, m in zip(params, grads, momenta):
        if not p.numel():
            continue
        p3, m3 = _stack(p, "params"), None if m is None else _stack(m, "momenta")
        g3 = g.reshape(-1, *g.shape[-2:]) if g.dim() > 3 else _stack(g, "grads")  # a copy where the leading axes ask for one
        held += (p3, g3, m3)
        count, rows, cols = p3.shape
        if rows * cols > 1 << 22:  # (a smaller one fits whatever its sides)
            _check_size(p, "params")
        by = math.sqrt(max(1.0, rows / cols)) if scale is None else scale
        items.append(_ITEM.pack(p3.data_ptr(), g3.data_ptr(), 0 if m is None else m3.data_ptr(), *p3.stride(), *g3.stride(),
                                *((0, 0, 0) if m is None else m3.stride()), count, rows, cols, _TYPES[p.dtype], _TYPES[g.dtype],
                                0 if m is None else _TYPES[m.dtype], -lr * by, decay, 0))
    return items, held


def _orthogonal_plain(u, steps, coefficients, eps):
    """In float32, whatever u's type; u: [..., rows, columns]."""
    a, b, c = coefficients
    x = u.float()
    turned = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2) if turned else x
    norm = torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True, dtype=torch.float64).clamp_min(eps)
    x = (x.double() / (norm + (norm == 0.0))).float()  # of float32's largest numbers the norm is beyond its range
    for _ in range(int(steps)):
        gram = x @ x.transpose(-1, -2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-1, -2) if turned else x


@torch.no_grad()
def orthogonalize(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7, out=None):
    """g / max(|g|_F, eps), then ``steps`` times X <- a X + (b A + c A^2) X with A = X X^T (of a tall matrix X^T X): the
    singular vectors stay, the singular values go towards 1 (with the default coefficients into about 0.7 to 1.2).
    Coefficients under which a singular value from [0, 1], or one that rounding has put above 1 by 1 / 512, may grow beyond 64 on
    the way are refused.

    g: [..., rows, columns], any strides; each matrix by itself; one that holds an infinity or a NaN becomes NaN, one of
    zeros stays.  ``out``: a tensor of g's shape, g itself among them (by default a new one of g's type).  The products are
    as exact as float32 ones for every type of g.  No gradient: an update is not differentiated.  On the GPU a matrix that does not fit
    a workgroup's LDS (128 x 208, 32 x 1024 ...) takes a workspace of 8 times its float32 size if it is square, 5 times if it is
    long; the matrices of a stack up to 4 GiB at a time."""
    _known_type(g, "g")
    if g.dim() < 2:
        raise ValueError(f"g: a matrix is wanted, not shape {tuple(g.shape)}")
    _check_iteration(steps, coefficients, eps)
    if out is None:
        out = torch.empty(g.shape, dtype=g.dtype, device=g.device)
    else:
        _known_type(out, "out")
        if out.shape != g.shape or out.device != g.device:
            raise ValueError(f"out: shape {tuple(g.shape)} on {g.device} is wanted, not {tuple(out.shape)} on {out.device}")
        _written(out, "out")
        if g.dim() > 3:
            _stack(out, "out")
    if g.numel() == 0:
        return out
    g = g.resolve_neg()
    if not g.is_cuda:
        return out.copy_(_orthogonal_plain(g, steps, coefficients, eps))
    _refuse_unseen("orthogonalize", g, out)
    _check_size(g, "g")
    if out.data_ptr() != g.data_ptr() or out.stride() != g.stride() or out.dtype != g.dtype:
        (g0, g1), (o0, o1) = _extent(g), _extent(out)
        if g0 < o1 and o0 < g1:  # a matrix of out may lie over another matrix of g
            g = g.clone()
    g3 = g.reshape(-1, *g.shape[-2:]) if g.dim() > 3 else _stack(g, "g")
    o3 = _stack(out, "out")
    item = _ITEM.pack(o3.data_ptr(), g3.data_ptr(), 0, *o3.stride(), *g3.stride(), 0, 0, 0, *g3.shape,
                      _TYPES[out.dtype], _TYPES[g.dtype], 0, 1.0, 0.0, 0)
    _muon_call(g.device, [item], 0.0, False, steps, coefficients, eps)
    torch.autograd.graph.increment_version(out)
    return out


@torch.no_grad()
def muon_step(params, grads, momenta=None, *, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
              coefficients=COEFFICIENTS, eps=1e-7, scale=None):
    """One step of the orthogonalised momentum update on a list of weights, in place:

        m <- momentum m + (1 - momentum) g;  u = (1 - momentum) g + momentum m  (nesterov; else m; g without ``momenta``)
        p <- (1 - lr weight_decay) p - lr scale orthogonalize(u)

    params, grads, momenta: lists of [..., rows, columns] of one device, each of its own type and strides (momenta best in
    float32); leading axes are a stack of weights.  ``scale``: None for sqrt(max(1, rows / columns)), or a number.  The
    weights of a list share their launches, so one call for all of a network's is best.  No written tensor may overlap
    another tensor of the call."""
    params, grads = list(params), [g.resolve_neg() for g in grads]
    momenta = [None] * len(params) if momenta is None else list(momenta)
    if not len(params) == len(grads) == len(momenta):
        raise ValueError(f"{len(params)} params, {len(grads)} grads and {len(momenta)} momenta")
    _check_iteration(steps, coefficients, eps)
    for v, name in ((lr, "lr"), (momentum, "momentum"), (weight_decay, "weight_decay"), (0.0 if scale is None else scale, "scale")):
        if not math.isfinite(v):
            raise ValueError(f"{name}: {v}")
    if not params:
        return
    device, seen = params[0].device, set()
    for p, g, m in zip(params, grads, momenta):
        for t, name in ((p, "params"), (g, "grads"), (m, "momenta")):
            if t is None and name == "momenta":
                continue
            _known_type(t, name)
            if t.dim() < 2 or t.shape != p.shape:
                raise ValueError(f"{name}: a matrix, and the shape of its weight {tuple(p.shape)} is wanted, not {tuple(t.shape)}")
            if t.device != device:
                raise ValueError(f"{name}: one device is wanted, not {t.device} and {device}")
            if name != "grads" and t.numel():
                _written(t, name)
                if t.data_ptr() in seen:
                    raise ValueError(f"{name}: a tensor is listed twice")
                seen.add(t.data_ptr())
    if any(g.numel() and g.data_ptr() in seen for g in grads):
        raise ValueError("grads: a tensor is among the written ones too")
    decay = 1.0 - lr * weight_decay
    if device.type != "cuda":
        for p, g, m in zip(params, grads, momenta):
            if not p.numel():
                continue
            u = g.float()
            if m is not None:
                m.copy_(momentum * m.float() + (1.0 - momentum) * u)
                u = (1.0 - momentum) * u + momentum * m.float() if nesterov else m.float()
            by = math.sqrt(max(1.0, p.shape[-2] / p.shape[-1])) if scale is None else scale
            p.copy_(decay * p.float() - lr * by * _orthogonal_plain(u, steps, coefficients, eps))
        return
    _refuse_unseen("muon_step", *params, *grads, *momenta)
    items, held = _muon_items(params, grads, momenta, lr, decay, scale)
    if items:
        _muon_call(device, items, momentum, nesterov, steps, coefficients, eps)
    del held  # (its memory is the stream's: what takes it next runs behind the launches)
    torch.autograd.graph.increment_version([t for t in params + momenta if t is not None])


class Muon(torch.optim.Optimizer):
    """``muon_step`` over the parameters that have a gradient; matrices only (what has one axis wants another optimiser).

    The momentum is held in float32.  A step may be captured in a HIP graph once one step has been taken: the buffers have
    to be there before, and the learning rate of the capture stays."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
        _check_iteration(steps, coefficients, eps)
        if not lr >= 0.0 or not 0.0 <= momentum < 1.0 or not weight_decay >= 0.0:
            raise ValueError(f"lr {lr}, momentum {momentum}, weight_decay {weight_decay}")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps))

    def add_param_group(self, group):
        super().add_param_group(group)
        try:
            for p in self.param_groups[-1]["params"]:
                _known_type(p, "params")
                if p.dim() < 2:
                    raise ValueError(f"Muon takes matrices, not a parameter of shape {tuple(p.shape)}")
        except (TypeError, ValueError):
            self.param_groups.pop()  # a refused group leaves the optimizer as it was
            raise

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)  # casts the state to the parameters' type: the momentum stays float32
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i, p in zip(saved, (p for group in self.param_groups for p in group["params"])):
            if "momentum" in state_dict["state"].get(i, ()):
                self.state[p]["momentum"] = state_dict["state"][i]["momentum"].to(device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_device = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if "momentum" not in self.state.get(p, ()):
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("Muon: take one step before the capture, or each replay clears the momentum")
                    self.state[p]["momentum"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                by_device.setdefault(p.device, []).append((p, p.grad, self.state[p]["momentum"]))
            for of in by_device.values():
                muon_step(*zip(*of), lr=group["lr"], momentum=group["momentum"], nesterov=group["nesterov"],
                          weight_decay=group["weight_decay"], steps=group["steps"], coefficients=group["coefficients"], eps=group["eps"])
        return loss
