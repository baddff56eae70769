"""Differentiable forward of the attentive pools and their set encoders.

Calls that need no autograd graph (``.eval()`` under ``torch.no_grad()``, or
nothing requiring a gradient) run through the fused MFMA layer-chain and
attention kernels (``dense.py``), which implement BatchNorm with running
statistics and record no graph.  In ``.train()``, and in ``.eval()`` whenever an
input or a parameter requires a gradient, the pools are composed here from
differentiable pieces instead (BatchNorm follows the module's mode): the Linear
of a dense layer is this package's streaming MFMA product for its output and
input gradient (``mvf_linear_rows``; a library GEMM for shapes it does not
take) and ``mvf_xty`` for its weight and bias gradients (``linear``), its
BatchNorm1d + LeakyReLU tail one pair of this package's kernels forward and
one backward (``batch_norm_act``), the attention-weighted sum one kernel each
way (``weighted_segment_sum``), and the CSR operations are this package's
kernels, all wrapped in ``torch.autograd.Function``
(``pooling.segment_csr`` / ``gather_csr`` / ``segment_softmax_csr``).

Inside ``keep_activations('int8')`` (or with ``keep='int8'``) the dense layers keep
8-bit rows (``packed``) for their backward instead of float32 ones: a Linear the
rows it got, BatchNorm + LeakyReLU its normalised rows, and a Linear behind such
an activation nothing of its own: its weight gradient is made of the packed
rows of the activation.  The forward computes the same (the order of a product's
sum may differ below 4096 rows); gradients are the formulas' on the rows as they
read back.

The computation follows modules/multimodal/pooling.py: ``DeepSetFeat.forward``
:658-681, ``MinMaxDiffSetFeat.forward`` :577-597, ``MLPSetFeat.forward``
:688-699, ``GroupBimodalCSRPool.forward`` :263-315 and
``QKVBimodalCSRPool.forward`` :454-547.
"""
import contextlib
import ctypes
import math
import threading

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import packed
from . import pooling as P

_FORMS = ("float32", "int8")
_kept = threading.local()


@contextlib.contextmanager
def keep_activations(form):
    """Form in which the dense layers (and ``residual.residual_norm``) of this thread
    keep rows for their backward pass: 'float32' (as they are, the default) or
    'int8' (``packed`` rows).  Read by the forward; a backward uses what its forward
    kept, wherever it runs."""
    if form not in _FORMS:
        raise ValueError(f"keep_activations: {form!r} is not one of {_FORMS}")
    before = getattr(_kept, "form", _FORMS[0])
    _kept.form = form
    try:
        yield
    finally:
        _kept.form = before


def kept_form(keep=None):
    """``keep``, or what ``keep_activations`` says where it is None."""
    if keep is None:
        return getattr(_kept, "form", _FORMS[0])
    if keep not in _FORMS:
        raise ValueError(f"keep={keep!r} is not one of {_FORMS}")
    return keep


def _keeps8(keep, *tensors):
    return (kept_form(keep) == "int8" and torch.is_grad_enabled()
            and any(t is not None and t.requires_grad for t in tensors))


class _BatchNormAct(torch.autograd.Function):
    """BatchNorm1d (+ LeakyReLU) of float32 rows on the kernels
    mvf_batch_norm_act_forward / _backward: two passes over the rows forward,
    two backward; only the layer's input is kept for the backward."""

    @staticmethod
    def forward(ctx, z, weight, bias, rm, rv, eps, slope, batch_stats, factor, col_sums):
        lib = L.load()
        z = z.detach().contiguous()
        rows, C = z.shape
        dev = z.device
        w = None if weight is None else weight.detach().float().contiguous()
        b = None if bias is None else bias.detach().float().contiguous()
        y = torch.empty_like(z)
        mean = torch.empty(C, dtype=torch.float32, device=dev)
        invstd = torch.empty(C, dtype=torch.float32, device=dev)
        nbytes = lib.mvf_batch_norm_act_workspace_bytes(C)
        ws = L.workspace(nbytes, dev)
        with torch.cuda.device(dev):
            L.check(lib.mvf_batch_norm_act_forward(
                L.ptr(z), rows, C, L.ptr(w), L.ptr(b), L.ptr(rm), L.ptr(rv), int(batch_stats),
                float(factor), float(eps), int(slope is not None),
                0.0 if slope is None else float(slope), L.ptr(y), L.ptr(mean), L.ptr(invstd),
                L.ptr(col_sums), 0 if col_sums is None else col_sums.shape[0],
                L.ptr(ws), nbytes, L.stream_ptr(dev)))
        ctx.save_for_backward(z, w, b, mean, invstd)
        ctx.slope, ctx.batch_stats = slope, bool(batch_stats)
        return y

    @staticmethod
    def backward(ctx, grad_y):
        lib = L.load()
        z, w, b, mean, invstd = ctx.saved_tensors
        rows, C = z.shape
        dev = z.device
        grad_y = grad_y.contiguous()
        gz = torch.empty_like(z)
        gw = torch.empty(C, dtype=torch.float32, device=dev) if w is not None and ctx.needs_input_grad[1] else None
        gb = torch.empty(C, dtype=torch.float32, device=dev) if b is not None and ctx.needs_input_grad[2] else None
        nbytes = lib.mvf_batch_norm_act_workspace_bytes(C)
        ws = L.workspace(nbytes, dev)
        slope = ctx.slope
        with torch.cuda.device(dev):
            L.check(lib.mvf_batch_norm_act_backward(
                L.ptr(grad_y), L.ptr(z), rows, C, L.ptr(w), L.ptr(b), L.ptr(mean), L.ptr(invstd),
                int(ctx.batch_stats), int(slope is not None), 0.0 if slope is None else float(slope),
                L.ptr(gz), L.ptr(gw), L.ptr(gb), L.ptr(ws), nbytes, L.stream_ptr(dev)))
        return gz, gw, gb, None, None, None, None, None, None, None


def _addr(t):
    return None if t is None else t.data_ptr()


def _bn8_forward(z, weight, bias, rm, rv, eps, slope, batch_stats, factor, counter, col_sums):
    """(y, codes, exps, invstd) of mvf_batch_norm_act8_forward."""
    lib = L.load()
    rows, C = z.shape
    dev = z.device
    y = torch.empty_like(z)
    codes, exps = packed.empty_codes(rows, C, dev)
    invstd = torch.empty(C, dtype=torch.float32, device=dev)
    nbytes = lib.mvf_batch_norm_act8_workspace_bytes(C)
    ws = L.workspace(nbytes, dev)
    L.launch(dev, lib.mvf_batch_norm_act8_forward, z.data_ptr(), rows, C, _addr(weight), _addr(bias), _addr(rm),
             _addr(rv), batch_stats, factor, eps, slope is not None, slope or 0.0, _addr(counter), y.data_ptr(), codes.data_ptr(),
             exps.data_ptr(), invstd.data_ptr(), _addr(col_sums), 0 if col_sums is None else col_sums.shape[0],
             ws.data_ptr(), nbytes)
    return y, codes, exps, invstd


def _bn8_backward(grad_y, codes, exps, weight, bias, invstd, batch_stats, slope, needs):
    """(grad_z, grad_weight, grad_bias) of mvf_batch_norm_act8_backward, those of `needs`."""
    lib = L.load()
    rows, C = codes.shape
    dev = codes.device
    grad_y = grad_y.contiguous()
    gz = torch.empty((rows, C), dtype=torch.float32, device=dev) if needs[0] else None
    gw = torch.empty(C, dtype=torch.float32, device=dev) if needs[1] else None
    gb = torch.empty(C, dtype=torch.float32, device=dev) if needs[2] else None
    nbytes = lib.mvf_batch_norm_act8_workspace_bytes(C)
    ws = L.workspace(nbytes, dev)
    L.launch(dev, lib.mvf_batch_norm_act8_backward, grad_y.data_ptr(), codes.data_ptr(), exps.data_ptr(), rows, C,
             _addr(weight), _addr(bias), invstd.data_ptr(), batch_stats, slope is not None, slope or 0.0,
             _addr(gz), _addr(gw), _addr(gb), ws.data_ptr(), nbytes)
    return gz, gw, gb


def _vector(t):
    return None if t is None else t.detach().contiguous()


def _fused8(rows, weight):
    """Do the kernels that pack rows within a Linear's own pass take these?"""
    return bool(L.load().mvf_linear_rows8_supported(weight.shape[1], weight.shape[0])) and rows.data_ptr() % 16 == 0


def _sums_buffer(lib, cout, want, dev):
    nbytes = lib.mvf_linear_rows_sums_bytes(cout) if want else 0
    return torch.empty(nbytes // 8, dtype=torch.float64, device=dev) if want else None, nbytes, ctypes.c_int32(0)


def _linear8_forward(x, weight, bias, want_sums):
    """(y, codes, exps, partial column sums or None) of mvf_linear_rows8_forward."""
    lib = L.load()
    rows, (cout, cin), dev = x.shape[0], weight.shape, x.device
    weight, bias = _vector(weight), _vector(bias)
    y = torch.empty((rows, cout), dtype=torch.float32, device=dev)
    codes, exps = packed.empty_codes(rows, cin, dev)
    sums, nbytes, n = _sums_buffer(lib, cout, want_sums, dev)
    L.launch(dev, lib.mvf_linear_rows8_forward, x.data_ptr(), cin, weight.data_ptr(), _addr(bias), cout, rows,
             y.data_ptr(), codes.data_ptr(), exps.data_ptr(), _addr(sums), nbytes, ctypes.addressof(n))
    return y, codes, exps, sums[:n.value * 2 * cout].view(n.value, 2, cout) if want_sums else None


def _linear8_backward(grad_y, codes, exps, weight, want_bias):
    """(grad_x, grad_weight, grad_bias or None) of mvf_linear_rows8_backward."""
    lib = L.load()
    rows, (cout, cin), dev = grad_y.shape[0], weight.shape, grad_y.device
    weight = _vector(weight)
    gx = torch.empty((rows, cin), dtype=torch.float32, device=dev)
    gw = torch.empty((cout, cin), dtype=torch.float32, device=dev)
    gb = torch.empty(cout, dtype=torch.float32, device=dev) if want_bias else None
    nbytes = lib.mvf_xty8_workspace_bytes()
    ws = L.workspace(nbytes, dev)
    L.launch(dev, lib.mvf_linear_rows8_backward, grad_y.data_ptr(), codes.data_ptr(), exps.data_ptr(),
             weight.data_ptr(), cin, cout, rows, gx.data_ptr(), gw.data_ptr(), _addr(gb), ws.data_ptr(), nbytes)
    return gx, gw, gb


def _bn_linear8_forward(z, w, b, rm, rv, eps, slope, batch_stats, factor, counter, col_sums, weight, bias, want_sums):
    """(out, codes, exps, invstd, partial column sums or None) of mvf_batch_norm_act_linear8_forward."""
    lib = L.load()
    rows, (cout, cin), dev = z.shape[0], weight.shape, z.device
    weight, bias = _vector(weight), _vector(bias)
    out = torch.empty((rows, cout), dtype=torch.float32, device=dev)
    codes, exps = packed.empty_codes(rows, cin, dev)
    invstd = torch.empty(cin, dtype=torch.float32, device=dev)
    sums, sbytes, n = _sums_buffer(lib, cout, want_sums, dev)
    nbytes = lib.mvf_batch_norm_act_linear8_workspace_bytes(cin)
    ws = L.workspace(nbytes, dev)
    L.launch(dev, lib.mvf_batch_norm_act_linear8_forward, z.data_ptr(), rows, cin, _addr(w), _addr(b), _addr(rm),
             _addr(rv), batch_stats, factor, eps, slope is not None, slope or 0.0, _addr(counter), weight.data_ptr(),
             _addr(bias), cout,
             out.data_ptr(), codes.data_ptr(), exps.data_ptr(), invstd.data_ptr(), _addr(col_sums),
             0 if col_sums is None else col_sums.shape[0], _addr(sums), sbytes, ctypes.addressof(n),
             ws.data_ptr(), nbytes)
    return out, codes, exps, invstd, sums[:n.value * 2 * cout].view(n.value, 2, cout) if want_sums else None


def _bn_linear8_backward(grad_out, codes, exps, w, b, invstd, batch_stats, slope, weight, needs):
    """Gradients of (z, BatchNorm's weight and bias, the Linear's weight and bias), those of `needs`, by
    mvf_batch_norm_act_linear8_backward."""
    lib = L.load()
    (rows, cin), cout, dev = codes.shape, weight.shape[0], codes.device
    weight = _vector(weight)

    def empty(wanted, *shape):
        return torch.empty(shape, dtype=torch.float32, device=dev) if wanted else None

    gz, gw, gb = empty(True, rows, cin), empty(needs[1], cin), empty(needs[2], cin)
    glw, glb = empty(True, cout, cin), empty(needs[4], cout)
    nbytes = lib.mvf_batch_norm_act_linear8_workspace_bytes(cin)
    ws = L.workspace(nbytes, dev)
    L.launch(dev, lib.mvf_batch_norm_act_linear8_backward, grad_out.data_ptr(), codes.data_ptr(), exps.data_ptr(), rows,
             cin, _addr(w), _addr(b), invstd.data_ptr(), batch_stats, slope is not None, slope or 0.0,
             weight.data_ptr(), cout, gz.data_ptr(), _addr(gw), _addr(gb), glw.data_ptr(), _addr(glb),
             ws.data_ptr(), nbytes)
    return gz, gw, gb, glw, glb


class _BatchNormAct8(torch.autograd.Function):
    """_BatchNormAct that keeps the normalised rows in 8 bits."""

    @staticmethod
    def forward(ctx, z, weight, bias, rm, rv, eps, slope, batch_stats, factor, counter, col_sums):
        w, b = _vector(weight), _vector(bias)
        y, codes, exps, invstd = _bn8_forward(z.detach().contiguous(), w, b, rm, rv, eps, slope, batch_stats,
                                              factor, counter, col_sums)
        ctx.save_for_backward(codes, exps, w, b, invstd)
        ctx.slope, ctx.batch_stats = slope, bool(batch_stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        codes, exps, w, b, invstd = ctx.saved_tensors
        return _bn8_backward(grad_y, codes, exps, w, b, invstd, ctx.batch_stats, ctx.slope,
                             ctx.needs_input_grad) + (None,) * 8


class _BatchNormActLinear8(torch.autograd.Function):
    """Linear(act(bn(z))) that keeps the normalised rows in 8 bits and nothing else of
    a row: the Linear's input is made of them again in its weight gradient."""

    @staticmethod
    def forward(ctx, z, bn_weight, bn_bias, weight, bias, rm, rv, eps, slope, batch_stats, factor, counter, col_sums,
                want_sums):
        w, b = _vector(bn_weight), _vector(bn_bias)
        z = z.detach().contiguous()
        ctx.fused = _fused8(z, weight)
        if ctx.fused:
            out, codes, exps, invstd, sums = _bn_linear8_forward(
                z, w, b, rm, rv, eps, slope, batch_stats, factor, counter, col_sums, weight, bias, want_sums)
        else:
            y, codes, exps, invstd = _bn8_forward(z, w, b, rm, rv, eps, slope, batch_stats, factor, counter, col_sums)
            out, sums = _product(y, weight, bias, want_sums)
        ctx.save_for_backward(codes, exps, w, b, invstd, weight)
        ctx.slope, ctx.batch_stats = slope, bool(batch_stats)
        if sums is None:
            return out, None
        ctx.mark_non_differentiable(sums)
        return out, sums

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, _grad_sums):
        codes, exps, w, b, invstd, weight = ctx.saved_tensors
        need = ctx.needs_input_grad
        grad_out = grad_out.contiguous()
        gz = gw = gb = glw = glb = None
        if ctx.fused and need[0] and need[3] and grad_out.data_ptr() % 16 == 0:
            return _bn_linear8_backward(grad_out, codes, exps, w, b, invstd, ctx.batch_stats, ctx.slope, weight,
                                        need) + (None,) * 9
        if any(need[:3]):
            gy = _product(grad_out, weight.t(), None)[0]
            gz, gw, gb = _bn8_backward(gy, codes, exps, w, b, invstd, ctx.batch_stats, ctx.slope, need)
        if need[3]:
            glw, glb = _xty8(grad_out, codes, exps, tail=(w, b, ctx.slope), want_sums=need[4])
        elif need[4]:
            glb = xty(grad_out).view(-1)
        return (gz, gw, gb, glw, glb) + (None,) * 9


def _takes_bn(z, bn):
    return (z.is_cuda and z.dtype == torch.float32 and z.dim() == 2 and z.shape[0] > 0
            and isinstance(bn, torch.nn.BatchNorm1d) and z.shape[1] == bn.num_features)


def _sums_for(z, col_sums):
    """col_sums, refused unless they are partial sums of z's columns."""
    if col_sums is not None and not (
            col_sums.dtype == torch.float64 and col_sums.dim() == 3 and col_sums.shape[0] > 0
            and col_sums.shape[1] == 2 and col_sums.shape[2] == z.shape[1] and col_sums.device == z.device
            and col_sums.is_contiguous()):
        raise ValueError(f"col_sums must be contiguous float64 [n, 2, {z.shape[1]}] on the device of the rows, as "
                         f"linear(..., want_sums=True) returns them, got {tuple(col_sums.shape)} {col_sums.dtype}")
    return col_sums


def _bn_plan(z, bn, weight, bias, kernel_counts=False, col_sums=None):
    """(running mean, running variance, batch_stats, factor, counter, the column sums to use) of the
    next call on z of an nn.BatchNorm1d with these parameters; None where this package's kernels do
    not take one of its tensors.  The batch is counted in num_batches_tracked here, or, with
    kernel_counts, by the kernel that is given the counter (None: already counted, or nothing to
    count)."""
    rm, rv, tracked = bn.running_mean, bn.running_var, bn.num_batches_tracked
    for t in (weight, bias, rm, rv):
        if t is not None and not (t.device == z.device and t.dtype == torch.float32 and t.shape == z.shape[1:]):
            return None
    batch_stats = bn.training or rm is None
    factor, counter = 0.0, None
    if batch_stats:
        if z.shape[0] < 2:
            raise ValueError(
                f"Expected more than 1 value per channel when training, got input size {tuple(z.shape)}")
        col_sums = _sums_for(z, col_sums)
        if bn.training and bn.track_running_stats and tracked is not None:
            if kernel_counts and bn.momentum is not None and tracked.device == z.device and tracked.dtype == torch.int64:
                counter = tracked
            else:
                tracked.add_(1)
            factor = (1.0 / float(tracked)) if bn.momentum is None else bn.momentum
    # running statistics: updated in train mode, read in eval mode, unused by an eval-mode
    # module that tracks none (it normalises with batch statistics)
    use_running = rm is not None and (bn.training or not batch_stats)
    return (rm if use_running else None, rv if use_running else None, batch_stats, factor, counter,
            col_sums if batch_stats else None)


def batch_norm_act(z, bn, act, col_sums=None, keep=None):
    """``act(bn(z))`` for an ``nn.BatchNorm1d`` (train or eval mode, running
    statistics and ``num_batches_tracked`` updated as the module does) followed
    by a LeakyReLU, on this package's kernels when z is a float32 [rows, C]
    tensor on the HIP device; other inputs and activations take the modules.
    col_sums: partial column sums of z and z * z as ``linear(..., want_sums=True)``
    returns them (batch statistics without another pass over z).
    keep: 'float32' keeps z for the backward, 'int8' its normalised rows in 8 bits
    (a value that is not finite then counts as not above the activation's kink);
    None: as ``keep_activations`` says."""
    fused_act = isinstance(act, torch.nn.LeakyReLU)
    kept_form(keep)
    if not _takes_bn(z, bn):
        return act(bn(z))
    weight, bias = bn.weight, bn.bias
    keeps8 = _keeps8(keep, z, weight, bias)
    plan = _bn_plan(z, bn, weight, bias, keeps8, col_sums)
    if plan is None:
        return act(bn(z))
    rm, rv, batch_stats, factor, counter, col_sums = plan
    slope = float(act.negative_slope) if fused_act else None
    if keeps8:
        y = _BatchNormAct8.apply(z, weight, bias, rm, rv, bn.eps, slope, batch_stats, factor, counter, col_sums)
    else:
        y = _BatchNormAct.apply(z, weight, bias, rm, rv, bn.eps, slope, batch_stats, factor, col_sums)
    return y if fused_act else act(y)


def batch_norm_act_linear(z, bn, act, lin, col_sums=None, want_sums=False, keep=None):
    """``linear(lin, batch_norm_act(z, bn, act, col_sums), want_sums)``.  With 'int8'
    rows (``keep``, ``keep_activations``) and a LeakyReLU the two keep one packed copy
    of the normalised rows between them; elsewhere they are two calls."""
    if isinstance(act, torch.nn.LeakyReLU) and _takes(lin, z) and _takes_bn(z, bn):
        weight, bias = bn.weight, bn.bias
        if _keeps8(keep, z, weight, bias, lin.weight, lin.bias):
            plan = _bn_plan(z, bn, weight, bias, True, col_sums)
            if plan is not None:
                rm, rv, batch_stats, factor, counter, col_sums = plan
                y, sums = _BatchNormActLinear8.apply(
                    z, weight, bias, lin.weight, lin.bias, rm, rv, bn.eps, float(act.negative_slope),
                    batch_stats, factor, counter, col_sums, bool(want_sums))
                return (y, sums) if want_sums else y
    form = {} if keep is None else {"keep": keep}
    return linear(lin, batch_norm_act(z, bn, act, col_sums=col_sums, **form), want_sums, **form)


def xty(x, y=None):
    """x^T . y of two float32 [rows, *] tensors on the HIP device (mvf_xty);
    without y the column sums of x, [A, 1]."""
    lib = L.load()
    x = x.contiguous()
    dev = x.device
    if y is None:
        out = torch.empty((x.shape[1], 1), dtype=torch.float32, device=dev)
        nbytes = lib.mvf_xty_workspace_bytes()
        ws = L.workspace(nbytes, dev)
        with torch.cuda.device(dev):
            L.check(lib.mvf_xty(L.ptr(x), x.stride(0), x.shape[1], None, 0, 1, x.shape[0],
                                L.ptr(out), 1, L.ptr(ws), nbytes, L.stream_ptr(dev)))
        return out
    y = y.contiguous()
    out = torch.empty((x.shape[1], y.shape[1]), dtype=torch.float32, device=dev)
    nbytes = lib.mvf_xty_workspace_bytes()
    ws = L.workspace(nbytes, dev)
    with torch.cuda.device(dev):
        L.check(lib.mvf_xty(L.ptr(x), x.stride(0), x.shape[1], L.ptr(y), y.stride(0), y.shape[1],
                            x.shape[0], L.ptr(out), out.stride(0), L.ptr(ws), nbytes,
                            L.stream_ptr(dev)))
    return out


class _Weights:
    """What dense.LayerSpec reads of an nn.Linear."""

    def __init__(self, weight, bias):
        self.weight, self.bias = weight, bias
        self.out_features, self.in_features = weight.shape


def _product(x, weight, bias, want_sums=False):
    """(x W^T + b, partial column sums or None) over many rows: the streaming
    float32 MFMA kernel (mvf_linear_rows, which can leave the column sums of its
    output for BatchNorm's batch statistics) for at most 64 input and output
    columns, one launch of the layer-chain kernel with a single plain layer for
    wider ones (both stream the rows at a higher rate than the library GEMM
    does for these shapes), the library GEMM otherwise."""
    if max(weight.shape) > 256 or x.shape[0] < 4096:
        return torch.nn.functional.linear(x, weight, bias), None
    dense = P._dense
    w = weight.detach()
    specs, xp = dense.aligned_input(
        [dense.LayerSpec(_Weights(w if w.is_contiguous() else w.contiguous(), bias))], x.detach())
    lib = L.load()
    cout, cin = specs[0].cout, specs[0].cin
    if not (lib.mvf_linear_rows_supported(cin, cout) and xp.is_contiguous() and xp.data_ptr() % 16 == 0):
        return dense.run_layers(specs, xp), None
    wp, bp = specs[0].weight.float().contiguous(), None if bias is None else bias.detach().float().contiguous()
    dev = xp.device
    y = torch.empty((xp.shape[0], cout), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        if not want_sums:
            L.check(lib.mvf_linear_rows(L.ptr(xp), cin, L.ptr(wp), L.ptr(bp), cout, xp.shape[0], L.ptr(y),
                                        L.stream_ptr(dev)))
            return y, None
        nbytes = lib.mvf_linear_rows_sums_bytes(cout)
        sums = torch.empty(nbytes // 8, dtype=torch.float64, device=dev)
        n = ctypes.c_int32(0)
        L.check(lib.mvf_linear_rows_sums(L.ptr(xp), cin, L.ptr(wp), L.ptr(bp), cout, xp.shape[0], L.ptr(y),
                                         L.ptr(sums), nbytes, ctypes.byref(n), L.stream_ptr(dev)))
    return y, sums[:n.value * 2 * cout].view(n.value, 2, cout)


class _Linear(torch.autograd.Function):
    """y = x W^T + b: the output and the input gradient (as many rows as the
    input) by ``_product``, the weight gradient by mvf_xty: a reduction over
    every row into a few thousand sums, where library GEMMs reach a few percent
    of the memory bandwidth."""

    @staticmethod
    def forward(ctx, x, weight, bias, want_sums):
        ctx.save_for_backward(x, weight)
        ctx.has_bias = bias is not None
        y, sums = _product(x, weight, bias, want_sums)
        if sums is None:
            sums = torch.empty(0, dtype=torch.float64, device=x.device)
        ctx.mark_non_differentiable(sums)
        return y, sums

    @staticmethod
    def backward(ctx, grad_y, _grad_sums):
        x, weight = ctx.saved_tensors
        grad_y = grad_y.contiguous()
        gx = _product(grad_y, weight.t(), None)[0] if ctx.needs_input_grad[0] else None
        gw = xty(grad_y, x) if ctx.needs_input_grad[1] else None
        gb = xty(grad_y).view(-1) if ctx.has_bias and ctx.needs_input_grad[2] else None
        return gx, gw, gb, None


def xty8(x, codes, exps, tail=None, want_sums=False):
    """(x^T . y, column sums of x or None) for float32 rows x [rows, A] and y read from 8-bit
    rows: codes int8 [rows, B], exps uint8 [rows, ceil(B / 32)] (mvf_xty8).  tail = (weight,
    bias, slope): the rows are those of ``mvf_batch_norm_act8_forward`` and y the activated
    values made of them; weight and bias float32 [B] or None, slope None: no activation."""
    if x.dtype != torch.float32:
        raise TypeError(f"mvfusion xty8 expects float32 rows, got {x.dtype}")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"xty8 expects rows [rows, A] with at least one column, got {tuple(x.shape)}")
    packed.check_codes(codes, exps, "xty8")
    if codes.shape[0] != x.shape[0] or codes.device != x.device:
        raise ValueError(f"xty8: {codes.shape[0]} packed rows on {codes.device} do not fit {x.shape[0]} rows on {x.device}")
    w, b, slope = tail if tail is not None else (None, None, None)
    for t in (w, b):
        if t is not None and (t.dtype != torch.float32 or t.shape != codes.shape[1:] or t.device != x.device):
            raise ValueError(f"xty8: weight and bias must be float32 [{codes.shape[1]}] on the device of the rows")
    if not x.is_cuda:
        raise RuntimeError("mvfusion xty8 runs on a HIP device only (there is no CPU fallback).")
    return _xty8(x, codes.contiguous(), exps.contiguous(), None if tail is None else (_vector(w), _vector(b), slope), want_sums)


def _xty8(x, codes, exps, tail=None, want_sums=False):
    """xty8 without its checks, for the rows a forward has kept."""
    lib = L.load()
    x = x.contiguous()
    dev = x.device
    A, B = x.shape[1], codes.shape[1]
    out = torch.empty((A, B), dtype=torch.float32, device=dev)
    sums = torch.empty(A, dtype=torch.float32, device=dev) if want_sums else None
    w, b, slope = tail if tail is not None else (None, None, None)
    nbytes = lib.mvf_xty8_workspace_bytes()
    ws = L.workspace(nbytes, dev)
    L.launch(dev, lib.mvf_xty8, x.data_ptr(), A, A, codes.data_ptr(), exps.data_ptr(), B, x.shape[0],
             tail is not None, _addr(w), _addr(b), slope is not None, slope or 0.0, out.data_ptr(), B, _addr(sums),
             ws.data_ptr(), nbytes)
    return out, sums


class _Linear8(torch.autograd.Function):
    """_Linear that keeps its input as 8-bit rows (nothing of it when the weight needs no
    gradient)."""

    @staticmethod
    def forward(ctx, x, weight, bias, want_sums):
        codes = exps = None
        x = x.detach().contiguous()
        ctx.fused = ctx.needs_input_grad[1] and _fused8(x, weight)
        if ctx.fused:
            y, codes, exps, sums = _linear8_forward(x, weight, bias, want_sums)
        else:
            if ctx.needs_input_grad[1]:
                codes, exps = packed.pack_codes(x)
            y, sums = _product(x, weight, bias, want_sums)
        ctx.save_for_backward(codes, exps, weight)
        if sums is None:
            return y, None
        ctx.mark_non_differentiable(sums)
        return y, sums

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y, _grad_sums):
        codes, exps, weight = ctx.saved_tensors
        need = ctx.needs_input_grad
        grad_y = grad_y.contiguous()
        if ctx.fused and need[0] and grad_y.data_ptr() % 16 == 0:
            return _linear8_backward(grad_y, codes, exps, weight, need[2]) + (None,)
        gx = _product(grad_y, weight.t(), None)[0] if need[0] else None
        gw = gb = None
        if need[1]:
            gw, gb = _xty8(grad_y, codes, exps, want_sums=need[2])
        elif need[2]:
            gb = xty(grad_y).view(-1)
        return gx, gw, gb, None


def _fits(x, weight, bias):
    """Can the kernels take rows x through this Linear?  (They read as many columns as the weight has,
    and parameters as float32 on the device of the rows.)"""
    return (x.is_cuda and x.dtype == torch.float32 and x.dim() == 2 and x.shape[0] > 0
            and weight.device == x.device and weight.dtype == torch.float32 and weight.shape[1] == x.shape[1]
            and (bias is None or (bias.device == x.device and bias.dtype == torch.float32)))


def _takes(lin, x):
    return _fits(x, lin.weight, lin.bias)


def _linear(x, weight, bias, want_sums=False, keep=None):
    fn = _Linear8 if _keeps8(keep, x, weight, bias) else _Linear
    return fn.apply(x, weight, bias, bool(want_sums))


def linear(lin, x, want_sums=False, keep=None):
    """``lin(x)`` for an ``nn.Linear`` on float32 [rows, C] device tensors,
    with the weight gradient on this package's kernel; anything else takes the
    module.  want_sums: returns (output, partial column sums of the output and
    its square or None) for ``batch_norm_act``.  keep: 'float32' keeps x for the
    weight gradient, 'int8' its 8-bit rows; None: as ``keep_activations`` says."""
    if _takes(lin, x):
        y, sums = _linear(x, lin.weight, lin.bias, want_sums, keep)
        return (y, sums if sums is not None and sums.numel() else None) if want_sums else y
    kept_form(keep)
    return (lin(x), None) if want_sums else lin(x)


def _batch_stats(block):
    bn = block[1].batch_norm
    return bn.training or bn.running_mean is None


def _mlp_tail(seq, z, sums=None):
    """What follows the first Linear of an MLP, from that Linear's output."""
    for i, block in enumerate(seq):
        bn, act = block[1].batch_norm, block[2]
        if i + 1 == len(seq):
            return batch_norm_act(z, bn, act, col_sums=sums)
        if _batch_stats(seq[i + 1]):
            z, sums = batch_norm_act_linear(z, bn, act, seq[i + 1][0], col_sums=sums, want_sums=True)
        else:
            z, sums = batch_norm_act_linear(z, bn, act, seq[i + 1][0], col_sums=sums), None


def mlp(seq, x):
    """MLP of base_modules.py:38-48: per block Linear (streaming MFMA products,
    weight gradient by mvf_xty), then BatchNorm1d and the activation in one pair
    of kernels; in train mode the Linear leaves the column sums the batch
    statistics are made of.  With 8-bit rows kept (``keep_activations``) an
    activation and the Linear behind it share one packed copy."""
    if len(seq) == 0:
        return x
    if _batch_stats(seq[0]):
        z, sums = linear(seq[0][0], x, want_sums=True)
    else:
        z, sums = linear(seq[0][0], x), None
    return _mlp_tail(seq, z, sums)


def mlp_on_rows_and_sets(seq, x, x_set, ptr):
    """``mlp(seq, cat((x, gather_csr(x_set, ptr)), 1))`` without the concatenated rows: the
    first Linear is split by columns, [x | x_set[seg]] W^T = x Wa^T + (x_set Wb^T + b)[seg],
    so the set features go through their half once per segment instead of once per row
    (DeepSetFeat's 'concatenation' fusion, pooling.py:669-681)."""
    lin = seq[0][0]
    d = x.shape[1]
    wa, wb = lin.weight[:, :d], lin.weight[:, d:]
    if not (_fits(x, wa, None) and _fits(x_set, wb, lin.bias)):
        return mlp(seq, torch.cat((x, P.gather_csr(x_set, ptr)), dim=1))
    za = _linear(x, wa, None)[0]
    zb = _linear(x_set, wb, lin.bias)[0]
    return _mlp_tail(seq, za + P.gather_csr(zb, ptr))


def deep_set_feat(m, x, ptr):
    x = mlp(m.mlp_elt_1, x)
    sets = [P.segment_csr(x, ptr, reduce=p) for p in m.pool]
    if m.use_num:
        sets.append(P._set_num(ptr).view(-1, 1))
    x_set = torch.cat(sets, dim=-1) if len(sets) > 1 else sets[0]
    x_set = mlp(m.mlp_set, x_set)
    if m.fusion == 'concatenation' and x.is_cuda and x.dtype == torch.float32:
        return mlp_on_rows_and_sets(m.mlp_elt_2, x, x_set, ptr)
    x_set = P.gather_csr(x_set, ptr)
    if m.fusion == 'residual':
        x_out = x + x_set
    elif m.fusion == 'concatenation':
        x_out = torch.cat((x, x_set), dim=-1)
    else:
        x_out = torch.cat((x, x + x_set), dim=-1)
    return mlp(m.mlp_elt_2, x_out)


def min_max_diff_set_feat(m, x, ptr):
    parts = [x]
    if m.use_min:
        parts.append(x - P.segment_gather_csr(x, ptr, reduce='min'))
    if m.use_max:
        parts.append(x - P.segment_gather_csr(x, ptr, reduce='max'))
    if m.use_num:
        parts.append(P._set_num(ptr).repeat_interleave(ptr[1:] - ptr[:-1]).view(-1, 1))
    return mlp(m.mlp, torch.cat(parts, dim=1) if len(parts) > 1 else x)


def map_encoder(m, x, ptr):
    if isinstance(m, P.DeepSetFeat):
        return deep_set_feat(m, x, ptr)
    if isinstance(m, P.MinMaxDiffSetFeat):
        return min_max_diff_set_feat(m, x, ptr)
    return mlp(m.mlp, x)


class _WeightedSegmentSum(torch.autograd.Function):
    """segment_csr(x * expand_group_feat(att), ptr, 'sum') in one pass over x,
    and both gradients in one pass (mvf_weighted_segment_sum / _backward)."""

    @staticmethod
    def forward(ctx, x, att, ptr, num_groups):
        lib = L.load()
        x, att = x.detach().contiguous(), att.detach().contiguous()
        dev = x.device
        nseg = ptr.shape[0] - 1
        out = torch.empty((nseg, x.shape[1]), dtype=torch.float32, device=dev)
        with torch.cuda.device(dev):
            L.check(lib.mvf_weighted_segment_sum(L.ptr(x), L.ptr(att), x.shape[1], num_groups,
                                                 L.ptr(ptr), nseg, L.ptr(out), L.stream_ptr(dev)))
        ctx.save_for_backward(x, att, ptr)
        ctx.num_groups = num_groups
        return out

    @staticmethod
    def backward(ctx, grad_out):
        lib = L.load()
        x, att, ptr = ctx.saved_tensors
        dev = x.device
        rows, C = x.shape
        grad_out = grad_out.contiguous()
        row2seg = P._dense.csr_row_segments(ptr, rows, outside=-1)
        gx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        gatt = torch.empty_like(att) if ctx.needs_input_grad[1] else None
        with torch.cuda.device(dev):
            L.check(lib.mvf_weighted_segment_sum_backward(
                L.ptr(grad_out), L.ptr(x), L.ptr(att), C, ctx.num_groups, L.ptr(row2seg), rows,
                ptr.shape[0] - 1, L.ptr(gx), L.ptr(gatt), L.stream_ptr(dev)))
        return gx, gatt, None, None


def weighted_segment_sum(x, att, ptr, num_groups):
    """Sum over the rows of every segment of ``x * expand_group_feat(att)``
    (pooling.py:289-296, 519-526): one kernel forward and one backward when the
    channels split into equal groups of a power-of-two multiple of 4 channels
    (rows outside every segment get zero gradients); the composition of
    ``expand_group_feat`` and ``segment_csr`` otherwise."""
    C = x.shape[1]
    cv = C // 4
    ok = (x.is_cuda and x.dtype == torch.float32 and att.dtype == torch.float32 and x.dim() == 2
          and x.shape[0] > 0 and C % 4 == 0 and C % num_groups == 0 and (C // num_groups) % 4 == 0
          and cv <= 64 and cv & (cv - 1) == 0
          and (cv // num_groups) & (cv // num_groups - 1) == 0
          and att.numel() == x.shape[0] * num_groups and ptr.dtype == torch.int64)
    if not ok:
        return P.segment_csr(x * P.expand_group_feat(att, num_groups, C), ptr, reduce='sum')
    return _WeightedSegmentSum.apply(x, att, ptr, num_groups)


def _group_shape_ok(C, num_groups):
    cv = C // 4
    return (C % 4 == 0 and C % num_groups == 0 and (C // num_groups) % 4 == 0 and 1 <= cv <= 64
            and cv & (cv - 1) == 0 and (cv // num_groups) & (cv // num_groups - 1) == 0)


class _SegmentDot(torch.autograd.Function):
    """comp[r, g] = sum over the channels c of group g of keys[r, c] * queries[segment of r, c]:
    the compatibilities of the views with the query of their point
    (pooling.py:497-512: ``(K * gather_csr(Q)).view(-1, G, D).sum(2)``) without the
    gathered queries or the products in memory.  Forward and both gradients are the
    kernels of the attention-weighted sum with the roles of the tensors exchanged."""

    @staticmethod
    def forward(ctx, keys, queries, ptr, num_groups):
        lib = L.load()
        keys, queries = keys.detach().contiguous(), queries.detach().contiguous()
        dev = keys.device
        rows, C = keys.shape
        nseg = ptr.shape[0] - 1
        row2seg = P._dense.csr_row_segments(ptr, rows, outside=-1)
        comp = torch.empty((rows, num_groups), dtype=torch.float32, device=dev)
        with torch.cuda.device(dev):
            # (the weights argument is only read for the row gradient, which is not asked for)
            L.check(lib.mvf_weighted_segment_sum_backward(
                L.ptr(queries), L.ptr(keys), L.ptr(keys), C, num_groups, L.ptr(row2seg), rows, nseg,
                None, L.ptr(comp), L.stream_ptr(dev)))
        ctx.save_for_backward(keys, queries, ptr, row2seg)
        ctx.num_groups = num_groups
        return comp

    @staticmethod
    def backward(ctx, grad_comp):
        lib = L.load()
        keys, queries, ptr, row2seg = ctx.saved_tensors
        dev = keys.device
        rows, C = keys.shape
        nseg = ptr.shape[0] - 1
        grad_comp = grad_comp.contiguous()
        gk = gq = None
        with torch.cuda.device(dev):
            if ctx.needs_input_grad[0]:
                gk = torch.empty_like(keys)
                L.check(lib.mvf_weighted_segment_sum_backward(
                    L.ptr(queries), L.ptr(keys), L.ptr(grad_comp), C, ctx.num_groups, L.ptr(row2seg),
                    rows, nseg, L.ptr(gk), None, L.stream_ptr(dev)))
            if ctx.needs_input_grad[1]:
                gq = torch.empty_like(queries)
                L.check(lib.mvf_weighted_segment_sum(L.ptr(keys), L.ptr(grad_comp), C, ctx.num_groups,
                                                     L.ptr(ptr), nseg, L.ptr(gq), L.stream_ptr(dev)))
        return gk, gq, None, None


def segment_dot(keys, queries, ptr, num_groups):
    """[rows, G] group-wise dot products of every key row with the query row of its segment
    (queries: one row per segment); the composition with ``gather_csr`` for shapes the
    kernels do not take."""
    C = keys.shape[1]
    if (keys.is_cuda and keys.dtype == torch.float32 and queries.dtype == torch.float32
            and keys.dim() == 2 and keys.shape[0] > 0 and queries.shape == (ptr.shape[0] - 1, C)
            and ptr.dtype == torch.int64 and _group_shape_ok(C, num_groups)):
        return _SegmentDot.apply(keys, queries, ptr, num_groups)
    q = P.gather_csr(queries, ptr)
    return (keys.view(-1, num_groups, C // num_groups) * q.view(-1, num_groups, C // num_groups)).sum(dim=2)


def attend(m, x_mod, comp, ptr):
    """Softmax of the compatibilities over the views of a point, attention-
    weighted sum of the values, optional gate from the best compatibility."""
    att = P.segment_softmax_csr(comp, ptr, scaling=m.group_scaling)
    x_pool = weighted_segment_sum(x_mod, att, ptr, m.num_groups)
    gate = None
    if m.G is not None:
        gate = m.G(P.segment_csr(comp, ptr, reduce='max'))
        x_pool = x_pool * P.expand_group_feat(gate, m.num_groups, m.out_mod)
    return x_pool, att, gate


def group_pool(m, x_main, x_mod, x_map, ptr):
    x_map = map_encoder(m.E_map, x_map, ptr)
    x_mod = mlp(m.E_mod, x_mod)
    x_mix = mlp(m.E_mix, torch.cat([x_map, x_mod], dim=1)) if m.use_mod else x_map
    comp = linear(m.E_score, x_mix)
    x_pool, att, gate = attend(m, x_mod, comp, ptr)
    return x_pool, dict(x_map=x_map, x_mod=x_mod, C=comp, A=att, G=gate)


def qkv_pool(m, x_main, x_mod, x_map, ptr):
    x_main = mlp(m.E_main, x_main)
    x_map = map_encoder(m.E_map, x_map, ptr)
    x_mod = mlp(m.E_mod, x_mod)
    if m.use_mod_k:
        keys = linear(m.K, mlp(m.E_mix_K, torch.cat([x_map, x_mod], dim=1)))
    else:
        keys = linear(m.K, x_map)
    if not m.use_mod_q and not m.save_last:
        # the queries stay one row per point: every view meets the row of its point in the kernel
        queries = linear(m.Q, x_main)
        if m.dim_scaling:
            queries = queries / math.sqrt(m.nc_qk)
        comp = segment_dot(keys, queries, ptr, m.num_groups)
    else:
        if m.use_mod_q:
            queries = linear(m.Q, mlp(m.E_mix_Q, torch.cat([P.gather_csr(x_main, ptr), x_mod], dim=1)))
        else:
            queries = P.gather_csr(linear(m.Q, x_main), ptr)
        comp = (keys.view(-1, m.num_groups, m.nc_qk) * queries.view(-1, m.num_groups, m.nc_qk)).sum(dim=2)
        if m.dim_scaling:
            comp = comp / math.sqrt(m.nc_qk)
    x_pool, att, gate = attend(m, x_mod, comp, ptr)
    return x_pool, dict(x_map=x_map, x_mod=x_mod, K=keys, Q=queries, C=comp, A=att, G=gate)
