"""Gated residual block between two norms: what a pooled image feature (or any
branch's output) goes through on its way onto a point's own feature,

    out = x + scale * gate * N(f; post),    h = N(out; pre)

in one kernel forward and one (and a fold of the column gradients) backward.
``h`` is the input of the next branch.  The gate is one value per row and channel
group, as ``pooling.Gating`` makes it (modules/multimodal/pooling.py:702-723);
rows without a view (``seen``) pass through.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import packed
from . import training

_MAX_C = 4096
_NONE, _RMS, _LAYER = 0, 1, 2


def _norm_args(norm, C, x, name):
    """(kind, weight, bias, eps) of an nn.RMSNorm / nn.LayerNorm over the channels (attributes: a
    parametrized or replicated weight is no entry of the module's own parameters)."""
    if norm is None:
        return _NONE, None, None, 0.0
    if isinstance(norm, torch.nn.LayerNorm):
        kind = _LAYER
    elif isinstance(norm, torch.nn.RMSNorm):
        kind = _RMS
    else:
        raise TypeError(f"residual_norm: {name} must be an nn.RMSNorm or nn.LayerNorm, got {type(norm).__name__}")
    if tuple(norm.normalized_shape) != (C,):
        raise ValueError(f"residual_norm: {name} normalises {tuple(norm.normalized_shape)}, the rows have {C} channels")
    eps = torch.finfo(x.dtype).eps if norm.eps is None else float(norm.eps)
    bias = norm.bias if kind == _LAYER else None        # (an RMS norm has none)
    return kind, _vector(norm.weight, C, x, name), _vector(bias, C, x, name), eps


def _vector(t, C, x, name):
    """t as C float32 values (autograd follows; t itself where it is that already)."""
    if t is None:
        return None
    if t.device != x.device:
        raise ValueError(f"residual_norm: {name} is on {t.device}, the rows are on {x.device}")
    if t.dtype == torch.float32 and t.shape == (C,):
        return t
    if not t.is_floating_point() or t.numel() not in (1, C):
        raise ValueError(f"residual_norm: {name} must hold 1 or {C} floating-point values, got {tuple(t.shape)} {t.dtype}")
    return t.float().reshape(-1).expand(C)


def _addr(t):
    return None if t is None else t.data_ptr()


class _ResidualNorm(torch.autograd.Function):
    """The kernels mvf_residual_norm_forward / _backward.  Kept for the backward:
    x (only with a pre-norm) and f as they are or as 8-bit rows, four statistics a
    row, and the parameters."""

    @staticmethod
    def forward(ctx, x, f, gate, scale, w_post, b_post, w_pre, b_pre, seen, post, pre, eps_post, eps_pre, keep):
        lib = L.load()
        x, f, gate, scale, w_post, b_post, w_pre, b_pre = (
            None if t is None else t.detach().contiguous()
            for t in (x, f, gate, scale, w_post, b_post, w_pre, b_pre))
        rows, C = x.shape
        dev = x.device
        G = 0 if gate is None else gate.shape[1]
        out = torch.empty_like(x)
        h = torch.empty_like(x) if pre else None
        wants = keep is not None
        keep8 = keep == "int8"
        xq = packed.empty_codes(rows, C, dev) if keep8 and pre else (None, None)
        fq = packed.empty_codes(rows, C, dev) if keep8 and f is not None else (None, None)
        stats = torch.empty((4, rows), dtype=torch.float32, device=dev) if wants and (pre or post) else None
        L.launch(dev, lib.mvf_residual_norm_forward, x.data_ptr(), _addr(f), packed.ROW_TYPES[x.dtype], rows, C,
                 _addr(gate), G, _addr(seen), _addr(scale), post, _addr(w_post), _addr(b_post), eps_post,
                 pre, _addr(w_pre), _addr(b_pre), eps_pre, out.data_ptr(), _addr(h), _addr(xq[0]), _addr(xq[1]),
                 _addr(fq[0]), _addr(fq[1]), _addr(stats))
        if wants:
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(
                x if pre and not keep8 else None, xq[0], xq[1], None if keep8 else f, fq[0], fq[1],
                gate, scale, w_post, b_post, w_pre, seen, stats)
            ctx.args = rows, C, G, post, pre, x.dtype, dev
        return (out, h) if pre else out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_h=None):
        nothing = (None,) * 14
        if d_out is None and d_h is None:
            return nothing
        lib = L.load()
        x, xc, xe, f, fc, fe, gate, scale, w_post, b_post, w_pre, seen, stats = ctx.saved_tensors
        rows, C, G, post, pre, dtype, dev = ctx.args
        d_out = None if d_out is None else d_out.contiguous()
        d_h = None if d_h is None else d_h.contiguous()
        need = ctx.needs_input_grad

        def empty(wanted, shape, kind=torch.float32):
            return torch.empty(shape, dtype=kind, device=dev) if wanted else None

        dx = empty(need[0], (rows, C), dtype)
        df = empty(need[1], (rows, C), dtype)
        dgate = empty(need[2], (rows, G))
        vectors = [empty(need[i], (C,)) for i in range(3, 8)]
        nbytes = lib.mvf_residual_norm_workspace_bytes(rows, C) if any(need[3:8]) else 0
        ws = L.workspace(nbytes, dev) if nbytes else None
        L.launch(dev, lib.mvf_residual_norm_backward, _addr(d_out), _addr(d_h), _addr(x), _addr(xc), _addr(xe),
                 _addr(f), _addr(fc), _addr(fe), packed.ROW_TYPES[dtype], rows, C, _addr(gate), G, _addr(seen),
                 _addr(scale), post, _addr(w_post), _addr(b_post), pre, _addr(w_pre), _addr(stats), _addr(dx),
                 _addr(df), _addr(dgate), *map(_addr, vectors), _addr(ws), nbytes)
        return (dx, df, dgate, *vectors) + nothing[8:]


def residual_norm(x, f, post=None, pre=None, gate=None, scale=None, seen=None, keep=None):
    """``out = x + scale * gate * post(f)`` and, with ``pre``, ``h = pre(out)``:
    returns ``out`` or ``(out, h)``, of the shape and type of x.

    :param x: [..., C] float32, bfloat16 or float16 rows on the HIP device, C <= 4096
    :param f: rows like x, the branch's output; None: out = x (the norm in front of
        the first branch)
    :param post, pre: nn.RMSNorm or nn.LayerNorm over the C channels, or None; their weights,
        biases and eps are read, the modules are not called (hooks on them do not run)
    :param gate: [...] or [..., G] with C % G == 0, G groups of neighbouring channels
    :param scale: [C], one element, or a number
    :param seen: [...] bool; where False nothing is added and f is not read, so
        whatever it holds there (NaN included) reaches neither out nor a gradient
    :param keep: what the backward keeps of x and f: 'float32' (the rows as they
        are, whatever their type), 'int8' (``packed`` rows, gradients then come from
        the values read back), or None: as ``training.keep_activations`` says

    Arithmetic is float32, out and h are rounded once (h from the unrounded out).
    Differentiable once with respect to x, f, gate, scale and the norms'
    parameters."""
    packed._check_rows(x, "residual_norm")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _MAX_C:
        raise ValueError(f"residual_norm expects rows of 1 to {_MAX_C} channels, got {tuple(x.shape)}")
    if f is None and not (post is None and gate is None and scale is None and seen is None):
        raise ValueError("residual_norm: post, gate, scale and seen need f")
    if f is None and pre is None:
        raise ValueError("residual_norm: nothing to do without f and without pre")
    shape, C = x.shape, x.shape[-1]
    if f is not None and (f.shape != shape or f.dtype != x.dtype or f.device != x.device):
        raise ValueError(f"residual_norm: f is {tuple(f.shape)} {f.dtype} on {f.device}, "
                         f"x is {tuple(shape)} {x.dtype} on {x.device}")
    k_post, w_post, b_post, eps_post = _norm_args(post, C, x, "post")
    k_pre, w_pre, b_pre, eps_pre = _norm_args(pre, C, x, "pre")
    flat = x.dim() == 2         # (views only where they are needed: each is a node of the graph)
    rows = x if flat else x.reshape(-1, C)
    if gate is not None:
        if gate.device != x.device or not gate.is_floating_point():
            raise ValueError("residual_norm: gate must hold floating-point values on the device of the rows")
        if gate.shape == shape[:-1]:
            gate = gate.unsqueeze(-1)
        if gate.shape[:-1] != shape[:-1] or gate.dim() != len(shape) or gate.shape[-1] < 1 or C % gate.shape[-1] != 0:
            raise ValueError(f"residual_norm: gate {tuple(gate.shape)} does not fit rows {tuple(shape)}: one value per "
                             f"row and channel group, in a number of groups that divides {C}")
        gate = gate.float() if flat else gate.float().reshape(-1, gate.shape[-1])
    if scale is not None:
        if not torch.is_tensor(scale):
            scale = torch.full((C,), float(scale), dtype=torch.float32, device=x.device)
        scale = _vector(scale, C, x, "scale")
    if seen is not None:
        if seen.dtype != torch.bool or seen.shape != shape[:-1] or seen.device != x.device:
            raise ValueError(f"residual_norm: seen must be a bool tensor {tuple(shape[:-1])} on the device of the rows")
        seen = (seen if flat else seen.reshape(-1)).contiguous()
    if f is not None and not flat:
        f = f.reshape(-1, C)
    leaves = (rows, f, gate, scale, w_post, b_post, w_pre, b_pre)
    keep = training.kept_form(keep)
    if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in leaves)):
        keep = None
    got = _ResidualNorm.apply(*leaves, seen, k_post, k_pre, eps_post, eps_pre, keep)
    if flat:
        return got
    return (got[0].view(shape), got[1].view(shape)) if k_pre else got.view(shape)
