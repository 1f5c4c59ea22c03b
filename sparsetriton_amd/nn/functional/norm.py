"""Per-sample batch normalisation of sparse features (``sparsetriton/nn/functional/norm.py:20-112``).

``sparse_batch_norm`` keeps the reference's signature and semantics: in
training each channel of each sample (rows with the same ``coords[:, 0]``) is
normalised by that sample's mean and biased variance, and the running
statistics move by ``momentum`` towards the mean over the batch's samples of
those statistics; in evaluation the running statistics are used.  Affine
``weight`` / ``bias`` are optional.

``sparse_batch_norm_act`` is the same normalisation with the residual add and
ReLU of the reference's blocks (``nn/modules/blocks.py:21-124``) fused into its
output pass: ``act(bn(x) + residual)``.

Both run as HIP kernels (``st_bn_forward`` / ``st_bn_backward``): two
deterministic statistics passes and one output pass forward, one statistics
pass and one gradient pass backward, each autograd-differentiable in the
features, the residual and the affine parameters.

``sparse_layer_norm`` normalises each row over its channels, with the residual
add of a pre-norm transformer block in the same pass (``st_ln_forward`` /
``st_ln_backward``).
"""

import ctypes
import functools
from typing import Optional, Tuple, Union

import torch

from sparsetriton_amd import _lib
from sparsetriton_amd.tensor import SparseTensor
from sparsetriton_amd.utils.utils import once_differentiable, refuse_tangents

__all__ = ["sparse_batch_norm", "sparse_batch_norm_act", "sparse_layer_norm"]


def _f32(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if t is None:
        return None
    return t.detach().to(torch.float32).contiguous()


@functools.lru_cache(maxsize=256)
def _workspace_floats(n: int, C: int, B: int) -> int:
    floats = ctypes.c_int64()
    _lib.call("st_bn_workspace", n, C, B, ctypes.byref(floats))
    return floats.value


def _workspace(n: int, C: int, B: int, device) -> torch.Tensor:
    return torch.empty((_workspace_floats(n, C, B),), dtype=torch.float32, device=device)


class _BatchNormAct(torch.autograd.Function):
    """out = act(bn(feats) + residual); statistics per sample in training."""

    @staticmethod
    def forward(ctx, feats, weight, bias, residual, coords, batch_size, running_mean, running_var, training, eps,
                momentum, relu):
        _lib.require_device(feats, "SparseTensor features")
        x = feats.contiguous()
        n, C = x.shape
        dev = x.device
        B = max(int(batch_size), 1)
        if B > 4096:
            raise ValueError(f"sparse batch norm supports at most 4096 samples per batch (got {B})")
        res = residual.contiguous() if residual is not None else None
        if res is not None and (res.shape != x.shape or res.dtype != x.dtype):
            raise ValueError("the residual must match the features' shape and dtype")
        w32, b32 = _f32(weight), _f32(bias)
        out = torch.empty_like(x)
        s = _lib.stream_of(dev)
        if training:
            mean, invstd = torch.empty((2, B, C), dtype=torch.float32, device=dev).unbind(0)
            counts = torch.empty((B,), dtype=torch.int32, device=dev)
            ws = _workspace(n, C, B, dev)
            rm = rv = None
            if running_mean is not None:
                rm = running_mean if running_mean.dtype == torch.float32 and running_mean.is_contiguous() else \
                    running_mean.float().contiguous()
            if running_var is not None:
                rv = running_var if running_var.dtype == torch.float32 and running_var.is_contiguous() else \
                    running_var.float().contiguous()
            _lib.call("st_bn_forward", _lib.ptr(x), n, C, _lib.feat_code(x.dtype), _lib.ptr(coords),
                      _lib.coord_code(coords.dtype), B, _lib.ptr(w32), _lib.ptr(b32), _lib.ptr(res), int(relu), 1,
                      float(eps), float(momentum), _lib.ptr(rm), _lib.ptr(rv), _lib.ptr(mean), _lib.ptr(invstd),
                      _lib.ptr(counts), _lib.ptr(ws), ws.numel(), _lib.ptr(out), s)
            if rm is not None and rm is not running_mean:
                running_mean.copy_(rm)
            if rv is not None and rv is not running_var:
                running_var.copy_(rv)
        else:
            if running_mean is None or running_var is None:
                raise ValueError("evaluation-mode batch norm needs running_mean and running_var")
            mean = torch.empty((C,), dtype=torch.float32, device=dev)
            invstd = torch.empty((C,), dtype=torch.float32, device=dev)
            counts = None
            rm32, rv32 = _f32(running_mean), _f32(running_var)
            _lib.call("st_bn_forward", _lib.ptr(x), n, C, _lib.feat_code(x.dtype), _lib.ptr(coords),
                      _lib.coord_code(coords.dtype), B, _lib.ptr(w32), _lib.ptr(b32), _lib.ptr(res), int(relu), 0,
                      float(eps), float(momentum), _lib.ptr(rm32), _lib.ptr(rv32), _lib.ptr(mean),
                      _lib.ptr(invstd), None, None, 0, _lib.ptr(out), s)
        # the output is needed only for the ReLU mask (so an in-place op on a plain output stays legal)
        ctx.save_for_backward(x, out if relu else None, coords, w32, mean, invstd, counts)
        ctx.meta = (B, bool(training), bool(relu), residual is not None, weight, bias)
        return out

    @staticmethod
    def backward(ctx, dout):
        x, out, coords, w32, mean, invstd, counts = ctx.saved_tensors
        B, training, relu, has_res, weight, bias = ctx.meta
        n, C = x.shape
        dev = x.device
        g = dout.contiguous()
        if g.dtype != x.dtype:
            g = g.to(x.dtype)
        need_x = ctx.needs_input_grad[0]
        dx = torch.empty_like(x)
        dres = torch.empty_like(x) if (has_res and ctx.needs_input_grad[3]) else None
        dw = torch.empty((C,), dtype=torch.float32, device=dev) if (weight is not None and ctx.needs_input_grad[1]) \
            else None
        db = torch.empty((C,), dtype=torch.float32, device=dev) if (bias is not None and ctx.needs_input_grad[2]) \
            else None
        ws = _workspace(n, C, B if training else 1, dev)
        _lib.call("st_bn_backward", _lib.ptr(x), _lib.ptr(out), _lib.ptr(g), n, C, _lib.feat_code(x.dtype),
                  _lib.ptr(coords), _lib.coord_code(coords.dtype), B, _lib.ptr(w32), int(relu), int(training),
                  _lib.ptr(mean), _lib.ptr(invstd), _lib.ptr(counts), _lib.ptr(ws), ws.numel(), _lib.ptr(dx),
                  _lib.ptr(dres), _lib.ptr(dw), _lib.ptr(db), _lib.stream_of(dev))
        dw = dw.to(weight.dtype) if dw is not None else None
        db = db.to(bias.dtype) if db is not None else None
        return (dx if need_x else None, dw, db, dres, None, None, None, None, None, None, None, None)


def sparse_batch_norm_act(
    tensor: SparseTensor,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    running_mean: Optional[torch.Tensor] = None,
    running_var: Optional[torch.Tensor] = None,
    training: bool = True,
    eps: float = 1e-5,
    momentum: float = 0.1,
    residual: Optional[torch.Tensor] = None,
    relu: bool = False,
) -> SparseTensor:
    """``act(bn(tensor.F) + residual)`` as one kernel pass (``act`` = ReLU or identity)."""
    if tensor.F.dim() != 2:
        raise ValueError(f"Expected 2D input, got {tensor.F.dim()}D")
    feats = _BatchNormAct.apply(tensor.F, weight, bias, residual, tensor.C.contiguous(), tensor.batch_size,
                                running_mean, running_var, bool(training), float(eps), float(momentum), bool(relu))
    return tensor.replace(feats)


def sparse_batch_norm(
    tensor: SparseTensor,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    running_mean: Optional[torch.Tensor] = None,
    running_var: Optional[torch.Tensor] = None,
    training: bool = True,
    eps: float = 1e-5,
    momentum: float = 0.1,
) -> SparseTensor:
    """Per-sample batch normalisation (reference ``norm.py:20-112``)."""
    return sparse_batch_norm_act(tensor, weight, bias, running_mean, running_var, training, eps, momentum)


@functools.lru_cache(maxsize=256)
def _ln_workspace_floats(n: int, C: int, code: int) -> int:
    floats = ctypes.c_int64()
    _lib.call("st_ln_backward_workspace", n, C, code, ctypes.byref(floats))
    return floats.value


def _ln_param(t, dtype):
    return t if t is None or (t.dtype is dtype and t.is_contiguous()) else t.detach().to(dtype).contiguous()


def _ln_params(x, weight, bias):
    """weight and bias as the kernels take them: one dtype for both, the features' or fp32."""
    given = weight if weight is not None else bias
    dt = torch.float32 if given is None else given.dtype
    if (dt is not x.dtype and dt is not torch.float32) or (weight is not None and bias is not None and bias.dtype is not dt):
        dt = torch.float32
    return _ln_param(weight, dt), _ln_param(bias, dt), _lib.FEAT_DTYPES[dt]


def _ln_forward(x, weight, bias, residual, eps, stats):
    C = x.shape[-1]
    x = x.contiguous()
    n = x.numel() // C
    res = residual.contiguous() if residual is not None else None
    w, b, wcode = _ln_params(x, weight, bias)
    y = torch.empty_like(x)
    h = torch.empty_like(x) if res is not None else None
    mean = rstd = None
    if stats:
        mean, rstd = torch.empty((2, n), dtype=torch.float32, device=x.device).unbind(0)
    ptr = _lib.ptr
    _lib.call("st_ln_forward", x.data_ptr(), ptr(res), n, C, _lib.FEAT_DTYPES[x.dtype], ptr(w), ptr(b), wcode, eps,
              ptr(h), y.data_ptr(), ptr(mean), ptr(rstd), _lib.stream_of(x.device))
    return y, h, x, w, wcode, mean, rstd


class _LayerNorm(torch.autograd.Function):
    """(y,) or, with a residual, (y, h): y = norm(h), h = x + residual."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        y, h, xc, w, wcode, mean, rstd = _ln_forward(x, weight, bias, residual, eps, True)
        ctx.save_for_backward(xc if h is None else h, w, mean, rstd)
        ctx.meta = (wcode, None if weight is None else weight.dtype, None if bias is None else bias.dtype)
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, w, mean, rstd = ctx.saved_tensors
        wcode, wdt, bdt = ctx.meta
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        C = h.shape[-1]
        n = h.numel() // C
        if dy is None:  # nothing arrives at y: the stream's gradient goes through
            def zero(dt):
                return torch.zeros((C,), dtype=dt, device=h.device)
            return dh, zero(wdt) if need_w else None, zero(bdt) if need_b else None, dh if need_r else None, None
        dy = dy.contiguous()
        dh = dh.contiguous() if dh is not None else None
        dx = torch.empty_like(h) if (need_x or need_r) else None
        wtype = torch.float32 if wcode == _lib.FEAT_DTYPES[torch.float32] else h.dtype
        dw = torch.empty((C,), dtype=wtype, device=h.device) if need_w else None
        db = torch.empty((C,), dtype=wtype, device=h.device) if need_b else None
        ws, floats = None, 0
        if need_w or need_b:
            floats = _ln_workspace_floats(n, C, _lib.FEAT_DTYPES[h.dtype])
            ws = torch.empty((floats,), dtype=torch.float32, device=h.device)
        _lib.call("st_ln_backward", _lib.ptr(h), _lib.ptr(dy), _lib.ptr(dh), n, C, _lib.FEAT_DTYPES[h.dtype],
                  _lib.ptr(w), wcode, _lib.ptr(mean), _lib.ptr(rstd), _lib.ptr(ws), floats, _lib.ptr(dx),
                  _lib.ptr(dw), _lib.ptr(db), _lib.stream_of(h.device))
        if dw is not None and dw.dtype != wdt:
            dw = dw.to(wdt)
        if db is not None and db.dtype != bdt:
            db = db.to(bdt)
        return dx if need_x else None, dw, db, dx if need_r else None, None


def sparse_layer_norm(
    input: Union[SparseTensor, torch.Tensor],
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    eps: float = 1e-5,
    residual: Optional[Union[SparseTensor, torch.Tensor]] = None,
) -> Union[SparseTensor, torch.Tensor, Tuple]:
    """Layer norm of each row over its channels: ``norm(x) * weight + bias``.

    With ``residual`` (same shape and dtype), the pre-norm block's add runs in the same pass and
    the result is ``(norm(h), h)`` with ``h = x + residual``, the stream that goes on.  ``input``
    (and ``residual``) are a ``SparseTensor`` or a tensor (..., C) of float32, float16 or bfloat16;
    the results are of the same kind.  Statistics and products are fp32; the gradients of
    ``weight`` and ``bias`` are added in a fixed order.  There is no forward-mode derivative: a tangent
    on an input raises.
    """
    x = input.F if isinstance(input, SparseTensor) else input
    res = residual.F if isinstance(residual, SparseTensor) else residual
    _lib.require_device(x, "layer norm input")
    _lib.feat_code(x.dtype)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"layer norm needs at least one channel (got shape {tuple(x.shape)})")
    for t, what in ((weight, "weight"), (bias, "bias")):
        if t is not None and (t.shape != x.shape[-1:] or t.device != x.device):
            raise ValueError(f"layer norm {what} must be ({x.shape[-1]},) on {x.device} "
                             f"(got {tuple(t.shape)} on {t.device})")
        if t is not None:
            _lib.feat_code(t.dtype)
    if res is not None and (res.shape != x.shape or res.dtype != x.dtype or res.device != x.device):
        raise ValueError("the residual must match the input's shape, dtype and device")
    refuse_tangents("sparse_layer_norm", x, weight, bias, res)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, res)):
        out = _LayerNorm.apply(x, weight, bias, res, float(eps))
        y, h = out if res is not None else (out, None)
    else:
        y, h = _ln_forward(x, weight, bias, res, float(eps), False)[:2]
    if isinstance(input, SparseTensor):
        y, h = input.replace(y), (input.replace(h) if h is not None else None)
    return y if h is None else (y, h)
