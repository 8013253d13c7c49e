"""Operators around a network's last matrix product, as HIP kernels of libazamd: the loss of a linear layer over many classes
with its gradient (the logits are never stored), dropout from a counter-based generator (the mask is never stored), and the product
in 8-bit integers with a scale for each token and channel.

They take GPU tensors of float32, bfloat16 or float16 and run on the current stream of the tensors' device; there is no CPU
fallback. Upstream computes the loss from stored logits (go_zero/train.py:537-541) and has no counterpart of the other two.
Derivatives are first ones in reverse mode: a dual tensor (torch.autograd.forward_ad) is refused, and a second derivative raises. So does
a call under torch.jit.trace or make_fx, whose record would lack the kernels; torch.cuda.graph captures them."""
from __future__ import annotations

import ctypes as C

import torch
from torch import nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from . import _native as N

_DTYPES = {torch.float32: N.AZ_DT_F32, torch.bfloat16: N.AZ_DT_BF16, torch.float16: N.AZ_DT_F16}
_REDUCE = {"none": N.AZ_REDUCE_NONE, "mean": N.AZ_REDUCE_MEAN, "sum": N.AZ_REDUCE_SUM}


def _need(ok: bool, what: str):
    if not ok:
        raise ValueError(what)


def _recorded() -> bool:
    """The call is being recorded by torch.jit.trace or make_fx. They see torch operations only: the record would allocate the result and
    return it as it is, without the kernel that fills it."""
    return torch._C._is_tracing() or (torch._C._len_torch_dispatch_stack() > 0 and get_proxy_mode() is not None)


def _on_gpu(name: str, x: torch.Tensor, *others):
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise N.NativeError(f"alphazero_amd.head.{name} needs tensors on a GPU (no CPU fallback)")
    dev = x.device
    for t in others:
        if t is not None and t.device != dev:
            raise ValueError(f"{name}: tensors on {x.device} and {t.device}")
    if _recorded():
        raise NotImplementedError(f"{name} cannot be traced: capture it into a HIP graph (torch.cuda.graph) instead")
    # a dual tensor does not ask for a gradient: without this its tangent would be lost and the derivative read as zero
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (x, *others)):
        raise NotImplementedError(f"{name} has no forward-mode derivative")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., n] as [rows, n] with neighbouring columns; a copy only where the layout asks for one."""
    t = t.reshape(-1, t.shape[-1]) if t.dim() != 2 else t
    if (t.stride(1) != 1 and t.shape[1] > 1) or (t.stride(0) < t.shape[1] and t.shape[0] > 1):
        t = t.contiguous()
    return t


def _pitch(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


# torch.cuda.current_device and current_stream without their checks and objects: 0.1 instead of 0.5 to 3 us of host time each
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device) -> int:
    return _raw_stream(device.index) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


def _native(device, name: str, *args) -> int:
    """A call of the library with `device` as the current one."""
    fn = getattr(N.lib(), name)
    if _current_device() == device.index:
        return N.check(fn(*args), name)
    with torch.cuda.device(device):
        return N.check(fn(*args), name)


def _scratch(size: int, device) -> torch.Tensor:
    return torch.empty(max(1, size), dtype=torch.uint8, device=device)


# ------------------------------------------------------------------------------------------------ loss of a linear layer
def _ce_args(x, weight, bias, target, ignore_index, reduction, entropy_coeff, precise):
    dense = target.dim() == 2
    return N.AzLinearCeArgs(x.data_ptr(), weight.data_ptr(), _ptr(bias), target.data_ptr(), x.shape[0], x.shape[1], weight.shape[0], _pitch(x),
                            _pitch(weight), _pitch(target) if dense else 0, ignore_index, _DTYPES[x.dtype], dense, _REDUCE[reduction] | (N.AZ_PRECISE_GRADIENT if precise else 0), entropy_coeff)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, target, ignore_index, reduction, entropy_coeff, precise, parts):
        a = _ce_args(x, weight, bias, target, ignore_index, reduction, entropy_coeff, precise)
        rows, dev = x.shape[0], x.device
        shape = (rows,) if reduction == "none" else ()
        out = tuple(torch.empty(shape, dtype=torch.float32, device=dev) for _ in range(3 if parts else 1))
        kept = torch.empty(4 * rows + 4, dtype=torch.float32, device=dev)
        if rows:
            r = C.byref(a)
            size = N.check(N.lib().az_linear_ce_workspace(r, 0), "az_linear_ce_workspace")
            ws = _scratch(size, dev)
            _native(dev, "az_linear_ce_forward", r, kept.data_ptr(), out[0].data_ptr(), out[1].data_ptr() if parts else None,
                    out[2].data_ptr() if parts else None, ws.data_ptr(), size, _stream(dev))
        else:       # an empty sum, a mean of nothing
            for o in out:
                o.fill_(float("nan") if reduction == "mean" else 0.0)
        ctx.save_for_backward(x, weight, bias, target, kept)
        ctx.args = (ignore_index, reduction, entropy_coeff, precise)
        if parts:
            ctx.mark_non_differentiable(out[1], out[2])
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    def backward(ctx, grad, *_parts):
        if grad is None:
            return (None,) * 9
        x, weight, bias, target, kept = ctx.saved_tensors
        with torch.no_grad():
            found = _ce_backward(x, weight, bias, target, kept, grad, ctx.args, ctx.needs_input_grad[:3])
        if torch.is_grad_enabled():        # create_graph: the gradients depend on all of these
            found = tuple(None if g is None else _NoSecondDerivative.apply(g, grad, x, weight, bias) for g in found)
        return (*found, None, None, None, None, None, None)


def _ce_backward(x, weight, bias, target, kept, grad, args, need):
    a = _ce_args(x, weight, bias, target, *args)
    need_x, need_w, need_b = need
    dev = x.device
    grad = grad.to(torch.float32).contiguous()
    gx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
    gw = torch.empty(weight.shape, dtype=x.dtype, device=dev) if need_w else None
    gb = torch.empty(bias.shape, dtype=x.dtype, device=dev) if bias is not None and need_b else None
    if not x.shape[0]:
        for g in (gw, gb):
            if g is not None:
                g.zero_()
        return gx, gw, gb
    r = C.byref(a)
    size = N.check(N.lib().az_linear_ce_workspace(r, 1), "az_linear_ce_workspace")
    ws = _scratch(size, dev)
    _native(dev, "az_linear_ce_backward", r, kept.data_ptr(), grad.data_ptr(), _ptr(gx), _ptr(gw), _ptr(gb), ws.data_ptr(), size, _stream(dev))
    return gx, gw, gb


class _NoSecondDerivative(torch.autograd.Function):
    """A gradient that says so when it is differentiated, instead of being taken for a constant."""

    @staticmethod
    def forward(ctx, g, *depends):
        ctx.mark_dirty(g)        # the same tensor, with this node behind it: a view could not be changed in place
        return g

    @staticmethod
    def backward(ctx, *_grads):
        raise NotImplementedError("linear_cross_entropy has no second derivative")


def linear_cross_entropy(x, weight, target, bias=None, *, ignore_index: int = -100, reduction: str = "mean", entropy_coeff: float = 0.0,
                         parts: bool = False, precise_gradient: bool = False):
    """Cross entropy of softmax(x weight^T + bias) minus entropy_coeff times that softmax' entropy, without ever holding the logits.

    x [..., features], weight [classes, features], bias [classes] or None: one dtype (float32, bfloat16, float16; under autocast they
    are cast to its dtype like the operands of a linear layer). target: int64 class indices of x's leading shape, or floating target
    weights [..., classes] (a search's visit distribution; they need not sum to one; no gradient). Rows whose index is ignore_index
    count nowhere: loss and gradient zero whatever they hold, and the mean is over the other rows. reduction "mean", "sum" or
    "none". Returns the float32 loss; with parts=True (loss, cross entropy, entropy), the last two without gradient.

    An index outside 0..classes-1 that is not ignore_index gives a NaN loss and NaN gradients (the check is on the device, nothing
    waits for it). Everything is accumulated in float32; between the products of the backward pass the gradient of the logits keeps
    22 bits for float32 inputs. For 16-bit ones it keeps 16 bits or more with up to 128 rows or 512 classes and is rounded to the
    inputs' type beyond, which adds up to 20 % to the error that rounding the results makes, with target weights up to 35 %;
    precise_gradient=True keeps 16 bits or more there too, in up to twice the time.

    float32 gradients, but for up to 16 rows of a large weight: the sums over the classes (for x) and over the rows (for the weight) hold
    weight and x to 22 bits each, and to 2^-49 of that matrix' largest value, so values below 2^-27 of the largest lose bits.

    Scratch memory of the backward pass: up to 2 GB whatever the number of classes, 6 to 8 bytes for each element of x (float32: 12), and with
    up to 16 rows 64 bytes for each class. Of the forward pass: for float32, and for rows that are not a multiple of 16 bytes, a copy of x and up
    to 512 MB of the weight; 16 bytes for each row and 64 to 256 classes (24 with target weights). More than a million rows or features
    take more: the smallest piece is 256 classes."""
    _on_gpu("linear_cross_entropy", x, weight, target, bias)
    _need(reduction in _REDUCE, 'reduction is "none", "mean" or "sum"')
    _need(x.dim() >= 1 and weight.dim() == 2 and x.shape[-1] == weight.shape[1], f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not fit")
    _need(weight.shape[0] >= 1 and weight.shape[1] >= 1, "classes and features are at least 1")
    _need(bias is None or tuple(bias.shape) == (weight.shape[0],), "bias has one value per class")
    if torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        x, weight, bias = x.to(dt), weight.to(dt), None if bias is None else bias.to(dt)
    _need(x.dtype in _DTYPES, f"x is float32, bfloat16 or float16, not {x.dtype}")
    _need(weight.dtype == x.dtype and (bias is None or bias.dtype == x.dtype), "x, weight and bias have one dtype")
    lead = x.shape[:-1]
    if target.is_floating_point():
        _need(target.shape == (*lead, weight.shape[0]), f"target weights {tuple(target.shape)} do not fit {(*lead, weight.shape[0])}")
        _need(not (target.requires_grad and torch.is_grad_enabled()), "the target has no gradient: detach it")
        target = _rows(target.to(torch.float32))
    else:
        _need(target.dtype == torch.int64, f"class indices are int64, not {target.dtype}")
        _need(target.shape == lead, f"target {tuple(target.shape)} does not fit {tuple(lead)}")
        target = target.reshape(-1).contiguous()
    x2 = _rows(x)
    out = _LinearCrossEntropy.apply(x2, _rows(weight), bias if bias is None else bias.contiguous(), target, int(ignore_index), reduction,
                                    float(entropy_coeff), bool(precise_gradient), bool(parts))
    if reduction == "none" and len(lead) != 1:
        out = tuple(t.reshape(lead) for t in out)
    return out if parts else out[0]


# ------------------------------------------------------------------------------------------------ dropout
class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, seed_tensor, threshold, seed, offset):
        ctx.save_for_backward(seed_tensor)
        ctx.args = (threshold, seed, offset)
        return _dropout(x, residual, seed_tensor, threshold, seed, offset)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        gx = None
        if ctx.needs_input_grad[0]:
            gx = _dropout(grad.contiguous(), None, ctx.saved_tensors[0], *ctx.args)
        return gx, grad if ctx.needs_input_grad[1] else None, None, None, None, None


def _dropout(x, residual, seed_tensor, threshold, seed, offset):
    y = torch.empty_like(x)      # contiguous, as x is here
    dev = x.device
    _native(dev, "az_dropout", x.data_ptr(), _ptr(residual), y.data_ptr(), x.numel(), _DTYPES[x.dtype], threshold, seed, _ptr(seed_tensor), offset,
            _stream(dev))
    return y


def dropout(x, p: float, seed, offset: int = 0, *, residual=None):
    """x with every element dropped (zero) with probability p and the others scaled by 1 / (1 - p), plus `residual`.

    The mask is a function of (seed, offset, position), made again in the backward pass instead of being stored: Philox4x32-10 with key
    `seed` and counter (position // 8 in row-major order, offset), 16 bits per element, so p is taken to the nearest 1 / 65536. Use
    another offset for every call that shall have another mask. seed and offset: whole numbers below 2^64; seed may also be an int64
    tensor of one element on x's device, read when the kernel runs (a captured graph then replays with whatever it holds; it has to
    hold the same value in the backward pass). What is dropped is selected away, never multiplied: it may be infinite or NaN."""
    _on_gpu("dropout", x, residual)
    _need(x.dtype in _DTYPES, f"x is float32, bfloat16 or float16, not {x.dtype}")
    _need(residual is None or (residual.shape == x.shape and residual.dtype == x.dtype), "residual has x's shape and dtype")
    _need(0.0 <= p <= 1.0, "p is a probability")
    _need(0 <= int(offset) < 1 << 64, "offset is 0..2^64-1")
    seed_tensor, number = None, 0
    if isinstance(seed, torch.Tensor):
        _need(seed.dtype == torch.int64 and seed.numel() == 1 and seed.device == x.device, "a seed tensor is one int64 on x's device")
        seed_tensor = seed
    else:
        number = int(seed)
        _need(0 <= number < 1 << 64, "seed is 0..2^64-1")
    x = x.contiguous()
    residual = None if residual is None else residual.contiguous()
    threshold = round(65536 * float(p))
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, seed_tensor, threshold, number, int(offset))
    return _dropout(x, residual, seed_tensor, threshold, number, int(offset))


# ------------------------------------------------------------------------------------------------ 8-bit integers
def quantize_rows(x):
    """(q int8 [..., n], scale float32 [...]) with x ~ q * scale: scale = max|row| / 127, q = the nearest whole number of
    127 x / max|row| (ties to even). A row of zeros has scale 0; a row with an infinity or NaN has q = 0 and scale NaN. Neither
    has a gradient."""
    _on_gpu("quantize_rows", x)
    _need(x.dtype in _DTYPES, f"x is float32, bfloat16 or float16, not {x.dtype}")
    _need(x.dim() >= 1 and x.shape[-1] >= 1, "a row has at least one element")
    x2 = _rows(x.detach())
    q = torch.empty(x2.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x2.shape[0], dtype=torch.float32, device=x.device)
    _native(x.device, "az_quantize_rows", x2.data_ptr(), _DTYPES[x.dtype], x2.shape[0], x2.shape[1], _pitch(x2), q.data_ptr(), q.shape[1],
            scale.data_ptr(), _stream(x.device))
    return q.reshape(x.shape), scale.reshape(x.shape[:-1])


def int8_linear(x, qweight, weight_scale, bias=None, *, x_scale=None, out_dtype=None):
    """y[..., n] = x_scale[...] * weight_scale[n] * sum_k x[..., k] qweight[n, k] + bias[n], the sum in 32-bit integers.

    x: float32, bfloat16 or float16, quantised row by row on the way as quantize_rows does it, or int8 with its x_scale (float32,
    x's leading shape). qweight int8 [channels, features] (at most 131071 features), weight_scale float32 [channels]. The output has
    x's dtype (float32 for int8 x) or out_dtype. Rows of qweight that start at multiples of 16 bytes are read in place. There is no
    gradient."""
    _on_gpu("int8_linear", x, qweight, weight_scale, bias, x_scale)
    shape, (channels, features) = x.shape, qweight.shape if qweight.dim() == 2 else (0, 0)
    whole = x.dtype == torch.int8
    if not (qweight.dtype == torch.int8 and channels >= 1 and 1 <= features <= 131071 and x.dim() >= 1 and shape[-1] == features
            and (whole or x.dtype in _DTYPES) and weight_scale.dtype == torch.float32 and weight_scale.shape == (channels,)
            and (bias is None or (bias.dtype in _DTYPES and bias.shape == (channels,))) and whole == (x_scale is not None)
            and (x_scale is None or (x_scale.dtype == torch.float32 and x_scale.shape == shape[:-1])) and (out_dtype is None or out_dtype in _DTYPES)):
        _int8_refuse(x, qweight, weight_scale, bias, x_scale, out_dtype)
    if torch.is_grad_enabled() and (x.requires_grad or weight_scale.requires_grad or (bias is not None and bias.requires_grad)
                                    or (x_scale is not None and x_scale.requires_grad)):
        raise ValueError("int8_linear has no gradient: call it under torch.no_grad() or with detached tensors")
    out_dtype = out_dtype or (torch.float32 if whole else x.dtype)
    dev = x.device
    y = torch.empty((*shape[:-1], channels), dtype=out_dtype, device=dev)
    if y.numel() == 0:
        return y
    x2, w = _rows(x), _rows(qweight)
    scale, wscale = None if x_scale is None else x_scale.reshape(-1).contiguous(), weight_scale.contiguous()
    b = None if bias is None else bias.contiguous()
    a = N.AzInt8Args(x2.data_ptr(), w.data_ptr(), _ptr(scale), wscale.data_ptr(), _ptr(b), y.data_ptr(), x2.shape[0], features, channels, _pitch(x2),
                     _pitch(w), N.AZ_DT_I8 if whole else _DTYPES[x.dtype], 0 if b is None else _DTYPES[b.dtype], _DTYPES[out_dtype])
    r = C.byref(a)
    size = N.check(N.lib().az_int8_workspace(r), "az_int8_workspace")
    ws = _scratch(size, dev) if size else None
    _native(dev, "az_int8_linear", r, _ptr(ws), size, _stream(dev))
    return y


def _int8_refuse(x, qweight, weight_scale, bias, x_scale, out_dtype):
    _need(x.dtype in _DTYPES or x.dtype == torch.int8, f"x is float32, bfloat16, float16 or int8, not {x.dtype}")
    _need(qweight.dtype == torch.int8 and qweight.dim() == 2, "qweight is an int8 matrix")
    _need(x.dim() >= 1 and x.shape[-1] == qweight.shape[1], f"x {tuple(x.shape)} and qweight {tuple(qweight.shape)} do not fit")
    _need(qweight.shape[0] >= 1 and 1 <= qweight.shape[1] <= 131071, "channels are at least 1, features 1..131071")
    _need(weight_scale.dtype == torch.float32 and tuple(weight_scale.shape) == (qweight.shape[0],), "weight_scale is one float32 per channel")
    _need(bias is None or (bias.dtype in _DTYPES and tuple(bias.shape) == (qweight.shape[0],)), "bias is one floating value per channel")
    _need((x_scale is not None) == (x.dtype == torch.int8), "x_scale comes with an int8 x, and only with it")
    _need(x_scale is None or (x_scale.dtype == torch.float32 and x_scale.shape == x.shape[:-1]), "x_scale is one float32 per row of x")
    raise ValueError(f"out_dtype is float32, bfloat16 or float16, not {out_dtype}")


class Int8Linear(nn.Module):
    """A linear layer whose weights are held in 8 bits with a scale per output channel and whose input is quantised per row: the
    serving form of a trained nn.Linear (on a GPU). Rows are laid out at multiples of 16 bytes once, here. As with int8_linear there is
    no gradient: an input that asks for one is refused."""

    def __init__(self, linear: nn.Linear):
        super().__init__()
        _on_gpu("Int8Linear", linear.weight)
        self.in_features, self.out_features = linear.in_features, linear.out_features
        q, scale = quantize_rows(linear.weight)
        store = torch.zeros((self.out_features, (self.in_features + 15) // 16 * 16), dtype=torch.int8, device=q.device)
        store[:, :self.in_features] = q
        self.register_buffer("qweight", store)
        self.register_buffer("weight_scale", scale)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().clone())

    def _apply(self, fn, recurse=True):
        """half(), bfloat16(), to(dtype) and type() are about the bias and the inputs: the 8-bit weights and their float32 scales are moved,
        never cast."""
        kept = {name: getattr(self, name) for name in ("qweight", "weight_scale")}
        super()._apply(fn, recurse)
        for name, v in kept.items():
            now = getattr(self, name)
            if now.dtype != v.dtype:
                setattr(self, name, v.to(now.device))
        return self

    def forward(self, x):
        return int8_linear(x, self.qweight[:, :self.in_features], self.weight_scale, self.bias)
