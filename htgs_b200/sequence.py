"""Operators for networks over sequences of Gaussians: what reads or refines a scene's Gaussians before they are rendered, one row for
each Gaussian in the order of a space-filling curve, 10^5 to 10^6 rows long.

* `add_rms_norm`, `add_rms_norm_fp8`   - root-mean-square norm of a residual stream with the residual's addition; the second leaves 8-bit codes
* `quantize_fp8`, `Fp8Matrix`          - 8-bit matrices with a power-of-two scale for each block of 128
* `fp8_matmul`, `fp8_linear`           - their matrix product; the second is differentiable and quantises its operands itself; `check_products` asks after their errors
* `gated_scan`, `gated_scan_step`      - gated linear recurrence over whole sequences (differentiable), and one step of it

Values are float32, float16 or bfloat16; sums, statistics and states are 32-bit.  Everything is queued on the current CUDA stream without a
host wait, can be captured in a CUDA graph, and gives the same bits for the same inputs.  There is no CPU fallback.  Derivatives
are reverse-mode: dual tensors of forward-mode differentiation are refused.  (No counterpart in the reference.)
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional, Tuple

import torch

from . import _native
from ._native import HtgsFp8Matrix, HtgsScan

__all__ = ["add_rms_norm", "add_rms_norm_fp8", "Fp8Matrix", "quantize_fp8", "fp8_matmul", "fp8_linear", "check_products", "gated_scan", "gated_scan_step"]

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_BLOCK = 128


def _compiled():
    """The compiled extension module where it is the active binding, else None: the functions here then do its work over ctypes."""
    mods = _native.pybind_modules()
    return mods[0] if mods else None


def _check(t, name: str, dtype=None, device=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must live on a CUDA device")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if dtype is None:
        if t.dtype not in _TYPES:
            raise TypeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    elif t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` as a matrix of its last dimension's rows; a copy only where its rows are not evenly spaced or not dense."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1]) if t.numel() else t.reshape(t.shape[:-1].numel(), t.shape[-1])
    if t.stride(1) != 1 and t.shape[1] != 1 or t.stride(0) < t.shape[1] and t.shape[0] > 1:
        t = t.contiguous()
    return t


def _call(device: torch.device, name: str, *args) -> None:
    """Calls a library function with the device current and its current stream as the last argument."""
    function = getattr(_native.lib(), name)
    stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() == device.index:
        _native.check(function(*args, stream))
    else:
        with torch.cuda.device(device):
            _native.check(function(*args, stream))


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _no_tangent(*tensors) -> None:
    """A tangent would be dropped without a word: a dual tensor need not want a gradient."""
    if any(t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("the sequence operators have no forward-mode derivative: unpack dual tensors first")


class _NoSecondDerivative(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *grads):
        return tuple(g.view_as(g) for g in grads)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("the sequence operators have no second derivative")


def _first_derivative(backward):
    """A backward pass whose gradients, where its graph is created, hang on a node that raises: a second derivative is an error where one is taken,
    and only there."""
    @functools.wraps(backward)
    def run(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        marked = iter(_NoSecondDerivative.apply(*(g.detach().requires_grad_() for g in out if g is not None)))
        return tuple(None if g is None else next(marked) for g in out)
    return run


# ---- norm ------------------------------------------------------------------------------------------------------------------


def _check_norm(x, weight, residual):
    _check(x, "x")
    _check(weight, "weight", x.dtype, x.device)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 8192:
        raise ValueError("x must have a last dimension of 1 to 8192 values")
    if weight.shape != x.shape[-1:]:
        raise ValueError(f"weight must have shape ({x.shape[-1]},), got {tuple(weight.shape)}")
    if residual is not None:
        _check(residual, "residual", x.dtype, x.device)
        if residual.shape != x.shape:
            raise ValueError(f"residual must have the shape of x, {tuple(x.shape)}, got {tuple(residual.shape)}")
    _no_tangent(x, weight, residual)


def _norm_forward(x, weight, residual, eps, with_rstd, to_codes):
    """(y or Fp8Matrix, sum or None, rstd or None) for matrices."""
    rows, width = x.shape
    weight = weight.contiguous()
    total = None if residual is None else torch.empty((rows, width), dtype=x.dtype, device=x.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if with_rstd else None
    if to_codes:
        y, out = None, _empty_fp8(rows, width, 1, x.device)
        codes, scales = out.codes, out.scales
    else:
        y = out = torch.empty((rows, width), dtype=x.dtype, device=x.device)
        codes = scales = None
    _call(x.device, "htgs_add_rms_norm", x.data_ptr(), x.stride(0), None if residual is None else residual.data_ptr(),
          0 if residual is None else residual.stride(0), weight.data_ptr(), _TYPES[x.dtype], rows, width, eps,
          None if y is None else y.data_ptr(), width, None if total is None else total.data_ptr(), width,
          None if rstd is None else rstd.data_ptr(), None if codes is None else codes.data_ptr(), 0 if codes is None else codes.stride(0),
          None if scales is None else scales.data_ptr(), 0 if scales is None else scales.stride(0))
    return out, total, rstd


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        xm, rm = _rows(x), None if residual is None else _rows(residual)
        y, total, rstd = _norm_forward(xm, weight, rm, eps, True, False)
        ctx.save_for_backward(xm, rm, weight, rstd)
        return (y.view(x.shape), total.view(x.shape)) if residual is not None else y.view(x.shape)

    @staticmethod
    @_first_derivative
    def backward(ctx, grad_y, grad_sum=None):
        x, residual, weight, rstd = ctx.saved_tensors
        if grad_y is None:
            return grad_sum, torch.zeros_like(weight), grad_sum, None
        shape = grad_y.shape
        rows, width = x.shape
        gy, gs = _rows(grad_y), None if grad_sum is None else _rows(grad_sum)
        grad_x = torch.empty((rows, width), dtype=x.dtype, device=x.device)
        grad_weight = torch.empty(width, dtype=x.dtype, device=x.device)
        size = _native.lib().htgs_add_rms_norm_backward_scratch_bytes(rows, width)
        scratch = torch.empty(size, dtype=torch.uint8, device=x.device)
        _call(x.device, "htgs_add_rms_norm_backward", gy.data_ptr(), gy.stride(0), None if gs is None else gs.data_ptr(),
              0 if gs is None else gs.stride(0), x.data_ptr(), x.stride(0), None if residual is None else residual.data_ptr(),
              0 if residual is None else residual.stride(0), weight.contiguous().data_ptr(), rstd.data_ptr(), _TYPES[x.dtype],
              rows, width, grad_x.data_ptr(), width, grad_weight.data_ptr(), scratch.data_ptr(), size)
        grad_x = grad_x.view(shape)
        return grad_x, grad_weight, None if residual is None else grad_x, None


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, stream) with stream = x + residual and y = stream / sqrt(mean(stream^2) + eps) * weight over the last dimension (1 to 8192
    values).  Without a residual the stream is x itself.  x, weight and residual have one type.  y is computed from the
    unrounded sum.  Differentiable in x, weight and residual."""
    compiled = _compiled()
    if compiled:
        return compiled.add_rms_norm(x, weight, residual, eps)
    _check_norm(x, weight, residual)
    if _wants_grad(x, weight, residual):
        return _AddRmsNorm.apply(x, weight, residual, float(eps)) if residual is not None else (_AddRmsNorm.apply(x, weight, None, float(eps)), x)
    y, total, _ = _norm_forward(_rows(x), weight, None if residual is None else _rows(residual), float(eps), False, False)
    return y.view(x.shape), x if total is None else total.view(x.shape)


def add_rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                     eps: float = 1e-6) -> Tuple["Fp8Matrix", torch.Tensor]:
    """`add_rms_norm` whose y leaves as an `Fp8Matrix` of x.shape[:-1].numel() rows, quantised from 32-bit values with a scale for each row and
    128 columns: what `fp8_matmul` takes.  For inference: it has no gradient and refuses inputs that want one."""
    compiled = _compiled()
    if compiled:
        codes, scales, total = compiled.add_rms_norm_fp8(x, weight, residual, eps)
        return _fp8(codes, scales, 1), total
    _check_norm(x, weight, residual)
    if _wants_grad(x, weight, residual):
        raise RuntimeError("add_rms_norm_fp8 has no gradient: use add_rms_norm and fp8_linear in training, or torch.no_grad()")
    q, total, _ = _norm_forward(_rows(x), weight, None if residual is None else _rows(residual), float(eps), False, True)
    return q, x if total is None else total.view(x.shape)


# ---- 8-bit matrices ----------------------------------------------------------------------------------------------------------


class Fp8Matrix:
    """A matrix [rows, width] of float8_e4m3fn codes and their float8_e8m0fnu scales, one for each block of 128 columns and
    `rows_per_scale` (1 or 128) rows: scales [ceil(rows / rows_per_scale), ceil(width / 128)].  Rows of codes begin on 16 bytes and rows of
    scales on 4.  Nothing is copied."""
    __slots__ = ("codes", "scales", "rows_per_scale")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows_per_scale: int = 1):
        compiled = _compiled()
        if compiled:
            compiled.check_fp8_matrix(codes, scales, rows_per_scale)
            self.codes, self.scales, self.rows_per_scale = codes, scales, rows_per_scale
            return
        _check(codes, "codes", torch.float8_e4m3fn)
        _check(scales, "scales", torch.float8_e8m0fnu, codes.device)
        if rows_per_scale not in (1, _BLOCK):
            raise ValueError("rows_per_scale must be 1 or 128")
        if codes.dim() != 2 or scales.dim() != 2:
            raise ValueError("codes and scales must be matrices")
        rows, width = codes.shape
        if tuple(scales.shape) != (-(-rows // rows_per_scale), -(-width // _BLOCK)):
            raise ValueError(f"scales must have shape {(-(-rows // rows_per_scale), -(-width // _BLOCK))}, got {tuple(scales.shape)}")
        for t, name, unit in ((codes, "codes", 16), (scales, "scales", 4)):
            if t.numel() and (t.data_ptr() % unit or t.shape[1] > 1 and t.stride(1) != 1 or
                              t.shape[0] > 1 and (t.stride(0) % unit or t.stride(0) < t.shape[1])):
                raise ValueError(f"{name} must have dense rows that begin on multiples of {unit} bytes")
        self.codes, self.scales, self.rows_per_scale = codes, scales, rows_per_scale

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def _struct(self) -> HtgsFp8Matrix:
        codes, scales = self.codes, self.scales
        rows, width = codes.shape
        # the stride of a single row says nothing
        return HtgsFp8Matrix(codes.data_ptr(), scales.data_ptr(), rows, width, codes.stride(0) if rows > 1 else -(-width // 16) * 16,
                             scales.stride(0) if scales.shape[0] > 1 else -(-scales.shape[1] // 4) * 4, self.rows_per_scale)

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values that the codes stand for; bfloat16 and float32 hold all of them exactly, except that float32's and
        bfloat16's largest exponent bounds them."""
        compiled = _compiled()
        if compiled:
            return compiled.dequantize_fp8(self.codes, self.scales, self.rows_per_scale, dtype)
        if dtype not in _TYPES:
            raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        out = torch.empty(self.codes.shape, dtype=dtype, device=self.codes.device)
        _call(out.device, "htgs_dequantize_fp8", ctypes.byref(self._struct()), out.data_ptr(), out.shape[1], _TYPES[dtype])
        return out


def _fp8(codes: torch.Tensor, scales: torch.Tensor, rows_per_scale: int) -> Fp8Matrix:
    """An `Fp8Matrix` of tensors that need no check."""
    m = Fp8Matrix.__new__(Fp8Matrix)
    m.codes, m.scales, m.rows_per_scale = codes, scales, rows_per_scale
    return m


def _empty_fp8(rows: int, width: int, rows_per_scale: int, device) -> Fp8Matrix:
    blocks = -(-width // _BLOCK)
    return _fp8(torch.empty_strided((rows, width), (-(-width // 16) * 16, 1), dtype=torch.float8_e4m3fn, device=device),
                torch.empty_strided((-(-rows // rows_per_scale), blocks), (-(-blocks // 4) * 4, 1), dtype=torch.float8_e8m0fnu, device=device), rows_per_scale)


def _quantize(x: torch.Tensor, rows_per_scale: int, straight: bool, transposed: bool):
    rows, width = x.shape
    q = _empty_fp8(rows, width, rows_per_scale, x.device) if straight else None
    t = _empty_fp8(width, rows, rows_per_scale, x.device) if transposed else None
    if rows and width:
        where = [p for m in (q, t) for p in ((None, 0, None, 0) if m is None else (m.codes.data_ptr(), m.codes.stride(0), m.scales.data_ptr(), m.scales.stride(0)))]
        _call(x.device, "htgs_quantize_fp8", x.data_ptr(), x.stride(0), _TYPES[x.dtype], rows, width, rows_per_scale, *where)
    return q, t


def quantize_fp8(x: torch.Tensor, rows_per_scale: int = 1, transpose: bool = False) -> Fp8Matrix:
    """The last dimension's rows of x (or, with `transpose`, the columns of the matrix x) as 8-bit codes: each block of 128 columns and
    `rows_per_scale` rows (1: activations, 128: weights) gets the least power of two with which its largest finite value is at most 448, and values are
    rounded to nearest even.  Infinities and NaN become NaN.  No gradient flows through it."""
    compiled = _compiled()
    if compiled:
        return _fp8(*compiled.quantize_fp8(x, rows_per_scale, transpose), rows_per_scale)
    _check(x, "x")
    if rows_per_scale not in (1, _BLOCK):
        raise ValueError("rows_per_scale must be 1 or 128")
    if x.dim() < 1 or transpose and x.dim() != 2:
        raise ValueError("x must have a dimension to quantise along (and be a matrix to be transposed)")
    q, t = _quantize(_rows(x.detach()), rows_per_scale, not transpose, transpose)
    return t if transpose else q


def _few(x: torch.Tensor) -> bool:
    """Whether one kernel codes and multiplies the rows of x."""
    return 1 <= x.shape[0] <= 8 and x.shape[1] >= 1 and x.shape[0] * -(-x.shape[1] // _BLOCK) * _BLOCK <= 32768


def _matmul(a: Fp8Matrix, b: Fp8Matrix, dtype: torch.dtype) -> torch.Tensor:
    out = torch.empty((a.codes.shape[0], b.codes.shape[0]), dtype=dtype, device=a.codes.device)
    _call(out.device, "htgs_fp8_matmul", ctypes.byref(a._struct()), ctypes.byref(b._struct()), out.data_ptr(), out.shape[1], _TYPES[dtype])
    return out


def fp8_matmul(x, weight: Fp8Matrix, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x times the transpose of `weight` [out, width].  x is an `Fp8Matrix` [rows, width], or a tensor [..., width] that is quantised first, with a scale
    for each row and 128 columns.  Sums are 32-bit; the result has `dtype`, by default x's type, and bfloat16 for an `Fp8Matrix`.  For
    inference: it refuses an x that wants a gradient (`fp8_linear` has one)."""
    if not isinstance(weight, Fp8Matrix):
        raise TypeError("weight must be an Fp8Matrix")
    compiled = _compiled()
    if compiled:
        if isinstance(x, Fp8Matrix):
            return compiled.fp8_matmul(x.codes, x.scales, x.rows_per_scale, weight.codes, weight.scales, weight.rows_per_scale, dtype)
        return compiled.fp8_matmul(x, None, 1, weight.codes, weight.scales, weight.rows_per_scale, dtype)
    if dtype is not None and dtype not in _TYPES:
        raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    if isinstance(x, Fp8Matrix):
        if x.device != weight.device:
            raise ValueError(f"x is on {x.device}, expected {weight.device}")
        if x.shape[1] != weight.shape[1]:
            raise ValueError(f"x has width {x.shape[1]}, weight {weight.shape[1]}")
        return _matmul(x, weight, dtype or torch.bfloat16)
    _check(x, "x", None, weight.device)
    if x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x must have a last dimension of {weight.shape[1]} values")
    _no_tangent(x)
    if _wants_grad(x):
        raise RuntimeError("fp8_matmul has no gradient: use fp8_linear in training, or torch.no_grad()")
    xm, dtype = _rows(x), dtype or x.dtype
    if _few(xm):
        out = torch.empty((*x.shape[:-1], weight.shape[0]), dtype=dtype, device=x.device)
        _call(x.device, "htgs_fp8_matmul_values", xm.data_ptr(), xm.stride(0), _TYPES[x.dtype], xm.shape[0], ctypes.byref(weight._struct()), out.data_ptr(),
              weight.shape[0], _TYPES[dtype])
        return out
    q, _ = _quantize(xm, 1, True, False)
    return _matmul(q, weight, dtype).view(*x.shape[:-1], weight.shape[0])


def check_products(device: Optional[torch.device] = None) -> None:
    """Raises if a product on `device` (default: the current one) gave up on a wait of its kernel, so that its result is not complete: NaN where something is missing.  The next product there
    raises by itself; this is for what no product follows: after a synchronisation, at the end of a training step or behind a graph's replay.  Waits for nothing."""
    index = None if device is None else torch.device(device).index
    _native.check(_native.lib().htgs_fp8_matmul_status(torch.cuda.current_device() if index is None else index))


class _Fp8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight):
        need_x, need_weight = ctx.needs_input_grad
        xm, wm = _rows(x), _rows(weight)
        xq, xt = _quantize(xm, 1, True, need_weight)          # the gradients sum over other axes, so their blocks run along those
        wq, wt = _quantize(wm, _BLOCK, True, need_x)
        ctx.save_for_backward(*(t for m in (xt, wt) for t in ((None, None) if m is None else (m.codes, m.scales))))
        ctx.types = (x.dtype, weight.dtype)
        return _matmul(xq, wq, x.dtype).view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @_first_derivative
    def backward(ctx, grad_y):
        x_codes, x_scales, w_codes, w_scales = ctx.saved_tensors
        need_x, need_weight = ctx.needs_input_grad
        xt, wt = _fp8(x_codes, x_scales, 1), _fp8(w_codes, w_scales, _BLOCK)
        gq, gt = _quantize(_rows(grad_y), 1, need_x, need_weight)
        grad_x = _matmul(gq, wt, ctx.types[0]).view(*grad_y.shape[:-1], wt.shape[0]) if need_x else None
        return grad_x, _matmul(gt, xt, ctx.types[1]) if need_weight else None


def fp8_linear(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """x [..., width] times the transpose of weight [out, width], with 8-bit operands: x quantised per row and 128 columns, weight per block of
    128 x 128.  Differentiable: grad_y is quantised along `out` for the gradient of x, and grad_y and x along the rows for the gradient of
    weight; quantisation itself counts as the identity."""
    compiled = _compiled()
    if compiled:
        return compiled.fp8_linear(x, weight)
    _check(x, "x")
    _check(weight, "weight", x.dtype, x.device)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError("weight must have shape (out, width), and x a last dimension of width values")
    _no_tangent(x, weight)
    if _wants_grad(x, weight):
        return _Fp8Linear.apply(x, weight)
    return fp8_matmul(x, quantize_fp8(weight, _BLOCK))


# ---- recurrence ----------------------------------------------------------------------------------------------------------------


_MOST_STRIDE = 1 << 22      # of a recurrence's rows, in elements


def _scan_rows(t: torch.Tensor) -> torch.Tensor:
    m = _rows(t)
    return m.clone(memory_format=torch.contiguous_format) if m.stride(0) > _MOST_STRIDE else m


def _scan_struct(x, gate, initial, offsets, sequences, reverse) -> HtgsScan:
    return HtgsScan(x.data_ptr(), gate.data_ptr(), None if initial is None else initial.data_ptr(), None if offsets is None else offsets.data_ptr(),
                    x.stride(0), gate.stride(0), x.shape[0], x.shape[1], sequences, _TYPES[x.dtype], int(reverse))


def _scan_forward(x, gate, initial, offsets, sequences, reverse, keep):
    rows, width = x.shape
    lib = _native.lib()
    h = torch.empty((rows, width), dtype=x.dtype, device=x.device)
    last = torch.empty((sequences, width), dtype=torch.float32, device=x.device)
    states = torch.empty(lib.htgs_gated_scan_state_bytes(rows, width), dtype=torch.uint8, device=x.device) if keep else None
    size = lib.htgs_gated_scan_workspace_bytes(rows, width)
    workspace = torch.empty(size, dtype=torch.uint8, device=x.device)
    _call(x.device, "htgs_gated_scan", ctypes.byref(_scan_struct(x, gate, initial, offsets, sequences, reverse)), h.data_ptr(), width, last.data_ptr(),
          None if states is None else states.data_ptr(), workspace.data_ptr(), size)
    return h, last, states


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, initial, offsets, sequences, reverse):
        ctx.set_materialize_grads(False)
        h, last, states = _scan_forward(x, gate, initial, offsets, sequences, reverse, True)
        ctx.save_for_backward(x, gate, initial, offsets, states)
        ctx.rest = (sequences, reverse)
        return h, last

    @staticmethod
    @_first_derivative
    def backward(ctx, grad_h, grad_last):
        x, gate, initial, offsets, states = ctx.saved_tensors
        sequences, reverse = ctx.rest
        rows, width = x.shape
        if grad_h is None:
            grad_h = torch.zeros((rows, width), dtype=x.dtype, device=x.device)
        grad_h = _scan_rows(grad_h)
        grad_last = None if grad_last is None else grad_last.contiguous()
        grad_x, grad_gate = (torch.empty((rows, width), dtype=x.dtype, device=x.device) for _ in range(2))
        grad_initial = torch.empty_like(initial) if initial is not None and ctx.needs_input_grad[2] else None
        size = _native.lib().htgs_gated_scan_workspace_bytes(rows, width)
        workspace = torch.empty(size, dtype=torch.uint8, device=x.device)
        _call(x.device, "htgs_gated_scan_backward", ctypes.byref(_scan_struct(x, gate, initial, offsets, sequences, reverse)), states.data_ptr(),
              grad_h.data_ptr(), grad_h.stride(0), None if grad_last is None else grad_last.data_ptr(), grad_x.data_ptr(), width, grad_gate.data_ptr(), width,
              None if grad_initial is None else grad_initial.data_ptr(), workspace.data_ptr(), size)
        return grad_x, grad_gate, grad_initial, None, None, None


def gated_scan(x: torch.Tensor, gate: torch.Tensor, initial: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None,
               reverse: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """(h, last) of the recurrence h_t = a_t h_{t-1} + (1 - a_t) x_t with a = sigmoid(gate), channel by channel.

    x and gate are [rows, width] (one sequence, or with `offsets` several behind one another) or [batch, rows, width]; views with evenly spaced rows, such as
    the halves of one projection, are read in place.  `offsets` is an int32 tensor of ascending row numbers, from 0 to rows, that
    begin the sequences (sequences may be empty).  `initial` [sequences, width] float32 is the state in front of each sequence (default zeros), `last` the float32
    state behind it.  With `reverse` each sequence is gone through from its last row to its first.  States are 32-bit; h has x's
    type.  Differentiable in x, gate and initial."""
    compiled = _compiled()
    if compiled:
        return compiled.gated_scan(x, gate, initial, offsets, reverse)
    _check(x, "x")
    _check(gate, "gate", x.dtype, x.device)
    if gate.shape != x.shape or x.dim() not in (2, 3):
        raise ValueError("x and gate must have one shape, [rows, width] or [batch, rows, width]")
    if not 1 <= x.shape[-1] <= 65536:
        raise ValueError("x must have 1 to 65536 channels")
    if offsets is not None:
        _check(offsets, "offsets", torch.int32, x.device)
        if x.dim() != 2 or offsets.dim() != 1 or offsets.numel() < 2:
            raise ValueError("offsets must hold sequences + 1 row numbers, for x of shape [rows, width]")
        offsets = offsets.contiguous()
    sequences = x.shape[0] if x.dim() == 3 else 1 if offsets is None else offsets.numel() - 1
    if initial is not None:
        _check(initial, "initial", torch.float32, x.device)
        if tuple(initial.shape) != (sequences, x.shape[-1]):
            raise ValueError(f"initial must have shape {(sequences, x.shape[-1])}, got {tuple(initial.shape)}")
    _no_tangent(x, gate, initial)
    shape = x.shape
    if sequences == 0:
        return torch.empty_like(x), torch.empty((0, shape[-1]), dtype=torch.float32, device=x.device)
    if _wants_grad(x, gate, initial):
        initial = None if initial is None else initial.contiguous()
        h, last = _GatedScan.apply(_scan_rows(x), _scan_rows(gate), initial, offsets, sequences, bool(reverse))
    else:
        h, last, _ = _scan_forward(_scan_rows(x), _scan_rows(gate), None if initial is None else initial.contiguous(), offsets, sequences, bool(reverse), False)
    return h.view(shape), last


def gated_scan_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
    """One step of `gated_scan` for each row: `state` [rows, width] float32 becomes a * state + (1 - a) * x, in place, and is returned in x's type.  For
    inference: it refuses inputs that want a gradient."""
    compiled = _compiled()
    if compiled:
        return compiled.gated_scan_step(x, gate, state)
    _check(x, "x")
    _check(gate, "gate", x.dtype, x.device)
    _check(state, "state", torch.float32, x.device)
    if x.dim() != 2 or gate.shape != x.shape or state.shape != x.shape or x.shape[1] < 1:
        raise ValueError("x, gate and state must have one shape, [rows, width]")
    if state.stride(1) != 1 and state.shape[1] != 1 or state.shape[0] > 1 and state.stride(0) < state.shape[1]:
        raise ValueError("state must have dense rows: it is updated in place")
    _no_tangent(x, gate, state)
    if _wants_grad(x, gate, state):
        raise RuntimeError("gated_scan_step has no gradient: use gated_scan in training, or torch.no_grad()")
    xm, gm = _rows(x), _rows(gate)
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _call(x.device, "htgs_gated_scan_step", xm.data_ptr(), xm.stride(0), gm.data_ptr(), gm.stride(0), state.data_ptr(), state.stride(0), h.data_ptr(),
          x.shape[1], _TYPES[x.dtype], x.shape[0], x.shape[1])
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)        # autograd learns of it; what inference mode made is kept by no gradient
    return h
