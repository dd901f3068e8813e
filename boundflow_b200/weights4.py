"""Linear layers whose weights are held in 4 bits with a scale for each group of columns.

`Weight4` stands where a Linear layer's weight does: in the `params` of a module that `CudaTaskExecutor.run_ibp`, `forward_ibp_trace_mlp`, `run_crown_ibp_mlp`
(`_from_forward_trace` and with ReLU influence too), `run_alpha_crown_mlp`, `run_alpha_beta_crown_mlp`, `first_layer_certificate` and `CudaQueryRuntime` bound (such modules
take the graph path of `dag.py`; L1 and L2 balls and the certificate make a dense copy of the first layer in every call), as the weight of
`CudaIntervalDomain.affine_transformer`, and in the products below.  `ibp_trace`, `bound_split_domains`, `run_crown_intermediate_mlp` and fused regions read dense
weights and refuse it; `dense()` makes one.

    linear4(x, weight, bias)                   x W^T + b, with gradients for x and bias (the weight is frozen)
    interval_linear4(lower, upper, weight, b)  bounds of it over boxes, with gradients for lower, upper and bias
    rows_times_weight4(A, weight)              A W: coefficient rows pushed back through the layer
    quantise_weight4(W, group)                 codes and scales of a given weight

The reference holds all weights in 32 bits; the bounds are those of the network whose weights the codes and scales stand for, computed as
`bf_ibp_linear` and `bf_crown_relu_linear_bwd` compute them for dense weights.  Like the rest of the package the functions queue their work on the current
stream of the tensors' device; tensors on the CPU are copied to the current CUDA device and results returned on the device the inputs came from.

Forward, a sum over at most 128 columns of one group is scaled when it is complete, so inputs of 1e35 and more may overflow it whatever the scale.  Infinity times a zero weight is
NaN, as are infinities of both signs in one sum.  Waits on the device are bounded: where one runs out, the results concerned are NaN, and so are all bounds that follow from them.
"""
from __future__ import annotations

from typing import Any, Optional, Tuple

import torch
from torch.autograd import forward_ad as _forward

from . import _lib
from .network import _cuda_device

_MOST_ROWS, _MOST_SIDE = 2 ** 31 - 1, 2 ** 30  # of a call, of a weight: the library counts them in 32 bits
_TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_F16}


class Weight4:
    """W [n_out, n_in] = scales[k // group, n] * (code[n, k] - 8).

    codes: uint8 [n_out, padded / 2], two codes in a byte (low nibble = even column), padded = n_in rounded up to a whole group;
    scales: fp32 [padded / group, n_out], finite.  Both contiguous, on one device, codes on a 16-byte boundary.  They are read where they are: a change
    in place is a change of the weight."""

    __slots__ = ("codes", "scales", "n_out", "n_in", "group")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, n_in: int):
        n_in = int(n_in)
        if not (torch.is_tensor(codes) and torch.is_tensor(scales)) or codes.dtype != torch.uint8 or scales.dtype != torch.float32:
            raise TypeError("Weight4 takes codes as uint8 and scales as float32 tensors")
        if codes.dim() != 2 or scales.dim() != 2 or n_in < 1 or codes.shape[0] < 1:
            raise ValueError(f"Weight4: codes {tuple(codes.shape)}, scales {tuple(scales.shape)}, n_in {n_in}")
        n_out, padded, groups = int(codes.shape[0]), 2 * int(codes.shape[1]), int(scales.shape[0])
        group = padded // groups if groups else 0
        if int(scales.shape[1]) != n_out or groups == 0 or group * groups != padded or not padded - group < n_in <= padded:
            raise ValueError(f"Weight4: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not hold rows of {n_in} weights")
        if n_out > _MOST_SIDE or n_in > _MOST_SIDE:
            raise ValueError(f"Weight4: {n_out} x {n_in} weights (at most 2^30 a side)")
        if group < 32 or group > 1 << 20 or group & (group - 1):
            raise ValueError(f"Weight4: groups of {group} weights (a power of two from 32 to 2^20 is wanted)")
        if codes.device != scales.device:
            raise ValueError("Weight4: codes and scales are on different devices")
        if not codes.is_contiguous() or not scales.is_contiguous() or codes.data_ptr() % 16:
            raise ValueError("Weight4: codes and scales must be contiguous, codes on a 16-byte boundary")
        self.codes, self.scales, self.n_out, self.n_in, self.group = codes, scales, n_out, n_in, group

    @classmethod
    def _of(cls, codes: torch.Tensor, scales: torch.Tensor, n_out: int, n_in: int, group: int) -> "Weight4":
        """Without the checks, for tensors made to measure."""
        w = cls.__new__(cls)
        w.codes, w.scales, w.n_out, w.n_in, w.group = codes, scales, n_out, n_in, group
        return w

    @property
    def shape(self) -> Tuple[int, int]:
        return (self.n_out, self.n_in)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dim(self) -> int:
        return 2

    def to(self, device: Any) -> "Weight4":
        return self if self.codes.device == (device if isinstance(device, torch.device) else torch.device(device)) else Weight4(self.codes.to(device), self.scales.to(device), self.n_in)

    def integers(self) -> torch.Tensor:
        """code - 8 as int8 [n_out, n_in]."""
        codes = self.codes if self.codes.is_cuda else self.codes.to(_cuda_device(self.codes))
        out = torch.empty((self.n_out, self.n_in), dtype=torch.int8, device=codes.device)
        _W4_INTEGERS(codes.device, codes.data_ptr(), out.data_ptr(), self.n_out, self.n_in, self.group)
        return out if self.codes.is_cuda else out.to(self.codes.device)

    def dense(self) -> torch.Tensor:
        """The weight in fp32."""
        device = _device_of(self.codes)
        w = self.to(device)
        out = torch.empty(w.shape, dtype=torch.float32, device=device)
        _W4_DENSE(device, w.codes.data_ptr(), w.scales.data_ptr(), out.data_ptr(), w.n_out, w.n_in, w.group)
        return out.to(self.device)

    def __repr__(self) -> str:
        return f"Weight4({self.n_out} x {self.n_in}, groups of {self.group}, {self.device})"


def _device_of(t: torch.Tensor) -> torch.device:
    return t.device if t.is_cuda else _cuda_device(t)


def quantise_weight4(W: torch.Tensor, group: int = 128) -> Weight4:
    """Codes and scales of W (fp32, bf16 or fp16, [n_out, n_in]): the scale of a group is its largest magnitude times 1/7, a code the nearest of -7..7
    (ties to even).  A group of zeros has scale 0; one that holds an infinity or a NaN is NaN throughout."""
    if not torch.is_tensor(W) or W.dtype not in _TYPES:
        raise TypeError("quantise_weight4 takes an fp32, bf16 or fp16 tensor")
    group = int(group)
    if W.dim() != 2 or W.shape[0] < 1 or W.shape[1] < 1:
        raise ValueError(f"quantise_weight4: a weight [n_out, n_in] is wanted, got {tuple(W.shape)}")
    if max(W.shape) > _MOST_SIDE:
        raise ValueError(f"quantise_weight4: {tuple(W.shape)} weights (at most 2^30 a side)")
    if group < 32 or group > 1 << 20 or group & (group - 1):
        raise ValueError(f"quantise_weight4: groups of {group} weights (a power of two from 32 to 2^20 is wanted)")
    device = _device_of(W)
    w = _placed(W.detach() if W.requires_grad else W, device)
    n_out, n_in = w.shape
    groups = -(-n_in // group)
    codes = torch.empty(n_out, groups * group // 2, dtype=torch.uint8, device=device)
    scales = torch.empty(groups, n_out, dtype=torch.float32, device=device)
    _W4_QUANTISE(device, w.data_ptr(), _TYPES[w.dtype], codes.data_ptr(), scales.data_ptr(), n_out, n_in, group)
    made = Weight4._of(codes, scales, n_out, n_in, group)
    return made if W.is_cuda else made.to(W.device)


# ---- launches: contiguous CUDA tensors of one device, rows [M, n] -----------------------
class _Entry:
    """An entry point of the library, called with the tensors' device current.  (torch.cuda.device and the arity check cost a call of few microseconds more than its
    kernel takes; the argument lists below are fixed.)"""

    def __init__(self, name: str):
        self.name, self.fn = name, None

    def __call__(self, device: torch.device, *args) -> None:
        fn = self.fn
        if fn is None:
            fn = self.fn = getattr(_lib.load(), self.name).unchecked
        index = device.index
        before = torch._C._cuda_getDevice()
        if before == index:
            code = fn(*args, torch._C._cuda_getCurrentRawStream(index))
        else:
            with torch.cuda.device(device):
                code = fn(*args, torch._C._cuda_getCurrentRawStream(index))
        if code:
            _lib.check(code)


_W4_LINEAR, _W4_INTERVAL, _W4_ROWS, _W4_INTERVAL_GRAD = (_Entry(n) for n in ("bf_w4_linear", "bf_w4_interval", "bf_w4_rows", "bf_w4_interval_grad"))
_W4_LINEAR_GRAD = _Entry("bf_w4_linear_grad")
_W4_LINEAR_MANY, _W4_INTERVAL_MANY, _W4_ROWS_MANY, _W4_INTERVAL_GRAD_MANY = (_Entry(f"bf_w4_{n}_many") for n in ("linear", "interval", "rows", "interval_grad"))
_W4_QUANTISE, _W4_INTEGERS, _W4_DENSE, _COLUMN_SUMS = (_Entry(n) for n in ("bf_w4_quantise", "bf_w4_integers", "bf_w4_dense", "bf_column_sums"))


_LEAST_MANY = 32  # rows from which the kernels for many are asked about


def _many_pays(M: int, w: Weight4, dtype: torch.dtype, backward: bool, pair: bool) -> bool:
    return bool(_lib.load().bf_w4_many_pays(M, w.n_in, w.n_out, w.group, _TYPES[dtype], backward, pair))


def _workspace(rows: torch.Tensor, w: Weight4, backward: bool, pair: bool = False) -> Optional[torch.Tensor]:
    """Workspace of the kernels for many rows, or None where those for few are taken."""
    M = rows.shape[0]
    if M < _LEAST_MANY or not _many_pays(M, w, rows.dtype, backward, pair):
        return None
    return torch.empty(_lib.load().bf_w4_workspace_bytes(M, rows.shape[1], _TYPES[rows.dtype]), dtype=torch.uint8, device=rows.device)


def _linear(x: torch.Tensor, w: Weight4, bias: Optional[torch.Tensor]) -> torch.Tensor:
    M = x.shape[0]
    y = x.new_empty((M, w.n_out))
    if M:
        work = _workspace(x, w, False)
        args = (x.data_ptr(), _TYPES[x.dtype], w.codes.data_ptr(), w.scales.data_ptr(), None if bias is None else bias.data_ptr(),
                0 if bias is None else _TYPES[bias.dtype], y.data_ptr(), M, w.n_in, w.n_out, w.group)
        if work is None:
            _W4_LINEAR(x.device, *args)
        else:
            _W4_LINEAR_MANY(x.device, *args, work.data_ptr())
    return y


def _interval(a: torch.Tensor, b: torch.Tensor, mode: int, relu_in: int, w: Weight4, bias: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    M = a.shape[0]
    lower, upper = a.new_empty((M, w.n_out)), a.new_empty((M, w.n_out))
    if M:
        work = _workspace(a, w, False, True)
        args = (a.data_ptr(), b.data_ptr(), mode, relu_in, w.codes.data_ptr(), w.scales.data_ptr(), None if bias is None else bias.data_ptr(),
                lower.data_ptr(), upper.data_ptr(), M, w.n_in, w.n_out, w.group)
        if work is None:
            _W4_INTERVAL(a.device, *args)
        else:
            _W4_INTERVAL_MANY(a.device, *args, work.data_ptr())
    return lower, upper


def _rows(a: torch.Tensor, w: Weight4) -> torch.Tensor:
    M = a.shape[0]
    z = a.new_empty((M, w.n_in))
    if M:
        work = _workspace(a, w, True)
        args = (a.data_ptr(), _TYPES[a.dtype], w.codes.data_ptr(), w.scales.data_ptr(), z.data_ptr(), M, w.n_in, w.n_out, w.group)
        if work is None:
            _W4_ROWS(a.device, *args)
        else:
            _W4_ROWS_MANY(a.device, *args, work.data_ptr())
    return z


def _column_sums(a: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    M, n = a.shape
    if M == 0:
        return a.new_zeros(n, dtype=dtype)
    out = a.new_empty(n, dtype=dtype)
    _COLUMN_SUMS(a.device, a.data_ptr(), _TYPES[a.dtype], out.data_ptr(), _TYPES[dtype], M, n)
    return out


class _Linear4(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bias, weight):
        ctx.weight, ctx.bias_type = weight, None if bias is None else bias.dtype
        return _linear(x, weight, bias)

    @staticmethod
    def backward(ctx, dy):
        need, w, M = ctx.needs_input_grad, ctx.weight, dy.shape[0]
        again = dy.requires_grad and torch.is_grad_enabled()  # a gradient of this gradient is asked for
        dy = dy.contiguous()
        if again:
            return _Rows4.apply(dy, w) if need[0] else None, dy.float().sum(0).to(ctx.bias_type) if need[1] else None, None
        if M == 0 or M >= _LEAST_MANY:
            return _rows(dy, w) if need[0] else None, _column_sums(dy, ctx.bias_type) if need[1] else None, None
        dx = dy.new_empty((M, w.n_in)) if need[0] else None
        db = dy.new_empty(w.n_out, dtype=ctx.bias_type) if need[1] else None
        _W4_LINEAR_GRAD(dy.device, dy.data_ptr(), _TYPES[dy.dtype], w.codes.data_ptr(), w.scales.data_ptr(), None if dx is None else dx.data_ptr(),
                        None if db is None else db.data_ptr(), 0 if db is None else _TYPES[ctx.bias_type], M, w.n_in, w.n_out, w.group)
        return dx, db, None


class _Rows4(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, weight):
        ctx.weight = weight
        return _rows(a, weight)

    @staticmethod
    def backward(ctx, dz):
        again = dz.requires_grad and torch.is_grad_enabled()
        dz = dz.contiguous()
        return (_Linear4.apply(dz, None, ctx.weight) if again else _linear(dz, ctx.weight, None)), None


class _Interval4(torch.autograd.Function):
    @staticmethod
    def forward(ctx, lower, upper, bias, weight):
        ctx.weight = weight
        return _interval(lower, upper, _lib.IN_LOWER_UPPER, 0, weight, bias)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dl, du):
        w = ctx.weight
        dl, du = dl.contiguous(), du.contiguous()
        M = dl.shape[0]
        gl = gu = db = None
        if ctx.needs_input_grad[0] or ctx.needs_input_grad[1]:
            gl, gu = dl.new_empty((M, w.n_in)), dl.new_empty((M, w.n_in))
            if M:
                work = _workspace(dl, w, True, True)
                args = (dl.data_ptr(), du.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), gl.data_ptr(), gu.data_ptr(), M, w.n_in, w.n_out, w.group)
                if work is None:
                    _W4_INTERVAL_GRAD(dl.device, *args)
                else:
                    _W4_INTERVAL_GRAD_MANY(dl.device, *args, work.data_ptr())
        if ctx.needs_input_grad[2]:
            db = _column_sums(dl, torch.float32) + _column_sums(du, torch.float32)
        return gl, gu, db, None


def _check_rows(name: str, x: Any, weight: Any, width: str) -> None:
    if not isinstance(weight, Weight4):
        raise TypeError(f"{name}: the weight is a Weight4 (quantise_weight4 makes one), got {type(weight)}")
    if not torch.is_tensor(x) or x.dtype not in _TYPES:
        raise TypeError(f"{name} takes fp32, bf16 or fp16 tensors")
    if x.dim() < 1 or x.shape[-1] != getattr(weight, width):
        raise ValueError(f"{name}: rows of {int(x.shape[-1]) if x.dim() else 0} do not match {weight!r}")
    if x.numel() > _MOST_ROWS * x.shape[-1]:
        raise ValueError(f"{name}: {x.numel() // x.shape[-1]} rows (at most 2^31 - 1 in a call)")


def _refuse_tangents(name: str, *tensors: Any) -> None:
    """A tensor that carries a forward-mode tangent asks for no gradient: without this the launch would drop it."""
    if _forward._current_level >= 0 and any(torch.is_tensor(t) and t.is_floating_point() and _forward.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative")


def _check_bias(name: str, bias: Any, weight: Weight4) -> None:
    if bias is not None and (not torch.is_tensor(bias) or bias.dtype not in _TYPES):
        raise TypeError(f"{name} takes an fp32, bf16 or fp16 bias")
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != weight.n_out):
        raise ValueError(f"{name}: bias {tuple(bias.shape)} does not match {weight!r}")


def _ready(x: Any, weight: Any, width: int, bias: Any) -> bool:
    """Whether a call can go straight to its launch: rows [M, width] and bias as the kernels read them, on the weight's device, and no gradient asked for.
    (All else takes the checks and copies below; microseconds that a small layer's kernel does not take.)"""
    return (x.is_cuda and x.dim() == 2 and x.shape[1] == width and x.shape[0] <= _MOST_ROWS and x.dtype in _TYPES and x.is_contiguous() and x.get_device() == weight.codes.get_device()
            and not (x.requires_grad and torch.is_grad_enabled())
            and (bias is None or (torch.is_tensor(bias) and bias.is_cuda and bias.dim() == 1 and bias.shape[0] == weight.n_out and bias.dtype in _TYPES and bias.is_contiguous()
                                  and bias.get_device() == x.get_device() and not (bias.requires_grad and torch.is_grad_enabled()))))


def _placed(t: torch.Tensor, device: torch.device) -> torch.Tensor:
    """`t` on `device`, contiguous: itself where it is so already."""
    return t if t.is_cuda and t.device == device and t.is_contiguous() else t.to(device).contiguous()


def linear4(x: torch.Tensor, weight: Weight4, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x W^T + bias for x [..., n_in] in fp32, bf16 or fp16 (sums in fp32, rounded once to x's type).  Differentiable in x and bias; beside 16-bit rows each
    product of the gradient of x is held to 2^-17 (`rows_times_weight4`)."""
    _refuse_tangents("linear4", x, bias)
    if type(weight) is Weight4 and torch.is_tensor(x) and _ready(x, weight, weight.n_in, bias):
        return _linear(x, weight, bias)
    _check_rows("linear4", x, weight, "n_in")
    _check_bias("linear4", bias, weight)
    device = _device_of(x)
    w, b = weight.to(device), bias if bias is None else _placed(bias, device)
    flat = x.dim() == 2
    rows = _placed(x if flat else x.reshape(-1, weight.n_in), device)
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        y = _Linear4.apply(rows, b, w)
    else:
        y = _linear(rows, w, b)
    if not flat:
        y = y.reshape(x.shape[:-1] + (weight.n_out,))
    return y if x.is_cuda else y.to(x.device)


def interval_linear4(lower: torch.Tensor, upper: torch.Tensor, weight: Weight4, bias: Optional[torch.Tensor] = None, *,
                     relu_in: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Bounds of x W^T + bias for lower <= x <= upper (fp32 [..., n_in]); `relu_in` clamps the input at zero first.  Differentiable once, for lower, upper
    and bias (without relu_in)."""
    _refuse_tangents("interval_linear4", lower, upper, bias)
    if (type(weight) is Weight4 and torch.is_tensor(lower) and torch.is_tensor(upper) and lower.dtype == upper.dtype == torch.float32 and lower.shape == upper.shape
            and _ready(lower, weight, weight.n_in, bias) and _ready(upper, weight, weight.n_in, None) and (bias is None or bias.dtype == torch.float32)):
        return _interval(lower, upper, _lib.IN_LOWER_UPPER, 1 if relu_in else 0, weight, bias)
    _check_rows("interval_linear4", lower, weight, "n_in")
    _check_rows("interval_linear4", upper, weight, "n_in")
    _check_bias("interval_linear4", bias, weight)
    if lower.shape != upper.shape or lower.device != upper.device:
        raise ValueError(f"interval_linear4: lower {tuple(lower.shape)} and upper {tuple(upper.shape)} differ in shape or device")
    if lower.dtype != torch.float32 or upper.dtype != torch.float32 or (bias is not None and bias.dtype != torch.float32):
        raise TypeError("interval_linear4 takes fp32: bounds rounded to 16 bits would not hold")
    device = _device_of(lower)
    w, b = weight.to(device), bias if bias is None else _placed(bias, device)
    flat = lower.dim() == 2
    lo, up = (_placed(t if flat else t.reshape(-1, weight.n_in), device) for t in (lower, upper))
    if torch.is_grad_enabled() and (lower.requires_grad or upper.requires_grad or (bias is not None and bias.requires_grad)):
        if relu_in:
            raise NotImplementedError("interval_linear4 has no gradient with relu_in; clamp the bounds before the call")
        yl, yu = _Interval4.apply(lo, up, b, w)
    else:
        yl, yu = _interval(lo, up, _lib.IN_LOWER_UPPER, 1 if relu_in else 0, w, b)
    if not flat:
        shape = lower.shape[:-1] + (weight.n_out,)
        yl, yu = yl.reshape(shape), yu.reshape(shape)
    return (yl, yu) if lower.is_cuda else (yl.to(lower.device), yu.to(lower.device))


def rows_times_weight4(A: torch.Tensor, weight: Weight4) -> torch.Tensor:
    """A W for coefficient rows A [..., n_out] in fp32, bf16 or fp16 (sums in fp32, rounded once; beside 16-bit rows each product is held to 2^-17): the
    gradient of `linear4`.  Differentiable in A."""
    _refuse_tangents("rows_times_weight4", A)
    if type(weight) is Weight4 and torch.is_tensor(A) and _ready(A, weight, weight.n_out, None):
        return _rows(A, weight)
    _check_rows("rows_times_weight4", A, weight, "n_out")
    device = _device_of(A)
    flat = A.dim() == 2
    rows, w = _placed(A if flat else A.reshape(-1, weight.n_out), device), weight.to(device)
    z = _Rows4.apply(rows, w) if A.requires_grad and torch.is_grad_enabled() else _rows(rows, w)
    if not flat:
        z = z.reshape(A.shape[:-1] + (weight.n_in,))
    return z if A.is_cuda else z.to(A.device)
