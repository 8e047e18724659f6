"""Microscaled 4-bit floating point: quantisation and product.

The SC engine's products run as e2m1 multiply-adds with unit scales; this
module offers the same tensor-core operands with real block scales, i.e. the
deterministic 4-bit linear that an SC linear is compared with.

* ``mx_quantize(x, fmt)`` -> ``MXTensor``: e2m1 codes with one scale per block
  of the last dimension.  ``"mxfp4"``: blocks of 32, power-of-two scales
  ``2^(floor(log2 max|x|) - 2)``.  ``"nvfp4"``: blocks of 16, e4m3 scales
  ``max|x| * fl32(1/6)`` under a power-of-two tensor scale ``2^scale_exp``.
  Codes are rounded to nearest even and saturate at 6.  A block with a NaN or
  an infinity stands for NaNs.
* ``MXTensor.dequantize()``: the values that the codes stand for.
* ``mx_matmul(a, b)``: ``a @ b^T`` (+ bias) with fp32 sums; ``a`` may be a
  plain tensor, which is quantised to ``b``'s format on the way in.
* ``MXLinear``: an ``nn.Linear`` with its weight in 4 bits.

Inference only: there is no gradient, and an input that asks for one is
refused.  There is no CPU path: CPU tensors raise.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Union

import torch
import torch.nn as nn

from . import _lib
from ._call import call, dtype_code, has_tangent

__all__ = ["MXTensor", "mx_quantize", "mx_matmul", "MXLinear", "tensor_scale_exp"]


def _check_fmt(fmt: str) -> str:
    if fmt not in _lib.MX_FORMAT:
        raise ValueError(f"unknown 4-bit format {fmt!r} (one of {sorted(_lib.MX_FORMAT)})")
    return fmt


def _check_exp(scale_exp: int) -> int:
    exp = int(scale_exp)
    if not -1024 <= exp <= 1024:  # (the engine has the formats' own limits)
        raise ValueError(f"scale_exp {scale_exp} is out of range")
    return exp


def _no_grad_wanted(name: str, *tensors) -> None:
    wanted = has_tangent(tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            wanted = wanted or (t is not None and t.requires_grad)
    if wanted:
        raise RuntimeError(f"{name} has no gradient; call it under torch.no_grad() or on "
                           "detached inputs")


def _sizes(rows: int, K: int, fmt: str):
    """Bytes of codes and of scales (``scmp_mx_data_size``, ``scmp_mx_scale_size``)."""
    kp = (K + 31) // 32 * 32
    groups = -(-kp // (4 * _lib.MX_BLOCK[fmt]))
    return rows * kp // 2, (rows + 127) // 128 * groups * 512


def _check_bytes(data: torch.Tensor, scales: torch.Tensor, sizes) -> None:
    if (data.dtype == scales.dtype == torch.uint8 and (data.numel(), scales.numel()) == sizes
            and data.is_contiguous() and scales.is_contiguous()):
        return
    for t, size, what in ((data, sizes[0], "data"), (scales, sizes[1], "scales")):
        if t.dtype != torch.uint8 or not t.is_contiguous() or t.numel() != size:
            raise ValueError(f"{what} must be {size} contiguous bytes, got {t.numel()} of {t.dtype}"
                             f" with strides {t.stride()}")


class MXTensor:
    """A quantised tensor ``[..., K]``: codes and block scales on the GPU.

    ``data`` and ``scales`` (uint8) have the layout of ``scmp_mx_quantize``
    (rows are the leading dimensions flattened); ``dtype`` is the type of the
    tensor it was made from, which products of it come out in by default."""

    __slots__ = ("shape", "rows", "fmt", "scale_exp", "dtype", "_data", "_scales", "_buf",
                 "data_ptr", "scales_ptr", "index")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, shape: Sequence[int], fmt: str,
                 scale_exp: int = 0, dtype: torch.dtype = torch.float32):
        shape = torch.Size(shape)
        if not shape or shape[-1] < 1 or min(shape) < 0:
            raise ValueError("an MXTensor has a last dimension of at least 1 and none below 0, got "
                             f"{tuple(shape)}")
        _check_bytes(data, scales, _sizes(math.prod(shape[:-1]), shape[-1], _check_fmt(fmt)))
        if data.device != scales.device:
            raise ValueError(f"data on {data.device}, scales on {scales.device}")
        if data.data_ptr() % 16 or scales.data_ptr() % 16:
            raise ValueError("data and scales must be 16-byte aligned")
        self._set(data, scales, None, data.data_ptr(), scales.data_ptr(), data.get_device(), shape,
                  fmt, _check_exp(scale_exp), dtype)

    def _set(self, data, scales, buf, data_ptr, scales_ptr, index, shape, fmt, scale_exp, dtype):
        self._data, self._scales, self._buf = data, scales, buf
        self.data_ptr, self.scales_ptr, self.index = data_ptr, scales_ptr, index
        self.shape, self.fmt, self.scale_exp, self.dtype = shape, fmt, scale_exp, dtype
        self.rows = math.prod(shape[:-1])
        return self

    @property
    def data(self) -> torch.Tensor:
        if self._data is None:
            self._data = self._buf[:_sizes(self.rows, self.shape[-1], self.fmt)[0]]
        return self._data

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            at = self.scales_ptr - self.data_ptr
            self._scales = self._buf[at:at + _sizes(self.rows, self.shape[-1], self.fmt)[1]]
        return self._scales

    @property
    def device(self) -> torch.device:
        return (self._data if self._buf is None else self._buf).device

    @property
    def is_cuda(self) -> bool:
        return self.index >= 0

    def dim(self) -> int:
        return len(self.shape)

    def __reduce__(self):
        # copies and loaded tensors are other memory: no address is carried over
        return MXTensor, (self.data, self.scales, tuple(self.shape), self.fmt, self.scale_exp,
                          self.dtype)

    def reshape(self, *shape) -> "MXTensor":
        """The same codes under other leading dimensions; the last one stays."""
        shape = shape[0] if len(shape) == 1 and not isinstance(shape[0], int) else shape
        shape = torch.empty(self.shape, device="meta").reshape(*shape).shape
        if shape[-1] != self.shape[-1]:
            raise ValueError("an MXTensor keeps its last dimension")
        return MXTensor.__new__(MXTensor)._set(
            self._data, self._scales, self._buf, self.data_ptr, self.scales_ptr, self.index, shape,
            self.fmt, self.scale_exp, self.dtype)

    def dequantize(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The values that the codes stand for, ``[..., K]`` (default: the
        type the tensor was made from; exact in it unless they leave its range)."""
        dtype = self.dtype if dtype is None else dtype
        code = dtype_code(dtype, "dtype")
        if self.index < 0:
            raise RuntimeError("dequantize runs on the CUDA engine only (no CPU path)")
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        call(_lib.load().scmp_mx_dequantize, self.index, self.data_ptr, self.scales_ptr, self.rows,
             self.shape[-1], _lib.MX_FORMAT[self.fmt], self.scale_exp, out.data_ptr(), code)
        return out

    def __repr__(self) -> str:
        return (f"MXTensor(shape={tuple(self.shape)}, fmt={self.fmt!r}, "
                f"scale_exp={self.scale_exp}, dtype={self.dtype}, device={self.device})")


def mx_empty(shape: torch.Size, fmt: str, device: torch.device, dtype: torch.dtype,
             scale_exp: int = 0) -> MXTensor:
    """An MXTensor whose codes and scales (one allocation) are still to be written."""
    data, scales = _sizes(math.prod(shape[:-1]), shape[-1], _check_fmt(fmt))
    at = (data + 255) & ~255
    buf = torch.empty(at + scales, dtype=torch.uint8, device=device)
    ptr = buf.data_ptr()
    return MXTensor.__new__(MXTensor)._set(None, None, buf, ptr, ptr + at, buf.get_device(), shape,
                                           fmt, scale_exp, dtype)


def _rows_of(x: torch.Tensor):
    """(x or a copy of it, row distance) with contiguous rows a fixed distance apart."""
    K = x.shape[-1]
    if x.is_contiguous():
        return x, K
    x2 = x.detach().reshape(-1, K)
    if (K > 1 and x2.stride(1) != 1) or (x2.shape[0] > 1 and x2.stride(0) < K):
        x2 = x2.contiguous()
    return x2, (x2.stride(0) if x2.shape[0] > 1 else K)


def _thin(rows: int, N: int, K: int) -> bool:
    """Whether a few rows are quantised inside the product's own launch, which
    needs no buffers (the engine's rule for products of codes)."""
    return (rows <= _lib.MX_THIN_ROWS and K <= _lib.MX_THIN_K
            and K / 1024 * (N / 1024 * (1 + 0.7 * rows) + rows - 5) < 12)


def _overlap(out: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether contiguous ``out`` and ``t`` (its span, where strided) share bytes."""
    if t.numel() == 0 or out.numel() == 0:
        return False
    span = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1
    start, end = out.data_ptr(), out.data_ptr() + out.numel() * out.element_size()
    return t.data_ptr() < end and start < t.data_ptr() + span * t.element_size()


def _overlap_codes(out: torch.Tensor, q: "MXTensor") -> bool:
    """The same for ``q``'s codes and scales."""
    start, end = out.data_ptr(), out.data_ptr() + out.numel() * out.element_size()
    sizes = _sizes(q.rows, q.shape[-1], q.fmt)
    return any([p < end and start < p + n for p, n in zip((q.data_ptr, q.scales_ptr), sizes)])


def _check_input(x: torch.Tensor, name: str) -> int:
    code = dtype_code(x.dtype, "x")
    if not x.is_cuda:
        raise RuntimeError(f"{name} runs on the CUDA engine only (no CPU path); got {x.device}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} needs a last dimension of at least 1, got {tuple(x.shape)}")
    return code


def mx_quantize(x: torch.Tensor, fmt: str = "mxfp4", *, scale_exp: int = 0) -> MXTensor:
    """Quantise ``x`` (``[..., K]``, float32 / bfloat16 / float16, CUDA) along
    its last dimension.  ``scale_exp`` is nvfp4's power-of-two tensor scale
    (``tensor_scale_exp`` gives the one that suits a tensor; 0 suits normalised
    activations)."""
    _check_fmt(fmt)
    code = _check_input(x, "mx_quantize")
    _no_grad_wanted("mx_quantize", x)
    out = mx_empty(x.shape, fmt, x.device, x.dtype, _check_exp(scale_exp))
    x, ld = _rows_of(x)
    call(_lib.load().scmp_mx_quantize, out.index, x.data_ptr(), code, out.rows, out.shape[-1], ld,
         _lib.MX_FORMAT[fmt], out.scale_exp, out.data_ptr, out.scales_ptr)
    return out


def mx_matmul(a: Union[torch.Tensor, MXTensor], b: MXTensor, *,
              bias: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``a @ b^T`` (+ ``bias``) for ``a`` ``[..., K]`` and ``b`` ``[N, K]`` ->
    ``[..., N]``: the exact products of the 4-bit values summed in fp32, the
    bias added, rounded once to ``out_dtype`` (default: a's type).  A plain
    ``a`` is quantised to ``b``'s format first (nvfp4 with tensor scale 1).
    ``out`` is contiguous and shares no memory with the operands or ``bias``."""
    if not isinstance(b, MXTensor) or len(b.shape) != 2:
        raise TypeError("b must be a 2-D MXTensor [N, K]")
    if b.index < 0:
        raise RuntimeError("mx_matmul runs on the CUDA engine only (no CPU path)")
    N, K = b.shape
    plain = not isinstance(a, MXTensor)
    index = a.get_device() if plain else a.index
    if index != b.index:
        raise ValueError(f"operands on different devices: {a.device} vs {b.device}")
    if len(a.shape) < 1 or a.shape[-1] != K:
        raise ValueError(f"inner-dim mismatch: a {tuple(a.shape)}, b {tuple(b.shape)}")
    qa = a
    if plain:
        x_code = _check_input(a, "mx_matmul")
        rows = a.numel() // K
        qa = None if _thin(rows, N, K) else mx_empty(a.shape, b.fmt, a.device, a.dtype)
    elif a.fmt != b.fmt:
        raise ValueError(f"operands of different formats: {a.fmt} vs {b.fmt}")
    else:
        rows = a.rows
    _no_grad_wanted("mx_matmul", a if plain else None, bias, out)
    shape = (*a.shape[:-1], N)
    given = out is not None
    if not given:
        dtype = a.dtype if out_dtype is None else out_dtype
        out_code = dtype_code(dtype, "out")
        out = torch.empty(shape, dtype=dtype, device=b.device)
    else:
        if (tuple(out.shape) != shape or not out.is_contiguous() or out.get_device() != index
                or out_dtype not in (None, out.dtype)):
            raise ValueError(f"out must be contiguous {shape} on {b.device} of out_dtype")
        out_code = dtype_code(out.dtype, "out")
        if ((_overlap if plain else _overlap_codes)(out, a) or _overlap_codes(out, b)
                or (bias is not None and _overlap(out, bias))):
            raise ValueError("out shares memory with an input")
    bias_code, bias_ptr = 0, 0
    if bias is not None:
        if bias.shape != (N,) or bias.get_device() != index:
            raise ValueError(f"bias must be [{N}] on {b.device}, got {tuple(bias.shape)} on "
                             f"{bias.device}")
        bias_code = dtype_code(bias.dtype, "bias")
        bias = bias if bias.is_contiguous() else bias.detach().contiguous()
        bias_ptr = bias.data_ptr()
    args = _lib.PACK_MX_MATMUL.pack(
        _lib.ABI_VERSION, _lib.MX_FORMAT[b.fmt], 0 if qa is None else qa.data_ptr,
        0 if qa is None else qa.scales_ptr, b.data_ptr, b.scales_ptr, rows, N, K,
        b.scale_exp if plain else a.scale_exp + b.scale_exp, bias_code, bias_ptr, out.data_ptr(),
        out_code, 0)
    if plain:
        x, ld = _rows_of(a)
        call(_lib.load().scmp_mx_linear, index, x.data_ptr(), x_code, ld, args)
    else:
        call(_lib.load().scmp_mx_matmul, index, args)
    if given:
        torch.autograd.graph.increment_version(out)  # a write in place, as autograd counts them
    return out


@torch.no_grad()
def tensor_scale_exp(x: torch.Tensor) -> int:
    """The nvfp4 ``scale_exp`` that brings the largest block scale of ``x`` to
    between half of e4m3's largest value and that value (0 for a zero tensor).
    Reads the maximum back to the host."""
    top = float(x.abs().amax()) if x.numel() else 0.0
    if not 0.0 < top < math.inf:
        return 0
    return max(-60, min(60, math.floor(math.log2(top / (6 * 448))) + 1))


class MXLinear(nn.Module):
    """``nn.Linear`` with its weight in 4 bits, laid out once from ``linear``
    (on the GPU) when the module is made; activations are quantised per call,
    or come as an ``MXTensor`` from a fused producer.  Its buffers move with
    ``.to(device)`` and are saved with the module."""

    def __init__(self, linear: nn.Linear, fmt: str = "mxfp4"):
        super().__init__()
        w = linear.weight.detach()
        if w.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            w = w.float()
        exp = tensor_scale_exp(w) if _check_fmt(fmt) == "nvfp4" else 0
        q = mx_quantize(w, fmt, scale_exp=exp)
        self.fmt = fmt
        self.scale_exp = exp
        self.out_features, self.in_features = w.shape
        self.register_buffer("data", q.data.clone())
        self.register_buffer("scales", q.scales.clone())
        bias = linear.bias
        self.register_buffer("bias", None if bias is None else bias.detach().clone())

    def get_extra_state(self):
        return {"fmt": self.fmt, "scale_exp": self.scale_exp}

    def set_extra_state(self, state):
        # (the format fixes the buffers' sizes and was chosen with them)
        if state["fmt"] != self.fmt:
            raise ValueError(f"saved in {state['fmt']}, this module is {self.fmt}")
        self.scale_exp = int(state["scale_exp"])

    def quantized_weight(self) -> MXTensor:
        data, scales = self.data, self.scales
        # (buffers can be assigned: a state dict's own tensors, of any kind)
        _check_bytes(data, scales, _sizes(self.out_features, self.in_features, self.fmt))
        return MXTensor.__new__(MXTensor)._set(
            data, scales, None, data.data_ptr(), scales.data_ptr(), data.get_device(),
            torch.Size((self.out_features, self.in_features)), self.fmt, self.scale_exp,
            torch.float32)

    def forward(self, x: Union[torch.Tensor, MXTensor]) -> torch.Tensor:
        return mx_matmul(x, self.quantized_weight(), bias=self.bias)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, fmt={self.fmt!r}")
