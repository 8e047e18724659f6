"""Microscaled 4-bit floating point: quantisation and product.

The SC engine's products run as e2m1 multiply-adds with unit scales; this
module offers the same tensor-core operands with real block scales, i.e. the
deterministic 4-bit linear that an SC linear is compared with.

* ``mx_quantize(x, fmt)`` -> ``MXTensor``: e2m1 codes with one scale per block
  of the last dimension.  ``"mxfp4"``: blocks of 32, power-of-two scales
  ``2^(floor(log2 max|x|) - 2)``.  ``"nvfp4"``: blocks of 16, e4m3 scales
  ``max|x| / 6`` under a power-of-two tensor scale ``2^scale_exp``.  Codes are
  rounded to nearest even and saturate at 6.  A block with a NaN or an
  infinity stands for NaNs.
* ``MXTensor.dequantize()``: the values that the codes stand for.
* ``mx_matmul(a, b)``: ``a @ b^T`` (+ bias) with fp32 sums; ``a`` may be a
  plain tensor, which is quantised to ``b``'s format on the way in.
* ``MXLinear``: an ``nn.Linear`` with its weight in 4 bits.

Inference only: there is no gradient, and an input that asks for one is
refused.  There is no CPU path: CPU tensors raise.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Union

import torch
import torch.nn as nn

from . import _lib

__all__ = ["MXTensor", "mx_quantize", "mx_matmul", "MXLinear", "tensor_scale_exp"]


def _dtype_code(dtype: torch.dtype, what: str) -> int:
    code = _lib.DTYPE.get(str(dtype))
    if code is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {dtype}")
    return code


def _check_fmt(fmt: str) -> str:
    if fmt not in _lib.MX_FORMAT:
        raise ValueError(f"unknown 4-bit format {fmt!r} (one of {sorted(_lib.MX_FORMAT)})")
    return fmt


def _no_grad_wanted(name: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no gradient; call it under torch.no_grad() or on "
                           "detached inputs")


def _stream(dev: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)


class MXTensor:
    """A quantised tensor ``[..., K]``: codes and block scales on the GPU.

    ``data`` and ``scales`` have the layout of ``scmp_mx_quantize`` (rows are
    the leading dimensions flattened); ``dtype`` is the type of the tensor it
    was made from, which products of it come out in by default."""

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, shape: Sequence[int], fmt: str,
                 scale_exp: int = 0, dtype: torch.dtype = torch.float32):
        self.data = data
        self.scales = scales
        self.shape = torch.Size(shape)
        self.fmt = _check_fmt(fmt)
        self.scale_exp = int(scale_exp)
        self.dtype = dtype
        lib = _lib.load()
        rows, K = self.rows, self.shape[-1]
        for t, size, what in ((data, lib.scmp_mx_data_size(rows, K, _lib.MX_FORMAT[fmt]), "data"),
                              (scales, lib.scmp_mx_scale_size(rows, K, _lib.MX_FORMAT[fmt]),
                               "scales")):
            if t.dtype != torch.uint8 or not t.is_contiguous() or t.numel() != size:
                raise ValueError(f"{what} must be {size} contiguous bytes for {tuple(self.shape)}")

    @property
    def rows(self) -> int:
        return math.prod(self.shape[:-1])

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def is_cuda(self) -> bool:
        return self.data.is_cuda

    def dim(self) -> int:
        return len(self.shape)

    def reshape(self, *shape) -> "MXTensor":
        """The same codes under other leading dimensions; the last one stays."""
        shape = shape[0] if len(shape) == 1 and not isinstance(shape[0], int) else shape
        shape = torch.empty(self.shape, device="meta").reshape(*shape).shape
        if shape[-1] != self.shape[-1]:
            raise ValueError("an MXTensor keeps its last dimension")
        return MXTensor(self.data, self.scales, shape, self.fmt, self.scale_exp, self.dtype)

    @torch.no_grad()
    def dequantize(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The values that the codes stand for, ``[..., K]`` (default: the
        type the tensor was made from; exact in it unless they leave its range)."""
        dtype = self.dtype if dtype is None else dtype
        code = _dtype_code(dtype, "dtype")
        if not self.is_cuda:
            raise RuntimeError("dequantize runs on the CUDA engine only (no CPU path)")
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        with torch.cuda.device(self.device):
            _lib.check(_lib.load().scmp_mx_dequantize(
                self.data.data_ptr(), self.scales.data_ptr(), self.rows, self.shape[-1],
                _lib.MX_FORMAT[self.fmt], self.scale_exp, out.data_ptr(), code,
                _stream(self.device)))
        return out

    def __repr__(self) -> str:
        return (f"MXTensor(shape={tuple(self.shape)}, fmt={self.fmt!r}, "
                f"scale_exp={self.scale_exp}, dtype={self.dtype}, device={self.device})")


def mx_empty(shape: Sequence[int], fmt: str, device: torch.device, dtype: torch.dtype,
             scale_exp: int = 0) -> MXTensor:
    """An MXTensor whose codes and scales are still to be written."""
    lib = _lib.load()
    rows, K = math.prod(shape[:-1]), shape[-1]
    code = _lib.MX_FORMAT[_check_fmt(fmt)]
    data = torch.empty(lib.scmp_mx_data_size(rows, K, code), dtype=torch.uint8, device=device)
    scales = torch.empty(lib.scmp_mx_scale_size(rows, K, code), dtype=torch.uint8, device=device)
    return MXTensor(data, scales, shape, fmt, scale_exp, dtype)


def _as_rows(x: torch.Tensor) -> torch.Tensor:
    """``[rows, K]`` with contiguous rows a fixed distance apart (a view where
    the strides allow it)."""
    K = x.shape[-1]
    x2 = x.reshape(-1, K)
    if K > 1 and x2.stride(1) != 1 or x2.shape[0] > 1 and x2.stride(0) < K:
        x2 = x2.contiguous()
    return x2


def mx_quantize(x: torch.Tensor, fmt: str = "mxfp4", *, scale_exp: int = 0) -> MXTensor:
    """Quantise ``x`` (``[..., K]``, float32 / bfloat16 / float16, CUDA) along
    its last dimension.  ``scale_exp`` is nvfp4's power-of-two tensor scale
    (``tensor_scale_exp`` gives the one that suits a tensor; 0 suits normalised
    activations)."""
    fmt = _check_fmt(fmt)
    code = _dtype_code(x.dtype, "x")
    if not x.is_cuda:
        raise RuntimeError(f"mx_quantize runs on the CUDA engine only (no CPU path); got {x.device}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"mx_quantize needs a last dimension of at least 1, got {tuple(x.shape)}")
    _no_grad_wanted("mx_quantize", x)
    out = mx_empty(x.shape, fmt, x.device, x.dtype, scale_exp)
    x2 = _as_rows(x.detach()) if out.rows else x
    K = x.shape[-1]
    ld = x2.stride(0) if out.rows > 1 else K
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().scmp_mx_quantize(
            x2.data_ptr(), code, out.rows, K, ld, _lib.MX_FORMAT[fmt], int(scale_exp),
            out.data.data_ptr(), out.scales.data_ptr(), _stream(x.device)))
    return out


def mx_matmul(a: Union[torch.Tensor, MXTensor], b: MXTensor, *,
              bias: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``a @ b^T`` (+ ``bias``) for ``a`` ``[..., K]`` and ``b`` ``[N, K]`` ->
    ``[..., N]``: the exact products of the 4-bit values summed in fp32, the
    bias added, rounded once to ``out_dtype`` (default: a's type).  A plain
    ``a`` is quantised to ``b``'s format first (nvfp4 with tensor scale 1)."""
    if not isinstance(b, MXTensor) or b.dim() != 2:
        raise TypeError("b must be a 2-D MXTensor [N, K]")
    if not isinstance(a, MXTensor):
        if a.device != b.device:
            raise ValueError(f"operands on different devices: {a.device} vs {b.device}")
        if a.dim() < 1 or a.shape[-1] != b.shape[-1]:
            raise ValueError(f"inner-dim mismatch: a {tuple(a.shape)}, b {tuple(b.shape)}")
        a = mx_quantize(a, b.fmt)
    if a.device != b.device or not b.is_cuda:
        raise ValueError(f"operands on different devices or on the CPU: {a.device} vs {b.device}")
    if a.fmt != b.fmt:
        raise ValueError(f"operands of different formats: {a.fmt} vs {b.fmt}")
    N, K = b.shape
    if a.shape[-1] != K:
        raise ValueError(f"inner-dim mismatch: a {tuple(a.shape)}, b {tuple(b.shape)}")
    _no_grad_wanted("mx_matmul", bias)
    shape = (*a.shape[:-1], N)
    if out is None:
        out = torch.empty(shape, dtype=a.dtype if out_dtype is None else out_dtype, device=b.device)
    elif (tuple(out.shape) != shape or not out.is_contiguous() or out.device != b.device
          or out_dtype not in (None, out.dtype)):
        raise ValueError(f"out must be contiguous {shape} on {b.device} of out_dtype")
    _no_grad_wanted("mx_matmul", out)
    args = _lib.MxMatmulArgs()
    args.abi_version = _lib.ABI_VERSION
    args.fmt = _lib.MX_FORMAT[b.fmt]
    args.a, args.a_scales = a.data.data_ptr(), a.scales.data_ptr()
    args.b, args.b_scales = b.data.data_ptr(), b.scales.data_ptr()
    args.M, args.N, args.K = a.rows, N, K
    args.scale_exp = a.scale_exp + b.scale_exp
    if bias is not None:
        if bias.shape != (N,) or bias.device != b.device:
            raise ValueError(f"bias must be [{N}] on {b.device}, got {tuple(bias.shape)}")
        args.bias_dtype = _dtype_code(bias.dtype, "bias")
        bias = bias.detach().contiguous()
        args.bias = bias.data_ptr()
    args.out_dtype = _dtype_code(out.dtype, "out")
    args.out = out.data_ptr()
    with torch.cuda.device(b.device):
        _lib.check(_lib.load().scmp_mx_matmul(ctypes.byref(args), _stream(b.device)))
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
        self.register_buffer("data", q.data)
        self.register_buffer("scales", q.scales)
        bias = linear.bias
        self.register_buffer("bias", None if bias is None else bias.detach().clone())

    def quantized_weight(self) -> MXTensor:
        return MXTensor(self.data, self.scales, (self.out_features, self.in_features), self.fmt,
                        self.scale_exp)

    def forward(self, x: Union[torch.Tensor, MXTensor]) -> torch.Tensor:
        return mx_matmul(x, self.quantized_weight(), bias=self.bias)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, fmt={self.fmt!r}")
