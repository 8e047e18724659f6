"""8-bit floating point with a scale per block of 128: quantisation, product and
a linear that is trained in it.

The 4-bit products of ``mx`` serve; this module trains as well, on the same
tensor-core path (e4m3 codes, power-of-two block scales that the hardware applies):

* ``fp8_quantize(x, blocks)`` -> ``FP8Tensor``: e4m3 codes with one scale
  ``2^E`` per block, the smallest (from ``2^-127`` on) under which the block's
  largest magnitude is at most 448.  ``"row"``: 128 consecutive elements of the
  last dimension (activations); ``"square"``: 128 x 128 elements (weights, whose
  transpose then has the same codes).  Codes are rounded to nearest even.  A block
  with a NaN or an infinity stands for NaNs.
* ``FP8Tensor.dequantize()``: the values that the codes stand for.
* ``fp8_matmul(a, b)``: ``a @ b^T`` (+ bias) with fp32 sums; ``a`` may be a plain
  tensor, which is quantised along its rows on the way in.  Inference only.
* ``fp8_linear(x, weight, bias)``: the same of a plain weight, differentiable: its
  three products take 8-bit operands.
* ``FP8Linear``: an ``nn.Linear`` served in 8 bits (its weight laid out once), or
  with ``train=True`` trained in 8 bits (its parameters stay what they were).

There is no CPU path: CPU tensors raise.
"""
from __future__ import annotations

import functools
import math
from typing import Optional, Sequence, Tuple, Union

import torch
import torch.nn as nn

from . import _lib
from ._call import DTYPE, call, dtype_code, has_tangent, once_differentiable
from .mx import _check_bytes, _check_input, _no_grad_wanted, _overlap, _rows_of

__all__ = ["FP8Tensor", "fp8_quantize", "fp8_matmul", "fp8_linear", "FP8Linear"]

BLOCKS = ("row", "square")


def _sizes(rows: int, K: int) -> Tuple[int, int]:
    """Bytes of codes and of scales (``scmp_fp8_data_size``, ``scmp_fp8_scale_size``)."""
    return rows * ((K + 127) // 128 * 128), (rows + 127) // 128 * ((K + 511) // 512) * 512


class FP8Tensor:
    """A quantised tensor ``[..., K]``: codes and block scales on the GPU.

    ``data`` and ``scales`` (uint8) have the layout of ``scmp_fp8_quantize`` (rows
    are the leading dimensions flattened); ``blocks`` is ``"row"`` or ``"square"``
    (for the record: both have one layout); ``dtype`` is the type of the tensor it
    was made from, which products of it come out in by default."""

    __slots__ = ("shape", "rows", "blocks", "dtype", "_data", "_scales", "_buf", "data_ptr",
                 "scales_ptr", "index")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, shape: Sequence[int],
                 blocks: str = "row", dtype: torch.dtype = torch.float32):
        shape = torch.Size(shape)
        if not shape or shape[-1] < 1 or min(shape) < 0:
            raise ValueError("an FP8Tensor has a last dimension of at least 1 and none below 0, "
                             f"got {tuple(shape)}")
        if blocks not in BLOCKS:
            raise ValueError(f"unknown blocks {blocks!r} (one of {BLOCKS})")
        self.rows = math.prod(shape[:-1])
        _check_bytes(data, scales, _sizes(self.rows, shape[-1]))
        if data.device != scales.device:
            raise ValueError(f"data on {data.device}, scales on {scales.device}")
        if data.data_ptr() % 16 or scales.data_ptr() % 16:
            raise ValueError("data and scales must be 16-byte aligned")
        self._set(data, scales, None, data.data_ptr(), scales.data_ptr(), data.get_device(), shape,
                  self.rows, blocks, dtype)

    def _set(self, data, scales, buf, data_ptr, scales_ptr, index, shape, rows, blocks, dtype):
        self._data, self._scales, self._buf = data, scales, buf
        self.data_ptr, self.scales_ptr, self.index = data_ptr, scales_ptr, index
        self.shape, self.rows, self.blocks, self.dtype = shape, rows, blocks, dtype
        return self

    @property
    def data(self) -> torch.Tensor:
        if self._data is None:
            self._data = self._buf[:_sizes(self.rows, self.shape[-1])[0]]
        return self._data

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            at = self.scales_ptr - self.data_ptr
            self._scales = self._buf[at:at + _sizes(self.rows, self.shape[-1])[1]]
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
        return FP8Tensor, (self.data, self.scales, tuple(self.shape), self.blocks, self.dtype)

    def reshape(self, *shape) -> "FP8Tensor":
        """The same codes under other leading dimensions; the last one stays."""
        shape = shape[0] if len(shape) == 1 and not isinstance(shape[0], int) else shape
        shape = torch.empty(self.shape, device="meta").reshape(*shape).shape
        if not shape or shape[-1] != self.shape[-1]:
            raise ValueError("an FP8Tensor keeps its last dimension")
        return FP8Tensor.__new__(FP8Tensor)._set(
            self._data, self._scales, self._buf, self.data_ptr, self.scales_ptr, self.index, shape,
            self.rows, self.blocks, self.dtype)

    def dequantize(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The values that the codes stand for, ``[..., K]`` (default: the type
        the tensor was made from; exact in it unless they leave its range)."""
        dtype = self.dtype if dtype is None else dtype
        code = dtype_code(dtype, "dtype")
        if self.index < 0:
            raise RuntimeError("dequantize runs on the CUDA engine only (no CPU path)")
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        call(_lib.load().scmp_fp8_dequantize, self.index, self.data_ptr, self.scales_ptr,
             self.rows, self.shape[-1], out.data_ptr(), code)
        return out

    def __repr__(self) -> str:
        return (f"FP8Tensor(shape={tuple(self.shape)}, blocks={self.blocks!r}, "
                f"dtype={self.dtype}, device={self.device})")


def fp8_empty(shape: Sequence[int], device: torch.device, dtype: torch.dtype,
              blocks: str = "row") -> FP8Tensor:
    """An FP8Tensor whose codes and scales (one allocation) are still to be written."""
    shape = torch.Size(shape)
    rows = math.prod(shape[:-1])
    data, scales = _sizes(rows, shape[-1])
    buf = torch.empty(data + scales, dtype=torch.uint8, device=device)
    ptr = buf.data_ptr()  # (rows of codes are whole 128-byte blocks: the scales are aligned)
    return FP8Tensor.__new__(FP8Tensor)._set(None, None, buf, ptr, ptr + data, buf.get_device(),
                                             shape, rows, blocks, dtype)


def fp8_quantize(x: torch.Tensor, blocks: str = "row", *, transpose: bool = False
                 ) -> Union[FP8Tensor, Tuple[FP8Tensor, FP8Tensor]]:
    """Quantise ``x`` (``[..., K]``, float32 / bfloat16 / float16, CUDA) in blocks
    of 128 elements of the last dimension (``"row"``) or, 2-D, of 128 x 128
    (``"square"``).  ``transpose`` (2-D) also returns its transpose ``[K, rows]``,
    quantised along its own rows, from the same pass: ``(q, q_t)``."""
    if blocks not in BLOCKS:
        raise ValueError(f"unknown blocks {blocks!r} (one of {BLOCKS})")
    code = _check_input(x, "fp8_quantize")
    if x.dim() != 2 and (blocks == "square" or transpose):
        raise ValueError(f"squares and transposes are of matrices, got {tuple(x.shape)}")
    if transpose and x.shape[0] < 1:
        raise ValueError("the transpose of no rows has no last dimension")
    _no_grad_wanted("fp8_quantize", x)
    q = fp8_empty(x.shape, x.device, x.dtype, blocks)
    t = fp8_empty((x.shape[1], x.shape[0]), x.device, x.dtype, blocks) if transpose else None
    x, ld = _rows_of(x)
    args = _lib.PACK_FP8_QUANTIZE.pack(
        _lib.ABI_VERSION, code, x.data_ptr(), q.rows, q.shape[-1], ld, blocks == "square", 0,
        q.data_ptr, q.scales_ptr, 0 if t is None else t.data_ptr,
        0 if t is None else t.scales_ptr)
    call(_lib.load().scmp_fp8_quantize, q.index, args)
    return q if t is None else (q, t)


def _thin(rows: int, N: int, K: int) -> bool:
    """Whether a few rows are quantised inside the product's own launch, which
    needs no buffers (the engine's rule for products of codes)."""
    return (rows <= _lib.FP8_THIN_ROWS and K <= _lib.FP8_THIN_K
            and K / 1024 * (N / 1024 * (0.03 + 0.17 * rows) + 0.2 * rows - 1.6) < 3.2)


def _overlap_codes(out: torch.Tensor, q: FP8Tensor) -> bool:
    """Whether contiguous ``out`` shares bytes with ``q``'s codes or scales."""
    return _overlap(out, q.data) or _overlap(out, q.scales)


def fp8_matmul(a: Union[torch.Tensor, FP8Tensor], b: FP8Tensor, *,
               bias: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``a @ b^T`` (+ ``bias``) for ``a`` ``[..., K]`` and ``b`` ``[N, K]`` ->
    ``[..., N]``: products of the 8-bit values summed in fp32, the bias added,
    rounded once to ``out_dtype`` (default: a's type).  A plain ``a`` is quantised
    along its rows first.  ``out`` is contiguous and shares no memory with the
    operands or ``bias``.  No gradient (``fp8_linear`` has one)."""
    if not isinstance(b, FP8Tensor) or len(b.shape) != 2:
        raise TypeError("b must be a 2-D FP8Tensor [N, K]")
    if b.index < 0:
        raise RuntimeError("fp8_matmul runs on the CUDA engine only (no CPU path)")
    N, K = b.shape
    plain = not isinstance(a, FP8Tensor)
    index = a.get_device() if plain else a.index
    if index != b.index:
        raise ValueError(f"operands on different devices: {a.device} vs {b.device}")
    if len(a.shape) < 1 or a.shape[-1] != K:
        raise ValueError(f"inner-dim mismatch: a {tuple(a.shape)}, b {tuple(b.shape)}")
    codes = None  # of a plain a: freed to the stream's later calls when this one returns
    a_ptr = a_scales_ptr = 0
    if plain:
        x_code = _check_input(a, "fp8_matmul")
        rows = a.numel() // K
        if not _thin(rows, N, K):
            data, scales = _sizes(rows, K)
            codes = a.new_empty(data + scales, dtype=torch.uint8)  # (cheaper than torch.empty)
            a_ptr = codes.data_ptr()
            a_scales_ptr = a_ptr + data
    else:
        rows, a_ptr, a_scales_ptr = a.rows, a.data_ptr, a.scales_ptr
    _no_grad_wanted("fp8_matmul", a if plain else None, bias, out)
    shape = (*a.shape[:-1], N)
    given = out is not None
    if not given:
        dtype = a.dtype if out_dtype is None else out_dtype
        out_code = dtype_code(dtype, "out")
        out = (a.new_empty(shape, dtype=dtype) if plain else
               torch.empty(shape, dtype=dtype, device=b.device))
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
        bias_code = _check_bias(bias, N, b.device, index)
        bias = bias if bias.is_contiguous() else bias.detach().contiguous()
        bias_ptr = bias.data_ptr()
    args = _lib.PACK_FP8_MATMUL.pack(
        _lib.ABI_VERSION, bias_code, a_ptr, a_scales_ptr, b.data_ptr, b.scales_ptr, rows, N, K,
        bias_ptr, out.data_ptr(), out_code, 0)
    if plain:
        x, ld = _rows_of(a)
        call(_lib.load().scmp_fp8_linear, index, x.data_ptr(), x_code, ld, args)
    else:
        call(_lib.load().scmp_fp8_matmul, index, args)
    if given:
        torch.autograd.graph.increment_version(out)  # a write in place, as autograd counts them
    return out


def _check_bias(bias, N, device, index) -> int:
    if bias.shape != (N,) or bias.get_device() != index:
        raise ValueError(f"bias must be [{N}] on {device}, got {tuple(bias.shape)} on "
                         f"{bias.device}")
    return dtype_code(bias.dtype, "bias")


@functools.lru_cache(maxsize=256)
def _train_sizes(M: int, N: int, K: int) -> Tuple[int, int, int, int]:
    """Bytes of both workspaces and of the saved codes of x and of the weight."""
    lib = _lib.load()
    return (lib.scmp_fp8_train_workspace(M, N, K, 0), lib.scmp_fp8_train_workspace(M, N, K, 1),
            lib.scmp_fp8_train_saved_size(M, K), lib.scmp_fp8_train_saved_size(N, K))


def _train_forward(x, weight, bias, save_x: bool, save_weight: bool):
    """(y, codes of x^T and of weight^T in one buffer or None, where the second begins)."""
    N, K = weight.shape
    y = x.new_empty((*x.shape[:-1], N))
    index = x.get_device()
    xr, ld = _rows_of(x)
    M = x.numel() // K
    if M == 0:
        return y, None, 0
    wr, weight_ld = _rows_of(weight)
    bias = bias if bias is None or bias.is_contiguous() else bias.detach().contiguous()
    workspace, _, x_bytes, w_bytes = _train_sizes(M, N, K)
    ws = x.new_empty(workspace, dtype=torch.uint8)
    x_bytes = x_bytes if save_x else 0  # (multiples of 256)
    saved, ptr = None, 0
    if save_x or save_weight:
        saved = x.new_empty(x_bytes + (w_bytes if save_weight else 0), dtype=torch.uint8)
        ptr = saved.data_ptr()
    args = _lib.PACK_FP8_TRAIN.pack(
        _lib.ABI_VERSION, DTYPE[x.dtype], DTYPE[weight.dtype],
        0 if bias is None else DTYPE[bias.dtype], xr.data_ptr(), wr.data_ptr(),
        0 if bias is None else bias.data_ptr(), y.data_ptr(),
        ptr if save_x else 0, ptr + x_bytes if save_weight else 0, ws.data_ptr(), workspace, M, N,
        K, ld, weight_ld)
    call(_lib.load().scmp_fp8_train_forward, index, args)
    return y, saved, x_bytes


class _FP8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        wants = ctx.needs_input_grad
        y, saved, ctx.weight_at = _train_forward(x, weight, bias, wants[1], wants[0])
        # (codes alone: nothing of x or weight is kept for the backward pass)
        ctx.save_for_backward(saved)
        ctx.like = (x.shape, weight.shape, x.dtype, weight.dtype,
                    None if bias is None else bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (saved,) = ctx.saved_tensors
        x_shape, (N, K), dtype, weight_dtype, bias_dtype = ctx.like
        wants = ctx.needs_input_grad
        M = math.prod(x_shape[:-1])
        new = dy.new_zeros if M == 0 else dy.new_empty  # (no rows: sums of nothing)
        dx = new(x_shape, dtype=dtype) if wants[0] else None
        dw = new((N, K), dtype=weight_dtype) if wants[1] else None
        db = new(N, dtype=bias_dtype) if wants[2] else None
        if M:
            dyr, ld = _rows_of(dy)
            size = _train_sizes(M, N, K)[1]
            ptr = 0 if saved is None else saved.data_ptr()
            ws = dy.new_empty(size, dtype=torch.uint8)
            args = _lib.PACK_FP8_TRAIN_BWD.pack(
                _lib.ABI_VERSION, DTYPE[dtype], DTYPE[weight_dtype],
                0 if db is None else DTYPE[bias_dtype], dyr.data_ptr(),
                ptr if wants[1] else 0, ptr + ctx.weight_at if wants[0] else 0,
                *[0 if t is None else t.data_ptr() for t in (dx, dw, db)], ws.data_ptr(), size,
                M, N, K, ld)
            call(_lib.load().scmp_fp8_train_backward, dy.get_device(), args)
        return dx, dw, db


def fp8_linear(x: torch.Tensor, weight: torch.Tensor,
               bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ weight^T`` (+ ``bias``) in 8 bits, for training: ``x`` ``[..., K]``,
    ``weight`` ``[N, K]``, ``bias`` ``[N]``, each float32, bfloat16 or float16 ->
    ``[..., N]`` of x's type.  With Q the values of 8-bit codes::

        y  = Q(x) Q(W)^T + bias    x in blocks of 128 along its rows, W in squares
        dx = Q(dy) Q(W)            dy in blocks along its rows
        dW = Q(dy)^T Q(x)          both in blocks of 128 tokens along their columns
        db = sum of dy over tokens

    Sums in fp32 (the tensor core's, which are cut off and not rounded; long ones in
    pieces: ``scmp_fp8_matmul``), each result rounded once to its tensor's type.  Differentiable
    (once, backward) in all three, as if Q passed gradients through.  Kept for the
    backward pass are codes only, one byte per element of ``x`` and ``weight``.
    The weight is quantised in every call.  Under autocast as anywhere else y is of
    x's own type."""
    _check_input(x, "fp8_linear")
    dtype_code(weight.dtype, "weight")
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must be [N, K], got {tuple(weight.shape)}")
    if x.shape[-1] != weight.shape[1]:
        raise ValueError(f"inner-dim mismatch: x {tuple(x.shape)}, weight {tuple(weight.shape)}")
    index = x.get_device()
    if weight.get_device() != index:
        raise ValueError(f"operands on different devices: {x.device} vs {weight.device}")
    leaves = (x, weight, bias)
    if bias is not None:
        _check_bias(bias, weight.shape[0], x.device, index)
    if (torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in leaves])
            ) or has_tangent(leaves):
        # (a forward-mode tangent is refused there: the function has no jvp)
        return _FP8Linear.apply(x, weight, bias)
    return _train_forward(x, weight, bias, False, False)[0]


class FP8Linear(nn.Module):
    """``nn.Linear`` in 8 bits.  Served (the default): its weight is laid out once
    from ``linear`` (on the GPU) when the module is made; activations are quantised
    per call, or come as an ``FP8Tensor``; buffers move with ``.to(device)`` and are
    saved with the module.  ``train=True``: ``linear``'s parameters themselves, in
    ``fp8_linear``."""

    def __init__(self, linear: nn.Linear, train: bool = False):
        super().__init__()
        self.out_features, self.in_features = linear.weight.shape
        self.trained = bool(train)
        if self.trained:
            self.weight, self.bias = linear.weight, linear.bias
            return
        w = linear.weight.detach()
        if w.dtype not in DTYPE:
            w = w.float()
        q = fp8_quantize(w, "square")
        self.register_buffer("data", q.data.clone())
        self.register_buffer("scales", q.scales.clone())
        bias = linear.bias
        self.register_buffer("bias", None if bias is None else bias.detach().clone())

    def quantized_weight(self) -> FP8Tensor:
        """The weight's codes (a trained module's present ones)."""
        if self.trained:
            return fp8_quantize(self.weight.detach(), "square")
        # (buffers can be assigned: a state dict's own tensors, of any kind)
        return FP8Tensor(self.data, self.scales, (self.out_features, self.in_features), "square")

    def forward(self, x: Union[torch.Tensor, FP8Tensor]) -> torch.Tensor:
        if self.trained:
            return fp8_linear(x, self.weight, self.bias)
        return fp8_matmul(x, self.quantized_weight(), bias=self.bias)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, train={self.trained}")
