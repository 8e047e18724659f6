"""DINOv2-style ViT-L/14 with a linear head, and the SC patcher the benchmark
uses.

The model carries the attribute names the reference's patchers rely on
(``cls/sc_attention_patch.py:335-341,459-636``): ``backbone.blocks[i].attn``
with ``qkv``, ``proj``, ``proj_drop``, ``num_heads``, ``scale``; an ``Mlp``
class with ``fc1`` / ``fc2``; and a 1000-way head on the concatenation of the
CLS token and the mean patch token (2048 -> 1000).  Weights are random
(seeded); there are no checkpoints in this environment.

With ``rope`` the attention turns q and k by the patches' (height, width), as
EVA-type blocks do, with ``qk_norm`` it normalises them first.  ``patch_vit_mx``
puts the linears in microscaled 4 bits instead (``mx.MXLinear``, the deterministic
counterpart of the SC linears), ``patch_vit_fp8`` in 8 bits, for training too, and
``set_fused_norm`` runs the blocks' residual adds and norms in one pass each,
with gradients.  ``set_dropout`` gives the blocks dropout and stochastic depth.

``patch_vit`` installs the SC operators per block: ``qkv_proj`` /
``out_proj`` / ``mlp_fc1`` / ``mlp_fc2`` as ``SCLinear``, Q@K^T and Attn@V
through the batched attention core, optional per-block pools (e.g. an
LFSR-16 pool seeded per block) and optional head-aligned compensation
``out = block(x) + comp(x)``.
"""
from __future__ import annotations

import functools
import threading
from typing import Callable, Dict, Iterable, Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _lib
from ._call import (DTYPE, call, has_tangent, in_backward, in_dual_level,
                    once_differentiable)
from .attention import GridRotary, QKNorm, make_sc_attention_forward
from .fp8 import FP8Linear
from .head_aligned_comp import HeadAlignedSCLinear
from .mp import SeededRandomMPConfig, quantile_counts, set_current_block_idx
from .mx import MXLinear
from .sc_linear import PackedWeights, SCLinear, _get_config, sc_linear_rows


def _fp_linear(lin: nn.Module, x: torch.Tensor) -> torch.Tensor:
    """``lin(x)``; a plain ``nn.Linear`` with a bias on a CUDA input runs as a
    matmul followed by an in-place bias add.  On B200 with fp32 operands that
    is the same cuBLAS GEMM kernel as ``F.linear`` and the same single
    rounding of ``acc + bias`` as its bias epilogue (identical bits), without
    the epilogue's extra pass: ViT-L/14 fc1 at 128 images 5.07 -> 4.72 ms,
    fc2 4.42 -> 4.33 ms.  CPU inputs keep ``F.linear``, whose ``addmm`` adds
    the bias inside the GEMM, and so do 16-bit ones (the epilogue adds the
    bias before the output is rounded)."""
    if (type(lin) is not nn.Linear or lin.bias is None or not x.is_cuda
            or x.dtype != torch.float32 or lin.weight.dtype != torch.float32):
        return lin(x)
    x2 = x.reshape(-1, x.shape[-1])
    y = torch.mm(x2, lin.weight.t()).add_(lin.bias)
    return y.reshape(*x.shape[:-1], y.shape[-1])


# Whether the blocks run their fp32 elementwise steps fused on the engine
# (scmp_bias_gelu, scmp_scale_residual); identical bits either way.
FUSED_GLUE = True


def set_fused_glue(flag: bool) -> None:
    """Turn the fused fp32 block glue on or off (results are identical)."""
    global FUSED_GLUE
    FUSED_GLUE = bool(flag)


# Whether the blocks run a residual add and the norm behind it in one pass
# (residual_norm), in training too.  The sums' order differs from
# nn.LayerNorm's, so this is off unless asked for; blocks with 4-bit linears
# always do.
FUSED_NORM = False


def set_fused_norm(flag: bool) -> None:
    """Turn the blocks' fused residual adds and norms on or off.  A block with
    hooks on its norms or its first layer scale, which one pass would not call,
    keeps the separate ones."""
    global FUSED_NORM
    FUSED_NORM = bool(flag)


def _check_glue(like: torch.Tensor, **tensors) -> None:
    """The glue kernels take fp32 CUDA tensors, contiguous and of one shape, and
    per-column parameters; anything else would be read past its end."""
    if not like.is_cuda:
        raise RuntimeError(f"the fused block glue runs on the CUDA engine only (no CPU path); "
                           f"got {like.device}")
    if not like.dim():
        raise ValueError("the fused block glue takes rows [..., C]")
    for name, t in tensors.items():
        if t is None:
            continue
        if t.dtype != torch.float32:
            raise TypeError(f"{name} must be float32, got {t.dtype}")
        want = like.shape[-1:] if name in ("gamma", "bias") else like.shape
        if t.shape != want or t.device != like.device or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous {list(want)} on {like.device}, got "
                             f"{tuple(t.shape)} strides {t.stride()} on {t.device}")


def bias_gelu_(t: torch.Tensor, bias: torch.Tensor) -> torch.Tensor:
    """``t = gelu(t + bias)`` in place (fp32 CUDA ``[..., C]``, exact GELU):
    the bias add and torch's erf-form GELU in one pass, same bits."""
    _check_glue(t, t=t, bias=bias)
    C = t.shape[-1]
    call(_lib.load().scmp_bias_gelu, t.get_device(), t.data_ptr(), bias.data_ptr(),
         t.numel() // max(1, C), C)
    return t


def scale_residual(x: torch.Tensor, y: torch.Tensor, gamma: torch.Tensor,
                   bias: Optional[torch.Tensor] = None, extra: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``(x + (y [+ bias]) * gamma) [+ extra]`` (fp32 CUDA ``[..., C]``, all
    contiguous and of one shape): a block's layer-scaled residual add, with an
    unfused bias and a compensation term, in one pass; each step rounded as
    the separate torch ops round it.  ``out`` may be ``x`` or ``y``."""
    _check_glue(x, x=x, y=y, gamma=gamma, bias=bias, extra=extra, out=out)
    C = x.shape[-1]
    out = torch.empty_like(x) if out is None else out
    call(_lib.load().scmp_scale_residual, x.get_device(), out.data_ptr(), x.data_ptr(),
         y.data_ptr(), _ptr(bias), gamma.data_ptr(), _ptr(extra), x.numel() // max(1, C), C)
    return out


def _watched(*modules: Optional[nn.Module]) -> bool:
    """Whether hooks watch the modules' calls."""
    return bool(torch.nn.modules.module._has_any_global_hook()) or any(
        m is not None and bool(m._forward_hooks or m._forward_pre_hooks or m._backward_hooks
                               or m._backward_pre_hooks) for m in modules)


_NORM_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check_norm(x, y, weight, norm_bias, kind, eps, gamma, gate, post_weight, post_bias) -> None:
    """Refuses what ``residual_norm`` does not take."""
    if kind not in ("layer", "rms"):
        raise ValueError(f"unknown norm kind {kind!r}")
    if not (isinstance(eps, (int, float)) and eps >= 0):
        raise ValueError(f"eps must be >= 0, got {eps!r}")
    if not x.is_cuda:
        raise RuntimeError(f"residual_norm runs on the CUDA engine only (no CPU path); got {x.device}")
    dtype = x.dtype
    if dtype not in _NORM_TYPES:
        raise TypeError(f"x must be float32, bfloat16 or float16, got {dtype}")
    shape = x.shape
    if not shape or not 1 <= shape[-1] <= 8192:
        raise ValueError(f"residual_norm takes rows of 1 to 8192 values, got {tuple(shape)}")
    index = x.get_device()
    if y is None:
        if gamma is not None or gate is not None or post_weight is not None:
            raise ValueError("gamma, gate and post_weight scale y, which is None")
    elif y.shape != shape or y.dtype != dtype or y.get_device() != index:
        raise ValueError(f"y must match x: {tuple(y.shape)} {y.dtype} {y.device} vs "
                         f"{tuple(shape)} {dtype} {x.device}")
    if post_bias is not None and post_weight is None:
        raise ValueError("post_bias without post_weight")
    param_dtype, row = weight.dtype, shape[-1:]
    if param_dtype != dtype and param_dtype != torch.float32:
        raise TypeError(f"parameters must be {dtype} or float32, got {param_dtype}")
    for name, p in (("weight", weight), ("norm_bias", norm_bias), ("gamma", gamma),
                    ("post_weight", post_weight), ("post_bias", post_bias)):
        if p is not None and (p.shape != row or p.dtype != param_dtype or p.get_device() != index):
            raise ValueError(f"{name} must be {list(row)} of {param_dtype} on {x.device}, got "
                             f"{tuple(p.shape)} {p.dtype} {p.device}")
    if gate is not None and (len(shape) < 2 or gate.shape != (shape[0], shape[-1])
                             or gate.dtype != param_dtype or gate.get_device() != index):
        raise ValueError(f"gate must be [x.shape[0], {shape[-1]}] of {param_dtype} on {x.device}, "
                         f"got {tuple(gate.shape)} {gate.dtype} {gate.device}")


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _dense(t: Optional[torch.Tensor]):
    return t if t is None or t.is_contiguous() else t.detach().contiguous()


def _norm_launch(x, y, weight, norm_bias, gamma, gate, post_weight, post_bias, kind, eps,
                 stats=None, h=None, mx=None):
    """One ``scmp_residual_norm`` call on contiguous tensors; returns r (None without y)."""
    r = None if y is None else torch.empty_like(x)
    C = x.shape[-1]
    rows = x.numel() // C
    args = _lib.PACK_NORM.pack(
        _lib.ABI_VERSION, DTYPE[x.dtype], DTYPE[weight.dtype], kind == "rms", x.data_ptr(),
        _ptr(y), weight.data_ptr(), _ptr(norm_bias), _ptr(gamma), _ptr(gate), _ptr(post_weight),
        _ptr(post_bias), _ptr(r), _ptr(h), _ptr(stats), 0 if mx is None else mx.data_ptr,
        0 if mx is None else mx.scales_ptr, rows, C,
        0 if gate is None else rows // max(1, x.shape[0]), eps,
        h is not None and h.dtype == torch.float32,
        0 if mx is None else _lib.MX_FORMAT[mx.fmt], 0)
    call(_lib.load().scmp_residual_norm, x.get_device(), args)
    return r


@functools.lru_cache(maxsize=256)
def _norm_bwd_workspace(rows: int, C: int, rows_per_gate: int) -> int:
    """Bytes, a function of the sizes alone."""
    return _lib.load().scmp_residual_norm_bwd_workspace(rows, C, rows_per_gate)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, weight, norm_bias, gamma, gate, post_weight, post_bias, kind, eps):
        t = [_dense(v) for v in (x, y, weight, norm_bias, gamma, gate, post_weight, post_bias)]
        x = t[0]
        stats = torch.empty(x.numel() // x.shape[-1] * (2 if post_weight is None else 4),
                            dtype=torch.float32, device=x.device)
        h = torch.empty_like(x)
        r = _norm_launch(*t, kind, eps, stats, h)
        ctx.kind = kind
        ctx.save_for_backward(x if r is None else r, t[1], stats, *t[2:])
        ctx.set_materialize_grads(False)
        return h if r is None else (r, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        r, y, stats, weight, norm_bias, gamma, gate, post_weight, post_bias = ctx.saved_tensors
        dr, dh = grads if y is not None else (None, grads[0])
        leaves = (r, y, weight, norm_bias, gamma, gate, post_weight, post_bias)
        if r.numel() == 0 or (dr is None and dh is None):
            return tuple(torch.zeros_like(t) if w and t is not None else None
                         for w, t in zip(ctx.needs_input_grad, leaves)) + (None, None)
        dr, dh = _dense(dr), _dense(dh)
        out = [torch.empty_like(t) if w and t is not None else None
               for w, t in zip(ctx.needs_input_grad, leaves)]
        C = r.shape[-1]
        rows = r.numel() // C
        per_gate = rows if gate is None else rows // r.shape[0]
        lib = _lib.load()
        ws, size = None, 0
        if any(t is not None for t in out[2:]):
            size = _norm_bwd_workspace(rows, C, per_gate)
            ws = torch.empty(size, dtype=torch.uint8, device=r.device)
        args = _lib.PACK_NORM_BWD.pack(
            _lib.ABI_VERSION, DTYPE[r.dtype], DTYPE[weight.dtype], ctx.kind == "rms", r.data_ptr(),
            _ptr(y), _ptr(dr), _ptr(dh), weight.data_ptr(), _ptr(gamma), _ptr(gate),
            _ptr(post_weight), _ptr(post_bias), stats.data_ptr(), *[_ptr(t) for t in out], _ptr(ws),
            size, rows, C, per_gate)
        call(lib.scmp_residual_norm_bwd, r.get_device(), args)
        return (*out, None, None)


def residual_norm(x: torch.Tensor, y: Optional[torch.Tensor], weight: torch.Tensor,
                  norm_bias: Optional[torch.Tensor] = None, *, kind: str = "layer",
                  eps: float = 1e-6, gamma: Optional[torch.Tensor] = None,
                  gate: Optional[torch.Tensor] = None,
                  post_weight: Optional[torch.Tensor] = None,
                  post_bias: Optional[torch.Tensor] = None, quantize: Optional[str] = None):
    """A block's gated residual add with the norms around it, in one pass ->
    ``(r, h)``::

        z = y, or N(y) * post_weight + post_bias     the norm behind the branch
        r = x + z * gamma * gate                     rounded to x's type
        h = N(r) * weight + norm_bias                the norm in front of the next one

    ``N`` is a layer norm or, with ``kind="rms"``, a root-mean-square norm over
    the last dimension (at most 8192), statistics in fp32.  ``x``, ``y``
    ``[..., C]`` of one type (float32, bfloat16, float16); ``weight``,
    ``norm_bias``, ``gamma`` (layer scale), ``post_weight``, ``post_bias``
    ``[C]`` and ``gate`` ``[x.shape[0], C]`` (one per sample) of that type or
    float32, all optional but ``weight``.  ``y=None`` is the norm alone: ``r``
    is ``x``.

    Differentiable (once, backward) in every tensor.  ``quantize="mxfp4"`` or ``"nvfp4"``
    returns ``h`` as an ``MXTensor`` quantised from its fp32 values (nvfp4 with
    tensor scale 1) for ``mx_matmul``; that form has no gradient.  The sums
    differ from ``F.layer_norm``'s in their order, so the bits may too."""
    _check_norm(x, y, weight, norm_bias, kind, eps, gamma, gate, post_weight, post_bias)
    leaves = (x, y, weight, norm_bias, gamma, gate, post_weight, post_bias)
    if (torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in leaves])
            ) or has_tangent(leaves):
        # (a forward-mode tangent is refused there: the function has no jvp)
        if quantize is not None:
            raise RuntimeError("residual_norm with quantize has no gradient; call it under "
                               "torch.no_grad() or on detached inputs")
        out = _ResidualNorm.apply(*leaves, kind, eps)
        return (x, out) if y is None else out
    t = [_dense(v) for v in leaves]
    if quantize is None:
        h = torch.empty_like(t[0])
        r = _norm_launch(*t, kind, eps, None, h)
        return (x if r is None else r), h
    from . import mx as _mx
    _mx._check_fmt(quantize)
    if x.numel() == 0 or (x.shape[-1] * x.element_size() % 16 == 0 and not any(
            [v is not None and v.data_ptr() % 16 for v in t])):
        q = _mx.mx_empty(x.shape, quantize, x.device, x.dtype)
        r = _norm_launch(*t, kind, eps, None, None, q)
    else:  # odd rows: through h's fp32 values, the same codes in two launches
        h = torch.empty(x.shape, dtype=torch.float32, device=x.device)
        r = _norm_launch(*t, kind, eps, None, h)
        q = _mx.mx_quantize(h, quantize)
        q.dtype = x.dtype
    return (x if r is None else r), q


PER = ("element", "row", "sample")


def _dropout_launch(x, residual, p, seed, offset, state, span):
    """One ``scmp_dropout`` call on contiguous tensors."""
    y = torch.empty_like(x)
    args = _lib.PACK_DROPOUT.pack(_lib.ABI_VERSION, DTYPE[x.dtype], x.data_ptr(), _ptr(residual),
                                  y.data_ptr(), _ptr(state), x.numel(), span, seed, offset, p)
    call(_lib.load().scmp_dropout, x.get_device(), args)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, state, p, seed, offset, span):
        ctx.draw = (p, seed, offset)
        ctx.span = span
        ctx.save_for_backward(state)
        return _dropout_launch(_dense(x), _dense(residual), p, seed, offset, state, span)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (state,) = ctx.saved_tensors
        dx = None
        if ctx.needs_input_grad[0]:
            dx = _dropout_launch(_dense(dy), None, *ctx.draw, state, ctx.span)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None, None, None


def dropout(x: torch.Tensor, p: float, seed, offset: int = 0, *, per: str = "element",
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Dropout whose mask is never stored: ``x / (1 - p)`` where a draw is kept, 0
    where it is dropped (whatever x holds there), ``+ residual``, in one pass, rounded
    once.  ``per``: one draw per ``"element"``, per ``"row"`` (last dimension) or per
    ``"sample"`` (first dimension: stochastic depth).

    Draw ``d`` (counted in row-major order) is word ``d % 4`` of Philox4x32-10 under
    the 64-bit key ``seed`` at the counter ``(d // 4, offset)``, and is dropped if it is
    below ``round(p * 2^32)``: the same call draws the same mask, another ``offset``
    another one.  ``seed`` may be an int64 tensor ``[seed, more]`` on x's device, which
    the kernel reads (``more`` is added to ``offset``): a captured call then draws anew
    when the tensor changes between replays.

    ``x`` ``[..., C]`` and ``residual`` of one shape and type (float32, bfloat16,
    float16), CUDA.  Differentiable (once, backward) in both: the backward pass draws
    the mask again, so a seed tensor must still hold what it held."""
    if per not in PER:
        raise ValueError(f"unknown per {per!r} (one of {PER})")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be within 0 and 1, got {p!r}")
    if not x.is_cuda:
        raise RuntimeError(f"dropout runs on the CUDA engine only (no CPU path); got {x.device}")
    if x.dtype not in _NORM_TYPES:
        raise TypeError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    if not x.dim() and per != "element":
        raise ValueError("rows and samples are of tensors with dimensions")
    index = x.get_device()
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype
                                 or residual.get_device() != index):
        raise ValueError(f"residual must match x: {tuple(residual.shape)} {residual.dtype} "
                         f"{residual.device} vs {tuple(x.shape)} {x.dtype} {x.device}")
    state = None
    if isinstance(seed, torch.Tensor):
        if (seed.dtype != torch.int64 or seed.shape != (2,) or seed.get_device() != index
                or not seed.is_contiguous()):
            raise ValueError(f"a seed tensor is [seed, more], int64 and contiguous on {x.device}, "
                             f"got {seed.dtype} {tuple(seed.shape)} {seed.device}")
        state, seed = seed, 0
    seed, offset = int(seed), int(offset)
    if not (-1 << 63 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
        raise ValueError(f"seed and offset are 64-bit, got {seed} and {offset}")
    n = x.numel()
    span = 1
    if per != "element" and n:
        span = x.shape[-1] if per == "row" else n // x.shape[0]
    seed &= (1 << 64) - 1
    if (torch.is_grad_enabled() and (x.requires_grad or (
            residual is not None and residual.requires_grad))) or has_tangent((x, residual)):
        # (a forward-mode tangent is refused there: the function has no jvp)
        return _Dropout.apply(x, residual, state, float(p), seed, offset, span)
    return _dropout_launch(_dense(x), _dense(residual), float(p), seed, offset, state, span)


class _Calls:
    """Numbers of a module's calls, each given out once: to its threads, and to its
    data-parallel replicas, which are copies made for one call and hold this same object
    (a sequence for each of their devices, so that what one draws does not depend on when
    the others run)."""

    def __init__(self, start: int = 0):
        self.start, self.taken, self.lock = start, {}, threading.Lock()

    def take(self, device: Optional[int] = None) -> int:
        with self.lock:
            n = self.taken.get(device, self.start)
            self.taken[device] = n + 1
        return n if device is None else (device + 1 << 40) + n

    def most(self) -> int:
        with self.lock:
            return max(self.taken.values(), default=self.start)

    def __reduce__(self):  # (copies count for themselves)
        return _Calls, (self.most(),)


class Dropout(nn.Module):
    """``dropout`` in a model: in training every call takes the next mask, in
    evaluation it passes through.  ``index`` tells the modules of a model apart, which
    may then share ``seed``; ranks that are to draw apart take seeds of their own.
    ``calls`` counts (and, set, repeats) the eager masks, over threads (who takes which is
    theirs to order) and data-parallel replicas (whose devices draw masks of their own);
    calls that a graph captures count on the device, so that every replay draws masks of
    its own (replays that share a module follow one another, as they do for its weights'
    sake).  Both counts go with a state dict, in its metadata (its keys are those of a
    model without dropout, so that either loads the other's), and a run that loads it draws
    on where the saved one stopped.  A call made
    while a backward pass runs (a checkpoint's recomputation) would take the next mask
    instead of the one to be repeated, and raises: ``dropout`` with an offset of the
    caller's own repeats it."""

    def __init__(self, p: float, *, per: str = "element", seed: int = 0, index: int = 0):
        super().__init__()
        if per not in PER:
            raise ValueError(f"unknown per {per!r} (one of {PER})")
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p must be within 0 and 1, got {p!r}")
        if not 0 <= index < 1 << 16:
            raise ValueError(f"index must be within 0 and 65535, got {index}")
        seed = int(seed)
        if not -1 << 63 <= seed < 1 << 64:
            raise ValueError(f"seed is 64-bit, got {seed}")
        self.p, self.per, self.index, self._calls = float(p), per, index, _Calls()
        self._captured = False  # whether a graph has captured a call
        self.seed = seed - (1 << 64) if seed >= 1 << 63 else seed  # (as int64 holds it)
        # (no buffer: wrappers that broadcast buffers would give every rank the first one's seed)
        self.state = torch.tensor([self.seed, 0])

    def _apply(self, fn, *args, **kwargs):
        super()._apply(fn, *args, **kwargs)
        device = fn(self.state).device  # (its values stay, where fn only allocates too)
        if device != self.state.device:
            state = torch.tensor([self.seed, 0], device="cpu") if self.state.is_meta else self.state
            self.state = state.to(device)
        return self

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        metadata = getattr(destination, "_metadata", None)
        if metadata is not None:
            counts = metadata.setdefault(prefix[:-1], {})
            counts["calls"] = self.calls
            if self._captured:  # (read back from the device)
                counts["captured"] = int(self.state[1])

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, *args):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, *args)
        if "calls" in local_metadata:
            self.calls = local_metadata["calls"]
        if "captured" in local_metadata:
            self._captured = True
            self.state[1:].fill_(local_metadata["captured"])

    def __setstate__(self, state):
        super().__setstate__(state)
        self.__dict__.setdefault("_captured", True)
        if "state" in self._buffers:
            state = self._buffers.pop("state")
            self._non_persistent_buffers_set.discard("state")
            self.state = state
        if "_calls" not in self.__dict__:  # (saved whole by an earlier version)
            self._calls = _Calls(self.__dict__.pop("calls", 0))

    @property
    def active(self) -> bool:
        return self.training and self.p > 0

    @property
    def calls(self) -> int:
        return self._calls.most()

    @calls.setter
    def calls(self, n: int) -> None:
        self._calls = _Calls(int(n))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if not self.active:
            return x if residual is None else residual + x
        inside = in_backward()
        if inside is None:
            raise RuntimeError("this torch does not tell whether a backward pass runs, in which a "
                               "Dropout module must not take the next mask; use dropout() with "
                               "an offset of your own")
        if inside:
            raise RuntimeError("a Dropout module called inside a backward pass (by an activation "
                               "checkpoint?) cannot repeat the mask of its first call; use "
                               "dropout() with an offset of your own there")
        at = self.index << 48  # (its calls below 2^40, replicas' and, from 2^47, captured ones above)
        if x.is_cuda and torch.cuda.is_current_stream_capturing():
            self._captured = True
            state = self.state.clone()
            self.state[1:] += 1
            return dropout(x, self.p, state, at + (1 << 47), per=self.per, residual=residual)
        replica = getattr(self, "_is_replica", False)
        offset = at + self._calls.take(x.get_device() if replica else None)
        return dropout(x, self.p, self.seed, offset, per=self.per, residual=residual)

    def extra_repr(self) -> str:
        return f"p={self.p}, per={self.per!r}, seed={self.seed}, index={self.index}"


def _active(m: Optional[nn.Module]) -> bool:
    """Whether a module drops anything in this call."""
    return m is not None and (type(m) is not Dropout or m.active) and type(m) is not nn.Identity


def _plain_linear(m: nn.Module) -> bool:
    return (type(m) is nn.Linear and m.bias is not None and m.weight.dtype == torch.float32
            and m.weight.is_contiguous() and m.bias.is_contiguous())


class Mlp(nn.Module):
    def __init__(self, dim: int, hidden: int):
        super().__init__()
        self.fc1 = nn.Linear(dim, hidden)
        self.act = nn.GELU()
        self.fc2 = nn.Linear(hidden, dim)
        self.drop = nn.Identity()

    def forward(self, x):
        y = _fp_linear(self.fc2, self.act(_fp_linear(self.fc1, x)))
        drop = getattr(self, "drop", None)  # (a module saved whole by an earlier version has none)
        return y if drop is None else drop(y)


class Attention(nn.Module):
    def __init__(self, dim: int, num_heads: int):
        super().__init__()
        self.num_heads = num_heads
        self.scale = (dim // num_heads) ** -0.5
        self.qkv = nn.Linear(dim, 3 * dim)
        self.proj = nn.Linear(dim, dim)
        self.attn_drop = nn.Identity()
        self.proj_drop = nn.Identity()
        self.rope: Optional[GridRotary] = None  # positions of q and k, if the model has them
        self.qk_norm: Optional[QKNorm] = None   # and their norms

    def forward(self, x, attn_bias=None):
        B, N, C = x.shape
        H = self.num_heads
        # (a module saved whole by an earlier version has neither)
        rope, qk_norm = getattr(self, "rope", None), getattr(self, "qk_norm", None)
        if qk_norm is not None:
            q, k, v = qk_norm.split(self.qkv(x), H, rope, transpose_v=False)
        elif rope is not None:
            q, k, v = rope.split(self.qkv(x), H, transpose_v=False)
        else:
            qkv = self.qkv(x).reshape(B, N, 3, H, C // H).permute(2, 0, 3, 1, 4)
            q, k, v = qkv.unbind(0)
        out = F.scaled_dot_product_attention(q, k, v)
        return self.proj_drop(self.proj(out.transpose(1, 2).reshape(B, N, C)))


class LayerScale(nn.Module):
    def __init__(self, dim: int, init: float):
        super().__init__()
        self.gamma = nn.Parameter(torch.full((dim,), float(init)))

    def forward(self, x):
        return x * self.gamma


class Block(nn.Module):
    def __init__(self, dim: int, heads: int, hidden: int, ls_init: float):
        super().__init__()
        self.norm1 = nn.LayerNorm(dim, eps=1e-6)
        self.attn = Attention(dim, heads)
        self.ls1 = LayerScale(dim, ls_init)
        self.norm2 = nn.LayerNorm(dim, eps=1e-6)
        self.mlp = Mlp(dim, hidden)
        self.ls2 = LayerScale(dim, ls_init)
        self.comp: Optional[nn.Module] = None  # head-aligned compensation, if installed
        self.drop_path: Optional[Dropout] = None  # stochastic depth, if the model has it
        self.block_idx = 0

    def forward(self, x):
        set_current_block_idx(self.block_idx)
        if self._fused_norm_applies(x):
            return self._forward_fused_norm(x)
        if self._fused_glue_applies(x):
            return self._forward_fused_glue(x)
        y = self._add(x, self.ls1(self.attn(self.norm1(x))))
        y = self._add(y, self.ls2(self.mlp(self.norm2(y))))
        if self.comp is not None:
            y = y + self.comp(x).to(y.dtype)
        return y

    def _add(self, x: torch.Tensor, branch: torch.Tensor) -> torch.Tensor:
        """The residual add, with stochastic depth in the same pass where types allow."""
        drop = getattr(self, "drop_path", None)
        if not _active(drop):
            return x + branch
        if x.dtype == branch.dtype and type(drop) is Dropout:
            return drop(branch, x)
        return x + drop(branch)

    def _fused_norm_applies(self, x: torch.Tensor) -> bool:
        qkv, fc1 = getattr(self.attn, "qkv", None), getattr(self.mlp, "fc1", None)
        if not (FUSED_NORM or type(qkv) is MXLinear or type(fc1) is MXLinear):
            return False
        norms = (self.norm1, self.norm2)
        # (autocast keeps a 16-bit x's norms and residual in fp32, which r would not)
        return (x.is_cuda and x.dtype in _NORM_TYPES and x.shape[-1] <= 8192
                and (x.dtype == torch.float32 or not torch.is_autocast_enabled("cuda"))
                and type(self.ls1) is LayerScale
                and all(type(n) is nn.LayerNorm and n.weight is not None and n.bias is not None
                        and n.weight.dtype in (x.dtype, torch.float32) for n in norms)
                and self.ls1.gamma.dtype == self.norm2.weight.dtype
                and not in_dual_level() and not _watched(*norms, self.ls1))

    def _forward_fused_norm(self, x):
        """The forward above with each norm in the pass of the residual add in
        front of it; a norm whose reader is a 4-bit linear writes codes only
        (``attn`` or ``mlp`` then get an ``MXTensor``)."""
        def norm(n, owner, name, y=None, gamma=None):
            # (the reader of a patched block that is not a 4-bit linear, one whose
            # input a hook sees, or any reader while gradients are recorded, takes
            # values)
            reader = getattr(owner, name, None)
            fmt = reader.fmt if (type(reader) is MXLinear and not torch.is_grad_enabled()
                                 and not _watched(owner, reader)) else None
            return residual_norm(x, y, n.weight, n.bias, eps=n.eps, gamma=gamma, quantize=fmt)

        drop = getattr(self, "drop_path", None)
        _, h = norm(self.norm1, self.attn, "qkv")
        a = self.attn(h)
        if _active(drop):  # (a sample's draw and the layer scale commute)
            a = drop(a)
        if torch.promote_types(a.dtype, x.dtype) == x.dtype:
            # (under autocast the branch comes in 16 bits: as wide as the sum it joins)
            y, h = norm(self.norm2, self.mlp, "fc1", a.to(x.dtype), self.ls1.gamma)
        else:
            y = x + self.ls1(a)
            h = self.norm2(y)
        u = self.mlp(h)
        e = None if self.comp is None else self.comp(x).to(y.dtype)
        if _active(drop):
            y = self._add(y, self.ls2(u))
            return y if e is None else y + e
        if self._fused_glue_applies(y) and u.dtype == torch.float32:
            return scale_residual(y, u.contiguous(), self.ls2.gamma, out=y,
                                  extra=None if e is None else e.contiguous())
        y = y + self.ls2(u)
        return y if e is None else y + e

    def _fused_glue_applies(self, x: torch.Tensor) -> bool:
        return (FUSED_GLUE and x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()
                and not torch.is_grad_enabled() and not torch.is_autocast_enabled("cuda")
                and not in_dual_level() and not _active(getattr(self, "drop_path", None))
                and all(type(ls) is LayerScale and ls.gamma.dtype == torch.float32
                        for ls in (self.ls1, self.ls2)))

    def _forward_fused_glue(self, x: torch.Tensor) -> torch.Tensor:
        """The forward above with its fp32 elementwise steps on the engine:
        ``x + ls1(a)`` in one pass, fc1's bias with the GELU, fc2's bias with
        ``ls2``, the residual add and the compensation term in another (the
        matmuls stay cuBLAS fp32).  Bit-identical to the unfused forward.  A
        branch in another type is added as there."""
        a = self.attn(self.norm1(x))
        if a.dtype == torch.float32:
            y = scale_residual(x, a.contiguous(), self.ls1.gamma)
        else:
            y = x + self.ls1(a)
        h = self.norm2(y)
        mlp = self.mlp
        ub = None
        if (type(mlp) is Mlp and _plain_linear(mlp.fc1) and _plain_linear(mlp.fc2)
                and type(mlp.act) is nn.GELU and mlp.act.approximate == "none"
                and not _active(getattr(mlp, "drop", None))):
            h2 = h.reshape(-1, h.shape[-1])
            t = bias_gelu_(torch.mm(h2, mlp.fc1.weight.t()), mlp.fc1.bias)
            u = torch.mm(t, mlp.fc2.weight.t())
            ub = mlp.fc2.bias
        else:
            u = mlp(h)
            if u.dtype != torch.float32:
                y = y + self.ls2(u)
                return y if self.comp is None else y + self.comp(x).to(y.dtype)
        e = None
        if self.comp is not None:
            e = self.comp(x).to(torch.float32).contiguous()
        return scale_residual(y, u.reshape(y.shape).contiguous(), self.ls2.gamma, bias=ub,
                              extra=e, out=y)


class Backbone(nn.Module):
    def __init__(self, img: int = 224, patch: int = 14, dim: int = 1024, depth: int = 24,
                 heads: int = 16, hidden: int = 4096, ls_init: float = 1.0, rope: bool = False,
                 rope_base: float = 10000.0, qk_norm: Optional[str] = None):
        super().__init__()
        self.patch_embed = nn.Conv2d(3, dim, kernel_size=patch, stride=patch)
        n = (img // patch) ** 2
        self.cls_token = nn.Parameter(torch.zeros(1, 1, dim))
        self.pos_embed = nn.Parameter(torch.zeros(1, n + 1, dim))
        self.blocks = nn.ModuleList([Block(dim, heads, hidden, ls_init) for _ in range(depth)])
        for i, b in enumerate(self.blocks):
            b.block_idx = i
        if rope:
            grid = GridRotary((img // patch, img // patch), dim // heads, base=rope_base)
            for b in self.blocks:
                b.attn.rope = grid
        if qk_norm is not None:  # "rms" or "layer"
            for b in self.blocks:
                b.attn.qk_norm = QKNorm(dim // heads, qk_norm)
        self.norm = nn.LayerNorm(dim, eps=1e-6)

    def forward(self, x):
        x = self.patch_embed(x).flatten(2).transpose(1, 2)
        x = torch.cat([self.cls_token.expand(x.shape[0], -1, -1), x], dim=1) + self.pos_embed
        for b in self.blocks:
            x = b(x)
        return self.norm(x)


class ViTClassifier(nn.Module):
    """ViT-L/14 backbone + linear head on [CLS, mean(patch)] (2048 -> 1000)."""

    def __init__(self, num_classes: int = 1000, **kw):
        super().__init__()
        self.backbone = Backbone(**kw)
        dim = self.backbone.norm.normalized_shape[0]
        self.linear_head = nn.Linear(2 * dim, num_classes)

    def forward(self, x):
        t = self.backbone(x)
        feat = torch.cat([t[:, 0], t[:, 1:].mean(dim=1)], dim=-1)
        return self.linear_head(feat)


def vit_l14(seed: int = 0, num_classes: int = 1000, **kw) -> ViTClassifier:
    """Random-initialised DINOv2-style ViT-L/14 (24 blocks, d=1024, 16 heads,
    MLP 4096, 257 tokens at 224x224)."""
    g = torch.Generator().manual_seed(seed)
    m = ViTClassifier(num_classes=num_classes, **kw)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if name.endswith("gamma"):
                continue
            if p.dim() >= 2:
                p.copy_(torch.nn.init.trunc_normal_(torch.empty_like(p), std=0.02, generator=g))
            elif "norm" in name and name.endswith("weight"):
                p.fill_(1.0)
            else:
                p.zero_()
        m.backbone.pos_embed.copy_(torch.randn(m.backbone.pos_embed.shape, generator=g) * 0.02)
        m.backbone.cls_token.copy_(torch.randn(m.backbone.cls_token.shape, generator=g) * 0.02)
    return m.eval()


class _RowMPLinear(nn.Module):
    """SC linear whose rows carry a seeded random level in each call."""

    def __init__(self, linear: nn.Linear, cfg: SeededRandomMPConfig, salt: int,
                 cfg_for: Callable[[int, int], dict]):
        super().__init__()
        self.weight = linear.weight
        self.bias = linear.bias
        self.cfg = cfg
        self.salt = salt
        self.cfg_for = cfg_for
        self.calls = 0
        self.packed = PackedWeights(self.weight, "bipolar")  # one per precision class

    def forward(self, x):
        shp = x.shape
        x2 = x.reshape(-1, shp[-1])
        if x2.dtype not in (torch.float32, torch.bfloat16):
            x2 = x2.float()
        row_L = self.cfg.assign(x2.shape[0], x2.device, salt=(self.salt << 16) + self.calls)
        self.calls += 1
        counts = quantile_counts(x2.shape[0], self.cfg.stoc_len_levels, self.cfg.level_fractions)
        y = sc_linear_rows(x2, self.weight, row_L, self.cfg.stoc_len_levels, "bipolar",
                           bias=self.bias, cfg_for=self.cfg_for, host_counts=counts,
                           packed_for=self.packed)
        return y.to(x.dtype).reshape(*shp[:-1], -1)


def patch_vit(model: ViTClassifier, sc_prec: int, ops: Iterable[str] = ("qk", "av", "proj"), *,
              av_mode: str = "bipolar", attn_mp_spec: Optional[Dict] = None,
              linear_random_mp: Optional[SeededRandomMPConfig] = None,
              linear_ops: Iterable[str] = ("qkv_proj", "out_proj"),
              block_cfg_for: Optional[Callable[[int], Callable[[int, int], dict]]] = None,
              comp_blocks: Iterable[int] = (), comp_sc_prec: Optional[int] = None,
              comp_seed: int = 1) -> dict:
    """Install SC operators on every block (see module docstring).

    ``ops`` uses the reference's op names (``cls/sc_attention_patch.py:332``,
    with ``"proj"`` meaning qkv_proj + out_proj).  ``block_cfg_for(i)`` gives
    block ``i`` its own pool factory ``(D, p) -> config``.  ``comp_blocks``
    get a ``HeadAlignedSCLinear`` compensation (random weights) that reuses the
    block's ``(head_dim, p)`` pool.
    """
    ops = set(ops)
    stats = {"attn": 0, "qkv_proj": 0, "out_proj": 0, "mlp_fc1": 0, "mlp_fc2": 0, "comp": 0}
    attn_mp_spec = attn_mp_spec or {}
    linear_ops = set(linear_ops)
    if "proj" in ops:
        ops |= {"qkv_proj", "out_proj"}
    comp_blocks = set(comp_blocks)
    g = torch.Generator().manual_seed(comp_seed)
    for i, blk in enumerate(model.backbone.blocks):
        cfg_for = block_cfg_for(i) if block_cfg_for is not None else _get_config
        attn = blk.attn
        if "qk" in ops or "av" in ops:
            fwd = make_sc_attention_forward(
                sc_prec, sc_av="av" in ops, sc_qk="qk" in ops,
                qk_mp_cfg=attn_mp_spec.get("qk"), av_mp_cfg=attn_mp_spec.get("av"),
                av_mode=av_mode, cfg_for=cfg_for)
            attn.forward = fwd.__get__(attn, type(attn))
            stats["attn"] += 1

        def wrap(lin: nn.Linear, op: str, salt: int):
            if linear_random_mp is not None and op in linear_ops:
                return _RowMPLinear(lin, linear_random_mp, salt, cfg_for)
            cfg = None if block_cfg_for is None else cfg_for(lin.in_features, sc_prec)
            return SCLinear(lin, sc_prec, mode="bipolar", cfg_override=cfg, operator=op)

        if "qkv_proj" in ops:
            attn.qkv = wrap(attn.qkv, "qkv_proj", 4 * i)
            stats["qkv_proj"] += 1
        if "out_proj" in ops:
            attn.proj = wrap(attn.proj, "out_proj", 4 * i + 1)
            stats["out_proj"] += 1
        if "mlp_fc1" in ops:
            blk.mlp.fc1 = wrap(blk.mlp.fc1, "mlp_fc1", 4 * i + 2)
            stats["mlp_fc1"] += 1
        if "mlp_fc2" in ops:
            blk.mlp.fc2 = wrap(blk.mlp.fc2, "mlp_fc2", 4 * i + 3)
            stats["mlp_fc2"] += 1
        if i in comp_blocks:
            dim = attn.proj.weight.shape[0] if hasattr(attn.proj, "weight") else 1024
            lin = nn.Linear(dim, dim).to(next(model.parameters()).device)
            with torch.no_grad():
                lin.weight.copy_(torch.randn(dim, dim, generator=g) * 0.002)
                lin.bias.zero_()
            head_dim = dim // attn.num_heads
            p = comp_sc_prec or sc_prec
            blk.comp = HeadAlignedSCLinear(lin, p, n_heads=attn.num_heads,
                                           cfg_override=cfg_for(head_dim, p))
            stats["comp"] += 1
    return stats


MX_OPS = ("qkv_proj", "out_proj", "mlp_fc1", "mlp_fc2")
_WHERE = {"qkv_proj": ("attn", "qkv"), "out_proj": ("attn", "proj"), "mlp_fc1": ("mlp", "fc1"),
          "mlp_fc2": ("mlp", "fc2")}


def _patch_linears(model: ViTClassifier, ops: Iterable[str], make: Callable) -> dict:
    ops = set(ops)
    unknown = ops - set(MX_OPS)
    if unknown:
        raise ValueError(f"unknown ops {sorted(unknown)} (of {MX_OPS})")
    stats = {op: 0 for op in MX_OPS}
    for blk in model.backbone.blocks:
        for op in ops:
            owner = getattr(blk, _WHERE[op][0])
            setattr(owner, _WHERE[op][1], make(getattr(owner, _WHERE[op][1])))
            stats[op] += 1
    return stats


def patch_vit_mx(model: ViTClassifier, ops: Iterable[str] = MX_OPS, *,
                 fmt: str = "mxfp4") -> dict:
    """Put the named linears of every block (the op names of ``patch_vit``) in
    microscaled 4 bits: ``mx.MXLinear`` from the present weights, which must be
    on the GPU.  The norms in front of qkv_proj and mlp_fc1 then write their
    codes, except where a hook watches the norm or the module that reads them.
    Inference only."""
    return _patch_linears(model, ops, lambda lin: MXLinear(lin, fmt))


def patch_vit_fp8(model: ViTClassifier, ops: Iterable[str] = MX_OPS, *,
                  train: bool = False) -> dict:
    """Put the named linears of every block (the op names of ``patch_vit``) in 8
    bits: ``fp8.FP8Linear`` from the present weights, which must be on the GPU, or
    with ``train`` on the present parameters, which stay trainable."""
    return _patch_linears(model, ops, lambda lin: FP8Linear(lin, train))


def set_dropout(model: ViTClassifier, p: float = 0.0, drop_path=0.0, *, seed: int = 0) -> None:
    """Dropout with probability ``p`` behind every block's projection and MLP, and
    stochastic depth with probability ``drop_path`` (one number, or one per block) of
    each branch, from one ``seed``; active in training mode.  0 takes them out."""
    blocks = model.backbone.blocks
    rates = [float(drop_path)] * len(blocks) if isinstance(drop_path, (int, float)) else [
        float(r) for r in drop_path]
    if len(rates) != len(blocks):
        raise ValueError(f"{len(rates)} drop_path rates for {len(blocks)} blocks")
    for i, (blk, rate) in enumerate(zip(blocks, rates)):
        made = [Dropout(q, per=per, seed=seed, index=3 * i + j).to(blk.ls1.gamma.device).train(
            blk.training) if q else None
                for j, (q, per) in enumerate(((p, "element"), (p, "element"), (rate, "sample")))]
        blk.attn.proj_drop = made[0] or nn.Identity()
        blk.mlp.drop = made[1] or nn.Identity()
        blk.drop_path = made[2]
