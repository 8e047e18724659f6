"""``vit.residual_norm`` against its definition in 64 bits: values, gradients
(formula and differences), 4-bit output and refusals.

Tolerances carry magnitudes through the formulas: a fp32 sum of C terms is off
by at most (C + 8) 2^-24 of the sum of their magnitudes, whatever its order,
and a value rounded to its type by half a step of it."""
import ctypes
import pathlib
import subprocess
import sys
import threading

import pytest
import torch

from scmp_vit_b200 import _lib, mx, vit

U = 2.0 ** -24
EPS = 1e-6
DTYPES = (torch.float32, torch.bfloat16, torch.float16)
NAMES = ("x", "y", "weight", "norm_bias", "gamma", "gate", "post_weight", "post_bias")


def make(shape, dtype, dev, *, kind="layer", bias=True, gamma=True, gate=False, post=False,
         branch=True, param_dtype=None, grad=False, seed=0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    C = shape[-1]
    pd = param_dtype or dtype

    def t(*s, scale=1.0, shift=0.0, d=pd):
        return (torch.randn(*s, generator=g) * scale + shift).to(d).to(dev).requires_grad_(grad)

    return dict(
        x=t(*shape, scale=2.0, shift=0.5, d=dtype),
        y=t(*shape, scale=0.7, shift=-0.2, d=dtype) if branch else None,
        weight=t(C, scale=0.3, shift=1.0),
        norm_bias=t(C, scale=0.2) if bias else None,
        gamma=t(C, scale=0.5, shift=0.5) if gamma and branch else None,
        gate=t(shape[0], C) if gate and branch else None,
        post_weight=t(C, scale=0.3, shift=1.0) if post and branch else None,
        post_bias=t(C, scale=0.2) if post and bias and branch else None), kind


def call(t, kind, **kw):
    return vit.residual_norm(t["x"], t["y"], t["weight"], t["norm_bias"], kind=kind, eps=EPS,
                             gamma=t["gamma"], gate=t["gate"], post_weight=t["post_weight"],
                             post_bias=t["post_bias"], **kw)


def norm64(v, kind):
    """N(v), 1 / deviation and the magnitude that N(v)'s error scales with."""
    mean = v.mean(-1, keepdim=True) if kind == "layer" else 0.0
    rstd = (((v - mean) ** 2).mean(-1, keepdim=True) + EPS) ** -0.5
    n = (v - mean) * rstd
    return n, rstd, n.abs() + v.abs().mean(-1, keepdim=True) * rstd


def forward64(t, kind, r_given=None):
    """Everything the bounds need; the norm in front sees ``r_given`` (the
    rounded residual that the call returned)."""
    d = {k: None if v is None else v.detach().double() for k, v in t.items()}
    f = {}
    if d["y"] is not None:
        z = d["y"]
        f["Z"] = z.abs()
        if d["post_weight"] is not None:
            f["m"], f["rstd_y"], f["M"] = norm64(d["y"], kind)
            z = f["m"] * d["post_weight"]
            f["Z"] = f["M"] * d["post_weight"].abs()
            if d["post_bias"] is not None:
                z, f["Z"] = z + d["post_bias"], f["Z"] + d["post_bias"].abs()
        s = torch.ones((), dtype=torch.float64, device=z.device)
        if d["gamma"] is not None:
            s = s * d["gamma"]
        if d["gate"] is not None:
            s = s * d["gate"].reshape(z.shape[0], *[1] * (z.dim() - 2), -1)
        f["z"], f["s"] = z, s
        f["r"] = d["x"] + z * s
        f["R"] = d["x"].abs() + f["Z"] * s.abs()
    else:
        f["r"], f["R"] = d["x"], d["x"].abs()
    r = f["r"] if r_given is None else r_given.detach().double()
    f["n"], f["rstd"], f["Nm"] = norm64(r, kind)
    f["h"] = f["n"] * d["weight"]
    f["H"] = f["Nm"] * d["weight"].abs()
    if d["norm_bias"] is not None:
        f["h"], f["H"] = f["h"] + d["norm_bias"], f["H"] + d["norm_bias"].abs()
    return d, f


def close(got, ref, bound, what):
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny if got.dtype == torch.float16 else 0.0
    err = (got.detach().double() - ref).abs()
    allow = bound + half * ref.abs() * (1 + 1e-3) + tiny * half * 2 + 1e-30
    assert bool((err <= allow).all()), (what, (err / allow).max().item())


# ------------------------------------------------------------ CPU: refusals

def norm_args(**kw):
    a = _lib.NormArgs()
    a.abi_version = _lib.ABI_VERSION
    a.rows, a.C, a.rows_per_gate, a.eps = 4, 8, 2, 1e-6
    a.x = a.weight = a.h = 16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code,msg", [
    (dict(abi_version=3), -1, "abi_version"),
    (dict(dtype=3), -1, "dtype"),
    (dict(param_dtype=2), -1, "dtype"),
    (dict(rows=-1), -1, "shape"),
    (dict(C=0), -1, "shape"),
    (dict(C=8193), -4, "8192"),
    (dict(eps=-1.0), -1, "eps"),
    (dict(eps=float("nan")), -1, "eps"),
    (dict(x=None), -1, "non-NULL"),
    (dict(weight=None), -1, "non-NULL"),
    (dict(h=None), -1, "non-NULL"),
    (dict(y=16), -1, "non-NULL"),
    (dict(gamma=16), -1, "y, which is NULL"),
    (dict(y=16, r=16, post_bias=16), -1, "post_bias"),
    (dict(y=16, r=16, gate=16, rows_per_gate=3), -1, "rows_per_gate"),
    (dict(y=16, r=16, gate=16, rows_per_gate=0), -1, "rows_per_gate"),
    (dict(mx_data=16), -1, "together"),
    (dict(mx_data=16, mx_scales=16, mx_fmt=2), -1, "format"),
    (dict(mx_data=16, mx_scales=16, C=7), -4, "16-byte"),
    (dict(mx_data=16, mx_scales=16, x=20), -4, "16-byte"),
    (dict(x=18), -1, "aligned to its elements"),
    (dict(dtype=1, weight=17, param_dtype=1), -1, "aligned to its elements"),
    (dict(dtype=1, h=18, h_f32=1), -1, "aligned to its elements"),
])
def test_forward_refusals(kw, code, msg):
    assert _lib.load().scmp_residual_norm(ctypes.byref(norm_args(**kw)), None) == code
    assert msg in _lib.last_error()


@pytest.mark.parametrize("kw,code,msg", [
    (dict(abi_version=3), -1, "abi_version"),
    (dict(dtype=4), -1, "dtype"),
    (dict(rows=0), -1, "shape"),
    (dict(C=9000), -4, "8192"),
    (dict(stats=None), -1, "non-NULL"),
    (dict(dy=16), -1, "y, which is NULL"),
    (dict(dpost_weight=16), -1, "post_bias"),
    (dict(y=16, dgate=16), -1, "dgate"),
    (dict(y=16, gate=16, rows_per_gate=3), -1, "rows_per_gate"),
    (dict(dweight=16), -3, "workspace"),
    (dict(dweight=16, workspace=16, workspace_bytes=4), -3, "workspace"),
    (dict(dx=18), -1, "aligned to its elements"),
    (dict(dbias=18), -1, "aligned to its elements"),
])
def test_backward_refusals(kw, code, msg):
    a = _lib.NormBwdArgs()
    a.abi_version = _lib.ABI_VERSION
    a.rows, a.C, a.rows_per_gate = 4, 8, 4
    a.r = a.weight = a.stats = a.dx = 16
    for k, v in kw.items():
        setattr(a, k, v)
    assert _lib.load().scmp_residual_norm_bwd(ctypes.byref(a), None) == code
    assert msg in _lib.last_error()


def test_workspace_sizes():
    size = _lib.load().scmp_residual_norm_bwd_workspace
    assert size(0, 8, 1) == 0 and size(4, 0, 1) == 0 and size(4, 8, 3) == 0
    assert size(4, 8, 4) >= 4 * 8 * 4
    assert size(6, 8, 2) >= 3 * 4 * 8 * 4


def test_python_refusals_on_cpu():
    x, w = torch.zeros(2, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        vit.residual_norm(x, x, w)
    with pytest.raises(ValueError, match="kind"):
        vit.residual_norm(x, x, w, kind="batch")


@pytest.mark.gpu
def test_python_refusals(cuda_device):
    x, w = torch.zeros(2, 3, 8, device=cuda_device), torch.ones(8, device=cuda_device)
    for kw, msg in ((dict(y=x[:1]), "y must match"), (dict(y=x.half()), "y must match"),
                    (dict(y=None, gamma=w), "y, which is None"),
                    (dict(y=x, post_bias=w), "post_bias"),
                    (dict(y=x, gamma=w[:4]), "gamma must"),
                    (dict(y=x, gamma=w.half()), "gamma must"),
                    (dict(y=x, gate=w), "gate must"),
                    (dict(y=x, eps=-1), "eps"),
                    (dict(y=x, quantize="fp4"), "format")):
        with pytest.raises(ValueError, match=msg):
            vit.residual_norm(x, kw.pop("y"), w, **kw)
    with pytest.raises(TypeError, match="parameters"):
        vit.residual_norm(x, x, w.half())
    with pytest.raises(TypeError, match="x must"):
        vit.residual_norm(x.double(), None, w)
    with pytest.raises(ValueError, match="8192"):
        vit.residual_norm(torch.zeros(2, 8200, device=cuda_device), None,
                          torch.ones(8200, device=cuda_device))
    with pytest.raises(RuntimeError, match="no gradient"):
        vit.residual_norm(x.clone().requires_grad_(), x, w, quantize="mxfp4")


# ------------------------------------------------------------- GPU: values

FORMS = [dict(), dict(bias=False, kind="rms"), dict(gamma=False, gate=True),
         dict(gate=True, post=True), dict(post=True, kind="rms", gate=True),
         dict(post=True, kind="rms", bias=False), dict(branch=False),
         dict(branch=False, kind="rms")]
SIZES = [(1, 1, 1), (1, 1, 8), (2, 3, 7), (3, 5, 64), (2, 37, 96), (1, 257, 1024), (4, 9, 1408),
         (2, 3, 1025), (2, 5, 4096), (1, 3, 8192), (3, 1, 33), (5, 70, 260)]


@pytest.mark.gpu
@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("shape", SIZES)
def test_forward(cuda_device, shape, form):
    for i, dtype in enumerate(DTYPES):
        t, kind = make(shape, dtype, cuda_device, **FORMS[form])
        r, h = call(t, kind)
        torch.cuda.synchronize()
        check_forward(t, kind, r, h)


def check_forward(t, kind, r, h):
    C = t["x"].shape[-1]
    _, f = forward64(t, kind, r)
    if t["y"] is None:
        assert r is t["x"]
    else:
        close(r, f["r"], (C + 16) * U * f["R"], "r")
    close(h, f["h"], (C + 16) * U * f["H"], "h")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(2, 37, 96), (2, 3, 7)])
def test_forward_fp32_parameters(cuda_device, dtype, shape):
    t, kind = make(shape, dtype, cuda_device, gate=True, post=True, param_dtype=torch.float32)
    r, h = call(t, kind)
    check_forward(t, kind, r, h)


@pytest.mark.gpu
def test_forward_strides_streams_graph(cuda_device):
    t, kind = make((3, 10, 64), torch.bfloat16, cuda_device, gate=True)
    base = torch.randn(10, 3, 128, device=cuda_device).bfloat16()
    t["x"] = base[:, :, 1:65].transpose(0, 1)       # strided and off alignment
    r, h = call(t, kind)
    check_forward(t, kind, r, h)
    off = torch.randn(3 * 10 * 64 + 1, device=cuda_device).bfloat16()
    t["x"] = off[1:].view(3, 10, 64)                # contiguous, two bytes off
    r, h = call(t, kind)
    check_forward(t, kind, r, h)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r2, h2 = call(t, kind)
    side.synchronize()
    assert torch.equal(r, r2) and torch.equal(h, h2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r3, h3 = call(t, kind)
    t["y"].mul_(-2)
    graph.replay()
    r4, h4 = call(t, kind)
    torch.cuda.synchronize()
    assert torch.equal(r3, r4) and torch.equal(h3, h4)


@pytest.mark.gpu
def test_forward_odd_values(cuda_device):
    """Constant rows (deviation 0), a NaN and an infinity stay in their rows."""
    t, kind = make((1, 4, 64), torch.float32, cuda_device)
    t["x"][0, 0] = 3.0
    t["y"][0, 0] = 0.0
    ref = call(t, kind)
    assert bool(ref[1].isfinite().all())
    t["x"][0, 1, 5] = float("nan")
    t["y"][0, 2, 7] = float("inf")
    r, h = call(t, kind)
    assert bool(h[0, 1].isnan().all()) and bool(h[0, 2].isnan().all())
    for row in (0, 3):
        assert torch.equal(r[0, row], ref[0][0, row]) and torch.equal(h[0, row], ref[1][0, row])
    empty = call({k: (v[:, :0] if k in ("x", "y") else v) for k, v in t.items()}, kind)
    assert empty[0].shape == (1, 0, 64) and empty[1].shape == (1, 0, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("shape", [(1, 1, 8), (2, 65, 96), (3, 5, 40), (2, 3, 7), (2, 70, 1025),
                                   (1, 257, 1024), (2, 130, 1408), (1, 3, 8192)])
def test_quantized_output(cuda_device, fmt, shape):
    """The codes are those of h's fp32 values: with fp32 input the unquantised
    call returns exactly them."""
    for dtype in DTYPES:
        t, kind = make(shape, dtype, cuda_device, gate=True, post=True)
        r, q = call(t, kind, quantize=fmt)
        r2, h = call(t, kind)
        assert torch.equal(r, r2) and q.shape == shape and q.dtype == dtype
        if dtype != torch.float32:
            # the same rows and parameters widened: x, y and the rounded r are
            # exact in fp32, so N(r) is computed from the same numbers
            t2 = {k: None for k in NAMES}
            t2.update(x=r.float(), weight=t["weight"].float(), norm_bias=t["norm_bias"].float())
            _, h = call(t2, kind)
        ref = mx.mx_quantize(h.float(), fmt)
        if dtype == torch.float32 or shape[-1] * 4 % 16 == 0:
            got, want = q.dequantize(torch.float32), ref.dequantize(torch.float32)
            if dtype == torch.float32:
                assert torch.equal(q.data, ref.data) and torch.equal(q.scales, ref.scales)
            else:
                # rows of 16-bit pieces deal their columns to lanes in another
                # order: a sum's last bit may move a value across a border
                assert ((got != want).float().mean() < 2e-3)


# ----------------------------------------------------------- GPU: gradients

def check_grads(t, kind, r, h, dr, dh):
    leaves = [k for k in NAMES if t[k] is not None]
    grads = dict(zip(leaves, torch.autograd.grad(
        [o for o, g in ((r, dr), (h, dh)) if g is not None], [t[k] for k in leaves],
        [g for g in (dr, dh) if g is not None], allow_unused=True)))
    torch.cuda.synchronize()
    d, f = forward64(t, kind, r)
    C = t["x"].shape[-1]
    rows = t["x"].numel() // C
    tol = (C + 16) * U

    def back(dn, Dn, n, Nm, rstd):
        g = dn - n * (dn * n).mean(-1, keepdim=True)
        G = Dn + Nm * (Dn * Nm).mean(-1, keepdim=True)
        if kind == "layer":
            g, G = g - dn.mean(-1, keepdim=True), G + Dn.mean(-1, keepdim=True)
        return g * rstd, G * rstd

    zero = torch.zeros_like(f["r"])
    dh64 = zero if dh is None else dh.double()
    dr64 = zero if dr is None else dr.double()
    dn = dh64 * d["weight"]
    g, G = back(dn, dn.abs(), f["n"], f["Nm"], f["rstd"])
    g, G = g + dr64, G + dr64.abs()

    def total(term, Term, name, keep_batch=False, extra=0):
        """A column sum of rows terms, each off by a few tol of its magnitude."""
        over = tuple(range(1 if keep_batch else 0, term.dim() - 1))
        ref = term.sum(over) if over else term
        mag = Term.sum(over) if over else Term
        close(grads[name], ref, (rows * U + (4 + extra) * tol) * mag, name)

    close(grads["x"], g, 4 * tol * G, "x")
    total(dh64 * f["n"], dh64.abs() * f["Nm"], "weight")
    if t["norm_bias"] is not None:
        total(dh64, dh64.abs(), "norm_bias")
    if t["y"] is None:
        return
    s = f["s"]
    gate = d["gate"].reshape(g.shape[0], *[1] * (g.dim() - 2), -1) if d["gate"] is not None else 1.0
    if t["gamma"] is not None:
        total(g * f["z"] * gate, G * f["Z"] * abs(gate), "gamma", extra=4)
    if t["gate"] is not None:
        gamma = d["gamma"] if d["gamma"] is not None else 1.0
        total(g * f["z"] * gamma, G * f["Z"] * abs(gamma), "gate", keep_batch=True, extra=4)
    dz, Dz = g * s, G * s.abs()
    if t["post_weight"] is not None:
        total(dz * f["m"], Dz * f["M"], "post_weight", extra=4)
        if t["post_bias"] is not None:
            total(dz, Dz, "post_bias", extra=4)
        pw = d["post_weight"]
        dz, Dz = back(dz * pw, Dz * pw.abs(), f["m"], f["M"], f["rstd_y"])
    close(grads["y"], dz, 12 * tol * Dz, "y")


@pytest.mark.gpu
@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("shape", SIZES)
def test_backward(cuda_device, shape, form):
    for dtype in DTYPES:
        t, kind = make(shape, dtype, cuda_device, grad=True, **FORMS[form])
        r, h = call(t, kind)
        g = torch.Generator().manual_seed(7)
        dr = torch.randn(shape, generator=g).to(dtype).to(cuda_device)
        dh = torch.randn(shape, generator=g).to(dtype).to(cuda_device)
        check_grads(t, kind, r, h, dr if t["y"] is not None else None, dh)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_backward_fp32_parameters(cuda_device, dtype):
    t, kind = make((3, 41, 104), dtype, cuda_device, grad=True, gate=True, post=True,
                   param_dtype=torch.float32)
    r, h = call(t, kind)
    check_grads(t, kind, r, h, torch.randn_like(r), torch.randn_like(h))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [(64, 257, 256), (300, 2, 72), (1, 5000, 24), (700, 1, 40),
                                  (297, 5, 1408), (2, 3000, 1032)])
def test_backward_many_rows_and_repeats(cuda_device, rows):
    """More rows than slots, more gate groups than blocks; the same bits again."""
    t, kind = make(rows, torch.float32, cuda_device, grad=True, gate=True)
    r, h = call(t, kind)
    dr, dh = torch.randn_like(r), torch.randn_like(h)
    check_grads(t, kind, r, h, dr, dh)
    leaves = [t[k] for k in NAMES if t[k] is not None]
    first = torch.autograd.grad(call(t, kind), leaves, (dr, dh))
    again = torch.autograd.grad(call(t, kind), leaves, (dr, dh))
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.gpu
def test_backward_partial(cuda_device):
    """One output's gradient alone, one leaf alone, strided and shared gradients."""
    t, kind = make((2, 9, 64), torch.float32, cuda_device, grad=True, post=True)
    r, h = call(t, kind)
    check_grads(t, kind, r, h, torch.randn_like(r), None)
    r, h = call(t, kind)
    check_grads(t, kind, r, h, None, torch.randn_like(h))
    full = torch.autograd.grad(sum(o.sum() for o in call(t, kind)),
                               [t[k] for k in NAMES if t[k] is not None])
    for k, want in zip([k for k in NAMES if t[k] is not None], full):
        one = {n: (v.detach().requires_grad_(n == k) if v is not None else None)
               for n, v in t.items()}
        sum(o.sum() for o in call(one, kind)).backward()
        assert torch.equal(one[k].grad, want), k
    # x and y the same tensor: both gradients add up
    x = t["x"].detach().requires_grad_()
    r, h = vit.residual_norm(x, x, t["weight"].detach())
    h.square().sum().backward()
    x64 = x.detach().double().requires_grad_()
    h64 = torch.nn.functional.layer_norm(2 * x64, (64,), t["weight"].detach().double(), eps=EPS)
    h64.square().sum().backward()
    # the gradient of a norm's square is small against its terms: those carry the error
    scale = (2 * h64.abs() * t["weight"].detach().abs()).detach().amax(-1, keepdim=True) / x64.std(
        -1, keepdim=True).detach()
    assert bool(((x.grad.double() - x64.grad).abs() <= 16 * 80 * U * scale + 1e-12).all())


@pytest.mark.gpu
def test_backward_empty(cuda_device):
    t, kind = make((2, 0, 64), torch.float32, cuda_device, grad=True, gate=True)
    r, h = call(t, kind)
    (r.sum() + h.sum()).backward()
    assert t["x"].grad.shape == (2, 0, 64)
    assert not t["weight"].grad.any() and not t["gate"].grad.any()


@pytest.mark.gpu
def test_gradient_against_differences(cuda_device):
    """<grad, d> against (L(+e) - L(-e)) / 2e of the call itself, along random
    directions of every leaf.  fp32 values of magnitude A carry an error of
    (C + 16) 2^-24 A each into L, and the third derivative of a norm along a
    direction of unit relative size is below a few A: 8 e^2 A."""
    t, kind = make((2, 12, 48), torch.float32, cuda_device, grad=True, gate=True, post=True)
    cr = torch.randn(2, 12, 48, device=cuda_device).double()
    ch = torch.randn(2, 12, 48, device=cuda_device).double()
    r, h = call(t, kind)
    leaves = [k for k in NAMES if t[k] is not None]
    grads = torch.autograd.grad((r, h), [t[k] for k in leaves], (cr.float(), ch.float()))
    e = 2.0 ** -7
    for k, grad in zip(leaves, grads):
        d = torch.randn_like(t[k])
        side = []
        for sign in (1, -1):
            moved = {n: None if v is None else v.detach() for n, v in t.items()}
            moved[k] = moved[k] + sign * e * d
            r2, h2 = call(moved, kind)
            side.append((cr.float().double() * r2.double()).sum()
                        + (ch.float().double() * h2.double()).sum())
        diff = (side[0] - side[1]) / (2 * e)
        dot = (grad.double() * d.double()).sum()
        A = (cr.abs() * r.detach().double().abs()).sum() + (ch.abs() * (
            h.detach().double().abs() + 3)).sum()
        assert abs(diff - dot) <= A * ((48 + 16) * U / e + 8 * e * e), (k, diff, dot)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [768, 1408])
def test_backward_first_call_of_a_process(cuda_device, C):
    """A kernel's first launch asks for the shared memory that it needs, whatever
    the size of later ones."""
    code = ("import torch\n"
            "from scmp_vit_b200.vit import residual_norm\n"
            f"x = torch.randn(64, {C}, device='cuda').bfloat16().requires_grad_()\n"
            f"w = torch.ones({C}, device='cuda').bfloat16()\n"
            "_, h = residual_norm(x, x.detach(), w)\n"
            "h.sum().backward()\n"
            "assert bool(x.grad.isfinite().all())\n")
    root = pathlib.Path(__file__).resolve().parent.parent
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root, timeout=120)


@pytest.mark.gpu
def test_calls_at_the_same_time(cuda_device):
    """Threads with sizes and streams of their own give the bits of one thread."""
    def step(C):
        g = torch.Generator().manual_seed(C)
        t = [torch.randn(300, C, generator=g).bfloat16().to(cuda_device).requires_grad_()
             for _ in range(2)]
        w = torch.randn(C, generator=g).bfloat16().to(cuda_device).requires_grad_()
        r, h = vit.residual_norm(*t, w, post_weight=w)
        return torch.autograd.grad((r, h), (*t, w), (r.detach(), h.detach()))

    sizes = (768, 1408, 2048, 1024)
    want = {C: step(C) for C in sizes}
    torch.cuda.synchronize()
    failed = []

    def work(C):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    got = step(C)
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(x, y) for x, y in zip(got, want[C]))
        except BaseException as e:  # seen by the test's own thread
            failed.append((C, e))

    threads = [threading.Thread(target=work, args=(C,)) for C in sizes]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@pytest.mark.gpu
def test_backward_in_a_graph(cuda_device):
    t, kind = make((2, 30, 96), torch.bfloat16, cuda_device, grad=True, gate=True)
    leaves = [t[k] for k in NAMES if t[k] is not None]
    dr = torch.randn(2, 30, 96, device=cuda_device).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(call(t, kind), leaves, (dr, dr))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(call(t, kind), leaves, (dr, dr))
    with torch.no_grad():
        t["y"].mul_(0.5)
    graph.replay()
    ref = torch.autograd.grad(call(t, kind), leaves, (dr, dr))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


# ------------------------------------- the variants that large calls take
# Slots that walk: 16-bit rows, and fp32 rows of warps that do not fill a block,
# from some 1200 rows on (148 SMs x 3 or 4 blocks x the rows of a block), the next
# row's loads issued into the registers of the one at work.  Backward slots with
# more rows than their ring has stages (148 x 1 or 2 blocks), and parameters read
# again from shared memory.

MANY = [(8, 600, 1024), (8, 601, 1408), (3, 700, 2504), (2, 900, 4104), (4, 700, 1001),
        (3, 500, 2501), (2, 500, 4101), (5, 500, 200)]


@pytest.mark.gpu
@pytest.mark.parametrize("form", [0, 3, 5, 6])
@pytest.mark.parametrize("shape", MANY)
def test_forward_many_rows(cuda_device, shape, form):
    for dtype in DTYPES:
        t, kind = make(shape, dtype, cuda_device, **FORMS[form])
        r, h = call(t, kind)
        check_forward(t, kind, r, h)
        again = call(t, kind)
        assert torch.equal(r, again[0]) and torch.equal(h, again[1])


@pytest.mark.gpu
def test_forward_of_a_training_batch(cuda_device):
    for post in (False, True):
        t, kind = make((16, 1025, 1408), torch.bfloat16, cuda_device, kind="rms", bias=False,
                       gate=True, post=post)
        check_forward(t, kind, *call(t, kind))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("shape", [(8, 600, 1024), (8, 601, 1408), (3, 700, 2504), (2, 900, 4104),
                                   (5, 500, 200)])
def test_quantized_output_many_rows(cuda_device, fmt, shape):
    """Byte for byte the codes of the same pass's h in fp32, rows past the last
    one (up to whole atoms of scales) included."""
    for dtype in DTYPES:
        for form in (dict(), dict(gate=True, post=True), dict(branch=False, kind="rms")):
            t, kind = make(shape, dtype, cuda_device, **form)
            r, q = call(t, kind, quantize=fmt)
            h32 = torch.empty(shape, dtype=torch.float32, device=cuda_device)
            r2 = vit._norm_launch(*[t[k] for k in NAMES], kind, EPS, None, h32)
            ref = mx.mx_quantize(h32, fmt)
            assert r is t["x"] if r2 is None else torch.equal(r, r2)
            assert torch.equal(q.data, ref.data) and torch.equal(q.scales, ref.scales)
            _, f = forward64(t, kind, r)
            close(h32, f["h"], (shape[-1] + 16) * U * f["H"], "h in fp32")


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("shape", [(2, 3, 7), (2, 70, 1025), (3, 90, 1001)])
def test_quantized_output_of_odd_rows(cuda_device, fmt, shape):
    """Rows in single elements deal their columns alike in every type: with the
    rounded r widened, N(r) is computed from the same numbers in the same order,
    so the codes are those of the fp32 call."""
    for dtype in (torch.bfloat16, torch.float16):
        t, kind = make(shape, dtype, cuda_device, gate=True, post=True)
        r, q = call(t, kind, quantize=fmt)
        t2 = {k: None for k in NAMES}
        t2.update(x=r.float(), weight=t["weight"].float(), norm_bias=t["norm_bias"].float())
        _, h = call(t2, kind)
        ref = mx.mx_quantize(h, fmt)
        assert q.dtype == dtype and q.shape == shape
        assert torch.equal(q.data, ref.data) and torch.equal(q.scales, ref.scales)


@pytest.mark.gpu
@pytest.mark.parametrize("form", [0, 3, 4, 6])
@pytest.mark.parametrize("shape", MANY)
def test_backward_many_rows(cuda_device, shape, form):
    for dtype in DTYPES:
        t, kind = make(shape, dtype, cuda_device, grad=True, **FORMS[form])
        r, h = call(t, kind)
        g = torch.Generator().manual_seed(7)
        dr = torch.randn(shape, generator=g).to(dtype).to(cuda_device)
        dh = torch.randn(shape, generator=g).to(dtype).to(cuda_device)
        check_grads(t, kind, r, h, dr if t["y"] is not None else None, dh)
        r, h = call(t, kind)
        leaves = [t[k] for k in NAMES if t[k] is not None]
        outs, grads = ((h,), (dh,)) if t["y"] is None else ((r, h), (dr, dh))
        first = torch.autograd.grad(outs, leaves, grads, retain_graph=True)
        again = torch.autograd.grad(outs, leaves, grads)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_rows_fp32_parameters(cuda_device, dtype):
    for shape in ((8, 600, 1024), (2, 900, 4104), (4, 700, 1001)):
        t, kind = make(shape, dtype, cuda_device, grad=True, gate=True, post=True,
                       param_dtype=torch.float32)
        r, h = call(t, kind)
        check_forward(t, kind, r, h)
        check_grads(t, kind, r, h, torch.randn_like(r), torch.randn_like(h))
