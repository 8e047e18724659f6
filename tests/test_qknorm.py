"""``attention.split_qkv_norm`` against norms and turned complex numbers in 64 bits:
values, gradients, layouts and refusals.

Bounds, with u = 2^-24 and D elements per row: the mean is off by at most (D + 2) u
A (A = mean |x|), the deviation relatively by (D / 2 + 8) u (its sum, the square root's
two steps), so n by (D + 10) u (|n| + A / deviation); weight, bias, rotation and the
products of the backward pass add a few u of what they multiply.  Sums over R rows
add R u of the sum of magnitudes.  Then the type's half step."""
import copy
import ctypes
import math
import pickle

import pytest
import torch

from scmp_vit_b200 import _lib, attention
from scmp_vit_b200.attention import (GridRotary, QKNorm, RotaryAxes, make_sc_attention_forward,
                                     split_qkv, split_qkv_norm)

DTYPES = (torch.float32, torch.bfloat16, torch.float16)
U = 2.0 ** -24


def positions(grid, cls=1):
    pos = torch.cartesian_prod(*[torch.arange(n) for n in grid]).reshape(-1, len(grid))
    return torch.cat([torch.full((cls, len(grid)), -1), pos]).to(torch.int32)


def turn64(x, dims, pos, interleaved, sign=1):
    """x [B, H, N, D] in 64 bits, turned; base 10000."""
    if not dims:
        return x
    pos = pos.to(x.device)
    pos = pos[None] if pos.dim() == 2 else pos
    parts, at = list(x.unbind(-1)), 0
    for a, d in enumerate(dims):
        for i in range(d // 2):
            e = (at + 2 * i, at + 2 * i + 1) if interleaved else (at + i, at + i + d // 2)
            c = pos[..., a].clamp(min=0).double()
            t = (sign * c * math.exp(-2.0 * i / d * math.log(10000.0)))[:, None]
            u, v = x[..., e[0]], x[..., e[1]]
            parts[e[0]], parts[e[1]] = u * t.cos() - v * t.sin(), v * t.cos() + u * t.sin()
        at += d
    return torch.stack(parts, -1)


def spread64(mag, dims, interleaved):
    """|u| + |v| of each element's pair (the element alone where it stays)."""
    parts, at = list(mag.unbind(-1)), 0
    for d in dims:
        for i in range(d // 2):
            e = (at + 2 * i, at + 2 * i + 1) if interleaved else (at + i, at + i + d // 2)
            parts[e[0]] = parts[e[1]] = mag[..., e[0]] + mag[..., e[1]]
        at += d
    return torch.stack(parts, -1)


def norm64(x, weight, bias, kind, eps):
    """(n weight + bias, n, deviation)."""
    v = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    dev = ((v * v).mean(-1, keepdim=True) + eps).sqrt()
    n = v / dev
    return n * weight + (0 if bias is None else bias), n, dev


def split64(qkv, H, Hk, weights, kind, eps, dims, pos, interleaved):
    B, N, width = qkv.shape
    heads = qkv.reshape(B, N, H + 2 * Hk, -1).transpose(1, 2)
    out = []
    for lo, hi, w, b in ((0, H, weights[0], weights[2]), (H, H + Hk, weights[1], weights[3])):
        t, _, _ = norm64(heads[:, lo:hi], w, b, kind, eps)
        out.append(turn64(t, dims, pos, interleaved))
    return (*out, heads[:, H + Hk:])


def close(got, ref, bound):
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny * 2 * half
    err = (got.double() - ref).abs()
    assert bool((err <= bound + half * ref.abs() * (1 + 1e-3) + tiny).all()), (
        err / (bound + half * ref.abs() + tiny)).max()


def check(qkv, H, Hk, weights, kind, eps, axes, pos, transpose_v, grads=None):
    """Values and, with grads of q, k, v, every gradient."""
    leaves = [t if t is None else t.detach().requires_grad_() for t in (qkv, *weights)]
    q, k, v = split_qkv_norm(leaves[0], H, *leaves[1:3], *leaves[3:], kind=kind, eps=eps,
                             axes=axes, pos=pos, num_kv_heads=Hk, transpose_v=transpose_v)
    dims = [] if axes is None else axes.dims
    inter = True if axes is None else axes.interleaved
    D = q.shape[-1]
    big = [t if t is None else t.detach().double().requires_grad_() for t in (qkv, *weights)]
    ref = split64(big[0], H, Hk, big[1:], kind, eps, dims, pos, inter)
    heads = big[0].detach().reshape(*qkv.shape[:2], H + 2 * Hk, D).transpose(1, 2)
    assert torch.equal(v, heads[:, H + Hk:].to(v.dtype))
    assert (v.transpose(-1, -2) if transpose_v else v).is_contiguous()
    sides = []
    for got, r, lo, hi, i in ((q, ref[0], 0, H, 0), (k, ref[1], H, H + Hk, 1)):
        x, w, b = heads[:, lo:hi], big[1 + i].detach(), big[3 + i]
        t, n, dev = norm64(x, w, None if b is None else b.detach(), kind, eps)
        wide = n.abs() + x.abs().mean(-1, keepdim=True) / dev
        mag = w.abs() * wide + (0 if b is None else b.detach().abs())
        close(got.detach(), r.detach(), (D + 16) * U * spread64(mag.expand_as(x), dims, inter))
        sides.append((w, n, dev, wide))
    # (v is one copy: its gradient is dv, bit for bit)
    if grads is None:
        return q, k, v
    wanted = [t for t in leaves if t is not None]
    got = torch.autograd.grad((q, k, v), wanted, grads)
    want = torch.autograd.grad(ref, [t for t in big if t is not None],
                               [g.double() for g in grads])
    back = got[0].reshape(*qkv.shape[:2], H + 2 * Hk, D).transpose(1, 2)
    bref = want[0].reshape(*qkv.shape[:2], H + 2 * Hk, D).transpose(1, 2)
    assert torch.equal(back[:, H + Hk:], grads[2])
    names = [i for i, t in enumerate(leaves) if t is not None]
    for i, (lo, hi) in enumerate(((0, H), (H, H + Hk))):
        w, n, dev, wide = sides[i]
        g = spread64(grads[i].double().abs(), dims, inter)  # |dt| at most
        gw = g * w.abs()
        m = gw + gw.mean(-1, keepdim=True) + wide * (gw * wide).mean(-1, keepdim=True)
        close(back[:, lo:hi], bref[:, lo:hi], 2 * (D + 20) * U * m / dev)
        rows = g[..., 0].numel()
        close(got[names.index(1 + i)], want[names.index(1 + i)],
              (rows + D + 20) * U * (g * wide).sum((0, 1, 2)))
        if big[3 + i] is not None:
            close(got[names.index(3 + i)], want[names.index(3 + i)],
                  (rows + 20) * U * g.sum((0, 1, 2)))
    for t, gr in zip(wanted, got):
        assert gr.dtype == t.dtype and gr.shape == t.shape
    return q, k, v


# ------------------------------------------------------------ CPU: refusals

def args(**kw):
    a = _lib.QkNormArgs()
    s = a.split
    s.abi_version = _lib.ABI_VERSION
    s.B, s.N, s.H, s.Hk, s.D, s.axes = 1, 2, 4, 2, 16, 2
    s.qkv = s.q = s.k = s.v = s.table = s.pos = 16
    for i in range(2):
        s.dims[i], s.sizes[i] = 8, 4
    a.q_weight = a.k_weight = 16
    a.eps = 1e-6
    for k, v in kw.items():
        if k in ("dims", "sizes"):
            for i, n in enumerate(v):
                getattr(s, k)[i] = n
        else:
            setattr(s if hasattr(s, k) and k != "x" else a, k, v)
    return a


@pytest.mark.parametrize("kw,code,msg", [
    (dict(abi_version=2), -1, "abi_version"),
    (dict(dtype=3), -1, "dtype"),
    (dict(param_dtype=2), -1, "parameters"),
    (dict(N=-1), -1, "shape"),
    (dict(H=0), -1, "shape"),
    (dict(Hk=3), -1, "multiple"),
    (dict(D=7), -4, "even"),
    (dict(D=258), -4, "256"),
    (dict(axes=-1), -1, "axes"),
    (dict(axes=5), -1, "axes"),
    (dict(dims=(3, 4)), -1, "axis 0"),
    (dict(sizes=(4, 0)), -1, "axis 1"),
    (dict(dims=(8, 10)), -1, "exceed"),
    (dict(pos=None), -1, "non-NULL"),
    (dict(q_weight=None), -1, "non-NULL"),
    (dict(k_weight=18), -1, "aligned to its elements"),
    (dict(k_bias=18), -1, "aligned to its elements"),
    (dict(table=12), -1, "aligned"),
    (dict(k=18), -1, "aligned to its elements"),
    (dict(B=1 << 20, N=1 << 20), -4, "tokens"),
    (dict(eps=-1.0), -1, "eps"),
    (dict(eps=math.nan), -1, "eps"),
    (dict(inverse=1), -1, "x (the forward"),
    (dict(inverse=1, x=18), -1, "aligned to its elements"),
    (dict(inverse=1, x=16, dq_weight=16), -3, "workspace"),
    (dict(inverse=1, x=16, dk_bias=16, workspace=16, workspace_bytes=100), -3, "workspace"),
])
def test_refusals(kw, code, msg):
    assert _lib.load().scmp_split_qkv_norm(ctypes.byref(args(**kw)), None) == code
    assert msg in _lib.last_error()


def test_packed_arguments_are_the_struct():
    a, values = _lib.QkNormArgs(), []
    for part in (a.split, a):
        for name, kind in part._fields_:
            for i in range(getattr(kind, "_length_", 0) or 1):
                if name == "split":
                    continue
                values.append(len(values) + 1)
                if hasattr(kind, "_length_"):
                    getattr(part, name)[i] = values[-1]
                else:
                    setattr(part, name, values[-1])
    assert _lib.PACK_QKNORM.pack(*values) == bytes(a)
    lib = _lib.load()
    for shape in ((0, 1, 8), (1, 0, 8), (1, 1, 0), (1, 1, 258)):
        assert lib.scmp_split_qkv_norm_workspace(*shape) == 0
    assert lib.scmp_split_qkv_norm_workspace(16, 4, 64) > 0


def test_python_refusals(monkeypatch):
    qkv, w = torch.zeros(1, 2, 96), torch.ones(16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        split_qkv_norm(qkv, 2, w, w)
    with pytest.raises(ValueError, match="kind"):
        QKNorm(16, "batch")
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    launched = []
    monkeypatch.setattr(attention, "call", lambda *a: launched.append(a))
    axes, pos = RotaryAxes([8, 8], [4, 4]), torch.zeros(2, 2, dtype=torch.int32)
    for kw, match in ((dict(kind="batch"), "kind"), (dict(eps=-1), "eps"),
                      (dict(num_heads=5), "qkv must"), (dict(num_kv_heads=3), "multiple"),
                      (dict(q_weight=w[:8]), "q_weight"), (dict(k_weight=w.half()), "k_weight"),
                      (dict(k_bias=torch.ones(4)), "k_bias"), (dict(axes=axes), "together"),
                      (dict(pos=pos), "together"), (dict(axes=axes, pos=pos.long()), "pos must"),
                      (dict(axes=RotaryAxes([20], [4]), pos=pos[:, :1]), "head size")):
        full = dict(dict(num_heads=2, q_weight=w, k_weight=w), **kw)
        with pytest.raises(ValueError, match=match):
            split_qkv_norm(qkv, **full)
    with pytest.raises(TypeError, match="parameters"):
        split_qkv_norm(qkv, 2, w.half(), w.half())
    with pytest.raises(TypeError, match="float32"):
        split_qkv_norm(qkv.double(), 2, w, w)
    assert launched == []
    split_qkv_norm(qkv, 2, w, w, w, w, axes=axes, pos=pos)
    split_qkv_norm(qkv.half(), 2, w, w)
    assert len(launched) == 2
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), torch.no_grad():
        for at in range(2):
            t = [qkv, w]
            t[at] = fwAD.make_dual(t[at], torch.ones_like(t[at]))
            with pytest.raises(NotImplementedError, match="jvp"):
                split_qkv_norm(t[0], 2, t[1], w)


def test_reference_gradients_by_differences():
    """The 64-bit formula's gradients against its own differences."""
    g = torch.Generator().manual_seed(1)
    pos = positions((2, 2))
    for kind in ("rms", "layer"):
        t = [torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()
             for s in ((2, 5, 4 * 10), (10,), (10,), (10,), (10,))]
        assert torch.autograd.gradcheck(
            lambda x, *w: split64(x, 2, 1, w, kind, 1e-3, [4, 4], pos, False), t)


def test_module_copies():
    m = QKNorm(16, "layer")
    for c in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        assert sorted(n for n, _ in c.named_parameters()) == ["k_bias", "k_weight", "q_bias",
                                                              "q_weight"]
    assert [n for n, _ in QKNorm(16).named_parameters()] == ["q_weight", "k_weight"]


# ------------------------------------------------------------ GPU

CASES = [  # B, H, Hk, D, dims, grid, cls: every width of pieces in every type
    (2, 16, 16, 64, [32, 32], (16, 16), 1),
    (1, 4, 2, 64, [16, 24, 24], (3, 5, 4), 1),
    (3, 4, 1, 40, [20, 20], (6, 7), 0),
    (2, 2, 2, 40, [24, 12], (5, 9), 2),
    (1, 12, 12, 128, [44, 42, 42], (2, 8, 8), 1),
    (2, 3, 3, 22, [10, 6, 4], (2, 3, 5), 1),
    (1, 2, 1, 256, [64, 64, 64, 64], (2, 2, 3, 3), 1),
    (1, 2, 2, 248, [124, 124], (3, 4), 1),
    (5, 8, 4, 80, [40, 40], (1, 1), 0),
    (2, 2, 2, 34, [30], (33,), 0),
    (2, 5, 1, 96, [], (50,), 0),
    (1, 1, 1, 2, [2], (7,), 1),
    (3, 1, 1, 254, [], (5,), 0),
    (33, 16, 4, 64, [64], (1,), 0),   # the next token of each sequence
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_values_and_gradients(cuda_device, case, interleaved, kind):
    B, H, Hk, D, dims, grid, cls = CASES[case]
    dev = cuda_device
    pos = positions(grid, cls).to(dev)
    N = pos.shape[0]
    axes = RotaryAxes(dims, grid, interleaved=interleaved, device=dev) if dims else None
    pos = pos if dims else None
    for i, dtype in enumerate(DTYPES):
        for transpose_v in (True, False):
            g = torch.Generator().manual_seed(case)

            def randn(*shape, dt=dtype):
                return torch.randn(*shape, generator=g).to(dt).to(dev)
            pdt = torch.float32 if transpose_v else dtype
            qkv = randn(B, N, (H + 2 * Hk) * D) * torch.exp(randn(B, N, 1)) + 0.3
            weights = [1 + 0.3 * randn(D, dt=pdt), 1 + 0.3 * randn(D, dt=pdt),
                       0.2 * randn(D, dt=pdt) if kind == "layer" else None,
                       0.2 * randn(D, dt=pdt) if kind == "layer" or i else None]
            grads = [randn(B, H, N, D), randn(B, Hk, N, D), randn(B, Hk, N, D)]
            if transpose_v:
                grads[2] = grads[2].transpose(-1, -2).contiguous().transpose(-1, -2)
            check(qkv, H, Hk, weights, kind, 1e-6, axes, pos, transpose_v, grads)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_tokens(cuda_device, dtype):
    """Threads that walk several heads, blocks that walk several units."""
    dev, g = cuda_device, torch.Generator().manual_seed(3)

    def randn(*shape):
        return torch.randn(*shape, generator=g).to(dtype).to(dev)
    axes = RotaryAxes([16, 16], [40, 40], interleaved=False, device=dev)
    pos = positions((40, 40)).to(dev)
    for H, Hk in ((8, 8), (6, 2)):
        check(randn(9, 1601, (H + 2 * Hk) * 32), H, Hk, [randn(32) for _ in range(4)], "layer",
              1e-5, axes, pos, H == 8, [randn(9, h, 1601, 32) for h in (H, Hk, Hk)])


@pytest.mark.gpu
def test_rows_that_are_odd(cuda_device):
    """Zero rows, constant rows, eps 0, one NaN or infinity (its head's row alone),
    values whose squares leave fp16's range."""
    dev, g = cuda_device, torch.Generator().manual_seed(5)
    qkv = torch.randn(1, 6, 3 * 2 * 16, generator=g).to(dev)
    w = torch.ones(16, device=dev)
    qkv[0, 0] = 0
    qkv[0, 1] = 3
    for kind in ("rms", "layer"):
        check(qkv, 2, 2, [w, w, None, None], kind, 1e-6, None, None, False)
    q, _, _ = split_qkv_norm(qkv, 2, w, w, eps=0.0, transpose_v=False)
    assert bool(q[0, :, 0].isnan().all()) and not bool(q[0, :, 1:].isnan().any())
    big = (qkv * 3000).half()
    check(big, 2, 2, [w.half(), w.half(), None, None], "rms", 1e-6, None, None, False)
    for bad in (math.nan, math.inf):
        t = qkv.clone()
        t[0, 3, 20] = bad  # q, head 1
        q2, k2, v2 = split_qkv_norm(t, 2, w, w, transpose_v=False)
        q, k, v = split_qkv_norm(qkv, 2, w, w, transpose_v=False)
        # (an infinite deviation leaves zeros beside the NaN)
        assert not torch.equal(q2[0, 1, 3], q[0, 1, 3]) and bool(q2[0, 1, 3].isnan().any())
        q2[0, 1, 3] = q[0, 1, 3]
        assert all(torch.equal(a, b) for a, b in ((q, q2), (k, k2), (v, v2)))


FAR = [  # D, dims, grid: every width of pieces
    (64, [32, 32], (4, 5)), (40, [20, 20], (5, 4)), (48, [24, 12], (3, 6)), (22, [10, 6, 4], (2, 3, 3)),
    (128, [44, 42, 42], (2, 3, 3)), (256, [128, 128], (4, 4)), (34, [30], (19,)), (2, [2], (7,))]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("D,dims,grid", FAR)
def test_layer_norm_far_from_zero(cuda_device, D, dims, grid, interleaved):
    """Rows whose mean is 100 to 1000 deviations, and constant ones, turned: what is
    normalised is x - mean, whose terms are no larger than the deviation.  Rows are m + d
    and m - d with few bits, so that every sum of them is exact, m is a representable mean
    and x - m exact: the error is the deviation's (D / 2 + 8) u and a few u of each
    product, all relative to |n|.  A constant row leaves 0, turned biases."""
    dev, g = cuda_device, torch.Generator().manual_seed(D)
    pos = positions(grid, 1).to(dev)
    axes = RotaryAxes(dims, grid, interleaved=interleaved, device=dev)
    N = pos.shape[0]
    for i, dtype in enumerate(DTYPES):
        step = (2.0 ** -14, 2.0 ** -4, 2.0 ** -7)[i]  # (8 + d is a number of each type)
        for size, deviation in ((8.0, 0.08), (8.0, 0.02 if i != 1 else 0.1), (0.0, 1.0)):
            d = (torch.randn(1, N, 3, D // 2, generator=g) * deviation / step).round() * step
            x = torch.cat([size + d, size - d], -1)[..., torch.randperm(D, generator=g)]
            qkv = x.reshape(1, N, 3 * D).to(dtype).to(dev)
            assert torch.equal(qkv.cpu().float(), x.reshape(1, N, 3 * D))
            w = [(1 + 0.3 * torch.randn(D, generator=g)).to(dev) for _ in range(2)]
            b = [0.2 * torch.randn(D, generator=g).to(dev) for _ in range(2)]
            for bias in ([None, None], b):
                q, k, _ = split_qkv_norm(qkv, 1, *w, *bias, kind="layer", axes=axes, pos=pos)
                heads = qkv.double().reshape(1, N, 3, D).transpose(1, 2)
                for j, got in enumerate((q, k)):
                    wj, bj = w[j].double(), None if bias[j] is None else bias[j].double()
                    t, n, _ = norm64(heads[:, j:j + 1], wj, bj, "layer", 1e-6)
                    mag = wj.abs() * n.abs() + (0 if bj is None else bj.abs())
                    close(got, turn64(t, dims, pos, interleaved),
                          (D / 2 + 16) * U * spread64(mag.expand_as(n), dims, interleaved))
        for c in (100.0, -10.0, 7.5, 0.375, 3000.0 if i != 1 else 3008.0):
            qkv = torch.full((1, N, 3 * D), c, dtype=dtype, device=dev)
            leaves = [t.detach().requires_grad_() for t in (qkv, *w)]
            q, k, _ = split_qkv_norm(leaves[0], 1, *leaves[1:], kind="layer", axes=axes, pos=pos)
            assert not q.any() and not k.any()
            _, dwq, dwk = torch.autograd.grad((q, k), leaves, (torch.ones_like(q),) * 2)
            assert not dwq.any() and not dwk.any()
            q, k, _ = split_qkv_norm(qkv, 1, *w, *b, kind="layer", axes=axes, pos=pos)
            for got, bj in ((q, b[0]), (k, b[1])):
                bj = bj.double().expand(1, 1, N, D)
                close(got, turn64(bj, dims, pos, interleaved),
                      4 * U * spread64(bj.abs(), dims, interleaved))


@pytest.mark.gpu
def test_batched_positions_and_range(cuda_device):
    dev, g = cuda_device, torch.Generator().manual_seed(1)
    axes = RotaryAxes([4, 4], [7, 9], device=dev)
    pos = torch.stack([torch.randint(0, 7, (3, 20), generator=g),
                       torch.randint(0, 9, (3, 20), generator=g)], -1).to(torch.int32).to(dev)
    pos[1, 4, 0] = -1
    qkv = torch.randn(3, 20, 3 * 2 * 8, generator=g).to(dev)
    w = torch.randn(8, generator=g).to(dev)
    grads = [torch.randn(3, 2, 20, 8, generator=g).to(dev) for _ in range(3)]
    q, k, _ = check(qkv, 2, 2, [w, w, None, None], "rms", 1e-6, axes, pos, False, grads)
    pos[2, 7, 1] = 9
    pos[0, 3, 0] = 2 ** 31 - 1
    q2, k2, _ = split_qkv_norm(qkv, 2, w, w, axes=axes, pos=pos)
    for a, b in ((q, q2), (k, k2)):
        a = a.detach()
        assert bool(b[2, :, 7, 4:].isnan().all()) and bool(b[0, :, 3, :4].isnan().all())
        b[2, :, 7, 4:], b[0, :, 3, :4] = a[2, :, 7, 4:], a[0, :, 3, :4]
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_strides_streams_graph_empty_repeats(cuda_device):
    dev = cuda_device
    axes = RotaryAxes([16, 16], [5, 5], device=dev)
    pos = positions((5, 5)).to(dev)
    w = torch.randn(65, device=dev).half()
    kw = dict(axes=axes, pos=pos)
    big = torch.randn(2, 26, 200, device=dev).half()
    for qkv in (big[..., 3:195], big[..., :192].contiguous()):
        got = split_qkv_norm(qkv, 2, w[::2][:32], w[1:33], **kw)
        ref = split_qkv_norm(qkv.clone(), 2, w[::2][:32].clone(), w[1:33].clone(), **kw)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    # an odd address takes narrower pieces, whose sums have another order
    odd = torch.randn(2 * 26 * 192 + 1, device=dev).half()[1:].view(2, 26, 192)
    grads = [torch.randn(2, 2, 26, 32, device=dev).half() for _ in range(3)]
    check(odd, 2, 2, [w[::2][:32], w[1:33], None, None], "rms", 1e-6, axes, pos, True, grads)
    wc = w[:32].contiguous()
    ref = split_qkv_norm(qkv, 2, wc, wc, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = split_qkv_norm(qkv, 2, wc, wc, **kw)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))

    def step(x):
        t = [v.detach().requires_grad_() for v in (x, wc, wc)]
        out = split_qkv_norm(t[0], 2, *t[1:], **kw)
        return [v.detach() for v in out] + list(torch.autograd.grad(out, t, out))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(qkv)
    torch.cuda.current_stream().wait_stream(side)
    static = qkv.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(static)
    static.copy_(qkv * 2 + 1)
    graph.replay()
    torch.cuda.synchronize()
    for _ in range(2):  # (the same bits from every call)
        assert all(torch.equal(a, b) for a, b in zip(got, step(qkv * 2 + 1)))
    t = [v.detach().clone().requires_grad_() for v in (qkv[:0], wc, wc)]
    out = split_qkv_norm(t[0], 2, *t[1:], **kw)
    assert [tuple(v.shape) for v in out] == [(0, 2, 26, 32)] * 3
    grads = torch.autograd.grad(out, t, out)
    assert grads[0].shape == (0, 26, 192) and not grads[1].any() and not grads[2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("empty", ["B", "N"])
def test_parameter_gradients_of_no_rows_at_the_c_entry(cuda_device, dtype, empty):
    """Sums over nothing: 0 in each gradient that is wanted, nothing behind it."""
    code = DTYPES.index(dtype)
    for wanted in range(16):
        out = torch.full((4, 40), math.nan, dtype=dtype, device=cuda_device)
        names = ("dq_weight", "dk_weight", "dq_bias", "dk_bias")
        at = {n: out[i].data_ptr() for i, n in enumerate(names) if wanted >> i & 1}
        a = args(inverse=1, D=32, dtype=code, param_dtype=code, **{empty: 0}, **at)
        attention.call(_lib.load().scmp_split_qkv_norm, 0, bytes(a))
        for i in range(4):
            n = 32 if wanted >> i & 1 else 0
            assert not out[i, :n].any() and bool(out[i, n:].isnan().all())


def test_no_rows_on_the_cpu():
    lib = _lib.load()
    assert lib.scmp_split_qkv_norm(ctypes.byref(args(inverse=1, B=0)), None) == 0
    assert lib.scmp_split_qkv_norm(ctypes.byref(args(inverse=1, N=0, dk_bias=18)), None) == -1
    assert "aligned to its elements" in _lib.last_error()


@pytest.mark.gpu
def test_wants_and_second_derivative(cuda_device):
    dev, g = cuda_device, torch.Generator().manual_seed(2)
    qkv, w, b = (torch.randn(*s, generator=g).to(dev) for s in ((2, 9, 96), (16,), (16,)))
    grads = [torch.randn(2, 2, 9, 16, generator=g).to(dev) for _ in range(3)]
    full = None
    for wants in range(31, 0, -1):
        t = [v.clone().requires_grad_(bool(wants >> i & 1)) for i, v in enumerate((qkv, w, w, b, b))]
        out = split_qkv_norm(t[0], 2, *t[1:], kind="layer", transpose_v=False)
        at = [i for i in range(5) if wants >> i & 1]
        out, gr = zip(*[(o, d) for o, d in zip(out, grads) if o.requires_grad])
        got = torch.autograd.grad(out, [t[i] for i in at], gr, allow_unused=True)
        full = full or got
        for i, d in zip(at, got):
            assert torch.equal(d, full[i])
    qkv.requires_grad_()
    (d,) = torch.autograd.grad(split_qkv_norm(qkv, 2, w, w)[0].sum(), qkv, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), qkv)


@pytest.mark.gpu
def test_in_the_attention(cuda_device):
    """Modules with ``qk_norm`` split by it, the SC forward included; others under
    that name are left alone."""
    from scmp_vit_b200 import vit
    dev = cuda_device
    for kind in ("rms", "layer"):
        m = vit.vit_l14(seed=0, dim=64, depth=1, heads=2, hidden=64, img=56, rope=True,
                        qk_norm=kind).to(dev)
        attn = m.backbone.blocks[0].attn
        with torch.no_grad():
            for p in attn.qk_norm.parameters():
                p.add_(0.3 * torch.randn_like(p))
        x = torch.randn(2, 17, 64, device=dev)
        qkv = attn.qkv(x)
        n = attn.qk_norm
        q, k, v = split_qkv_norm(qkv, 2, n.q_weight, n.k_weight, n.q_bias, n.k_bias, kind=kind,
                                 eps=n.eps, axes=attn.rope.axes, pos=attn.rope.pos,
                                 transpose_v=False)
        a = torch.nn.functional.scaled_dot_product_attention(q, k, v).transpose(1, 2)
        assert torch.equal(attn(x), attn.proj(a.reshape(2, 17, 64)))
        m(torch.randn(1, 3, 56, 56, device=dev)).sum().backward()
        assert all(p.grad is not None for p in n.parameters())
        with torch.no_grad():
            fwd = make_sc_attention_forward(7, sc_av=False, sc_qk=False)
            s = (q @ k.transpose(-2, -1)) * attn.scale
            a = (s.softmax(-1) @ v).transpose(1, 2).reshape(2, 17, 64)
            torch.testing.assert_close(fwd(attn, x), attn.proj(a))
            attn.qk_norm = torch.nn.Identity()
            attn.rope = None
            q, k, v = split_qkv(qkv, 2)
            s = (q @ k.transpose(-2, -1)) * attn.scale
            a = (s.softmax(-1) @ v).transpose(1, 2).reshape(2, 17, 64)
            torch.testing.assert_close(fwd(attn, x), attn.proj(a))
