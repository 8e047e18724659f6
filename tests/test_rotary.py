"""``attention.split_qkv_rotary`` against turned complex numbers in 64 bits:
values, gradient, layouts and refusals.  A turned element is one product and
one fused multiply-add of fp32 numbers whose cos and sin are rounded once:
off by at most 3 2^-24 (|u| + |v|), plus its type's half step."""
import copy
import ctypes
import math
import pickle

import pytest
import torch

from scmp_vit_b200 import _lib
from scmp_vit_b200.attention import (GridRotary, RotaryAxes, make_sc_attention_forward, split_qkv,
                                     split_qkv_rotary)

DTYPES = (torch.float32, torch.bfloat16, torch.float16)
U = 2.0 ** -24


def positions(grid, cls=1):
    pos = torch.cartesian_prod(*[torch.arange(n) for n in grid]).reshape(-1, len(grid))
    return torch.cat([torch.full((cls, len(grid)), -1), pos]).to(torch.int32)


def rotate64(x, dims, pos, base, scales, interleaved, sign=1):
    """x [B, H, N, D], pos [N or B x N, axes]; (turned, |u| + |v| per element)."""
    out, mag = x.double().clone(), x.double().abs()
    pos = pos.to(x.device)
    pos = pos[None] if pos.dim() == 2 else pos
    at = 0
    for a, d in enumerate(dims):
        for i in range(d // 2):
            e = (at + 2 * i, at + 2 * i + 1) if interleaved else (at + i, at + i + d // 2)
            c = pos[..., a].clamp(min=0).double()
            angle = (sign * c * scales[a] * math.exp(-2.0 * i / d * math.log(base)))[:, None]
            u, v = x[..., e[0]].double(), x[..., e[1]].double()
            out[..., e[0]] = u * angle.cos() - v * angle.sin()
            out[..., e[1]] = v * angle.cos() + u * angle.sin()
            mag[..., e[0]] = mag[..., e[1]] = u.abs() + v.abs()
        at += d
    return out, mag


def close(got, ref, mag):
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny * 2 * half
    assert bool(((got.double() - ref).abs() <= 3 * U * mag + half * ref.abs() * (1 + 1e-3)
                 + tiny).all())


# ------------------------------------------------------------ CPU: refusals

@pytest.mark.parametrize("kw,code,msg", [
    (dict(abi_version=2), -1, "abi_version"),
    (dict(dtype=3), -1, "dtype"),
    (dict(N=-1), -1, "shape"),
    (dict(H=0), -1, "shape"),
    (dict(Hk=3), -1, "multiple"),
    (dict(D=7), -4, "even"),
    (dict(D=258), -4, "256"),
    (dict(axes=0), -1, "axes"),
    (dict(axes=5), -1, "axes"),
    (dict(dims=(3, 4)), -1, "axis 0"),
    (dict(sizes=(4, 0)), -1, "axis 1"),
    (dict(dims=(8, 10)), -1, "exceed"),
    (dict(pos=None), -1, "non-NULL"),
    (dict(table=12), -1, "aligned"),
    (dict(pos=18), -1, "aligned"),
    (dict(k=18), -1, "aligned to its elements"),
    (dict(B=1 << 20, N=1 << 20), -4, "tokens"),
])
def test_refusals(kw, code, msg):
    a = _lib.RotaryArgs()
    a.abi_version = _lib.ABI_VERSION
    a.B, a.N, a.H, a.Hk, a.D, a.axes = 1, 2, 4, 2, 16, 2
    a.qkv = a.q = a.k = a.v = a.table = a.pos = 16
    kw = dict(dict(dims=(8, 8), sizes=(4, 4)), **kw)
    for k, v in kw.items():
        if k in ("dims", "sizes"):
            for i, n in enumerate(v):
                getattr(a, k)[i] = n
        else:
            setattr(a, k, v)
    assert _lib.load().scmp_split_qkv_rotary(ctypes.byref(a), None) == code
    assert msg in _lib.last_error()


def test_python_refusals_on_cpu():
    with pytest.raises(ValueError, match="even"):
        RotaryAxes([3], [4])
    with pytest.raises(ValueError, match="axes"):
        RotaryAxes([2] * 5, [4] * 5)
    with pytest.raises(ValueError, match="size"):
        RotaryAxes([2, 2], [4])
    with pytest.raises(ValueError, match="base"):
        RotaryAxes([2], [4], base=0)
    axes = RotaryAxes([8, 8], [4, 4])
    with pytest.raises(RuntimeError, match="no CPU path"):
        split_qkv_rotary(torch.zeros(1, 2, 96), 2, axes, torch.zeros(2, 2, dtype=torch.int32))


def test_copies():
    """Modules with positions are copied and pickled like others."""
    rope = GridRotary((3, 2), 8)
    for c in (copy.deepcopy(rope), pickle.loads(pickle.dumps(rope))):
        assert c.axes.dims == [4, 4] and c.axes.sizes == [3, 2]
        assert torch.equal(c.axes.table_bits, rope.axes.table_bits)
        assert torch.equal(c.pos, rope.pos)


def test_table():
    """cos and sin of far coordinates are those of the 64-bit angle, and a cast
    of the module leaves them."""
    axes = RotaryAxes([4, 2], [5, 100000], base=100.0, scales=[0.5, 1.0]).half()
    t = axes.table_bits.view(torch.float32).reshape(-1, 2)
    assert t.shape == (5 * 2 + 100000, 2)
    for c in range(5):
        for i, f in enumerate((1.0, 0.1)):
            assert t[2 * c + i].tolist() == pytest.approx(
                [math.cos(0.5 * c * f), math.sin(0.5 * c * f)], abs=2 ** -24)
    assert t[10 + 99999].tolist() == pytest.approx([math.cos(99999), math.sin(99999)],
                                                   abs=2 ** -24)


# ------------------------------------------------------------- GPU: values

CASES = [  # B, H, Hk, D, dims, grid, cls
    (1, 1, 1, 2, [2], (1,), 0),
    (2, 16, 16, 64, [32, 32], (16, 16), 1),
    (1, 4, 2, 64, [16, 24, 24], (3, 5, 4), 1),
    (3, 4, 1, 40, [20, 20], (6, 7), 0),
    (2, 2, 2, 40, [24, 12], (5, 9), 2),
    (1, 12, 12, 128, [44, 42, 42], (2, 8, 8), 1),
    (2, 3, 3, 22, [10, 6, 4], (2, 3, 5), 1),
    (1, 2, 1, 256, [64, 64, 64, 64], (2, 2, 3, 3), 1),
    (5, 8, 4, 80, [40, 40], (1, 1), 0),
    (2, 2, 2, 34, [30], (33,), 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_values_and_gradient(cuda_device, case, interleaved):
    B, H, Hk, D, dims, grid, cls = CASES[case]
    dev = cuda_device
    pos = positions(grid, cls).to(dev)
    N = pos.shape[0]
    scales = [1.0, 0.5, 2.0, 1.5][:len(dims)]
    axes = RotaryAxes(dims, grid, base=1000.0, scales=scales, interleaved=interleaved, device=dev)
    for dtype in DTYPES:
        for transpose_v in (True, False):
            g = torch.Generator().manual_seed(case)
            qkv = torch.randn(B, N, (H + 2 * Hk) * D, generator=g).to(dtype).to(dev)
            qkv.requires_grad_()
            q, k, v = split_qkv_rotary(qkv, H, axes, pos, num_kv_heads=Hk, transpose_v=transpose_v)
            heads = qkv.detach().reshape(B, N, H + 2 * Hk, D).transpose(1, 2)
            for got, x in ((q, heads[:, :H]), (k, heads[:, H:H + Hk])):
                close(got.detach(), *rotate64(x, dims, pos, 1000.0, scales, interleaved))
                rest = sum(dims)
                assert torch.equal(got[..., rest:], x[..., rest:])
                if cls:
                    assert torch.equal(got[:, :, :cls], x[:, :, :cls])
            assert torch.equal(v, heads[:, H + Hk:])
            assert (v.transpose(-1, -2) if transpose_v else v).is_contiguous()
            grads = [torch.randn(t.shape, generator=g).to(dtype).to(dev) for t in (q, k, v)]
            if transpose_v:
                grads[2] = grads[2].transpose(-1, -2).contiguous().transpose(-1, -2)
            (dqkv,) = torch.autograd.grad((q, k, v), (qkv,), grads)
            back = dqkv.reshape(B, N, H + 2 * Hk, D).transpose(1, 2)
            close(back[:, :H], *rotate64(grads[0], dims, pos, 1000.0, scales, interleaved, -1))
            close(back[:, H:H + Hk],
                  *rotate64(grads[1], dims, pos, 1000.0, scales, interleaved, -1))
            assert torch.equal(back[:, H + Hk:], grads[2])


@pytest.mark.gpu
def test_equals_split_without_positions(cuda_device):
    qkv = torch.randn(2, 50, 3 * 4 * 64, device=cuda_device).bfloat16()
    axes = RotaryAxes([32, 32], [4, 4], device=cuda_device)
    pos = torch.full((50, 2), -1, dtype=torch.int32, device=cuda_device)
    for a, b in zip(split_qkv(qkv, 4), split_qkv_rotary(qkv, 4, axes, pos)):
        assert torch.equal(a, b) and a.stride() == b.stride()


@pytest.mark.gpu
def test_batched_positions_and_range(cuda_device):
    """Positions per sample; a coordinate past the table gives NaN, a negative
    one leaves its axis alone."""
    dims, dev = [4, 4], cuda_device
    axes = RotaryAxes(dims, [7, 9], device=dev)
    g = torch.Generator().manual_seed(1)
    pos = torch.stack([torch.randint(0, 7, (3, 20), generator=g),
                       torch.randint(0, 9, (3, 20), generator=g)], -1).to(torch.int32).to(dev)
    pos[1, 4, 0] = -1
    qkv = torch.randn(3, 20, 3 * 2 * 8, generator=g).to(dev)
    q, k, v = split_qkv_rotary(qkv, 2, axes, pos)
    heads = qkv.reshape(3, 20, 6, 8).transpose(1, 2)
    close(q, *rotate64(heads[:, :2], dims, pos, 10000.0, [1, 1], True))
    assert torch.equal(q[1, :, 4, :4], heads[1, :2, 4, :4])
    pos[2, 7, 1] = 9
    pos[0, 3, 0] = 2 ** 31 - 1
    q2, k2, _ = split_qkv_rotary(qkv, 2, axes, pos)
    for a, b in ((q, q2), (k, k2)):
        assert bool(b[2, :, 7, 4:].isnan().all()) and bool(b[0, :, 3, :4].isnan().all())
        b[2, :, 7, 4:], b[0, :, 3, :4] = a[2, :, 7, 4:], a[0, :, 3, :4]
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_strides_streams_graph_empty(cuda_device):
    dev = cuda_device
    axes = RotaryAxes([16, 16], [5, 5], device=dev)
    pos = positions((5, 5)).to(dev)
    big = torch.randn(2, 26, 200, device=dev).half()
    for qkv in (big[..., 3:195], big[..., :192].contiguous(),
                torch.randn(2 * 26 * 192 + 1, device=dev).half()[1:].view(2, 26, 192)):
        q, k, v = split_qkv_rotary(qkv, 2, axes, pos)
        ref = split_qkv_rotary(qkv.clone(), 2, axes, pos)
        assert all(torch.equal(a, b) for a, b in zip((q, k, v), ref))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = split_qkv_rotary(qkv, 2, axes, pos)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = split_qkv_rotary(qkv, 2, axes, pos)
    qkv.mul_(-3)
    graph.replay()
    ref = split_qkv_rotary(qkv, 2, axes, pos)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    for shape in ((0, 26, 192), (2, 0, 192)):
        e = torch.zeros(shape, device=dev, requires_grad=True)
        q, k, v = split_qkv_rotary(e, 2, axes, pos if shape[1] else pos[:0])
        (q.sum() + v.sum()).backward()
        assert q.shape == (shape[0], 2, shape[1], 32) and e.grad.shape == shape


@pytest.mark.gpu
def test_partial_and_strided_gradients(cuda_device):
    """One output used alone; gradients that come expanded or transposed."""
    dev = cuda_device
    axes = RotaryAxes([4, 4], [3, 3], interleaved=False, device=dev)
    pos = positions((3, 3)).to(dev)
    for transpose_v in (True, False):
        x = torch.randn(2, 10, 3 * 2 * 8, device=dev, requires_grad=True)
        q, k, v = split_qkv_rotary(x, 2, axes, pos, transpose_v=transpose_v)
        v.sum().backward()                      # dv expanded from one number, dq and dk absent
        g = x.grad.reshape(2, 10, 3, 16)
        assert not g[:, :, :2].any() and bool((g[:, :, 2] == 1).all())
        x.grad = None
        q, k, v = split_qkv_rotary(x, 2, axes, pos, transpose_v=transpose_v)
        w = torch.randn(2, 8, 10, 2, device=dev)
        (q * w.permute(0, 3, 2, 1)).sum().backward()
        head = x.grad.reshape(2, 10, 6, 8).transpose(1, 2)[:, :2]
        close(head, *rotate64(w.permute(0, 3, 2, 1), [4, 4], pos, 10000.0, [1, 1], False, -1))


@pytest.mark.gpu
def test_gradient_against_differences(cuda_device):
    """The map is linear: the difference along a direction is the map itself,
    up to the rounding of two outputs (2 x 4 2^-24 of their magnitude, over 2e
    with e = 1)."""
    dev = cuda_device
    axes = RotaryAxes([6, 2], [4, 4], device=dev)
    pos = positions((4, 4)).to(dev)
    x = torch.randn(1, 17, 3 * 2 * 8, device=dev, requires_grad=True)
    outs = split_qkv_rotary(x, 2, axes, pos)
    cs = [torch.randn_like(o) for o in outs]
    (grad,) = torch.autograd.grad(outs, (x,), cs)
    d = torch.randn_like(x)
    side = []
    for s in (1, -1):
        moved = split_qkv_rotary(x.detach() + s * d, 2, axes, pos)
        side.append(sum((c.double() * o.double()).sum() for c, o in zip(cs, moved)))
    size = sum((c.abs().double() * 6 * o.detach().abs().double().amax()).sum()
               for c, o in zip(cs, outs))
    assert abs((side[0] - side[1]) / 2 - (grad.double() * d.double()).sum()) <= 8 * U * size


@pytest.mark.gpu
def test_python_refusals(cuda_device):
    dev = cuda_device
    axes = RotaryAxes([8, 8], [4, 4], device=dev)
    x = torch.zeros(1, 4, 3 * 2 * 16, device=dev)
    pos = torch.zeros(4, 2, dtype=torch.int32, device=dev)
    for args, kw, msg in (((x, 4, axes, pos), dict(num_kv_heads=3), "multiple"),
                          ((x[0], 2, axes, pos), {}, "must be"),
                          ((x, 5, axes, pos), {}, "must be"),
                          ((x, 8, axes, pos), {}, "axes' dims"),
                          ((x, 2, axes, pos.long()), {}, "pos must"),
                          ((x, 2, axes, pos[:3]), {}, "pos must"),
                          ((x, 2, axes, pos.cpu()), {}, "pos must"),
                          ((x, 2, RotaryAxes([8, 8], [4, 4]), pos), {}, "axes are on")):
        with pytest.raises(ValueError, match=msg):
            split_qkv_rotary(*args, **kw)
    with pytest.raises(TypeError, match="float32"):
        split_qkv_rotary(x.double(), 2, axes, pos)


def test_sc_attention_leaves_a_foreign_rope_alone():
    """Attention modules of other models keep an embedding, a function or a flag
    under that name and turn q and k themselves, or elsewhere."""
    class Attn(torch.nn.Module):
        def __init__(self, rope):
            super().__init__()
            self.num_heads, self.scale, self.rope = 2, 0.5, rope
            self.qkv, self.proj = torch.nn.Linear(8, 24), torch.nn.Linear(8, 8)
            self.proj_drop = torch.nn.Identity()

    x = torch.randn(2, 3, 8, generator=torch.Generator().manual_seed(1))
    forward = make_sc_attention_forward(8, False, sc_qk=False)
    torch.manual_seed(0)
    want = forward(Attn(None), x)
    for rope in (lambda q: q, True, torch.nn.Embedding(3, 4), "axial"):
        torch.manual_seed(0)
        m = Attn(None)
        m.rope = rope
        assert torch.equal(forward(m, x), want)


def test_sc_attention_refuses_positions_on_the_cpu():
    torch.manual_seed(0)
    from scmp_vit_b200.vit import Attention
    m = Attention(8, 2)
    m.rope = GridRotary((1, 2), 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        make_sc_attention_forward(8, False, sc_qk=False)(m, torch.zeros(2, 3, 8))


# ------------------------------------- the variants that large calls take

LARGE = [  # B, H, Hk, D, dims, grid: a thread walks three heads or more, in batches of four
    (16, 16, 16, 64, [32, 32], (16, 16)),
    (24, 12, 4, 64, [16, 24, 24], (3, 9, 9)),
    (120, 5, 5, 40, [20, 20], (13, 15)),
    (16, 10, 2, 128, [44, 42, 42], (4, 8, 9)),
    (30, 7, 7, 34, [30], (200,)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("case", range(len(LARGE)))
def test_values_and_gradient_of_many_tokens(cuda_device, case, interleaved):
    B, H, Hk, D, dims, grid = LARGE[case]
    dev = cuda_device
    pos = positions(grid, 1).to(dev)
    N = pos.shape[0]
    # the heads that one thread takes with the widest pieces, v in blocks of its own
    widest = next(v for v in (8, 4, 2) if D % v == 0)
    assert (H + Hk) * (B * N * (D // widest) // 256) // (148 * 6) >= 3
    scales = [1.0, 0.5, 2.0][:len(dims)]
    axes = RotaryAxes(dims, grid, base=1000.0, scales=scales, interleaved=interleaved, device=dev)
    for dtype in DTYPES:
        g = torch.Generator().manual_seed(case)
        qkv = torch.randn(B, N, (H + 2 * Hk) * D, generator=g).to(dtype).to(dev).requires_grad_()
        heads = qkv.detach().reshape(B, N, H + 2 * Hk, D).transpose(1, 2)
        want = rotate64(heads[:, :H + Hk], dims, pos, 1000.0, scales, interleaved)
        grad = torch.randn(heads.shape, generator=g).to(dtype).to(dev)
        back = rotate64(grad[:, :H + Hk], dims, pos, 1000.0, scales, interleaved, -1)
        for transpose_v in (True, False):
            q, k, v = split_qkv_rotary(qkv, H, axes, pos, num_kv_heads=Hk, transpose_v=transpose_v)
            close(torch.cat([q, k], 1).detach(), *want)
            assert torch.equal(v, heads[:, H + Hk:])
            dv = grad[:, H + Hk:]
            if transpose_v:
                dv = dv.transpose(-1, -2).contiguous().transpose(-1, -2)
            (dqkv,) = torch.autograd.grad((q, k, v), (qkv,), (grad[:, :H], grad[:, H:H + Hk], dv))
            dqkv = dqkv.reshape(B, N, H + 2 * Hk, D).transpose(1, 2)
            close(dqkv[:, :H + Hk], *back)
            assert torch.equal(dqkv[:, H + Hk:], dv)
