"""The 4-bit block operators in the model that uses them: rotary positions,
residual adds with their norms and 4-bit linears in a small ViT, bit for bit
against the same calls made one by one, and the fused norms' training step
against 64 bits."""
import copy
import pickle
import threading

import pytest
import torch
import torch.nn.functional as F

from scmp_vit_b200 import mx, vit
from scmp_vit_b200.attention import GridRotary, make_sc_attention_forward

U = 2.0 ** -24


def small(dev, dtype=torch.float32, **kw):
    m = vit.vit_l14(seed=0, dim=128, depth=2, heads=2, hidden=256, img=56, **kw)
    g = torch.Generator().manual_seed(1)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if name.endswith("gamma") or "norm" in name:
                p.add_(0.2 * torch.randn(p.shape, generator=g))
            elif name.endswith("bias"):
                p.add_(0.05 * torch.randn(p.shape, generator=g))
    return m.to(dev, dtype)


def test_patch_refuses_unknown_ops():
    with pytest.raises(ValueError, match="unknown ops"):
        vit.patch_vit_mx(vit.vit_l14(dim=64, depth=1, heads=1, hidden=64, img=28), ("qk",))


def test_grid_positions():
    g = GridRotary((2, 3), 20, prefix=2)
    assert g.axes.dims == [10, 10] and g.axes.sizes == [2, 3]
    assert g.pos.tolist() == [[-1, -1], [-1, -1], [0, 0], [0, 1], [0, 2], [1, 0], [1, 1], [1, 2]]
    assert not g.state_dict()


def block_by_calls(blk, x):
    """A patched block from the public calls, one operator at a time."""
    dt = x.dtype
    _, h = vit.residual_norm(x, None, blk.norm1.weight, blk.norm1.bias, eps=blk.norm1.eps,
                             quantize=blk.attn.qkv.fmt)
    qkv = mx.mx_matmul(h, blk.attn.qkv.quantized_weight(), bias=blk.attn.qkv.bias)
    B, N, C = x.shape
    q, k, v = vit.GridRotary.split(blk.attn.rope, qkv, blk.attn.num_heads, transpose_v=False)
    a = F.scaled_dot_product_attention(q, k, v).transpose(1, 2).reshape(B, N, C)
    a = mx.mx_matmul(a, blk.attn.proj.quantized_weight(), bias=blk.attn.proj.bias)
    y, h = vit.residual_norm(x, a, blk.norm2.weight, blk.norm2.bias, eps=blk.norm2.eps,
                             gamma=blk.ls1.gamma, quantize=blk.mlp.fc1.fmt)
    t = F.gelu(mx.mx_matmul(h, blk.mlp.fc1.quantized_weight(), bias=blk.mlp.fc1.bias))
    u = mx.mx_matmul(t, blk.mlp.fc2.quantized_weight(), bias=blk.mlp.fc2.bias)
    assert u.dtype == dt
    return y + u * blk.ls2.gamma


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_patched_model_is_its_calls(cuda_device, fmt, dtype):
    m = small(cuda_device, dtype, rope=True)
    stats = vit.patch_vit_mx(m, fmt=fmt)
    assert all(n == 2 for n in stats.values())
    x = torch.randn(3, 3, 56, 56, generator=torch.Generator().manual_seed(2)).to(cuda_device, dtype)
    with torch.no_grad():
        got = m(x)
        bb = m.backbone
        t = bb.patch_embed(x).flatten(2).transpose(1, 2)
        t = torch.cat([bb.cls_token.expand(3, -1, -1), t], dim=1) + bb.pos_embed
        for blk in bb.blocks:
            t = block_by_calls(blk, t)
        t = bb.norm(t)
        ref = m.linear_head(torch.cat([t[:, 0], t[:, 1:].mean(dim=1)], dim=-1))
    assert torch.equal(got, ref)


@pytest.mark.gpu
def test_linears_alone_and_beside_sc(cuda_device):
    """Some linears in 4 bits, the attention through SC, positions on."""
    for ops in (("mlp_fc1",), ("qkv_proj", "mlp_fc2"), vit.MX_OPS):
        m = small(cuda_device, rope=True)
        vit.patch_vit(m, 8, ("qk", "av"))
        vit.patch_vit_mx(m, ops)
        check_beside_sc(m, cuda_device)


def check_beside_sc(m, cuda_device):
    x = torch.randn(2, 3, 56, 56, generator=torch.Generator().manual_seed(3)).to(cuda_device)
    with torch.no_grad():
        a, b = m(x), m(x)
    assert torch.equal(a, b) and bool(a.isfinite().all())
    # the SC attention turns q and k: positions change its result
    for blk in m.backbone.blocks:
        blk.attn.rope = None
    with torch.no_grad():
        assert not torch.equal(m(x), a)


@pytest.mark.gpu
def test_sc_attention_with_positions(cuda_device):
    """The SC forward on turned q and k equals the one that gets them turned."""
    m = small(cuda_device, rope=True)
    attn = m.backbone.blocks[0].attn
    x = torch.randn(2, 17, 128, device=cuda_device)
    with torch.no_grad():
        got = make_sc_attention_forward(8, True)(attn, x)
        plain = copy.deepcopy(attn)
        plain.rope = None
        q, k, v = attn.rope.split(attn.qkv(x), 2)
        turned = torch.stack([q, k, v], 2).permute(0, 3, 2, 1, 4).reshape(2, 17, -1).contiguous()

        class Given(torch.nn.Module):
            def forward(self, _):
                return turned

        plain.qkv = Given()
        want = make_sc_attention_forward(8, True)(plain, x)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_mx_model_in_a_graph(cuda_device):
    m = small(cuda_device, torch.bfloat16, rope=True)
    vit.patch_vit_mx(m)
    x = torch.randn(2, 3, 56, 56, device=cuda_device).bfloat16()
    with torch.no_grad():
        m(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(x)
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, m(x))


@pytest.mark.gpu
def test_4bit_linears_refuse_training(cuda_device):
    m = small(cuda_device)
    vit.patch_vit_mx(m)
    with pytest.raises(RuntimeError, match="no gradient"):
        m(torch.randn(1, 3, 56, 56, device=cuda_device))


@pytest.mark.gpu
def test_training_step_against_64_bits(cuda_device):
    """Loss gradients of a fp32 model with positions and fused norms against
    the plain modules in 64 bits.  Some 40 operators lie between a parameter and
    the loss, each off by at most (C + 16) 2^-24 of its magnitude with C = 256
    its longest sum: 6.5e-4 of the largest gradient of a tensor."""
    m = small(cuda_device, rope=True).train()
    ref = copy.deepcopy(m).double()
    x = torch.randn(2, 3, 56, 56, generator=torch.Generator().manual_seed(4)).to(cuda_device)
    target = torch.randn(2, 1000, generator=torch.Generator().manual_seed(5)).to(cuda_device)

    class Turn:  # the positions in 64 bits
        def __init__(self, rope):
            self.rope = rope

        def split(self, qkv, H, transpose_v=True):
            B, N, C3 = qkv.shape
            D = C3 // (3 * H)
            q, k, v = qkv.reshape(B, N, 3, H, D).permute(2, 0, 3, 1, 4)
            pos, d = self.rope.pos.clamp(min=0).double(), self.rope.axes.dims[0]
            freq = 10000.0 ** (-torch.arange(0, d, 2, device=qkv.device).double() / d)
            angle = torch.cat([pos[:, :1] * freq, pos[:, 1:] * freq], -1)

            def turn(t):
                u, w = t[..., 0::2], t[..., 1::2]
                return torch.stack([u * angle.cos() - w * angle.sin(),
                                    w * angle.cos() + u * angle.sin()], -1).flatten(-2)

            return turn(q), turn(k), v

    for blk, b64 in zip(m.backbone.blocks, ref.backbone.blocks):
        rope = b64.attn.rope
        del b64.attn.rope
        b64.attn.rope = Turn(rope)
    vit.set_fused_norm(True)
    try:
        out = m(x)
        (out * target).sum().backward()
    finally:
        vit.set_fused_norm(False)
    (ref(x.double()) * target.double()).sum().backward()
    for (name, p), (_, p64) in zip(m.named_parameters(), ref.named_parameters()):
        err = (p.grad.double() - p64.grad).abs().max()
        assert err <= 40 * (256 + 16) * U * p64.grad.abs().max(), name


@pytest.mark.gpu
def test_fused_norm_off_keeps_the_bits(cuda_device):
    """Without 4-bit linears and without the switch nothing changes."""
    m = small(cuda_device)
    x = torch.randn(2, 3, 56, 56, device=cuda_device)
    with torch.no_grad():
        blk = m.backbone.blocks[0]
        t = torch.randn(2, 17, 128, device=cuda_device)
        assert not blk._fused_norm_applies(t)
        a = m(x)
        vit.set_fused_norm(True)
        try:
            b = m(x)
        finally:
            vit.set_fused_norm(False)
        assert torch.equal(m(x), a)
    # the fused norms differ in the order of their sums only (see above)
    assert (a - b).abs().max() <= 40 * (256 + 16) * U * a.abs().max()


def block_in_autocast(blk, x, ops=()):
    """A block's forward from the public calls, its branch widened to x's type."""
    def norm(n, y=None, gamma=None, fmt=None):
        return vit.residual_norm(x, y, n.weight, n.bias, eps=n.eps, gamma=gamma, quantize=fmt)

    _, h = norm(blk.norm1, fmt="mxfp4" if "qkv_proj" in ops else None)
    a = blk.attn(h)
    assert a.dtype == torch.bfloat16 and x.dtype == torch.float32
    y, h = norm(blk.norm2, a.float(), blk.ls1.gamma, "mxfp4" if "mlp_fc1" in ops else None)
    return y + blk.ls2(blk.mlp(h))


@pytest.mark.gpu
@pytest.mark.parametrize("ops", [("mlp_fc1",), ("qkv_proj", "mlp_fc2"), vit.MX_OPS])
def test_4bit_linears_under_autocast(cuda_device, ops):
    """The residual stream is fp32, the attention's output bf16."""
    m = small(cuda_device)
    vit.patch_vit_mx(m, ops)
    x = torch.randn(2, 17, 128, generator=torch.Generator().manual_seed(6)).to(cuda_device)
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
        for blk in m.backbone.blocks:
            got, want = blk(x), block_in_autocast(blk, x, ops)
            assert got.dtype == torch.float32 and torch.equal(got, want)
            x = got
        assert bool(m(torch.randn(2, 3, 56, 56, device=cuda_device)).isfinite().all())


@pytest.mark.gpu
def test_fused_norm_training_under_autocast(cuda_device):
    """The switch in mixed precision: a step's output and gradients are those of
    the calls made one by one, in the same types as without it."""
    from torch.nn.attention import SDPBackend, sdpa_kernel
    m = small(cuda_device, rope=True)
    blk = m.backbone.blocks[0]
    g = torch.Generator().manual_seed(7)
    x = torch.randn(2, 17, 128, generator=g).to(cuda_device).requires_grad_()
    t = torch.randn(2, 17, 128, generator=g).to(cuda_device)
    leaves = [x, *blk.parameters()]
    with sdpa_kernel(SDPBackend.MATH):
        with torch.autocast("cuda", torch.bfloat16):
            plain = blk(x)
            want = block_in_autocast(blk, x)
            vit.set_fused_norm(True)
            try:
                got = blk(x)
                wide = blk(x.detach().bfloat16())
            finally:
                vit.set_fused_norm(False)
        assert got.dtype == plain.dtype == wide.dtype == torch.float32
        assert torch.equal(got, want)
        grads = [torch.autograd.grad((o * t).sum(), leaves) for o in (got, want)]
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_fused_norm_beside_a_wider_branch(cuda_device):
    """A 16-bit block whose attention returns fp32 adds it as torch does."""
    class Wide(torch.nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner, self.qkv = inner, inner.qkv

        def forward(self, x):
            return self.inner(x).float()

    m = small(cuda_device, torch.bfloat16)
    blk = m.backbone.blocks[0]
    blk.attn, blk.norm2 = Wide(blk.attn), blk.norm2.float()
    blk.mlp, blk.ls1 = blk.mlp.float(), blk.ls1.float()
    x = torch.randn(2, 17, 128, device=cuda_device).bfloat16()
    with torch.no_grad():
        _, h = vit.residual_norm(x, None, blk.norm1.weight, blk.norm1.bias, eps=blk.norm1.eps)
        y = x + blk.ls1(blk.attn(h))
        want = y + blk.ls2(blk.mlp(blk.norm2(y)))
        vit.set_fused_norm(True)
        try:
            got = blk(x)
        finally:
            vit.set_fused_norm(False)
    assert got.dtype == torch.float32 and torch.equal(got, want)


def test_modules_saved_before_positions_run():
    """An attention module pickled whole by an earlier version has no ``rope``."""
    attn = vit.Attention(16, 2)
    x = torch.randn(2, 5, 16, generator=torch.Generator().manual_seed(1))
    want = attn(x)
    del attn.rope
    assert torch.equal(attn(x), want)
    assert torch.equal(pickle.loads(pickle.dumps(attn))(x), want)


@pytest.mark.gpu
def test_beside_sc_under_autocast(cuda_device):
    """4-bit linears, SC attention and fp32 linears under autocast: every branch is
    joined in the residual's type, as without the fused norms."""
    m = small(cuda_device, rope=True)
    vit.patch_vit(m, 8, ("qk", "av"))
    x = torch.randn(2, 3, 56, 56, generator=torch.Generator().manual_seed(3)).to(cuda_device)
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
        plain = m(x)
        vit.patch_vit_mx(m, ("mlp_fc1", "mlp_fc2"))
        a, b = m(x), m(x)
    assert plain.dtype == a.dtype and bool(plain.isfinite().all())
    assert torch.equal(a, b) and bool(a.isfinite().all())


@pytest.mark.gpu
def test_models_at_the_same_time(cuda_device):
    """Threads with models, formats and streams of their own, whose products, norms
    and splits share the GPU, give the bits of one thread."""
    jobs = []
    for i, (fmt, dtype) in enumerate((("mxfp4", torch.float32), ("nvfp4", torch.bfloat16),
                                      ("mxfp4", torch.bfloat16))):
        m = small(cuda_device, dtype, rope=True)
        vit.patch_vit_mx(m, fmt=fmt)
        x = torch.randn(8 * (i + 1), 3, 56, 56, device=cuda_device).to(dtype)
        with torch.no_grad():
            jobs.append((m, x, m(x)))
    torch.cuda.synchronize()
    failed = []

    def work(m, x, want):
        try:
            with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = m(x)
                    torch.cuda.current_stream().synchronize()
                    assert torch.equal(got, want)
        except BaseException as e:  # seen by the test's own thread
            failed.append(e)

    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
