"""The 8-bit linears, the norms of queries and keys and the dropout together, in the
model that uses them: a block's forward and gradients bit for bit those of the same
calls one by one, served and trained, eager and captured."""
import copy

import pytest
import torch
import torch.nn.functional as F

from scmp_vit_b200 import fp8, vit
from scmp_vit_b200.attention import split_qkv_norm


def small(dev, dtype=torch.float32, **kw):
    m = vit.vit_l14(seed=0, dim=128, depth=2, heads=2, hidden=256, img=56, rope=True,
                    qk_norm="rms", **kw)
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
        vit.patch_vit_fp8(vit.vit_l14(dim=64, depth=1, heads=1, hidden=64, img=28), ("qk",))


def test_trained_modules_keep_the_parameters():
    m = vit.vit_l14(dim=64, depth=2, heads=1, hidden=64, img=28)
    before = {n: id(p) for n, p in m.named_parameters()}
    assert vit.patch_vit_fp8(m, ("qkv_proj", "mlp_fc2"), train=True) == {
        "qkv_proj": 2, "out_proj": 0, "mlp_fc1": 0, "mlp_fc2": 2}
    assert {n: id(p) for n, p in m.named_parameters()} == before
    assert type(m.backbone.blocks[0].attn.qkv) is fp8.FP8Linear
    m.load_state_dict(vit.vit_l14(seed=1, dim=64, depth=2, heads=1, hidden=64, img=28).state_dict())
    assert all(type(lin) is torch.nn.Linear for b in m.backbone.blocks
               for lin in (b.attn.proj, b.mlp.fc1))


def block_by_calls(blk, x, drops=None):
    """A patched block from the public calls; drops: (p, rate, seed, offsets of
    projection, MLP and both branches)."""
    B, N, C = x.shape
    a, n = blk.attn, blk.attn.qk_norm

    def linear(lin, t):
        if lin.trained:
            return fp8.fp8_linear(t, lin.weight, lin.bias)
        return fp8.fp8_matmul(t, lin.quantized_weight(), bias=lin.bias)

    def add(t, branch, i):
        if drops is None:
            return t + branch
        return vit.dropout(branch, drops[1], drops[2], drops[3][i], per="sample", residual=t)

    def drop(t, i):
        return t if drops is None else vit.dropout(t, drops[0], drops[2], drops[3][i])
    q, k, v = split_qkv_norm(linear(a.qkv, blk.norm1(x)), a.num_heads, n.q_weight, n.k_weight,
                             eps=n.eps, axes=a.rope.axes, pos=a.rope.pos, transpose_v=False)
    o = F.scaled_dot_product_attention(q, k, v).transpose(1, 2).reshape(B, N, C)
    y = add(x, blk.ls1(drop(linear(a.proj, o), 0)), 2)
    u = linear(blk.mlp.fc2, blk.mlp.act(linear(blk.mlp.fc1, blk.norm2(y))))
    return add(y, blk.ls2(drop(u, 1)), 3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_served_block(cuda_device, dtype):
    m = small(cuda_device, dtype)
    ref = m.backbone.blocks[1]
    x = torch.randn(3, 17, 128, device=cuda_device).to(dtype)
    with torch.no_grad():
        plain = ref(x)
        assert vit.patch_vit_fp8(m)["mlp_fc1"] == 2
        blk = m.backbone.blocks[1]
        vit.set_fused_glue(False)
        try:
            got = blk(x)
            assert torch.equal(got, block_by_calls(blk, x))
        finally:
            vit.set_fused_glue(True)
        # (the fused glue rounds the fp32 steps as torch does)
        assert torch.equal(blk(x), got)
        # every product's operands are off by at most 2^-4: of the branches' size
        scale = (plain - x).float().abs().max()
        assert float((got - plain).float().abs().max()) < 0.5 * float(scale)
        again = small(cuda_device, dtype)
        vit.patch_vit_fp8(again)
        again.load_state_dict(copy.deepcopy(m.state_dict()))
        images = torch.randn(2, 3, 56, 56, device=cuda_device).to(dtype)
        assert torch.equal(again(images), m(images))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_trained_block(cuda_device, dtype):
    """Forward and every gradient of a block in training mode, with dropout and
    stochastic depth."""
    m = small(cuda_device, dtype)
    vit.patch_vit_fp8(m, train=True)
    vit.set_dropout(m, 0.2, 0.4, seed=5)
    m.train()
    blk = m.backbone.blocks[1]
    x = torch.randn(4, 17, 128, device=cuda_device).to(dtype).requires_grad_()
    dy = torch.randn(4, 17, 128, device=cuda_device).to(dtype)
    params = [x, *blk.parameters()]
    got = blk(x)
    grads = torch.autograd.grad(got, params, dy)
    drops = (0.2, 0.4, 5, (3 << 48, 4 << 48, 5 << 48, (5 << 48) + 1))
    want = block_by_calls(blk, x, drops)
    assert torch.equal(got, want)
    for a, b in zip(grads, torch.autograd.grad(want, params, dy)):
        assert torch.equal(a, b) and bool(a.isfinite().all())
    assert not torch.equal(blk(x), got)  # (the next masks)


@pytest.mark.gpu
def test_gradient_is_the_plain_model_s_up_to_8_bits(cuda_device):
    """Against the same model without 8 bits: each gradient within a quarter of the
    plain one's norm (codes are off by at most 2^-4 and on average by a third of
    that, over the dozen operands on the way)."""
    m = small(cuda_device)
    p = copy.deepcopy(m)
    vit.patch_vit_fp8(m, train=True)
    images = torch.randn(4, 3, 56, 56, device=cuda_device)
    for model in (m, p):
        model(images).square().sum().backward()
    for (name, a), b in zip(m.named_parameters(), p.parameters()):
        if b.grad is not None and float(b.grad.norm()) > 1e-6:
            assert float((a.grad - b.grad).norm()) < 0.25 * float(b.grad.norm()), name


@pytest.mark.gpu
def test_training_steps_captured(cuda_device):
    """A whole step, optimizer included, replayed: masks of its own in every replay,
    the eager model's updates where nothing is dropped."""
    dev = cuda_device
    images = torch.randn(2, 3, 56, 56, device=dev)
    m = small(dev)
    vit.patch_vit_fp8(m, train=True)
    m.train()
    other = copy.deepcopy(m)
    loss_of = lambda model: model(images).square().mean()  # noqa: E731

    def step(model):
        leaves = [q for q in model.parameters() if q.requires_grad]
        loss = loss_of(model)
        grads = torch.autograd.grad(loss, leaves, allow_unused=True)
        with torch.no_grad():
            for q, gr in zip(leaves, grads):
                if gr is not None:
                    q.sub_(1e-3 * gr)
        return loss.detach()
    start = {n: q.detach().clone() for n, q in m.named_parameters()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(m)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step(m)
    with torch.no_grad():
        for n, q in m.named_parameters():
            q.copy_(start[n])
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, step(other))
    for a, b in zip(m.parameters(), other.parameters()):
        assert torch.equal(a, b)
    vit.set_dropout(m, 0.3, seed=1)
    m.train()
    with torch.cuda.stream(side):
        m(images)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        out = m(images)
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        seen.append(out.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


@pytest.mark.gpu
def test_autocast_and_hooks(cuda_device):
    """Under autocast the 8-bit linears take what comes (fp32 behind a norm, 16 bits
    behind attention) and gradients reach every parameter; hooks see their calls."""
    m = small(cuda_device)
    vit.patch_vit_fp8(m, train=True)
    vit.set_dropout(m, 0.1, 0.2, seed=2)
    m.train()
    seen = []
    h = m.backbone.blocks[0].attn.qkv.register_forward_hook(lambda mod, i, o: seen.append(o.dtype))
    images = torch.randn(3, 3, 56, 56, device=cuda_device)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = m(images).float().square().mean()
    loss.backward()
    h.remove()
    assert len(seen) == 1
    assert all(p.grad is not None and bool(p.grad.isfinite().all())
               for p in m.backbone.blocks.parameters())


@pytest.mark.gpu
def test_threads_and_streams(cuda_device):
    """Two threads with streams of their own give the bits of one."""
    import threading
    m = small(cuda_device)
    vit.patch_vit_fp8(m, train=True)
    images = [torch.randn(2, 3, 56, 56, device=cuda_device) for _ in range(2)]
    params = list(m.backbone.blocks.parameters())

    def step(x):
        return torch.autograd.grad(m(x).square().sum(), params)
    want = [step(x) for x in images]
    got = [None, None]

    def work(i):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                got[i] = step(images[i])
        s.synchronize()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
