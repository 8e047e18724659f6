"""The fused fp32 block glue passes raw pointers to kernels that read fp32 rows
of one shape: other operands are refused, and a block whose branch comes in
another type adds it the ordinary way.  The library call is replaced on the
CPU, so nothing here reads memory that it should not."""
import pytest
import torch

from scmp_vit_b200 import _lib, attention, vit


class Recorder:
    """Stands for the library: keeps its calls' names and device indices."""

    def __init__(self):
        self.made = []

    def __getattr__(self, name):
        return name

    @property
    def calls(self):
        return len(self.made)


@pytest.fixture
def lib(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(_lib, "load", lambda: rec)
    for module in (vit, attention):
        monkeypatch.setattr(module, "call", lambda fn, index, *args: rec.made.append((fn, index)))
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    return rec


X, G = torch.zeros(2, 3, 8), torch.ones(8)


@pytest.mark.parametrize("kw", [
    dict(x=X.bfloat16()), dict(y=X.bfloat16()), dict(gamma=G.bfloat16()), dict(y=X[:1]),
    dict(y=X[..., :4]), dict(y=torch.zeros(3, 2, 8).transpose(0, 1)), dict(gamma=G[:4]),
    dict(gamma=torch.ones(16)[::2]), dict(bias=G.half()), dict(bias=torch.ones(1)),
    dict(extra=X.double()), dict(extra=X[:1]), dict(out=X.half()), dict(out=X[:1]),
    dict(y=torch.zeros(2, 3, 8, device="meta")), dict(x=torch.zeros(2, 3, 8)[..., ::2]),
])
def test_scale_residual_refuses(lib, kw):
    args = dict(x=X, y=X.clone(), gamma=G)
    args.update(kw)
    with pytest.raises((TypeError, ValueError)):
        vit.scale_residual(**args)
    assert lib.calls == 0


@pytest.mark.parametrize("t,bias", [
    (X.bfloat16(), G), (X, G.bfloat16()), (X, G[:4]), (X.transpose(0, 1), G), (X, X)])
def test_bias_gelu_refuses(lib, t, bias):
    with pytest.raises((TypeError, ValueError)):
        vit.bias_gelu_(t, bias)
    assert lib.calls == 0


def small(**kw):
    m = vit.vit_l14(seed=0, dim=32, depth=1, heads=2, hidden=64, img=28, **kw).eval()
    return m, m.backbone.blocks[0]


class Bf16Branch(torch.nn.Module):
    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x):
        return self.inner(x).bfloat16()


def test_calls_go_to_their_tensors_device(lib, monkeypatch):
    """On the default stream, whose handle every device shares, a launch on the
    current device would be given another device's memory."""
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 3)
    vit.scale_residual(X, X.clone(), G)
    vit.bias_gelu_(X.clone(), G)
    attention.split_qkv(torch.zeros(2, 3, 24), 2)
    assert lib.made == [("scmp_scale_residual", 3), ("scmp_bias_gelu", 3), ("scmp_split_qkv", 3)]


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU path"):
        vit.scale_residual(X, X, G)
    with pytest.raises(RuntimeError, match="no CPU path"):
        vit.bias_gelu_(X, G)
    with pytest.raises(RuntimeError):  # (a machine without a GPU says so itself)
        attention.split_qkv(torch.zeros(2, 3, 24), 2)


@pytest.mark.parametrize("where", ["attn", "mlp", "both"])
def test_fused_glue_adds_a_16_bit_branch_as_torch_does(lib, where):
    """The kernels would read a 16-bit branch as twice its bytes."""
    _, blk = small()
    if where in ("attn", "both"):
        blk.attn = Bf16Branch(blk.attn)
    if where in ("mlp", "both"):
        blk.mlp = Bf16Branch(blk.mlp)
    x = torch.randn(2, 5, 32, generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        if where == "both":
            assert torch.equal(blk._forward_fused_glue(x), blk(x)) and lib.calls == 0
        else:  # the fp32 branch still goes to the library, the other does not
            blk._forward_fused_glue(x)
            assert lib.calls == 1 + (where == "attn")


def test_fused_glue_does_not_apply_under_autocast_or_to_16_bit_scales(monkeypatch):
    _, blk = small()
    x = torch.zeros(1, 5, 32)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    with torch.no_grad():
        assert blk._fused_glue_applies(x)
        torch.set_autocast_enabled("cuda", True)
        try:
            assert not blk._fused_glue_applies(x)
        finally:
            torch.set_autocast_enabled("cuda", False)
        blk.ls2.gamma.data = blk.ls2.gamma.data.bfloat16()
        assert not blk._fused_glue_applies(x)


@pytest.mark.gpu
def test_autocast_gives_the_unfused_bits(cuda_device):
    m, _ = small()
    m = m.to(cuda_device)
    x = torch.randn(2, 3, 28, 28, generator=torch.Generator().manual_seed(2)).to(cuda_device)
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
        got = m(x)
        vit.set_fused_glue(False)
        try:
            want = m(x)
        finally:
            vit.set_fused_glue(True)
    assert torch.equal(got, want) and bool(got.isfinite().all())
