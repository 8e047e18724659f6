"""Which forward a block takes with fused norms, on the CPU: ``residual_norm``
is replaced by its formula and CPU tensors pass for CUDA ones."""
import pytest
import torch
import torch.nn.functional as F

from scmp_vit_b200 import vit


@pytest.fixture
def calls(monkeypatch):
    seen = []

    def stand_in(x, y, weight, norm_bias=None, *, eps, gamma=None, quantize=None):
        seen.append(quantize)
        r = x if y is None else x + y * gamma
        return r, F.layer_norm(r, x.shape[-1:], weight, norm_bias, eps)

    monkeypatch.setattr(vit, "residual_norm", stand_in)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(vit, "FUSED_GLUE", False)
    monkeypatch.setattr(vit, "FUSED_NORM", True)
    return seen


def block():
    m = vit.vit_l14(seed=0, dim=32, depth=1, heads=2, hidden=64, img=28).eval()
    return m.backbone.blocks[0], torch.randn(2, 5, 32, generator=torch.Generator().manual_seed(1))


def test_attention_without_a_qkv_linear(calls):
    """A block whose attention was replaced by one of another make."""
    class Other(torch.nn.Module):
        def forward(self, x):
            return x * 2

    blk, x = block()
    blk.attn = Other()
    with torch.no_grad():
        y = x + blk.ls1(blk.attn(blk.norm1(x)))
        want = y + blk.ls2(blk.mlp(blk.norm2(y)))
        assert torch.equal(blk(x), want)
    assert calls == [None, None]
