"""Forward-mode derivatives: the block operators have none and say so.  A dual
tensor has no ``requires_grad``, so a call that looked at that alone would
return values without a tangent, i.e. a derivative of zero.  CUDA tensors are
played by CPU ones and the launches replaced, since nothing may get that far."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from scmp_vit_b200 import attention, mx, vit
from scmp_vit_b200._call import has_tangent


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    launched = []
    for module in (attention, mx, vit):
        monkeypatch.setattr(module, "call", lambda *a: launched.append(a))
    return launched


def dual(t):
    return fwAD.make_dual(t, torch.ones_like(t))


X, W = torch.randn(2, 3, 32), torch.ones(32)
NORM = dict(x=X, y=X.clone(), weight=W, norm_bias=W.clone(), gamma=W.clone(),
            gate=torch.ones(2, 32), post_weight=W.clone(), post_bias=W.clone())


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("leaf", list(NORM))
def test_residual_norm(no_launch, leaf, grad):
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        t = dict(NORM, **{leaf: dual(NORM[leaf])})
        with pytest.raises(NotImplementedError, match="jvp"):
            vit.residual_norm(**t)
        with pytest.raises(RuntimeError, match="no gradient"):
            vit.residual_norm(**t, quantize="mxfp4")


@pytest.mark.parametrize("grad", [True, False])
def test_split_qkv_rotary(no_launch, grad):
    axes = attention.RotaryAxes([8, 8], [4, 4])
    pos = torch.zeros(3, 2, dtype=torch.int32)
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError, match="jvp"):
            attention.split_qkv_rotary(dual(torch.randn(2, 3, 96)), 2, axes, pos)


@pytest.mark.parametrize("grad", [True, False])
def test_quantise_and_product(no_launch, grad):
    w = mx.mx_empty(torch.Size((16, 32)), "mxfp4", torch.device("cpu"), torch.float32)
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(RuntimeError, match="no gradient"):
            mx.mx_quantize(dual(X))
        for kw in (dict(a=dual(X)), dict(a=X, bias=dual(torch.zeros(16))),
                   dict(a=X, out=dual(torch.zeros(2, 3, 16)))):
            with pytest.raises(RuntimeError, match="no gradient"):
                mx.mx_matmul(b=w, **kw)
    assert no_launch == []


def test_values_of_dual_tensors_are_taken(no_launch):
    """The primal, or a tensor whose level has ended, is a value like others."""
    with fwAD.dual_level():
        d = dual(X)
        assert not has_tangent((None, fwAD.unpack_dual(d).primal, X)) and has_tangent((X, d))
    assert not has_tangent((d,))
