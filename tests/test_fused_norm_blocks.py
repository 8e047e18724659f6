"""Which forward a block takes with fused norms, on the CPU: ``residual_norm``
is replaced by its formula and CPU tensors pass for CUDA ones."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
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


def patched(monkeypatch):
    """Every linear in 4 bits, as modules that take values and codes alike."""
    blk, x = block()

    class Linear4(torch.nn.Linear):
        fmt = "mxfp4"

    monkeypatch.setattr(vit, "MXLinear", Linear4)
    for owner, name in ((blk.attn, "qkv"), (blk.mlp, "fc1")):
        getattr(owner, name).__class__ = Linear4
    return blk, x


def test_hooks_see_every_module_they_watch(calls):
    """A block whose norms or layer scale are watched calls them as modules."""
    blk, x = block()
    with torch.no_grad():
        want = blk(x)
        assert calls == [None, None]
        for m in (blk.norm1, blk.norm2, blk.ls1):
            for register in ("register_forward_hook", "register_forward_pre_hook"):
                fired = []
                handle = getattr(m, register)(lambda *a: fired.append(1))
                assert torch.equal(blk(x), want) and fired == [1]
                handle.remove()
        fired = []
        handle = torch.nn.modules.module.register_module_forward_hook(
            lambda m, *a: fired.append(m))
        blk(x)
        handle.remove()
        assert {blk.norm1, blk.norm2, blk.ls1} <= set(fired)
    assert calls == [None, None]
    fired = []
    handle = blk.norm2.register_full_backward_hook(lambda *a: fired.append(1))
    blk(x.requires_grad_()).sum().backward()
    handle.remove()
    assert fired == [1] and calls == [None, None]


def test_codes_only_where_nobody_watches(calls, monkeypatch):
    blk, x = patched(monkeypatch)
    with torch.no_grad():
        blk(x)
        assert calls == ["mxfp4", "mxfp4"]
        for m, want in ((blk.attn, [None, "mxfp4"]), (blk.attn.qkv, [None, "mxfp4"]),
                        (blk.mlp, ["mxfp4", None]), (blk.mlp.fc1, ["mxfp4", None])):
            for register in ("register_forward_hook", "register_forward_pre_hook"):
                del calls[:]
                fired = []
                handle = getattr(m, register)(lambda m, a, *out: fired.append(type(a[0])))
                blk(x)
                handle.remove()
                assert calls == want and fired == [torch.Tensor]
        del calls[:]
        blk(x)
        assert calls == ["mxfp4", "mxfp4"]


@pytest.mark.parametrize("glue", [False, True])
def test_forward_mode_takes_the_separate_modules(calls, monkeypatch, glue):
    """The fused steps have no forward-mode derivative; a block under one, or with
    a dual parameter, is differentiated as the modules are."""
    monkeypatch.setattr(vit, "FUSED_GLUE", glue)
    monkeypatch.setattr(vit, "FUSED_NORM", not glue)
    monkeypatch.setattr(vit, "call", lambda *a: calls.append(a))
    blk, x = block()
    blk.attn = torch.nn.Linear(32, 32)
    t = torch.randn(x.shape, generator=torch.Generator().manual_seed(2))
    with torch.no_grad(), fwAD.dual_level():
        got = fwAD.unpack_dual(blk(fwAD.make_dual(x, t))).tangent
        scaled = torch.func.functional_call(
            blk, {"ls1.gamma": fwAD.make_dual(blk.ls1.gamma.detach(), torch.ones(32))}, (x,))
        assert fwAD.unpack_dual(scaled).tangent is not None
    assert calls == []
    e = 2.0 ** -10
    with torch.no_grad():
        monkeypatch.setattr(vit, "FUSED_GLUE", False)
        monkeypatch.setattr(vit, "FUSED_NORM", False)
        diff = (blk.double()(x.double() + e * t) - blk(x.double() - e * t)) / (2 * e)
    # differences are off by e^2 times the third derivative, of the order of the values
    assert (got - diff).abs().max() <= 100 * e * e * diff.abs().max()
