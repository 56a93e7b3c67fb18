"""The 4-bit products have no gradient: a backward pass that reaches one fails and is not cut off in silence."""
import pytest
import torch

from test_gpu_w4 import layer, routing, weights

pytestmark = pytest.mark.gpu
H, I, E = 128, 64, 4


def _experts(pkg, x, idx, w, l13, l2, **kw):
    return pkg.experts_w4(x, idx, w, l13[0], l13[1], l2[0], l2[1], group=32, **kw)


@pytest.mark.parametrize("T", [3, 40])
def test_linear(pkg, T):
    codes, scale, _ = weights((), 96, H, 32, False, torch.bfloat16, 1)
    x = torch.randn((T, H), device="cuda").to(torch.bfloat16)
    plain = pkg.linear_w4(x, codes, scale, group=32)
    assert not plain.requires_grad
    for leaf in ("x", "scale"):
        a = dict(x=x, codes=codes, scale=scale)
        a[leaf] = a[leaf].clone().requires_grad_()
        y = pkg.linear_w4(**a, group=32)
        assert y.requires_grad and torch.equal(y, plain)
        with pytest.raises(RuntimeError, match="linear_w4 has no gradient"):
            (y.float().sum() + a[leaf].float().sum()).backward()
        with pytest.raises(RuntimeError, match="out"):
            pkg.linear_w4(**a, group=32, out=torch.empty_like(plain))
        with torch.no_grad():
            assert not pkg.linear_w4(**a, group=32).requires_grad


@pytest.mark.parametrize("T", [3, 40])
def test_experts_and_a_gate_behind_them(pkg, T):
    l13, l2 = layer(E, H, I, 32, False, torch.bfloat16, 3)
    x = torch.randn((T, H), device="cuda").to(torch.bfloat16)
    idx, w = routing(T, E, 2, 1)
    plain = _experts(pkg, x, idx, w, l13, l2)
    assert not plain.requires_grad
    for args in ((x.clone().requires_grad_(), idx, w, l13, l2), (x, idx, w.clone().requires_grad_(), l13, l2),
                 (x, idx, w, (l13[0], l13[1].clone().requires_grad_()), l2), (x, idx, w, l13, (l2[0], l2[1].clone().requires_grad_()))):
        y = _experts(pkg, *args)
        assert torch.equal(y, plain)
        with pytest.raises(RuntimeError, match="experts_w4 has no gradient"):
            y.float().sum().backward()
        with pytest.raises(RuntimeError, match="out"):
            _experts(pkg, *args, out=torch.empty_like(plain))
        with torch.no_grad():
            assert not _experts(pkg, *args).requires_grad
    # A gate whose gradient would have to come through the experts, next to a path that has one.
    gate = torch.randn((E, H), device="cuda").requires_grad_()
    idx, w = pkg.route_experts(x.float() @ gate.T, 2)
    out = _experts(pkg, x, idx, w, l13, l2).float() + (x.float() @ gate.T).sum()
    with pytest.raises(RuntimeError, match="experts_w4 has no gradient"):
        out.sum().backward()
    assert not _experts(pkg, x, idx, w.detach(), l13, l2).requires_grad
