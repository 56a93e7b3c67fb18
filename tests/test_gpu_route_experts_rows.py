"""The general router at rows where it is easily wrong: no expert left, scores that round together, small differences.

The gradient of a row without a pick is exactly zero: its weights are constants."""
import numpy as np
import pytest
import torch

from oracle import experts_oracle as X

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("E", [1, 60, 64, 256, 1000])
def test_gradient_of_a_row_without_experts(pkg, E, score, renormalize, dtype):
    k = min(E, 6)
    x = torch.randn((9, E), generator=torch.Generator().manual_seed(E)).to(dtype).cuda()
    x[2] = x[8] = -INF
    live = [0, 1, 3, 4, 5, 6, 7]
    g = torch.randn((9, k), generator=torch.Generator().manual_seed(1)).cuda()
    leaf = x.clone().requires_grad_()
    idx, w = pkg.route_experts(leaf, k, score=score, renormalize=renormalize, scale=1.5)
    (w * g).sum().backward()
    assert (idx[[2, 8]] == -1).all() and (w.detach()[[2, 8]] == 0).all()
    assert (leaf.grad[[2, 8]] == 0).all()
    alone = pkg.route_experts_backward(g[live], x[live], idx[live], score=score, renormalize=renormalize, scale=1.5)
    assert torch.equal(leaf.grad[live], alone) and torch.isfinite(alone.float()).all()
    # a row whose places are all -1 is a constant whatever its logits are
    none = torch.full_like(idx, -1)
    assert (pkg.route_experts_backward(g, x, none, score=score, renormalize=renormalize) == 0).all()
    ref = X.route_grad(g.cpu().numpy(), x.double().cpu().numpy(), idx.cpu().numpy(), score, renormalize, 1.5)
    assert (ref[[2, 8]] == 0).all()


@pytest.mark.parametrize("renormalize", [False, True])
def test_gradient_shows_a_nan_logit(pkg, renormalize):
    """A NaN among excluded experts is picked, so its row's gradient is NaN; other rows do not see it."""
    x = torch.full((3, 64), -INF, device="cuda")
    x[0, :8] = x[2, :8] = torch.arange(8.0, device="cuda")
    x[1, 5] = float("nan")
    leaf = x.requires_grad_()
    idx, w = pkg.route_experts(leaf, 4, renormalize=renormalize)
    assert idx[1].tolist() == [5, -1, -1, -1]
    w.sum().backward()
    assert torch.isnan(leaf.grad[1]).any() and torch.isfinite(leaf.grad[[0, 2]]).all()


def _same_order(pkg, x, k, bias=None, **rule):
    idx, _ = pkg.route_experts(x, k, bias=bias, **rule)
    score = rule.pop("score")
    ref, _ = X.route(x.double().cpu().numpy(), k, score, None if bias is None else bias.double().cpu().numpy(), **rule)
    np.testing.assert_array_equal(idx.cpu().numpy(), ref)


@pytest.mark.parametrize("E", [64, 48])
def test_scores_that_round_together_without_a_bias(pkg, E):
    """Without a bias the kept groups' experts are ordered by their logits, also where 32-bit scores are equal: sigmoids of
    18 and more are 1, exponentials 110 below the maximum are 0. The groups themselves are far apart."""
    rng, per = np.random.default_rng(E), E // 8
    x = np.full((20, 8, per), -5.0, np.float32) - np.arange(8, dtype=np.float32)[:, None]
    for t in range(20):
        x[t, :4] = rng.permutation(np.linspace(18.0, 30.0, 4 * per)).reshape(4, per)
    group = dict(n_group=8, topk_group=4, group_score="top2")
    _same_order(pkg, torch.from_numpy(x.reshape(20, E)).cuda(), 12, score="sigmoid", **group)
    for t in range(20):
        x[t, :4] = -rng.permutation(np.linspace(110.0, 130.0, 4 * per)).reshape(4, per)
        x[t, 4:] = -200.0
        x[t, :4, 0] = [0.0, -0.5, -1.0, -1.5]
    _same_order(pkg, torch.from_numpy(x.reshape(20, E)).cuda(), 12, score="softmax", **group)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("base", [-9.0, -13.0, -15.5, -20.0, -29.0, -50.0])
def test_choice_by_scores_of_32_bits(pkg, base, grouped, score):
    """Neighbouring float32 logits around `base`, in any order, under a bias of zero, so that the scores are compared. They
    are 2^-20 (8 to 16), 2^-19 or 2^-18 (32 to 64) apart, which is as much between their scores: 8 units of 2^-23 at least.
    An exponential of 2 units, a sum of half a unit and a reciprocal or product of one are 7 for the two of them."""
    rng, E = np.random.default_rng(0), 64
    step = np.spacing(np.float32(abs(base)))
    x = np.stack([base - 40 * step * t + step * rng.permutation(E) for t in range(30)]).astype(np.float32)
    assert (np.diff(np.sort(x, 1), axis=1) == step).all()
    group = dict(n_group=8, topk_group=8, group_score="top2") if grouped else {}
    if score == "softmax":
        x[:, 7] = 0.0
    _same_order(pkg, torch.from_numpy(x).cuda(), 16, torch.zeros(E, device="cuda"), score=score, **group)


@pytest.mark.parametrize("renormalize", [False, True])
def test_weights_of_32_bits(pkg, renormalize):
    """Sigmoid weights. Units of 2^-24: exponential 4, sum 1, quotient 1, so 6 of a score. Without renormalisation 1 more for
    the scale. With it the row's sum has the scores' 6 and 5 additions, then a quotient and the scale: 19."""
    x = (3 * torch.randn((4096, 64), generator=torch.Generator().manual_seed(0))).cuda()
    idx, w = pkg.route_experts(x, 6, score="sigmoid", renormalize=renormalize, scale=2.5)
    ref = X.weights(X.scores(x.double().cpu().numpy(), "sigmoid"), idx.cpu().numpy(), renormalize, 2.5)
    assert (np.abs(w.double().cpu().numpy() / ref - 1) <= (19 if renormalize else 7) * 2.0 ** -24).all()
