"""The general expert router and its gradient against the 64-bit formulas.

The chosen experts must be a valid answer: at each place the pick's 64-bit value is within 2e-6 of the
value that the exact order has there (32-bit scores carry an error below 4 units of 2^-24 of values of
at most about 1.5), and exactly the exact order where the picks are equal or well apart. Weights are
within 4e-6 relative (a few 32-bit roundings), gradients within 1e-5 of the row's largest (32-bit
results) plus half a unit of the output type."""
import numpy as np
import pytest
import torch

from oracle import experts_oracle as X

pytestmark = pytest.mark.gpu
UNIT = {torch.float32: 0.0, **{t: torch.finfo(t).eps for t in (torch.bfloat16, torch.float16)}}


def _logits(T, E, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn((T, E), generator=g)).to(dtype).cuda()


def _check_route(pkg, logits, k, bias=None, exact=False, **rule):
    idx, w = pkg.route_experts(logits, k, bias=bias, **rule)
    torch.cuda.synchronize()
    idx, w = idx.cpu().numpy(), w.cpu().numpy()
    x = logits.double().cpu().numpy()
    b = None if bias is None else bias.double().cpu().numpy()
    score, renorm, scale = rule.get("score", "softmax"), rule.get("renormalize", True), rule.get("scale", 1.0)
    group = {n: rule[n] for n in ("n_group", "topk_group", "group_score") if n in rule}
    s, pick = X.picks(x, score, b, **group)
    eidx, _ = X.route(x, k, score, b, renormalize=renorm, scale=scale, **group)
    assert ((idx < 0) == (eidx < 0)).all()
    got = np.where(idx < 0, -np.inf, np.take_along_axis(pick, np.maximum(idx, 0), 1))
    want = np.where(eidx < 0, -np.inf, np.take_along_axis(pick, np.maximum(eidx, 0), 1))
    if exact or not group or rule.get("n_group") == 1:
        fin = np.isfinite(want)
        assert (np.abs(got[fin] - want[fin]) <= 2e-6).all() and (got[~fin] == want[~fin]).all()
    for row in idx:
        real = row[row >= 0]
        assert len(set(real.tolist())) == len(real) and (real < x.shape[1]).all()
    if exact:
        np.testing.assert_array_equal(idx, eidx)
    else:
        assert (idx == eidx).mean() > 0.999
    ref = X.weights(s, idx, renorm, scale)
    assert (np.abs(w - ref) <= 4e-6 * np.abs(ref) + 1e-30).all()
    return idx, w


V3 = dict(score="sigmoid", n_group=8, topk_group=4, group_score="top2", scale=2.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,rule", [
    (1, 256, 8, V3), (77, 256, 8, V3), (3001, 256, 8, V3),
    (33, 1, 1, {}), (9, 2, 2, dict(renormalize=False)), (130, 31, 5, dict(score="sigmoid")),
    (65, 32, 32, {}), (65, 33, 7, dict(renormalize=False, scale=0.5)), (400, 60, 6, dict(n_group=4, topk_group=2)),
    (50, 64, 6, dict(renormalize=False)), (50, 100, 12, dict(score="sigmoid", n_group=5, topk_group=5, group_score="top2")),
    (40, 128, 1, {}), (40, 160, 6, dict(n_group=8, topk_group=3)), (20, 512, 10, dict(score="sigmoid", n_group=32, topk_group=4)),
    (20, 600, 32, {}), (10, 1024, 32, dict(score="sigmoid", n_group=2, topk_group=1)),
])
@pytest.mark.parametrize("with_bias", [False, True])
def test_router(pkg, T, E, k, rule, dtype, with_bias):
    bias = (0.1 * torch.randn(E, generator=torch.Generator().manual_seed(E))).cuda() if with_bias else None
    _check_route(pkg, _logits(T, E, dtype, T + E), k, bias, **rule)


def test_same_choice_as_the_fixed_router(pkg):
    inp = pkg.make_inputs(pkg.CONFIGS[2].with_(E_local=1), "cuda")
    lg, b = inp["routing_logits"], inp["routing_bias"].float()
    idx, w = pkg.route_experts(lg, 8, bias=b, **V3)
    ridx, rw = pkg.route(lg, b, 2.5)
    same = (idx == ridx).all(1)
    assert same.float().mean() > 0.999          # rows whose picks differ by less than the 32-bit error
    assert ((w - rw).abs()[same] <= 4e-6 * rw[same]).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k", [(32, 4), (64, 8), (256, 8), (250, 32), (1024, 20)])
def test_ties_go_to_the_lower_expert(pkg, E, k, score):
    # All equal; two values only; a sorted row (its best experts sit in neighbouring registers of few lanes).
    flat = torch.zeros((3, E))
    two = (torch.arange(E) % 3 == 1).float().expand(2, E)
    rows = torch.cat((flat, two, torch.arange(E).float()[None] / 64, -torch.arange(E).float()[None] / 64))
    for dtype in (torch.float32, torch.float16):
        idx, _ = _check_route(pkg, rows.to(dtype).cuda(), k, exact=True, score=score)
        assert (idx[0] == np.arange(k)).all()
    idx, _ = _check_route(pkg, flat.cuda(), k, torch.zeros(E).cuda(), exact=True, score=score)
    zeros = torch.zeros((1, E)).cuda()
    zeros[0, E // 2] = -0.0                      # -0 ties with +0
    idx, _ = pkg.route_experts(zeros, k, score=score)
    assert (idx.cpu().numpy()[0] == np.arange(k)).all()


def test_equal_groups_go_to_the_lower_group(pkg):
    idx, _ = pkg.route_experts(torch.zeros((2, 64)).cuda(), 6, n_group=8, topk_group=2, group_score="top2", score="sigmoid")
    assert (idx.cpu().numpy() == np.arange(6)).all()
    x = torch.zeros((1, 64)).cuda()
    x[0, 40] = 1.0
    idx, _ = pkg.route_experts(x, 6, n_group=8, topk_group=2)
    assert idx.cpu().numpy()[0].tolist() == [40, 0, 1, 2, 3, 4]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [{}, dict(n_group=4, topk_group=2, group_score="top2"), dict(n_group=4, topk_group=1)])
@pytest.mark.parametrize("E", [64, 60])
def test_excluded_experts(pkg, E, groups, score):
    x = _logits(64, E, torch.float32, 5)
    x[0] = -float("inf")                         # no expert allowed
    x[1, 1:] = -float("inf")                     # one allowed
    x[2, : E - 3] = -float("inf")                # three allowed, all in the last group
    x[3, ::2] = -float("inf")
    x[4] = torch.finfo(torch.float32).min        # the type's lowest value is a logit like any other
    x[5, 10:] = torch.finfo(torch.float32).min
    idx, w = _check_route(pkg, x, 8, score=score, **groups)
    assert (idx[0] == -1).all() and (w[0] == 0).all()
    if not groups:
        assert idx[1].tolist() == [0] + [-1] * 7
        assert sorted(idx[2].tolist()) == [-1] * 5 + [E - 3, E - 2, E - 1]
    bias = torch.zeros(E).cuda()
    bias[5:] = -float("inf")
    idx, w = _check_route(pkg, x[6:], 8, bias, score=score, **groups)
    assert idx.max() <= 4
    g = pkg.route_experts_backward(torch.ones((64, 8)).cuda(), x, torch.from_numpy(np.full((64, 8), -1, np.int32)).cuda(),
                                   score=score)
    assert (torch.nan_to_num(g) == 0).all()


def test_nan_and_infinity(pkg):
    x = _logits(4, 64, torch.float32, 6)
    x[1, 7] = float("nan")
    x[2, 9] = float("inf")
    for score in ("softmax", "sigmoid"):
        idx, w = pkg.route_experts(x, 6, score=score)
        assert ((idx >= 0) & (idx < 64)).all()
        assert torch.isnan(w[1]).all() and torch.isfinite(w[[0, 3]]).all()
        assert torch.isnan(w[2]).any() if score == "softmax" else torch.isfinite(w[2]).all()
        assert idx[1, 0] == 7 and idx[2, 0] == 9


def test_strided_and_shifted_rows_and_streams(pkg):
    for dtype in (torch.float32, torch.bfloat16):
        big = _logits(70, 300, dtype, 8)
        for view in (big[:, :256], big[:, 1:257], big[:, 3:67], big[::3, 8:264]):
            i0, w0 = pkg.route_experts(view.contiguous(), 8)
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                i1, w1 = pkg.route_experts(view, 8)
                g1 = pkg.route_experts_backward(w1, view, i1)
            s.synchronize()
            assert torch.equal(i0, i1) and torch.equal(w0, w1)
            assert torch.equal(g1, pkg.route_experts_backward(w0, view.contiguous(), i0))
    i, w = pkg.route_experts(torch.empty((0, 64), device="cuda"), 4)
    assert i.shape == (0, 4) and pkg.route_experts_backward(w, torch.empty((0, 64), device="cuda"), i).shape == (0, 64)


GRAD = [(1, 256, 8), (67, 256, 8), (40, 1, 1), (33, 31, 5), (20, 60, 6), (9, 1024, 32), (5, 600, 17), (50, 128, 2)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("T,E,k", GRAD)
def test_gradient(pkg, T, E, k, score, renormalize, dtype):
    x = _logits(T, E, dtype, 3 * T + E)
    g = torch.randn((T, k), generator=torch.Generator().manual_seed(E)).cuda()
    idx, _ = pkg.route_experts(x, k, score=score)
    if T > 4 and k > 1:
        idx[1, 0] = -1                           # a place without an expert
        idx[2] = -1
    got = pkg.route_experts_backward(g, x, idx, score=score, renormalize=renormalize, scale=1.5)
    ref = X.route_grad(g.cpu().numpy(), x.double().cpu().numpy(), idx.cpu().numpy(), score, renormalize, 1.5)
    got = got.double().cpu().numpy()
    # One-place rows renormalise to a constant: the exact gradient is about 1e-20 and 32 bits see s/s = 1.
    size = np.abs(g.cpu().numpy()).max(axis=1, keepdims=True) * 1.5
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0     # half of the type's smallest step below 2^-14
    assert (np.abs(got - ref) <= 1e-5 * size + UNIT[dtype] / 2 * np.abs(ref) + tiny).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gradient_against_differences(pkg, score, renormalize):
    T, E, k, eps = 5, 24, 4, 1e-6
    x = _logits(T, E, torch.float32, 1)
    idx, _ = pkg.route_experts(x, k, score=score)
    g = torch.randn((T, k), generator=torch.Generator().manual_seed(2)).cuda()
    got = pkg.route_experts_backward(g, x, idx, score=score, renormalize=renormalize, scale=2.0).cpu().numpy()
    x64, i, g64 = x.double().cpu().numpy(), idx.cpu().numpy(), g.double().cpu().numpy()
    f = lambda z: (g64 * X.weights(X.scores(z, score), i, renormalize, 2.0)).sum(1)  # noqa: E731
    for e in range(E):
        d = np.zeros((T, E))
        d[:, e] = eps
        diff = (f(x64 + d) - f(x64 - d)) / (2 * eps)
        # differences: eps^2 in the third derivative plus 1e-16 / eps of rounding; the gradient: 32 bits
        assert (np.abs(got[:, e] - diff) <= 2e-5).all()


@pytest.mark.parametrize("rule", [V3, dict(score="softmax", renormalize=False), dict(score="softmax")])
def test_autograd(pkg, rule):
    x = _logits(12, 256, torch.float32, 4).requires_grad_()
    idx, w = pkg.route_experts(x, 8, **rule)
    g = torch.randn(w.shape, generator=torch.Generator().manual_seed(0)).cuda()
    (w * g).sum().backward()
    args = dict(score=rule["score"], renormalize=rule.get("renormalize", True), scale=rule.get("scale", 1.0))
    assert torch.equal(x.grad, pkg.route_experts_backward(g, x.detach(), idx, **args))
    with torch.no_grad():
        assert not pkg.route_experts(x, 8, **rule)[1].requires_grad


def test_refusals(pkg):
    x = _logits(4, 64, torch.float32, 0)
    bad = [(dict(top_k=0), "top_k"), (dict(top_k=33), "top_k"), (dict(top_k=9, n_group=8, topk_group=1), "top_k"),
           (dict(top_k=2, n_group=3), "n_group"), (dict(top_k=2, n_group=0), "n_group"), (dict(top_k=2, n_group=64), "n_group"),
           (dict(top_k=2, n_group=4, topk_group=5), "topk_group"), (dict(top_k=2, score="tanh"), "score"),
           (dict(top_k=2, group_score="mean"), "group_score"),
           (dict(top_k=2, bias=torch.zeros(63).cuda()), "bias"), (dict(top_k=2, bias=torch.zeros(64)), "bias"),
           (dict(top_k=2, bias=torch.zeros(64, dtype=torch.bfloat16).cuda()), "bias")]
    for kw, word in bad:
        with pytest.raises(RuntimeError, match=word):
            pkg.route_experts(x, **kw)
    for t in (x.cpu(), x[0], x.double(), x.t(), torch.zeros((2, 1025)).cuda(), torch.zeros((2, 0)).cuda()):
        with pytest.raises(RuntimeError, match="logits"):
            pkg.route_experts(t, 1)
    with pytest.raises(RuntimeError, match="top2"):
        pkg.route_experts(x[:, :32], 2, n_group=32, topk_group=4, group_score="top2")
    idx, w = pkg.route_experts(x, 4)
    for a, b in ((w.double(), idx), (w[:, :3], idx), (w, idx.long()), (w, idx[:2]), (w.cpu(), idx), (w, idx.cpu())):
        with pytest.raises(RuntimeError, match="idx|grad_weights"):
            pkg.route_experts_backward(a, x, b)
