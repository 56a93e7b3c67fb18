"""Arguments of the expert operators that are no whole numbers, no numbers or, for whole ones, too large: RuntimeError, as for every other bad argument."""
import numpy as np
import pytest
import torch

from test_gpu_w4 import layer, routing, weights

pytestmark = pytest.mark.gpu


def test_router(pkg):
    x = torch.randn((4, 64), device="cuda")
    for leaf in (x, x.clone().requires_grad_()):
        for kw, word in [(dict(top_k=2.0), "top_k"), (dict(top_k="2"), "top_k"), (dict(top_k=None), "top_k"), (dict(top_k=2 ** 40), "top_k"),
                         (dict(top_k=2, n_group=4.0, topk_group=2), "n_group"), (dict(top_k=2, n_group=4, topk_group=1.5), "topk_group"),
                         (dict(top_k=2, scale=None), "scale"), (dict(top_k=2, scale="1"), "scale"),
                         (dict(top_k=2, score=["softmax"]), "score"), (dict(top_k=2, group_score=None), "group_score")]:
            with pytest.raises(RuntimeError, match=word):
                pkg.route_experts(leaf, **kw)
    idx, w = pkg.route_experts(x, np.int64(2), n_group=np.int32(4), topk_group=torch.tensor(2), scale=np.float32(2.0))
    same = pkg.route_experts(x, 2, n_group=4, topk_group=2, scale=2)
    assert torch.equal(idx, same[0]) and torch.equal(w, same[1])
    for kw, word in [(dict(scale=None), "scale"), (dict(score=["softmax"]), "score")]:
        with pytest.raises(RuntimeError, match=word):
            pkg.route_experts_backward(w, x, idx, **kw)


def test_products(pkg):
    dtype = torch.bfloat16
    x = torch.zeros((3, 64), dtype=dtype, device="cuda")
    codes, scale, zero = weights((), 16, 64, 32, True, dtype, 0)
    for group in (32.0, "32", None, 2 ** 40):
        with pytest.raises(RuntimeError, match="group"):
            pkg.linear_w4(x, codes, scale, zero, group=group)
    (w13, s13, _), (w2, s2, _) = layer(3, 64, 32, 32, False, dtype, 0)
    idx, wt = routing(3, 3, 2, 0)
    for kw, word in [(dict(local_offset=2 ** 31), "local_offset"), (dict(local_offset=-2 ** 40), "local_offset"),
                     (dict(local_offset=1.0), "local_offset"), (dict(local_offset=None), "local_offset"), (dict(group=32.0), "group")]:
        with pytest.raises(RuntimeError, match=word):
            pkg.experts_w4(x, idx, wt, w13, s13, w2, s2, **{"group": 32, **kw})
    far = pkg.experts_w4(x, idx, wt, w13, s13, w2, s2, group=32, local_offset=2 ** 31 - 1)
    assert (far == 0).all()                                            # no pick lies there
    assert pkg.experts_w4_workspace_bytes(2 ** 32 + 3, 2, 3, 64, 32) == 0
