"""experts_w4 beyond 1024 picks, where the picks' places come from atomics and a gather, against 64-bit sums.

Tolerances as for the smaller calls: half a unit of the output type, 2^-15 of the absolute sum, half of float16's smallest
step. Calls repeat bit for bit although the order within an expert's list does not."""
import pytest
import torch

from test_gpu_w4 import check_experts, layer, routing

pytestmark = pytest.mark.gpu


def tokens(T, H, dtype, seed=0):
    return torch.randn((T, H), generator=torch.Generator().manual_seed(T + seed)).to(dtype).cuda()


def call(pkg, x, idx, wt, l13, l2, group, **kw):
    return pkg.experts_w4(x, idx, wt, l13[0], l13[1], l2[0], l2[1], w13_zero=l13[2], w2_zero=l2[2], group=group, **kw)


# Picks per expert of this GPU decide the tile: up to 32, up to 64, more.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,EG,k,H,I,group", [
    (512, 8, 8, 2, 128, 64, 32), (205, 8, 8, 5, 128, 64, 32), (1025, 4, 4, 1, 64, 96, 32),      # the limit from both sides
    (300, 64, 64, 4, 128, 64, 32), (300, 64, 64, 4, 256, 128, 64), (260, 40, 80, 8, 128, 128, 128),
    (260, 24, 24, 5, 256, 64, 64), (260, 24, 48, 5, 128, 192, 128), (330, 30, 30, 4, 320, 96, 32),
    (400, 5, 10, 4, 128, 128, 128), (700, 6, 6, 2, 192, 64, 64),
    (300, 64, 64, 4, 99, 53, 32), (260, 24, 24, 5, 131, 77, 64), (400, 5, 10, 4, 1, 1, 128), (350, 7, 7, 3, 161, 200, 32),
])
def test_experts(pkg, T, E, EG, k, H, I, group, dtype):
    x = tokens(T, H, dtype)
    idx, wt = routing(T, EG, k, T + E)
    for zero in (False, True):
        check_experts(pkg, x, idx, wt, *layer(E, H, I, group, zero, dtype, H + I), group)


@pytest.mark.parametrize("E", [6, 20, 60])
def test_uneven_routing(pkg, E):
    dtype, T, H, I, group, k = torch.bfloat16, 400, 128, 64, 64, 3
    x, (l13, l2) = tokens(T, H, dtype), layer(E, H, I, group, True, dtype, 9)
    idx, wt = routing(T, E, k, 2)
    one = torch.full_like(idx, -1)
    one[:, 1] = 4
    check_experts(pkg, x, one, wt, l13, l2, group)                     # every token to one expert
    check_experts(pkg, x, torch.full_like(idx, 3), wt, l13, l2, group)  # the same expert in every place
    some = idx.clone()
    some[::2] = -1
    some[0, 0], some[-1, 0], some[5, 1] = 2 ** 31 - 1, -2 ** 31, E
    y = check_experts(pkg, x, some, wt, l13, l2, group)                # tokens without a pick, picks that are no experts
    assert (y[2] == 0).all()
    assert (check_experts(pkg, x, torch.full_like(idx, -1), wt, l13, l2, group) == 0).all()
    check_experts(pkg, x, idx + 10, wt, l13, l2, group, offset=10)     # a slice of a larger layer
    check_experts(pkg, x, idx + 10, wt, l13, l2, group, offset=12)
    most = torch.where(torch.rand(idx.shape, generator=torch.Generator().manual_seed(1)).cuda() < 0.9, 0, idx)
    check_experts(pkg, x, most, -wt, l13, l2, group)                   # nine of ten picks on one expert


@pytest.mark.parametrize("dtype,H,I", [(torch.bfloat16, 128, 96), (torch.float16, 99, 53)])
@pytest.mark.parametrize("E", [5, 25, 50])
def test_views_workspace_streams_and_graphs(pkg, E, dtype, H, I):
    T, group, k = 400, 32, 4
    l13, l2 = layer(E, H, I, group, True, dtype, 4)
    big = tokens(T, H + 24, dtype)
    idx, wt = routing(T, E, k, T)
    ws = torch.full((pkg.experts_w4_workspace_bytes(T, k, E, H, I),), 255, dtype=torch.uint8, device="cuda")
    for view in (big[:, :H], big[:, 3:H + 3], big[:, 8:H + 8]):
        ws.fill_(255)                                                  # NaN in both types
        out = torch.full((T, H), 3.0, dtype=dtype, device="cuda")
        y = check_experts(pkg, view, idx, wt, l13, l2, group, out=out, workspace=ws)
        assert y is out
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            z = call(pkg, view.contiguous(), idx, wt, l13, l2, group)
        s.synchronize()
        assert torch.equal(y, z)
        for _ in range(10):
            assert torch.equal(y, call(pkg, view, idx, wt, l13, l2, group))
    x = big[:, :H].contiguous()
    out, graph = torch.empty_like(x), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(pkg, x, idx, wt, l13, l2, group, out=out, workspace=ws)
    x.neg_()
    idx.copy_(idx.flip(0))
    for _ in range(3):
        ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(pkg, x, idx, wt, l13, l2, group))


@pytest.mark.parametrize("E", [4, 20, 50])
def test_rows_do_not_mix(pkg, E):
    dtype, T, H, I, group = torch.bfloat16, 600, 128, 64, 32
    l13, l2 = layer(E, H, I, group, False, dtype, 4)
    x = tokens(T, H, dtype)
    idx, wt = routing(T, E, 2, T)
    y = call(pkg, x, idx, wt, l13, l2, group)
    x2 = x.clone()
    x2[T - 1, 5], x2[3, 7] = float("nan"), float("inf")
    y2 = call(pkg, x2, idx, wt, l13, l2, group)
    keep = torch.ones(T, dtype=torch.bool)
    keep[T - 1] = keep[3] = False
    assert torch.equal(y[keep], y2[keep]) and torch.isnan(y2[T - 1]).all()
