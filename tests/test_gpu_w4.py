"""Products with 4-bit weights against 64-bit sums.

Tolerance of one product: half a unit of the output type (the one rounding), plus 2^-18 of the sum of
absolute values (32-bit accumulation of at most a few thousand terms), plus half of float16's smallest
step. For the experts' pair of products the intermediate may carry 16 bits: 2^-15 of the absolute sum
in place of 2^-18."""
import importlib

import numpy as np
import pytest
import torch

from oracle import experts_oracle as X

pytestmark = pytest.mark.gpu
UNIT = {t: torch.finfo(t).eps for t in (torch.bfloat16, torch.float16)}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def weights(lead, N, K, group, zero, dtype, seed, std=0.05):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (*lead, N, (K + 1) // 2), generator=g, dtype=torch.uint8)
    scale = (std * (0.5 + torch.rand((*lead, N, -(-K // group)), generator=g))).to(dtype)
    z = torch.randint(0, 16, scale.shape, generator=g, dtype=torch.uint8) if zero else None
    return codes.cuda(), scale.cuda(), None if z is None else z.cuda()


def full(codes, scale, zero, K, group):
    return X.unpack_w4(codes.cpu().numpy(), scale.double().cpu().numpy(), None if zero is None else zero.cpu().numpy(), K, group)


def check_linear(pkg, x, codes, scale, zero, group, out=None):
    y = pkg.linear_w4(x, codes, scale, zero, group=group, out=out)
    torch.cuda.synchronize()
    assert pkg.device_status(reset=True) == 0
    w, x64 = full(codes, scale, zero, x.shape[1], group), x.double().cpu().numpy()
    ref, size = x64 @ w.T, np.abs(x64) @ np.abs(w).T
    err = np.abs(y.double().cpu().numpy() - ref)
    assert (err <= UNIT[x.dtype] / 2 * np.abs(ref) + 2.0 ** -18 * size + TINY[x.dtype]).all(), float(err.max())
    return y


MS = [1, 2, 7, 8, 9, 16, 17, 33, 64, 65, 127, 128, 129, 200, 300]
SHAPES = [(64, 128, 128), (128, 256, 64), (257, 96, 32), (1, 32, 32), (1, 1, 128), (16, 31, 32), (300, 333, 64),
          (127, 1024, 128), (130, 1056, 128), (96, 4096, 32), (512, 2080, 64), (33, 10000, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,K,group", SHAPES)
def test_linear(pkg, N, K, group, dtype):
    for i, M in enumerate(MS):
        x = torch.randn((M, K), generator=torch.Generator().manual_seed(M)).to(dtype).cuda()
        check_linear(pkg, x, *weights((), N, K, group, i % 2 == 0, dtype, N + K), group)


@pytest.mark.parametrize("M", [1, 5, 8, 20, 150])
def test_linear_views_and_out(pkg, M):
    dtype, N, K, group = torch.bfloat16, 192, 512, 64
    w = weights((), N, K, group, True, dtype, 3)
    big = torch.randn((2 * M, K + 40), generator=torch.Generator().manual_seed(M)).to(dtype).cuda()
    for view in (big[:M, :K], big[:M, 1:K + 1], big[::2, 8:K + 8], big[:M, 40:]):
        out = torch.full((M, N), 7.0, dtype=dtype, device="cuda")
        y = check_linear(pkg, view, *w, group, out=out)
        assert y is out
        assert torch.equal(y, pkg.linear_w4(view.contiguous(), *w, group=group))
    # codes, scales and zero points that start anywhere
    codes, scale, zero = w
    shifted = [torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t) for t in w]
    x = big[:M, :K].contiguous()
    assert torch.equal(pkg.linear_w4(x, *shifted, group=group), pkg.linear_w4(x, *w, group=group))
    assert pkg.linear_w4(x[:0], *w, group=group).shape == (0, N)


@pytest.mark.parametrize("M", [1, 8, 40, 200])
def test_linear_rows_do_not_mix(pkg, M):
    """Infinities and NaN stay in their own row; a row's result does not depend on the others' values."""
    dtype, N, K = torch.bfloat16, 100, 320
    w = weights((), N, K, 128, True, dtype, 1)
    x = torch.randn((M, K), generator=torch.Generator().manual_seed(0)).to(dtype).cuda()
    y = pkg.linear_w4(x, *w)
    x2 = x.clone()
    x2[M - 1, 3], x2[M - 1, 100] = float("nan"), float("inf")
    y2 = pkg.linear_w4(x2, *w)
    assert torch.equal(y[:M - 1], y2[:M - 1]) and torch.isnan(y2[M - 1]).all()
    x2[M - 1, 3] = 0.0                            # one infinity times weights that are not zero
    ref = x2[M - 1].double().cpu().numpy()
    y2 = pkg.linear_w4(x2, *w)[M - 1].double().cpu().numpy()
    at = full(*w, K, 128)[:, 100]
    assert np.isfinite(ref[np.arange(K) != 100]).all()
    assert (np.sign(y2[at != 0]) == np.sign(at[at != 0])).all() and np.isinf(y2[at != 0]).all()
    # every code and zero point, against the plain value
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(16, 1)
    zero = torch.arange(16, dtype=torch.uint8, device="cuda")[:, None].repeat(1, 4)
    scale = torch.ones((16, 4), dtype=dtype, device="cuda")
    eye = torch.eye(512, dtype=dtype, device="cuda")[: max(M, 1)]
    got = pkg.linear_w4(eye, codes, scale, zero)
    np.testing.assert_array_equal(got.double().cpu().numpy(), full(codes, scale, zero, 512, 128).T[: max(M, 1)])


def test_linear_repeats_bit_for_bit_and_captures(pkg):
    dtype = torch.bfloat16
    w = weights((), 640, 2048, 128, False, dtype, 5)
    for M in (1, 8, 100):
        x = torch.randn((M, 2048), device="cuda").to(dtype)
        y = pkg.linear_w4(x, *w)
        for _ in range(5):
            assert torch.equal(y, pkg.linear_w4(x, *w))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            z = pkg.linear_w4(x, *w)
        s.synchronize()
        assert torch.equal(y, z)
        out, graph = torch.empty_like(y), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pkg.linear_w4(x, *w, out=out)
        x.copy_(x.flip(0).neg())
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, pkg.linear_w4(x, *w))


@pytest.mark.parametrize("M", [20, 100])
def test_alternating_weights_of_an_odd_width(pkg, M):
    """Rows that TMA cannot read are copied within the call: every call has to see its own weights."""
    dtype, N, K = torch.bfloat16, 3000, 1999
    sets = [weights((), N, K, 64, True, dtype, seed) for seed in (1, 2, 3)]
    x = torch.randn((M, K), generator=torch.Generator().manual_seed(M)).to(dtype).cuda()
    first = [check_linear(pkg, x, *w, 64) for w in sets]
    for i in range(30):
        assert torch.equal(pkg.linear_w4(x, *sets[i % 3], group=64), first[i % 3])


def test_overlapping_output_is_refused(pkg):
    dtype = torch.bfloat16
    w = weights((), 64, 64, 32, False, dtype, 1)
    for M in (2, 40):
        x = torch.zeros((M, 64), dtype=dtype, device="cuda")
        with pytest.raises(RuntimeError, match="overlaps"):
            pkg.linear_w4(x, *w, group=32, out=x)
    l13, l2 = layer(2, 64, 32, 32, False, dtype, 0)
    idx, wt = routing(40, 2, 1, 0)
    with pytest.raises(RuntimeError, match="overlaps"):
        pkg.experts_w4(x, idx, wt, l13[0], l13[1], l2[0], l2[1], group=32, out=x)
    with pytest.raises(RuntimeError, match="local_offset"):
        pkg.experts_w4(x, idx, wt, l13[0], l13[1], l2[0], l2[1], group=32, local_offset=-1)


def test_offsets_past_32_bits(pkg):
    """Codes of more than 2^32 bytes: the last rows of a very tall matrix."""
    N, K = 2 ** 20 + 77, 8192
    codes = torch.zeros((N, K // 2), dtype=torch.uint8, device="cuda")
    codes.fill_(0x88)                             # zero weights
    codes[-5:] = torch.arange(5, dtype=torch.uint8, device="cuda")[:, None] * 0x11 + 0x33
    scale = torch.ones((N, K // 128), dtype=torch.bfloat16, device="cuda")
    for M in (1, 12):
        x = torch.ones((M, K), dtype=torch.bfloat16, device="cuda")
        y = pkg.linear_w4(x, codes, scale)
        assert (y[:, :-5] == 0).all()
        assert y[0, -5:].tolist() == [float((3 + i - 8) * K) for i in range(5)]


# ------------------------------------------------------------------------------------- experts
def layer(E, H, I, group, zero, dtype, seed):
    return weights((E,), 2 * I, H, group, zero, dtype, seed), weights((E,), H, I, group, zero, dtype, seed + 1)


def check_experts(pkg, x, idx, wt, l13, l2, group, offset=0, **kw):
    (w13, s13, z13), (w2, s2, z2) = l13, l2
    y = pkg.experts_w4(x, idx, wt, w13, s13, w2, s2, w13_zero=z13, w2_zero=z2, group=group, local_offset=offset, **kw)
    torch.cuda.synchronize()
    assert pkg.device_status(reset=True) == 0
    ref, size = X.experts(x.double().cpu().numpy(), idx.cpu().numpy(), wt.double().cpu().numpy(),
                          full(*l13, x.shape[1], group), full(*l2, w13.shape[1] // 2, group), offset)
    err = np.abs(y.double().cpu().numpy() - ref)
    bound = UNIT[x.dtype] / 2 * np.abs(ref) + 2.0 ** -15 * size + TINY[x.dtype]
    assert (err <= bound).all(), float((err - bound).max())
    return y


def routing(T, EG, k, seed):
    g = torch.Generator().manual_seed(seed)
    idx = torch.rand((T, EG), generator=g).topk(k, dim=1).indices.to(torch.int32)
    return idx.cuda(), (torch.rand((T, k), generator=g) + 0.1).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,EG,k,H,I,group", [
    (1, 4, 4, 2, 128, 64, 64), (1, 8, 8, 8, 512, 256, 128), (3, 8, 32, 4, 256, 96, 32), (8, 4, 4, 3, 384, 160, 64),
    (9, 3, 3, 2, 128, 128, 128), (40, 6, 12, 4, 192, 224, 32), (70, 16, 16, 6, 256, 64, 64), (300, 2, 4, 2, 128, 96, 32),
    (150, 1, 1, 1, 320, 128, 128), (5, 4, 4, 2, 99, 53, 32), (33, 5, 5, 3, 131, 77, 64), (64, 40, 40, 8, 128, 32, 32),
    (2, 300, 300, 32, 64, 32, 32), (16, 1, 1, 1, 1, 1, 32),
])
def test_experts(pkg, T, E, EG, k, H, I, group, dtype):
    x = torch.randn((T, H), generator=torch.Generator().manual_seed(T)).to(dtype).cuda()
    idx, wt = routing(T, EG, k, T + E)
    for zero in (False, True):
        check_experts(pkg, x, idx, wt, *layer(E, H, I, group, zero, dtype, H + I), group)


@pytest.mark.parametrize("T", [1, 6, 8, 9, 50, 140])
def test_experts_uneven_routing(pkg, T):
    dtype, E, H, I, group, k = torch.bfloat16, 6, 256, 128, 64, 3
    x = torch.randn((T, H), generator=torch.Generator().manual_seed(T)).to(dtype).cuda()
    l13, l2 = layer(E, H, I, group, True, dtype, 9)
    idx, wt = routing(T, E, k, 2)
    one = torch.full_like(idx, -1)
    one[:, 1] = 4
    check_experts(pkg, x, one, wt, l13, l2, group)                     # every token to one expert
    some = idx.clone()
    some[::2] = -1
    some[0, 0] = 2 ** 31 - 1
    some[-1, 0] = -2 ** 31
    y = check_experts(pkg, x, some, wt, l13, l2, group)                # tokens without a pick
    if T > 2:
        assert (y[2] == 0).all()
    y = check_experts(pkg, x, torch.full_like(idx, -1), wt, l13, l2, group)
    assert (y == 0).all()                                             # no token here
    check_experts(pkg, x, idx + 10, wt, l13, l2, group, offset=10)     # a slice of a larger layer
    check_experts(pkg, x, idx + 10, wt, l13, l2, group, offset=12)
    check_experts(pkg, x, torch.full_like(idx, 3), wt, l13, l2, group)  # the same expert in every place
    check_experts(pkg, x, idx, -wt, l13, l2, group)


def test_experts_views_workspace_and_streams(pkg):
    dtype, E, H, I, group, k = torch.bfloat16, 5, 256, 96, 32, 2
    l13, l2 = layer(E, H, I, group, True, dtype, 4)
    for T in (1, 4, 30, 150):
        big = torch.randn((T, H + 24), generator=torch.Generator().manual_seed(T)).to(dtype).cuda()
        idx, wt = routing(T, E, k, T)
        ws = torch.full((pkg.experts_w4_workspace_bytes(T, k, E, H, I),), 255, dtype=torch.uint8, device="cuda")
        for view in (big[:, :H], big[:, 3:H + 3], big[:, 8:H + 8]):
            out = torch.full((T, H), 3.0, dtype=dtype, device="cuda")
            y = check_experts(pkg, view, idx, wt, l13, l2, group, out=out, workspace=ws)
            assert y is out
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                z = pkg.experts_w4(view.contiguous(), idx, wt, l13[0], l13[1], l2[0], l2[1], w13_zero=l13[2], w2_zero=l2[2], group=group)
            s.synchronize()
            assert torch.equal(y, z)
        out, graph = torch.empty_like(y), torch.cuda.CUDAGraph()
        x = big[:, :H].contiguous()
        with torch.cuda.graph(graph):
            pkg.experts_w4(x, idx, wt, l13[0], l13[1], l2[0], l2[1], w13_zero=l13[2], w2_zero=l2[2], group=group, out=out, workspace=ws)
        x.neg_()
        idx.copy_(idx.flip(0))
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, pkg.experts_w4(x, idx, wt, l13[0], l13[1], l2[0], l2[1], w13_zero=l13[2], w2_zero=l2[2], group=group))
    assert pkg.experts_w4(x[:0], idx[:0], wt[:0], l13[0], l13[1], l2[0], l2[1], w13_zero=l13[2], w2_zero=l2[2], group=group).shape == (0, H)


def test_experts_rows_do_not_mix(pkg):
    dtype, E, H, I, group = torch.bfloat16, 4, 128, 64, 32
    l13, l2 = layer(E, H, I, group, False, dtype, 4)
    for T in (2, 8, 40):
        x = torch.randn((T, H), generator=torch.Generator().manual_seed(T)).to(dtype).cuda()
        idx, wt = routing(T, E, 2, T)
        call = lambda a: pkg.experts_w4(a, idx, wt, l13[0], l13[1], l2[0], l2[1], group=group)  # noqa: E731
        y = call(x)
        x2 = x.clone()
        x2[T - 1, 5] = float("nan")
        y2 = call(x2)
        assert torch.equal(y[:T - 1], y2[:T - 1]) and torch.isnan(y2[T - 1]).all()
        # large intermediate values that a 16-bit float of either kind must not clip
        big = pkg.experts_w4(300.0 * x, idx, wt, l13[0], l13[1], l2[0], l2[1], group=group)
        assert torch.isfinite(big).all()


def test_refusals(pkg):
    dtype = torch.bfloat16
    x = torch.zeros((3, 64), dtype=dtype, device="cuda")
    codes, scale, zero = weights((), 16, 64, 32, True, dtype, 0)
    ok = dict(x=x, codes=codes, scale=scale, zero=zero, group=32)
    for change, word in [(dict(x=x.float()), "x must"), (dict(x=x[0]), "x must"), (dict(x=x.cpu()), "x must"),
                         (dict(x=torch.zeros((64, 3), dtype=dtype, device="cuda").t()), "stride 1"),
                         (dict(x=x[:, :62]), "codes"), (dict(codes=codes.int()), "codes"), (dict(codes=codes[:, ::2]), "codes"),
                         (dict(codes=codes.cpu()), "one device"), (dict(codes=codes[0]), "codes"),
                         (dict(scale=scale.float()), "scale"), (dict(scale=scale[:, :1]), "scale"), (dict(scale=scale.half()), "scale"),
                         (dict(zero=zero[:8]), "zero"), (dict(zero=zero.int()), "zero"), (dict(zero=zero.cpu()), "zero"),
                         (dict(group=16), "group"), (dict(group=256), "group"),
                         (dict(out=torch.zeros((3, 16), device="cuda")), "out"),
                         (dict(out=torch.zeros((16, 3), dtype=dtype, device="cuda").t()), "out")]:
        with pytest.raises(RuntimeError, match=word):
            pkg.linear_w4(**{**ok, **change})
    (w13, s13, z13), (w2, s2, z2) = layer(3, 64, 32, 32, True, dtype, 0)
    idx, wt = routing(3, 3, 2, 0)
    ok = dict(x=x, idx=idx, weights=wt, w13=w13, w13_scale=s13, w2=w2, w2_scale=s2, w13_zero=z13, w2_zero=z2, group=32)
    pkg.experts_w4(**ok)
    for change, word in [(dict(x=x.float()), "x must"), (dict(x=x.half()), "scale"), (dict(idx=idx.long()), "idx"),
                         (dict(idx=idx[:2]), "idx"), (dict(weights=wt.double()), "weights"), (dict(weights=wt[:, :1]), "weights"),
                         (dict(w13=w13[:, :63]), "w13"), (dict(w13=w13[0]), "w13"), (dict(w2=w2[:2]), "w2"),
                         (dict(w2=w2.cpu()), "one device"), (dict(s13=None), "s13"), (dict(w13_scale=s13[:, :, :1]), "w13"),
                         (dict(w2_zero=z2[:, :5]), "w2"), (dict(group=48), "group"), (dict(idx=idx.cpu()), "idx"),
                         (dict(workspace=torch.zeros(8, dtype=torch.uint8, device="cuda")), "workspace"),
                         (dict(out=torch.zeros((3, 63), dtype=dtype, device="cuda")), "out")]:
        with pytest.raises((RuntimeError, TypeError), match=word):
            pkg.experts_w4(**{**ok, **change})
    native, ex = (importlib.import_module("15642_moe_b200." + n) for n in ("_native", "experts"))
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    rc = native.cuda_lib().moe_experts_w4(ex._EXPERTS(
        x.data_ptr(), idx.data_ptr(), wt.data_ptr(), w13.data_ptr(), s13.data_ptr(), 0, w2.data_ptr(), s2.data_ptr(), 0, x.data_ptr(),
        ws.data_ptr() + 16, 0, 64, 1 << 19, 1, 32, 3, 2, 3, 0, 64, 32))
    assert rc == 1 and b"256-byte aligned" in native.cuda_lib().moe_last_error()
