"""Host side of the expert operators at the edges of what their integers hold. Nothing here launches a kernel."""
import ctypes
import importlib

import pytest

INT_MAX = 2 ** 31 - 1


@pytest.fixture(scope="module")
def lib(pkg):
    return importlib.import_module("15642_moe_b200._native").cuda_lib()


@pytest.fixture(scope="module")
def ex(pkg):
    return importlib.import_module("15642_moe_b200.experts")


@pytest.fixture(scope="module")
def p():
    buf = (ctypes.c_uint8 * 4096)()
    yield (ctypes.addressof(buf) + 255) & ~255


def test_columns_beyond_the_limit_are_refused(lib, ex, p):
    """Rounding a column count up to whole steps must stay inside 32 bits."""
    far = 1 << 50                                                      # an output that overlaps nothing
    linear = lambda M=2, N=8, K=64: lib.moe_linear_w4(  # noqa: E731
        ex._LINEAR(p, p, p, 0, far, far // 2, 0, K, 1 << 62, 1, 128, M, N, K))
    for M in (1, 8, 9, 65535):
        for K in (INT_MAX, INT_MAX - 1, INT_MAX - 62, INT_MAX - 254):
            assert linear(M=M, K=K) == 1 and b"moe_linear_w4" in lib.moe_last_error(), (M, K)
            assert lib.moe_linear_w4_workspace_bytes(M, 8, K) == 0
        assert linear(M=M, N=INT_MAX, K=2) == 1 and b"moe_linear_w4" in lib.moe_last_error()
    experts = lambda E=1, H=64, I=64: lib.moe_experts_w4(  # noqa: E731
        ex._EXPERTS(p, p, p, p, p, 0, p, p, 0, far, far // 2, 0, H, 1 << 62, 1, 128, 2, 2, E, 0, H, I))
    for big in (INT_MAX, INT_MAX - 62, INT_MAX - 254, 2 ** 30 + 1):
        for kw in (dict(H=big), dict(I=big)):
            assert experts(**kw) == 1 and b"moe_experts_w4" in lib.moe_last_error(), kw
        assert lib.moe_experts_w4_workspace_bytes(2, 2, 1, big, 64) == 0
        assert lib.moe_experts_w4_workspace_bytes(2, 2, 1, 64, big) == 0


def test_workspace_sizes_up_to_the_limit(lib):
    """Sizes of widths that need no copy of the codes grow up to the largest that is taken."""
    sizes = [lib.moe_linear_w4_workspace_bytes(9, 8, K) for K in (64, 4096, 2 ** 20, 2 ** 27)]
    assert sizes == sorted(sizes) and sizes[0] > 0 and sizes[-1] >= 9 * 2 ** 27 * 2
    sizes = [lib.moe_experts_w4_workspace_bytes(2, 2, 1, H, 64) for H in (64, 4096, 2 ** 20, 2 ** 30)]
    assert sizes == sorted(sizes) and sizes[0] > 0 and sizes[-1] >= 4 * 2 ** 30 * (2 + 4)


def test_a_workspace_over_an_input_is_refused(lib, ex, p):
    """Every input in turn lies in the workspace's first or last bytes."""
    far = lambda i: (1 << 50) + (i << 24)  # noqa: E731
    M, N, K = 9, 8, 64
    need = lib.moe_linear_w4_workspace_bytes(M, N, K)
    ws = far(20)
    for at in range(4):                                                # x, codes, scale, zero
        for place in (ws, ws + need - 1):
            a = [far(i) for i in range(4)]
            a[at] = place
            rc = lib.moe_linear_w4(ex._LINEAR(*a, far(10), ws, 0, K, need, 1, 32, M, N, K))
            assert rc == 1 and b"workspace overlaps an input" in lib.moe_last_error(), at
    T, k, E, H, I = 2, 2, 4, 64, 32
    need = lib.moe_experts_w4_workspace_bytes(T, k, E, H, I)
    for at in range(9):                                                # x, idx, weights, w13, scale, zero, w2, scale, zero
        for place in (ws, ws + need // 256 * 256 - 256):
            a = [far(i) for i in range(9)]
            a[at] = place
            rc = lib.moe_experts_w4(ex._EXPERTS(*a, far(10), ws, 0, H, need, 1, 32, T, k, E, 0, H, I))
            assert rc == 1 and b"workspace overlaps an input" in lib.moe_last_error(), at


def test_calls_hand_over_whole_structs(ex, monkeypatch):
    """The C side copies its struct, padding at the end included: the bytes handed over must be as many."""
    P, L, I, F = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int, ctypes.c_float
    monkeypatch.setattr(ex.torch.cuda, "current_device", lambda: 0)
    for pack, members in ((ex._ROUTE, [P] * 5 + [L] + [I] * 9 + [F]), (ex._ROUTE_BACKWARD, [P] * 5 + [L] + [I] * 6 + [F]),
                          (ex._LINEAR, [P] * 7 + [L] * 2 + [I] * 5), (ex._EXPERTS, [P] * 12 + [L] * 2 + [I] * 8)):
        layout = type("Args", (ctypes.Structure,), {"_fields_": [("m%d" % i, t) for i, t in enumerate(members)]})
        args, seen = pack(*(1.5 if t is F else i for i, t in enumerate(members))), []
        ex._call(lambda a: seen.append(a) or 0, 0, args)
        assert len(seen[0]) >= ctypes.sizeof(layout) and seen[0].startswith(args)
