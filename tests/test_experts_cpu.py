"""Host side of the expert router and the 4-bit products: the C ABI refuses bad arguments before any launch, the Python
layer refuses CPU tensors, and the 64-bit oracle agrees with differences and with itself."""
import ctypes
import importlib

import numpy as np
import pytest

from oracle import experts_oracle as X


@pytest.fixture(scope="module")
def lib(pkg):
    return importlib.import_module("15642_moe_b200._native").cuda_lib()


@pytest.fixture(scope="module")
def ptr():
    buf = (ctypes.c_uint8 * 4096)()
    return (ctypes.addressof(buf) + 255) & ~255, buf


def test_router_refuses(lib, ptr):
    p = ptr[0]
    ex = importlib.import_module("15642_moe_b200.experts")
    call = lambda dtype=0, T=4, E=64, k=4, score=0, ng=1, tg=1, gs=0, lg=p: lib.moe_route_experts(  # noqa: E731
        ex._ROUTE(lg, 0, p, p, 0, 64, dtype, T, E, k, score, ng, tg, gs, 1, 1.0))
    for kw, word in [(dict(dtype=3), b"dtype"), (dict(T=-1), b"[T, E]"), (dict(E=0), b"[T, E]"), (dict(E=1025), b"[T, E]"),
                     (dict(k=0), b"top_k"), (dict(k=33), b"top_k"), (dict(k=9, ng=8), b"top_k"), (dict(ng=3), b"n_group"),
                     (dict(ng=64), b"n_group"), (dict(ng=4, tg=5), b"topk_group"), (dict(score=2), b"score"),
                     (dict(E=32, ng=32, tg=8, gs=1), b"two"), (dict(lg=0), b"null")]:
        assert call(**kw) == 1 and word in lib.moe_last_error(), kw
    assert call(T=0, lg=0) == 0
    assert lib.moe_route_experts(None) == 1 and b"null" in lib.moe_last_error()
    back = lambda dtype=0, T=4, E=64, k=4, score=0, g=p: lib.moe_route_experts_backward(  # noqa: E731
        ex._ROUTE_BACKWARD(g, p, p, p, 0, 64, dtype, T, E, k, score, 1, 1.0))
    for kw, word in [(dict(dtype=-1), b"dtype"), (dict(E=0), b"[T, E]"), (dict(k=33), b"top_k"), (dict(score=5), b"score"),
                     (dict(g=0), b"null")]:
        assert back(**kw) == 1 and word in lib.moe_last_error(), kw
    assert back(T=0) == 0
    assert lib.moe_route_experts_backward(None) == 1


def test_products_refuse(lib, ptr):
    p = ptr[0]
    ex = importlib.import_module("15642_moe_b200.experts")
    call = lambda dtype=1, group=128, M=2, N=8, K=64, x=p, out=p + 2048: lib.moe_linear_w4(  # noqa: E731
        ex._LINEAR(x, p, p, 0, out, 0, 0, 64, 0, dtype, group, M, N, K))
    for kw, word in [(dict(dtype=0), b"bf16"), (dict(group=16), b"group"), (dict(M=-1), b"[M, K]"), (dict(M=65536), b"65535"),
                     (dict(M=60000, K=70000), b"2^31"), (dict(N=0), b"[M, K]"), (dict(K=0), b"[M, K]"), (dict(x=0), b"null"),
                     (dict(out=p + 64), b"overlaps")]:
        assert call(**kw) == 1 and word in lib.moe_last_error(), kw
    assert call(M=0) == 0
    assert call(M=9) == 3 and b"workspace too small" in lib.moe_last_error()
    assert lib.moe_linear_w4_workspace_bytes(8, 64, 64) == 0 and lib.moe_linear_w4_workspace_bytes(9, 64, 64) > 0
    assert lib.moe_linear_w4(None) == 1 and b"null" in lib.moe_last_error()
    call = lambda dtype=1, group=128, T=2, k=2, E=4, H=64, I=32, ws=p, n=0, x=p, w2=p, off=0: lib.moe_experts_w4(  # noqa: E731
        ex._EXPERTS(x, p, p, p, p, 0, w2, p, 0, p, ws, 0, 64, n, dtype, group, T, k, E, off, H, I))
    for kw, word in [(dict(dtype=0), b"bf16"), (dict(group=1), b"group"), (dict(T=65536), b"65535"), (dict(k=0), b"top_k"),
                     (dict(E=1025), b"E must"), (dict(H=0), b"H and I"), (dict(x=0), b"null"), (dict(ws=0), b"null"),
                     (dict(w2=p + 8), b"16-byte"), (dict(off=-1), b"local_offset"), (dict(n=1 << 40), b"overlaps")]:
        assert call(**kw) == 1 and word in lib.moe_last_error(), kw
    assert call(n=16) == 3 and b"workspace too small" in lib.moe_last_error()
    assert call(T=0) == 0
    need = lib.moe_experts_w4_workspace_bytes(2, 2, 4, 64, 32)
    assert need > 0 and lib.moe_experts_w4_workspace_bytes(65535, 32, 256, 7168, 2048) > need
    assert lib.moe_experts_w4_workspace_bytes(65536, 2, 4, 64, 32) == 0
    assert call(ws=p + 16, n=1 << 40) == 1 and b"256-byte aligned" in lib.moe_last_error()
    assert lib.moe_experts_w4(None) == 1


def test_packed_arguments_have_the_structs_layout():
    """Sizes of the packed arguments against the header's structs, compiled by a C compiler."""
    import os
    import struct
    import subprocess
    import tempfile
    ex = importlib.import_module("15642_moe_b200.experts")
    names = ["moe_route_experts_args", "moe_route_experts_backward_args", "moe_linear_w4_args", "moe_experts_w4_args"]
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "a.c"), os.path.join(d, "a")
        with open(src, "w") as f:
            f.write('#include <stdio.h>\n#include <stddef.h>\n#include "moe_b200.h"\nint main(void) {\n'
                    + "".join('printf("%%zu ", sizeof(%s));\n' % n for n in names)
                    + 'printf("%zu %zu %zu %zu", offsetof(moe_route_experts_args, scale), offsetof(moe_route_experts_backward_args, scale),'
                      ' offsetof(moe_linear_w4_args, K), offsetof(moe_experts_w4_args, I));\nreturn 0; }\n')
        subprocess.run(["gcc", "-I", os.path.join(repo, "include"), "-o", exe, src], check=True)
        got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    packs = [ex._ROUTE.__self__, ex._ROUTE_BACKWARD.__self__, ex._LINEAR.__self__, ex._EXPERTS.__self__]
    for size, at, pack in zip(got[:4], got[4:], packs):
        assert pack.size - struct.calcsize("i") == at and pack.size <= size <= pack.size + 4   # the struct's own padding


def test_python_layer_refuses_cpu_tensors(pkg):
    import torch
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.route_experts(torch.zeros((2, 8)), 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.linear_w4(torch.zeros((2, 8), dtype=torch.bfloat16), torch.zeros((4, 4), dtype=torch.uint8),
                      torch.zeros((4, 1), dtype=torch.bfloat16))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_oracle_gradient_against_differences(score, renormalize):
    rng = np.random.default_rng(0)
    x, g = rng.normal(size=(6, 20)), rng.normal(size=(6, 5))
    idx, w = X.route(x, 5, score, renormalize=renormalize, scale=2.5)
    grad = X.route_grad(g, x, idx, score, renormalize, 2.5)
    f = lambda z: (g * X.weights(X.scores(z, score), idx, renormalize, 2.5)).sum(1)  # noqa: E731
    for e in range(20):
        d = np.zeros_like(x)
        d[:, e] = 1e-6
        np.testing.assert_allclose(grad[:, e], (f(x + d) - f(x - d)) / 2e-6, atol=1e-8)
    assert (np.diff(np.take_along_axis(X.picks(x, score)[1], idx, 1)) <= 0).all() and w.shape == idx.shape


def test_oracle_agrees_with_the_fixed_router(oracle):
    rng = np.random.default_rng(1)
    x, b = rng.normal(size=(300, 256)).astype(np.float32), (0.1 * rng.normal(size=256)).astype(np.float32)
    idx, w = X.route(x, 8, "sigmoid", b, 8, 4, "top2", True, 2.5)
    ridx, rw = oracle.route(x, b, 2.5)
    same = (idx == ridx).all(1)
    assert same.mean() > 0.99
    np.testing.assert_allclose(w[same], rw[same], rtol=1e-6)
