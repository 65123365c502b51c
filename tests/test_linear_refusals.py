"""What the linear-layer operators and the gradient norm refuse, on the host and before anything is launched: no device
is needed to see the status codes, and pl_last_error() names the entry point."""
import ctypes as C
import random

import pytest

from linear_util import shipped_fit, takes_copies

A, B, CM, D, Z, DB, WS = (0x10000000 * i for i in range(1, 8))   # addresses nobody dereferences


def call(L, pkg, **over):
    a = dict(type=3, ta=b"T", tb=b"N", M=64, N=32, K=16, alpha=1.0, A=A, lda=16, B=B, ldb=16, beta=0.0, C=None, ldc=0, D=D, ldd=64, ws=None, wsb=0,
             bias=None, act=0, type_d=None, preact=None, ldp=0, ep=True)
    a.update(over)
    ep = pkg.epilogue(bias=a["bias"], activation=a["act"], type_d=a["type"] if a["type_d"] is None else a["type_d"], preact=a["preact"], ld_preact=a["ldp"])
    return L.pl_gemm_epilogue(a["type"], a["ta"], a["tb"], a["M"], a["N"], a["K"], a["alpha"], a["A"], a["lda"], a["B"], a["ldb"],
                              C.byref(ep) if a["ep"] else None, a["beta"], a["C"], a["ldc"], a["D"], a["ldd"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("over,code", [
    (dict(ep=False), 5), (dict(type=4), 7), (dict(type=-1), 7), (dict(type=1, type_d=0), 7), (dict(type=3, type_d=2), 7), (dict(act=5), 7), (dict(act=-1), 7),
    (dict(ta=b"X"), 1), (dict(tb=b"C"), 1), (dict(M=-1), 2), (dict(K=-1), 2), (dict(N=1 << 31), 2), (dict(M=1 << 21, N=1 << 21), 2),
    (dict(lda=15), 3), (dict(ta=b"N", lda=63), 3), (dict(ldb=15), 3), (dict(tb=b"T", ldb=31), 3), (dict(ldd=63), 3), (dict(beta=1.0, C=CM, ldc=63), 3),
    (dict(preact=Z, ldp=63), 3), (dict(A=None), 5), (dict(B=None), 5), (dict(D=None), 5), (dict(beta=1.0), 3), (dict(beta=1.0, ldc=64), 5),
    (dict(A=A + 1), 7), (dict(D=D + 1), 7), (dict(bias=Z + 1), 7), (dict(preact=Z + 1, ldp=64), 7), (dict(type_d=1, D=D + 2), 7),
    (dict(D=A), 7), (dict(D=B + 64), 7), (dict(preact=D, ldp=64), 7), (dict(preact=A, ldp=64), 7), (dict(beta=1.0, C=D + 2, ldc=64), 7),
    (dict(beta=1.0, C=D, ldc=65), 7), (dict(beta=1.0, C=CM, ldc=64, preact=CM, ldp=64), 7), (dict(bias=D), 7), (dict(bias=Z, preact=Z, ldp=64), 7),
])
def test_product_refuses(pkg, L, over, code):
    assert call(L, pkg, **over) == code
    assert b"pl_gemm_epilogue:" in L.pl_last_error()


@pytest.mark.parametrize("M,N,K", [(2048, 2048, 2048), (512, 8, 512)])
def test_workspace_of_32_and_64_bit_products(pkg, L, M, N, K):
    """A large product passes through the workspace, a long and narrow one in slices; a small one needs none."""
    for kind in (0, 1):
        need = L.pl_gemm_epilogue_workspace_bytes(kind, b"T", b"N", M, N, K, 0)
        assert need >= M * N * (8 if kind == 0 else 4)
        assert L.pl_gemm_epilogue_workspace_bytes(kind, b"T", b"N", M, N, K, 1) > need
        shape = dict(M=M, N=N, K=K, lda=K, ldb=K, ldd=M)
        assert call(L, pkg, type=kind, ws=None, wsb=0, **shape) == 7
        assert call(L, pkg, type=kind, ws=WS, wsb=need - 1, **shape) == 7
        assert call(L, pkg, type=kind, ws=WS + 8, wsb=need, **shape) == 7
        assert L.pl_gemm_epilogue_workspace_bytes(kind, b"T", b"N", 64, 32, 16, 0) == 0
        assert L.pl_gemm_epilogue_workspace_bytes(kind, b"T", b"N", 64, 32, 16, 1) >= 64 * (8 if kind == 0 else 4)
    assert L.pl_gemm_epilogue_workspace_bytes(9, b"T", b"N", 64, 32, 16, 0) == 0
    assert L.pl_gemm_epilogue_workspace_bytes(3, b"T", b"N", 0, 32, 16, 1) == 0


def grad(L, **over):
    a = dict(type=3, ta=b"N", tb=b"N", M=64, N=32, K=16, alpha=1.0, A=A, lda=64, B=B, ldb=16, act=2, Z=Z, ldz=64, beta=0.0, C=None, ldc=0, D=D, ldd=64, db=DB, ws=WS, wsb=1 << 20)
    a.update(over)
    return L.pl_gemm_epilogue_grad(a["type"], a["ta"], a["tb"], a["M"], a["N"], a["K"], a["alpha"], a["A"], a["lda"], a["B"], a["ldb"], a["act"], a["Z"], a["ldz"],
                                   a["beta"], a["C"], a["ldc"], a["D"], a["ldd"], a["db"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("over,code", [
    (dict(type=7), 7), (dict(act=9), 7), (dict(Z=None), 5), (dict(ldz=63), 3), (dict(ws=None), 7), (dict(wsb=8), 7), (dict(ws=WS + 4), 7), (dict(db=D), 7),
    (dict(db=Z), 7), (dict(db=A), 7), (dict(db=DB + 1), 7), (dict(Z=D + 2), 7), (dict(Z=D, ldz=65), 7), (dict(Z=Z + 1), 7), (dict(D=B), 7), (dict(ta=b"H"), 1),
])
def test_product_gradient_refuses(L, over, code):
    assert grad(L, **over) == code
    assert b"pl_gemm_epilogue_grad:" in L.pl_last_error()


def act_grad(L, **over):
    a = dict(type=3, act=2, M=64, N=32, dY=A, lddy=64, Z=Z, ldz=64, dZ=D, lddz=64, db=DB, ws=WS, wsb=1 << 20)
    a.update(over)
    return L.pl_bias_act_grad(a["type"], a["act"], a["M"], a["N"], a["dY"], a["lddy"], a["Z"], a["ldz"], a["dZ"], a["lddz"], a["db"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("over,code", [
    (dict(type=-1), 7), (dict(act=5), 7), (dict(M=-1), 2), (dict(N=1 << 31), 2), (dict(lddy=63), 3), (dict(ldz=63), 3), (dict(lddz=63), 3), (dict(dY=None), 5),
    (dict(Z=None), 5), (dict(dZ=None, db=None), 5), (dict(dY=A + 1), 7), (dict(db=DB + 1), 7), (dict(ws=None), 5), (dict(wsb=16), 7), (dict(ws=WS + 8), 7),
    (dict(dZ=A + 2), 7), (dict(dZ=Z + 64), 7), (dict(dZ=A, lddz=65), 7), (dict(db=D + 64), 7),
])
def test_bias_and_activation_gradient_refuses(L, over, code):
    assert act_grad(L, **over) == code
    assert b"pl_bias_act_grad:" in L.pl_last_error()


def clip(L, ptrs, counts, types, outs, max_norm=1.0, eps=1e-6, norm=DB, ws=WS, wsb=None, n=None):
    n_ = len(ptrs) if n is None else n
    vp, ll, it = (C.c_void_p * len(ptrs))(*ptrs), (C.c_longlong * len(ptrs))(*counts), (C.c_int * len(ptrs))(*types)
    ov = (C.c_void_p * len(ptrs))(*outs) if outs is not None else None
    return L.pl_grad_norm_clip(n_, vp, ll, it, ov, max_norm, eps, norm, ws, L.pl_grad_norm_workspace_bytes(n_) if wsb is None else wsb, None)


def test_gradient_clipping_refuses(L):
    good = ([A, B], [100, 200], [1, 3], [A, B])
    nan = float("nan")
    for over, code in ((dict(n=-1), 2), (dict(max_norm=-1.0), 7), (dict(max_norm=nan), 7), (dict(eps=-1.0), 7), (dict(eps=nan), 7), (dict(norm=None), 5), (dict(norm=DB + 4), 7),
                       (dict(ws=None), 7), (dict(ws=WS + 8), 7), (dict(wsb=8), 7)):
        assert clip(L, *good, **over) == code, over
        assert b"pl_grad_norm_clip:" in L.pl_last_error()
    assert clip(L, [A, B], [100, -1], [1, 3], [A, B]) == 2
    assert clip(L, [A, B], [100, 1 << 38], [1, 3], [A, B]) == 2
    assert clip(L, [A, B], [100, 200], [1, 4], [A, B]) == 7
    assert clip(L, [A, None], [100, 200], [1, 3], [A, B]) == 5
    assert clip(L, [A, B], [100, 200], [1, 3], [A, None]) == 5
    assert clip(L, [A, B], [100, 200], [1, 3], None) == 5
    assert clip(L, [A + 2, B], [100, 200], [1, 3], [A + 2, B]) == 7          # not a multiple of its element size
    # written twice, or written over another tensor's gradients: in place and out of place, in any order of the list
    assert clip(L, [A, A], [100, 100], [1, 1], [A, A]) == 7
    assert clip(L, [A, A + 4], [100, 100], [1, 1], [A, A + 4]) == 7
    assert clip(L, [B, A, A + 396], [10, 100, 100], [1, 1, 1], [B, A, A + 396]) == 7
    assert clip(L, [A, B], [100, 100], [1, 1], [CM, CM + 200]) == 7
    assert clip(L, [A, B], [100, 100], [1, 1], [B, CM]) == 7
    assert clip(L, [A, B], [100, 100], [1, 1], [A + 4, B]) == 7
    assert b"written" in L.pl_last_error()
    ptrs, counts, types = (C.c_void_p * 1)(A), (C.c_longlong * 1)(10), (C.c_int * 1)(1)
    assert L.pl_grad_norm(1, None, counts, types, DB, WS, 1 << 20, None) == 5
    assert L.pl_grad_norm(1, ptrs, counts, types, None, WS, 1 << 20, None) == 5
    assert L.pl_grad_clip(1, ptrs, counts, types, ptrs, 1.0, 0.0, None, None) == 5
    assert L.pl_grad_clip(1, ptrs, counts, types, None, 1.0, 0.0, DB, None) == 5
    assert L.pl_grad_clip(0, None, None, None, None, 1.0, 0.0, DB, None) == 0
    assert L.pl_grad_norm_workspace_bytes(0) == 0 and L.pl_grad_norm_workspace_bytes(1) >= 8192


def test_workspaces_that_overlap_operands_are_refused(pkg, L):
    need = L.pl_gemm_epilogue_workspace_bytes(3, b"N", b"N", 64, 32, 16, 1)
    for at in (A, B + 128, D - need + 16, Z, DB - 16):
        assert grad(L, ws=at & ~15, wsb=1 << 20) == 7, hex(at)
        assert b"workspace" in L.pl_last_error()
    for at in (A, Z, D, DB):
        assert act_grad(L, ws=at, wsb=1 << 20) == 7
    assert act_grad(L, db=A + 64) == 7 and act_grad(L, db=Z) == 7
    for over in (dict(norm=A + 8), dict(norm=B + 392), dict(ws=A), dict(ws=A - 4096)):
        assert clip(L, [A, B], [100, 200], [1, 3], [A, B], **over) == 7
        assert b"overlaps a tensor" in L.pl_last_error()


def test_a_norm_inside_the_workspace_is_refused(L):
    """The scaling reads the workspace's partial sums while its first workgroup stores the norm."""
    need = L.pl_grad_norm_workspace_bytes(2)
    ptrs, counts, types = (C.c_void_p * 2)(A, B), (C.c_longlong * 2)(100, 200), (C.c_int * 2)(1, 3)
    for norm in (WS, WS + 8, WS + need - 8):
        assert clip(L, [A, B], [100, 200], [1, 3], [A, B], norm=norm) == 7, hex(norm)
        assert b"pl_grad_norm_clip: norm overlaps the workspace" in L.pl_last_error()
        assert L.pl_grad_norm(2, ptrs, counts, types, norm, WS, need, None) == 7, hex(norm)
        assert b"pl_grad_norm: norm overlaps the workspace" in L.pl_last_error()
    # right behind the bytes that a call uses it is taken: the next check answers
    assert clip(L, [A, B], [100, 200], [1, 3], [A, B], norm=WS + need, max_norm=-1.0) == 7
    assert b"max_norm" in L.pl_last_error()


def test_rows_beyond_the_fold(L):
    assert act_grad(L, M=(1 << 27) + 1, N=1, lddy=1 << 28, ldz=1 << 28, lddz=1 << 28) == 2
    assert grad(L, M=(1 << 27) + 1, N=1, K=1, lda=1 << 28, ldz=1 << 28, ldd=1 << 28) == 2


def test_nothing_to_do_is_no_error(pkg, L):
    assert call(L, pkg, M=0, lda=16, ldd=1) == 0
    assert call(L, pkg, N=0) == 0
    assert act_grad(L, M=0) == 0
    assert act_grad(L, N=0, db=None) == 0


def test_the_workspace_is_a_function_of_the_shape_alone(pkg, L, monkeypatch):
    """What a program asked for at its start is enough after a routine has installed the database's launcher constants, and
    whatever the environment pins for the routines' own products."""
    rng = random.Random(7)
    shapes = [(0, b"T", b"N", 128, 1216, 5824), (1, b"T", b"N", 256, 6848, 1024), (1, b"N", b"T", 2560, 400, 384), (0, b"N", b"T", 5516, 74, 2205)]
    for _ in range(4000):
        shapes.append((rng.choice([0, 1]), rng.choice([b"N", b"T"]), rng.choice([b"N", b"T"]), *(int(round(2 ** rng.uniform(3, 13))) for _ in range(3))))
    ask = lambda: [L.pl_gemm_epilogue_workspace_bytes(*s, db) for s in shapes for db in (0, 1)]  # noqa: E731
    before = ask()
    try:
        assert L.pl_gemm_set_fit(C.byref(shipped_fit(pkg, L))) == 0
        assert ask() == before
        for s, need in list(zip(shapes, before[::2]))[:4]:
            if need == 0:
                continue
            kind, ta, tb, M, N, K = s
            # (an operand inside the workspace, so that the check behind its size answers, and nothing is launched)
            over = dict(type=kind, ta=ta, tb=tb, M=M, N=N, K=K, lda=max(M, K), ldb=max(N, K), ldd=M, A=WS, ws=WS, wsb=need, D=WS * 16)
            assert call(L, pkg, **over) == 7
            assert b"overlaps an operand" in L.pl_last_error()
    finally:
        assert L.pl_gemm_set_fit(None) == 0
    for name, value in (("PARALIA_GEMM_TAIL", "0"), ("PARALIA_GEMM_LARGE_TILE", "0"), ("PARALIA_GEMM_LARGE_TILE", "1"), ("PARALIA_GEMM_LARGE_TILE", "2")):
        with monkeypatch.context() as m:
            m.setenv(name, value)
            assert ask() == before, (name, value)


@pytest.mark.parametrize("ta", ["N", "T"])
@pytest.mark.parametrize("tb", ["N", "T"])
def test_which_products_are_multiplied_from_copies(L, ta, tb):
    """Measured on 68 shapes both ways: large products of odd extents are faster from copies in the tile GEMM's tiles, small and
    narrow ones in 64 x 64 tiles."""
    for kind, M, N, K in (("f32", 3878, 1869, 4113), ("f32", 829, 10936, 2184), ("f32", 10936, 829, 2184), ("f32", 2253, 1029, 2616), ("f32", 3400, 1809, 424),
                          ("f32", 5991, 921, 5269), ("f32", 2061, 6226, 1334), ("f64", 3878, 1869, 4113), ("f64", 5510, 4977, 663)):
        assert takes_copies(L, kind, ta, tb, M, N, K), (kind, M, N, K)
    for kind, M, N, K in (("f32", 605, 195, 174), ("f64", 605, 195, 174), ("f32", 10474, 17, 2943), ("f64", 2304, 300, 1024), ("f32", 4893, 190, 1539)):
        assert not takes_copies(L, kind, ta, tb, M, N, K), (kind, M, N, K)


def test_a_failed_launch_says_so(pkg, L):
    """Without a device every launch fails: the status says so and pl_last_error() is this call's, not an older one's."""
    count = C.c_int(0)
    if L.pl_device_count(C.byref(count)) == 0 and count.value > 0:
        pytest.skip("a device would run kernels on these addresses")
    big = 1 << 30
    calls = {"few columns": lambda: call(L, pkg, K=64, lda=64, ldb=64), "tiles": lambda: call(L, pkg, ta=b"N", lda=64), "64 x 64": lambda: call(L, pkg, type=1),
             "tile GEMM": lambda: call(L, pkg, type=0, M=2048, N=2048, K=2048, lda=2048, ldb=2048, ldd=2048, B=16 * B, D=32 * D, ws=64 * WS, wsb=big),
             "its epilogue": lambda: call(L, pkg, type=0, act=1, M=2048, N=2048, K=2048, lda=2048, ldb=2048, ldd=2048, B=16 * B, D=32 * D, ws=64 * WS, wsb=big),
             "gradient": lambda: grad(L), "activation": lambda: act_grad(L), "clipping": lambda: clip(L, [A, B], [100, 200], [1, 3], [A, B]),
             "no columns": lambda: act_grad(L, N=0)}
    for name, f in calls.items():
        assert act_grad(L, type=-1) == 7 and b"unknown element type" in L.pl_last_error()
        assert f() == 4, name
        assert b"launch" in L.pl_last_error(), name
