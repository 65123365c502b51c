"""pl_gemm_epilogue, pl_gemm_epilogue_grad and pl_bias_act_grad on the GPU, against their definitions in 64 bits."""
import ctypes as C

import pytest
import torch

from linear_util import ACTS, TORCH, TYPES, Mat, check, forward, gradient, half_step, slope_product

pytestmark = pytest.mark.gpu
NAN = float("nan")


def rand_ints(rows, cols, seed, lo=-2, hi=2):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(lo, hi + 1, (rows, cols), generator=g).double().cuda()


def rand(rows, cols, seed, kind, scale=1.0):
    """What the operand's type holds of normal values, in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, cols, generator=g, dtype=torch.float64) * scale).to(TORCH[kind]).double().cuda()


class Layout:
    """Where the operands of a test lie: extra leading dimension and the first element's offset, for all of them."""

    def __init__(self, pad=0, offset=0):
        self.pad, self.offset = pad, offset

    def put(self, values, kind):
        rows, cols = values.shape
        return Mat(rows, cols, max(1, rows + self.pad), kind, self.offset).set(values)

    def empty(self, rows, cols, kind, gap=7.0):
        return Mat(rows, cols, max(1, rows + self.pad), kind, self.offset, gap=gap).set(torch.full((rows, cols), NAN, dtype=torch.float64, device="cuda"))


def workspace(nbytes):
    return torch.full((max(int(nbytes), 16) // 8 + 2,), NAN, dtype=torch.float64, device="cuda")


def product(pkg, L, kind, ta, tb, opA, opB, *, alpha=1.0, beta=0.0, bias=None, name="none", keep=False, Cm=None, in_place=False, kind_d=None, lay=Layout(), stream=None):
    """op(A), op(B), C in 64 bits through pl_gemm_epilogue -> D, z in 64 bits."""
    kind_d = kind_d or kind
    M, K, N = opA.shape[0], opA.shape[1], opB.shape[1]
    A = lay.put(opA if ta == "N" else opA.T.contiguous(), kind)
    B = lay.put(opB if tb == "N" else opB.T.contiguous(), kind)
    D = lay.empty(M, N, kind_d)
    Cbuf = None
    if Cm is not None:
        Cbuf = D.set(Cm) if in_place else lay.put(Cm, kind_d)
    elif not in_place:
        Cbuf = lay.put(torch.full((M, N), NAN, dtype=torch.float64, device="cuda"), kind_d)   # beta == 0: never read
    Z = lay.empty(M, N, kind) if keep else None
    b = lay.put(bias[:, None], kind) if bias is not None else None
    ep = pkg.epilogue(bias=b.ptr if b else None, activation=ACTS[name], type_d=TYPES[kind_d], preact=Z.ptr if keep else None, ld_preact=Z.ld if keep else 0)
    need = L.pl_gemm_epilogue_workspace_bytes(TYPES[kind], ta.encode(), tb.encode(), M, N, K, 0)
    ws = workspace(need)
    print("pl_gemm_epilogue", kind, kind_d, ta, tb, M, N, K, alpha, beta, name, "pad", lay.pad, "offset", lay.offset, flush=True)
    s = torch.cuda.current_stream().cuda_stream if stream is None else stream
    pkg.check(L.pl_gemm_epilogue(TYPES[kind], ta.encode(), tb.encode(), M, N, K, alpha, A.ptr, A.ld, B.ptr, B.ld, C.byref(ep), beta,
                                 Cbuf.ptr if Cbuf else None, Cbuf.ld if Cbuf else 0, D.ptr, D.ld, ws.data_ptr(), need, s), "pl_gemm_epilogue")
    torch.cuda.synchronize()
    assert D.gaps_untouched() and (not keep or Z.gaps_untouched())
    return D.get(), Z.get() if keep else None


def product_grad(pkg, L, kind, ta, tb, opA, opB, Zm, *, alpha=1.0, beta=0.0, name="none", Cm=None, in_place=None, with_db=True, lay=Layout()):
    M, K, N = opA.shape[0], opA.shape[1], opB.shape[1]
    A = lay.put(opA if ta == "N" else opA.T.contiguous(), kind)
    B = lay.put(opB if tb == "N" else opB.T.contiguous(), kind)
    Z = lay.put(Zm, kind)
    D = {None: None, "C": None, "Z": Z}[in_place]
    D = D or lay.empty(M, N, kind)
    Cbuf = (D.set(Cm) if in_place == "C" else lay.put(Cm, kind)) if Cm is not None else None
    if in_place == "Z":
        Z.set(Zm)
    db = Mat(M, 1, M, kind, lay.offset, gap=5.0)
    need = L.pl_gemm_epilogue_workspace_bytes(TYPES[kind], ta.encode(), tb.encode(), M, N, K, int(with_db))
    ws = workspace(need)
    print("pl_gemm_epilogue_grad", kind, ta, tb, M, N, K, alpha, beta, name, "pad", lay.pad, "offset", lay.offset, in_place, flush=True)
    pkg.check(L.pl_gemm_epilogue_grad(TYPES[kind], ta.encode(), tb.encode(), M, N, K, alpha, A.ptr, A.ld, B.ptr, B.ld, ACTS[name], Z.ptr, Z.ld, beta,
                                      Cbuf.ptr if Cbuf else None, Cbuf.ld if Cbuf else 0, D.ptr, D.ld, db.ptr if with_db else None, ws.data_ptr(), need,
                                      torch.cuda.current_stream().cuda_stream), "pl_gemm_epilogue_grad")
    torch.cuda.synchronize()
    if in_place != "Z":
        assert D.gaps_untouched()
    assert db.gaps_untouched()
    return D.get(), db.get()[:, 0]


TRANS = [("N", "N"), ("N", "T"), ("T", "N"), ("T", "T")]
# (M, N, K): one element, tile edges from both sides, K around a panel, short and long extents of each
SHAPES = [(1, 1, 1), (8, 8, 64), (128, 128, 64), (127, 129, 63), (129, 127, 65), (256, 256, 128), (257, 255, 129), (64, 1, 4096), (1, 64, 1000),
          (300, 200, 0), (130, 5, 2000), (1000, 33, 264), (520, 776, 200), (33, 1000, 7), (4, 3, 70)]


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32", "f64"])
@pytest.mark.parametrize("ta,tb", TRANS)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_is_exact_on_integers(pkg, L, kind, ta, tb, M, N, K):
    """Small integers: every sum is exact in 32 bits, so D is the rounding of the exact result, whatever the tiles, splits
    and edges.  Bias, beta, and a relu; NaN in every gap between columns and in a C that beta = 0 must not read."""
    opA, opB, bias, Cm = rand_ints(M, K, 1), rand_ints(K, N, 2), rand_ints(M, 1, 3, -9, 9)[:, 0], rand_ints(M, N, 4, -9, 9)
    exact = 2.0 * (opA @ opB if K else torch.zeros(M, N, dtype=torch.float64, device="cuda")) + bias[:, None]
    for lay in (Layout(), Layout(pad=8), Layout(pad=3), Layout(pad=8, offset=1), Layout(pad=24, offset=8)):
        got, z = product(pkg, L, kind, ta, tb, opA, opB, alpha=2.0, bias=bias, name="relu", keep=True, lay=lay)
        assert torch.equal(z, exact.to(TORCH[kind]).double())
        assert torch.equal(got, exact.clamp(min=0).to(TORCH[kind]).double())
    lay = Layout(pad=16)
    want = (exact + 3.0 * Cm).to(TORCH[kind]).double()
    for in_place in (False, True):
        got, _ = product(pkg, L, kind, ta, tb, opA, opB, alpha=2.0, beta=3.0, bias=bias, Cm=Cm, in_place=in_place, lay=lay)
        assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(128, 256, 512), (1000, 321, 1030), (4096, 16, 256), (77, 2050, 65)])
def test_weight_gradient_accumulates_in_32_bits(pkg, L, kind, M, N, K):
    """16-bit operands into an fp32 accumulator, in place, three micro-batches in a row: exact on integers, far past what
    16 bits hold."""
    acc = rand_ints(M, N, 9, -70000, 70000)
    want = acc.clone()
    D = Mat(M, N, M + 4, "f32", gap=7.0).set(acc)
    need = L.pl_gemm_epilogue_workspace_bytes(TYPES[kind], b"N", b"T", M, N, K, 0)
    ws = workspace(need)
    ep = pkg.epilogue(type_d=TYPES["f32"])
    for step in range(3):
        a, b = rand_ints(M, K, 20 + step), rand_ints(K, N, 30 + step)
        A, B = Mat(M, K, M, kind).set(a), Mat(N, K, N, kind).set(b.T.contiguous())
        pkg.check(L.pl_gemm_epilogue(TYPES[kind], b"N", b"T", M, N, K, 1.0, A.ptr, A.ld, B.ptr, B.ld, C.byref(ep), 1.0, D.ptr, D.ld, D.ptr, D.ld, ws.data_ptr(),
                                     need, torch.cuda.current_stream().cuda_stream), "pl_gemm_epilogue")
        want += a @ b
    torch.cuda.synchronize()
    assert torch.equal(D.get(), want) and D.gaps_untouched()


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32", "f64"])
@pytest.mark.parametrize("name", list(ACTS))
@pytest.mark.parametrize("M,N,K", [(200, 130, 96), (512, 1, 1024), (1025, 70, 520)])
def test_activations(pkg, L, kind, name, M, N, K):
    opA, opB, bias, Cm = rand(M, K, 5, kind, 2.0 * K ** -0.5), rand(K, N, 6, kind), rand(M, 1, 7, kind)[:, 0], rand(M, N, 8, kind)
    z, ez, y, ey = forward(opA, opB, bias, Cm, 1.25, -0.5, name, kind, kind)
    got, zs = product(pkg, L, kind, "T", "N", opA, opB, alpha=1.25, beta=-0.5, bias=bias, name=name, keep=True, Cm=Cm)
    check(zs, z, ez, "z")
    check(got, y, ey, "y")
    if kind in ("bf16", "f16"):
        got, _ = product(pkg, L, kind, "T", "N", opA, opB, bias=bias, name=name, kind_d="f32")
        z, ez, y, ey = forward(opA, opB, bias, None, 1.0, 0.0, name, kind, "f32")
        check(got, y, ey, "y in 32 bits")


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32", "f64"])
@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu"])
def test_activations_and_slopes_at_their_ends(pkg, L, kind, name):
    """Values from the subnormal to the largest: act(z) -> z or 0 and act'(z) -> 1 or 0 without 0 * inf on the way."""
    big = float(torch.finfo(TORCH[kind]).max)
    zs = torch.tensor([0.0, -0.0, 1e-7, -1e-7, 0.5, -0.5, 3.0, -3.0, 8.0, -8.0, 11.0, -11.0, 30.0, -30.0, 300.0, -300.0, 6e4, -6e4, big, -big], dtype=torch.float64, device="cuda")
    zs = zs.to(TORCH[kind]).double()
    one = torch.ones(1, 1, dtype=torch.float64, device="cuda")
    z, ez, y, ey = forward(zs[:, None], one, None, None, 1.0, 0.0, name, kind, kind)
    got, _ = product(pkg, L, kind, "N", "N", zs[:, None].contiguous(), one, name=name)
    y = torch.where(zs[:, None].abs() > 1e15, zs[:, None].clamp(min=0), y)   # (z^3 leaves 64 bits)
    check(got, y, ey.nan_to_num(nan=1e-30, posinf=1e300), "y")
    M = zs.numel()
    dz, db = act_grad(pkg, L, kind, name, torch.ones(M, 1, dtype=torch.float64, device="cuda"), zs[:, None])
    d, ed, _, _ = slope_product(torch.ones(M, 1, dtype=torch.float64, device="cuda"), torch.zeros(M, 1, dtype=torch.float64, device="cuda"), zs[:, None].clamp(-40, 40), name, kind)
    check(dz, d, ed, "slope")


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32", "f64"])
@pytest.mark.parametrize("name", list(ACTS))
@pytest.mark.parametrize("ta,tb,M,N,K", [("N", "N", 300, 257, 130), ("N", "N", 129, 1, 64), ("T", "N", 64, 1000, 200), ("N", "T", 1030, 40, 333)])
def test_gradient_through_the_activation(pkg, L, kind, name, ta, tb, M, N, K):
    opA, opB, Z, Cm = rand(M, K, 11, kind, K ** -0.5), rand(K, N, 12, kind), rand(M, N, 13, kind, 2.0), rand(M, N, 14, kind)
    for lay, beta, in_place in ((Layout(), 0.0, None), (Layout(pad=5, offset=3), 0.75, None), (Layout(pad=8), 0.75, "C"), (Layout(), 0.0, "Z")):
        d, ed, db, edb = gradient(opA, opB, Z, Cm, 0.5, beta, name, kind)
        got, gdb = product_grad(pkg, L, kind, ta, tb, opA, opB, Z, alpha=0.5, beta=beta, name=name, Cm=Cm if beta else None, in_place=in_place, lay=lay)
        check(got, d, ed, "D")
        check(gdb, db, edb, "dbias")


def test_gradient_without_dbias_and_dbias_of_nothing(pkg, L):
    opA, opB, Z = rand(40, 30, 1, "bf16"), rand(30, 20, 2, "bf16"), rand(40, 20, 3, "bf16")
    d, ed, _, _ = gradient(opA, opB, Z, None, 1.0, 0.0, "silu", "bf16")
    got, db = product_grad(pkg, L, "bf16", "N", "N", opA, opB, Z, name="silu", with_db=False)
    check(got, d, ed, "D")
    assert torch.isnan(db).all() or bool((db != 0).all())            # not written
    # no columns: the sum over them is zero, no rows: nothing to do
    db = torch.full((40,), NAN, dtype=torch.bfloat16, device="cuda")
    one = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    pkg.check(L.pl_gemm_epilogue_grad(3, b"N", b"N", 40, 0, 1, 1.0, one.data_ptr(), 40, one.data_ptr(), 1, 4, one.data_ptr(), 40, 0.0, None, 0, one.data_ptr(), 40,
                                      db.data_ptr(), None, 0, torch.cuda.current_stream().cuda_stream), "N == 0")
    assert bool((db == 0).all())
    db.fill_(NAN)
    pkg.check(L.pl_bias_act_grad(3, 4, 40, 0, None, 40, None, 40, None, 40, db.data_ptr(), None, 0, torch.cuda.current_stream().cuda_stream), "N == 0")
    assert bool((db == 0).all())


def act_grad(pkg, L, kind, name, dYm, Zm, *, lay=Layout(), with_db=True, with_dz=True, in_place=None):
    M, N = dYm.shape
    dY, Z = lay.put(dYm, kind), lay.put(Zm, kind)
    dZ = {None: None, "dY": dY, "Z": Z}[in_place] or lay.empty(M, N, kind)
    db = Mat(M, 1, M, kind, lay.offset, gap=5.0).set(torch.full((M, 1), NAN, dtype=torch.float64, device="cuda"))
    need = L.pl_bias_act_grad_workspace_bytes(TYPES[kind], M, N) if with_db else 0
    ws = workspace(need)
    print("pl_bias_act_grad", kind, name, M, N, "pad", lay.pad, "offset", lay.offset, in_place, flush=True)
    pkg.check(L.pl_bias_act_grad(TYPES[kind], ACTS[name], M, N, dY.ptr, dY.ld, Z.ptr, Z.ld, dZ.ptr if with_dz else None, dZ.ld, db.ptr if with_db else None,
                                 ws.data_ptr() if with_db else None, need, torch.cuda.current_stream().cuda_stream), "pl_bias_act_grad")
    torch.cuda.synchronize()
    if in_place is None:
        assert dZ.gaps_untouched()
    assert db.gaps_untouched()
    return dZ.get(), db.get()[:, 0]


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32", "f64"])
@pytest.mark.parametrize("name", list(ACTS))
@pytest.mark.parametrize("M,N", [(1, 1), (1, 3000), (517, 9), (2048, 64), (1031, 517), (7, 8), (513, 4097)])
def test_gradient_of_bias_and_activation(pkg, L, kind, name, M, N):
    dY, Z = rand(M, N, 21, kind), rand(M, N, 22, kind, 2.0)
    d, ed, db, edb = slope_product(dY, torch.zeros_like(dY), Z, name, kind)
    for lay, in_place in ((Layout(), None), (Layout(pad=1, offset=3), None), (Layout(pad=8), "dY"), (Layout(), "Z")):
        got, gdb = act_grad(pkg, L, kind, name, dY, Z, lay=lay, in_place=in_place)
        check(got, d, ed, "dZ")
        check(gdb, db, edb, "dbias")
    got, _ = act_grad(pkg, L, kind, name, dY, Z, with_db=False)
    check(got, d, ed, "dZ alone")
    _, gdb = act_grad(pkg, L, kind, name, dY, Z, with_dz=False)
    check(gdb, db, edb, "dbias alone")


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_infinities_and_nan_go_where_the_formula_sends_them(pkg, L, kind):
    """One NaN and one infinity among the operands reach their own row or column of D and nothing else."""
    M, N, K = 140, 150, 100
    opA, opB = rand_ints(M, K, 1, 1, 2), rand_ints(K, N, 2, 1, 2)
    clean, _ = product(pkg, L, kind, "T", "N", opA, opB)
    a = opA.clone()
    a[3, 7] = NAN
    b = opB.clone()
    b[99, 149] = float("inf")
    got, _ = product(pkg, L, kind, "T", "N", a, b)
    assert torch.isnan(got[3]).all() and torch.isinf(got[:, 149][torch.arange(M) != 3]).all()
    keep = torch.ones(M, N, dtype=torch.bool)
    keep[3], keep[:, 149] = False, False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_alpha_zero_and_k_zero_do_not_read_the_operands(pkg, L, kind):
    M, N = 70, 50
    nan = torch.full((M, 30), NAN, dtype=torch.float64, device="cuda")
    bias = rand_ints(M, 1, 3)[:, 0]
    got, _ = product(pkg, L, kind, "N", "N", nan, torch.full((30, N), NAN, dtype=torch.float64, device="cuda"), alpha=0.0, bias=bias)
    assert torch.equal(got, bias[:, None].expand(M, N).to(TORCH[kind]).double())


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_row_ranges_of_larger_matrices(pkg, L, kind):
    """Operands and results that are row ranges of packed buffers (three projections side by side): only the named rows
    are read and written."""
    M, N, K = 192, 75, 160
    w, x = rand_ints(K, 3 * M, 1), rand_ints(2 * K, N, 2)
    W, X = Mat(K, 3 * M, K, kind).set(w), Mat(2 * K, N, 2 * K, kind).set(x)
    D = Mat(3 * M, N, 3 * M, kind).set(torch.full((3 * M, N), 5.0, dtype=torch.float64, device="cuda"))
    ep = pkg.epilogue(type_d=TYPES[kind])
    need = L.pl_gemm_epilogue_workspace_bytes(TYPES[kind], b"T", b"N", M, N, K, 0)
    ws = workspace(need)
    size = 2
    pkg.check(L.pl_gemm_epilogue(TYPES[kind], b"T", b"N", M, N, K, 1.0, W.ptr + M * K * size, K, X.ptr + K * size, 2 * K, C.byref(ep), 0.0, None, 0,
                                 D.ptr + M * size, 3 * M, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream), "pl_gemm_epilogue")
    torch.cuda.synchronize()
    want = torch.full((3 * M, N), 5.0, dtype=torch.float64, device="cuda")
    want[M:2 * M] = (w[:, M:2 * M].T @ x[K:]).to(TORCH[kind]).double()
    assert torch.equal(D.get(), want)


def test_results_repeat_bit_for_bit(pkg, L):
    opA, opB, Z = rand(700, 900, 1, "bf16"), rand(900, 90, 2, "bf16"), rand(700, 90, 3, "bf16")
    first = product_grad(pkg, L, "bf16", "N", "N", opA, opB, Z, name="gelu")
    for _ in range(3):
        again = product_grad(pkg, L, "bf16", "N", "N", opA, opB, Z, name="gelu")
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
