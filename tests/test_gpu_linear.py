"""pl_gemm_epilogue, pl_gemm_epilogue_grad and pl_bias_act_grad on the GPU, against their definitions in 64 bits."""
import ctypes as C
import math

import pytest
import torch

from linear_util import ACTS, TORCH, TYPES, Mat, act, act_error, check, forward, gradient, half_step, shipped_fit, slope_product, takes_copies

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


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("ta,tb,M,N,K", [("T", "N", 300, 2, 64), ("N", "N", 300, 80, 64), ("T", "T", 2048, 2048, 72), ("N", "N", 256, 256, 4096), ("N", "N", 300, 9, 3)])
def test_activations_into_32_bits(pkg, L, kind, name, ta, tb, M, N, K):
    """An fp32 D of 16-bit operands shows what 16 bits would hide: the activation of an exact z to the accuracy of fp32 (few
    columns, tiles, large tiles, slices, thin rows)."""
    z = torch.linspace(-9.0, 9.0, M, dtype=torch.float64, device="cuda").to(TORCH[kind]).double()
    opA, opB = torch.zeros(M, K, dtype=torch.float64, device="cuda"), torch.zeros(K, N, dtype=torch.float64, device="cuda")
    opA[:, 1], opB[1] = z, 1.0
    got, _ = product(pkg, L, kind, ta, tb, opA, opB, name=name, kind_d="f32")
    y, bound = act(z, name), act_error(z, name, "f32")
    if name == "gelu":
        # (torch's ndtr loses the lower tail, -9 Phi(-9) = -1.0157e-18; erfc keeps it.)  u = 2^-24: 4 for an erfc of 2 ulp, 2 (1 + z^2) for the
        # two roundings of its argument, 1 for the product
        y, bound = z * 0.5 * torch.erfc(z * -0.5 ** 0.5), (8 + 2 * z * z) * 2.0 ** -24
    y, bound = y[:, None].expand(M, N), bound[:, None]
    check(got, y, bound * y.abs() + half_step(y, "f32"), "y")


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


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32", "f64"])
def test_a_closed_relu_lets_nothing_through(pkg, L, kind):
    """Infinite and NaN gradients where z <= 0 are zeros of D and add nothing to dbias; where z > 0 they arrive."""
    M, N, K = 150, 70, 40
    g, Z = rand_ints(M, N, 1, 1, 9), rand_ints(M, N, 2, -3, 3)
    closed = Z <= 0
    bad = g.clone()
    bad[closed & (rand_ints(M, N, 3) > 0)] = float("inf")
    bad[closed & (rand_ints(M, N, 3) < 0)] = NAN
    want = torch.where(closed, torch.zeros_like(g), g)
    for lay, in_place in ((Layout(), None), (Layout(pad=3, offset=1), None), (Layout(), "dY"), (Layout(), "Z")):
        got, db = act_grad(pkg, L, kind, "relu", bad, Z, lay=lay, in_place=in_place)
        assert torch.equal(got, want) and torch.equal(db, want.sum(1).to(TORCH[kind]).double())
    # the same arriving in C, in front of a product
    opA, opB = rand_ints(M, K, 4), rand_ints(K, N, 5)
    want = torch.where(closed, torch.zeros_like(g), g + opA @ opB)
    got, db = product_grad(pkg, L, kind, "T", "N", opA, opB, Z, beta=1.0, Cm=bad, name="relu")
    assert torch.equal(got, want.to(TORCH[kind]).double()) and torch.equal(db, want.sum(1).to(TORCH[kind]).double())
    open_ = g.clone()
    m, n = (Z > 0).nonzero()[0].tolist()
    open_[m, n] = float("inf")
    got, db = act_grad(pkg, L, kind, "relu", open_, Z)
    assert torch.isinf(got[m, n]) and torch.isinf(db[m]) and int(torch.isinf(got).sum()) == 1


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_alpha_zero_and_k_zero_do_not_read_the_operands(pkg, L, kind):
    M, N = 70, 50
    nan = torch.full((M, 30), NAN, dtype=torch.float64, device="cuda")
    bias = rand_ints(M, 1, 3)[:, 0]
    got, _ = product(pkg, L, kind, "N", "N", nan, torch.full((30, N), NAN, dtype=torch.float64, device="cuda"), alpha=0.0, bias=bias)
    assert torch.equal(got, bias[:, None].expand(M, N).to(TORCH[kind]).double())


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", [(128, 1, 8192), (128, 130, 8192), (40, 3, 5), (700, 300, 1001)])
def test_an_empty_gradient_stays_inside_its_workspace(pkg, L, kind, M, N, K):
    """alpha = 0 where the product would be split, copied or thin: dZ = beta C act'(Z), its sums, and nothing behind the
    workspace."""
    Cm, Z = rand_ints(M, N, 1, -9, 9), rand_ints(M, N, 2, -3, 3)
    Cb, Zb, D, db = Mat(M, N, M, kind).set(Cm), Mat(M, N, M, kind).set(Z), Mat(M, N, M, kind, gap=7.0), Mat(M, 1, M, kind, gap=5.0)
    need = L.pl_gemm_epilogue_workspace_bytes(TYPES[kind], b"N", b"N", M, N, K, 1)
    ws = torch.full((need + 8192,), 0xA5, dtype=torch.uint8, device="cuda")
    pkg.check(L.pl_gemm_epilogue_grad(TYPES[kind], b"N", b"N", M, N, K, 0.0, None, M, None, K, ACTS["relu"], Zb.ptr, M, 2.0, Cb.ptr, M, D.ptr, M, db.ptr, ws.data_ptr(), need,
                                      torch.cuda.current_stream().cuda_stream), "pl_gemm_epilogue_grad")
    torch.cuda.synchronize()
    want = 2.0 * Cm * (Z > 0)
    assert torch.equal(D.get(), want) and torch.equal(db.get()[:, 0], want.sum(1).to(TORCH[kind]).double())
    assert bool((ws[need:] == 0xA5).all())


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


@pytest.mark.parametrize("kind,ta,tb,M,N,K", [("f64", "T", "N", 128, 1216, 5824), ("f32", "T", "N", 256, 6848, 1024), ("f32", "N", "T", 2560, 400, 384), ("f64", "N", "T", 5516, 74, 2205)])
def test_results_do_not_depend_on_the_routines_constants(pkg, L, kind, ta, tb, M, N, K):
    """The same bits before and after a routine has installed the database's launcher constants, in the workspace asked for
    before."""
    opA, opB, Z = rand(M, K, 1, kind, K ** -0.5), rand(K, N, 2, kind), rand(M, N, 3, kind)
    first, plain = product_grad(pkg, L, kind, ta, tb, opA, opB, Z, name="silu"), product(pkg, L, kind, ta, tb, opA, opB)
    need = [L.pl_gemm_epilogue_workspace_bytes(TYPES[kind], ta.encode(), tb.encode(), M, N, K, db) for db in (0, 1)]
    try:
        assert L.pl_gemm_set_fit(C.byref(shipped_fit(pkg, L))) == 0
        assert need == [L.pl_gemm_epilogue_workspace_bytes(TYPES[kind], ta.encode(), tb.encode(), M, N, K, db) for db in (0, 1)]
        again = product_grad(pkg, L, kind, ta, tb, opA, opB, Z, name="silu")
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
        assert torch.equal(plain[0], product(pkg, L, kind, ta, tb, opA, opB)[0])
    finally:
        assert L.pl_gemm_set_fit(None) == 0


# ---- the launcher's other ways: large tiles, split K, few columns, copies of unaligned operands ----

def exact_product(pkg, L, kind, ta, tb, M, N, K, lay, kind_d=None, seed=1):
    opA, opB, bias = rand_ints(M, K, seed), rand_ints(K, N, seed + 1), rand_ints(M, 1, seed + 2, -9, 9)[:, 0]
    exact = opA @ opB + bias[:, None]
    got, z = product(pkg, L, kind, ta, tb, opA, opB, bias=bias, name="relu", keep=True, lay=lay, kind_d=kind_d)
    assert torch.equal(z, exact.to(TORCH[kind]).double())
    assert torch.equal(got, exact.clamp(min=0).to(TORCH[kind_d or kind]).double())


@pytest.mark.parametrize("kind,kind_d", [("bf16", None), ("f16", "f32")])
@pytest.mark.parametrize("ta,tb", TRANS)
@pytest.mark.parametrize("M,N,K", [(4096, 4096, 200), (4104, 4072, 648), (4100, 4099, 129), (2600, 8200, 321)])
def test_large_products(pkg, L, kind, kind_d, ta, tb, M, N, K):
    """Enough 256 x 256 tiles for every compute unit: whole and ragged, aligned and (pad 1) not."""
    for lay in (Layout(), Layout(pad=8), Layout(pad=1, offset=1)):
        exact_product(pkg, L, kind, ta, tb, M, N, K, lay, kind_d)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("ta,tb", TRANS)
@pytest.mark.parametrize("M,N,K", [(256, 256, 4096), (128, 130, 8200), (257, 100, 5000), (1030, 70, 3001), (700, 300, 1001), (520, 1500, 2047)])
def test_split_and_copied_products(pkg, L, kind, ta, tb, M, N, K):
    """Few tiles and a long K; extents that are no multiple of 8, whose operands are copied."""
    for lay in (Layout(), Layout(pad=8), Layout(pad=3, offset=5)):
        exact_product(pkg, L, kind, ta, tb, M, N, K, lay)
    opA, opB, Z = rand(M, K, 31, kind, K ** -0.5), rand(K, N, 32, kind), rand(M, N, 33, kind, 2.0)
    d, ed, db, edb = gradient(opA, opB, Z, None, 1.0, 0.0, "gelu_tanh", kind)
    got, gdb = product_grad(pkg, L, kind, ta, tb, opA, opB, Z, name="gelu_tanh", lay=Layout(pad=1))
    check(got, d, ed, "D")
    check(gdb, db, edb, "dbias")


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 31, 32, 33])
@pytest.mark.parametrize("M,K", [(5, 64), (100, 4096), (4100, 576), (5000, 64), (16400, 320), (33000, 128)])
def test_few_columns(pkg, L, kind, N, M, K):
    """Single tokens and small batches: fewer panels than waves, a panel count that does not divide, ragged last rows."""
    exact_product(pkg, L, kind, "T", "N", M, N, K, Layout())
    exact_product(pkg, L, kind, "T", "N", M, N, K, Layout(pad=8), kind_d="f32", seed=4)
    opA, opB, Cm = rand_ints(M, K, 7), rand_ints(K, N, 8), rand_ints(M, N, 9, -9, 9)
    got, _ = product(pkg, L, kind, "T", "N", opA, opB, alpha=2.0, beta=-1.0, Cm=Cm, in_place=True)
    assert torch.equal(got, (2.0 * (opA @ opB) - Cm).to(TORCH[kind]).double())


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(300, 9, 4103), (4263, 2, 1387), (130, 32, 2051), (600, 33, 1999)])
def test_few_columns_of_unaligned_operands(pkg, L, kind, M, N, K):
    """Odd strides and a ragged k: multiplied from copies whose k is filled up to whole panels."""
    for lay in (Layout(), Layout(pad=1), Layout(pad=3, offset=5)):
        exact_product(pkg, L, kind, "T", "N", M, N, K, lay)
    exact_product(pkg, L, kind, "T", "N", M, N, K, Layout(pad=1), kind_d="f32", seed=4)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("ta,tb,M,N,K", [("N", "T", 4096, 1, 16384), ("N", "T", 770, 7, 20001), ("T", "T", 300, 3, 17000), ("T", "T", 9, 1, 100003), ("N", "N", 5, 300, 16391),
                                         ("N", "T", 3, 2, 65537), ("N", "N", 1, 64, 500), ("N", "T", 2, 5, 129), ("T", "N", 300, 200, 7), ("N", "N", 7, 70001, 65)])
def test_products_of_rows_below_eight_elements(pkg, L, kind, ta, tb, M, N, K):
    """The weight gradient of a head with one to seven outputs over many tokens, and its like: K in slices, exact on whole
    numbers, close on normal ones, with nothing behind the workspace."""
    for lay in (Layout(), Layout(pad=1), Layout(pad=3, offset=5)):
        exact_product(pkg, L, kind, ta, tb, M, N, K, lay, kind_d="f32")
    opA, opB, bias, Cm = rand(M, K, 5, kind, 2.0 * K ** -0.5), rand(K, N, 6, kind), rand(M, 1, 7, kind)[:, 0], rand(M, N, 8, "f32")
    z, ez, y, ey = forward(opA, opB, bias, Cm, 1.25, -0.5, "silu", kind, "f32")
    got, zs = product(pkg, L, kind, ta, tb, opA, opB, alpha=1.25, beta=-0.5, bias=bias, name="silu", keep=True, Cm=Cm, kind_d="f32")
    check(zs, z, ez, "z")
    check(got, y, ey, "y")
    Z = rand(M, N, 33, kind, 2.0)
    d, ed, db, edb = gradient(opA, opB, Z, None, 1.0, 0.0, "gelu", kind)
    got, gdb = product_grad(pkg, L, kind, ta, tb, opA, opB, Z, name="gelu", lay=Layout(pad=1))
    check(got, d, ed, "D")
    check(gdb, db, edb, "dbias")


def test_the_gradient_of_one_output_costs_no_more_than_that_of_eight(pkg, L):
    """4096 features, 16384 tokens, into fp32: rows of one element are no 16-byte vectors, and were summed by one thread per
    element over all tokens (1346 us against 37)."""
    M, K = 4096, 16384
    x = torch.randn(K, M, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").bfloat16()
    ep, best = pkg.epilogue(type_d=TYPES["f32"]), {}
    for N in (1, 7, 8):
        dy, g = torch.randn(K, N, device="cuda").bfloat16(), torch.zeros(N, M, device="cuda")
        need = L.pl_gemm_epilogue_workspace_bytes(3, b"N", b"T", M, N, K, 0)
        ws, times = workspace(need), []
        for _ in range(8):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            pkg.check(L.pl_gemm_epilogue(3, b"N", b"T", M, N, K, 1.0, x.data_ptr(), M, dy.data_ptr(), N, C.byref(ep), 0.0, None, 0, g.data_ptr(), M, ws.data_ptr(), need,
                                         stream()), "pl_gemm_epilogue")
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        best[N] = min(times[2:])
    print(best, flush=True)
    assert best[1] <= 3 * best[8] and best[7] <= 5 * best[8]


@pytest.mark.parametrize("kind", ["f32", "f64"])
@pytest.mark.parametrize("ta,tb", TRANS)
@pytest.mark.parametrize("M,N,K", [(256, 256, 4096), (1700, 1500, 1600), (700, 300, 1001)])
def test_wide_products_split_and_cut(pkg, L, kind, ta, tb, M, N, K):
    for lay in (Layout(), Layout(pad=1)):
        exact_product(pkg, L, kind, ta, tb, M, N, K, lay)
    opA, opB = rand_ints(M, K, 7), rand_ints(K, N, 8)
    Cm, Z = rand_ints(M, N, 9, -9, 9), rand_ints(M, N, 10, -3, 3)
    for in_place in (False, True):
        got, _ = product(pkg, L, kind, ta, tb, opA, opB, alpha=3.0, beta=2.0, Cm=Cm, in_place=in_place)
        assert torch.equal(got, 3.0 * (opA @ opB) + 2.0 * Cm)
    got, db = product_grad(pkg, L, kind, ta, tb, opA, opB, Z, name="relu")
    want = (opA @ opB) * (Z > 0)
    assert torch.equal(got, want) and torch.equal(db, want.sum(1))


@pytest.mark.parametrize("kind,M,N,K", [("f32", 1501, 1301, 2003), ("f32", 3000, 130, 8192), ("f32", 8193, 2050, 257), ("f64", 2501, 2001, 2003), ("f64", 1280, 5001, 1536)])
@pytest.mark.parametrize("ta,tb", TRANS)
def test_wide_products_of_unaligned_operands(pkg, L, kind, ta, tb, M, N, K):
    """Large enough to be multiplied from aligned copies: ragged extents, and whole ones in rows of an odd stride."""
    for lay in (Layout(pad=1), Layout(pad=3, offset=1)):
        exact_product(pkg, L, kind, ta, tb, M, N, K, lay)
    opA, opB, Cm = rand_ints(M, K, 7), rand_ints(K, N, 8), rand_ints(M, N, 9, -9, 9)
    got, _ = product(pkg, L, kind, ta, tb, opA, opB, alpha=2.0, beta=-1.0, Cm=Cm, in_place=True, lay=Layout(pad=1))
    assert torch.equal(got, 2.0 * (opA @ opB) - Cm)
    opA, opB, Z = rand(M, K, 31, kind, K ** -0.5), rand(K, N, 32, kind), rand(M, N, 33, kind, 2.0)
    d, ed, db, edb = gradient(opA, opB, Z, None, 1.0, 0.0, "gelu_tanh", kind)
    got, gdb = product_grad(pkg, L, kind, ta, tb, opA, opB, Z, name="gelu_tanh", lay=Layout(pad=1))
    check(got, d, ed, "D")
    check(gdb, db, edb, "dbias")


@pytest.mark.parametrize("kind,M,N,K", [("f32", 2061, 1803, 1003), ("f32", 3400, 1809, 424), ("f32", 2100, 2052, 1500), ("f64", 2305, 2305, 1301)])
@pytest.mark.parametrize("ta,tb", TRANS)
def test_wide_products_from_copies(pkg, L, kind, ta, tb, M, N, K):
    """Products that do set space aside for copies, none with a K of whole panels: what fills it up has to count as zero,
    whatever lies behind the operands' rows and in the workspace (NaN, both)."""
    assert takes_copies(L, kind, ta, tb, M, N, K) and K % 32 != 0
    for lay in (Layout(), Layout(pad=1), Layout(pad=3, offset=1), Layout(pad=4)):
        exact_product(pkg, L, kind, ta, tb, M, N, K, lay)
    opA, opB, Cm = rand_ints(M, K, 7), rand_ints(K, N, 8), rand_ints(M, N, 9, -9, 9)
    for lay in (Layout(), Layout(pad=1)):
        got, _ = product(pkg, L, kind, ta, tb, opA, opB, alpha=2.0, beta=-1.0, Cm=Cm, in_place=True, lay=lay)   # (nothing but the product)
        assert torch.equal(got, 2.0 * (opA @ opB) - Cm)
    opA, opB, Z = rand(M, K, 31, kind, K ** -0.5), rand(K, N, 32, kind), rand(M, N, 33, kind, 2.0)
    d, ed, db, edb = gradient(opA, opB, Z, None, 1.0, 0.0, "gelu_tanh", kind)
    got, gdb = product_grad(pkg, L, kind, ta, tb, opA, opB, Z, name="gelu_tanh", lay=Layout(pad=1))
    check(got, d, ed, "D")
    check(gdb, db, edb, "dbias")


@pytest.mark.parametrize("kind", ["f32", "f64"])
@pytest.mark.parametrize("ta,tb", TRANS)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 70, 33), (65, 1, 16), (300, 200, 3), (605, 195, 174), (512, 8, 512), (3001, 17, 700), (64, 129, 2050)])
def test_small_wide_products(pkg, L, kind, ta, tb, M, N, K):
    """64 x 64 tiles: one element, one row, one column, less than a panel of k, whole panels and one more, K split."""
    for lay in (Layout(), Layout(pad=1), Layout(pad=3, offset=1)):
        exact_product(pkg, L, kind, ta, tb, M, N, K, lay)
    opA, opB, Cm = rand_ints(M, K, 7), rand_ints(K, N, 8), rand_ints(M, N, 9, -9, 9)
    got, _ = product(pkg, L, kind, ta, tb, opA, opB, alpha=2.0, beta=-1.0, Cm=Cm, in_place=True)
    assert torch.equal(got, 2.0 * (opA @ opB) - Cm)
    opA, opB, Z, Cm = rand(M, K, 31, kind, K ** -0.5), rand(K, N, 32, kind), rand(M, N, 33, kind, 2.0), rand(M, N, 34, kind)
    for name in ("none", "relu", "gelu"):
        d, ed, db, edb = gradient(opA, opB, Z, Cm, 1.0, 0.5, name, kind)
        got, gdb = product_grad(pkg, L, kind, ta, tb, opA, opB, Z, beta=0.5, Cm=Cm, name=name, lay=Layout(pad=1))
        check(got, d, ed, "D")
        check(gdb, db, edb, "dbias")


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("ta,tb,M,N,K", [("T", "N", 700, 300, 1001), ("N", "N", 256, 256, 4096), ("N", "T", 300, 200, 64), ("T", "T", 3, 5, 9), ("N", "N", 2051, 1701, 2003), ("T", "N", 605, 195, 174), ("N", "N", 512, 8, 512)])
def test_nothing_is_written_behind_the_workspace(pkg, L, kind, ta, tb, M, N, K):
    opA, opB, Z = rand_ints(M, K, 1), rand_ints(K, N, 2), rand_ints(M, N, 3)
    A, B = Mat(*((M, K) if ta == "N" else (K, M)), M if ta == "N" else K, kind).set(opA if ta == "N" else opA.T), Mat(*((K, N) if tb == "N" else (N, K)), K if tb == "N" else N, kind).set(opB if tb == "N" else opB.T)
    Zb, D, db = Mat(M, N, M, kind).set(Z), Mat(M, N, M, kind, gap=7.0), Mat(M, 1, M, kind, gap=5.0)
    need = L.pl_gemm_epilogue_workspace_bytes(TYPES[kind], ta.encode(), tb.encode(), M, N, K, 1)
    ws = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    pkg.check(L.pl_gemm_epilogue_grad(TYPES[kind], ta.encode(), tb.encode(), M, N, K, 1.0, A.ptr, A.ld, B.ptr, B.ld, ACTS["relu"], Zb.ptr, M, 0.0, None, 0, D.ptr, M, db.ptr,
                                      ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream), "pl_gemm_epilogue_grad")
    torch.cuda.synchronize()
    assert bool((ws[need:] == 0xA5).all())
    want = (opA @ opB) * (Z > 0)
    assert torch.equal(D.get(), want.to(TORCH[kind]).double()) and torch.equal(db.get()[:, 0], want.sum(1).to(TORCH[kind]).double())


@pytest.mark.parametrize("ta,tb", TRANS)
def test_leading_dimensions_beyond_the_request_offsets(pkg, L, ta, tb):
    """Columns 2^22 + 8 elements apart: what 32-bit offsets from a panel's start cannot span."""
    M, N, K, ld = 20, 24, 20, (1 << 22) + 8
    opA, opB = rand_ints(M, K, 1), rand_ints(K, N, 2)
    A = Mat(*((M, K) if ta == "N" else (K, M)), ld, "bf16").set(opA if ta == "N" else opA.T)
    B = Mat(*((K, N) if tb == "N" else (N, K)), ld, "bf16").set(opB if tb == "N" else opB.T)
    D = Mat(M, N, ld, "bf16", gap=7.0)
    ep = pkg.epilogue(type_d=3)
    need = L.pl_gemm_epilogue_workspace_bytes(3, ta.encode(), tb.encode(), M, N, K, 0)
    ws = workspace(need)
    pkg.check(L.pl_gemm_epilogue(3, ta.encode(), tb.encode(), M, N, K, 1.0, A.ptr, ld, B.ptr, ld, C.byref(ep), 0.0, None, 0, D.ptr, ld, ws.data_ptr(), need,
                                 torch.cuda.current_stream().cuda_stream), "pl_gemm_epilogue")
    assert torch.equal(D.get(), (opA @ opB).to(torch.bfloat16).double()) and D.gaps_untouched()


def test_a_result_beyond_4_gib(pkg, L):
    """70000 x 40000 in 16 bits, 5.6 GB, with its gradient: rows and columns far behind 2^32 bytes."""
    M, N, K = 70000, 40000, 64
    g = torch.Generator(device="cuda").manual_seed(5)
    w = torch.randint(-2, 3, (M, K), generator=g, device="cuda").to(torch.bfloat16)
    x = torch.randint(-2, 3, (N, K), generator=g, device="cuda").to(torch.bfloat16)
    y = torch.full((N, M), 9.0, dtype=torch.bfloat16, device="cuda")
    ep = pkg.epilogue(type_d=3, activation=ACTS["relu"])
    s = torch.cuda.current_stream().cuda_stream
    need = L.pl_gemm_epilogue_workspace_bytes(3, b"T", b"N", M, N, K, 0)
    ws = workspace(need)
    pkg.check(L.pl_gemm_epilogue(3, b"T", b"N", M, N, K, 1.0, w.data_ptr(), K, x.data_ptr(), K, C.byref(ep), 0.0, None, 0, y.data_ptr(), M, ws.data_ptr(), need, s), "pl_gemm_epilogue")
    rows = torch.tensor([0, 1, 255, 256, 20000, 30679, 30680, 39999], device="cuda")
    assert torch.equal(y[rows].float(), (x[rows].float() @ w.float().T).clamp(min=0))
    db = torch.zeros(M, dtype=torch.bfloat16, device="cuda")
    need = L.pl_bias_act_grad_workspace_bytes(3, M, N)
    ws = workspace(need)
    before = y[rows].clone()
    pkg.check(L.pl_bias_act_grad(3, ACTS["relu"], M, N, y.data_ptr(), M, y.data_ptr(), M, y.data_ptr(), M, db.data_ptr(), ws.data_ptr(), need, s), "pl_bias_act_grad")
    assert torch.equal(y[rows], before)
    # whole numbers: columns summed in 32 bits are exact (below 2^24)
    some = torch.tensor([0, 1, 35000, M - 1], device="cuda")
    assert torch.equal(db[some].float(), y[:, some].float().sum(0).to(torch.bfloat16).float())


# ---- as they are used together ----

class Layer2:
    """Two linear layers with an activation between them, row-major as a program holds them: the calls of a training step."""

    def __init__(self, pkg, L, kind, tokens, width, hidden, name, seed):
        self.pkg, self.L, self.kind, self.t, self.w, self.h, self.name = pkg, L, kind, tokens, width, hidden, name
        self.code, self.act = TYPES[kind], ACTS[name]
        g = torch.Generator().manual_seed(seed)
        new = lambda *shape, scale=1.0: (torch.randn(*shape, generator=g, dtype=torch.float64) * scale).to(TORCH[kind]).cuda()  # noqa: E731
        self.x, self.r, self.dy = new(tokens, width), new(tokens, width), new(tokens, width, scale=0.1)
        self.w1, self.b1 = new(hidden, width, scale=width ** -0.5), new(hidden, scale=0.3)
        self.w2, self.b2 = new(width, hidden, scale=hidden ** -0.5), new(width, scale=0.3)
        z = lambda *shape, t=kind: torch.zeros(*shape, dtype=TORCH[t], device="cuda")  # noqa: E731
        wide = "f64" if kind == "f64" else "f32"
        self.wide = wide
        self.z1, self.a1, self.y = z(tokens, hidden), z(tokens, hidden), z(tokens, width)
        self.dz1, self.dx = z(tokens, hidden), z(tokens, width)
        self.gb1, self.gb2 = z(hidden), z(width)
        self.gw1, self.gw2 = z(hidden, width, t=wide), z(width, hidden, t=wide)
        self.norm = torch.zeros(1, dtype=torch.float64, device="cuda")
        q = lambda ta, tb, m, n, k, d: L.pl_gemm_epilogue_workspace_bytes(self.code, ta, tb, m, n, k, d)  # noqa: E731
        need = max(q(b"T", b"N", hidden, tokens, width, 0), q(b"T", b"N", width, tokens, hidden, 0), q(b"N", b"N", hidden, tokens, width, 1), q(b"N", b"N", width, tokens, hidden, 0),
                   q(b"N", b"T", hidden, width, tokens, 0), q(b"N", b"T", width, hidden, tokens, 0), L.pl_bias_act_grad_workspace_bytes(self.code, width, tokens), L.pl_grad_norm_workspace_bytes(4))
        self.need, self.ws = need, workspace(need)
        grads = [self.gw1, self.gb1, self.gw2, self.gb2]
        self.n = len(grads)
        self.ptrs, self.counts = (C.c_void_p * 4)(*[t.data_ptr() for t in grads]), (C.c_longlong * 4)(*[t.numel() for t in grads])
        self.types = (C.c_int * 4)(TYPES[wide], self.code, TYPES[wide], self.code)

    def gemm(self, s, ta, tb, m, n, k, a, b, d, ep, beta=0.0, c=None):
        ld = lambda t: t.stride(0)  # noqa: E731
        self.pkg.check(self.L.pl_gemm_epilogue(self.code, ta, tb, m, n, k, 1.0, a.data_ptr(), ld(a), b.data_ptr(), ld(b), C.byref(ep), beta, c.data_ptr() if c is not None else None,
                                               ld(c) if c is not None else 0, d.data_ptr(), ld(d), self.ws.data_ptr(), self.need, s), "pl_gemm_epilogue")

    def step(self, s, limit):
        pkg, L, t, w, h = self.pkg, self.L, self.t, self.w, self.h
        ep = pkg.epilogue
        up = ep(bias=self.b1.data_ptr(), activation=self.act, type_d=self.code, preact=self.z1.data_ptr(), ld_preact=h)
        self.gemm(s, b"T", b"N", h, t, w, self.w1, self.x, self.a1, up)
        self.gemm(s, b"T", b"N", w, t, h, self.w2, self.a1, self.y, ep(bias=self.b2.data_ptr(), type_d=self.code), beta=1.0, c=self.r)
        pkg.check(L.pl_bias_act_grad(self.code, 0, w, t, self.dy.data_ptr(), w, None, 0, None, 0, self.gb2.data_ptr(), self.ws.data_ptr(), self.need, s), "db2")
        pkg.check(L.pl_gemm_epilogue_grad(self.code, b"N", b"N", h, t, w, 1.0, self.w2.data_ptr(), h, self.dy.data_ptr(), w, self.act, self.z1.data_ptr(), h, 0.0, None, 0,
                                          self.dz1.data_ptr(), h, self.gb1.data_ptr(), self.ws.data_ptr(), self.need, s), "dz1")
        wide = ep(type_d=TYPES[self.wide])
        self.gemm(s, b"N", b"T", h, w, t, self.a1, self.dy, self.gw2, wide, beta=1.0, c=self.gw2)
        self.gemm(s, b"N", b"T", w, h, t, self.x, self.dz1, self.gw1, wide, beta=1.0, c=self.gw1)
        self.gemm(s, b"N", b"N", w, t, h, self.w1, self.dz1, self.dx, ep(type_d=self.code))
        pkg.check(L.pl_grad_norm_clip(self.n, self.ptrs, self.counts, self.types, self.ptrs, limit, 1e-6, self.norm.data_ptr(), self.ws.data_ptr(), self.need, s), "clip")

    def outputs(self):
        return [t.clone() for t in (self.y, self.z1, self.a1, self.dz1, self.dx, self.gw1, self.gw2, self.gb1, self.gb2, self.norm)]


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu"])
def test_a_training_step_against_differences(pkg, L, name):
    """fp64, 5 tokens: every gradient of loss = sum(dy * y) against central differences of the library's own forward pass.
    With a step of 1e-6 the differences are off by about 1e-12 (third derivatives) + 1e-16 * |loss| / 1e-6."""
    m = Layer2(pkg, L, "f64", 5, 6, 9, name, 3)
    m.step(stream(), 1e30)
    torch.cuda.synchronize()
    grads = {"w1": m.gw1.clone(), "b1": m.gb1.clone(), "w2": m.gw2.clone(), "b2": m.gb2.clone(), "x": m.dx.clone()}
    assert abs(float(m.norm) - math.sqrt(sum(float((grads[k] ** 2).sum()) for k in ("w1", "b1", "w2", "b2")))) < 1e-12
    for k, g in grads.items():
        p = getattr(m, k)
        flat, want = p.view(-1), []
        for i in range(flat.numel()):
            old = float(flat[i])
            loss = []
            for e in (1e-6, -1e-6):
                flat[i] = old + e
                up = pkg.epilogue(bias=m.b1.data_ptr(), activation=m.act, type_d=0)
                m.gemm(stream(), b"T", b"N", m.h, m.t, m.w, m.w1, m.x, m.a1, up)
                m.gemm(stream(), b"T", b"N", m.w, m.t, m.h, m.w2, m.a1, m.y, pkg.epilogue(bias=m.b2.data_ptr(), type_d=0), beta=1.0, c=m.r)
                loss.append(float((m.y * m.dy).sum()))
            flat[i] = old
            want.append((loss[0] - loss[1]) / 2e-6)
        want = torch.tensor(want, dtype=torch.float64, device="cuda").view(g.shape)
        assert float((g - want).abs().max()) < 1e-8, k


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tokens,width,hidden", [(64, 128, 256), (333, 136, 1000), (37, 130, 259)])
def test_a_training_step_against_64_bits(pkg, L, kind, tokens, width, hidden):
    """A whole step, each call held to its definition on what the call before it really left."""
    m = Layer2(pkg, L, kind, tokens, width, hidden, "gelu_tanh", 5)
    m.step(stream(), 1e30)
    torch.cuda.synchronize()
    T = lambda t: t.double().T  # noqa: E731
    x, w1, w2, dy = (t.double() for t in (m.x, m.w1, m.w2, m.dy))
    z, ez, a, ea = forward(w1, x.T, m.b1.double(), None, 1.0, 0.0, "gelu_tanh", kind, kind)
    check(T(m.z1), z, ez, "z1")
    check(T(m.a1), a, ea, "a1")
    _, _, y, ey = forward(w2, T(m.a1), m.b2.double(), m.r.double().T, 1.0, 1.0, "none", kind, kind)
    check(T(m.y), y, ey, "y")
    d, ed, db, edb = gradient(w2.T, dy.T, T(m.z1), None, 1.0, 0.0, "gelu_tanh", kind)
    check(T(m.dz1), d, ed, "dz1")
    check(m.gb1.double(), db, edb, "gb1")
    wide = "f32"
    _, _, g, eg = forward(m.a1.double().T, dy, None, None, 1.0, 0.0, "none", kind, wide)
    check(T(m.gw2), g, eg, "gw2")
    _, _, g, eg = forward(x.T, m.dz1.double(), None, None, 1.0, 0.0, "none", kind, wide)
    check(T(m.gw1), g, eg, "gw1")
    _, _, g, eg = forward(w1.T, T(m.dz1), None, None, 1.0, 0.0, "none", kind, kind)
    check(T(m.dx), g, eg, "dx")


@pytest.mark.parametrize("kind,tokens,width,hidden", [("bf16", 96, 256, 512), ("f16", 41, 130, 515), ("f32", 64, 96, 200), ("bf16", 1, 4096, 512)])
def test_a_captured_step_replays(pkg, L, kind, tokens, width, hidden):
    """The step recorded into a graph, replayed on new inputs with eager work and synchronisations in between, against the
    eager step on the same inputs, bit for bit."""
    eager, captured = (Layer2(pkg, L, kind, tokens, width, hidden, "silu", 7) for _ in range(2))
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    captured.step(stream(), 0.5)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        captured.step(torch.cuda.current_stream().cuda_stream, 0.5)
    g = torch.Generator().manual_seed(1)
    for m in (eager, captured):
        for t in (m.gw1, m.gw2, m.gb1, m.gb2):
            t.zero_()
    for replay in range(4):
        x = torch.randn(tokens, width, generator=g).to(TORCH[kind]).cuda()
        eager.x.copy_(x), captured.x.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        eager.step(stream(), 0.5)
        torch.cuda.synchronize()
        for a, b in zip(eager.outputs(), captured.outputs()):
            assert torch.equal(a, b), replay


def test_two_streams_and_two_threads_at_once(pkg, L):
    """Steps with workspaces of their own on two streams, issued by two host threads, leave what they leave alone."""
    import threading
    alone = Layer2(pkg, L, "bf16", 200, 512, 1030, "gelu", 9)
    alone.step(stream(), 0.5)
    torch.cuda.synchronize()
    want = alone.outputs()
    models = [Layer2(pkg, L, "bf16", 200, 512, 1030, "gelu", 9) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    failed = []

    def work(m, s):
        try:
            for _ in range(10):
                with torch.cuda.stream(s):
                    for t in (m.gw1, m.gw2):
                        t.zero_()
                m.step(s.cuda_stream, 0.5)
        except Exception as e:   # reported by the main thread
            failed.append(e)
    threads = [threading.Thread(target=work, args=a) for a in zip(models, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for m in models:
        for a, b in zip(want, m.outputs()):
            assert torch.equal(a, b)



@pytest.mark.parametrize("kind,ta,tb,M,N,K", [("bf16", "N", "T", 1030, 3, 9000), ("f16", "N", "N", 5, 300, 4100), ("f32", "T", "N", 2061, 1803, 1003), ("f64", "N", "T", 700, 300, 1001)])
def test_captured_products_replay(pkg, L, kind, ta, tb, M, N, K):
    """Slices of thin products, copies, 64 x 64 slices: recorded, replayed on new operands with eager calls and synchronisations
    in between, bit for bit what the eager call leaves; nothing behind the workspace."""
    need = L.pl_gemm_epilogue_workspace_bytes(TYPES[kind], ta.encode(), tb.encode(), M, N, K, 1)
    A, B, Z = Mat(*((M, K) if ta == "N" else (K, M)), (M if ta == "N" else K) + 1, kind), Mat(*((K, N) if tb == "N" else (N, K)), (K if tb == "N" else N) + 1, kind), Mat(M, N, M, kind)
    outs = [(Mat(M, N, M, kind, gap=7.0), Mat(M, 1, M, kind, gap=5.0), torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device="cuda")) for _ in range(2)]

    def step(D, db, ws, s):
        pkg.check(L.pl_gemm_epilogue_grad(TYPES[kind], ta.encode(), tb.encode(), M, N, K, 0.5, A.ptr, A.ld, B.ptr, B.ld, ACTS["silu"], Z.ptr, Z.ld, 0.0, None, 0, D.ptr, D.ld,
                                          db.ptr, ws.data_ptr(), need, s), "pl_gemm_epilogue_grad")

    def fill(seed):
        A.set(rand(A.rows, A.cols, seed, kind)), B.set(rand(B.rows, B.cols, seed + 1, kind, K ** -0.5)), Z.set(rand(M, N, seed + 2, kind))

    fill(1)
    step(*outs[0], stream())
    step(*outs[1], stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        step(*outs[1], torch.cuda.current_stream().cuda_stream)
    for replay in range(4):
        fill(10 * replay + 20)
        graph.replay()
        torch.cuda.synchronize()
        step(*outs[0], stream())
        torch.cuda.synchronize()
        assert torch.equal(outs[0][0].get(), outs[1][0].get()) and torch.equal(outs[0][1].get(), outs[1][1].get()), replay
        assert all(bool((ws[need:] == 0xA5).all()) for _, _, ws in outs)
