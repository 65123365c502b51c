"""Column-major matrices in torch memory, and the definitions of the linear-layer operators in 64 bits, with the error
that 32-bit (64-bit) arithmetic may leave.

Notation of the bounds: u = 2^-24 (2^-53 for fp64 operands), S = |alpha| |A| |B| + |bias| with the operands' magnitudes.
A product summed in any order, with the accumulator rounded (or truncated) after every step, is off by at most
2 (K + 2) u S.  An activation's slope is below 1.13, so that error grows by at most that much on its way through it."""
import ctypes as C
import math
import os

import torch

TYPES = {"f64": 0, "f32": 1, "f16": 2, "bf16": 3}
TORCH = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
MAX_SLOPE = 1.13


class Mat:
    """rows x cols, column-major with leading dimension ld, starting `offset` elements into its buffer.  What is not the
    matrix (the rows behind it in every column, what lies in front and behind) is filled with `gap`."""

    def __init__(self, rows, cols, ld, kind, offset=0, gap=float("nan"), device="cuda"):
        self.rows, self.cols, self.ld, self.kind, self.offset, self.gap = rows, cols, ld, kind, offset, gap
        self.buf = torch.full((offset + cols * ld + 8,), gap, dtype=TORCH[kind], device=device)
        self.view = self.buf[offset:offset + cols * ld].view(cols, ld)[:, :rows]   # [n][m]

    def set(self, values):
        """values: rows x cols"""
        self.view.copy_(values.T.to(self.buf.dtype))
        return self

    def get(self):
        return self.view.T.double()

    @property
    def ptr(self):
        return self.buf.data_ptr() + self.offset * self.buf.element_size()

    def gaps_untouched(self):
        seen = self.buf.clone()
        seen[self.offset:self.offset + self.cols * self.ld].view(self.cols, self.ld)[:, :self.rows] = self.gap
        return bool(torch.isnan(seen).all()) if math.isnan(self.gap) else bool((seen == self.gap).all())


def unit(kind):
    return 2.0 ** -53 if kind == "f64" else 2.0 ** -24


def half_step(values, kind):
    """Half a unit in the last place of a rounding of `values` to `kind`, its smallest subnormal step included."""
    info = torch.finfo(TORCH[kind])
    return values.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def act(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(8 / math.pi)
        s = torch.sigmoid(c * (z + 0.044715 * z ** 3))
        return s + z * s * (1 - s) * c * (1 + 0.134145 * z * z)
    if name == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    return torch.ones_like(z)


def act_error(z, name, kind):
    """Relative error of the factor an activation multiplies z with, and (twice that) absolute error of the slope's terms:
    a few roundings, the rounding of the exponent's argument (z^2 / 2, or 2u of the tanh form), and for 16-bit operands
    the 4.2e-6 of the short polynomial."""
    if name in ("none", "relu"):
        return torch.zeros_like(z)
    a = z.abs().clamp(max=40)
    arg = {"gelu": a * a, "gelu_tanh": 8 * (a + 0.0448 * a ** 3), "silu": 2 * a}[name]
    return (16 + arg) * 2 * unit(kind) + (6e-6 if kind in ("f16", "bf16") and name == "gelu" else 0.0)


def forward(A, B, bias, C, alpha, beta, name, kind, kind_d):
    """op(A) M x K and op(B) K x N in 64 bits -> z, y and their error bounds."""
    K, u = A.shape[1], unit(kind)
    prod = A @ B if K else torch.zeros(A.shape[0], B.shape[1], dtype=torch.float64, device=A.device)
    size = A.abs() @ B.abs() if K else torch.zeros_like(prod)
    z, S = alpha * prod, abs(alpha) * size
    if bias is not None:
        z, S = z + bias[:, None], S + bias.abs()[:, None]
    ez = 2 * (K + 4) * u * S
    y = act(z, name)
    ey = MAX_SLOPE * ez + act_error(z, name, kind) * y.abs()
    if beta:
        ey = ey + 2 * u * (y.abs() + abs(beta) * C.abs())
        y = y + beta * C
    return z, ez + half_step(z.abs() + ez, kind), y, ey + half_step(y.abs() + ey, kind_d)


def gradient(A, B, Z, C, alpha, beta, name, kind):
    """-> D, dbias and their error bounds."""
    K, u = A.shape[1], unit(kind)
    prod = A @ B if K else torch.zeros(A.shape[0], B.shape[1], dtype=torch.float64, device=A.device)
    size = A.abs() @ B.abs() if K else torch.zeros_like(prod)
    g, S = alpha * prod, abs(alpha) * size
    if beta:
        g, S = g + beta * C, S + abs(beta) * C.abs()
    return slope_product(g, 2 * (K + 4) * u * S, Z, name, kind)


def slope_product(g, eg, Z, name, kind):
    u = unit(kind)
    s = slope(Z, name)
    d = g * s
    ed = MAX_SLOPE * eg + g.abs() * 2.5 * act_error(Z, name, kind) + 4 * u * d.abs()
    db, N = d.sum(1), d.shape[1]
    edb = ed.sum(1) + 2 * (N + 2) * u * d.abs().sum(1)
    return d, ed + half_step(d.abs() + ed, kind), db, edb + half_step(db.abs() + edb, kind)


def check(got, want, bound, what):
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), "%s: %d of %d elements off, worst %.3g of the bound, first at %s: %r instead of %r" % (
        what, int(bad.sum()), bad.numel(), float((off / bound).nan_to_num(nan=float("inf")).max()), bad.nonzero()[0].tolist(),
        float(got[bad][0]), float(want[bad][0]))


def shipped_fit(pkg, L):
    """The launcher constants of the shipped database, as the library's first routine call installs them."""
    import sys
    f = sys.modules[pkg.__name__ + ".binding"].gemm_fit()
    L.pl_gemm_fit_defaults(C.byref(f))
    names = {"lone_us_per_k_f64": ("lone_us_per_k", 0), "lone_us_per_k_f32": ("lone_us_per_k", 1), "f32_wide_fixed_us_beta0": ("f32_wide_fixed_us", 0),
             "f32_wide_fixed_us_beta1": ("f32_wide_fixed_us", 1), "edge_rounds_small": ("edge_rounds", 0), "edge_rounds_large": ("edge_rounds", 1)}
    for t, trans in enumerate(("NN", "NT", "TN", "TT")):
        names["f32_large_gain_" + trans] = ("f32_large_gain", t)
        for b in range(2):
            names["f32_large_fixed_us_beta%d_%s" % (b, trans)] = ("f32_large_fixed_us", t, b)
    fields = {name for name, _ in f._fields_}
    for line in open(os.path.join(pkg.PKG_DIR, "db", "mi355x", "Processed", "Kernel-fit_dev-0.log")):
        name, _, value = line.partition(":")
        if name in names:
            field, at = names[name][0], names[name][1:]
            array = getattr(f, field)
            for i in at[:-1]:
                array = array[i]
            array[at[-1]] = float(value)
        elif name in fields:
            setattr(f, name, float(value))
    return f


def takes_copies(L, kind, ta, tb, M, N, K):
    """Whether an fp32 or fp64 product sets space aside for aligned copies of its operands: behind the product, rows in whole
    tiles of 256 and k in whole panels of 32."""
    up = lambda n, unit: -(-n // unit) * unit  # noqa: E731
    es = 8 if kind == "f64" else 4
    need = L.pl_gemm_epilogue_workspace_bytes(TYPES[kind], ta.encode(), tb.encode(), M, N, K, 0)
    return need >= M * N * es + (up(M, 256) + up(N, 256)) * up(K, 32) * es
