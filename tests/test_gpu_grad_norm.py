"""pl_grad_norm, pl_grad_clip and pl_grad_norm_clip on the GPU, against their definition in 64 bits."""
import ctypes as C
import math

import pytest
import torch

from linear_util import TORCH, TYPES, half_step

pytestmark = pytest.mark.gpu
EPS = 1e-6


class Tensors:
    """Gradients of the given (count, type, offset in elements) in guarded buffers, and as many outputs."""

    def __init__(self, specs, seed, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.kinds = [k for _, k, _ in specs]
        self.bufs, self.outs, self.views, self.out_views = [], [], [], []
        for count, kind, offset in specs:
            buf = torch.full((offset + count + 16,), float("nan"), dtype=TORCH[kind], device="cuda")
            out = torch.full_like(buf, 7.0)
            buf[offset:offset + count] = (torch.randn(count, generator=g, dtype=torch.float64) * scale).to(TORCH[kind]).cuda()
            self.bufs.append(buf), self.outs.append(out)
            self.views.append(buf[offset:offset + count]), self.out_views.append(out[offset:offset + count])

    def lists(self, views):
        n = len(views)
        return (n, (C.c_void_p * max(n, 1))(*[v.data_ptr() for v in views]), (C.c_longlong * max(n, 1))(*[v.numel() for v in views]),
                (C.c_int * max(n, 1))(*[TYPES[k] for k in self.kinds]))

    def norm(self):
        return math.sqrt(math.fsum(float((v.double() ** 2).sum()) for v in self.views))


def stream():
    return torch.cuda.current_stream().cuda_stream


def norm_buffers(L, n):
    need = L.pl_grad_norm_workspace_bytes(n)
    return torch.full((1,), -1.0, dtype=torch.float64, device="cuda"), torch.full((max(need // 8, 2),), float("nan"), dtype=torch.float64, device="cuda"), need


def clip(pkg, L, t, max_norm, in_place):
    n, src, counts, types = t.lists(t.views)
    dst = src if in_place else t.lists(t.out_views)[1]
    norm, ws, need = norm_buffers(L, n)
    pkg.check(L.pl_grad_norm_clip(n, src, counts, types, dst, max_norm, EPS, norm.data_ptr(), ws.data_ptr(), need, stream()), "pl_grad_norm_clip")
    torch.cuda.synchronize()
    return float(norm)


def mixed(n, seed, biggest=30000):
    g = torch.Generator().manual_seed(seed)
    kinds = ["bf16", "f16", "f32", "f64"]
    out = []
    for i in range(n):
        count = int(torch.randint(0, biggest, (1,), generator=g)) if i % 3 else int(torch.randint(0, 40, (1,), generator=g))
        out.append((count, kinds[int(torch.randint(0, 4, (1,), generator=g))], int(torch.randint(0, 9, (1,), generator=g))))
    return out


LISTS = {
    "one element": [(1, "f32", 0)],
    "one of each": [(5, "f64", 1), (1000, "f32", 3), (77, "f16", 5), (8191, "bf16", 7)],
    "around a chunk": [(8192, "f32", 0), (8193, "bf16", 0), (8191, "f16", 1), (16384, "bf16", 3), (7, "f32", 0)],
    "empty among them": [(0, "f32", 0), (10, "bf16", 0), (0, "f64", 0), (0, "bf16", 0), (3, "f16", 0), (0, "f32", 0)],
    "exactly one launch": mixed(112, 1, 300),
    "one more than a launch": mixed(113, 2, 300),
    "several launches": mixed(400, 3, 20000),
    "one large": [(20_000_001, "bf16", 3)],
    "large and small": [(9_000_000, "f32", 1), (1, "bf16", 0), (5_000_000, "f16", 0), (3, "f64", 0)],
}


@pytest.mark.parametrize("which", list(LISTS))
def test_norm_and_clipping(pkg, L, which):
    """The norm: squares of at most 64-bit values added in 64 bits, so its relative error is below (count + 2) 2^-53 / 2 in
    any order, half that for the square root's share.  The scaled values: the factor's and the product's rounding in the wide
    type, then one to the tensor's."""
    for in_place, factor in ((False, 0.25), (True, 0.25), (False, 4.0), (True, 4.0)):
        t = Tensors(LISTS[which], 5)
        before = [v.double().clone() for v in t.views]
        total = sum(v.numel() for v in t.views)
        norm = t.norm()
        got = clip(pkg, L, t, factor * norm, in_place)
        assert abs(got - norm) <= norm * (total + 4) * 2.0 ** -53
        scale = min(1.0, factor * norm / (norm + EPS))
        for v, o, b, kind in zip(t.views, t.out_views, before, t.kinds):
            u = 2.0 ** -52 if kind == "f64" else 2.0 ** -23
            out = (v if in_place else o).double()
            if scale == 1.0:
                assert torch.equal(out, b)
            else:
                err = (b * scale).abs() * (u * 2 + (total + 4) * 2.0 ** -52)
                assert bool(((out - b * scale).abs() <= err + half_step((b * scale).abs() + err, kind)).all())
            if not in_place:
                assert torch.equal(v.double(), b)
        for buf, out, v, o in zip(t.bufs, t.outs, t.views, t.out_views):
            v.fill_(float("nan")), o.fill_(7.0)
            assert bool(torch.isnan(buf).all()) and bool((out == 7.0).all())       # nothing in front or behind was written


def test_the_three_entry_points_agree(pkg, L):
    t = Tensors(mixed(130, 9, 5000), 6)
    n, src, counts, types = t.lists(t.views)
    norm, ws, need = norm_buffers(L, n)
    pkg.check(L.pl_grad_norm(n, src, counts, types, norm.data_ptr(), ws.data_ptr(), need, stream()), "pl_grad_norm")
    limit = 0.3 * float(norm)
    pkg.check(L.pl_grad_clip(n, src, counts, types, t.lists(t.out_views)[1], limit, EPS, norm.data_ptr(), stream()), "pl_grad_clip")
    torch.cuda.synchronize()
    two = [o.clone() for o in t.out_views]
    assert clip(pkg, L, t, limit, False) == float(norm)
    assert all(torch.equal(a, b) for a, b in zip(two, t.out_views))
    # as over two ranks: the norm of both halves from their own norms
    halves = []
    for lo, hi in ((0, 60), (60, n)):
        part = Tensors([], 0)
        part.kinds = t.kinds[lo:hi]
        m, s, c, ty = part.lists(t.views[lo:hi])
        pkg.check(L.pl_grad_norm(m, s, c, ty, norm.data_ptr(), ws.data_ptr(), need, stream()), "pl_grad_norm")
        halves.append(float(norm))
    assert abs(math.hypot(*halves) - t.norm()) <= 1e-12 * t.norm()


def test_extreme_values(pkg, L):
    """Squares that 32 bits lose, infinities and NaN."""
    for value in (1e-30, 1e30):
        t = Tensors([(1000, "f32", 0)], 1)
        t.views[0].fill_(value)
        v = float(t.views[0][0].double())
        assert abs(clip(pkg, L, t, 1.0, False) / (v * math.sqrt(1000)) - 1) < 1e-12
    t = Tensors([(1000, "bf16", 0), (50, "f32", 0)], 1)
    t.views[0][999] = float("inf")
    assert clip(pkg, L, t, 1.0, True) == float("inf")
    assert bool((t.views[0][:999] == 0).all()) and math.isnan(float(t.views[0][999])) and bool((t.views[1] == 0).all())
    t = Tensors([(1000, "bf16", 0), (50, "f32", 0)], 1)
    t.views[1][3] = float("nan")
    assert math.isnan(clip(pkg, L, t, 1.0, True))
    assert all(bool(torch.isnan(v).all()) for v in t.views)
    t = Tensors([(100, "f32", 0)], 1)
    t.views[0].zero_()
    assert clip(pkg, L, t, 1.0, True) == 0.0 and bool((t.views[0] == 0).all())
    t = Tensors([(100, "f32", 0)], 1)
    clip(pkg, L, t, 0.0, True)
    assert bool((t.views[0] == 0).all())


def test_no_tensors(pkg, L):
    norm, ws, need = norm_buffers(L, 1)
    pkg.check(L.pl_grad_norm(0, None, None, None, norm.data_ptr(), None, 0, stream()), "pl_grad_norm")
    assert float(norm) == 0.0
    t = Tensors([(0, "f32", 0), (0, "bf16", 0)], 1)
    assert clip(pkg, L, t, 1.0, True) == 0.0


def test_repeats_bit_for_bit(pkg, L):
    t = Tensors(mixed(50, 4, 100000), 3)
    first = clip(pkg, L, t, 1.0, False)
    outs = [o.clone() for o in t.out_views]
    for _ in range(3):
        assert clip(pkg, L, t, 1.0, False) == first
        assert all(torch.equal(a, b) for a, b in zip(outs, t.out_views))


def whole_lists(n, seed, biggest):
    """n tensors, none of them empty."""
    return [(count + 1, kind, offset) for count, kind, offset in mixed(n, seed, biggest)]


@pytest.mark.parametrize("n", [127, 128, 129, 255, 256, 257])
def test_lists_around_a_launch(pkg, L, n):
    """128 tensors go into a launch: one fewer, as many, one more, and the same around the second; bounds as above."""
    for in_place, factor in ((False, 0.25), (True, 0.25), (True, 4.0)):
        t = Tensors(whole_lists(n, n, 300), 5)
        before = [v.double().clone() for v in t.views]
        total = sum(v.numel() for v in t.views)
        norm = t.norm()
        got = clip(pkg, L, t, factor * norm, in_place)
        assert abs(got - norm) <= norm * (total + 4) * 2.0 ** -53
        scale = min(1.0, factor * norm / (norm + EPS))
        for v, o, b, kind in zip(t.views, t.out_views, before, t.kinds):
            u = 2.0 ** -52 if kind == "f64" else 2.0 ** -23
            err = (b * scale).abs() * (u * 2 + (total + 4) * 2.0 ** -52) if scale < 1.0 else torch.zeros_like(b)
            out = (v if in_place else o).double()
            assert bool(((out - b * scale).abs() <= err + (half_step((b * scale).abs() + err, kind) if scale < 1.0 else 0.0)).all())


def test_a_long_list_costs_what_its_parts_cost(pkg, L):
    """3000 tensors: the norm and the clipping in one call do what they do in two, bit for bit, and take no longer than half
    as long again (with a fold of all partial sums in every workgroup of every launch 0.78 ms against 0.42)."""
    n, count = 3000, 70000
    flat = torch.randn(n * count, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").bfloat16()
    out = [torch.zeros_like(flat) for _ in range(2)]
    lists = [(C.c_void_p * n)(*[b.data_ptr() + 2 * count * i for i in range(n)]) for b in (flat, *out)]
    counts, types = (C.c_longlong * n)(*[count] * n), (C.c_int * n)(*[TYPES["bf16"]] * n)
    norm, ws, need = norm_buffers(L, n)
    norms = [norm, norm.clone()]

    def one():
        pkg.check(L.pl_grad_norm_clip(n, lists[0], counts, types, lists[1], 1.0, EPS, norms[0].data_ptr(), ws.data_ptr(), need, stream()), "pl_grad_norm_clip")

    def two():
        pkg.check(L.pl_grad_norm(n, lists[0], counts, types, norms[1].data_ptr(), ws.data_ptr(), need, stream()), "pl_grad_norm")
        pkg.check(L.pl_grad_clip(n, lists[0], counts, types, lists[2], 1.0, EPS, norms[1].data_ptr(), stream()), "pl_grad_clip")

    def best_ms(call):
        times = []
        for _ in range(6):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            call()
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times[1:])

    together, apart = best_ms(one), best_ms(two)
    print("one call %.3f ms, two calls %.3f ms" % (together, apart), flush=True)
    assert torch.equal(norms[0], norms[1]) and torch.equal(out[0], out[1])
    want = math.sqrt(float((flat.double() ** 2).sum()))
    assert abs(float(norm) - want) <= want * n * count * 2.0 ** -53
    assert together <= 1.5 * apart


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("limit", [1.0, 1e-3, 1e-6, 1e-30])
@pytest.mark.parametrize("in_place", [False, True])
def test_factors_below_the_normal_numbers_of_32_bits(pkg, L, kind, limit, in_place):
    """Gradients of 5e37 against a small limit: a factor that 32 bits hold in a few bits or not at all (1e-40 .. 1e-70) scales
    like any other.  Bounds as above: factor and product in the wide type, then one rounding to the tensor's."""
    t = Tensors([(1000, kind, 3), (20, "f64", 0)], 5, 5e37)
    before = [v.double().clone() for v in t.views]
    norm = t.norm()
    assert abs(clip(pkg, L, t, limit, in_place) - norm) <= norm * 1024 * 2.0 ** -53
    scale = limit / (norm + EPS)
    assert scale < 2.0 ** -126
    for v, o, b, k in zip(t.views, t.out_views, before, t.kinds):
        want = b * scale
        err = want.abs() * (2.0 ** -51 if k == "f64" else 2.0 ** -22) + want.abs() * 1024 * 2.0 ** -52
        assert bool((((v if in_place else o).double() - want).abs() <= err + half_step(want.abs() + err, k)).all())


def test_a_captured_long_list_replays(pkg, L):
    """300 tensors whose norm is folded by a launch of its own: recorded, replayed on new gradients, norms and outputs bit for
    bit those of the eager call, with nothing behind the workspace."""
    n, count = 300, 70001
    flat = torch.empty(n * count, device="cuda")
    outs, norms = [torch.zeros_like(flat) for _ in range(2)], [torch.zeros(1, dtype=torch.float64, device="cuda") for _ in range(2)]
    lists = [(C.c_void_p * n)(*[b.data_ptr() + 4 * count * i for i in range(n)]) for b in (flat, *outs)]
    counts, types = (C.c_longlong * n)(*[count] * n), (C.c_int * n)(*[TYPES["f32"]] * n)
    need = L.pl_grad_norm_workspace_bytes(n)
    ws = [torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device="cuda") for _ in range(2)]

    def call(i, s):
        pkg.check(L.pl_grad_norm_clip(n, lists[0], counts, types, lists[1 + i], 1.0, EPS, norms[i].data_ptr(), ws[i].data_ptr(), need, s), "pl_grad_norm_clip")

    g = torch.Generator(device="cuda").manual_seed(3)
    flat.normal_(generator=g)
    call(1, stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        call(1, torch.cuda.current_stream().cuda_stream)
    for replay in range(4):
        flat.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        call(0, stream())
        torch.cuda.synchronize()
        want = math.sqrt(float((flat.double() ** 2).sum()))
        assert abs(float(norms[0]) - want) <= want * n * count * 2.0 ** -53
        assert torch.equal(norms[0], norms[1]) and torch.equal(outs[0], outs[1]), replay
        assert all(bool((w[need:] == 0xA5).all()) for w in ws)
