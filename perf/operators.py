"""Workloads of the linear-layer operators and of gradient clipping: what one call computes, on which sizes.

Tensors are row-major as a torch program holds them: activations [tokens, features], weights [out, in].  The library
is column-major, so the same memory is a features x tokens matrix there.  `own = False` computes every operator from
elementary torch operations in 32 bits (64 where the tensors are); `own = True` calls the library.

    linear     y = act(x w^T + b) + beta r, optionally keeping z = x w^T + b      pl_gemm_epilogue
    wgrad      g = dz^T x + g0, the accumulated weight gradient                   pl_gemm_epilogue
    dgrad      dz = (dy w) * act'(z) and db = its sum over the tokens             pl_gemm_epilogue_grad
    act_grad   dz = dy * act'(z) and db = its sum over the tokens                 pl_bias_act_grad
    clip       n = |all gradients|, g * min(1, limit / (n + eps))                 pl_grad_norm_clip
"""
import ctypes as C
import importlib.util
import math
import os
import sys

import torch

own = False

TYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f64": 0, "f32": 1, "f16": 2, "bf16": 3}
ACTS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
EPS = 1e-6


def listed():
    return [
        # one token through an attention output projection with its residual: latency and one read of the weights
        {"name": "linear_1_token", "op": "linear", "type": "bf16", "tokens": 1, "fin": 4096, "fout": 4096, "act": "none",
         "bias": True, "residual": True, "keep": False, "pad": 0},
        # a batch of decoding sequences through the first half of a feed-forward block
        {"name": "linear_32_tokens", "op": "linear", "type": "f16", "tokens": 32, "fin": 4096, "fout": 16384, "act": "gelu_tanh",
         "bias": True, "residual": False, "keep": False, "pad": 0},
        # a training step's forward product of a feed-forward block, keeping what the backward pass needs
        {"name": "linear_train", "op": "linear", "type": "bf16", "tokens": 16384, "fin": 4096, "fout": 16384, "act": "gelu_tanh",
         "bias": True, "residual": False, "keep": True, "pad": 0},
        # a packed batch of prompts: no size a multiple of a tile, rows with padding behind them
        {"name": "linear_ragged", "op": "linear", "type": "f16", "tokens": 1023, "fin": 2052, "fout": 4100, "act": "silu",
         "bias": True, "residual": True, "keep": False, "pad": 3},
        # a layer kept in single precision
        {"name": "linear_f32", "op": "linear", "type": "f32", "tokens": 2048, "fin": 2048, "fout": 8192, "act": "gelu",
         "bias": True, "residual": False, "keep": True, "pad": 0},
        # a weight gradient added to the accumulator of earlier micro-batches, which is kept in 32 bits
        {"name": "wgrad_accumulate", "op": "wgrad", "type": "bf16", "out": "f32", "tokens": 8192, "fin": 4096, "fout": 4096, "pad": 0},
        # the gradient that reaches a feed-forward block's hidden layer, through its activation
        {"name": "dgrad_train", "op": "dgrad", "type": "bf16", "tokens": 8192, "fin": 4096, "fout": 16384, "act": "gelu_tanh", "pad": 0},
        # the same for a short fine-tuning batch of odd sizes
        {"name": "dgrad_ragged", "op": "dgrad", "type": "f16", "tokens": 333, "fin": 1024, "fout": 2050, "act": "silu", "pad": 1},
        # the activation's gradient where it arrives from outside the layer, at the size of a training batch
        {"name": "act_grad_train", "op": "act_grad", "type": "bf16", "tokens": 8192, "width": 16384, "act": "gelu_tanh", "pad": 0},
        # a small single-precision layer of odd sizes
        {"name": "act_grad_small", "op": "act_grad", "type": "f32", "tokens": 517, "width": 1031, "act": "gelu", "pad": 0},
        # a small network late in training: in place, the norm below the limit
        {"name": "clip_small", "op": "clip", "type": "f32", "vectors": "f32", "blocks": 6, "width": 128, "hidden": 500, "norm": 0.5,
         "limit": 1.0, "in_place": True},
        # a large network early in training: 16-bit matrices with 32-bit vectors, the norm above the limit, into another buffer
        {"name": "clip_large", "op": "clip", "type": "bf16", "vectors": "f32", "blocks": 16, "width": 2048, "hidden": 8192, "norm": 7.5,
         "limit": 1.0, "in_place": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "wgrad", "dgrad", "act_grad", "clip"])
    kind = rng.choice(["bf16", "bf16", "f16", "f16", "f32", "f64"])
    act = rng.choice(list(ACTS))
    if op == "clip":
        return {"op": op, "type": rng.choice(["bf16", "f16", "f32", "f64"]), "vectors": rng.choice(["f32", "bf16"]), "blocks": _log(rng, 1, 20),
                "width": _log(rng, 32, 1900), "hidden": _log(rng, 64, 7000), "norm": rng.choice([0.3, 0.9, 3.0, 40.0]), "limit": 1.0,
                "in_place": False}
    tokens = _log(rng, 1, 9000)
    if op == "act_grad":
        return {"op": op, "type": kind, "tokens": tokens, "width": _log(rng, 64, 14000), "act": act, "pad": rng.choice([0, 0, 1, 8])}
    fin, fout = _log(rng, 64, 6000), _log(rng, 64, 12000)
    if rng.random() < 0.5:  # multiples of 64 as often as any size
        fin, fout = -(-fin // 64) * 64, -(-fout // 64) * 64
    if kind in ("f32", "f64"):  # the same range of time: these products run at a sixteenth of the 16-bit rate and less
        tokens = min(tokens, 3000)
    case = {"op": op, "type": kind, "tokens": tokens, "fin": fin, "fout": fout, "pad": rng.choice([0, 0, 1, 8])}
    if op == "linear":
        case.update(act=act, bias=rng.random() < 0.7, residual=rng.random() < 0.5, keep=rng.random() < 0.5)
    elif op == "dgrad":
        case.update(act=act)
    else:
        case.update(out=rng.choice([kind, kind if kind == "f64" else "f32"]))
    return case


def _shapes(case):
    """The parameters of `blocks` feed-forward blocks with their norms, and an embedding: (shape, type) each."""
    w, h = case["width"], case["hidden"]
    block = [((w,), "vectors"), ((w, w), "type"), ((w,), "vectors"), ((h, w), "type"), ((h,), "vectors"), ((w, h), "type"), ((w,), "vectors")]
    return [(s, case[k]) for s, k in [((2 * h + 1, w), "type")] + block * case["blocks"]]


def _sizes(case):
    """A program keeps the gradients of each type in one buffer: how many elements each holds."""
    sizes = {}
    for shape, kind in _shapes(case):
        sizes[kind] = sizes.get(kind, 0) + math.prod(shape)
    return sizes


def _views(case, flat):
    used, views = dict.fromkeys(flat, 0), []
    for shape, kind in _shapes(case):
        count = math.prod(shape)
        views.append(flat[kind][used[kind]:used[kind] + count].view(shape))
        used[kind] += count
    return views


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _inputs(case, seed):
    """Everything random, from the seed alone."""
    dev = _device()
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(rows, cols, scale, kind, pad=0):
        t = torch.empty(rows, cols + pad, device=dev, dtype=TYPES[kind])
        t.normal_(0.0, scale, generator=gen)
        return t[:, :cols]

    op = case["op"]
    if op == "clip":
        sizes = _sizes(case)
        std = case["norm"] / math.sqrt(sum(sizes.values()))
        return {"flat": {k: torch.empty(n, device=dev, dtype=TYPES[k]).normal_(0.0, std, generator=gen) for k, n in sizes.items()}}
    kind, tokens, pad = case["type"], case["tokens"], case["pad"]
    if op == "act_grad":
        return {"dy": normal(tokens, case["width"], 0.1, kind, pad), "z": normal(tokens, case["width"], 1.0, kind, pad)}
    fin, fout = case["fin"], case["fout"]
    if op == "linear":
        d = {"x": normal(tokens, fin, 1.0, kind, pad), "w": normal(fout, fin, fin ** -0.5, kind, pad)}
        d["b"] = normal(1, fout, 0.5, kind)[0] if case["bias"] else None
        d["r"] = normal(tokens, fout, 1.0, kind, pad) if case["residual"] else None
        return d
    if op == "wgrad":
        return {"dz": normal(tokens, fout, 0.1, kind, pad), "x": normal(tokens, fin, 1.0, kind, pad),
                "g0": normal(fout, fin, 0.1 * tokens ** 0.5, case["out"], pad)}
    return {"dy": normal(tokens, fin, 0.1, kind, pad), "w": normal(fin, fout, fin ** -0.5, kind, pad), "z": normal(tokens, fout, 1.0, kind, pad)}


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    dev, op = _device(), case["op"]

    def rows(n, cols, kind):
        return torch.zeros(n, cols + case["pad"], device=dev, dtype=TYPES[kind])[:, :cols]

    if op == "clip":
        state["clipped"] = state["flat"] if case["in_place"] else {k: torch.zeros_like(t) for k, t in state["flat"].items()}
        state["grads"], state["out"] = _views(case, state["flat"]), _views(case, state["clipped"])
        state["norm"] = torch.zeros(1, device=dev, dtype=torch.float64)
    elif op == "act_grad":
        state["dz"] = rows(case["tokens"], case["width"], case["type"])
        state["db"] = torch.zeros(case["width"], device=dev, dtype=TYPES[case["type"]])
    elif op == "linear":
        state["y"] = rows(case["tokens"], case["fout"], case["type"])
        state["kept"] = rows(case["tokens"], case["fout"], case["type"]) if case["keep"] else None
    elif op == "wgrad":
        state["g"] = rows(case["fout"], case["fin"], case["out"])
    else:
        state["dz"] = rows(case["tokens"], case["fout"], case["type"])
        state["db"] = torch.zeros(case["fout"], device=dev, dtype=TYPES[case["type"]])
    return state


# ---- the plain form ----

def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


def _act(z, act):
    if act == "relu":
        return z * (z > 0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if act == "gelu_tanh":
        t = torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * (2 / math.pi) ** 0.5 * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "clip":
        norm = torch.sqrt(torch.stack([(_wide(g) * _wide(g)).sum(dtype=torch.float64) for g in s["grads"]]).sum())
        scale = torch.clamp(case["limit"] / (norm + EPS), max=1.0)
        s["norm"].copy_(norm.reshape(1))
        scaled = [o.copy_(_wide(g) * scale.to(_wide(g).dtype)) for o, g in zip(s["out"], s["grads"])]
        assert len(scaled) == len(s["grads"])
        return {"norm": s["norm"], "grads": s["clipped"]}
    kind = TYPES[case["type"]]
    if op == "linear":
        z = _wide(s["x"]) @ _wide(s["w"]).T
        if case["bias"]:
            z = z + _wide(s["b"])
        y = _act(z, case["act"])
        if case["residual"]:
            y = y + _wide(s["r"])
        return {"y": y.to(kind), "z": z.to(kind) if case["keep"] else None}
    if op == "wgrad":
        return {"g": (_wide(s["dz"]).T @ _wide(s["x"]) + _wide(s["g0"])).to(TYPES[case["out"]])}
    d = _wide(s["dy"]) @ _wide(s["w"]) if op == "dgrad" else _wide(s["dy"])
    d = d * _slope(_wide(s["z"]), case["act"])
    return {"dz": d.to(kind), "db": d.sum(0).to(kind)}


# ---- the library's calls ----

def _library():
    name = "paralia_framework_amd"
    if name not in sys.modules:
        folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "paralia-framework_amd")
        spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


def _kept(s):
    """What a program keeps between its calls: the library, a workspace and, for a list of gradients, its tables."""
    if "lib" not in s:
        pkg, case = _library(), s["case"]
        lib = s["lib"] = pkg.load()
        s["check"] = pkg.check
        op = case["op"]
        if op == "clip":
            n = len(s["grads"])
            s["n"] = n
            s["src"] = (C.c_void_p * n)(*[g.data_ptr() for g in s["grads"]])
            s["dst"] = (C.c_void_p * n)(*[g.data_ptr() for g in s["out"]])
            s["counts"] = (C.c_longlong * n)(*[g.numel() for g in s["grads"]])
            s["types"] = (C.c_int * n)(*[CODES[k] for _, k in _shapes(case)])
            need = lib.pl_grad_norm_workspace_bytes(n)
        elif op == "act_grad":
            need = lib.pl_bias_act_grad_workspace_bytes(CODES[case["type"]], case["width"], case["tokens"])
        else:
            m, n, k, ta, tb = {"linear": (case["fout"], case["tokens"], case["fin"], b"T", b"N"),
                               "wgrad": (case["fin"], case["fout"], case["tokens"], b"N", b"T"),
                               "dgrad": (case["fout"], case["tokens"], case["fin"], b"N", b"N")}[op]
            s["shape"] = (ta, tb, m, n, k)
            need = lib.pl_gemm_epilogue_workspace_bytes(CODES[case["type"]], ta, tb, m, n, k, 1 if op == "dgrad" else 0)
        s["ws_bytes"] = need
        s["ws"] = torch.empty(max(need, 16), device=_device(), dtype=torch.uint8)
        if op == "linear":
            kept = s["kept"]
            s["ep"] = pkg.epilogue(bias=s["b"].data_ptr() if case["bias"] else None, activation=ACTS[case["act"]],
                                   type_d=CODES[case["type"]], preact=kept.data_ptr() if case["keep"] else None,
                                   ld_preact=kept.stride(0) if case["keep"] else 0)
        elif op == "wgrad":
            s["ep"] = pkg.epilogue(type_d=CODES[case["out"]])
    return s["lib"]


def _own(s):
    lib, case = _kept(s), s["case"]
    op = case["op"]
    stream = torch.cuda.current_stream().cuda_stream
    ws, ws_bytes = s["ws"].data_ptr(), s["ws_bytes"]
    if op == "clip":
        rc = lib.pl_grad_norm_clip(s["n"], s["src"], s["counts"], s["types"], s["dst"], case["limit"], EPS, s["norm"].data_ptr(),
                                   ws, ws_bytes, stream)
        out = {"norm": s["norm"], "grads": s["clipped"]}
    elif op == "act_grad":
        dy, z, dz = s["dy"], s["z"], s["dz"]
        rc = lib.pl_bias_act_grad(CODES[case["type"]], ACTS[case["act"]], case["width"], case["tokens"], dy.data_ptr(), dy.stride(0),
                                  z.data_ptr(), z.stride(0), dz.data_ptr(), dz.stride(0), s["db"].data_ptr(), ws, ws_bytes, stream)
        out = {"dz": dz, "db": s["db"]}
    elif op == "dgrad":
        w, dy, z, dz = s["w"], s["dy"], s["z"], s["dz"]
        rc = lib.pl_gemm_epilogue_grad(CODES[case["type"]], *s["shape"], 1.0, w.data_ptr(), w.stride(0), dy.data_ptr(), dy.stride(0),
                                       ACTS[case["act"]], z.data_ptr(), z.stride(0), 0.0, None, 0, dz.data_ptr(), dz.stride(0),
                                       s["db"].data_ptr(), ws, ws_bytes, stream)
        out = {"dz": dz, "db": s["db"]}
    elif op == "wgrad":
        x, dz, g0, g = s["x"], s["dz"], s["g0"], s["g"]
        rc = lib.pl_gemm_epilogue(CODES[case["type"]], *s["shape"], 1.0, x.data_ptr(), x.stride(0), dz.data_ptr(), dz.stride(0), s["ep"],
                                  1.0, g0.data_ptr(), g0.stride(0), g.data_ptr(), g.stride(0), ws, ws_bytes, stream)
        out = {"g": g}
    else:
        x, w, r, y = s["x"], s["w"], s["r"], s["y"]
        rc = lib.pl_gemm_epilogue(CODES[case["type"]], *s["shape"], 1.0, w.data_ptr(), w.stride(0), x.data_ptr(), x.stride(0), s["ep"],
                                  1.0 if r is not None else 0.0, r.data_ptr() if r is not None else None, r.stride(0) if r is not None else 0,
                                  y.data_ptr(), y.stride(0), ws, ws_bytes, stream)
        out = {"y": y, "z": s["kept"]}
    s["check"](rc, op)
    return out


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    size = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}
    op = case["op"]
    if op == "clip":
        held = sum(math.prod(s) * size[k] for s, k in _shapes(case))
        count = sum(math.prod(s) for s, _ in _shapes(case))
        return {"bytes": held if case["in_place"] and case["norm"] < case["limit"] else 2 * held, "flops": 3 * count}
    e, t = size[case["type"]], case["tokens"]
    if op == "act_grad":
        return {"bytes": (3 * t + 1) * case["width"] * e, "flops": 12 * t * case["width"]}
    i, o = case["fin"], case["fout"]
    flops = 2 * t * i * o
    if op == "linear":
        outs = 1 + case["residual"] + case["keep"]
        return {"bytes": e * (t * i + i * o + outs * t * o + (o if case["bias"] else 0)), "flops": flops}
    if op == "wgrad":
        return {"bytes": e * t * (i + o) + 2 * size[case["out"]] * i * o, "flops": flops}
    return {"bytes": e * (t * i + i * o + 2 * t * o + o), "flops": flops}


# ---- the definitions in 64 bits ----

def _normal_cdf(z):
    return torch.special.ndtr(z)


def exact(case, seed):
    d = _inputs(case, seed)
    op = case["op"]
    if op == "clip":
        norm = math.sqrt(math.fsum(torch.linalg.vector_norm(t.double()).item() ** 2 for t in d["flat"].values()))
        scale = min(1.0, case["limit"] / (norm + EPS))
        return {"norm": torch.tensor([norm], dtype=torch.float64, device=_device()), "grads": {k: t.double() * scale for k, t in d["flat"].items()}}
    act = case.get("act", "none")
    if op == "wgrad":
        return {"g": torch.addmm(d["g0"].double(), d["dz"].double().T, d["x"].double())}
    if op == "linear":
        z = torch.mm(d["x"].double(), d["w"].double().T)
        if d["b"] is not None:
            z += d["b"].double()
        if act == "gelu":
            y = z * _normal_cdf(z)
        elif act == "gelu_tanh":
            y = z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))
        elif act == "silu":
            y = z * torch.sigmoid(z)
        else:
            y = z.clamp(min=0) if act == "relu" else z.clone()
        if d["r"] is not None:
            y += d["r"].double()
        return {"y": y, "z": z if case["keep"] else None}
    z = d["z"].double()
    g = torch.mm(d["dy"].double(), d["w"].double()) if op == "dgrad" else d["dy"].double()
    if act == "gelu":
        g = g * (_normal_cdf(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
    elif act == "gelu_tanh":
        c = math.sqrt(8 / math.pi)
        p = torch.sigmoid(c * (z + 0.044715 * z ** 3))
        g = g * (p + z * p * (1 - p) * c * (1 + 0.134145 * z ** 2))
    elif act == "silu":
        p = torch.sigmoid(z)
        g = g * (p + z * p * (1 - p))
    elif act == "relu":
        g = torch.where(z > 0, g, torch.zeros_like(g))
    return {"dz": g, "db": g.sum(0)}
