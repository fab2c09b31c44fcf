"""The training operators around a Transformer block's gated MLP, as this package's users call them: the residual's addition with its
RMS norm, the gated MLP, both with their pullbacks, and the clipping of all gradients by their global norm.

``own`` False: each operator in its plain form, elementary torch operations in 32 bits; True: the package's own entry points.
"""
from __future__ import annotations

import random

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-5
_MAX_NORM = 1.0
_E4M3_MOST = 448.0


def listed():
    return [
        # one generated token through the norm before a block's MLP: latency
        {"name": "norm token", "op": "norm", "rows": 1, "dim": 768, "dtype": "bf16", "residual": "f32", "scaled": False},
        # the same norm over a training batch of 8 x 1024 positions, fp32 residual stream
        {"name": "norm batch", "op": "norm", "rows": 8192, "dim": 768, "dtype": "bf16", "residual": "f32", "scaled": False},
        # a wide model's prefill of a ragged batch, the norm's output in 8 bits for an 8-bit product
        {"name": "norm wide scaled", "op": "norm", "rows": 5003, "dim": 8192, "dtype": "bf16", "residual": "bf16", "scaled": True},
        # the training batch's norm, backwards: cotangents of both inputs and of the weight
        {"name": "norm backward", "op": "norm_backward", "rows": 8192, "dim": 768, "dtype": "bf16", "residual": "f32"},
        # one generated token through the MLP: the weights' way through the chip
        {"name": "mlp token", "op": "mlp", "rows": 1, "dim": 768, "hidden": 2048, "dtype": "bf16", "bias": False, "keep": False},
        # a small ragged batch of a larger model with biases, served
        {"name": "mlp ragged", "op": "mlp", "rows": 77, "dim": 2048, "hidden": 5632, "dtype": "f16", "bias": True, "keep": False},
        # the training batch's MLP, forwards, with what the backward pass needs
        {"name": "mlp batch", "op": "mlp", "rows": 8192, "dim": 768, "hidden": 2048, "dtype": "bf16", "bias": False, "keep": True},
        # a wide model's MLP over a ragged prefill
        {"name": "mlp wide", "op": "mlp", "rows": 6007, "dim": 4096, "hidden": 11008, "dtype": "bf16", "bias": False, "keep": False},
        # the training batch's MLP, backwards: the cotangent of its input and both weights' gradients
        {"name": "mlp backward", "op": "mlp_backward", "rows": 8192, "dim": 768, "hidden": 2048, "dtype": "bf16", "bias": False},
        # the same of a larger model, an odd number of positions, half precision and biases
        {"name": "mlp backward wide", "op": "mlp_backward", "rows": 6007, "dim": 2560, "hidden": 6912, "dtype": "f16", "bias": True},
        # the gradients of a small interface: a few tensors of fp32
        {"name": "clip interface", "op": "clip", "layers": 0, "dim": 256, "hidden": 0, "vocab": 0, "regions": 2, "width": 32},
        # the gradients of a 12-layer model, matrices in bf16, interface and norms in fp32
        {"name": "clip model", "op": "clip", "layers": 12, "dim": 768, "hidden": 2048, "vocab": 50257, "regions": 6, "width": 64},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even in its logarithm."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(("norm", "norm", "norm_backward", "norm_backward", "mlp", "mlp", "mlp_backward", "clip", "clip"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    if op in ("norm", "norm_backward"):
        dim = _spread(rng, 64, 8192)
        if rng.random() < 0.75:  # mostly widths that models have, some that end anywhere
            dim = max(64, dim // 64 * 64)
        rows = _spread(rng, 1, min(32768, 32_000_000 // dim))
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        case = {"op": op, "rows": rows, "dim": dim, "dtype": dtype, "residual": rng.choice((dtype, "f32"))}
        return {**case, "scaled": rng.random() < 0.4} if op == "norm" else case
    if op in ("mlp", "mlp_backward"):
        dim, hidden = _spread(rng, 128, 4096), _spread(rng, 128, 11008)
        if rng.random() < 0.75:
            dim, hidden = max(64, dim // 64 * 64), max(64, hidden // 64 * 64)
        rows = _spread(rng, 1, max(1, min(16384, 100_000_000_000 // (dim * hidden))))
        case = {"op": op, "rows": rows, "dim": dim, "hidden": hidden, "dtype": dtype, "bias": rng.random() < 0.3}
        return {**case, "keep": rng.random() < 0.5} if op == "mlp" else case
    return {"op": "clip", "layers": rng.randint(0, 12), "dim": _spread(rng, 64, 768), "hidden": _spread(rng, 64, 2048),
            "vocab": _spread(rng, 16, 50000), "regions": rng.randint(1, 6), "width": _spread(rng, 4, 64)}


def _gradient_shapes(case):
    """(matrices in bf16, the rest in fp32) of a model's gradients, shapes only."""
    dim, hidden, width = case["dim"], case["hidden"], case["width"]
    block = [(3 * dim, dim), (3 * dim, 4), (dim, dim), (2 * hidden, dim), (dim, hidden)]
    half = block * case["layers"] + ([(case["vocab"], dim)] * 2 if case["layers"] else [])
    region = [(width, dim), (width,), (dim, width), (dim,), (width,), (width,), (1,)]
    single = [(dim,), (dim,)] * case["layers"] + region * case["regions"] + [(width, dim), (width,), (dim,)]
    return half, single


def _elements(shapes):
    total = 0
    for shape in shapes:
        count = 1
        for extent in shape:
            count *= extent
        total += count
    return total


def _views(flat, shapes):
    """Tensors of these shapes one behind the other in ``flat``."""
    views, at = [], 0
    for shape in shapes:
        count = _elements([shape])
        views.append(flat[at:at + count].view(shape))
        at += count
    return views


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, std=1.0, dtype=None):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype or _TYPES[case["dtype"]])

    state = {"case": case}
    if case["op"] == "clip":
        half, single = _gradient_shapes(case)
        # gradients whose global norm is between a half and eight times what it is clipped to
        norm = 0.5 * 16.0 ** random.Random(seed).random()
        std = norm * (_elements(half) + _elements(single)) ** -0.5
        for name, shapes, dtype in (("half", half, torch.bfloat16), ("single", single, torch.float32)):
            state[name] = rand(_elements(shapes), std=std, dtype=dtype)
            state[name + "_out"] = torch.empty_like(state[name])
        state["grads"] = _views(state["half"], half) + _views(state["single"], single)
        state["outs"] = _views(state["half_out"], half) + _views(state["single_out"], single)
        return state
    rows, dim = case["rows"], case["dim"]
    if case["op"] in ("norm", "norm_backward"):
        stream = _TYPES[case["residual"]]
        state["weight"] = (1.0 + rand(dim, std=0.1, dtype=torch.float32)).to(_TYPES[case["dtype"]])
        state["residual"] = rand(rows, dim, std=2.0, dtype=stream)
        if case["op"] == "norm":
            state["hidden"] = rand(rows, dim)
        else:
            state["g_normed"], state["g_residual"] = rand(rows, dim), rand(rows, dim, std=0.5, dtype=stream)
        return state
    hidden = case["hidden"]
    state["x"] = rand(rows, dim)
    state["fc1"], state["fc2"] = rand(2 * hidden, dim, std=dim ** -0.5), rand(dim, hidden, std=hidden ** -0.5)
    state["fc1_bias"] = rand(2 * hidden, std=0.1) if case["bias"] else None
    state["fc2_bias"] = rand(dim, std=0.1) if case["bias"] else None
    if case["op"] == "mlp_backward":
        # what the forward pass left, with its distributions
        state["fc1_output"] = rand(rows, 2 * hidden)
        up, gate = state["fc1_output"].float().chunk(2, dim=1)
        state["down_input"] = (up * gate * torch.sigmoid(gate)).to(_TYPES[case["dtype"]])
        state["g_out"] = rand(rows, dim)
    return state


def _run_own(s):
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients
    from latent_bounded_interfaces_amd.hip.transformer.block import (gated_mlp, gated_mlp_vjp, residual_rmsnorm,
                                                                     residual_rmsnorm_pullback)

    case = s["case"]
    if case["op"] == "norm":
        return residual_rmsnorm(s["hidden"], s["residual"], s["weight"], _EPS, scaled=case["scaled"])
    if case["op"] == "norm_backward":
        return residual_rmsnorm_pullback(s["g_normed"], s["residual"], s["weight"], _EPS, g_residual=s["g_residual"])
    if case["op"] == "mlp":
        return gated_mlp(s["x"], s["fc1"], s["fc2"], s["fc1_bias"], s["fc2_bias"], keep=case["keep"])
    if case["op"] == "mlp_backward":
        return gated_mlp_vjp(s["g_out"], s["x"], s["fc1_output"], s["down_input"], s["fc1"], s["fc2"], bias=case["bias"])
    norm = clip_gradients(s["grads"], _MAX_NORM, out=s["outs"])
    return norm, s["half_out"], s["single_out"]


def _norm(s):
    case = s["case"]
    total = s["hidden"].float() + s["residual"].float()
    normed = total * torch.rsqrt((total * total).mean(dim=1, keepdim=True) + _EPS) * s["weight"].float()
    stream = total.to(s["residual"].dtype)
    if not case["scaled"]:
        return normed.to(s["hidden"].dtype), stream
    most = normed.abs().amax(dim=1)
    scales = torch.where(most == 0, torch.ones_like(most), most / _E4M3_MOST)
    return (normed / scales[:, None]).to(torch.float8_e4m3fn), scales, stream


def _norm_backward(s):
    x, g = s["residual"].float(), s["g_normed"].float()
    inv = torch.rsqrt((x * x).mean(dim=1, keepdim=True) + _EPS)
    unit = x * inv
    pulled = g * s["weight"].float()
    total = inv * (pulled - unit * (unit * pulled).mean(dim=1, keepdim=True)) + s["g_residual"].float()
    return total.to(s["g_normed"].dtype), total.to(s["residual"].dtype), (g * unit).sum(dim=0)


def _mlp(s):
    dtype = s["x"].dtype
    fc1_output = s["x"].float() @ s["fc1"].float().t()
    if s["fc1_bias"] is not None:
        fc1_output = fc1_output + s["fc1_bias"].float()
    up, gate = fc1_output.chunk(2, dim=1)
    down_input = up * (gate * torch.sigmoid(gate))
    out = down_input @ s["fc2"].float().t()
    if s["fc2_bias"] is not None:
        out = out + s["fc2_bias"].float()
    return (out.to(dtype), fc1_output.to(dtype), down_input.to(dtype)) if s["case"]["keep"] else out.to(dtype)


def _mlp_backward(s):
    dtype = s["x"].dtype
    g_out = s["g_out"].float()
    up, gate = s["fc1_output"].float().chunk(2, dim=1)
    g_down = g_out @ s["fc2"].float()
    open_ = torch.sigmoid(gate)
    g_up, g_gate = g_down * (gate * open_), g_down * up * (open_ * (1.0 + gate * (1.0 - open_)))
    g_fc1 = torch.cat((g_up, g_gate), dim=1)
    grads = [g_fc1 @ s["fc1"].float(), g_fc1.t() @ s["x"].float(), g_out.t() @ s["down_input"].float()]
    if s["case"]["bias"]:
        grads += [g_fc1.sum(dim=0), g_out.sum(dim=0)]
    return tuple(g.to(dtype) for g in grads)


def _clip(s):
    half, single = s["half"].float(), s["single"]
    norm = torch.sqrt((half * half).sum(dtype=torch.float64) + (single * single).sum(dtype=torch.float64)).float()
    factor = torch.clamp(_MAX_NORM / (norm + 1e-6), max=1.0)
    return norm, (half * factor).to(torch.bfloat16), single * factor


_PLAIN = {"norm": _norm, "norm_backward": _norm_backward, "mlp": _mlp, "mlp_backward": _mlp_backward, "clip": _clip}


def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state["case"]["op"]](state)


def work(case):
    """Every input read once, every output written once; the products' multiplications and additions."""
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "clip":
        half, single = _gradient_shapes(case)
        return {"bytes": 2 * (2 * _elements(half) + 4 * _elements(single)) + 4, "flops": 3 * (_elements(half) + _elements(single))}
    rows, dim, b = case["rows"], case["dim"], size[case["dtype"]]
    if case["op"] == "norm":
        r = size[case["residual"]]
        return {"bytes": rows * dim * (b + 2 * r + (1 if case["scaled"] else b)) + dim * b + (4 * rows if case["scaled"] else 0),
                "flops": 5 * rows * dim}
    if case["op"] == "norm_backward":
        r = size[case["residual"]]
        return {"bytes": rows * dim * (2 * b + 3 * r) + dim * (b + 4), "flops": 12 * rows * dim}
    hidden = case["hidden"]
    weights = 3 * hidden * dim + (2 * hidden + dim if case["bias"] else 0)
    if case["op"] == "mlp":
        values = rows * (2 * dim + (3 * hidden if case["keep"] else 0)) + weights
        return {"bytes": b * values, "flops": 6 * rows * dim * hidden}
    return {"bytes": b * (rows * (3 * dim + 3 * hidden) + 2 * weights), "flops": 12 * rows * dim * hidden}


def exact(case, seed):
    """The definitions in 64 bits; of values in 8 bits, what they are rounded from."""
    s = prepare(case, seed)
    d = {name: value.double() for name, value in s.items() if isinstance(value, torch.Tensor) and name not in ("half_out", "single_out")}
    if case["op"] == "clip":
        norm = (torch.linalg.vector_norm(d["half"]) ** 2 + torch.linalg.vector_norm(d["single"]) ** 2) ** 0.5
        factor = min(1.0, _MAX_NORM / (float(norm) + 1e-6))
        return norm, d["half"].mul_(factor), d["single"].mul_(factor)
    if case["op"] == "norm":
        x = d["residual"].add_(d["hidden"])
        y = x / (x.pow(2).sum(1) / case["dim"] + _EPS).sqrt()[:, None] * d["weight"]
        if not case["scaled"]:
            return y, x
        scales = y.abs().max(dim=1).values / _E4M3_MOST
        scales[scales == 0] = 1.0
        return y / scales[:, None], scales, x
    if case["op"] == "norm_backward":
        # y_j = w_j x_j / m with m = sqrt(mean(x^2) + eps), so dy_j/dx_i = w_j (delta_ij / m - x_i x_j / (n m^3))
        x, g, n = d["residual"], d["g_normed"], case["dim"]
        m = (x.pow(2).sum(1, keepdim=True) / n + _EPS).sqrt()
        along = (g * d["weight"] * x).sum(1, keepdim=True)
        g_x = g * d["weight"] / m - x * along / (n * m ** 3) + d["g_residual"]
        return g_x, g_x, (g * x / m).sum(0)
    silu = torch.nn.functional.silu
    if case["op"] == "mlp":
        z = torch.addmm(d["fc1_bias"], d["x"], d["fc1"].t()) if case["bias"] else torch.mm(d["x"], d["fc1"].t())
        a = z[:, :case["hidden"]] * silu(z[:, case["hidden"]:])
        out = torch.addmm(d["fc2_bias"], a, d["fc2"].t()) if case["bias"] else torch.mm(a, d["fc2"].t())
        return (out, z, a) if case["keep"] else out
    up, gate = d["fc1_output"][:, :case["hidden"]], d["fc1_output"][:, case["hidden"]:].requires_grad_()
    with torch.enable_grad():
        opened = silu(gate)
        slope, = torch.autograd.grad(opened.sum(), gate)
    g_a = torch.mm(d["g_out"], d["fc2"])
    g_z = torch.cat((g_a * opened.detach(), g_a * up * slope), dim=1)
    grads = (torch.mm(g_z, d["fc1"]), torch.mm(g_z.t(), d["x"]), torch.mm(d["g_out"].t(), d["down_input"]))
    return grads + (g_z.sum(0), d["g_out"].sum(0)) if case["bias"] else grads
