"""The operators of a block's mixer half, as this package's users call them: the rotary positions of a packed projection, linear attention
with a decay for each head (over prompts, for single tokens, and its pullback for a basis of cotangents), and the norms behind and
before a block with its gate and residual scale.

``own`` False: each operator in its plain form, elementary torch operations in 32 bits; True: the package's own entry points.
"""
from __future__ import annotations

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZES = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-5
_CHUNK = 64


def listed():
    return [
        # a padded batch of eight prompts of up to 1024 tokens through one layer of the 12-head model
        {"name": "prompt ragged", "op": "prompt", "batch": 8, "heads": 12, "kv_heads": 12, "length": 1024, "dk": 64, "dv": 64, "dtype": "bf16",
         "lengths": True, "state": False},
        # long contexts of a larger model, the states of what came before them at hand
        {"name": "prompt long", "op": "prompt", "batch": 4, "heads": 16, "kv_heads": 16, "length": 4096, "dk": 128, "dv": 128, "dtype": "bf16",
         "lengths": False, "state": True},
        # one odd prompt in half precision, keys and values shared by four heads, widths that fill no tile
        {"name": "prompt odd", "op": "prompt", "batch": 1, "heads": 8, "kv_heads": 2, "length": 2999, "dk": 80, "dv": 112, "dtype": "f16",
         "lengths": False, "state": False},
        # one generated token: latency
        {"name": "token", "op": "token", "batch": 1, "heads": 12, "kv_heads": 12, "dk": 64, "dv": 64, "dtype": "bf16"},
        # one token each of a hundred sequences of the larger model: the states' way through the chip
        {"name": "token batch", "op": "token", "batch": 100, "heads": 16, "kv_heads": 4, "dk": 128, "dv": 128, "dtype": "bf16"},
        # the training batch's layer, backwards
        {"name": "pullback batch", "op": "pullback", "batch": 8, "basis": 1, "heads": 12, "kv_heads": 12, "length": 1024, "dk": 64, "dv": 64,
         "dtype": "bf16", "lengths": False, "state": False},
        # a few directions of an interface through a long layer
        {"name": "pullback basis", "op": "pullback", "batch": 4, "basis": 4, "heads": 16, "kv_heads": 16, "length": 4096, "dk": 128, "dv": 128,
         "dtype": "bf16", "lengths": False, "state": False},
        # one token far into its context takes its position
        {"name": "rotary token", "op": "rotary", "batch": 1, "heads": 12, "kv_heads": 12, "length": 1, "dim": 64, "rotary": 64, "table": 32768,
         "interleaved": False, "positions": True, "dtype": "bf16"},
        # the training batch: queries and keys out of the packed projection, turned
        {"name": "rotary batch", "op": "rotary", "batch": 8, "heads": 12, "kv_heads": 12, "length": 1024, "dim": 64, "rotary": 64, "table": 1024,
         "interleaved": False, "positions": False, "dtype": "bf16"},
        # back from heads that share keys and values, half of each head turned, neighbours in pairs
        {"name": "rotary backward", "op": "rotary_backward", "batch": 4, "basis": 1, "heads": 16, "kv_heads": 4, "length": 4096, "dim": 128,
         "rotary": 64, "table": 4096, "interleaved": True, "positions": False, "dtype": "bf16"},
        # the training batch between two halves of a block, an fp32 residual stream, a gate for each channel
        {"name": "norms batch", "op": "norms", "batch": 8, "length": 1024, "dim": 768, "dtype": "bf16", "residual": "f32", "gate": "channel"},
        # backwards, a wider model with a gate for each sequence
        {"name": "norms backward", "op": "norms_backward", "batch": 5, "length": 1003, "dim": 2048, "dtype": "bf16", "residual": "bf16",
         "gate": "sequence"},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even in its logarithm."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(("prompt", "prompt", "token", "pullback", "pullback", "rotary", "rotary_backward", "norms", "norms_backward"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    if op in ("norms", "norms_backward"):
        dim = _spread(rng, 64, 8192)
        if rng.random() < 0.75:  # mostly widths that models have, some that end anywhere
            dim = max(64, dim // 64 * 64)
        rows = _spread(rng, 1, min(32768, 32_000_000 // dim))
        batch = rng.randint(1, min(rows, 8))
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        return {"op": op, "batch": batch, "length": rows // batch, "dim": dim, "dtype": dtype, "residual": rng.choice((dtype, "f32")),
                "gate": rng.choice(("none", "channel", "sequence", "position"))}
    kv_heads, group = rng.choice((1, 2, 3, 4, 8, 12, 16)), rng.choice((1, 1, 1, 2, 4))
    heads = kv_heads * group
    if op in ("rotary", "rotary_backward"):
        dim = rng.choice((64, 64, 128, 128, 2 * rng.randint(4, 128)))
        rotary = dim if rng.random() < 0.5 else 2 * rng.randint(1, dim // 2)
        batch, basis = _spread(rng, 1, 16), _spread(rng, 1, 8) if op == "rotary_backward" else 1
        length = _spread(rng, 1, max(1, min(8192, 100_000_000 // (batch * basis * heads * 3 * dim))))
        case = {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "length": length, "dim": dim, "rotary": rotary,
                "table": length, "interleaved": rng.random() < 0.5, "positions": rng.random() < 0.5, "dtype": rng.choice((dtype, dtype, "f32"))}
        if case["positions"]:
            case["table"] = _spread(rng, length, 32768)
        return {**case, "basis": basis} if op == "rotary_backward" else case
    dk, dv = rng.choice((64, 128)), rng.choice((64, 128))
    if rng.random() < 0.6:
        dv = dk
    elif rng.random() < 0.5:
        dk, dv = rng.randint(8, 128), rng.randint(8, 128)
    case = {"op": op, "batch": _spread(rng, 1, 128 if op == "token" else 16), "heads": heads, "kv_heads": kv_heads, "dk": dk, "dv": dv, "dtype": dtype}
    if op == "token":
        return case
    basis = _spread(rng, 1, 16) if op == "pullback" else 1
    length = _spread(rng, 1, max(1, min(8192, 60_000_000 // (case["batch"] * basis * heads * (dk + dv)))))
    case.update(length=length, lengths=rng.random() < 0.4, state=rng.random() < 0.4)
    if op == "pullback":
        case.update(basis=basis, lengths=case["lengths"] and not case["state"])
    return case


def _rotary_tables(length, rotary):
    """cos and sin of the angles of ``length`` positions, [length, rotary / 2]."""
    frequency = 10000.0 ** (-torch.arange(rotary // 2, dtype=torch.float64, device="cuda") * 2 / rotary)
    angle = torch.arange(length, dtype=torch.float64, device="cuda")[:, None] * frequency
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, std=1.0, dtype=None):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype or _TYPES[case["dtype"]])

    state = {"case": case}
    op, batch = case["op"], case["batch"]
    if op in ("norms", "norms_backward"):
        length, dim, stream = case["length"], case["dim"], _TYPES[case["residual"]]
        shape = {"none": None, "channel": (dim,), "sequence": (batch, 1, dim), "position": (batch, length, dim)}[case["gate"]]
        state["post_weight"] = (1.0 + rand(dim, std=0.1, dtype=torch.float32)).to(_TYPES[case["dtype"]])
        state["weight"] = (1.0 + rand(dim, std=0.1, dtype=torch.float32)).to(_TYPES[case["dtype"]])
        state["gate"] = None if shape is None else rand(*shape, std=0.5)
        state["branch"] = rand(batch, length, dim)
        state["residual"] = rand(batch, length, dim, std=2.0, dtype=stream)
        if op == "norms_backward":
            state["g_normed"], state["g_residual"] = rand(batch, length, dim), rand(batch, length, dim, std=0.5, dtype=stream)
        state["residual_scale"] = 0.875
        return state
    heads, kv_heads = case["heads"], case["kv_heads"]
    if op in ("rotary", "rotary_backward"):
        length, dim = case["length"], case["dim"]
        state["cos"], state["sin"] = _rotary_tables(case["table"], case["rotary"])
        state["positions"] = None
        if case["positions"]:  # somewhere in their contexts, each sequence's one after the other
            first = torch.randint(0, case["table"] - length + 1, (batch, 1), generator=gen, device="cuda")
            state["positions"] = first + torch.arange(length, device="cuda")
        if op == "rotary":
            state["qkv"] = rand(batch, length, (heads + 2 * kv_heads) * dim)
        else:
            state["dq"], state["dk"], state["dv"] = (rand(batch, case["basis"], heads, length, dim) for _ in range(3))
        return state
    dk, dv = case["dk"], case["dv"]
    # heads that remember from two tokens to five hundred
    state["log_decay"] = -(2.0 ** -torch.linspace(1, 9, heads, device="cuda"))
    state["scale"] = dk ** -0.5
    if op == "token":
        state["q"], state["k"], state["v"] = rand(batch, heads, dk), rand(batch, kv_heads, dk), rand(batch, kv_heads, dv)
        state["state"] = rand(batch, heads, dk, dv, std=2.0, dtype=torch.float32)
        return state
    length = case["length"]
    state["q"], state["k"], state["v"] = rand(batch, heads, length, dk), rand(batch, kv_heads, length, dk), rand(batch, kv_heads, length, dv)
    state["lengths"] = torch.randint(0, length + 1, (batch,), generator=gen, device="cuda") if case["lengths"] else None
    state["state"] = rand(batch, heads, dk, dv, std=2.0, dtype=torch.float32) if case["state"] else None
    if op == "pullback":
        state["g_out"] = rand(batch, case["basis"], heads, length, dv)
        state["g_state"] = rand(batch, case["basis"], heads, dk, dv, std=0.5, dtype=torch.float32) if case["state"] else None
    return state


def _run_own(s):
    from latent_bounded_interfaces_amd.hip.transformer.block import gated_residual_rmsnorm, gated_residual_rmsnorm_pullback
    from latent_bounded_interfaces_amd.hip.transformer.mixer import (linear_attention, linear_attention_input_pullback_basis,
                                                                     linear_attention_step, rotary_heads, rotary_heads_pullback)

    case = s["case"]
    if case["op"] == "prompt":
        return linear_attention(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"], state=s["state"], lengths=s["lengths"])
    if case["op"] == "token":
        return linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], scale=s["scale"]), s["state"]
    if case["op"] == "pullback":
        grads = linear_attention_input_pullback_basis(s["q"], s["k"], s["v"], s["g_out"], s["log_decay"], scale=s["scale"], state=s["state"],
                                                      g_state=s["g_state"], lengths=s["lengths"])
        return grads if case["state"] else grads[:3]
    if case["op"] == "rotary":
        return rotary_heads(s["qkv"], s["cos"], s["sin"], n_heads=case["heads"], n_kv_heads=case["kv_heads"], interleaved=case["interleaved"],
                            positions=s["positions"])
    if case["op"] == "rotary_backward":
        return rotary_heads_pullback(s["dq"], s["dk"], s["dv"], s["cos"], s["sin"], n_kv_heads=case["kv_heads"],
                                     interleaved=case["interleaved"], positions=s["positions"])
    if case["op"] == "norms":
        return gated_residual_rmsnorm(s["branch"], s["residual"], s["post_weight"], s["weight"], _EPS, gate=s["gate"],
                                      residual_scale=s["residual_scale"])
    grads = gated_residual_rmsnorm_pullback(s["g_normed"], s["branch"], s["residual"], s["post_weight"], s["weight"], _EPS, gate=s["gate"],
                                            residual_scale=s["residual_scale"], g_residual=s["g_residual"], sequence_gate=case["gate"] == "sequence")
    return tuple(g for g in grads if g is not None)


def _mix(a, b, c, log_decay, first=None, on_first=1):
    """out_i = sum over j <= i of decay^(i - j) (a_i . b_j) c_j, plus decay^(i + on_first) a_i first: chunks of 64, a triangle in each and a
    state in front of each.  a, b, c [..., H, T, D] in 32 bits."""
    length = a.shape[-2]
    chunks = -(-length // _CHUNK)

    def cut(t):
        t = torch.nn.functional.pad(t, (0, 0, 0, chunks * _CHUNK - length))
        return t.reshape(*t.shape[:-2], chunks, _CHUNK, t.shape[-1])

    a, b, c = cut(a), cut(b), cut(c)
    rate = log_decay.double()[:, None, None, None]
    at = torch.arange(_CHUNK, device=a.device)
    apart = (at[:, None] - at).clamp(min=0)
    inside = torch.where(at[:, None] >= at, (rate * apart).exp(), 0.0).float()
    out = ((a @ b.transpose(-1, -2)) * inside) @ c
    left = (rate * (_CHUNK - 1 - at)[:, None]).exp().float()
    ends = (b * left).transpose(-1, -2) @ c
    number = torch.arange(chunks, device=a.device)
    behind = (number[:, None] - 1 - number).clamp(min=0)
    carried = torch.where(number[:, None] > number, (rate[..., 0] * (_CHUNK * behind)).exp(), 0.0).float()
    starts = (carried @ ends.flatten(-2)).view(ends.shape)
    out = out + (a * (rate * (at + 1)[:, None]).exp().float()) @ starts
    if first is not None:
        since = number[:, None] * _CHUNK + at + on_first
        out = out + (a * (rate * since[:, :, None]).exp().float()) @ first[..., None, :, :]
    out = out.flatten(-3, -2)
    return out[..., :length, :]


def _valid(s, t):
    """``t`` [B, ..., T, D] in 32 bits, zero behind each sequence's end."""
    t = t.float()
    if s["lengths"] is None:
        return t
    inside = torch.arange(t.shape[-2], device=t.device) < s["lengths"][:, None]
    return torch.where(inside.view(t.shape[0], *[1] * (t.dim() - 3), -1, 1), t, 0.0)


def _prompt(s):
    dtype, group = s["q"].dtype, s["case"]["heads"] // s["case"]["kv_heads"]
    q, k, v = (_valid(s, s[name]) for name in ("q", "k", "v"))
    k, v = k.repeat_interleave(group, dim=1), v.repeat_interleave(group, dim=1)
    out = _mix(q, k, v, s["log_decay"], s["state"])
    batch, length = q.shape[0], q.shape[2]
    ends = torch.full((batch,), length, device=q.device) if s["lengths"] is None else s["lengths"]
    rate = s["log_decay"].double()
    behind = (ends[:, None] - 1 - torch.arange(length, device=q.device)).clamp(min=0)
    left = (rate[:, None] * behind[:, None]).exp().float()
    final = (k * left[..., None]).transpose(-1, -2) @ v
    if s["state"] is not None:
        final = final + (rate * ends[:, None]).exp().float()[..., None, None] * s["state"]
    return (out * s["scale"]).to(dtype), final


def _token(s):
    dtype, group = s["q"].dtype, s["case"]["heads"] // s["case"]["kv_heads"]
    k, v = s["k"].float().repeat_interleave(group, dim=1), s["v"].float().repeat_interleave(group, dim=1)
    s["state"].mul_(s["log_decay"].exp()[:, None, None]).add_(k[..., None] * v[..., None, :])
    return ((s["q"].float()[..., None] * s["state"]).sum(dim=-2) * s["scale"]).to(dtype), s["state"]


def _pullback(s):
    dtype, group = s["q"].dtype, s["case"]["heads"] // s["case"]["kv_heads"]
    q, k, v, g = (_valid(s, s[name]) for name in ("q", "k", "v", "g_out"))
    k, v = k.repeat_interleave(group, dim=1), v.repeat_interleave(group, dim=1)
    q, k, v = q[:, None], k[:, None], v[:, None]
    g = g * s["scale"]
    rate = s["log_decay"]
    state, g_state = s["state"], s["g_state"]
    dq = _mix(g, v, k, rate, None if state is None else state[:, None].transpose(-1, -2))
    q, k, v, g = (t.flip(-2) for t in (q, k, v, g))
    # the later tokens first; the cotangent of the last state meets the last token undiminished
    dk = _mix(v, g, q, rate, None if g_state is None else g_state.transpose(-1, -2), on_first=0).flip(-2)
    dv = _mix(k, q, g, rate, g_state, on_first=0).flip(-2)
    grads = tuple(t.to(dtype) for t in (dq, dk, dv))
    if state is None:
        return grads
    length = q.shape[-2]
    left = (rate.double()[:, None] * (length - torch.arange(length, device=q.device))).exp().float()
    back = (q * left[..., None]).transpose(-1, -2) @ g
    return (*grads, back + (rate.double() * length).exp().float()[:, None, None] * g_state)


def _turned(s, x, back):
    """``x`` [..., T, D] turned by the angles of its positions, or back."""
    rotary, length = s["case"]["rotary"], x.shape[-2]
    at = torch.arange(length, device=x.device) if s["positions"] is None else s["positions"]
    cos, sin = s["cos"][at], s["sin"][at]
    if s["positions"] is not None:
        cos, sin = (t.view(t.shape[0], *[1] * (x.dim() - 3), *t.shape[1:]) for t in (cos, sin))
    if back:
        sin = -sin
    turned, rest = x[..., :rotary].float(), x[..., rotary:].float()
    if s["case"]["interleaved"]:
        first, second = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((first * cos - second * sin, first * sin + second * cos), dim=-1).flatten(-2)
    else:
        first, second = turned.chunk(2, dim=-1)
        turned = torch.cat((first * cos - second * sin, first * sin + second * cos), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _rotary(s):
    case = s["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    x = s["qkv"].view(case["batch"], case["length"], heads + 2 * kv_heads, dim).transpose(1, 2)
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    return _turned(s, q, False).to(q.dtype), _turned(s, k, False).to(q.dtype), v


def _rotary_backward(s):
    case, dtype = s["case"], s["dq"].dtype
    shared = (case["batch"], case["basis"], case["kv_heads"], -1, case["length"], case["dim"])
    dq = _turned(s, s["dq"], True)
    dk = _turned(s, s["dk"].float().view(shared).sum(dim=3), True)
    dv = s["dv"].float().view(shared).sum(dim=3)
    return torch.cat((dq, dk, dv), dim=2).transpose(2, 3).flatten(-2).to(dtype)


def _norms(s):
    branch = s["branch"].float()
    unit = branch * torch.rsqrt((branch * branch).mean(dim=-1, keepdim=True) + _EPS)
    added = unit * s["post_weight"].float()
    if s["gate"] is not None:
        added = added * s["gate"].float()
    total = s["residual_scale"] * s["residual"].float() + added
    normed = total * torch.rsqrt((total * total).mean(dim=-1, keepdim=True) + _EPS) * s["weight"].float()
    return normed.to(s["branch"].dtype), total.to(s["residual"].dtype)


def _norms_backward(s):
    dtype, stream = s["branch"].dtype, s["residual"].dtype
    x, g = s["residual"].float(), s["g_normed"].float()
    inv = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + _EPS)
    unit, pulled = x * inv, g * s["weight"].float()
    total = inv * (pulled - unit * (unit * pulled).mean(dim=-1, keepdim=True)) + s["g_residual"].float()
    g_weight = (g * unit).sum(dim=(0, 1))
    branch = s["branch"].float()
    inv = torch.rsqrt((branch * branch).mean(dim=-1, keepdim=True) + _EPS)
    unit = branch * inv
    post = s["post_weight"].float()
    opened = total if s["gate"] is None else total * s["gate"].float()
    pulled = opened * post
    g_branch = inv * (pulled - unit * (unit * pulled).mean(dim=-1, keepdim=True))
    grads = [g_branch.to(dtype), (s["residual_scale"] * total).to(stream)]
    if s["case"]["gate"] == "position":
        grads.append((total * unit * post).to(dtype))
    elif s["case"]["gate"] == "sequence":
        grads.append((total * unit * post).sum(dim=1, keepdim=True))
    elif s["case"]["gate"] == "channel":
        grads.append((total * unit * post).sum(dim=(0, 1)))
    return (*grads, (opened * unit).sum(dim=(0, 1)), g_weight)


_PLAIN = {"prompt": _prompt, "token": _token, "pullback": _pullback, "rotary": _rotary, "rotary_backward": _rotary_backward,
          "norms": _norms, "norms_backward": _norms_backward}


def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state["case"]["op"]](state)


def work(case):
    """Every input read once, every output written once.  Of linear attention the operations of its recurrence, which has the fewest."""
    op, batch, b = case["op"], case["batch"], _SIZES[case["dtype"]]
    if op in ("norms", "norms_backward"):
        rows, dim, r = batch * case["length"], case["dim"], _SIZES[case["residual"]]
        gates = {"none": 0, "channel": 1, "sequence": batch, "position": rows}[case["gate"]]
        if op == "norms":
            return {"bytes": rows * dim * (2 * b + 2 * r) + dim * b * (2 + gates), "flops": 10 * rows * dim}
        of_gate = b if case["gate"] == "position" else 4
        return {"bytes": rows * dim * (3 * b + 3 * r) + dim * (2 * b + 8 + gates * (b + of_gate)), "flops": 25 * rows * dim}
    heads, kv_heads = case["heads"], case["kv_heads"]
    if op in ("rotary", "rotary_backward"):
        rows = batch * case["length"] * case.get("basis", 1)
        angles = 4 * case["rotary"] * (batch if case["positions"] else 1) * case["length"]
        if op == "rotary":  # the values stay where they are
            return {"bytes": rows * 2 * (heads + kv_heads) * case["dim"] * b + angles, "flops": 3 * rows * (heads + kv_heads) * case["rotary"]}
        return {"bytes": rows * (4 * heads + 2 * kv_heads) * case["dim"] * b + angles, "flops": rows * (heads * (2 * case["dim"] + 3 * case["rotary"]))}
    dk, dv = case["dk"], case["dv"]
    states = 4 * batch * heads * dk * dv
    if op == "token":
        return {"bytes": 2 * states + b * batch * (heads + kv_heads) * (dk + dv) + 4 * heads, "flops": 5 * batch * heads * dk * dv}
    rows = batch * case["length"]
    inputs = b * rows * (heads * dk + kv_heads * (dk + dv))
    if op == "prompt":
        return {"bytes": inputs + b * rows * heads * dv + states * (2 if case["state"] else 1), "flops": 4 * rows * heads * dk * dv}
    basis = case["basis"]
    moved = inputs + b * rows * basis * heads * (2 * dk + 2 * dv) + (states * (1 + 2 * basis) if case["state"] else 0)
    return {"bytes": moved, "flops": rows * heads * dk * dv * (2 + 8 * basis)}


def _sums(a, b, c, log_decay, reverse=False):
    """The sums of linear attention by their definition, a triangle of pairs for each head; a, b, c [N, T, D], log_decay [N]."""
    length = a.shape[1]
    at = torch.arange(length, device=a.device, dtype=torch.float64)
    apart = at[None, :] - at[:, None] if reverse else at[:, None] - at[None, :]
    out = torch.empty(*a.shape[:2], c.shape[2], dtype=torch.float64, device=a.device)
    step = max(1, (1 << 25) // length ** 2)
    for n in range(0, a.shape[0], step):
        part = slice(n, n + step)
        pairs = torch.exp(log_decay[part, None, None] * apart.clamp(min=0)).mul_(apart >= 0)
        pairs.mul_(torch.matmul(a[part], b[part].mT.contiguous()))
        out[part] = torch.matmul(pairs, c[part])
    return out


def _exact_linear(case, s, d):
    group, scale, rate = case["heads"] // case["kv_heads"], s["scale"], d["log_decay"]
    shared = [d["k"].repeat_interleave(group, 1), d["v"].repeat_interleave(group, 1)]
    if case["op"] == "token":
        new = rate.exp().view(-1, 1, 1) * d["state"] + torch.einsum("bhi,bhj->bhij", *shared)
        return torch.einsum("bhi,bhij->bhj", d["q"], new) * scale, new
    batch, heads, length = d["q"].shape[:3]
    ends = torch.full((batch,), length, device="cuda") if s["lengths"] is None else s["lengths"]
    live = (torch.arange(length, device="cuda") < ends[:, None]).double()
    q, k, v = (t * live[:, None, :, None] for t in (d["q"], *shared))
    t_at = torch.arange(length, device="cuda", dtype=torch.float64)
    past = torch.exp(rate.view(1, -1, 1) * (t_at + 1.0))  # of the first state, at each token
    flat = lambda t: t.reshape(-1, *t.shape[-2:])  # noqa: E731
    if case["op"] == "prompt":
        out = _sums(flat(q), flat(k), flat(v), rate.repeat(batch)).view(batch, heads, length, -1)
        weights = torch.exp(rate.view(1, -1, 1) * (ends.view(-1, 1, 1) - 1 - t_at).clamp(min=0))
        final = torch.matmul((k * weights[..., None]).mT.contiguous(), v)
        if s["state"] is not None:
            out = out + torch.matmul(q * past[..., None], d["state"])
            final = final + torch.exp(rate * ends[:, None])[..., None, None] * d["state"]
        return out * scale, final
    g = d["g_out"] * live[:, None, None, :, None] * scale
    basis = case["basis"]
    rates = rate.repeat(batch)
    found = []
    for p in range(basis):
        gp = g[:, p]
        dq = _sums(flat(gp), flat(v), flat(k), rates).view_as(q)
        dk = _sums(flat(v), flat(gp), flat(q), rates, reverse=True).view_as(k)
        dv = _sums(flat(k), flat(q), flat(gp), rates, reverse=True).view_as(v)
        if s["state"] is None:
            found.append((dq, dk, dv))
            continue
        # through the first state and the last one: S_T = decay^T S_0 + sum of decay^(T-1-j) k_j v_j
        gs = d["g_state"][:, p]
        dq = dq + torch.matmul(gp * past[..., None], d["state"].mT.contiguous())
        rest = torch.exp(rate.view(1, -1, 1) * (length - 1 - t_at))[..., None]
        dk = dk + rest * torch.matmul(v, gs.mT.contiguous())
        dv = dv + rest * torch.matmul(k, gs)
        ds = torch.exp(rate * length).view(1, -1, 1, 1) * gs + torch.matmul((q * past[..., None]).mT.contiguous(), gp)
        found.append((dq, dk, dv, ds))
    return tuple(torch.stack(parts, dim=1) for parts in zip(*found))


def _exact_rotary(case, s, d):
    rotary, length, kv = case["rotary"], case["length"], case["kv_heads"]
    at = torch.arange(length, device="cuda").expand(case["batch"], length) if s["positions"] is None else s["positions"]
    turn = torch.complex(d["cos"], d["sin"])[at]  # [B, T, rotary / 2]

    def turned(x, by):  # x [B, T, ..., D]
        by = by.view(*by.shape[:2], *[1] * (x.dim() - 3), by.shape[2])
        pairs = x[..., :rotary].unflatten(-1, (-1, 2) if case["interleaved"] else (2, -1))
        along = -1 if case["interleaved"] else -2
        z = torch.complex(*(t.contiguous() for t in pairs.unbind(along))) * by
        return torch.cat((torch.stack((z.real, z.imag), dim=along).flatten(-2), x[..., rotary:]), dim=-1)

    if case["op"] == "rotary":
        x = d["qkv"].view(case["batch"], length, -1, case["dim"])
        q, k, v = x.split((case["heads"], kv, kv), dim=2)
        return tuple(t.transpose(1, 2) for t in (turned(q, turn), turned(k, turn), v))
    dq, dk, dv = (d[name].permute(0, 3, 1, 2, 4) for name in ("dq", "dk", "dv"))  # [B, T, P, H, D]
    dk, dv = (t.unflatten(3, (kv, -1)).sum(4) for t in (dk, dv))
    back = turn.conj().resolve_conj()
    return torch.cat((turned(dq, back), turned(dk, back), dv), dim=3).permute(0, 2, 1, 3, 4).flatten(-2)


def _exact_norms(case, s, d):
    n, alpha = case["dim"], s["residual_scale"]
    gate = d["gate"] if s["gate"] is not None else torch.ones((), dtype=torch.float64, device="cuda")
    root = lambda t: (t.pow(2).sum(-1, keepdim=True) / n + _EPS).sqrt()  # noqa: E731
    if case["op"] == "norms":
        total = alpha * d["residual"] + gate * (d["branch"] / root(d["branch"]) * d["post_weight"])
        return total / root(total) * d["weight"], total
    # y_j = w_j x_j / m with m = sqrt(mean(x^2) + eps), so dy_j/dx_i = w_j (delta_ij / m - x_i x_j / (n m^3))
    x, g = d["residual"], d["g_normed"]
    m = root(x)
    g_total = g * d["weight"] / m - x * (g * d["weight"] * x).sum(-1, keepdim=True) / (n * m ** 3) + d["g_residual"]
    y, m2 = d["branch"], root(d["branch"])
    g_u = g_total * gate
    g_branch = g_u * d["post_weight"] / m2 - y * (g_u * d["post_weight"] * y).sum(-1, keepdim=True) / (n * m2 ** 3)
    through = g_total * d["post_weight"] * y / m2
    g_gate = {"none": [], "channel": [through.sum((0, 1))], "sequence": [through.sum(1, keepdim=True)], "position": [through]}[case["gate"]]
    return (g_branch, alpha * g_total, *g_gate, (g_u * y / m2).sum((0, 1)), (g * x / m).sum((0, 1)))


def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    d = {name: value.double() for name, value in s.items() if isinstance(value, torch.Tensor) and value.is_floating_point()}
    if case["op"] in ("prompt", "token", "pullback"):
        return _exact_linear(case, s, d)
    if case["op"] in ("rotary", "rotary_backward"):
        return _exact_rotary(case, s, d)
    return _exact_norms(case, s, d)
