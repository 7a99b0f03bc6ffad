"""The operators of a rotary, gated ViT block, as a user's program calls them.

Newer vision transformers differ from the classic block in three places, and
each is an operator here:

* `rotary`: positions on several axes (row and column of an image's patch; time,
  row and column of a video's) rotate pairs of a head's values, instead of a
  table added to the tokens. The gradient is the rotation backwards.
* `qk_norm`: queries and keys are normalised for each head (root mean square or
  LayerNorm) and rotated, in one pass over the packed QKV projection; with its
  backward pass. The packed result is what attention takes next.
* `gated`: the MLP's first product, activation(gate) * value, both halves in one
  weight; for training it keeps the preactivations, from which `gated_backward`
  gives their gradient.

Sizes: 197 tokens are a 224-pixel image in 16-pixel patches and the class token,
577 a 384-pixel one; 192 columns and 3 heads are ViT-Tiny, 768 and 12 ViT-Base.
A gated MLP's hidden width is 2/3 of a classic one's: 512 for 192 columns, 2048
for 768. A video is frames of such patches, a token each.
"""

from __future__ import annotations

import functools
import math
import os
import sys

import torch

own = False

DEVICE = "cuda:0"
EPSILON = 1.0e-6
STORAGE = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}


@functools.lru_cache(maxsize=1)
def _cuvit():
    path = os.path.abspath("cu-vit_amd")  # imported from the repository's root
    if path not in sys.path:
        sys.path.insert(0, path)
    import cuvit_amd

    return cuvit_amd


def listed():
    return [
        # One image through a single-image forward: the smallest rotation, where
        # the call itself is most of the time. Heads split into halves.
        {"name": "rotary_f32_image", "op": "rotary", "dtype": "f32", "images": 1, "frames": 1, "rows": 14,
         "columns": 14, "lead": 1, "heads": 3, "head_dim": 64, "pairs": "16,16", "pairing": "halves",
         "inverse": False, "heads_first": False, "shared": True, "start": 0.0},
        # Four clips of 16 frames in bf16, time, row and column, adjacent pairs,
        # queries as attention by heads keeps them: the gradient's direction.
        {"name": "rotary_bf16_video_inverse", "op": "rotary", "dtype": "bf16", "images": 4, "frames": 16,
         "rows": 14, "columns": 14, "lead": 0, "heads": 12, "head_dim": 64, "pairs": "8,12,12",
         "pairing": "adjacent", "inverse": True, "heads_first": True, "shared": True, "start": 0.0},
        # ViT-Tiny's QKV projection at the reference's precision and a serving batch.
        {"name": "qk_norm_f32_tiny_b32", "op": "qk_norm", "dtype": "f32", "images": 32, "frames": 1, "rows": 14,
         "columns": 14, "lead": 1, "heads": 3, "kv_heads": 3, "head_dim": 64, "pairs": "16,16",
         "pairing": "halves", "norm": "rms", "beta": False, "shared": True, "start": 0.0},
        # ViT-Base's at a large batch in bf16: throughput.
        {"name": "qk_norm_bf16_base_b64", "op": "qk_norm", "dtype": "bf16", "images": 64, "frames": 1, "rows": 14,
         "columns": 14, "lead": 1, "heads": 12, "kv_heads": 12, "head_dim": 64, "pairs": "16,16",
         "pairing": "halves", "norm": "rms", "beta": False, "shared": True, "start": 0.0},
        # A long video in one sequence: heads of 80, keys shared by groups of
        # heads, LayerNorm with its shift, a part of each head left unrotated.
        {"name": "qk_norm_bf16_long_video", "op": "qk_norm", "dtype": "bf16", "images": 1, "frames": 16,
         "rows": 28, "columns": 28, "lead": 1, "heads": 12, "kv_heads": 4, "head_dim": 80, "pairs": "8,12,12",
         "pairing": "halves", "norm": "layer", "beta": True, "shared": False, "start": 1000.0},
        # The backward pass at ViT-Base's fine-tuning batch.
        {"name": "qk_norm_backward_bf16_b16", "op": "qk_norm_backward", "dtype": "bf16", "images": 16,
         "frames": 1, "rows": 14, "columns": 14, "lead": 1, "heads": 12, "kv_heads": 12, "head_dim": 64,
         "pairs": "16,16", "pairing": "halves", "norm": "rms", "beta": False, "shared": True, "start": 0.0},
        # And at 384 pixels in fp32, LayerNorm with its shift, adjacent pairs.
        {"name": "qk_norm_backward_f32_577", "op": "qk_norm_backward", "dtype": "f32", "images": 4,
         "frames": 1, "rows": 24, "columns": 24, "lead": 1, "heads": 6, "kv_heads": 6, "head_dim": 64,
         "pairs": "16,16", "pairing": "adjacent", "norm": "layer", "beta": True, "shared": False, "start": 0.0},
        # One token (a class token attended to last) through ViT-Base's gated MLP.
        {"name": "gated_bf16_one_token", "op": "gated", "dtype": "bf16", "m": 1, "n": 2048, "k": 768,
         "activation": "silu", "bias": True, "keep": False},
        # ViT-Base's at a large batch: the largest case.
        {"name": "gated_bf16_base_b64", "op": "gated", "dtype": "bf16", "m": 64 * 197, "n": 2048, "k": 768,
         "activation": "silu", "bias": True, "keep": False},
        # A training forward in fp32 at odd sizes: the preactivations are kept.
        {"name": "gated_f32_train_odd", "op": "gated", "dtype": "f32", "m": 4 * 577, "n": 1365, "k": 512,
         "activation": "gelu_tanh", "bias": True, "keep": True},
        # The gate's gradient at the fine-tuning batch.
        {"name": "gated_backward_bf16_b16", "op": "gated_backward", "dtype": "bf16", "m": 16 * 197, "n": 2048,
         "activation": "silu"},
        # And of one fp32 image at an odd width.
        {"name": "gated_backward_f32_image", "op": "gated_backward", "dtype": "f32", "m": 197, "n": 683,
         "activation": "gelu"},
    ]


# -- drawn cases ----------------------------------------------------------------

_LARGEST_FLOPS = 4 * 64 * 197 * 2048 * 768
_LARGEST_BYTES = 2 * 2 * 64 * 197 * 3 * 768


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _draw_grid(rng):
    """Images or clips, their patches and their head layout."""
    head_dim = rng.choice([32, 48, 64, 64, 64, 72, 80, 88, 96, 128, 128, 256])
    half = head_dim // 2
    rotated = rng.choice([half, half, half, half // 2])
    axes = rng.choice([1, 2, 2, 3])
    pairs = [rotated // axes] * axes
    pairs[-1] += rotated - sum(pairs)
    frames = rng.choice([1, 1, 1, _log_uniform(rng, 2, 32)])
    side = rng.randint(1, 32)
    return {"images": _log_uniform(rng, 1, 64), "frames": frames, "rows": side,
            "columns": rng.choice([side, rng.randint(1, 32)]), "lead": rng.choice([0, 1, 1, 5]),
            "heads": rng.choice([1, 2, 3, 6, 8, 12, 16]), "head_dim": head_dim,
            "pairs": ",".join(str(p) for p in pairs), "pairing": rng.choice(["halves", "adjacent"]),
            "shared": rng.random() < 0.6, "start": rng.choice([0.0, 0.0, float(rng.randint(1, 100000))])}


def draw(rng):
    """A case of the same ranges, other than the listed ones."""
    while True:
        op = rng.choice(["rotary", "rotary", "qk_norm", "qk_norm", "qk_norm_backward", "gated", "gated",
                         "gated_backward"])
        case = {"op": op, "dtype": rng.choice(["f32", "bf16", "bf16"])}
        if op in ("rotary", "qk_norm", "qk_norm_backward"):
            case.update(_draw_grid(rng))
        if op == "rotary":
            case.update(inverse=rng.random() < 0.5, heads_first=rng.random() < 0.3)
        elif op in ("qk_norm", "qk_norm_backward"):
            heads = case["heads"]
            case["kv_heads"] = rng.choice([heads, heads] + [d for d in (1, 2, 4) if heads % d == 0])
            case["norm"] = rng.choice(["rms", "layer"])
            case["beta"] = rng.random() < (0.7 if case["norm"] == "layer" else 0.1)
        else:
            width = rng.choice([192, 384, 768, rng.randint(24, 1100)])
            case["m"] = rng.choice([_log_uniform(rng, 1, 64 * 197), _log_uniform(rng, 1, 64 * 197),
                                    _log_uniform(rng, 1, 16)])
            case["n"] = rng.choice([8 * width // 3, 2 * width, rng.randint(17, 2100)])
            if op == "gated":
                case["k"] = width
                case.update(bias=rng.random() < 0.7, keep=rng.random() < 0.3)
            case["activation"] = rng.choice(["silu", "silu", "gelu", "gelu_tanh"])
        cost = work(case)
        dear = (cost["flops"] * (10 if case["dtype"] == "f32" and op == "gated" else 1) > _LARGEST_FLOPS
                or cost["bytes"] > _LARGEST_BYTES)
        if not dear and not any({**case, "name": known["name"]} == known for known in listed()):
            return case


# -- sizes ----------------------------------------------------------------------


def _tokens(case):
    return case["lead"] + case["frames"] * case["rows"] * case["columns"]


def _pairs(case):
    return [int(p) for p in case["pairs"].split(",")]


def _slots(case):
    return case["heads"] + 2 * case["kv_heads"]


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "gated":
        m, n, k = case["m"], case["n"], case["k"]
        outputs = m * n * (3 if case["keep"] else 1)
        return {"bytes": size * (m * k + 2 * n * k + outputs) + 4 * (2 * n if case["bias"] else 0),
                "flops": 4 * m * n * k}
    if case["op"] == "gated_backward":
        return {"bytes": size * 5 * case["m"] * case["n"], "flops": 20 * case["m"] * case["n"]}
    tokens, images, width = _tokens(case), case["images"], case["head_dim"]
    positions = 4 * tokens * len(_pairs(case)) * (1 if case["shared"] else images)
    if case["op"] == "rotary":
        values = images * tokens * case["heads"] * width
        return {"bytes": 2 * size * values + positions, "flops": 3 * values}
    normed = images * tokens * (case["heads"] + case["kv_heads"]) * width
    values = images * tokens * _slots(case) * width
    if case["op"] == "qk_norm":
        return {"bytes": 2 * size * values + positions, "flops": 8 * normed}
    return {"bytes": size * (normed + 2 * values) + positions, "flops": 20 * normed}


# -- what a program has in hand -------------------------------------------------


def _positions(case):
    """[tokens, axes] or [images, tokens, axes]: leading tokens at the origin, a
    patch at its place; where images do not share them, each is shifted."""
    axes = len(_pairs(case))
    grid = torch.stack(torch.meshgrid(torch.arange(case["frames"]), torch.arange(case["rows"]),
                                      torch.arange(case["columns"]), indexing="ij"), dim=-1).reshape(-1, 3)
    grid = grid.float()
    grid[:, 0] += case["start"]
    if axes == 1:
        grid = torch.arange(grid.shape[0], dtype=torch.float32)[:, None] + case["start"]
    else:
        grid = grid[:, 3 - axes:]
    table = torch.cat([torch.zeros(case["lead"], axes), grid])
    if not case["shared"]:
        table = table[None] + torch.arange(case["images"], dtype=torch.float32)[:, None, None]
    return table.contiguous().to(DEVICE)


def _frequencies(case):
    """Each axis its own ladder, 10000^(-i / pairs)."""
    ladders = [torch.pow(torch.tensor(10000.0, dtype=torch.float64), -torch.arange(n, dtype=torch.float64) / max(n, 1))
               for n in _pairs(case)]
    return torch.cat(ladders).float().to(DEVICE)


def prepare(case, seed):
    generator = torch.Generator(device=DEVICE)
    generator.manual_seed(seed)
    kind = STORAGE[case["dtype"]]

    def normal(*shape, mean=0.0, scale=1.0, dtype=kind):
        return (torch.randn(*shape, generator=generator, device=DEVICE) * scale + mean).to(dtype)

    state = {"case": case}
    op = case["op"]
    if op in ("gated", "gated_backward"):
        m, n = case["m"], case["n"]
        if op == "gated":
            k = case["k"]
            state["a"] = normal(m, k)
            state["w"] = normal(2 * n, k, scale=1.0 / math.sqrt(k))
            state["bias"] = normal(2 * n, scale=0.1, dtype=torch.float32) if case["bias"] else None
            state["out"] = torch.empty(m, n, dtype=kind, device=DEVICE)
            state["pre"] = torch.empty(m, 2 * n, dtype=kind, device=DEVICE) if case["keep"] else None
        else:
            state["pre"] = normal(m, 2 * n)
            state["grad"] = normal(m, n)
            state["out"] = torch.empty(m, 2 * n, dtype=kind, device=DEVICE)
        if own:
            cuvit = _cuvit()
            activation = {"silu": cuvit.GATE_SILU, "gelu": cuvit.GATE_GELU,
                          "gelu_tanh": cuvit.GATE_GELU_TANH}[case["activation"]]
            state["problem"] = cuvit.gated_problem(m, n, case.get("k", 1), activation)
        return state
    images, tokens, heads, width = case["images"], _tokens(case), case["heads"], case["head_dim"]
    state["positions"] = _positions(case)
    state["frequencies"] = _frequencies(case)
    stride = 0 if case["shared"] else tokens * len(_pairs(case))
    if op == "rotary":
        shape = (images, heads, tokens, width) if case["heads_first"] else (images, tokens, heads, width)
        state["x"] = normal(*shape)
        state["out"] = torch.empty(*shape, dtype=kind, device=DEVICE)
        if own:
            cuvit = _cuvit()
            pairing = cuvit.ROTARY_HALVES if case["pairing"] == "halves" else cuvit.ROTARY_ADJACENT
            problem = cuvit.rotary_problem(images, tokens, heads, width, _pairs(case), pairing)
            problem.rotation.position_stride = stride
            problem.inverse = int(case["inverse"])
            if case["heads_first"]:
                for strides in (problem.input, problem.output):
                    strides.image, strides.token, strides.head = heads * tokens * width, width, tokens * width
            state["problem"] = problem
        return state
    slots = _slots(case)
    state["qkv"] = normal(images, tokens, slots, width, scale=1.5)
    for name in ("q", "k"):
        state[name + "_gamma"] = normal(width, mean=1.0, scale=0.2, dtype=torch.float32)
        state[name + "_beta"] = normal(width, scale=0.1, dtype=torch.float32) if case["beta"] else None
    state["out"] = torch.empty(images, tokens, slots, width, dtype=kind, device=DEVICE)
    if op == "qk_norm_backward":
        state["grad"] = normal(images, tokens, slots, width)
        for name in ("q_gamma", "k_gamma", "q_beta", "k_beta"):
            wanted = name.endswith("gamma") or case["beta"]
            state["grad_" + name] = torch.empty(width, device=DEVICE) if wanted else None
    if own:
        cuvit = _cuvit()
        pairing = cuvit.ROTARY_HALVES if case["pairing"] == "halves" else cuvit.ROTARY_ADJACENT
        norm = cuvit.NORM_RMS if case["norm"] == "rms" else cuvit.NORM_LAYER
        problem = cuvit.qk_norm_problem(images, tokens, heads, width, _pairs(case), pairing, norm, EPSILON,
                                        kv_heads=case["kv_heads"])
        problem.rotation.position_stride = stride
        state["problem"] = problem
        if op == "qk_norm_backward":
            state["workspace"] = torch.empty(cuvit.qk_norm_rotary_workspace(problem), dtype=torch.uint8,
                                             device=DEVICE)
    return state


# -- one pass -------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _own_rotary(s):
    _cuvit().rotary(s["x"], s["positions"], s["frequencies"], s["out"], s["problem"])
    return s["out"]


def _own_qk_norm(s):
    _cuvit().qk_norm_rotary(s["qkv"], s["q_gamma"], s["k_gamma"], s["positions"], s["frequencies"], s["out"],
                            s["problem"], q_beta=s["q_beta"], k_beta=s["k_beta"])
    return s["out"]


def _own_qk_norm_backward(s):
    _cuvit().qk_norm_rotary_backward(s["qkv"], s["q_gamma"], s["k_gamma"], s["positions"], s["frequencies"],
                                     s["grad"], s["out"], s["problem"], workspace=s["workspace"],
                                     grad_q_gamma=s["grad_q_gamma"], grad_k_gamma=s["grad_k_gamma"],
                                     grad_q_beta=s["grad_q_beta"], grad_k_beta=s["grad_k_beta"])
    return _gradients(s["case"], s["out"], s["grad_q_gamma"], s["grad_k_gamma"], s["grad_q_beta"], s["grad_k_beta"])


def _own_gated(s):
    _cuvit().gated_gemm(s["a"], s["w"], s["bias"], s["out"], s["problem"], preactivations=s["pre"])
    return (s["out"], s["pre"]) if s["case"]["keep"] else s["out"]


def _own_gated_backward(s):
    _cuvit().gated_backward(s["pre"], s["grad"], s["out"], s["problem"])
    return s["out"]


_OWN = {"rotary": _own_rotary, "qk_norm": _own_qk_norm, "qk_norm_backward": _own_qk_norm_backward,
        "gated": _own_gated, "gated_backward": _own_gated_backward}


def _gradients(case, grad_qkv, q_gamma, k_gamma, q_beta, k_beta):
    outputs = {"qkv": grad_qkv, "q_gamma": q_gamma, "k_gamma": k_gamma}
    if case["beta"]:
        outputs.update(q_beta=q_beta, k_beta=k_beta)
    return outputs


# -- the plain forms ------------------------------------------------------------


def _angles(case, positions, frequencies):
    """cos and sin of each token's pairs, [.., tokens, pairs], from angles in 64
    bits: a far position times a frequency of 1 keeps no fraction in 32."""
    axis = torch.repeat_interleave(torch.arange(len(_pairs(case)), device=DEVICE),
                                   torch.tensor(_pairs(case), device=DEVICE), output_size=frequencies.shape[0])
    angle = positions.double()[..., axis] * frequencies.double()
    return torch.cos(angle).float(), torch.sin(angle).float()


def _rotate(case, x, cos, sin):
    """x [.., head_dim] in fp32, cos and sin [.., pairs]."""
    pairs = cos.shape[-1]
    turned, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if case["pairing"] == "halves":
        first, second = turned[..., :pairs], turned[..., pairs:]
        turned = torch.cat([first * cos - second * sin, second * cos + first * sin], dim=-1)
    else:
        first, second = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([first * cos - second * sin, second * cos + first * sin], dim=-1).flatten(-2)
    return torch.cat([turned, rest], dim=-1)


def _plain_rotary(s):
    case = s["case"]
    cos, sin = _angles(case, s["positions"], s["frequencies"])
    if case["inverse"]:
        sin = -sin
    at = -3 if case["heads_first"] else -2  # tokens before heads, or heads before tokens
    return _rotate(case, s["x"].float(), cos.unsqueeze(at), sin.unsqueeze(at)).to(s["x"].dtype)


def _plain_parts(s, x):
    """Queries and keys as [.., heads, head_dim], and the values."""
    heads, kv_heads = s["case"]["heads"], s["case"]["kv_heads"]
    return x[:, :, :heads], x[:, :, heads:heads + kv_heads], x[:, :, heads + kv_heads:]


def _plain_normalised(case, x):
    """The normalised rows and 1 / their spread."""
    if case["norm"] == "layer":
        x = x - x.mean(dim=-1, keepdim=True)
    scale = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPSILON)
    return x * scale, scale


def _plain_qk_norm(s):
    case = s["case"]
    cos, sin = _angles(case, s["positions"], s["frequencies"])
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    q, k, v = _plain_parts(s, s["qkv"].float())
    done = []
    for part, gamma, beta in ((q, s["q_gamma"], s["q_beta"]), (k, s["k_gamma"], s["k_beta"])):
        y = _plain_normalised(case, part)[0] * gamma
        if beta is not None:
            y = y + beta
        done.append(_rotate(case, y, cos, sin))
    return torch.cat(done + [v], dim=2).to(s["qkv"].dtype)


def _plain_qk_norm_backward(s):
    case = s["case"]
    cos, sin = _angles(case, s["positions"], s["frequencies"])
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    parts = _plain_parts(s, s["qkv"].float())
    grads = _plain_parts(s, s["grad"].float())
    done, gammas, betas = [], [], []
    for part, grad, gamma in ((parts[0], grads[0], s["q_gamma"]), (parts[1], grads[1], s["k_gamma"])):
        x, scale = _plain_normalised(case, part)
        d = _rotate(case, grad, cos, -sin)
        gammas.append((d * x).sum(dim=(0, 1, 2), dtype=torch.float64).float())
        betas.append(d.sum(dim=(0, 1, 2), dtype=torch.float64).float())
        d = d * gamma
        dx = d - x * (d * x).mean(dim=-1, keepdim=True)
        if case["norm"] == "layer":
            dx = dx - d.mean(dim=-1, keepdim=True)
        done.append(dx * scale)
    grad_qkv = torch.cat(done + [grads[2]], dim=2).to(s["qkv"].dtype)
    return _gradients(case, grad_qkv, gammas[0], gammas[1], betas[0], betas[1])


_TANH_SCALE = math.sqrt(2.0 / math.pi)
_TANH_CUBE = 0.044715


def _plain_activation(kind, x):
    if kind == "silu":
        return x / (1.0 + torch.exp(-x))
    if kind == "gelu":
        return 0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5)))
    return 0.5 * x * (1.0 + torch.tanh(_TANH_SCALE * (x + _TANH_CUBE * x * x * x)))


def _plain_slope(kind, x):
    if kind == "silu":
        sigmoid = 1.0 / (1.0 + torch.exp(-x))
        return sigmoid * (1.0 + x * (1.0 - sigmoid))
    if kind == "gelu":
        return 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) / math.sqrt(2.0 * math.pi)
    t = torch.tanh(_TANH_SCALE * (x + _TANH_CUBE * x * x * x))
    return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * _TANH_SCALE * (1.0 + 3.0 * _TANH_CUBE * x * x)


def _plain_gated(s):
    case = s["case"]
    z = s["a"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"]
    out = (_plain_activation(case["activation"], z[:, :case["n"]]) * z[:, case["n"]:]).to(s["a"].dtype)
    return (out, z.to(s["a"].dtype)) if case["keep"] else out


def _plain_gated_backward(s):
    case = s["case"]
    z, grad = s["pre"].float(), s["grad"].float()
    gate, value = z[:, :case["n"]], z[:, case["n"]:]
    return torch.cat([grad * value * _plain_slope(case["activation"], gate),
                      grad * _plain_activation(case["activation"], gate)], dim=1).to(s["pre"].dtype)


_PLAIN = {"rotary": _plain_rotary, "qk_norm": _plain_qk_norm, "qk_norm_backward": _plain_qk_norm_backward,
          "gated": _plain_gated, "gated_backward": _plain_gated_backward}


# -- the definitions in 64 bits ---------------------------------------------------


def _turn(case, x, positions, frequencies, sign):
    """Every pair (x, y) of a token as the complex number x + i y, times
    exp(sign i angle); x is [images, tokens, heads, head_dim] in 64 bits."""
    counts = _pairs(case)
    table = positions.double()
    if table.dim() == 2:
        table = table[None]
    columns, at = [], 0
    for axis, count in enumerate(counts):
        columns.append(table[..., axis:axis + 1] * frequencies[at:at + count].double())
        at += count
    phase = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE), sign * torch.cat(columns, dim=-1))
    phase = phase[:, :, None, :]
    total = sum(counts)
    if case["pairing"] == "halves":
        number = torch.complex(x[..., :total].contiguous(), x[..., total:2 * total].contiguous()) * phase
        return torch.cat([number.real, number.imag, x[..., 2 * total:]], dim=-1)
    number = torch.complex(x[..., 0:2 * total:2].contiguous(), x[..., 1:2 * total:2].contiguous()) * phase
    return torch.cat([torch.view_as_real(number.contiguous()).reshape(*x.shape[:-1], 2 * total),
                      x[..., 2 * total:]], dim=-1)


def _define_qk_norm(case, qkv, weights, positions, frequencies):
    heads, kv_heads = case["heads"], case["kv_heads"]
    rows = qkv[:, :, :heads + kv_heads]
    gamma = torch.cat([weights["q_gamma"].expand(heads, -1), weights["k_gamma"].expand(kv_heads, -1)])
    mean = rows.mean(-1, keepdim=True) if case["norm"] == "layer" else 0.0
    spread = torch.sqrt(((rows - mean) ** 2).sum(-1, keepdim=True) / case["head_dim"] + EPSILON)
    y = (rows - mean) / spread * gamma
    if case["beta"]:
        y = y + torch.cat([weights["q_beta"].expand(heads, -1), weights["k_beta"].expand(kv_heads, -1)])
    return torch.cat([_turn(case, y, positions, frequencies, 1.0), qkv[:, :, heads + kv_heads:]], dim=2)


def _define_gated(kind, gate, value):
    if kind == "silu":
        return gate * torch.sigmoid(gate) * value
    if kind == "gelu":
        return gate * torch.special.ndtr(gate) * value
    inner = math.sqrt(8.0 / math.pi) * (gate + 0.044715 * gate ** 3)
    return gate * torch.sigmoid(inner) * value


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rotary":
        x = s["x"].double()
        x = x.transpose(1, 2) if case["heads_first"] else x
        y = _turn(case, x, s["positions"], s["frequencies"], -1.0 if case["inverse"] else 1.0)
        return (y.transpose(1, 2) if case["heads_first"] else y).contiguous()
    if op in ("qk_norm", "qk_norm_backward"):
        names = ["q_gamma", "k_gamma"] + (["q_beta", "k_beta"] if case["beta"] else [])
        weights = {name: s[name].double() for name in names}
        qkv = s["qkv"].double()
        if op == "qk_norm":
            return _define_qk_norm(case, qkv, weights, s["positions"], s["frequencies"])
        leaves = [qkv.requires_grad_()] + [weights[name].requires_grad_() for name in names]
        y = _define_qk_norm(case, qkv, weights, s["positions"], s["frequencies"])
        grads = torch.autograd.grad(y, leaves, s["grad"].double())
        return dict(zip(["qkv"] + names, grads))
    n = case["n"]
    if op == "gated":
        z = torch.nn.functional.linear(s["a"].double(), s["w"].double(),
                                       None if s["bias"] is None else s["bias"].double())
        out = _define_gated(case["activation"], z[:, :n], z[:, n:])
        return (out, z) if case["keep"] else out
    z = s["pre"].double().requires_grad_()
    out = _define_gated(case["activation"], z[:, :n], z[:, n:])
    return torch.autograd.grad(out, z, s["grad"].double())[0]
