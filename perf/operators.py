"""What the operators of a decoder layer's training step are measured on, each in a plain form of elementary torch operations and through
`lumen_b200.runtime`:

  rotate  norms of queries and keys for each head with the position rotation, in one pass; forward and backward
  gated   the gated feed-forward block: both projections, the activation and the product, the projection back; forward and backward
  clip    the global norm over a step's gradients, and clipping by it

Inputs are made on the GPU from the seed alone."""

import math
import random

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ITEM = {"float32": 4, "bfloat16": 2, "float16": 2}
EPS = 1e-6


def listed():
    return [
        # One new token of four sequences far into a cache (16 heads x 64): what a call costs.
        {"name": "rotate_token_bf16", "op": "rotate", "batch": 4, "seq": 1, "heads": 16, "kv_heads": 16, "dim": 64, "rotary": 64,
         "interleaved": False, "table": 131072, "weights": True, "backward": False, "dtype": "bfloat16"},
        # Prefill of two prompts of a length nobody rounded, four query heads to a key head, views of a packed projection.
        {"name": "rotate_prefill_f16", "op": "rotate", "batch": 2, "seq": 1531, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "table": 4096, "weights": True, "backward": False, "dtype": "float16"},
        # The backward pass at the benchmark's attention shape, grouped heads: memory bandwidth.
        {"name": "rotate_train_bf16", "op": "rotate", "batch": 8, "seq": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "table": 4096, "weights": True, "backward": True, "dtype": "bfloat16"},
        # A float32 model with a head dim off the powers of two, a rotation of part of it and neighbouring pairs; backward.
        {"name": "rotate_partial_f32", "op": "rotate", "batch": 3, "seq": 1021, "heads": 10, "kv_heads": 5, "dim": 80, "rotary": 32,
         "interleaved": True, "table": 2048, "weights": True, "backward": True, "dtype": "float32"},
        # Decode of four sequences at the 12-layer model's width: the weights are read once.
        {"name": "gated_token_bf16", "op": "gated", "tokens": 4, "width": 1024, "hidden": 4096, "activation": "silu", "backward": False,
         "dtype": "bfloat16"},
        # A short ragged batch at sizes that are no multiples of a tile.
        {"name": "gated_ragged_f16", "op": "gated", "tokens": 1531, "width": 1120, "hidden": 2808, "activation": "silu", "backward": False,
         "dtype": "float16"},
        # A rank's eight sequences of 2048 tokens at the 12-layer model's width, forward with what the backward pass needs kept.
        {"name": "gated_train_bf16", "op": "gated", "tokens": 16384, "width": 1024, "hidden": 4096, "activation": "silu", "backward": False,
         "dtype": "bfloat16"},
        # The backward pass of a ragged batch, gelu.
        {"name": "gated_backward_ragged", "op": "gated", "tokens": 2600, "width": 840, "hidden": 2056, "activation": "gelu", "backward": True,
         "dtype": "bfloat16"},
        # The backward pass of the rank's eight sequences.
        {"name": "gated_train_backward", "op": "gated", "tokens": 16384, "width": 1024, "hidden": 4096, "activation": "silu", "backward": True,
         "dtype": "bfloat16"},
        # The gradients of the 2-layer float32 model, clipped: launches.
        {"name": "clip_small_f32", "op": "clip", "layers": 2, "width": 128, "hidden": 512, "vocab": 256, "seq": 64, "clipped": True,
         "in_place": False, "dtype": "float32"},
        # The gradients of the benchmark's model at seven of its layers, clipped: memory bandwidth.
        {"name": "clip_model_bf16", "op": "clip", "layers": 7, "width": 1024, "hidden": 4096, "vocab": 32768, "seq": 2048, "clipped": True,
         "in_place": False, "dtype": "bfloat16"},
        # Tensors of all types and of sizes that nothing divides, in place, under the bound: the usual step, whose gradients stay as they are.
        {"name": "clip_mixed_in_place", "op": "clip", "tensors": 41, "elements": 60000000, "spread": 7, "clipped": False, "in_place": True,
         "dtype": "mixed"},
    ]


def _size(rng, low, high, multiple=1):
    n = int(math.exp(rng.uniform(math.log(low), math.log(high))))
    return max(low, n // multiple * multiple)


def draw(rng):
    op = rng.choice(["rotate", "rotate", "gated", "gated", "clip"])
    if op == "rotate":
        dim, kv_heads, group = rng.choice([48, 64, 80, 96, 128, 256]), rng.randint(1, 16), rng.choice([1, 1, 2, 4, 5, 8])
        if rng.random() < 0.3:  # serving: one token or a few of some sequences
            batch, seq = _size(rng, 1, 256), rng.choice([1, 1, 2, 5])
        else:
            batch, seq = rng.randint(1, 8), _size(rng, 3, 8192)
        most = 8 * 4096 * 40 * 128 // 2  # half of the largest listed one's elements: float32 has twice the bytes
        while batch * seq * kv_heads * (group + 1) * dim > most:
            seq, batch = max(1, seq * 2 // 3), max(1, batch * 3 // 4)
        return {"op": "rotate", "batch": batch, "seq": seq, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
                "rotary": rng.choice([dim, dim, dim // 2 // 16 * 16]), "interleaved": rng.random() < 0.3, "table": seq + _size(rng, 1, 100000),
                "weights": rng.random() < 0.8, "backward": rng.random() < 0.5, "dtype": rng.choice(["float32", "bfloat16", "bfloat16", "float16"])}  # fmt: skip
    if op == "gated":
        width, hidden, backward = _size(rng, 128, 4096, 8), _size(rng, 256, 16384, 8), rng.random() < 0.5
        tokens = rng.randint(1, 32) if not backward and rng.random() < 0.3 else _size(rng, 16, 32768)
        while tokens * width * hidden > 16384 * 1024 * 4096 or tokens * hidden > 16384 * 4096:
            tokens = max(1, tokens * 2 // 3)
        return {"op": "gated", "tokens": tokens, "width": width, "hidden": hidden, "activation": rng.choice(["silu", "gelu", "relu"]),
                "backward": backward, "dtype": rng.choice(["bfloat16", "float16"])}  # fmt: skip
    return {"op": "clip", "tensors": rng.randint(1, 60), "elements": _size(rng, 1000, 60000000), "spread": rng.randrange(1 << 20),
            "clipped": rng.random() < 0.6, "in_place": False, "dtype": rng.choice(["float32", "bfloat16", "float16", "mixed"])}  # fmt: skip


def _sizes(case):
    """The element counts and types of a step's gradients."""
    if "layers" in case:
        d, f = case["width"], case["hidden"]
        layer = [d, d, 3 * d * d, d * d, d, d, f * d, d * f]
        counts = [case["vocab"] * d, case["seq"] * d] + layer * case["layers"] + [d, d, case["vocab"] * d]
    else:
        r = random.Random(case["spread"])
        shares = [math.exp(r.uniform(0.0, 9.0)) for _ in range(case["tensors"])]
        counts = [max(1, int(case["elements"] * s / sum(shares))) for s in shares]
    kinds = ["bfloat16", "float32", "float16"] if case["dtype"] == "mixed" else [case["dtype"]]
    return [(n, kinds[k % len(kinds)]) for k, n in enumerate(counts)]


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(TYPES.get(dtype, dtype))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] == "rotate":
        b, n, nq, nk, h, t = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["dim"], case["dtype"]
        packed = _normal(g, (b, n, nq + 2 * nk, h), t, 1.5)  # the projection that q, k and v are views of
        s["q"], s["k"] = packed[:, :, :nq], packed[:, :, nq : nq + nk]
        half = case["rotary"] // 2
        rate = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / max(half, 1))
        angle = torch.arange(case["table"], device="cuda", dtype=torch.float64)[:, None] * rate
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        # where each sequence's tokens stand: behind what it has had before
        start = torch.randint(0, case["table"] - n + 1, (b, 1), generator=g, device="cuda")
        s["positions"] = start + torch.arange(n, device="cuda")
        s["wq"], s["wk"] = ((1.0 + 0.2 * torch.randn(h, generator=g, device="cuda")).to(TYPES[t]) if case["weights"] else None for _ in "qk")
        if case["backward"]:
            s["dq"], s["dk"] = _normal(g, (b, n, nq, h), t, 0.1), _normal(g, (b, n, nk, h), t, 0.1)
    elif case["op"] == "gated":
        m, d, f, t = case["tokens"], case["width"], case["hidden"], case["dtype"]
        s["x"] = _normal(g, (m, d), t)
        s["wgu"], s["wd"] = _normal(g, (2 * f, d), t, d**-0.5), _normal(g, (d, f), t, f**-0.5)
        if case["backward"]:  # what the forward pass has left
            gate_up = s["x"].float() @ s["wgu"].float().t()
            s["gate_up"] = gate_up.to(TYPES[t])
            s["h"] = (_act(gate_up[:, :f], case["activation"])[0] * gate_up[:, f:]).to(TYPES[t])
            s["dy"] = _normal(g, (m, d), t, 0.1)
    else:
        scale = random.Random(seed)
        s["grads"] = [_normal(g, (n,), t, 10.0 ** scale.uniform(-3.0, -1.0)) for n, t in _sizes(case)]
        total = math.sqrt(sum(float(x.double().square().sum()) for x in s["grads"]))
        s["max_norm"] = total * (0.37 if case["clipped"] else 2.0)
        s["out"] = s["grads"] if case["in_place"] else [torch.empty_like(x) for x in s["grads"]]
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _act(a, kind):
    """The activation and its derivative, float32."""
    if kind == "relu":
        on = (a > 0).float()
        return a * on, on
    if kind == "silu":
        p = 1.0 / (1.0 + torch.exp(-a))
        return a * p, p * (1.0 + a * (1.0 - p))
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (a + 0.044715 * a * a * a))
    return 0.5 * a * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * a * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * a * a)


def _halves(x, rotary, interleaved):
    """The two members of each pair, and the elements that are not rotated."""
    r = x[..., :rotary]
    pair = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., : rotary // 2], r[..., rotary // 2 :])
    return (*pair, x[..., rotary:])


def _joined(a, b, rest, interleaved):
    r = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((r, rest), -1)


def _rotate(s, x, w):
    x = x.float()
    z = x * torch.rsqrt(torch.mean(x * x, -1, keepdim=True) + EPS)
    if w is not None:
        z = z * w.float()
    a, b, rest = _halves(z, s["rotary"], s["interleaved"])
    c, n = s["cos"][s["positions"]].unsqueeze(2), s["sin"][s["positions"]].unsqueeze(2)
    return _joined(a * c - b * n, b * c + a * n, rest, s["interleaved"])


def _rotate_backward(s, x, w, dy):
    x, dy = x.float(), dy.float()
    r = torch.rsqrt(torch.mean(x * x, -1, keepdim=True) + EPS)
    a, b, rest = _halves(dy, s["rotary"], s["interleaved"])
    c, n = s["cos"][s["positions"]].unsqueeze(2), s["sin"][s["positions"]].unsqueeze(2)
    dz = _joined(a * c + b * n, b * c - a * n, rest, s["interleaved"])
    unit = x * r
    dw = None if w is None else (dz * unit).sum((0, 1, 2)).to(w.dtype)
    du = dz if w is None else dz * w.float()
    return r * (du - unit * torch.mean(du * unit, -1, keepdim=True)), dw


def _run_plain(s):
    if s["op"] == "rotate":
        t = s["q"].dtype
        if not s["backward"]:
            return {"q": _rotate(s, s["q"], s["wq"]).to(t), "k": _rotate(s, s["k"], s["wk"]).to(t)}
        (dq, dwq), (dk, dwk) = _rotate_backward(s, s["q"], s["wq"], s["dq"]), _rotate_backward(s, s["k"], s["wk"], s["dk"])
        return {"dq": dq.to(t), "dk": dk.to(t), "dwq": dwq, "dwk": dwk}
    if s["op"] == "gated":
        t, f, kind = s["x"].dtype, s["hidden"], s["activation"]
        x, wgu, wd = s["x"].float(), s["wgu"].float(), s["wd"].float()
        if not s["backward"]:
            gate_up = x @ wgu.t()
            h = _act(gate_up[:, :f], kind)[0] * gate_up[:, f:]
            return {"y": (h @ wd.t()).to(t), "gate_up": gate_up.to(t), "h": h.to(t)}
        gate_up, dy = s["gate_up"].float(), s["dy"].float()
        value, slope = _act(gate_up[:, :f], kind)
        dh = dy @ wd
        d_gate_up = torch.cat((dh * gate_up[:, f:] * slope, dh * value), -1)
        return {"dx": (d_gate_up @ wgu).to(t), "dwgu": (d_gate_up.t() @ x).to(t), "dwd": (dy.t() @ s["h"].float()).to(t)}
    norm = torch.sqrt(sum(x.float().square().sum() for x in s["grads"]))
    factor = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    clipped = [o.copy_((x.float() * factor).to(x.dtype)) for o, x in zip(s["out"], s["grads"])]
    return {"norm": norm, "grads": clipped}


# ---- the framework's calls -----------------------------------------------------------------------------------------


def _run_own(s):
    from lumen_b200 import runtime

    if s["op"] == "rotate":
        common = {"positions": s["positions"], "q_weight": s["wq"], "k_weight": s["wk"], "eps": EPS, "interleaved": s["interleaved"]}
        if not s["backward"]:
            q, k = runtime.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], **common)
            return {"q": q, "k": k}
        dq, dk, dwq, dwk = runtime.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["cos"], s["sin"], **common)
        return {"dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    if s["op"] == "gated":
        if not s["backward"]:
            y, gate_up, h = runtime.gated_mlp_forward(s["x"], s["wgu"], s["wd"], activation=s["activation"])
            return {"y": y, "gate_up": gate_up, "h": h}
        dx, dwgu, dwd = runtime.gated_mlp_backward(s["dy"], s["x"], s["wgu"], s["wd"], s["gate_up"], s["h"], activation=s["activation"])
        return {"dx": dx, "dwgu": dwgu, "dwd": dwd}
    norm = runtime.clip_grad_norm(s["grads"], s["max_norm"], out=None if s["in_place"] else s["out"])
    return {"norm": norm, "grads": s["out"]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        phase = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]][:, :, None]
        half = case["rotary"] // 2

        def turned(x, w):
            z = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
            z = z if w is None else z * w
            head, rest = z[..., : 2 * half], z[..., 2 * half :]
            pairs = head.unflatten(-1, (half, 2)) if case["interleaved"] else head.unflatten(-1, (2, half)).transpose(-1, -2)
            pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * phase)
            pairs = pairs if case["interleaved"] else pairs.transpose(-1, -2)
            return torch.cat((pairs.flatten(-2), rest), -1)

        out = {}
        for name in "qk":
            x, w = s[name].double(), s["w" + name]
            w = None if w is None else w.double()
            if not case["backward"]:
                out[name] = turned(x, w)
                continue
            x.requires_grad_()
            leaves = (x,) if w is None else (x, w.requires_grad_())
            got = torch.autograd.grad(turned(*leaves) if w is not None else turned(x, None), leaves, s["d" + name].double())
            out["d" + name], out["dw" + name] = got[0], got[1] if w is not None else None
        return out
    if case["op"] == "gated":
        f = case["hidden"]

        def unit(pre):
            a, b = pre.split(f, -1)
            if case["activation"] == "silu":
                return a.sigmoid() * a * b
            if case["activation"] == "relu":
                return torch.where(a > 0, a, 0.0) * b
            return a * torch.sigmoid(math.sqrt(8.0 / math.pi) * (a + 0.044715 * a.pow(3))) * b

        x, wgu, wd = s["x"].double(), s["wgu"].double(), s["wd"].double()
        if not case["backward"]:
            pre = torch.matmul(x, wgu.T)
            h = unit(pre)
            return {"y": torch.matmul(h, wd.T), "gate_up": pre, "h": h}
        pre, dy = s["gate_up"].double().requires_grad_(), s["dy"].double()
        (d_pre,) = torch.autograd.grad(unit(pre), pre, torch.matmul(dy, wd))
        return {"dx": torch.matmul(d_pre, wgu), "dwgu": torch.matmul(d_pre.T, x), "dwd": torch.matmul(dy.T, s["h"].double())}
    norm = torch.stack([torch.linalg.vector_norm(x.double()) for x in s["grads"]])
    norm = torch.linalg.vector_norm(norm)
    factor = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    return {"norm": norm, "grads": [x.double() * factor for x in s["grads"]]}


def work(case):
    if case["op"] == "rotate":
        item, tokens, h = ITEM[case["dtype"]], case["batch"] * case["seq"], case["dim"]
        values = tokens * (case["heads"] + case["kv_heads"]) * h
        tables = min(tokens, case["table"]) * case["rotary"] * 4 + tokens * 8
        weights = (4 if case["backward"] else 2) * h * item * case["weights"]
        return {"bytes": values * item * (3 if case["backward"] else 2) + tables + weights, "flops": values * (20 if case["backward"] else 8)}
    if case["op"] == "gated":
        item, m, d, f = ITEM[case["dtype"]], case["tokens"], case["width"], case["hidden"]
        if not case["backward"]:
            return {"bytes": item * (2 * m * d + 3 * d * f + 3 * m * f), "flops": 6.0 * m * d * f}
        return {"bytes": item * (3 * m * d + 6 * d * f + 3 * m * f), "flops": 12.0 * m * d * f}
    sizes = _sizes(case)
    held = sum(n * ITEM[t] for n, t in sizes)
    return {"bytes": held + 4 + (held if case["clipped"] or not case["in_place"] else 0), "flops": 3 * sum(n for n, _ in sizes)}
