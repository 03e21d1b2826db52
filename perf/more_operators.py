"""What the operators at the two ends of a training step's backward pass are measured on, each in a plain form of elementary torch operations and
through `lumen_b200.runtime`:

  loss    softmax cross entropy of a projection to a vocabulary, straight from the hidden states and the head's weights: each token's loss and
          log-sum-exp, and the gradients of hidden states and weights
  adamw   the AdamW step over all of a model's tensors, with float32 moments or with moments in 8 bits

Inputs are made on the GPU from the seed alone."""

import math
import random

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ITEM = {"float32": 4, "bfloat16": 2, "float16": 2}
IGNORED = -100
BETAS, EPS, DECAY, LR = (0.9, 0.999), 1e-8, 0.01, 1e-3
BLOCK = 256  # elements that share a scale where moments are held in 8 bits
MOST = 448.0  # the largest e4m3 value


def listed():
    return [
        # One token of four sequences, scored at the 12-layer model's width and vocabulary: what a call costs beside reading the head once.
        {"name": "loss_token_bf16", "op": "loss", "tokens": 4, "width": 1024, "vocab": 32768, "ignored": 0.0, "reduction": "none", "backward": False,
         "dtype": "bfloat16"},
        # A prompt's tokens against a wide model's vocabulary: the head is what there is to read.
        {"name": "loss_prompt_bf16", "op": "loss", "tokens": 61, "width": 4096, "vocab": 131072, "ignored": 0.0, "reduction": "none", "backward": False,
         "dtype": "bfloat16"},
        # Evaluation of a batch of texts whose lengths nobody rounded, a part of it padding, a vocabulary of an odd size.
        {"name": "loss_ragged_f16", "op": "loss", "tokens": 1531, "width": 1120, "vocab": 30011, "ignored": 0.3, "reduction": "mean", "backward": False,
         "dtype": "float16"},
        # A rank's eight sequences of 2048 tokens at the 12-layer model's head: the forward pass of its training step.
        {"name": "loss_train_bf16", "op": "loss", "tokens": 16384, "width": 1024, "vocab": 32768, "ignored": 0.0, "reduction": "mean", "backward": False,
         "dtype": "bfloat16"},
        # The 2-layer float32 model's head: launches.
        {"name": "loss_backward_small_f32", "op": "loss", "tokens": 256, "width": 128, "vocab": 256, "ignored": 0.0, "reduction": "mean", "backward": True,
         "dtype": "float32"},
        # The backward pass of a ragged batch with padding, a weight for each token.
        {"name": "loss_backward_ragged", "op": "loss", "tokens": 2600, "width": 840, "vocab": 10007, "ignored": 0.3, "reduction": "none", "backward": True,
         "dtype": "bfloat16"},
        # The backward pass of the rank's eight sequences.
        {"name": "loss_train_backward", "op": "loss", "tokens": 16384, "width": 1024, "vocab": 32768, "ignored": 0.0, "reduction": "mean", "backward": True,
         "dtype": "bfloat16"},
        # The step of the 2-layer float32 model: launches.
        {"name": "adamw_small_f32", "op": "adamw", "layers": 2, "width": 128, "hidden": 512, "vocab": 256, "seq": 64, "grads": "same", "bits": 32,
         "masters": False, "clipped": False, "packed": False, "step": 3, "dtype": "float32"},
        # The step of the benchmark's model at seven of its layers, gradients clipped on the way: memory bandwidth.
        {"name": "adamw_model_bf16", "op": "adamw", "layers": 7, "width": 1024, "hidden": 4096, "vocab": 32768, "seq": 2048, "grads": "same", "bits": 32,
         "masters": False, "clipped": True, "packed": False, "step": 1000, "dtype": "bfloat16"},
        # The same step with both moments in 8 bits.
        {"name": "adamw_model_8bit", "op": "adamw", "layers": 7, "width": 1024, "hidden": 4096, "vocab": 32768, "seq": 2048, "grads": "same", "bits": 8,
         "masters": False, "clipped": True, "packed": False, "step": 1000, "dtype": "bfloat16"},
        # Tensors of all types and of sizes that nothing divides, views of one arena, float32 gradients and float32 copies of the 16-bit weights.
        {"name": "adamw_mixed_masters", "op": "adamw", "tensors": 41, "elements": 30000000, "spread": 7, "grads": "float32", "bits": 32, "masters": True,
         "clipped": False, "packed": True, "step": 17, "dtype": "mixed"},
    ]


def _size(rng, low, high, multiple=1):
    n = int(math.exp(rng.uniform(math.log(low), math.log(high))))
    return max(low, n // multiple * multiple)


def draw(rng):
    if rng.random() < 0.6:
        backward, dtype = rng.random() < 0.5, rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        width, vocab = _size(rng, 64, 4096, 8), _size(rng, 200, 131072)
        tokens = rng.randint(1, 32) if rng.random() < 0.3 else _size(rng, 33, 16384)
        most = 16384 * 1024 * 32768 // (32 if dtype == "float32" else 1)  # float32 products run on other cores
        while tokens * width * vocab > most or tokens * vocab > 16384 * 32768:
            tokens, vocab = max(1, tokens * 2 // 3), max(200, vocab * 3 // 4)
        return {"op": "loss", "tokens": tokens, "width": width, "vocab": vocab, "ignored": rng.choice([0.0, 0.0, 0.1, 0.5]),
                "reduction": rng.choice(["mean", "sum", "none"]), "backward": backward, "dtype": dtype}  # fmt: skip
    bits, dtype = rng.choice([32, 8]), rng.choice(["float32", "bfloat16", "float16", "mixed"])
    return {"op": "adamw", "tensors": rng.randint(1, 60), "elements": _size(rng, 1000, 60000000), "spread": rng.randrange(1 << 20),
            "grads": rng.choice(["same", "same", "float32"]), "bits": bits, "masters": rng.random() < 0.3, "clipped": rng.random() < 0.5,
            "packed": bits == 32 and rng.random() < 0.5, "step": _size(rng, 1, 100000), "dtype": dtype}  # fmt: skip


def _sizes(case):
    """The element counts and types of a model's tensors."""
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
    if case["op"] == "loss":
        t, d, v, kind = case["tokens"], case["width"], case["vocab"], case["dtype"]
        s["w"] = _normal(g, (v, d), kind, 1.5 * d**-0.5)
        s["targets"] = torch.randint(0, v, (t,), generator=g, device="cuda")
        # hidden states of a model that has learnt something: each leans towards its target
        lean = 2.0 * torch.rand((t, 1), generator=g, device="cuda")
        s["x"] = (torch.randn((t, d), generator=g, device="cuda") + lean * s["w"][s["targets"]].float()).to(TYPES[kind])
        s["targets"][1:][torch.rand(t, generator=g, device="cuda")[1:] < case["ignored"]] = IGNORED  # the first one counts
        if case["backward"]:
            logits = s["x"].float() @ s["w"].float().t()
            s["lse"] = torch.logsumexp(logits, -1)  # what the forward pass has left
            scale = 4096.0 if kind == "float16" and case["reduction"] == "mean" else 1.0
            s["d_loss"] = 0.5 + torch.rand(t, generator=g, device="cuda") if case["reduction"] == "none" else torch.full((), scale, device="cuda")
        return s
    sizes, buffers = _sizes(case), {}
    spans, ends = [], {}
    for n, kind in sizes:  # where each tensor lies in its type's arena: one behind the other, or at the start of a block
        at = ends.get(kind, 0)
        spans.append((kind, at, n))
        ends[kind] = at + n if case["packed"] else (at + n + BLOCK - 1) // BLOCK * BLOCK
    scale = random.Random(seed)
    masters = case["masters"]
    for kind, end in ends.items():
        grad = "float32" if case["grads"] == "float32" else kind
        buffers[kind] = {"grads": torch.zeros(end, dtype=TYPES[grad], device="cuda"), "weights": torch.zeros(end, device="cuda"),
                         "exp_avg": torch.zeros(end, device="cuda"), "exp_avg_sq": torch.zeros(end, device="cuda")}  # fmt: skip
    for kind, at, n in spans:
        b, size = buffers[kind], 10.0 ** scale.uniform(-4.0, -2.0)
        rms = size * torch.exp(torch.randn(n, generator=g, device="cuda"))  # what the gradients of each element have been like
        b["grads"][at : at + n] = (rms * torch.randn(n, generator=g, device="cuda")).to(b["grads"].dtype)
        b["exp_avg"][at : at + n] = 0.3 * rms * torch.randn(n, generator=g, device="cuda")
        b["exp_avg_sq"][at : at + n] = rms.square() * (0.2 + torch.rand(n, generator=g, device="cuda")) * (1.0 - BETAS[1] ** (case["step"]))
        b["weights"][at : at + n] = 0.05 * torch.randn(n, generator=g, device="cuda")
    for kind, b in buffers.items():
        weights = b.pop("weights")
        b["params"] = weights.to(TYPES[kind])
        if masters:
            b["masters"] = weights if kind != "float32" else None
        if case["bits"] == 8:
            b["exp_avg"], b["exp_avg_scale"] = _to_bits(b["exp_avg"])
            b["exp_avg_sq"], b["exp_avg_sq_scale"] = _to_bits(torch.sqrt(b["exp_avg_sq"]), lowest=True)
    total = math.sqrt(sum(float(b["grads"].double().square().sum()) for b in buffers.values()))
    s["norm"] = torch.full((), total, device="cuda")
    s["max_norm"] = 0.37 * total
    s["buffers"] = buffers

    def views(name):
        if name not in next(iter(buffers.values())):
            return None
        if name.endswith("_scale"):
            return [buffers[kind][name][at // BLOCK : (at + n + BLOCK - 1) // BLOCK] for kind, at, n in spans]
        return [None if buffers[kind][name] is None else buffers[kind][name][at : at + n] for kind, at, n in spans]

    s["lists"] = {name: views(name) for name in ("params", "grads", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "masters")}
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _to_bits(x, lowest=False):
    """e4m3 codes (a byte each) and the scale of each block of `x`, whose largest value becomes the largest that e4m3 has. `lowest`: what is not zero
    does not become zero."""
    x = x.view(-1, BLOCK)
    most = x.abs().amax(-1, keepdim=True)
    q = x * torch.where(most < 2.0**-100, 0.0, MOST / most)
    q = q.to(torch.float8_e4m3fn).float()
    if lowest:
        q = torch.where((q == 0) & (x > 0), 2.0**-9, q)
    scale = torch.where(most < 2.0**-100, 0.0, most / MOST)
    return q.to(torch.float8_e4m3fn).view(torch.uint8).view(-1), scale.view(-1)


def _of_bits(codes, scale):
    return (codes.view(torch.float8_e4m3fn).float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _token_grads(s):
    """The gradient of each token's loss; what does not count has none."""
    counts = s["targets"] != IGNORED
    g = s["d_loss"] * counts
    return g / counts.sum().clamp(min=1) if s["reduction"] == "mean" else g


def _loss(s):
    logits = s["x"].float() @ s["w"].float().t()
    if not s["backward"]:
        most = logits.amax(-1, keepdim=True)
        lse = most.squeeze(-1) + torch.log(torch.exp(logits - most).sum(-1))
        counts = s["targets"] != IGNORED
        at = torch.where(counts, s["targets"], 0)
        losses = torch.where(counts, lse - logits.gather(-1, at[:, None]).squeeze(-1), 0.0)
        if s["reduction"] == "none":
            return {"loss": losses, "lse": lse}
        total = losses.double().sum()
        return {"loss": (total / counts.sum().clamp(min=1) if s["reduction"] == "mean" else total).float(), "lse": lse}
    d = torch.exp(logits - s["lse"][:, None])
    at = torch.where(s["targets"] == IGNORED, 0, s["targets"])
    d[torch.arange(len(at), device="cuda"), at] -= 1.0
    d *= _token_grads(s)[:, None]
    t = s["x"].dtype
    return {"d_x": (d @ s["w"].float()).to(t), "d_w": (d.t() @ s["x"].float()).to(t)}


def _adamw(s):
    b1, b2 = BETAS
    c1, c2 = 1.0 / (1.0 - b1 ** s["step"]), 1.0 / (1.0 - b2 ** s["step"])
    out = {}
    for kind, b in s["buffers"].items():
        g = b["grads"].float()
        if s["clipped"]:
            g = g * torch.clamp(s["max_norm"] / (s["norm"] + 1e-6), max=1.0)
        if s["bits"] == 8:
            m, v = _of_bits(b["exp_avg"], b["exp_avg_scale"]), _of_bits(b["exp_avg_sq"], b["exp_avg_sq_scale"]).square()
        else:
            m, v = b["exp_avg"], b["exp_avg_sq"]
        m = m * b1 + g * (1.0 - b1)
        v = v * b2 + g * g * (1.0 - b2)
        master = b.get("masters")
        w = b["params"].float() if master is None else master
        w = w * (1.0 - LR * DECAY) - m * c1 * LR / (torch.sqrt(v * c2) + EPS)
        b["params"].copy_(w.to(b["params"].dtype))
        if master is not None:
            master.copy_(w)
        if s["bits"] == 8:
            for name, x in (("exp_avg", m), ("exp_avg_sq", torch.sqrt(v))):
                codes, scale = _to_bits(x, lowest=name == "exp_avg_sq")
                b[name].copy_(codes), b[name + "_scale"].copy_(scale)
        else:
            b["exp_avg"].copy_(m), b["exp_avg_sq"].copy_(v)
        out[kind] = _updated(s, b)
    return out


def _updated(s, b):
    """What a step leaves of a type's tensors; moments of 8 bits as the e4m3 values that they are, beside their blocks' scales."""
    out = {name: b[name] for name in ("params", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "masters") if b.get(name) is not None}
    if s["bits"] == 8:
        for name in ("exp_avg", "exp_avg_sq"):
            out[name] = b[name].view(torch.float8_e4m3fn)
    return out


# ---- the framework's calls -----------------------------------------------------------------------------------------


def _run_own(s):
    from lumen_b200 import runtime

    if s["op"] == "loss":
        if not s["backward"]:
            loss, lse = runtime.linear_cross_entropy(s["x"], s["w"], s["targets"], reduction=s["reduction"], ignore_index=IGNORED)
            return {"loss": loss, "lse": lse}
        d_x, d_w = runtime.linear_cross_entropy_backward(s["d_loss"], s["x"], s["w"], s["targets"], s["lse"], reduction=s["reduction"], ignore_index=IGNORED)
        return {"d_x": d_x, "d_w": d_w}
    lists = s["lists"]
    clip = {"norm": s["norm"], "max_norm": s["max_norm"]} if s["clipped"] else {}
    runtime.adamw_step(lists["params"], lists["grads"], lists["exp_avg"], lists["exp_avg_sq"], s["step"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY,
                       exp_avg_scale=lists["exp_avg_scale"], exp_avg_sq_scale=lists["exp_avg_sq_scale"], masters=lists["masters"], **clip)  # fmt: skip
    return {kind: _updated(s, b) for kind, b in s["buffers"].items()}


def run(state):
    if own:
        return _run_own(state)
    return _loss(state) if state["op"] == "loss" else _adamw(state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def _nearest_e4m3(x):
    """The nearest e4m3 values to float64 `x` (ties to even): three bits behind the leading one, multiples of 2^-9 below 2^-6."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 4).clamp(min=-9).double())
    return (torch.round(x / step) * step).clamp(-MOST, MOST)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "loss":
        x, w, targets = s["x"].double(), s["w"].double(), s["targets"]
        counts = (targets != IGNORED).double()
        if not case["backward"]:
            lse, hit = [], []
            for rows, at in zip(x.split(2048), targets.clamp(min=0).split(2048)):  # some rows of 64-bit logits at a time
                z = torch.matmul(rows, w.T)
                lse.append(torch.logsumexp(z, 1)), hit.append((rows * w[at]).sum(1))
            lse, losses = torch.cat(lse), (torch.cat(lse) - torch.cat(hit)) * counts
            loss = {"none": lambda: losses, "sum": lambda: losses.sum(), "mean": lambda: losses.sum() / max(1.0, float(counts.sum()))}
            return {"loss": loss[case["reduction"]](), "lse": lse}
        share = counts * s["d_loss"].double()
        if case["reduction"] == "mean":
            share = share / max(1.0, float(counts.sum()))
        d_x, d_w = torch.empty_like(x), torch.zeros_like(w)
        for i in range(0, len(x), 2048):
            rows = slice(i, i + 2048)
            p = torch.softmax(torch.cat((torch.matmul(x[rows], w.T),), 1), 1)
            p *= torch.exp(torch.logsumexp(torch.matmul(x[rows], w.T), 1) - s["lse"][rows].double())[:, None]  # by the log-sum-exp that was given
            p -= torch.nn.functional.one_hot(targets[rows].clamp(min=0), case["vocab"])
            p *= share[rows, None]
            d_x[rows] = torch.matmul(p, w)
            d_w += torch.matmul(p.T, x[rows])
        return {"d_x": d_x, "d_w": d_w}
    b1, b2, t, out = *BETAS, case["step"], {}
    factor = min(1.0, s["max_norm"] / (float(s["norm"]) + 1e-6)) if case["clipped"] else 1.0
    for kind, b in s["buffers"].items():
        g = b["grads"].double() * factor
        if case["bits"] == 8:
            m, r = ((b[n].view(torch.float8_e4m3fn).double().unflatten(0, (-1, BLOCK)) * b[n + "_scale"].double().unsqueeze(1)).flatten() for n in ("exp_avg", "exp_avg_sq"))
            v = r * r
        else:
            m, v = b["exp_avg"].double(), b["exp_avg_sq"].double()
        m, v = torch.lerp(g, m, b1), torch.lerp(g.pow(2), v, b2)
        start = b["masters"] if b.get("masters") is not None else b["params"]
        bias = math.sqrt(-math.expm1(t * math.log(b2))) / -math.expm1(t * math.log(b1))
        moved = start.double() * (1.0 - LR * DECAY) - LR * bias * m / (v.sqrt() + EPS * math.sqrt(-math.expm1(t * math.log(b2))))
        out[kind] = {"params": moved}
        if b.get("masters") is not None:
            out[kind]["masters"] = moved
        if case["bits"] == 32:
            out[kind] |= {"exp_avg": m, "exp_avg_sq": v}
            continue
        for name, held in (("exp_avg", m), ("exp_avg_sq", v.sqrt())):
            blocks = held.unflatten(0, (-1, BLOCK))
            top = blocks.abs().max(1).values
            unit = torch.where(top < 2.0**-100, 1.0, top / MOST).unsqueeze(1)
            value = _nearest_e4m3(blocks / unit)
            if name == "exp_avg_sq":
                value = torch.where(blocks > 0, value.clamp(min=2.0**-9), value)
            out[kind] |= {name: value.flatten(), name + "_scale": top / MOST}
    return out


def work(case):
    if case["op"] == "loss":
        item, t, d, v = ITEM[case["dtype"]], case["tokens"], case["width"], case["vocab"]
        if not case["backward"]:
            return {"bytes": item * (t + v) * d + t * (8 + 4) + (t if case["reduction"] == "none" else 1) * 4, "flops": 2.0 * t * d * v}
        return {"bytes": 2 * item * (t + v) * d + t * (8 + 4) + (t if case["reduction"] == "none" else 1) * 4, "flops": 6.0 * t * d * v}
    total = elements = 0
    for n, kind in _sizes(case):
        moments = 16 * n if case["bits"] == 32 else 4 * n + 16 * ((n + BLOCK - 1) // BLOCK)
        weights = 2 * ITEM[kind] * n
        if case["masters"] and kind != "float32":
            weights = (8 + ITEM[kind]) * n  # the copies are read and written, the weights themselves written alone
        total += moments + weights + (4 if case["grads"] == "float32" else ITEM[kind]) * n
        elements += n
    return {"bytes": total, "flops": 16 * elements}
