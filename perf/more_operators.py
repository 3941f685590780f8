"""Cases of the dense blocks that stand beside the routed experts (shared experts, dense layers), and of the int8 recipe.

* ``linear``: the matrix product in 8-bit integers with a scale for each token and for each output channel, from 16-bit
  rows that are quantised on the way (``torch.ops._xpu_C.b200_int8_linear``).
* ``layer``: a Mixture-of-Experts layer whose weights and activations are multiplied as 8-bit integers
  (``XpuFusedMoe`` with int8 weights).
* ``gated``: both projections of a gated feed-forward block, its activation and the product
  (``torch.ops._xpu_C.b200_gated_linear``), as a serving step calls it.
* ``gated_grad``: the same in a training step: forward and the gradients of the rows and of the weights
  (``vllm_xpu_kernels.gated_linear``).

Shapes are the ones of ``perf/cases.py``.  Inputs are seeded synthetic draws: rows ~N(0,1), weights ~N(0, 1/fan_in),
gradients ~N(0,1), routing by random scores.
"""
import math
import os
import sys

import torch

own = False

# layers of the int8 recipe: hidden size, intermediate size, experts, experts a token
LAYERS = {
    "small": dict(hidden=2048, inter=1408, experts=8, topk=2),
    "mixtral": dict(hidden=4096, inter=14336, experts=8, topk=2),
    "qwen3": dict(hidden=2048, inter=768, experts=128, topk=8),
}
LEAST = 1e-10       # least largest value of a row that is quantised


def _linear(tokens, n, k, dtype="bfloat16", bias=False):
    return dict(op="linear", tokens=tokens, n=n, k=k, dtype=dtype, bias=bias)


def _layer(family, tokens, dtype="bfloat16", **other):
    return dict(dict(op="layer", tokens=tokens, dtype=dtype, **LAYERS[family]), **other)


def _gated(op, tokens, hidden, inter, dtype="bfloat16"):
    return dict(op=op, tokens=tokens, hidden=hidden, inter=inter, dtype=dtype)


def listed():
    return [
        # one decoded token through a projection: latency and the weights' bytes
        dict(_linear(1, 4096, 4096), name="linear_bf16_t1"),
        # a few users, with a bias
        dict(_linear(13, 2880, 2880, "float16", True), name="linear_fp16_t13_bias"),
        # a chunk of a prompt, odd in every size that may be
        dict(_linear(1001, 2011, 2032), name="linear_bf16_t1001_odd"),
        # the largest prefill batch through a shared expert's first product
        dict(_linear(8192, 4096, 7168), name="linear_bf16_t8192"),
        # one decoded token: eight small experts and the latency of a layer
        dict(_layer("qwen3", 1), name="layer_qwen3_t1"),
        # a decode batch on large experts
        dict(_layer("mixtral", 61, "float16"), name="layer_mixtral_fp16_t61"),
        # a prompt over many small experts
        dict(_layer("qwen3", 2048), name="layer_qwen3_t2048"),
        # one decoded token through a shared expert
        dict(_gated("gated", 1, 7168, 2048), name="gated_bf16_t1"),
        # the largest prefill batch through it
        dict(_gated("gated", 8192, 7168, 2048), name="gated_bf16_t8192"),
        # the smallest training step: latency
        dict(_gated("gated_grad", 48, 512, 256), name="gated_grad_bf16_t48"),
        # a ragged batch of a small layer, fp16
        dict(_gated("gated_grad", 1001, 2048, 1408, "float16"), name="gated_grad_fp16_t1001"),
        # a long batch through a shared expert
        dict(_gated("gated_grad", 4096, 7168, 2048), name="gated_grad_bf16_t4096"),
    ]


def _log_uniform(rng, least, most):
    return int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))


def draw(rng):
    """Any of the operators: 1 to 8192 tokens (a layer 1 to 2048, a training step up to 4096), sizes up to the listed ones, odd
    ones where they may be (rows are multiples of 16 bytes); layers of fewer experts, experts a token or shorter ones."""
    op = rng.choice(["linear", "layer", "gated", "gated_grad"])
    dtype = rng.choice(["bfloat16", "float16"])
    if op == "linear":
        return _linear(_log_uniform(rng, 1, 8192), _log_uniform(rng, 100, 4096), 16 * _log_uniform(rng, 16, 448), dtype,
                       rng.random() < 0.5)
    if op == "layer":
        family = rng.choice(sorted(LAYERS))
        f = LAYERS[family]
        other = dict(topk=rng.randint(1, f["topk"]))
        if f["experts"] > 8:
            other["experts"] = f["experts"] // rng.choice([1, 2, 4])
        else:
            other["inter"] = f["inter"] // rng.choice([1, 2, 4])
        return _layer(family, _log_uniform(rng, 1, 2048 if family != "mixtral" else 256), dtype, **other)
    return _gated(op, _log_uniform(rng, 1, 8192 if op == "gated" else 4096), 8 * _log_uniform(rng, 32, 896),
                  _log_uniform(rng, 100, 2048), dtype)


# ---- inputs -----------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _int8_rows(g, *shape):
    """Rows of N(0, 1/k) weights [..., n, k] as codes and a scale per row."""
    q = torch.empty(shape, dtype=torch.int8, device="cuda")
    s = torch.empty(shape[:-1], device="cuda")
    for i in range(shape[0] if len(shape) == 3 else 1):
        w = _randn(g, *shape[-2:]).mul_(shape[-1] ** -0.5)
        top = w.abs().amax(dim=-1).div_(127.0)
        (s[i] if len(shape) == 3 else s).copy_(top)
        (q[i] if len(shape) == 3 else q).copy_(w.div_(top[:, None]).round_())
    return q, s


def _import_package():
    sys.path.insert(0, os.path.join(os.getcwd(), "vllm-xpu-kernels_b200"))
    import vllm_xpu_kernels.fused_moe_interface as fmi
    import vllm_xpu_kernels.gated_linear as gl
    return fmi, gl


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, T = getattr(torch, case["dtype"]), case["tokens"]
    s = dict(op=case["op"])
    if case["op"] == "linear":
        s["w"], s["ws"] = _int8_rows(g, case["n"], case["k"])
        s["x"] = _randn(g, T, case["k"]).to(dtype)
        s["bias"] = _randn(g, case["n"]).to(dtype) if case["bias"] else None
        s["out"] = torch.empty(T, case["n"], dtype=dtype, device="cuda")
        if own:
            _import_package()
    elif case["op"] == "layer":
        H, I, E, K = (case[k] for k in ("hidden", "inter", "experts", "topk"))
        s["w13"], s["s13"] = _int8_rows(g, E, 2 * I, H)
        s["w2"], s["s2"] = _int8_rows(g, E, H, I)
        s["x"] = _randn(g, T, H).to(dtype)
        top = torch.rand(T, E, generator=g, device="cuda").topk(K, dim=-1)
        s["weights"], s["ids"] = torch.softmax(2.0 * top.values, dim=-1), top.indices.to(torch.int32)
        s["out"] = torch.empty(T, H, dtype=dtype, device="cuda")
        if own:
            fmi, _ = _import_package()
            s["layer"] = fmi.XpuFusedMoe(s["w13"], s["s13"], None, s["w2"], s["s2"], None, K, "silu", E)
    else:
        H, I = case["hidden"], case["inter"]
        s["x"], s["w"] = _randn(g, T, H).to(dtype), _randn(g, 2 * I, H).mul_(H ** -0.5).to(dtype)
        if case["op"] == "gated":
            s["out"] = torch.empty(T, I, dtype=dtype, device="cuda")
        else:
            s["grad"] = _randn(g, T, I).to(dtype)
            s["x"].requires_grad_(True)
            s["w"].requires_grad_(True)
        if own:
            s["module"] = _import_package()[1]
    return s


# ---- the passes ---------------------------------------------------------------

def _plain_codes(rows):
    """Rows as whole numbers from -127 to 127, and their scales."""
    scale = rows.abs().amax(dim=-1).clamp(min=LEAST) / 127.0
    return torch.round(rows / scale[..., None]), scale


def _plain_linear(s):
    q, scale = _plain_codes(s["x"].float())
    y = torch.matmul(q, s["w"].float().t()) * scale[:, None] * s["ws"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    s["out"].copy_(y)
    return s["out"]


def _plain_layer(s):
    """Every expert's product with every token, of which a token's own experts have a weight."""
    q, scale = _plain_codes(s["x"].float())
    E, T = s["w13"].shape[0], q.shape[0]
    a = torch.bmm(q.expand(E, T, -1), s["w13"].float().transpose(1, 2)) * scale[:, None] * s["s13"][:, None, :]
    gate, up = a.chunk(2, dim=-1)
    q, scale = _plain_codes(gate / (1.0 + torch.exp(-gate)) * up)
    y = torch.bmm(q, s["w2"].float().transpose(1, 2)) * scale[..., None] * s["s2"][:, None, :]
    mine = torch.zeros(T, E, device=y.device).scatter_(1, s["ids"].long(), s["weights"])
    s["out"].copy_((mine.t()[:, :, None] * y).sum(dim=0))
    return s["out"]


def _plain_gated(x, w):
    gate, up = torch.matmul(x.float(), w.float().t()).chunk(2, dim=-1)
    return gate, up, 1.0 / (1.0 + torch.exp(-gate))


def _plain_gated_grad(s):
    with torch.no_grad():
        dtype = s["x"].dtype
        gate, up, sig = _plain_gated(s["x"], s["w"])
        d = s["grad"].float()
        both = torch.cat((d * up * sig * (1.0 + gate * (1.0 - sig)), d * gate * sig), dim=-1)
        return dict(out=(gate * sig * up).to(dtype), dx=torch.matmul(both, s["w"].float()).to(dtype),
                    dw=torch.matmul(both.t(), s["x"].float()).to(dtype))


def run(state):
    s = state
    if s["op"] == "linear":
        if not own:
            return _plain_linear(s)
        torch.ops._xpu_C.b200_int8_linear(s["out"], s["x"], None, s["w"], s["ws"], s["bias"])
        return s["out"]
    if s["op"] == "layer":
        if not own:
            return _plain_layer(s)
        s["layer"].apply(s["out"], s["x"], s["weights"], s["ids"])
        return s["out"]
    if s["op"] == "gated":
        if not own:
            gate, up, sig = _plain_gated(s["x"], s["w"])
            s["out"].copy_(gate * sig * up)
            return s["out"]
        torch.ops._xpu_C.b200_gated_linear(s["out"], s["x"], s["w"])
        return s["out"]
    if not own:
        return _plain_gated_grad(s)
    out = s["module"].gated_linear(s["x"], s["w"])
    dx, dw = torch.autograd.grad(out, (s["x"], s["w"]), s["grad"])
    return dict(out=out.detach(), dx=dx, dw=dw)


# ---- what a pass needs, and what it gives in 64 bits ------------------------------

def work(case):
    """Linear: rows, weights and scales read, rows written.  Layer: the weights of the experts that a random routing reaches, tokens,
    ids and weights read, rows written.  Gated: rows and weights read, rows written; its gradients also read a gradient and write two."""
    T = case["tokens"]
    if case["op"] == "linear":
        n, k = case["n"], case["k"]
        return {"bytes": 2 * T * k + n * k + 4 * n + 2 * T * n + (2 * n if case["bias"] else 0), "flops": 2.0 * T * n * k}
    H, I = case["hidden"], case["inter"]
    if case["op"] == "layer":
        E, K = case["experts"], case["topk"]
        active = max(1.0, E * (1.0 - (1.0 - K / E) ** T))
        return {"bytes": active * (3 * H * I + 4 * (2 * I + H)) + 4 * T * H + 8 * T * K, "flops": 6.0 * T * K * H * I}
    forward = 2 * (T * H + 2 * I * H + T * I)
    if case["op"] == "gated":
        return {"bytes": forward, "flops": 4.0 * T * H * I}
    return {"bytes": forward + 2 * (T * I + T * H + 2 * I * H), "flops": 12.0 * T * H * I}


def _exact_codes(rows):
    scale = torch.clamp(rows.abs().max(dim=1).values, min=LEAST) / 127.0
    return torch.round(rows / scale.unsqueeze(1)), scale


def _exact_linear(s):
    q, scale = _exact_codes(s["x"].double())
    y = q.mm(s["w"].double().t())       # whole numbers that 64 bits hold
    y = y.mul(torch.outer(scale, s["ws"].double()))
    return y if s["bias"] is None else y.add(s["bias"].double())


def _exact_layer(s):
    q, scale = _exact_codes(s["x"].double())
    out = torch.zeros_like(q)
    for e in range(s["w13"].shape[0]):
        token, slot = torch.nonzero(s["ids"] == e, as_tuple=True)
        if token.numel() == 0:
            continue
        a = q[token].mm(s["w13"][e].double().t()) * torch.outer(scale[token], s["s13"][e].double())
        half = a.shape[1] // 2
        h, hs = _exact_codes(a[:, :half] * torch.sigmoid(a[:, :half]) * a[:, half:])
        y = h.mm(s["w2"][e].double().t()) * torch.outer(hs, s["s2"][e].double())
        out.index_add_(0, token, y * s["weights"][token, slot].double().unsqueeze(1))
    return out


def _exact_gated(s):
    x, w = s["x"].detach().double(), s["w"].detach().double()
    half = w.shape[0] // 2
    gate, up = x.mm(w[:half].t()), x.mm(w[half:].t())
    out = torch.nn.functional.silu(gate) * up
    if s["op"] == "gated":
        return out
    d, sig = s["grad"].double(), torch.sigmoid(gate)
    dgate, dup = d * up * (sig + gate * sig * (1 - sig)), d * gate * sig
    return dict(out=out, dx=dgate.mm(w[:half]) + dup.mm(w[half:]), dw=torch.cat((dgate.t().mm(x), dup.t().mm(x))))


def exact(case, seed):
    """In 64 bits, with no rounding behind the inputs' but that to the codes of rows."""
    s = prepare(case, seed)
    return {"linear": _exact_linear, "layer": _exact_layer}.get(case["op"], _exact_gated)(s)
