"""Cases of two operators that a decoding step runs one after the other around its router.

* ``norm``: the residual's addition, the root-mean-square norm and the 8-bit copy of its rows with
  scales (``torch.ops._C.b200_add_rms_norm``).  The 16-bit rows go to the router and to layers that
  take 16-bit rows, the e4m3 rows and their scales to layers of quantised activations.
* ``layer``: a whole Mixture-of-Experts layer for a few tokens in two kernels
  (``XpuFusedMoe(..., few_tokens=True)``): the top-k op's ids and weights in, the weighted sum of
  the experts out, activations in 16 bits or more all the way.

Shapes are the ones of ``perf/cases.py``.  Inputs are seeded synthetic draws: rows ~N(0,1), norm weights
around 1, expert weights ~N(0, 1/fan_in) in the layer's storage format, routing by random scores.
"""
import math
import os
import sys

import torch

own = False

# family -> what its layers have in common; `experts` are the routed experts of the whole layer, of which one
# process holds experts / ranks
FAMILIES = {
    "small": dict(recipe="w16", hidden=2048, inter=1408, experts=8, topk=2, most=16),
    "mixtral": dict(recipe="w16", hidden=4096, inter=14336, experts=8, topk=2, most=16),
    "mixtral_int4": dict(recipe="int4", hidden=4096, inter=14336, experts=8, topk=2, most=16),
    "qwen3": dict(recipe="fp8", hidden=2048, inter=768, experts=128, topk=8, most=16),
    "deepseek": dict(recipe="fp8", hidden=7168, inter=2048, experts=256, topk=8, most=8),
    "deepseek_ep8": dict(recipe="fp8", hidden=7168, inter=2048, experts=256, topk=8, most=16, ranks=8),
    "gptoss": dict(recipe="mxfp4", hidden=2880, inter=2880, experts=128, topk=4, most=16, act="swigluoai"),
}
RANK = 3            # the rank whose share of an expert-parallel layer is run
LEAST_SCALE = 1.0 / (448.0 * 512.0)
ALPHA, LIMIT = 1.702, 7.0


def _layer(family, tokens, **other):
    f = FAMILIES[family]
    c = dict(op="layer", family=family, tokens=tokens, hidden=f["hidden"], inter=f["inter"], experts=f["experts"],
             topk=f["topk"], dtype="bfloat16")
    c.update(other)
    return c


def _norm(tokens, hidden, group, **other):
    """`group`: values of a row per scale, 0 for one scale a row."""
    c = dict(op="norm", tokens=tokens, hidden=hidden, group=group, dtype="bfloat16", residual=True, rows16=True,
             power_of_two=False)
    c.update(other)
    return c


def listed():
    return [
        # one user decoding on 4-bit experts: the shortest weight stream, launches and latency
        dict(_layer("gptoss", 1), name="layer_gptoss_mxfp4_t1"),
        # a few users on 4-bit experts
        dict(_layer("gptoss", 7), name="layer_gptoss_mxfp4_t7"),
        # a small decode batch over many small fp8 experts
        dict(_layer("qwen3", 16), name="layer_qwen3_fp8_t16"),
        # one user decoding on large fp8 experts
        dict(_layer("deepseek", 1), name="layer_deepseek_fp8_t1"),
        # one expert-parallel rank: an eighth of the slots is local
        dict(_layer("deepseek_ep8", 16), name="layer_deepseek_fp8_ep8_t16"),
        # speculative tokens of one user on int4 experts
        dict(_layer("mixtral_int4", 4), name="layer_mixtral_int4_t4"),
        # a small 16-bit layer: two experts' weights and latency
        dict(_layer("small", 1), name="layer_small_bf16_t1"),
        # the largest batch of this form on large 16-bit experts
        dict(_layer("mixtral", 16, dtype="float16"), name="layer_mixtral_fp16_t16"),
        # one decoded token: latency
        dict(_norm(1, 7168, 128), name="norm_bf16_t1_group128"),
        # a decode batch, one scale a row
        dict(_norm(61, 2880, 0), name="norm_bf16_t61_row"),
        # a chunk of a prompt: no residual, 8-bit rows alone, power-of-two scales
        dict(_norm(1001, 4096, 64, dtype="float16", residual=False, rows16=False, power_of_two=True),
             name="norm_fp16_t1001_group64"),
        # the largest prefill batch
        dict(_norm(8192, 7168, 128), name="norm_bf16_t8192_group128"),
    ]


def _log_uniform(rng, most):
    return int(round(math.exp(rng.uniform(0.0, math.log(most)))))


def draw(rng):
    """A layer family with 1 to 16 tokens, also with fewer experts (a token's or the layer's) or shorter ones, or a norm of
    1 to 8192 rows; small layers, and norms with one scale a row, also in other sizes."""
    if rng.random() < 0.5:
        family = rng.choice(sorted(FAMILIES))
        f = FAMILIES[family]
        other = dict(topk=rng.randint(1, f["topk"]))
        if f["experts"] > 8:
            other["experts"] = f["experts"] // rng.choice([1, 2, 4])
        else:
            other["inter"] = f["inter"] // rng.choice([1, 2, 4])
        if f["recipe"] in ("w16", "int4"):
            other["dtype"] = rng.choice(["bfloat16", "float16"])
        if family == "small":
            other.update(hidden=rng.choice([512, 1024, 2048]), inter=rng.choice([256, 704, 1408, 1536, 2048]),
                         experts=rng.choice([8, 16, 32, 60]), topk=rng.choice([1, 2, 4, 6]))
        return _layer(family, rng.randint(1, f["most"]), **other)
    group = rng.choice([0, 32, 64, 128])
    hidden = rng.choice([512, 2048, 4096, 7168]) if group else rng.choice([2880, rng.randint(100, 7168)])
    return _norm(_log_uniform(rng, 8192), hidden, group, dtype=rng.choice(["bfloat16", "float16", "float32"]),
                 residual=rng.random() < 0.7, rows16=rng.random() < 0.7, power_of_two=rng.random() < 0.3)


# ---- inputs -----------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _fp8_blocks(g, experts, n, k):
    """[experts, n, k] e4m3 weights drawn from N(0, 1/k) and their scale per 128x128 block."""
    q = torch.empty(experts, n, k, dtype=torch.float8_e4m3fn, device="cuda")
    s = torch.empty(experts, n // 128, k // 128, dtype=torch.float32, device="cuda")
    for e in range(experts):
        w = _randn(g, n // 128, 128, k // 128, 128).mul_(k ** -0.5)
        top = w.abs().amax(dim=(1, 3), keepdim=True).div_(448.0)
        q[e] = w.div_(top).view(n, k).to(torch.float8_e4m3fn)
        s[e] = top.view(n // 128, k // 128)
    return q, s


def _w16(g, experts, k, n, dtype):
    w = torch.empty(experts, k, n, dtype=dtype, device="cuda")
    for e in range(experts):
        w[e] = _randn(g, k, n).mul_(k ** -0.5)
    return w, None


def _int4(g, experts, n, k, dtype):
    """Two uint4 codes a byte (zero point 8) of N(0, 1/k) weights, scale per 128 values."""
    q = torch.empty(experts, n, k // 2, dtype=torch.uint8, device="cuda")
    for e in range(experts):
        c = _randn(g, n, k // 2, 2).mul_(2.5).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
        q[e] = c[..., 0] | (c[..., 1] << 4)
    s = torch.empty(experts, n, k // 128, device="cuda").uniform_(0.3, 0.5, generator=g).mul_(k ** -0.5).to(dtype)
    return q, s


def _mxfp4(g, experts, n, k):
    """Uniform e2m1 codes, e8m0 exponents in [-10, -4] per 32 values."""
    def some(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.uint8)
    return some(0, 256, experts, n, k // 2).view(torch.float4_e2m1fn_x2), some(117, 124, experts, n, k // 32)


def _prepare_layer(case, seed):
    f = FAMILIES[case["family"]]
    T, H, I, E, K = (case[k] for k in ("tokens", "hidden", "inter", "experts", "topk"))
    dtype = getattr(torch, case["dtype"])
    g = torch.Generator(device="cuda").manual_seed(seed)
    local = E // f.get("ranks", 1)
    b13 = b2 = None
    if f["recipe"] == "w16":
        (w13, s13), (w2, s2) = _w16(g, local, H, 2 * I, dtype), _w16(g, local, I, H, dtype)
    elif f["recipe"] == "int4":
        (w13, s13), (w2, s2) = _int4(g, local, 2 * I, H, dtype), _int4(g, local, H, I, dtype)
    elif f["recipe"] == "fp8":
        (w13, s13), (w2, s2) = _fp8_blocks(g, local, 2 * I, H), _fp8_blocks(g, local, H, I)
    else:
        (w13, s13), (w2, s2) = _mxfp4(g, local, 2 * I, H), _mxfp4(g, local, H, I)
        b13, b2 = (_randn(g, local, 2 * I) * 0.02).to(dtype), (_randn(g, local, H) * 0.02).to(dtype)
    top = torch.rand(T, E, generator=g, device="cuda").topk(K, dim=-1)
    expert_map = None
    if local < E:
        expert_map = torch.arange(E, dtype=torch.int32, device="cuda") - RANK * local
        expert_map[(expert_map < 0) | (expert_map >= local)] = -1
    state = dict(op="layer", recipe=f["recipe"], act=f.get("act", "silu"), w13=w13, s13=s13, b13=b13, w2=w2, s2=s2, b2=b2,
                 x=_randn(g, T, H).to(dtype), weights=torch.softmax(2.0 * top.values, dim=-1),
                 ids=top.indices.to(torch.int32), map=expert_map, out=torch.empty(T, H, dtype=dtype, device="cuda"))
    if own:
        sys.path.insert(0, os.path.join(os.getcwd(), "vllm-xpu-kernels_b200"))
        import vllm_xpu_kernels.fused_moe_interface as fmi
        state["layer"] = fmi.XpuFusedMoe(w13, s13, b13, w2, s2, b2, K, state["act"], local, ep_rank=RANK if local < E else 0,
                                         ep_size=E // local, expert_map=expert_map, few_tokens=True)
    return state


def _prepare_norm(case, seed):
    T, H = case["tokens"], case["hidden"]
    dtype = getattr(torch, case["dtype"])
    g = torch.Generator(device="cuda").manual_seed(seed)
    group = case["group"] or H
    if own:
        sys.path.insert(0, os.path.join(os.getcwd(), "vllm-xpu-kernels_b200"))
        import vllm_xpu_kernels.fused_moe_interface  # noqa: F401  (registers the ops)
    return dict(op="norm", group=group, power_of_two=case["power_of_two"], x=_randn(g, T, H).to(dtype),
                residual=(2.0 * _randn(g, T, H)).to(dtype) if case["residual"] else None,
                weight=(1.0 + 0.2 * _randn(g, H)).to(dtype), eps=1e-6,
                out=torch.empty(T, H, dtype=dtype, device="cuda") if case["rows16"] else None,
                q=torch.empty(T, H, dtype=torch.float8_e4m3fn, device="cuda"),
                scales=torch.empty(T, H // group, dtype=torch.float32, device="cuda"))


def prepare(case, seed):
    return _prepare_layer(case, seed) if case["op"] == "layer" else _prepare_norm(case, seed)


# ---- the passes ---------------------------------------------------------------

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _experts_matrix(s, w, scale, slots):
    """Rows [features, inputs] of the slots' experts, in 32 bits."""
    recipe = s["recipe"]
    if recipe == "w16":
        return w[slots].float().transpose(-1, -2)
    codes = w.view(torch.uint8)[slots]
    if recipe == "fp8":
        e, n, k = codes.shape
        blocks = codes.view(torch.float8_e4m3fn).float().view(e, n // 128, 128, k // 128, 128)
        return (blocks * scale[slots][:, :, None, :, None]).view(e, n, k)
    low, high = codes & 15, codes >> 4
    e, n, k = codes.shape[0], codes.shape[1], 2 * codes.shape[2]
    if recipe == "int4":
        values = torch.stack((low, high), dim=-1).float() - 8.0
        each = scale[slots].float()
    else:
        table = torch.tensor(_E2M1, device=w.device)
        values = torch.stack((table[low.int()], table[high.int()]), dim=-1)
        each = torch.exp2(scale[slots].float() - 127.0)
    return (values.view(e, n, each.shape[-1], k // each.shape[-1]) * each[..., None]).view(e, n, k)


def _plain_layer(s):
    x = s["x"].float()
    T, K = s["ids"].shape
    slots, weights = s["ids"].long().flatten(), s["weights"]
    if s["map"] is not None:
        slots = s["map"].long()[slots]
        weights = torch.where(slots.view(T, K) >= 0, weights, 0.0)
        slots = slots.clamp(min=0)
    rows = x[:, None, :].expand(T, K, -1).reshape(T * K, -1, 1)
    up = torch.matmul(_experts_matrix(s, s["w13"], s["s13"], slots), rows)[..., 0]
    if s["b13"] is not None:
        up = up + s["b13"].float()[slots]
    if s["act"] == "silu":
        gate, up = up.chunk(2, dim=-1)
        h = gate / (1.0 + torch.exp(-gate)) * up
    else:
        gate, up = up[:, 0::2].clamp(max=LIMIT), up[:, 1::2].clamp(-LIMIT, LIMIT)
        h = (up + 1.0) * gate / (1.0 + torch.exp(-ALPHA * gate))
    y = torch.matmul(_experts_matrix(s, s["w2"], s["s2"], slots), h[..., None])[..., 0]
    if s["b2"] is not None:
        y = y + s["b2"].float()[slots]
    s["out"].copy_((weights[..., None] * y.view(T, K, -1)).sum(dim=1))
    return s["out"]


def _plain_norm(s):
    x, group = s["x"], s["group"]
    if s["residual"] is not None:
        x = s["residual"].copy_(x.float() + s["residual"].float())
    f = x.float()
    y = f * torch.rsqrt((f * f).mean(dim=-1, keepdim=True) + s["eps"]) * s["weight"].float()
    if s["out"] is not None:
        s["out"].copy_(y)
    groups = y.view(y.shape[0], -1, group)
    scale = (groups.abs().amax(dim=-1) / 448.0).clamp(min=LEAST_SCALE)
    if s["power_of_two"]:
        scale = torch.exp2(torch.ceil(torch.log2(scale)))
    s["scales"].copy_(scale)
    s["q"].copy_((groups / scale[..., None]).clamp(-448.0, 448.0).view_as(y))
    return _norm_outputs(s)


def _norm_outputs(s):
    return {k: s[k] for k in ("residual", "out", "q", "scales") if s[k] is not None}


def run(state):
    s = state
    if s["op"] == "layer":
        if not own:
            return _plain_layer(s)
        s["layer"].apply(s["out"], s["x"], s["weights"], s["ids"], s["map"])
        return s["out"]
    if not own:
        return _plain_norm(s)
    torch.ops._C.b200_add_rms_norm(s["x"], s["residual"], s["weight"], s["eps"], s["out"], s["q"], s["scales"], s["group"],
                                   s["power_of_two"])
    return _norm_outputs(s)


# ---- what a pass needs, and what it gives in 64 bits ------------------------------

def work(case):
    """Layer: the weights of the experts that a random routing reaches, tokens, ids and weights read, rows written; two
    multiplications of every local slot.  Norm: rows, residual and weight read; residual, 16-bit and 8-bit rows and scales written."""
    T, H = case["tokens"], case["hidden"]
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "norm":
        values = T * H * (size + 1 + (2 * size if case["residual"] else 0) + (size if case["rows16"] else 0))
        return {"bytes": values + size * H + 4 * T * H // (case["group"] or H), "flops": 6.0 * T * H}
    f = FAMILIES[case["family"]]
    I, E, K = case["inter"], case["experts"], case["topk"]
    local = E // f.get("ranks", 1)
    active = max(1.0, local * (1.0 - (1.0 - K / E) ** T))
    n = 3 * H * I
    each = {"w16": 2 * n, "fp8": n + 4 * n // 16384, "int4": n // 2 + 2 * n // 128,
            "mxfp4": n // 2 + n // 32 + 2 * (2 * I + H)}[f["recipe"]]
    return {"bytes": active * each + 4 * T * H + 8 * T * K, "flops": 6.0 * T * K * local / E * H * I}


def _exact_matrix(s, w, scale, e):
    """One expert's [features, inputs] in 64 bits."""
    if s["recipe"] == "w16":
        return w[e].double().t()
    if s["recipe"] == "fp8":
        return w[e].double() * scale[e].double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    byte = w[e].view(torch.uint8).long()
    codes = torch.empty(byte.shape[0], 2 * byte.shape[1], dtype=torch.long, device=byte.device)
    codes[:, 0::2], codes[:, 1::2] = byte % 16, byte // 16
    if s["recipe"] == "int4":
        values, each = (codes - 8).double(), scale[e].double()
    else:
        values = torch.tensor(_E2M1, dtype=torch.float64, device=byte.device)[codes]
        each = torch.pow(2.0, scale[e].double() - 127.0)
    return values * each.repeat_interleave(values.shape[1] // each.shape[1], 1)


def _exact_layer(s):
    x, ids, w = s["x"].double(), s["ids"].tolist(), s["weights"].double()
    out = torch.zeros_like(x)
    for t, row in enumerate(ids):
        for k, e in enumerate(row):
            if s["map"] is not None:
                e = int(s["map"][e])
            if e < 0:
                continue
            a = torch.mv(_exact_matrix(s, s["w13"], s["s13"], e), x[t])
            if s["b13"] is not None:
                a += s["b13"][e].double()
            if s["act"] == "silu":
                half = a.numel() // 2
                h = a[:half] * torch.sigmoid(a[:half]) * a[half:]
            else:
                gate, up = torch.clamp(a[0::2], max=LIMIT), torch.clamp(a[1::2], min=-LIMIT, max=LIMIT)
                h = (1.0 + up) * (gate * torch.sigmoid(ALPHA * gate))
            y = torch.mv(_exact_matrix(s, s["w2"], s["s2"], e), h)
            if s["b2"] is not None:
                y += s["b2"][e].double()
            out[t] += w[t, k] * y
    return out


def _exact_norm(s):
    dtype, group = s["x"].dtype, s["group"]
    v = s["x"].double()
    got = {}
    if s["residual"] is not None:
        got["residual"] = v + s["residual"].double()
        v = got["residual"].to(dtype).double()      # the rows that are normalised are the ones that are stored
    y = v / torch.sqrt(v.square().sum(dim=1, keepdim=True) / v.shape[1] + s["eps"]) * s["weight"].double()
    if s["out"] is not None:
        got["out"] = y
    parts = y.unflatten(1, (-1, group))
    scale = torch.clamp(parts.abs().max(dim=2).values / 448.0, min=LEAST_SCALE)
    if s["power_of_two"]:
        scale = torch.pow(2.0, torch.ceil(torch.log2(scale)))
    got["q"] = (parts / scale.unsqueeze(2)).flatten(1)      # before its rounding
    got["scales"] = scale
    return got


def exact(case, seed):
    """In 64 bits, with no rounding behind the inputs' but that of the stored residual."""
    s = prepare(case, seed)
    return _exact_layer(s) if case["op"] == "layer" else _exact_norm(s)
