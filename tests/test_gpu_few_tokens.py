"""GPU: a whole layer for a few tokens (``XpuFusedMoe(few_tokens=True)``) against its formula in 64 bits.

The bound of an output comes from the roundings on its way, with the sums of magnitudes taken in 64 bits:

* a sum of n products in fp32, in any order, with additions that may truncate: (n + 32) 2^-23 of the sum of magnitudes;
* an operand of the tensor cores in 16 bits: half a step of its type, 2^-11 where rows are scaled to float16 (which
  keeps a bfloat16 as it is), 2^-8 for h next to bfloat16 weights, and 2^-30 of the row's largest magnitude for what
  falls below the type's range;
* the activation passes an error of gate on with a factor of at most 1.2 max(1, |up|) (|d silu|, |d gelu| and |d (g
  sigmoid(1.702 g))| are all below 1.2), one of up with |act(gate)|, and adds 2^-20 of its value by itself (exp, erf, tanh and
  division of fp32; 2^-20 absolute times (1 + |up|) for the tanh and erf forms, which cancel for negative gates);
* the output's own rounding, half a step.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]
BF16, F16 = torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def make_matrix(recipe, g, E, N, K, dtype, group):
    """-> (weights, scales as the layer takes them, [E, N, K] in 64 bits)."""
    def rand(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=torch.uint8)
    if recipe == "w16":
        w = (torch.randn(E, K, N, generator=g, device=DEV) * K ** -0.5).to(dtype)
        return w, None, w.double().transpose(1, 2)
    if recipe in ("fp8", "fp8_kn"):
        q = (torch.randn(E, N, K, generator=g, device=DEV) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        s = (torch.rand(E, N // 128, K // 128, generator=g, device=DEV) + 0.5) * K ** -0.5 / 100
        d = q.double() * s.double().repeat_interleave(128, 1).repeat_interleave(128, 2)
        return (q.transpose(1, 2).contiguous() if recipe == "fp8_kn" else q), s, d
    q = rand(0, 256, E, N, K // 2)
    codes = torch.stack((q & 15, q >> 4), -1).view(E, N, K).long()
    if recipe == "mxfp4":
        s = rand(117, 124, E, N, K // 32)
        d = torch.tensor(E2M1, device=DEV, dtype=torch.float64)[codes] * torch.exp2(s.double() - 127).repeat_interleave(32, 2)
        return q.view(torch.float4_e2m1fn_x2), s, d
    s = ((torch.rand(E, N, K // group, generator=g, device=DEV) + 0.5) * K ** -0.5 / 4).to(dtype)
    return q, s, (codes - 8).double() * s.double().repeat_interleave(group, 2)


def act64(kind, gate, up, limit=7.0, alpha=1.702):
    if kind == "silu":
        a = gate * torch.sigmoid(gate)
    elif kind == "gelu":
        a = gate * 0.5 * (1 + torch.erf(gate * 0.5 ** 0.5))
    elif kind == "gelu_tanh":
        a = 0.5 * gate * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (gate + 0.044715 * gate ** 3)))
    elif kind == "swigluoai":
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
        a, up = gate * torch.sigmoid(alpha * gate), up + 1
    else:
        a, up = (gate * torch.sigmoid(gate)).clamp(max=limit), up.clamp(-limit, limit)
    return a, up


def sum_bound(n):
    return (n + 32) * 2.0 ** -23


def reference(x, weights, ids, w13, b13, w2, b2, act, clamp, emap, h_half, half):
    """-> output and its bound, [T, H] in 64 bits."""
    T, K = ids.shape
    E = w13.shape[0]
    xd = x.double()
    out = torch.zeros(T, w2.shape[1], dtype=torch.float64, device=DEV)
    err = torch.zeros_like(out)
    for t in range(T):
        for k in range(K):
            e = int(ids[t, k])
            limit = E if emap is None else emap.numel()
            if not 0 <= e < limit:
                continue
            e = e if emap is None else int(emap[e])
            if not 0 <= e < E:
                continue
            a, mag = w13[e] @ xd[t], w13[e].abs() @ xd[t].abs()
            mag = mag + 2.0 ** -30 / sum_bound(x.shape[1]) * w13[e].abs().sum(1) * xd[t].abs().max()
            if b13 is not None:
                a, mag = a + b13[e].double(), mag + b13[e].double().abs()
            pairs = act == "swigluoai"
            split = (lambda v: (v[0::2], v[1::2])) if pairs else (lambda v: v.chunk(2))
            (gate, up), (mg, mu) = split(a), split(mag)
            if clamp:
                gate, up = gate.clamp(max=clamp), up.clamp(-clamp, clamp)
            av, uv = act64(act, gate, up)
            h = av * uv
            c = sum_bound(x.shape[1])
            dh = c * (1.2 * mg * uv.abs().clamp(min=1) + av.abs() * mu) + 2.0 ** -20 * (h.abs() + (uv.abs() + 1 if "gelu" in act else 0))
            dh = dh + h_half * (h.abs() + dh) + 2.0 ** -30 * h.abs().max()
            y = w2[e] @ h
            my = w2[e].abs() @ h.abs()
            if b2 is not None:
                y, my = y + b2[e].double(), my + b2[e].double().abs()
            wt = weights[t, k].double()
            out[t] += wt * y
            err[t] += wt.abs() * (w2[e].abs() @ dh + sum_bound(h.numel() + K) * (my + w2[e].abs() @ dh))
    return out, err + half * (out.abs() + err) + 2.0 ** -25


class Case:
    def __init__(self, native, recipe, T, H, I, E, K, dtype=BF16, act="silu", bias=False, clamp=None, group=128, seed=0, ranks=1, rank=0,
                 few=True, group2=None, **kw):
        g = gen(seed)
        self.T, self.H, self.dtype = T, H, dtype
        self.w13, self.s13, self.d13 = make_matrix(recipe, g, E, 2 * I, H, dtype, group)
        self.w2, self.s2, self.d2 = make_matrix(recipe, g, E, H, I, dtype, group2 or group)
        rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
        self.b13 = (rnd(E, 2 * I) * 0.1).to(dtype) if bias else None
        self.b2 = (rnd(E, H) * 0.1).to(dtype) if bias else None
        self.map = None
        if ranks > 1:
            self.map = torch.arange(E * ranks, device=DEV, dtype=torch.int32) - rank * E
            self.map[(self.map < 0) | (self.map >= E)] = -1
        self.layer = native.XpuFusedMoe(self.w13, self.s13, self.b13, self.w2, self.s2, self.b2, K, act, E, ep_rank=rank,
                                        ep_size=ranks, expert_map=self.map, gemm1_clamp_limit=clamp, few_tokens=few, **kw)
        self.act, self.clamp = act, clamp
        self.x = rnd(T, H).to(dtype)
        self.ids = torch.rand(T, E * ranks, generator=g, device=DEV).topk(min(K, E * ranks), -1).indices.to(torch.int32)
        if K > E * ranks:
            self.ids = torch.randint(0, E * ranks, (T, K), generator=g, device=DEV, dtype=torch.int32)
        self.weights = torch.rand(T, K, generator=g, device=DEV) + 0.1
        self.h_half = 2.0 ** -8 if recipe == "w16" and dtype == BF16 else 2.0 ** -11

    def run(self, out=None):
        out = torch.full((self.T, self.H), float("nan"), dtype=self.dtype, device=DEV) if out is None else out
        self.layer.apply(out, self.x, self.weights, self.ids, self.map)
        return out

    def check(self, out):
        ref, bound = reference(self.x, self.weights, self.ids, self.d13, self.b13, self.d2, self.b2, self.act, self.clamp, self.map,
                               self.h_half, torch.finfo(self.dtype).eps / 2)
        worst = ((out.double() - ref).abs() / bound).max().item()
        assert worst <= 1, worst
        return worst


SHAPES = [
    # recipe, hidden, inter, experts, topk, group
    ("w16", 64, 32, 4, 2, 0), ("w16", 72, 20, 3, 1, 0), ("w16", 512, 256, 8, 2, 0), ("w16", 2048, 1408, 8, 2, 0),
    ("w16", 264, 136, 60, 6, 0), ("w16", 8, 8, 1, 1, 0), ("w16", 1032, 1000, 2, 2, 0),
    ("fp8", 128, 128, 4, 2, 0), ("fp8", 256, 384, 16, 4, 0), ("fp8", 2048, 768, 32, 8, 0), ("fp8", 7168, 256, 4, 2, 0),
    ("fp8", 384, 2048, 3, 3, 0), ("fp8_kn", 256, 384, 4, 2, 0),
    ("mxfp4", 64, 64, 4, 2, 0), ("mxfp4", 32, 32, 2, 1, 0), ("mxfp4", 96, 160, 5, 3, 0), ("mxfp4", 2880, 2880, 4, 4, 0),
    ("mxfp4", 416, 608, 32, 4, 0),
    ("int4", 128, 128, 4, 2, 128), ("int4", 256, 512, 8, 2, 256), ("int4", 96, 160, 3, 2, 32), ("int4", 4096, 1024, 4, 2, 128),
    ("int4", 192, 320, 6, 2, 64),
]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("recipe,H,I,E,K,group", SHAPES)
def test_formats_and_sizes(native, recipe, H, I, E, K, group, dtype):
    for T in (1, 3, 16):
        c = Case(native, recipe, T, H, I, E, K, dtype, group=group, seed=T)
        c.check(c.run())


@pytest.mark.parametrize("group,group2", [(32, 128), (128, 32), (64, 256), (256, 64), (32, 64), (128, 256)])
def test_int4_groups_of_both(native, group, group2):
    """The two matrices may have groups of different lengths."""
    c = Case(native, "int4", 5, 768, 512, 6, 3, group=group, group2=group2, seed=group + group2)
    c.check(c.run())


@pytest.mark.parametrize("recipe", ["w16", "fp8", "mxfp4", "int4"])
@pytest.mark.parametrize("H,I,experts", [(8192, 256, 1), (16384, 128, 2), (256, 8192, 1), (256, 4096, 3)])
def test_more_tokens_than_a_block_holds(native, recipe, H, I, experts):
    """Tokens that a block's shared memory holds a part of, all with the same experts: several passes over the features, several
    stretches of h."""
    c = Case(native, recipe, 16, H, I, 4, 1, group=128, seed=H + I)
    c.ids[:, 0] = torch.arange(16, device=DEV, dtype=torch.int32) % experts
    c.check(c.run())


@pytest.mark.parametrize("recipe", ["w16", "fp8", "mxfp4", "int4"])
@pytest.mark.parametrize("T", [2, 13])
def test_more_experts_than_blocks(native, recipe, T):
    """Blocks whose features belong to many experts: small ones, most of them with one token."""
    c = Case(native, recipe, T, 128, 128, 300, 24, group=64, seed=T)
    c.check(c.run())


@pytest.mark.parametrize("T", range(1, 17))
@pytest.mark.parametrize("recipe", ["w16", "fp8", "mxfp4", "int4"])
def test_every_number_of_tokens(native, recipe, T):
    c = Case(native, recipe, T, 256, 256, 6, 3, seed=T)
    c.check(c.run())


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "swigluoai", "swiglustep"])
@pytest.mark.parametrize("clamp", [None, 0.5])
@pytest.mark.parametrize("recipe", ["w16", "fp8", "mxfp4", "int4"])
def test_activations_biases_and_limits(native, recipe, act, clamp):
    c = Case(native, recipe, 5, 256, 384, 6, 2, act=act, bias=True, clamp=clamp)
    c.x *= 4
    c.check(c.run())


@pytest.mark.parametrize("recipe", ["w16", "fp8", "mxfp4", "int4"])
def test_routing_that_is_not_even(native, recipe):
    c = Case(native, recipe, 16, 256, 256, 6, 3, seed=7)
    for kind in ("one expert", "same twice", "all alike", "unused tokens", "nobody", "ids of 64 bits"):
        ids = c.ids.clone()
        if kind == "one expert":
            ids.fill_(2)
        elif kind == "same twice":
            ids[:, 1] = ids[:, 0]
        elif kind == "all alike":
            ids[:] = ids[0]
        elif kind == "unused tokens":
            ids[3], ids[7], ids[0, 1], ids[15, 2] = -1, 6, 1 << 30, -(1 << 31)
        elif kind == "nobody":
            ids.fill_(-1)
        else:
            ids = ids.long()
            ids[2, 1], ids[4, 0] = 1 << 40, (1 << 32) + 1
        out = torch.full((16, 256), float("nan"), dtype=BF16, device=DEV)
        c.layer.apply(out, c.x, c.weights, ids)
        kept, c.ids = c.ids, ids
        c.check(out)
        c.ids = kept
        if kind == "nobody":
            assert (out == 0).all()


@pytest.mark.parametrize("recipe", ["w16", "fp8", "mxfp4", "int4"])
def test_a_rank_of_an_expert_parallel_layer(native, recipe):
    """The ranks' shares add up; rank 3 alone has the caller's map, the others the layer's own."""
    for rank in range(4):
        c = Case(native, recipe, 9, 256, 256, 4, 4, ranks=4, rank=rank, seed=3)
        c.check(c.run())
        if rank != 3:
            c.layer.expert_map, given = c.map, c.map
            out = torch.empty_like(c.x)
            c.layer.apply(out, c.x, c.weights, c.ids)
            assert torch.equal(out, c.run()) and c.map is given


@pytest.mark.parametrize("recipe", ["w16", "fp8", "mxfp4", "int4"])
@pytest.mark.parametrize("power", [-40, 30])
def test_rows_of_any_magnitude(native, recipe, power):
    """bfloat16 rows far outside float16's range, each with its own magnitude."""
    c = Case(native, recipe, 4, 256, 256, 4, 2, bias=False, act="silu")
    c.x[1] = (c.x[1].float() * 2.0 ** power).to(BF16)
    c.x[3, ::2] = (c.x[3, ::2].float() * 2.0 ** (power // 2)).to(BF16)
    c.check(c.run())


@pytest.mark.parametrize("recipe", ["w16", "fp8", "mxfp4", "int4"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_row_that_is_not_finite_stays_by_itself(native, recipe, value):
    c = Case(native, recipe, 5, 256, 256, 4, 2, seed=5)
    clean = c.run()
    c.x[2, 17] = value
    out = c.run()
    assert out[2].isnan().any()
    keep = [0, 1, 3, 4]
    assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("recipe", ["w16", "fp8", "mxfp4", "int4"])
def test_same_results_every_time_and_for_each_token_alone(native, recipe):
    """No atomics, no order that changes; a token's row does not depend on the others."""
    c = Case(native, recipe, 11, 512, 384, 8, 3, seed=9)
    first = c.run()
    for _ in range(3):
        assert torch.equal(c.run(), first)
    for t in (0, 10):
        one = torch.empty(1, 512, dtype=BF16, device=DEV)
        c.layer.apply(one, c.x[t:t + 1], c.weights[t:t + 1].contiguous(), c.ids[t:t + 1].contiguous())
        c2 = one.double() - first[t:t + 1].double()
        assert (c2.abs() <= 2.0 ** -6 * first[t].double().abs() + 2.0 ** -6 * first[t].double().abs().mean()).all()


def test_other_calls_of_the_layer_run_as_before(native):
    """More tokens than a few, and calls with quantised rows, are those of a layer without the option, bit for bit."""
    c = Case(native, "fp8", 16, 256, 256, 6, 2, seed=2)
    plain = Case(native, "fp8", 16, 256, 256, 6, 2, seed=2, few=False)
    x = torch.randn(17, 256, device=DEV).to(BF16)
    ids, w = torch.randint(0, 6, (17, 2), device=DEV, dtype=torch.int32), torch.rand(17, 2, device=DEV)
    a, b = torch.empty_like(x), torch.empty_like(x)
    c.layer.apply(a, x, w, ids)
    plain.layer.apply(b, x, w, ids)
    assert torch.equal(a, b)
    q, s = torch.empty(16, 256, device=DEV, dtype=torch.float8_e4m3fn), torch.empty(16, 2, device=DEV)
    torch.ops._C.per_token_group_fp8_quant(c.x, q, s, 128, 1e-10, -448.0, 448.0, False, False, False)
    a, b = torch.empty_like(c.x), torch.empty_like(c.x)
    c.layer.apply(a, q, c.weights, c.ids, a1q_scale=s)
    plain.layer.apply(b, q, c.weights, c.ids, a1q_scale=s)
    assert torch.equal(a, b)
    empty = torch.empty(0, 256, device=DEV, dtype=BF16)
    c.layer.apply(torch.empty_like(empty), empty, c.weights[:0], c.ids[:0])


def test_streams_graphs_and_workspaces(native):
    """Two captured graphs and eager calls, in turn and on streams of their own."""
    cases = [Case(native, r, 6, 256, 256, 6, 2, seed=4 + i) for i, r in enumerate(("fp8", "mxfp4"))]
    want = [c.run() for c in cases]
    torch.cuda.synchronize()
    graphs = []
    for c in cases:
        out = torch.zeros(6, 256, dtype=BF16, device=DEV)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            c.run(out)
        graphs.append((graph, out))
    for _ in range(3):
        streams = [torch.cuda.Stream() for _ in cases]
        eager = []
        for s, (graph, out), c in zip(streams, graphs, cases):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                out.zero_()
                graph.replay()
                eager.append(c.run())
        torch.cuda.synchronize()
        for (graph, out), e, w in zip(graphs, eager, want):
            assert torch.equal(out, w) and torch.equal(e, w)
    c = cases[0]
    c.x.copy_(torch.randn(6, 256, device=DEV))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    c.check(graphs[0][1])


@pytest.mark.parametrize("recipe", ["fp8", "mxfp4"])
def test_decoding_steps(native, recipe):
    """What a decoder block does between its attention and the next one's, as it would be called: norm with the residual's
    addition, router, layer for a few tokens; with the same results eagerly and replayed, over steps that follow one another."""
    from gpu_utils import topk_softmax
    T, H, E, K = 5, 512, 16, 4
    c = Case(native, recipe, T, H, 256, E, K, seed=11)
    router, weight = torch.randn(H, E, device=DEV) * H ** -0.5, torch.rand(H, device=DEV) + 0.5
    hidden, residual = torch.zeros(T, H, dtype=BF16, device=DEV), torch.zeros(T, H, dtype=BF16, device=DEV)
    rows, q, s = torch.empty_like(hidden), torch.empty(T, H, dtype=torch.float8_e4m3fn, device=DEV), torch.empty(T, H // 128, device=DEV)

    def step():
        torch.ops._C.b200_add_rms_norm(hidden, residual, weight, 1e-6, rows, q, s, 128)
        w, ids, _ = topk_softmax((rows.float() @ router).contiguous(), K, True)
        c.layer.apply(hidden, rows, w, ids)
        return w, ids

    start = c.x.clone()
    hidden.copy_(start)
    residual.copy_(start * 0.5)
    eager = []
    for _ in range(3):
        before = (hidden.double() + residual.double()).to(BF16)
        w, ids = step()
        assert torch.equal(residual, before)
        want = before.double() * (before.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt() * weight.double()
        # fp32 on the way (2^-18), then half a step of bfloat16
        assert ((rows.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -18) * want.abs()).all()
        back = q.double().view(T, H // 128, 128) * s.double()[..., None]
        # half a step of e4m3 and of the scale's reciprocal; below the normal codes half of 2^-9 scales
        assert ((back.view(T, H) - want).abs() <= (2.0 ** -4 + 2.0 ** -18) * want.abs() + 2.0 ** -10 * s.double().repeat_interleave(128, 1)).all()
        c.x, c.weights, c.ids = rows, w, ids
        c.check(hidden)
        eager.append(hidden.clone())
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    hidden.copy_(start)
    residual.copy_(start * 0.5)
    for want in eager:
        graph.replay()
        assert torch.equal(hidden, want)


def test_a_limit_on_the_blocks_changes_nothing(native):
    for recipe in ("w16", "fp8", "mxfp4"):
        c = Case(native, recipe, 7, 512, 384, 8, 3, seed=1)
        c.layer.gemm_max_ctas = 20
        c.check(c.run())


def test_refusals(native):
    c = Case(native, "fp8", 4, 256, 256, 4, 2)
    out = torch.empty_like(c.x)
    for args, error, message in [
            ((out.float(), c.x, c.weights, c.ids), RuntimeError, "bfloat16 or float16"),
            ((out, c.x.half(), c.weights, c.ids), RuntimeError, "same dtype"),
            ((out, c.x, c.weights.half(), c.ids), RuntimeError, "topk_weights must be float32"),
            ((out, c.x, c.weights, c.ids.short()), RuntimeError, "int64 or int32"),
            ((out, c.x, c.weights, c.ids[:, :1]), RuntimeError, "num_rows, TopK"),
            ((out[:3], c.x, c.weights, c.ids), RuntimeError, "num_rows, hidden_size"),
            ((out, c.x.t().contiguous().t(), c.weights, c.ids), RuntimeError, "contiguous"),
            ((out, c.x, c.weights.cpu(), c.ids), RuntimeError, "device of hidden_states"),
            ((out, c.x[:, :128].contiguous(), c.weights, c.ids), RuntimeError, ""),
            ((out, c.x, c.weights, c.ids, torch.zeros(3, device=DEV, dtype=torch.int32)), RuntimeError, "total_experts_num")]:
        with pytest.raises(error, match=message):
            c.layer.apply(*args)
    with pytest.raises(NotImplementedError):
        Case(native, "w16", 1, 64, 64, 2, 1, act="relu2_no_mul")
    w = torch.zeros(2, 64, 128, device=DEV).to(torch.float8_e4m3fn)
    with pytest.raises(NotImplementedError, match="few_tokens"):
        native.XpuFusedMoe(w, torch.ones(2, device=DEV), None, w, torch.ones(2, device=DEV), None, 1, "silu", 2, few_tokens=True)


def test_a_decoding_step(native):
    """Norm, router, top-k, the layer on 16-bit rows and, next to it, on the norm's 8-bit rows; captured and replayed."""
    T, H, I, E, K = 4, 512, 256, 8, 2
    c = Case(native, "fp8", T, H, I, E, K, seed=6)
    plain = Case(native, "fp8", T, H, I, E, K, seed=6, few=False)
    router = torch.randn(H, E, device=DEV).to(BF16)
    weight, residual = torch.rand(H, device=DEV).to(BF16), torch.randn(T, H, device=DEV).to(BF16)
    start = residual.clone()
    rows, q, s = torch.empty_like(c.x), torch.empty(T, H, device=DEV, dtype=torch.float8_e4m3fn), torch.empty(T, H // 128, device=DEV)
    w, ids, src = torch.empty(T, K, device=DEV), torch.empty(T, K, device=DEV, dtype=torch.int32), torch.empty(T, K, device=DEV, dtype=torch.int32)
    few, quant = torch.empty_like(c.x), torch.empty_like(c.x)

    def step():
        torch.ops._C.b200_add_rms_norm(c.x, residual, weight, 1e-6, rows, q, s, 128)
        torch.ops._moe_C.topk_softmax(w, ids, src, (rows @ router).float(), True, None)
        c.layer.apply(few, rows, w, ids)
        plain.layer.apply(quant, q, w, ids, a1q_scale=s)

    step()
    torch.cuda.synchronize()
    eager = [t.clone() for t in (residual, few, quant)]
    residual.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    residual.copy_(start)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip((residual, few, quant), eager):
        assert torch.equal(a, b)
    c.x, c.weights, c.ids = rows, w, ids
    c.check(few)
    # two roundings to e4m3 (rows and h, half a step each) against none: 2^-4 of what is multiplied, at random signs
    assert (few.double() - quant.double()).norm() <= 2.0 ** -4 * few.double().norm()
