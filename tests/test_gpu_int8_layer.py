"""XpuFusedMoe with int8 weights, against its definition in 64 bits; runs of the operators one after the other."""
import copy

import pytest
import torch

import int8_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
B16, F16 = torch.bfloat16, torch.float16
U = 2.0 ** -24


def _weights(E, H, I, gen):
    def some(n, k):
        q = torch.randint(-127, 128, (E, n, k), generator=gen, dtype=torch.int8)
        return q.to(DEV), ((torch.rand(E, n, generator=gen) + 0.5) * k ** -0.5 / 73).to(DEV)
    return some(2 * I, H) + some(H, I)


def _routing(T, E, K, gen):
    top = torch.rand(T, E, generator=gen).topk(K, dim=-1)
    return torch.softmax(top.values, -1).to(DEV), top.indices.to(torch.int32).to(DEV)


def _exact_rows(x, w13, s13, b13, w2, s2, b2, act, clamp=None):
    """One expert's rows in 64 bits, and what they may be off by before their rounding: codes of h that lie within `near` of a tie may
    be the neighbouring ones."""
    q, qs = ref.quant_rows(x)
    q, qs = q.to(DEV), qs.to(DEV)
    a, p = ref.linear(q, qs, w13, s13, b13)
    ea = (3.01 * p.abs() + a.abs()) * U
    g, u, eg, eu = *a.chunk(2, -1), *ea.chunk(2, -1)
    if clamp:
        g, u = g.clamp(max=clamp), u.clamp(-clamp, clamp)
    h, eh = act(g, u, eg, eu)
    top = h.abs().amax(-1, keepdim=True)
    scale = top.clamp(min=ref.LEAST) / 127
    rel = eh.amax(-1, keepdim=True) / top.clamp(min=ref.LEAST) + 2 * U     # of the scale
    near = eh / scale + (h.abs() / scale) * (rel + 2 * U) + 127 * U
    v = h / scale
    q2 = torch.round(v)
    tie = ((v - torch.floor(v) - 0.5).abs() <= near).double()
    wide = torch.clamp(near - 0.5, min=0).ceil() + tie                      # steps that a code may be off
    y, p2 = ref.linear(q2, scale[:, 0], w2, s2, b2)
    off = (wide * scale) @ (w2.double() * s2.double()[:, None]).abs().t()
    return y, off + p2.abs() * (rel + 3 * U) + y.abs() * U


def _silu(g, u, eg, eu):
    h = ref.silu(g) * u
    return h, 1.1 * u.abs() * eg + ref.silu(g).abs() * eu + h.abs() * (2.0 ** -20 + g.abs() * 2.0 ** -23)


def _check(out, x, weights, ids, w13, s13, b13, w2, s2, b2, act=_silu, clamp=None, emap=None, parts=0.0):
    """`parts`: half a step of parts of a token's sum that are rounded before they are added up."""
    dtype = out.dtype
    step = torch.finfo(dtype).eps / 2
    want, tol = torch.zeros_like(out, dtype=torch.float64), torch.full_like(out, torch.finfo(dtype).smallest_normal * step, dtype=torch.float64)
    for e in range(w13.shape[0]):
        local = ids.long() if emap is None else emap.long()[ids.long()]
        t, k = torch.nonzero(local == e, as_tuple=True)
        if t.numel() == 0:
            continue
        b = lambda v: None if v is None else v[e]  # noqa: E731
        y, off = _exact_rows(x[t], w13[e], s13[e], b(b13), w2[e], s2[e], b(b2), act, clamp)
        w = weights[t, k].double()[:, None]
        want.index_add_(0, t, w * y)
        # rows are rounded, half a step of their size or of the type's subnormal numbers (a row's -1.208e-5 of float16, weight 0.47, may be off by
        # 2^-25 of them: 1.4e-8, and their sum by as much as that and 2^-25), then added up in fp32
        tol.index_add_(0, t, w.abs() * (off + (y.abs() + off) * (step + 10 * U + parts * (1 + step)) + torch.finfo(dtype).smallest_normal * step))
    tol = tol + (want.abs() + tol) * step * (1 + 2.0 ** -10)
    err = (out.double() - want).abs()
    assert torch.all(err <= tol), float((err / tol).max())


@pytest.mark.parametrize("dtype", [B16, F16])
@pytest.mark.parametrize("T,E,K,H,I,bias", [(1, 8, 2, 128, 64, False), (3, 4, 1, 48, 16, True), (16, 8, 2, 256, 144, False),
                                            (33, 4, 2, 64, 304, True), (200, 8, 2, 272, 128, False), (600, 2, 2, 128, 48, True),
                                            (40, 128, 8, 128, 64, False)])
def test_layer(native, T, E, K, H, I, bias, dtype):
    gen = torch.Generator().manual_seed(T + E + H + I)
    w13, s13, w2, s2 = _weights(E, H, I, gen)
    b13 = torch.randn(E, 2 * I, generator=gen).to(dtype).to(DEV) if bias else None
    b2 = torch.randn(E, H, generator=gen).to(dtype).to(DEV) if bias else None
    x = torch.randn(T, H, generator=gen).to(dtype).to(DEV)
    weights, ids = _routing(T, E, K, gen)
    layer = native.XpuFusedMoe(w13, s13, b13, w2, s2, b2, K, "silu", E)
    assert layer.recipe == "int8"
    for ids_ in (ids, ids.long()):
        out = torch.full((T, H), float("nan"), dtype=dtype, device=DEV)
        layer.apply(out, x, weights, ids_)
        _check(out, x, weights, ids, w13, s13, b13, w2, s2, b2)


@pytest.mark.parametrize("T", [2, 100])
def test_clamp_and_the_form_of_two_kernels(native, T):
    gen = torch.Generator().manual_seed(T)
    E, K, H, I = 4, 2, 64, 32
    w13, s13, w2, s2 = _weights(E, H, I, gen)
    x = torch.randn(T, H, generator=gen).to(F16).to(DEV)
    weights, ids = _routing(T, E, K, gen)
    out = torch.empty(T, H, dtype=F16, device=DEV)
    native.XpuFusedMoe(w13, s13, None, w2, s2, None, K, "silu", E, gemm1_clamp_limit=0.7).apply(out, x, weights, ids)
    _check(out, x, weights, ids, w13, s13, None, w2, s2, None, clamp=0.7)

    def rounded(g, u, eg, eu):     # gates and ups go through 16 bits
        h, eh = _silu(g, u, eg + g.abs() * 2.0 ** -11 * 1.01, eu + u.abs() * 2.0 ** -11 * 1.01)
        return h, eh + 1.1 * 2.0 ** -11 * g.abs() * u.abs() * 2.0 ** -11
    native.XpuFusedMoe(w13, s13, None, w2, s2, None, K, "silu", E, gemm1_clamp_limit=0.7, fuse_activation=False).apply(out, x, weights, ids)
    _check(out, x, weights, ids, w13, s13, None, w2, s2, None, act=rounded, clamp=0.7)


@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "swigluoai", "swiglustep", "relu2_no_mul"])
def test_other_activations(native, name):
    """Through 16 bits before and behind the activation: a code may be a few steps off; h is compared before its rounding to codes."""
    T, E, K, H, I = 20, 4, 2, 64, 32
    gen = torch.Generator().manual_seed(len(name))
    w13, s13, w2, s2 = _weights(E, H, I, gen)
    if name == "relu2_no_mul":
        w2 = torch.randint(-127, 128, (E, H, 2 * I), generator=gen, dtype=torch.int8).to(DEV)
    x = torch.randn(T, H, generator=gen).to(F16).to(DEV)
    weights, ids = _routing(T, E, K, gen)
    out = torch.empty(T, H, dtype=F16, device=DEV)
    native.XpuFusedMoe(w13, s13, None, w2, s2, None, K, name, E).apply(out, x, weights, ids)

    def act(a):
        g, u = a.chunk(2, -1)
        if name == "gelu":
            return torch.nn.functional.gelu(g) * u
        if name == "gelu_tanh":
            return torch.nn.functional.gelu(g, approximate="tanh") * u
        if name == "swiglustep":
            return ref.silu(g).clamp(max=7.0) * u.clamp(-7.0, 7.0)
        if name == "relu2_no_mul":
            return a.clamp(min=0) ** 2
        g, u = a[:, 0::2].clamp(max=7.0), a[:, 1::2].clamp(-7.0, 7.0)
        return (u + 1) * g * torch.sigmoid(1.702 * g)
    want, tol = torch.zeros(T, H, dtype=torch.float64, device=DEV), torch.zeros(T, H, dtype=torch.float64, device=DEV)
    for e in range(E):
        t, k = torch.nonzero(ids == e, as_tuple=True)
        q, qs = ref.quant_rows(x[t])
        a, _ = ref.linear(q.to(DEV), qs.to(DEV), w13[e], s13[e])
        h = act(a)
        w = weights[t, k].double()[:, None]
        dense = (w2[e].double() * s2[e].double()[:, None])
        y = h @ dense.t()
        # half a step of the row, and what 2^-11 of a gate and an up and of h itself move it: derivatives are below 2 (1 + |a|) each
        big = a.abs().amax(-1, keepdim=True)
        move = 4 * (1 + big) ** 2 * 2.0 ** -11
        off = (h.abs().amax(-1, keepdim=True) / 127 * 0.51 + move) * dense.abs().sum(-1)[None]
        want.index_add_(0, t, w * y)
        tol.index_add_(0, t, w * (off + y.abs() * 2.0 ** -10))
    assert torch.all((out.double() - want).abs() <= tol + want.abs() * 2.0 ** -10)
    assert float((out.double() - want).norm() / want.norm()) < 0.05          # (no sum of bounds: two quantisations of 1/254 of a row's largest)


@pytest.mark.parametrize("T", [4, 150])
def test_experts_of_one_rank(native, T):
    gen = torch.Generator().manual_seed(T)
    E, K, H, I, ep = 16, 4, 64, 48, 4
    w13, s13, w2, s2 = _weights(E, H, I, gen)
    x = torch.randn(T, H, generator=gen).to(B16).to(DEV)
    weights, ids = _routing(T, E, K, gen)
    n = E // ep
    for rank in range(ep):
        mine = slice(rank * n, (rank + 1) * n)
        layer = native.XpuFusedMoe(w13[mine].contiguous(), s13[mine].contiguous(), None, w2[mine].contiguous(), s2[mine].contiguous(), None,
                                   K, "silu", n, ep_rank=rank, ep_size=ep)
        out = torch.full((T, H), float("nan"), dtype=B16, device=DEV)
        layer.apply(out, x, weights, ids)
        _check(out, x, weights, ids, w13[mine], s13[mine], None, w2[mine], s2[mine], None, emap=layer.expert_map)


@pytest.mark.parametrize("T", [3, 80])
def test_graphs_streams_copies_and_hooks(native, T):
    gen = torch.Generator().manual_seed(T)
    E, K, H, I = 8, 2, 128, 64
    w13, s13, w2, s2 = _weights(E, H, I, gen)
    x = torch.randn(T, H, generator=gen).to(B16).to(DEV)
    weights, ids = _routing(T, E, K, gen)
    layer = native.XpuFusedMoe(w13, s13, None, w2, s2, None, K, "silu", E)
    want = torch.empty(T, H, dtype=B16, device=DEV)
    layer.apply(want, x, weights, ids)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.apply(out, x, weights, ids)
    graph.replay()
    assert torch.equal(out, want)
    x2 = torch.randn(T, H, generator=gen).to(B16).to(DEV)
    x.copy_(x2)
    layer.apply(want, x, weights, ids)
    graph.replay()
    assert torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.empty_like(want)
        copy.copy(layer).apply(got, x, weights, ids)
    side.synchronize()
    assert torch.equal(got, want)
    stages = []
    layer.stage_hook = stages.append
    layer.persistent_workspace = False
    layer.apply(got, x, weights, ids)
    assert torch.equal(got, want) and stages == ["routing", "permute", "gemm1", "activation", "gemm2", "gather"]
    assert torch.equal(native.xpu_fused_moe(x, w13, s13, None, w2, s2, None, weights, ids, K, "silu", E), want)


def test_refusals(native):
    gen = torch.Generator().manual_seed(0)
    E, K, H, I = 4, 2, 64, 32
    w13, s13, w2, s2 = _weights(E, H, I, gen)
    x = torch.randn(5, H, generator=gen).to(B16).to(DEV)
    weights, ids = _routing(5, E, K, gen)
    out = torch.empty(5, H, dtype=B16, device=DEV)
    make = native.XpuFusedMoe
    with pytest.raises(NotImplementedError, match="few_tokens"):
        make(w13, s13, None, w2, s2, None, K, "silu", E, few_tokens=True)
    with pytest.raises(ValueError, match="no fused epilogue"):
        make(w13, s13, None, w2, s2, None, K, "swigluoai", E, fuse_activation=True)
    with pytest.raises(ValueError, match="both|w13 and w2"):
        make(w13, s13, None, w2.to(B16), None, None, K, "silu", E)
    layer = make(w13, s13, None, w2, s2, None, K, "silu", E)
    with pytest.raises(NotImplementedError, match="quantise their rows"):
        layer.apply(out, x, weights, ids, a1q_scale=torch.ones(5, 1, device=DEV))
    with pytest.raises(NotImplementedError, match="apply_sorted"):
        layer.apply_sorted(out, x, torch.tensor([5, 0, 0, 0], dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="int8 must be"):
        make(w13, s13[:, :32].contiguous(), None, w2, s2, None, K, "silu", E).apply(out, x, weights, ids)
    with pytest.raises(RuntimeError, match="divisible by 16"):
        make(w13[..., :56].contiguous(), s13, None, w2[:, :56].contiguous(), s2[:, :56].contiguous(), None, K, "silu",
             E).apply(out[:, :56].contiguous(), x[:, :56].contiguous(), weights, ids)
    with pytest.raises(RuntimeError, match="dtype"):
        layer.apply(out, x.half(), weights, ids)


@pytest.mark.parametrize("T", [2, 90])
def test_a_block_with_a_shared_expert(native, T):
    """What a decoder block runs one after the other: norm, routed int8 experts, and a shared expert in int8 beside them."""
    gen = torch.Generator().manual_seed(T)
    E, K, H, I = 8, 2, 128, 64
    w13, s13, w2, s2 = _weights(E, H, I, gen)
    v13, t13 = ref.weights(2 * I, H, gen)
    v2, t2 = ref.weights(H, I, gen)
    v13[v13 == -128], v2[v2 == -128] = -127, -127
    t13, t2 = t13 * 0.2, t2 * 0.2
    x = torch.randn(T, H, generator=gen).to(B16).to(DEV)
    res = torch.randn(T, H, generator=gen).to(B16).to(DEV)
    weights, ids = _routing(T, E, K, gen)
    normed = torch.empty_like(x)
    torch.ops._C.b200_add_rms_norm(x, res, None, 1e-6, normed)
    routed = torch.empty_like(x)
    native.XpuFusedMoe(w13, s13, None, w2, s2, None, K, "silu", E).apply(routed, normed, weights, ids)
    both = torch.empty(T, 2 * I, dtype=B16, device=DEV)
    torch.ops._xpu_C.b200_int8_linear(both, normed, None, v13, t13)
    q, qs = torch.empty(T, I, dtype=torch.int8, device=DEV), torch.empty(T, device=DEV)
    torch.ops._C.b200_silu_and_mul_quant_int8_rows(q, both, qs)
    shared = torch.empty_like(x)
    torch.ops._xpu_C.b200_int8_linear(shared, q, qs, v2, t2)
    _check(routed, normed, weights, ids, w13, s13, None, w2, s2, None)

    def rounded(g, u, eg, eu):     # the products go through bfloat16
        return _silu(g, u, eg + g.abs() * 2.0 ** -8 * 1.01, eu + u.abs() * 2.0 ** -8 * 1.01)
    one = torch.ones(T, 1, device=DEV)
    _check(shared, normed, one, torch.zeros(T, 1, dtype=torch.int32, device=DEV), v13[None], t13[None], None, v2[None], t2[None], None, act=rounded)


# T, E, K, H, I: rows of more pieces than a block of the permutation keeps, more slots than its small form takes, more than eight experts a token
@pytest.mark.parametrize("T,E,K,H,I", [(5, 2, 1, 8448, 16), (3, 4, 2, 33024, 16), (40, 2, 2, 20016, 16), (1100, 8, 4, 128, 32), (1100, 4, 2, 8448, 16),
                                       (30, 16, 10, 64, 32), (300, 32, 16, 48, 16), (1, 256, 8, 64, 16)])
def test_permutations(native, T, E, K, H, I):
    gen = torch.Generator().manual_seed(T + H)
    w13, s13, w2, s2 = _weights(E, H, I, gen)
    x = torch.randn(T, H, generator=gen).to(B16).to(DEV)
    weights, ids = _routing(T, E, K, gen)
    out = torch.full((T, H), float("nan"), dtype=B16, device=DEV)
    native.XpuFusedMoe(w13, s13, None, w2, s2, None, K, "silu", E).apply(out, x, weights, ids)
    _check(out, x, weights, ids, w13, s13, None, w2, s2, None)


def test_nothing_to_do(native):
    """No tokens; experts that get none; a token none of whose experts are here; a row of zeros."""
    gen = torch.Generator().manual_seed(3)
    E, K, H, I = 4, 2, 64, 32
    w13, s13, w2, s2 = _weights(E, H, I, gen)
    layer = native.XpuFusedMoe(w13, s13, None, w2, s2, None, K, "silu", E)
    empty = torch.empty(0, H, dtype=B16, device=DEV)
    layer.apply(empty, empty.clone(), torch.empty(0, K, device=DEV), torch.empty(0, K, dtype=torch.int32, device=DEV))
    x = torch.randn(6, H, generator=gen).to(B16).to(DEV)
    x[2] = 0
    weights, ids = torch.rand(6, K, generator=gen).to(DEV), torch.tensor([[1, 1], [1, 3], [1, 3], [-1, -1], [3, -1], [1, 3]], dtype=torch.int32, device=DEV)
    out = torch.full((6, H), float("nan"), dtype=B16, device=DEV)
    layer.apply(out, x, weights, ids)
    # (an id that is not an expert's drops its slot)
    _check(out, x, weights, ids, w13, s13, None, w2, s2, None)
    assert not out[2].any() and not out[3].any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_row_that_is_not_finite_stays_visible_and_alone(native, bad):
    gen = torch.Generator().manual_seed(4)
    E, K, H, I, T = 4, 2, 64, 32, 40
    w13, s13, w2, s2 = _weights(E, H, I, gen)
    x = torch.randn(T, H, generator=gen).to(B16).to(DEV)
    weights, ids = _routing(T, E, K, gen)
    layer = native.XpuFusedMoe(w13, s13, None, w2, s2, None, K, "silu", E)
    want, got = (torch.empty(T, H, dtype=B16, device=DEV) for _ in range(2))
    layer.apply(want, x, weights, ids)
    x[7, 5] = bad
    layer.apply(got, x, weights, ids)
    assert torch.isnan(got[7]).all()
    others = torch.arange(T, device=DEV) != 7
    assert torch.equal(got[others], want[others])


@pytest.mark.parametrize("T", [3, 90])
def test_two_graphs_replayed_in_turn(native, T):
    """Two layers of one shape captured after each other, on one stream's workspace, with a dense product in the second graph."""
    gen = torch.Generator().manual_seed(T)
    E, K, H, I = 8, 2, 128, 64
    graphs, outs, inputs, eager = [], [], [], []
    for _ in range(2):
        w13, s13, w2, s2 = _weights(E, H, I, gen)
        layer = native.XpuFusedMoe(w13, s13, None, w2, s2, None, K, "silu", E)
        v, t = ref.weights(48, H, gen)
        x = torch.randn(T, H, generator=gen).to(B16).to(DEV)
        weights, ids = _routing(T, E, K, gen)
        out, dense = torch.empty(T, H, dtype=B16, device=DEV), torch.empty(T, 48, dtype=B16, device=DEV)

        def run(out=out, dense=dense, x=x, layer=layer, v=v, t=t, weights=weights, ids=ids):
            layer.apply(out, x, weights, ids)
            torch.ops._xpu_C.b200_int8_linear(dense, x, None, v, t)
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        graphs.append(graph), outs.append((out, dense)), inputs.append(x), eager.append(run)
    for step in range(3):
        for x in inputs:
            x.copy_(torch.randn(T, H, generator=gen).to(B16))
        wants = []
        for run, pair in zip(eager, outs):
            run()
            wants.append([o.clone() for o in pair])
            for o in pair:
                o.fill_(float("nan"))
        for i in (step % 2, 1 - step % 2):
            graphs[i].replay()
        for pair, want in zip(outs, wants):
            assert all(torch.equal(o, w) for o, w in zip(pair, want))


@pytest.mark.parametrize("ep,tokens", [(2, (5, 9)), (4, (33, 0, 64, 7))])
def test_expert_parallel_over_peer_memory(native, ep, tokens):
    """All ranks in this process, one phase after the other; every rank's part of a token's sum travels as a 16-bit row."""
    from vllm_xpu_kernels.ep_moe import EpPeerFusedMoe, LocalPeerWorld
    gen = torch.Generator().manual_seed(ep)
    E, K, H, I = 8, 4, 128, 64
    w13, s13, w2, s2 = _weights(E, H, I, gen)
    n, world = E // ep, LocalPeerWorld(ep, DEV)
    layers = []
    for r in range(ep):
        mine = slice(r * n, (r + 1) * n)
        layers.append(EpPeerFusedMoe(w13[mine].contiguous(), s13[mine].contiguous(), None, w2[mine].contiguous(), s2[mine].contiguous(), None,
                                     K, "silu", n, world.member(r), max(tokens), H))
    for _ in range(2):      # the second call runs over the first one's leftovers
        given = []
        for r in range(ep):
            weights, ids = _routing(max(tokens[r], 1), E, K, gen)
            given.append((torch.randn(tokens[r], H, generator=gen).to(B16).to(DEV), weights[:tokens[r]], ids[:tokens[r]]))
            layers[r].dispatch(*given[r])
        for r in range(ep):
            layers[r].experts_and_combine()
        for r in range(ep):
            out = torch.full((tokens[r], H), float("nan"), dtype=B16, device=DEV)
            layers[r].finish(out)
            if tokens[r]:
                _check(out, *given[r], w13, s13, None, w2, s2, None, parts=2.0 ** -8)


def test_first_calls_under_capture():
    """A process whose first call of every operator is captured, and replayed on other inputs."""
    import subprocess
    import sys

    from conftest import PKG_DIR
    code = f"""
import sys
sys.path.insert(0, {str(PKG_DIR)!r})
import torch
import vllm_xpu_kernels.fused_moe_interface as fmi
from vllm_xpu_kernels.gated_linear import gated_linear
gen = torch.Generator().manual_seed(1)
B16, DEV = torch.bfloat16, "cuda"
def codes(*shape):
    return torch.randint(-127, 128, shape, generator=gen, dtype=torch.int8).to(DEV), (torch.rand(shape[:-1], generator=gen) * 1e-3).to(DEV)
E, K, H, I = 8, 2, 128, 64
layer = fmi.XpuFusedMoe(*codes(E, 2 * I, H), None, *codes(E, H, I), None, K, "silu", E)
w, ws = codes(48, H)
g = torch.randn(2 * I, H, generator=gen).to(B16).to(DEV).requires_grad_(True)
runs = []
for T in (3, 40, 300):
    x = torch.randn(T, H, generator=gen).to(B16).to(DEV)
    top = torch.rand(T, E, generator=gen).topk(K, dim=-1)
    weights, ids = torch.softmax(top.values, -1).to(DEV), top.indices.int().to(DEV)
    d = torch.randn(T, I, generator=gen).to(B16).to(DEV)
    out, dense = torch.empty(T, H, dtype=B16, device=DEV), torch.empty(T, 48, dtype=B16, device=DEV)
    def run(T=T, x=x, weights=weights, ids=ids, d=d, out=out, dense=dense):
        layer.apply(out, x, weights, ids)
        torch.ops._xpu_C.b200_int8_linear(dense, x, None, w, ws)
        y = gated_linear(x, g)
        return out, dense, y.detach(), torch.autograd.grad(y, g, d)[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    runs.append((run, x, graph, got))
for run, x, graph, got in runs:
    for _ in range(2):
        x.copy_(torch.randn(x.shape, generator=gen))
        graph.replay()
        got2 = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(got2, run()))
print("the same")
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "the same" in done.stdout, done.stderr[-2000:]
