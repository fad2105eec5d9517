"""The layer on a given routing (ops.routed_moe_layer, the module with softmax scores or groups), and the paged attention,
the routing and the experts run as a model runs them, against float64.

Bounds.  fp32: 1e-5 of a result's largest value (sums of at most a few hundred products of 2^-24 each, three deep).
bf16: relative L2 error of roundings x 2^-8, a result behind at most 5 roundings in a chain (g and u, dh, dg and du, the
slots' dx, the sum); products with matrices that do not depend on the errors keep the relative L2 error."""
import pytest
import torch
import torch.nn.functional as F

from oracle.paged_ref import append_ref, attend_ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16 = 5 * 2.0 ** -8


def _experts(n, D, I, g, dtype):
    rnd = lambda *s: (torch.randn(*s, generator=g) * s[-1] ** -0.5).to(dtype)
    return [rnd(I, D) for _ in range(n)], [rnd(D, I) for _ in range(n)], [rnd(I, D) for _ in range(n)]


def _layer64(x, weights, idx, w1, w2, w3, s1, s2, s3):
    """The layer in float64; ids outside and repeated ids of a token count for nothing."""
    y = torch.zeros_like(x)
    ffn = lambda r, a, b, c: (F.silu(r @ a.T) * (r @ c.T)) @ b.T
    for e in range(len(w1)):
        first = (idx == e) & ((idx == e).cumsum(1) == 1)
        for t, j in first.nonzero().tolist():
            y[t] = y[t] + weights[t, j] * ffn(x[t:t + 1], w1[e], w2[e], w3[e])[0]
    for a, b, c in zip(s1, s2, s3):
        y = y + ffn(x, a, b, c)
    return y


def _close(got, want, dtype, what):
    got, want = got.detach().double().cpu(), want.detach().double()
    assert torch.isfinite(got).all(), what
    if dtype == torch.float32:
        assert (got - want).abs().max() <= 1e-5 * max(want.abs().max(), 1e-30), what
    else:
        assert (got - want).norm() <= BF16 * max(want.norm(), 1e-30), what


def _both(x, weights, idx, experts, dy, dtype):
    """((name, on the GPU, in float64)) of the output and every gradient."""
    from dsmoe import ops
    leaf = lambda t, f: f(t.detach()).requires_grad_(True)
    runs = []
    for f, layer in ((lambda t: t.to(DEV), ops.routed_moe_layer), (lambda t: t.double(), _layer64)):
        xl, wl, el = leaf(x, f), leaf(weights, f), [[leaf(t, f) for t in ws] for ws in experts]
        y = layer(xl, wl, idx.to(xl.device), *el)
        y.backward(f(dy))
        flat = [(f"{n}[{i}]", t) for n, ws in zip(("w1", "w2", "w3", "s1", "s2", "s3"), el) for i, t in enumerate(ws)]
        grads = [("y", y), ("dx", xl.grad), ("dweights", wl.grad)]
        runs.append(grads + [(n, t.grad if t.grad is not None else torch.zeros_like(t)) for n, t in flat])
    return [(n, a, b) for (n, a), (_, b) in zip(*runs)]


def _inputs(T, D, E, k, I, S, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x, dy = (torch.randn(T, D, generator=g).to(dtype) for _ in range(2))
    idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]) if T else torch.zeros(0, k, dtype=torch.int64)
    weights = torch.rand(T, k, generator=g)
    return x, weights, idx, (*_experts(E, D, I, g, dtype), *_experts(S, D, I, g, dtype)), dy


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,D,E,k,I,S", [(1, 64, 4, 2, 32, 1), (37, 64, 16, 4, 48, 0), (130, 128, 8, 8, 64, 2),
                                         (65, 72, 20, 16, 40, 1), (300, 64, 3, 1, 64, 1)])
def test_against_the_definition(T, D, E, k, I, S, dtype):
    for name, got, want in _both(*_inputs(T, D, E, k, I, S, dtype, seed=T), dtype):
        _close(got, want, dtype, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ids_that_are_not_there_or_come_twice(dtype):
    x, weights, idx, experts, dy = _inputs(40, 64, 6, 4, 32, 1, dtype, seed=3)
    idx[0] = -1                                                            # a token without experts
    idx[1] = torch.tensor([5, 5, 5, 5])
    idx[2] = torch.tensor([6, 0, -7, 0])
    idx[3] = torch.tensor([2 ** 32 + 1, 2, -2 ** 40, 2 ** 31])              # outside, whatever their low 32 bits are
    idx[4] = torch.tensor([1, 0, 1, 0])
    idx[39, 3] = idx[39, 0]
    weights[0] = float("nan")                                              # of ids that count for nothing
    weights[1, 1:] = float("inf")
    dead = torch.zeros(40, 4, dtype=torch.bool)
    dead[0], dead[1, 1:], dead[2, [0, 2, 3]], dead[3, [0, 2, 3]], dead[4, 2:], dead[39, 3] = (True,) * 6
    for name, got, want in _both(x, weights, idx, experts, dy, dtype):
        if name == "dweights":
            assert (got.cpu()[dead] == 0).all()
        _close(got, want, dtype, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_gates_own_routing_gives_the_fused_layer(dtype):
    """y and the experts' gradients bit for bit, from the weights in the layer's workspace (the layer's gate may sum its
    logits in parts, gate_forward's does not)."""
    from dsmoe import _lib, moe_layer, ops
    x, _, _, experts, dy = _inputs(200, 128, 16, 4, 64, 1, dtype, seed=5)
    gw, gb = torch.randn(16, 128, device=DEV) * 0.1, torch.zeros(16, device=DEV)
    ex = [[t.to(DEV).requires_grad_(True) for t in ws] for ws in experts]
    leaves = [t for ws in ex for t in ws]
    x, dy = x.to(DEV).requires_grad_(True), dy.to(DEV)
    y, idx64, _, _ = moe_layer(x, gw, gb, *ex, k=4, route_scale=1.5)
    want = torch.autograd.grad(y, leaves, dy)
    d = _lib.make_dims(200, 128, 16, 4, 64, 1, 64, dtype, 1.5)
    ws = torch.ops.dsmoe.moe_fwd(x.detach(), gw, gb, [t.detach() for t in leaves], [], 16, 1, 4, 64, 64, 1.5, True)[4]
    at = _lib.load().dsmoe_moe_fwd_workspace_offset(d, 1, _lib.WS_WEIGHTS)
    w = ws[at:at + 200 * 4 * 4].view(torch.float32).view(200, 4).clone().requires_grad_(True)
    z = ops.routed_moe_layer(x, w, idx64, *ex)
    got = torch.autograd.grad(z, leaves, dy)
    assert torch.equal(y, z) and all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        assert torch.equal(ops.routed_moe_layer(x, w, idx64.int(), *ex), z)


def test_no_tokens():
    from dsmoe import ops
    x, weights, idx, experts, dy = _inputs(0, 64, 4, 2, 32, 1, torch.bfloat16, seed=1)
    ex = [[t.to(DEV).requires_grad_(True) for t in ws] for ws in experts]
    x, weights = x.to(DEV).requires_grad_(True), weights.to(DEV).requires_grad_(True)
    y = ops.routed_moe_layer(x, weights, idx.to(DEV), *ex)
    y.backward(dy.to(DEV))
    assert y.shape == (0, 64) and weights.grad.shape == (0, 2) and all((t.grad == 0).all() for ws in ex for t in ws)
    m = _module(GATES[2])
    e = torch.zeros(2, 0, 64, device=DEV, requires_grad=True)
    m(e).sum().backward()
    assert e.grad.shape == e.shape and (m.gate.weight.grad == 0).all() and (m._last_counts == 0).all()


CONFIG = dict(dim=64, n_routed_experts=16, n_shared_experts=1, moe_inter_dim=48, n_activated_experts=4)
GATES = [dict(score_func="softmax"), dict(n_expert_groups=4, n_limited_groups=2, route_scale=2.5),
         dict(score_func="softmax", n_expert_groups=8, n_limited_groups=3, group_score="max", norm_topk_prob=False, route_scale=4.0)]


def _module(gate, dtype=torch.float32):
    from dsmoe import DeepSeekMoE
    torch.manual_seed(0)
    m = DeepSeekMoE(dict(CONFIG, **gate))
    with torch.no_grad():
        for n, p in m.named_parameters():
            p.copy_(torch.randn(p.shape) * p.shape[-1] ** -0.5)
        m.gate.bias.copy_(torch.randn(16) * 0.05)
    return m.to(DEV).to(dtype)


def _module64(m, x, idx, gate):
    """The module's output in float64 from double leaves, on the experts that it chose; (y, leaves by name)."""
    p = {n: t.detach().double().cpu().requires_grad_(True) for n, t in m.named_parameters()}
    logits = x @ p["gate.weight"].T
    s = torch.softmax(logits, -1) if gate.get("score_func") == "softmax" else torch.sigmoid(logits)
    w = s.gather(1, idx)
    if gate.get("norm_topk_prob", True):
        w = w / w.sum(1, keepdim=True)
    w = w * gate.get("route_scale", 1.0)
    ws = [[p[f"{kind}.{e}.{n}.weight"] for e in range(c)] for kind, c in (("experts", 16), ("shared_experts", 1))
          for n in ("w1", "w2", "w3")]
    return _layer64(x, w, idx, *ws), p, (s + m.gate.bias.double().cpu()).detach()


@pytest.mark.parametrize("gate", GATES)
def test_module(gate):
    m = _module(gate)
    g = torch.Generator().manual_seed(2)
    x, dy = torch.randn(3, 41, 64, generator=g), torch.randn(3, 41, 64, generator=g)
    xl = x.to(DEV).requires_grad_(True)
    y = m(xl)
    y.backward(dy.to(DEV))
    idx = m._last_indices.cpu()
    x64 = x.double().reshape(-1, 64).requires_grad_(True)
    y64, p64, scores = _module64(m, x64, idx, gate)
    y64.backward(dy.double().reshape(-1, 64))
    _close(y.reshape(-1, 64), y64, torch.float32, "y")
    _close(xl.grad.reshape(-1, 64), x64.grad, torch.float32, "dx")
    for n, p in m.named_parameters():
        _close(p.grad, p64[n].grad if p64[n].grad is not None else torch.zeros_like(p64[n]), torch.float32, n)
    # the choice: of the groups kept, the best
    G, keep = gate.get("n_expert_groups", 1), gate.get("n_limited_groups", gate.get("n_expert_groups", 1))
    by = scores.view(-1, G, 16 // G)
    best = by.amax(2) if gate.get("group_score") == "max" else by.topk(min(2, 16 // G), 2).values.sum(2)
    kept = torch.zeros_like(best).scatter(1, best.topk(keep, 1).indices, 1.0).bool()
    want = by.masked_fill(~kept[..., None], float("-inf")).flatten(1).topk(4, 1).indices
    assert torch.equal(want.sort(1).values, idx.sort(1).values)
    assert torch.equal(m._last_counts.cpu().long(), torch.bincount(idx.flatten(), minlength=16))
    assert m.get_load_balance_loss().isfinite() if hasattr(m, "get_load_balance_loss") else True


def test_module_under_autocast_and_without_gradients():
    """fp32 parameters: their gradients come in fp32 from the bf16 products; without gradients the same output."""
    gate = GATES[1]
    m = _module(gate)
    g = torch.Generator().manual_seed(3)
    x, dy = torch.randn(70, 64, generator=g).bfloat16(), torch.randn(70, 64, generator=g).bfloat16()
    xl = x.to(DEV).requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(xl)
    y.backward(dy.to(DEV))
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        z = m(x.to(DEV))
    assert torch.equal(y, z)
    x64 = x.double().requires_grad_(True)
    y64, p64, _ = _module64(m, x64, m._last_indices.cpu(), gate)
    y64.backward(dy.double())
    # one more rounding than the layer's: the experts' weights to bf16
    for name, got, want in [("y", y, y64), ("dx", xl.grad, x64.grad)] + [(n, p.grad, p64[n].grad) for n, p in m.named_parameters()]:
        want = torch.zeros_like(got.double().cpu()) if want is None else want
        assert got.dtype == (torch.float32 if "weight" in name else torch.bfloat16)
        assert (got.double().cpu() - want).norm() <= (BF16 + 2.0 ** -8) * max(want.norm(), 1e-30), name


def test_module_captured():
    """Forward and backward in a graph, replayed on other inputs between eager steps."""
    m = _module(GATES[1], torch.bfloat16)
    m.gate.weight.data = m.gate.weight.data.float()
    x, dy = torch.randn(50, 64, device=DEV).bfloat16().requires_grad_(True), torch.randn(50, 64, device=DEV).bfloat16()
    leaves = [x, *m.parameters()]

    def step():
        y = m(x)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(50, 64, generator=torch.Generator().manual_seed(i)))
            dy.normal_()
        graph.replay()
        got = [o.clone() for o in out]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_module_compiled():
    """The operators break the graph; outputs and gradients are the eager module's."""
    m = _module(GATES[0])
    f = torch.compile(m, backend="eager")
    x = torch.randn(20, 64, device=DEV, requires_grad=True)
    y, z = m(x), f(x)
    assert torch.equal(y, z)
    a = torch.autograd.grad(y.square().sum(), [x, *m.parameters()])
    b = torch.autograd.grad(z.square().sum(), [x, *m.parameters()])
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_refusals():
    from dsmoe import ops
    x, weights, idx, experts, _ = _inputs(5, 64, 4, 2, 32, 1, torch.bfloat16, seed=7)
    x, weights, idx, ex = x.to(DEV), weights.to(DEV), idx.to(DEV), [[t.to(DEV) for t in ws] for ws in experts]
    for w, i in ((weights[:4], idx), (weights, idx[:, :1]), (weights, idx.float()), (weights[0], idx[0])):
        with pytest.raises(ValueError, match="weights and idx"):
            ops.routed_moe_layer(x, w, i, *ex)
    with pytest.raises(ValueError, match="k <="):
        ops.routed_moe_layer(x, weights.repeat(1, 3), idx.repeat(1, 3), *ex)
    with pytest.raises(ValueError, match="k <="):
        ops.routed_moe_layer(x, weights[:, :0], idx[:, :0], *ex)
    with pytest.raises(ValueError, match="master"):
        ops.routed_moe_layer(x, weights, idx, *ex, master_weights=[t for ws in ex for t in ws])
    with pytest.raises(ValueError, match="w1|expert"):
        ops.routed_moe_layer(x, weights, idx, ex[0][:3], *ex[1:])
    with pytest.raises(ValueError, match="gate_logits"):
        ops.gate_logits(x, torch.zeros(4, 63, device=DEV))


# ---------------------------------------------------------------------------- a decoder layer as it serves
def test_append_attend_route_experts():
    """Chunks of two prompts, then single tokens: append (with the norm) -> attention over the pages -> output projection ->
    grouped routing -> experts; every stage against float64 on the inputs that it had."""
    from dsmoe import DeepSeekMoE
    from dsmoe.mla import mla_attention_paged, mla_cache_append
    H, R, Dn, Dr, Dv, D, page = 4, 32, 16, 16, 16, 64, 8
    g = torch.Generator().manual_seed(11)
    rnd = lambda *s: (torch.randn(*s, generator=g) * s[-1] ** -0.5).to(DEV, torch.bfloat16)
    wq, wc, w_k, w_v, wo, nw = rnd(H * (Dn + Dr), D), rnd(R + Dr, D), rnd(H, Dn, R), rnd(H, Dv, R), rnd(D, H * Dv), torch.ones(R, device=DEV)
    gate = GATES[1]
    m = _module(gate, torch.bfloat16)
    m.gate.weight.data = m.gate.weight.data.float()
    kv, pe = torch.zeros(12, page, R, device=DEV, dtype=torch.bfloat16), torch.zeros(12, page, Dr, device=DEV, dtype=torch.bfloat16)
    table = torch.randperm(12, generator=g)[:12].view(2, 6).int().to(DEV)
    lens = [0, 0]
    for new in ([20, 7], [13, 1], [1, 1], [1, 30], [1, 1]):
        lens = [n + a for n, a in zip(lens, new)]
        x = torch.randn(sum(new), D, generator=g).to(DEV, torch.bfloat16)
        kv_lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        off = torch.tensor([0, *new]).cumsum(0).int().to(DEV)
        with torch.no_grad():
            q, c = (x @ wq.T).view(-1, H, Dn + Dr), x @ wc.T
            before = (kv.cpu(), pe.cpu())
            mla_cache_append(c[:, :R], c[:, R:], kv, pe, table, kv_lens, off, norm_weight=nw)
            a = mla_attention_paged(q[..., :Dn], q[..., Dn:], kv, pe, table, kv_lens, off, w_k, w_v, (Dn + Dr) ** -0.5,
                                    max_q=max(new), max_kv=max(lens))
            h = a.flatten(1) @ wo.T
            y = m(h)
        host = [t.cpu() for t in (table, kv_lens, off)]
        kv64, pe64, _ = append_ref(c[:, :R].cpu(), c[:, R:].cpu(), *before, *host, nw.cpu())
        assert ((kv.cpu().double() - kv64).abs() <= 2.0 ** -8 * kv64.abs() + 1e-6).all() and torch.equal(pe.cpu().double(), pe64)
        a64, spread, _ = attend_ref(q[..., :Dn].cpu(), q[..., Dn:].cpu(), kv.cpu(), pe.cpu(), *host, w_k.cpu(), w_v.cpu(), (Dn + Dr) ** -0.5)
        assert ((a.cpu().double() - a64).abs() <= 2.0 ** -8 * a64.abs() + 2.0 ** -6 * spread).all()
        y64, _, _ = _module64(m, h.cpu().double(), m._last_indices.cpu(), gate)
        _close(y, y64, torch.bfloat16, "y")
    assert lens == [36, 40]
