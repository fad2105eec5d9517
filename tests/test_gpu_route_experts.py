"""dsmoe.ops.route_experts (csrc/route_experts.hip) against its definition in numpy, in 64 bits.

idx and counts are equal; scores are 64-bit values rounded to fp32 once (an error of 2^-24 of them), a sum of k <= 16
of them and two more operations add at most (k + 1) 2^-24: weights within (k + 4) 2^-23 of themselves.  Gradients in fp32
from fp32 scores: every term of the formula is off by at most (E / 8 + k + 24) 2^-24 of its size (sums over lanes and slots,
exp within 2^-22, the steps of the formula), so a value by that of its sum of absolute terms."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TINY = 1e-10


def _scores(x, score):
    with np.errstate(over="ignore", invalid="ignore"):
        if score == "sigmoid":
            return 1.0 / (1.0 + np.exp(-x))
        e = np.exp(x - x.max(1, keepdims=True))
        return e / e.sum(1, keepdims=True)


def _ref(logits, k, bias, score, G, keep, top2, normalise, scale):
    """Indices, float64 weights and counts, one token at a time."""
    T, E = logits.shape
    full = _scores(logits.astype(np.float64), score)
    c = full.astype(np.float32)
    with np.errstate(invalid="ignore"):
        if bias is not None:
            c = c + bias.astype(np.float32)
        key = np.where(np.isnan(c), -np.inf, c)
        nan = np.isnan(c)
        gs = E // G
        idx = np.zeros((T, k), np.int64)
        for t in range(T):
            order = lambda ids: sorted(ids, key=lambda e: (nan[t, e], -key[t, e], e))
            groups = [order(range(g * gs, g * gs + gs)) for g in range(G)]
            gscore = [c[t, o[0]] + c[t, o[1]] if top2 and gs > 1 else c[t, o[0]] for o in groups]
            best = sorted(range(G), key=lambda g: (np.isnan(gscore[g]), -np.nan_to_num(gscore[g], nan=0.0, posinf=np.inf, neginf=-np.inf), g))[:keep]
            idx[t] = order([e for g in best for e in groups[g]])[:k]
    w = np.take_along_axis(full, idx, 1)
    if normalise:
        w = w / np.maximum(w.sum(1, keepdims=True), TINY)
    return idx, w * scale, np.bincount(idx.reshape(-1), minlength=E)


def _grad(logits, idx, dw, score, normalise, scale):
    """The gradient in float64 and the sum of its absolute terms."""
    full = _scores(logits.astype(np.float64), score)
    s = np.take_along_axis(full, idx, 1)
    g, ga = dw * scale, np.abs(dw * scale)
    if normalise:
        S = s.sum(1, keepdims=True)
        held = S < TINY
        S = np.maximum(S, TINY)
        g, ga = (g / S - np.where(held, 0, (g * s).sum(1, keepdims=True) / S ** 2),
                 ga / S + np.where(held, 0, (ga * s).sum(1, keepdims=True) / S ** 2))
    ds, dsa = np.zeros_like(full), np.zeros_like(full)
    np.put_along_axis(ds, idx, g, 1)
    np.put_along_axis(dsa, idx, ga, 1)
    if score == "sigmoid":
        return ds * full * (1 - full), dsa * full
    return full * (ds - (g * s).sum(1, keepdims=True)), full * (dsa + (ga * s).sum(1, keepdims=True))


def _inputs(T, E, seed, bias=True, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(T, E, generator=g) * std, torch.randn(E, generator=g) * 0.05 if bias else None


def _check(logits, bias, k, score="sigmoid", G=1, keep=1, group_score="top2", normalise=True, scale=1.5, grad=True):
    from dsmoe.ops import route_experts
    T, E = logits.shape
    idx, w, counts = _ref(logits.numpy(), k, None if bias is None else bias.numpy(), score, G, keep, group_score == "top2",
                          normalise, scale)
    x = logits.to(DEV).requires_grad_(grad)
    gw, gi, gc = route_experts(x, k, None if bias is None else bias.to(DEV), score=score, n_groups=G, topk_groups=keep,
                               group_score=group_score, normalise=normalise, route_scale=scale)
    assert gw.dtype == torch.float32 and gi.dtype == gc.dtype == torch.int32
    assert np.array_equal(gi.cpu().numpy(), idx) and np.array_equal(gc.cpu().numpy(), counts)
    got = gw.detach().cpu().double().numpy()
    assert (np.abs(got - w) <= (k + 4) * 2.0 ** -23 * np.abs(w) + 1e-37).all()
    if not grad:
        return
    dw = torch.randn(T, k, generator=torch.Generator().manual_seed(1))
    d, = torch.autograd.grad(gw, x, dw.to(DEV))
    ref, size = _grad(logits.numpy(), idx, dw.double().numpy(), score, normalise, scale)
    err = np.abs(d.cpu().double().numpy() - ref)
    assert (err <= size * (E / 8 + k + 24) * 2.0 ** -24 + 1e-37).all()


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("T,E,k,G,keep", [
    (1, 1, 1, 1, 1), (1, 4, 2, 1, 1), (5, 16, 4, 4, 2), (65, 17, 3, 1, 1), (7, 32, 16, 2, 2), (130, 64, 6, 8, 3),
    (64, 64, 6, 1, 1), (33, 60, 8, 5, 3), (19, 63, 2, 7, 1), (3, 128, 8, 64, 40), (21, 160, 6, 8, 3), (300, 256, 8, 8, 4),
    (18, 250, 16, 2, 1), (9, 257, 4, 1, 1), (10, 512, 16, 16, 2), (11, 384, 7, 3, 3), (40, 20, 4, 1, 1), (8, 8, 3, 8, 3)])
def test_against_the_definition(T, E, k, G, keep, score, normalise):
    _check(*_inputs(T, E, seed=E + k, bias=(T + E) % 3 != 0), k, score, G, keep, "top2" if E % 2 == 0 else "max", normalise)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_largest_group_score(score):
    _check(*_inputs(50, 64, seed=2), 6, score, 8, 2, "max")


@pytest.mark.parametrize("E,G,keep,k", [(16, 1, 1, 4), (64, 8, 3, 6), (256, 8, 4, 8), (320, 4, 2, 8), (30, 5, 2, 3)])
def test_ties_go_to_the_lower_id(E, G, keep, k):
    """Few distinct values: groups and experts tie everywhere."""
    g = torch.Generator().manual_seed(E)
    x = torch.randint(-2, 2, (200, E), generator=g).float()
    for score in ("sigmoid", "softmax"):
        _check(x, None, k, score, G, keep)
        _check(x, torch.randint(0, 2, (E,), generator=g).float() * 0.25, k, score, G, keep, "max")
    _check(torch.zeros(9, E), None, k, "softmax", G, keep)
    # neighbouring fp32 scores: the next value up, and scores that round to one value
    x = torch.zeros(64, E) + torch.arange(E)[torch.randperm(E, generator=g)] * 2.0 ** -24
    _check(x, None, k, "sigmoid", G, keep)
    _check(x * 8, None, k, "sigmoid", G, keep)
    _check(x * 64, None, k, "softmax", G, keep)


def test_extreme_logits():
    """Saturated and vanishing scores, sums under the floor, -infinity for experts that are switched off."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(40, 64, generator=g) * 40
    x[0] = -200.0
    x[1] = 200.0
    x[2] = -60.0
    x[3, ::2] = float("-inf")
    x[4, 5:] = float("-inf")
    x[5, 7] = 3e38
    for score in ("sigmoid", "softmax"):
        for normalise in (True, False):
            _check(x, None, 4, score, 8, 4, "max", normalise)
    bias = torch.zeros(64)
    bias[::3] = float("-inf")
    bias[5] = float("inf")
    bias[6] = -torch.finfo(torch.float32).max
    _check(x, bias, 4, "sigmoid", 1, 1)


def test_nan_comes_last():
    x, bias = _inputs(30, 64, seed=6)
    x[::2, 3::7] = float("nan")
    x[7] = float("nan")
    from dsmoe.ops import route_experts
    for G, keep in ((1, 1), (8, 3)):
        idx, _, counts = _ref(x.numpy(), 6, bias.numpy(), "sigmoid", G, keep, True, True, 1.0)
        _, gi, gc = route_experts(x.to(DEV), 6, bias.to(DEV), n_groups=G, topk_groups=keep)
        assert np.array_equal(gi.cpu().numpy(), idx) and np.array_equal(gc.cpu().numpy(), counts)
    idx = _ref(x.numpy(), 6, bias.numpy(), "softmax", 1, 1, True, True, 1.0)[0]
    assert np.array_equal(route_experts(x.to(DEV), 6, bias.to(DEV), score="softmax")[1].cpu().numpy(), idx)


def test_defaults_are_route_from_logits():
    from dsmoe.ops import route_experts, route_from_logits
    for T, E, k in ((1, 4, 2), (700, 64, 6), (129, 16, 4), (50, 256, 8), (40, 200, 16)):
        x, bias = _inputs(T, E, seed=T)
        old = route_from_logits(x.to(DEV), bias.to(DEV), k, 2.5)
        w, idx, counts = route_experts(x.to(DEV), k, bias.to(DEV), route_scale=2.5)
        assert torch.equal(w, old["weights"]) and torch.equal(idx, old["idx"]) and torch.equal(counts, old["counts"])


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("normalise", [True, False])
def test_gradient_against_differences(score, normalise):
    """Central differences of the float64 definition with the choice held: steps of 2^-17, whose own error is under 2^-24 of the
    largest third derivative and of the rounding 2^-53 / 2^-17."""
    x, bias = _inputs(6, 24, seed=8)
    from dsmoe.ops import route_experts
    g = x.to(DEV).requires_grad_(True)
    w, idx, _ = route_experts(g, 4, bias.to(DEV), score=score, n_groups=4, topk_groups=2, normalise=normalise, route_scale=1.3)
    dw = torch.randn(6, 4, generator=torch.Generator().manual_seed(2))
    d, = torch.autograd.grad(w, g, dw.to(DEV))
    ids, h = idx.cpu().numpy().astype(np.int64), 2.0 ** -17

    def f(z):
        s = np.take_along_axis(_scores(z, score), ids, 1)
        s = s / np.maximum(s.sum(1, keepdims=True), TINY) if normalise else s
        return (s * 1.3 * dw.double().numpy()).sum(1)
    z = x.double().numpy()
    for e in range(24):
        up, dn = z.copy(), z.copy()
        up[:, e] += h
        dn[:, e] -= h
        assert np.abs((f(up) - f(dn)) / (2 * h) - d[:, e].cpu().double().numpy()).max() < 5e-6


def test_strides_types_and_an_empty_call():
    from dsmoe.ops import route_experts
    x, bias = _inputs(40, 64, seed=9)
    want = route_experts(x.to(DEV), 6, bias.to(DEV), n_groups=8, topk_groups=4)
    wide = torch.full((40, 80), float("nan"), device=DEV)
    wide[:, 9:73] = x.to(DEV)
    for y in (wide[:, 9:73], x.to(DEV).T.contiguous().T):
        got = route_experts(y, 6, bias.to(DEV).double(), n_groups=8, topk_groups=4)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    b16 = x.to(DEV).bfloat16().requires_grad_(True)
    w, idx, _ = route_experts(b16, 6, bias.to(DEV))
    f = b16.detach().float().requires_grad_(True)
    w2, idx2, _ = route_experts(f, 6, bias.to(DEV))
    assert torch.equal(w, w2) and torch.equal(idx, idx2)
    g, = torch.autograd.grad(w.sum() + (w * w).sum(), b16)
    g2, = torch.autograd.grad(w2.sum() + (w2 * w2).sum(), f)
    assert g.dtype == torch.bfloat16 and torch.equal(g, g2.bfloat16())
    # rows whose start is not 16-byte aligned, contiguous all the same
    odd = torch.empty(40 * 64 + 1, device=DEV)[1:].view(40, 64)
    odd.copy_(x)
    assert all(torch.equal(a, b) for a, b in zip(route_experts(odd, 6, bias.to(DEV), n_groups=8, topk_groups=4), want))
    w, idx, counts = route_experts(x[:0].to(DEV).requires_grad_(True), 6, bias.to(DEV))
    assert w.shape == idx.shape == (0, 6) and (counts == 0).all()
    assert torch.autograd.grad(w.sum(), w, allow_unused=True)[0].shape == (0, 6)


def test_gradient_reaches_a_shared_and_broadcast_input():
    """Two calls on one leaf add up; an expanded gradient is read as it stands."""
    from dsmoe.ops import route_experts
    x, bias = _inputs(33, 64, seed=10)
    g = x.to(DEV).requires_grad_(True)
    a = route_experts(g, 6, bias.to(DEV))[0]
    b = route_experts(g, 4, None, score="softmax", normalise=False)[0]
    both, = torch.autograd.grad([a, b], g, [torch.ones((), device=DEV).expand(33, 6), torch.ones((), device=DEV).expand(33, 4)])
    one = [torch.autograd.grad(w, g, torch.ones_like(w))[0]
           for w in (route_experts(g, 6, bias.to(DEV))[0], route_experts(g, 4, None, score="softmax", normalise=False)[0])]
    assert torch.equal(both, one[0] + one[1])
    row = torch.randn(1, 64, device=DEV, requires_grad=True)
    w = route_experts(row.expand(50, 64), 6)[0]
    d, = torch.autograd.grad(w[:, 0].sum(), row)
    r = route_experts(row, 6)[0]
    d1, = torch.autograd.grad(r[:, 0].sum(), row)
    assert torch.allclose(d, 50 * d1, rtol=1e-5, atol=1e-7)


def test_captured_forward_and_backward():
    from dsmoe.ops import route_experts
    x, bias = _inputs(300, 64, seed=11)
    leaf, b = x.to(DEV).requires_grad_(True), bias.to(DEV)
    dw = torch.randn(300, 6, device=DEV)

    def step():
        w, idx, counts = route_experts(leaf, 6, b, n_groups=8, topk_groups=4)
        return w.detach(), idx, counts, torch.autograd.grad(w, leaf, dw)[0]
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
            leaf.copy_(torch.randn(300, 64, generator=torch.Generator().manual_seed(i)))
            dw.normal_()
        graph.replay()
        got = [o.clone() for o in out]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_groups_across_lanes_with_as_many_tokens_as_a_block_holds():
    """64 tokens' keys and group scores in a block's shared memory, more than 64 KiB of it."""
    x, bias = _inputs(64, 250, seed=17)
    _check(x, bias, 8, G=10, keep=4)


def test_compiled_with_a_graph_break():
    from dsmoe.ops import route_experts
    x, bias = _inputs(40, 64, seed=18)
    b = bias.to(DEV)

    def f(x):
        w, idx, counts = route_experts(x * 2, 6, b, n_groups=8, topk_groups=3)
        return w.square().sum(), idx
    grads = []
    for fn in (f, torch.compile(f, backend="eager")):
        leaf = x.to(DEV).requires_grad_(True)
        y, idx = fn(leaf)
        y.backward()
        grads.append((y.detach(), idx, leaf.grad))
    assert all(torch.equal(p, q) for p, q in zip(*grads))


def test_refusals():
    from dsmoe.ops import route_experts
    x, bias = _inputs(4, 64, seed=12)
    g, b = x.to(DEV), bias.to(DEV)
    for kw, text in ((dict(k=0), "k must"), (dict(k=17), "16"), (dict(k=65), "k must"), (dict(n_groups=7), "divide"),
                     (dict(n_groups=0), "n_groups"), (dict(n_groups=8, topk_groups=9), "topk_groups"),
                     (dict(n_groups=8, topk_groups=0), "topk_groups"), (dict(k=9, n_groups=8, topk_groups=1), "k must"),
                     (dict(score="relu"), "score"), (dict(group_score="mean"), "group_score")):
        with pytest.raises(ValueError, match=text):
            route_experts(g, **{"k": 6, "bias": b, **kw})
    with pytest.raises(ValueError, match="bias"):
        route_experts(g, 6, b[:5])
    with pytest.raises(ValueError, match="logits"):
        route_experts(g[0], 6)
    with pytest.raises(ValueError, match="logits"):
        route_experts(g.int(), 6)
    with pytest.raises(ValueError, match="512"):
        route_experts(torch.zeros(2, 513, device=DEV), 6)
    torch.cuda.synchronize()
