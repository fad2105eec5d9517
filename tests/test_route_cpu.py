"""What the routing of experts and the layer on a given routing refuse (CPU only)."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import dsmoe._lib as L
    if not L.LIB_PATH.exists():
        from dsmoe import build
        build.build(verbose=False)
    return L.load()


def _dims(**kw):
    import dsmoe._lib as L
    base = dict(T=4, E=64, k=6, score=0, n_groups=8, topk_groups=4, group_top2=1, normalise=1, route_scale=1.0)
    d = L.RouteDims()
    for name, v in {**base, **kw}.items():
        assert hasattr(d, name)
        setattr(d, name, v)
    return d


def test_struct_matches_the_header():
    import dsmoe._lib as L
    assert ctypes.sizeof(L.RouteDims) == 9 * 4


@pytest.mark.parametrize("bad,text", [
    (dict(T=-1), b"T must"), (dict(T=2 ** 31 - 4096), b"too many"), (dict(E=0), b"E"), (dict(E=513), b"512"), (dict(k=0), b"k must"), (dict(k=17), b"16"),
    (dict(E=8, n_groups=1, topk_groups=1, k=9), b"k must"), (dict(n_groups=0), b"n_groups"), (dict(n_groups=7), b"divide"),
    (dict(n_groups=65), b"n_groups"), (dict(topk_groups=0), b"topk_groups"), (dict(topk_groups=9), b"topk_groups"),
    (dict(topk_groups=1, k=9), b"k must"), (dict(score=2), b"score"), (dict(score=-1), b"score")])
def test_refuses(lib, bad, text):
    import dsmoe._lib as L
    d = _dims(**bad)
    assert lib.dsmoe_route_experts_workspace_size(d) == 0
    for rc in (lib.dsmoe_route_experts(None, None, d, None, None, None, None, 0, None),
               lib.dsmoe_route_experts_bwd(None, None, None, d, None, None)):
        assert rc in (L.DSMOE_ERR_INVALID, L.DSMOE_ERR_UNSUPPORTED) and text in lib.dsmoe_last_error(), lib.dsmoe_last_error()


def test_pointers_and_workspace_are_checked(lib):
    import dsmoe._lib as L
    p, d = 4096, _dims()   # no device memory: refused before any use
    for bad in ((None, p, p), (p, None, p), (p, p, None)):
        assert lib.dsmoe_route_experts(bad[0], p, d, bad[1], bad[2], None, None, 0, None) == L.DSMOE_ERR_INVALID
    need = lib.dsmoe_route_experts_workspace_size(d)
    assert need >= 256
    assert lib.dsmoe_route_experts(p, p, d, p, p, p, p, need - 1, None) == L.DSMOE_ERR_WORKSPACE
    assert lib.dsmoe_route_experts(p, p, d, p, p, p, None, need, None) == L.DSMOE_ERR_WORKSPACE
    for i in range(4):
        a = [None if i == j else p for j in range(4)]
        assert lib.dsmoe_route_experts_bwd(a[0], a[1], a[2], d, a[3], None) == L.DSMOE_ERR_INVALID
    # nothing to do is no error, whatever the pointers
    assert lib.dsmoe_route_experts(None, None, _dims(T=0), None, None, None, None, 0, None) == 0
    assert lib.dsmoe_route_experts_bwd(None, None, None, _dims(T=0), None, None) == 0


def test_workspace_holds_the_largest_calls_counts(lib):
    small, large = (lib.dsmoe_route_experts_workspace_size(_dims(T=t, E=512, n_groups=1, topk_groups=1)) for t in (1, 2 ** 31 - 4097))
    assert 256 <= small < large < 1 << 34


def test_layer_on_a_routing_refuses(lib):
    import dsmoe._lib as L
    p, d = 4096, L.make_dims(4, 64, 4, 2, 32, 0, 0, torch.bfloat16, 1.0)
    pp = ctypes.cast((ctypes.c_void_p * 4)(p, p, p, p), ctypes.POINTER(ctypes.c_void_p))
    fwd = lambda idx, w: lib.dsmoe_moe_fwd_routed(p, idx, w, pp, pp, pp, None, None, None, d, 1, p, p, 0, None)
    assert fwd(None, p) == L.DSMOE_ERR_INVALID and fwd(p, None) == L.DSMOE_ERR_INVALID
    assert fwd(p, p) == L.DSMOE_ERR_WORKSPACE
    bwd = lambda dw: lib.dsmoe_moe_bwd_routed(p, pp, pp, pp, None, None, None, d, p, p, p, dw, pp, pp, pp, None, None, None,
                                              L.DSMOE_BF16, p, 0, None)
    assert bwd(None) == L.DSMOE_ERR_INVALID and bwd(p) == L.DSMOE_ERR_WORKSPACE


def test_no_cpu_implementation():
    from dsmoe import DeepSeekMoE
    from dsmoe.ops import gate_logits, route_experts, routed_moe_layer
    x = torch.zeros(3, 8)
    with pytest.raises(RuntimeError):
        route_experts(x, 2)
    with pytest.raises(RuntimeError):
        route_experts(x, 2, torch.zeros(8))
    with pytest.raises(RuntimeError):
        gate_logits(x, torch.zeros(4, 8))
    e = [torch.zeros(4, 8)] * 2
    with pytest.raises(RuntimeError):
        routed_moe_layer(x, torch.zeros(3, 1), torch.zeros(3, 1, dtype=torch.int64), e, [torch.zeros(8, 4)] * 2, e)
    m = DeepSeekMoE(dict(dim=8, n_routed_experts=4, n_shared_experts=0, moe_inter_dim=8, n_activated_experts=2, score_func="softmax"))
    with pytest.raises(RuntimeError):
        m(x)


def test_the_defaults_keep_the_fused_gate():
    from dsmoe import AuxLossFreeGate
    base = dict(dim=8, n_routed_experts=4, n_activated_experts=2)
    assert AuxLossFreeGate(base).fused
    for kw in (dict(score_func="softmax"), dict(n_expert_groups=2), dict(norm_topk_prob=False)):
        assert not AuxLossFreeGate({**base, **kw}).fused
