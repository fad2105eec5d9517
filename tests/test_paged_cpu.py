"""What the paged latent cache refuses, and its oracle against the contiguous attention's (CPU only)."""
import ctypes

import pytest
import torch

from oracle.mla_ref import mla_attention_oracle
from oracle.paged_ref import append_ref, attend_ref


@pytest.fixture(scope="module")
def lib():
    import dsmoe._lib as L
    if not L.LIB_PATH.exists():
        from dsmoe import build
        build.build(verbose=False)
    return L.load()


def _dims(**kw):
    import dsmoe._lib as L
    d = L.MlaPagedDims()
    base = dict(T=4, B=2, H=12, R=192, D_nope=48, D_rope=24, D_v=64, pages=8, page_size=16, table_width=3, max_q=4,
                max_kv=48, softmax_scale=0.1)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return d


def test_struct_matches_the_header():
    import dsmoe._lib as L
    assert ctypes.sizeof(L.MlaPagedDims) == 12 * 4 + 9 * 8 + 8


@pytest.mark.parametrize("bad,text", [
    (dict(T=-1), b"negative"), (dict(B=-1), b"negative"), (dict(H=0), b"H must"), (dict(R=0), b"R and D_rope"),
    (dict(R=257), b"R and D_rope"), (dict(D_rope=0), b"R and D_rope"), (dict(D_nope=0), b"D_nope"), (dict(D_v=257), b"D_v"),
    (dict(D_nope=200, D_rope=57), b"D_nope + D_rope"), (dict(pages=0), b"pages"), (dict(page_size=0), b"pages"),
    (dict(table_width=-1), b"pages"), (dict(kv_page_stride=-1), b"stride"), (dict(T=1 << 22), b"2^24"), (dict(H=65536), b"heads"),
    (dict(max_q=-1), b"max_q")])
def test_attention_refuses(lib, bad, text):
    import dsmoe._lib as L
    d = _dims(**bad)
    assert lib.dsmoe_mla_attn_paged_workspace_size(d) == 0
    rc = lib.dsmoe_mla_attn_paged(None, None, None, None, None, None, None, None, 0, None, 0, d, None, None, 0, None)
    assert rc in (L.DSMOE_ERR_INVALID, L.DSMOE_ERR_UNSUPPORTED) and text in lib.dsmoe_last_error()


def test_too_many_sequences(lib):
    import dsmoe._lib as L
    for call in (lambda d: lib.dsmoe_mla_attn_paged(*[None] * 8, 0, None, 0, d, None, None, 0, None),
                 lambda d: lib.dsmoe_mla_cache_append(None, 0, None, 0, 1, None, 1e-6, *[None] * 5, d, None)):
        assert call(_dims(B=1 << 24)) == L.DSMOE_ERR_UNSUPPORTED and b"2^24" in lib.dsmoe_last_error()
    # K and V are not built where the attention's grid had no room: the workspace is the latent rows' alone
    few, many = (lib.dsmoe_mla_attn_paged_workspace_size(_dims(T=256, H=16, B=b, max_q=256, max_kv=256)) for b in (1 << 20, (1 << 24) - 1))
    assert 0 < few and 0 < many


def test_pointers_workspace_and_strides_are_checked(lib):
    import dsmoe._lib as L
    d = _dims()
    rc = lib.dsmoe_mla_attn_paged(None, None, None, None, None, None, None, None, 0, None, 0, d, None, None, 0, None)
    assert rc == L.DSMOE_ERR_INVALID and b"NULL" in lib.dsmoe_last_error()
    p = 4096   # no device memory: refused before any use
    call = lambda d, ws=p, n=1 << 40, wk=0: lib.dsmoe_mla_attn_paged(p, p, p, p, p, p, p, p, wk, p, 0, d, p, ws, n, None)
    assert call(d, n=lib.dsmoe_mla_attn_paged_workspace_size(d) - 256) == L.DSMOE_ERR_WORKSPACE
    assert call(d, ws=p + 8) == L.DSMOE_ERR_INVALID and b"aligned" in lib.dsmoe_last_error()
    assert call(d, wk=-1) == L.DSMOE_ERR_INVALID and b"stride" in lib.dsmoe_last_error()
    assert call(_dims(qn_token_stride=-1)) == L.DSMOE_ERR_INVALID
    assert lib.dsmoe_mla_cache_append(p, 0, p, 0, 7, None, 1e-6, p, p, p, p, p, d, None) == L.DSMOE_ERR_UNSUPPORTED
    assert lib.dsmoe_mla_cache_append(p, -1, p, 0, 1, None, 1e-6, p, p, p, p, p, d, None) == L.DSMOE_ERR_INVALID
    assert lib.dsmoe_mla_cache_append(None, 0, p, 0, 1, None, 1e-6, p, p, p, p, p, d, None) == L.DSMOE_ERR_INVALID
    # nothing to do is no error, whatever the pointers
    assert lib.dsmoe_mla_cache_append(None, 0, None, 0, 1, None, 1e-6, None, None, None, None, None, _dims(T=0), None) == 0
    assert lib.dsmoe_mla_attn_paged(None, None, None, None, None, None, None, None, 0, None, 0, _dims(B=0), None, None, 0, None) == 0


def test_no_cpu_implementation():
    from dsmoe.mla import mla_attention_paged, mla_cache_append
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        mla_cache_append(bf(2, 16), bf(2, 8), bf(4, 16, 16), bf(4, 16, 8), i32(1, 2), i32(1), i32(2))
    with pytest.raises(RuntimeError, match="GPU"):
        mla_attention_paged(bf(2, 4, 16), bf(2, 4, 8), bf(4, 16, 16), bf(4, 16, 8), i32(1, 2), i32(1), i32(2), bf(4, 16, 16),
                            bf(4, 16, 16), 0.1)


def test_oracle_is_the_contiguous_attention_of_each_sequence():
    g = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    H, R, Dn, Dr, Dv, page = 3, 20, 10, 6, 12, 5
    new, kv = [4, 1], [13, 7]
    table = torch.tensor([[5, 0, 3], [1, 4, -1]], dtype=torch.int32)
    qn, qp, wk, wv = rnd(5, H, Dn), rnd(5, H, Dr), rnd(H, Dn, R), rnd(H, Dv, R)
    c, pe = rnd(20, R), rnd(20, Dr)
    kvp, pep = torch.full((6, page, R), float("nan")).double(), torch.full((6, page, Dr), float("nan")).double()
    lens, off = torch.tensor(kv), torch.tensor([0, 4, 5])
    # every position written as a new token of its sequence
    kvp, pep, written = append_ref(c, pe, kvp, pep, table, lens, torch.tensor([0, 13, 20]))
    assert int(written.sum()) == 20
    out, spread, size = attend_ref(qn, qp, kvp, pep, table, lens, off, wk, wv, 0.3)
    for b, (t, s) in enumerate(((slice(0, 4), slice(0, 13)), (slice(4, 5), slice(13, 20)))):
        ref = mla_attention_oracle(qn[t].transpose(0, 1)[None], qp[t].transpose(0, 1)[None], c[s][None], pe[s][None], wk, wv, 0.3,
                                   is_causal=True, q_start=kv[b] - new[b])
        assert abs(out[t].numpy() - ref[0]).max() < 1e-12
    assert (spread >= out.abs() - 1e-12).all() and (size > 0).all()
