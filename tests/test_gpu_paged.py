"""The paged latent cache and its attention (csrc/mla_cache.hip, csrc/mla_paged.hip, csrc/mla_paged_kv.hip) against the float64 oracle.

Bounds, derived from the arithmetic.  Append: one rounding to bf16 (2^-8 of the value) behind fp32 arithmetic of R + 8
roundings at most (2^-24 each).  Attention: the output's rounding (2^-8 of it), the probabilities' (2^-8 of
spread = sum_j p_j |v_j|), and the scores' errors: a score is off by at most d = size (2^-16 + (D_nope + 2 R + D_rope)
2^-24), size its sum of absolute terms (q_nope W_k is kept to 2^-16, then fp32 sums), which moves every probability by
a factor within e^(2 d) of one, another 2 d of spread and more; where K and V are built, in fp16, k and v add
2^-11 each: d = size 2^-11 and 2^-11 of spread."""
import pytest
import torch

from oracle.mla_ref import mla_attention_oracle
from oracle.paged_ref import append_ref, attend_ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
MID = dict(H=12, R=192, Dn=48, Dr=24, Dv=64)
WIDE = dict(H=32, R=256, Dn=128, Dr=64, Dv=128)
SMALL = dict(H=4, R=16, Dn=16, Dr=16, Dv=16)
ODD = dict(H=3, R=20, Dn=10, Dr=6, Dv=12)


def _batch(new, kv, page, seed, shape, spare=3, behind=0, width=None, H=0, R=0, Dn=0, Dr=0, Dv=0):
    """CPU tensors of a batch: sequences of `new` new tokens and `kv` positions, pages handed out in no order."""
    d = dict(shape)
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in kv]
    order = torch.randperm(sum(need) + spare, generator=g)
    table = torch.full((len(kv), width or max(1, *need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].int()[:table.shape[1]]
        at += n
    T = sum(new) + behind
    rnd = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).bfloat16()
    off = torch.tensor([0, *new]).cumsum(0).int()
    return dict(q_nope=rnd(T, d["H"], d["Dn"]), q_pe=rnd(T, d["H"], d["Dr"]), kv_pages=rnd(len(order), page, d["R"]),
                pe_pages=rnd(len(order), page, d["Dr"]), table=table, kv_lens=torch.tensor(kv, dtype=torch.int32),
                offsets=off, w_k=rnd(d["H"], d["Dn"], d["R"], std=d["R"] ** -0.5),
                w_v=rnd(d["H"], d["Dv"], d["R"], std=d["R"] ** -0.5)), (d["Dn"] + d["Dr"]) ** -0.5


ORDER = ("q_nope", "q_pe", "kv_pages", "pe_pages", "table", "kv_lens", "offsets", "w_k", "w_v")


def _gpu(x):
    return {k: v.to(DEV) for k, v in x.items()}


def _call(x, scale, **kw):
    from dsmoe.mla import mla_attention_paged
    return mla_attention_paged(*[x[k] for k in ORDER], scale, **kw)


def _check(got, x, scale):
    ref, spread, size = attend_ref(*[x[k] for k in ORDER], scale)
    rows = ~torch.isnan(ref).all(-1).all(-1)
    got = got.detach().cpu().double()
    Dn, R, Dr = x["q_nope"].shape[2], x["kv_pages"].shape[2], x["pe_pages"].shape[2]
    built = int((x["offsets"][1:] - x["offsets"][:-1]).max()) > 16   # K and V are built for some sequence, maybe
    d = size * (2.0 ** -11 if built else 2.0 ** -16) + size * (Dn + 2 * R + Dr) * 2.0 ** -24
    bound = 2.0 ** -8 * ref.abs() + spread * (2.0 ** -8 + 2.0 ** -10 + torch.expm1(2 * d)[..., None]) + 1e-30
    off = (got - ref).abs()[rows]
    assert torch.isfinite(got[rows]).all()
    assert (off <= bound[rows]).all(), f"max {off.max():.3g}, {(off / bound[rows]).max():.3g} of the bound"


@pytest.mark.parametrize("new,kv,page,shape", [
    ([1], [1], 64, MID),                                 # one position
    ([1], [300], 64, MID),
    ([1, 1, 1], [33, 1, 2000], 64, MID),                 # ragged decode
    ([1] * 70, [5 + 7 * i for i in range(70)], 16, SMALL),   # more sequences than lanes
    ([5, 0, 1, 33], [5, 40, 64, 700], 37, MID),          # a fresh prompt, a sequence without new tokens, odd pages
    ([3, 2], [3, 130], 1, ODD),                          # pages of one row, element loads
    ([7], [129], 128, dict(MID, H=5)),                   # a row tile over several tokens
    ([2], [70], 48, dict(MID, H=40)),                    # a token over two row tiles
    ([1, 1], [5000, 17], 64, WIDE),
    ([40, 9], [300, 9], 16, WIDE),
    ([64], [64], 64, ODD),
    ([2, 1], [65, 8], 16, dict(H=2, R=8, Dn=16, Dr=8, Dv=16)),   # a latent row of one 16-byte chunk
    ([1], [9000], 64, dict(H=1, R=64, Dn=32, Dr=16, Dv=32)),     # as many ranges as there may be
    ([2, 3], [50, 60], 16, dict(H=2, R=250, Dn=200, Dr=50, Dv=250)),
    ([2, 3], [50, 60], 16, dict(H=2, R=128, Dn=16, Dr=240, Dv=256)),
])
def test_attention(new, kv, page, shape):
    x, scale = _batch(new, kv, page, seed=len(new) + kv[0], shape=shape)
    _check(_call(_gpu(x), scale, max_q=max(new), max_kv=max(kv)), x, scale)


@pytest.mark.parametrize("new,kv,page,shape", [
    ([300], [300], 64, MID),                             # a fresh prompt, key ranges
    ([500, 1, 47, 46, 0, 1], [1400, 900, 47, 300, 50, 1], 48, MID),   # chunks beside decoding sequences, both sides of the line
    ([129, 200], [129, 1000], 16, WIDE),
    ([1300], [2000], 128, WIDE),
    ([33] * 70 + [1] * 5, [33 + 3 * i for i in range(75)], 16, SMALL),  # more sequences than lanes
    ([64, 130, 17], [64, 131, 300], 37, ODD),            # element loads of queries, latent rows and weights
    ([128], [128], 1, MID),                              # whole tiles
    ([257], [513], 64, dict(MID, H=5)),
    ([70, 60], [70, 161], 16, dict(H=2, R=250, Dn=200, Dr=50, Dv=250)),
    ([200], [333], 16, dict(H=2, R=128, Dn=16, Dr=240, Dv=256)),
    ([200, 150], [200, 400], 16, dict(H=40, R=64, Dn=32, Dr=16, Dv=32)),
])
def test_chunks(new, kv, page, shape):
    x, scale = _batch(new, kv, page, seed=len(new) + kv[0], shape=shape)
    _check(_call(_gpu(x), scale, max_q=max(new), max_kv=max(kv)), x, scale)
    _check(_call(_gpu(x), scale), x, scale)


@pytest.mark.parametrize("new,kv,page,shape", [
    ([300, 130, 17], [300, 131, 300], 37, ODD),          # element loads of queries, latent rows and weights
    ([400, 300], [400, 461], 16, dict(H=2, R=250, Dn=200, Dr=50, Dv=250)),
    ([700], [833], 16, dict(H=2, R=128, Dn=16, Dr=240, Dv=256)),
    ([330, 1, 5], [330, 40, 9], 1, SMALL),
    ([24, 20, 18, 17, 16, 40], [24, 90, 400, 17, 16, 900], 16, MID),     # near the line, together with K and V
    ([24, 20, 18, 17, 30, 20], [2000, 90, 900, 1100, 1500, 700], 16, MID),   # and together without
    ([200, 20, 1], [220, 3000, 700], 64, MID),           # far on either side in one batch
])
def test_chunks_of_as_many_rows_as_pay(new, kv, page, shape):
    """Batches of at least 1280 (token, head) rows, from where on K and V may be built."""
    assert sum(new) * shape["H"] >= 1280
    x, scale = _batch(new, kv, page, seed=len(new) + kv[0] + 1, shape=shape)
    _check(_call(_gpu(x), scale, max_q=max(new), max_kv=max(kv)), x, scale)
    _check(_call(_gpu(x), scale), x, scale)


@pytest.mark.parametrize("scale", [-0.3, 2.0, 0.0])
def test_scales_of_many_rows(scale):
    x, _ = _batch([1, 330], [200, 400], 16, seed=48, shape=SMALL)
    _check(_call(_gpu(x), scale), x, scale)


def test_tiny_values_keep_their_weight_in_chunks():
    """As test_tiny_values_keep_their_weight, with enough rows and tokens for K and V."""
    x, scale = _batch([128], [8192], 64, seed=49, shape=MID)
    pages = x["table"][0].long()
    x["kv_pages"][pages] = (x["kv_pages"][pages].float() * 1e-36).bfloat16()
    x["kv_pages"][pages[0], 0] = torch.randn(192, generator=torch.Generator().manual_seed(1)).bfloat16()
    x["q_nope"].zero_()
    x["q_pe"].fill_(1.0)
    x["pe_pages"].zero_()
    x["pe_pages"][pages[0], 0] = 14 * 0.6931 / (24 * scale)
    _check(_call(_gpu(x), scale), x, scale)


def test_offsets_out_of_range_with_many_rows():
    n = 353
    x, scale = _batch([2, n], [30, 400], 16, seed=50, shape=SMALL)
    clean = _call(_gpu(x), scale)
    for offsets, rows in (([0, 2, 10 ** 9], slice(None)), ([0, 2, -5], slice(0, 2)), ([-9, 2, 2 + n], slice(None))):
        x["offsets"] = torch.tensor(offsets, dtype=torch.int32)
        assert (_call(_gpu(x), scale)[rows].float() - clean[rows].float()).abs().max() <= 2e-2 * clean.float().abs().max()


def test_chunks_in_several_passes():
    """K and V of one pass hold 4 GiB: a table far wider than the sequences are long."""
    new = [129] * 8 + [1]
    x, scale = _batch(new, [n + 40 for n in new], 64, seed=31, shape=WIDE, width=512)
    _check(_call(_gpu(x), scale), x, scale)


@pytest.mark.parametrize("c,pe,w", [(1e20, 1e20, 1e-10), (1e-20, 1e-20, 1e-10), (3e4, 1.0, 1e3), (1e-6, 1e6, 1.0)])
def test_magnitudes_past_half_precision(c, pe, w):
    """Keys, values, queries far above and below what 16-bit floats of five exponent bits hold, in one batch with ordinary ones."""
    x, scale = _batch([150, 100, 3], [150, 333, 90], 16, seed=33, shape=MID)
    lo = x["kv_pages"].shape[0] // 2
    x["kv_pages"][:lo] = (x["kv_pages"][:lo].float() * c).bfloat16()
    x["pe_pages"][:lo] = (x["pe_pages"][:lo].float() * pe).bfloat16()
    x["w_k"], x["w_v"] = (x["w_k"].float() * w).bfloat16(), (x["w_v"].float() * w).bfloat16()
    z = max(1.0, c * w, pe)
    x["q_nope"], x["q_pe"] = (x["q_nope"].float() / z).bfloat16(), (x["q_pe"].float() / z).bfloat16()
    _check(_call(_gpu(x), scale), x, scale)


@pytest.mark.parametrize("scale", [-0.3, 2.0, 0.0])
@pytest.mark.parametrize("n", [6, 60])
def test_scales(scale, n):
    x, _ = _batch([1, n], [200, 90], 16, seed=3, shape=SMALL)
    _check(_call(_gpu(x), scale), x, scale)


def test_hints_do_not_change_what_is_computed():
    """max_q and max_kv far too small or large: every position and token still counts."""
    x, scale = _batch([1, 60, 3], [900, 400, 64], 16, seed=5, shape=MID)
    g = _gpu(x)
    for kw in (dict(), dict(max_q=1, max_kv=1), dict(max_q=0, max_kv=0), dict(max_q=10 ** 6, max_kv=2 ** 40)):
        _check(_call(g, scale, **kw), x, scale)


def test_strides_and_views():
    """Queries as halves of one projection, pages as halves of one pool with a gap, a table inside a wider one, head views
    of one weight: read in place, with equal bits."""
    x, scale = _batch([4, 1], [70, 130], 16, seed=7, shape=MID)
    g = _gpu(x)
    want = _call(g, scale)
    v = dict(g)
    T, H, Dn, Dr, R, Dv = 5, 12, 48, 24, 192, 64
    q = torch.cat([g["q_nope"], g["q_pe"]], -1).transpose(0, 1).contiguous().transpose(0, 1)   # heads outermost
    v["q_nope"], v["q_pe"] = q[..., :Dn], q[..., Dn:]
    pool = torch.full((g["kv_pages"].shape[0], 17, R + Dr), float("nan"), dtype=torch.bfloat16, device=DEV)
    v["kv_pages"], v["pe_pages"] = pool[:, :16, :R], pool[:, :16, R:]
    v["kv_pages"].copy_(g["kv_pages"])
    v["pe_pages"].copy_(g["pe_pages"])
    wide = torch.full((2, 40), 10 ** 9, dtype=torch.int32, device=DEV)
    v["table"] = wide[:, 3:3 + g["table"].shape[1]]
    v["table"].copy_(g["table"])
    w = torch.cat([g["w_k"], g["w_v"]], 1)
    v["w_k"], v["w_v"] = w[:, :Dn], w[:, Dn:]
    assert torch.equal(_call(v, scale), want)
    # the last dimension not contiguous: copied
    v["q_nope"] = g["q_nope"].transpose(1, 2).contiguous().transpose(1, 2)
    v["w_v"] = g["w_v"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(_call(v, scale), want)
    _check(want, x, scale)


def test_rows_without_anything():
    """No positions, fewer positions than new tokens, rows behind the last sequence, sequences without tokens."""
    x, scale = _batch([3, 4, 0, 2], [10, 10, 5, 10], 16, seed=9, shape=SMALL, behind=6)
    x["kv_lens"] = torch.tensor([0, 2, 5, -7], dtype=torch.int32)
    out = torch.full((15, 4, 16), 7.0, dtype=torch.bfloat16, device=DEV)
    got = _call(_gpu(x), scale, out=out)
    assert got is out
    _check(got, x, scale)
    assert (got[9:] == 7.0).all()                    # as they were
    assert (got[:5] == 0).all() and (got[7:9] == 0).all()
    # nothing to do at all
    y = _gpu(x)
    y["q_nope"], y["q_pe"] = y["q_nope"][:0], y["q_pe"][:0]
    assert _call(y, scale).shape == (0, 4, 16)
    y = dict(_gpu(x), table=y["table"][:0], kv_lens=y["kv_lens"][:0], offsets=y["offsets"][:1])
    assert (_call(y, scale, out=out.fill_(3.0)) == 3.0).all()


@pytest.mark.parametrize("n", [5, 55])
def test_pages_that_are_not_there_and_lengths_past_the_table(n):
    x, scale = _batch([2, n, 1], [100, 90, 60], 16, seed=11, shape=MID)
    x["table"][0, 2] = -1
    x["table"][1, 0] = 10 ** 6
    x["table"][1, 5] = x["kv_pages"].shape[0]
    x["table"][2, :] = -5
    x["kv_lens"][0] = 130                            # the table ends at 112: the new tokens stand behind it
    _check(_call(_gpu(x), scale), x, scale)
    x["kv_lens"][0] = 2 ** 31 - 1
    got = _call(_gpu(x), scale)
    _check(got, x, scale)
    assert (got[n + 2] == 0).all()                   # a sequence without a single page


def test_offsets_that_are_out_of_range_stay_inside():
    """Offsets past T, or decreasing ones: clamped, the sound sequences unharmed."""
    for n in (3, 53):
        x, scale = _batch([2, n], [30, 60], 16, seed=12, shape=SMALL)
        clean = _call(_gpu(x), scale)
        x["offsets"] = torch.tensor([0, 2, 10 ** 9], dtype=torch.int32)
        assert torch.equal(_call(_gpu(x), scale), clean)
        x["offsets"] = torch.tensor([0, 2, -5], dtype=torch.int32)
        assert torch.equal(_call(_gpu(x), scale)[:2], clean[:2])
        x["offsets"] = torch.tensor([-9, 2, 2 + n], dtype=torch.int32)
        assert torch.equal(_call(_gpu(x), scale), clean)


@pytest.mark.parametrize("H", [4, 31])
@pytest.mark.parametrize("offsets", [[1, 5, 0, 3], [100, 200, 0, 50], [0, 150, 151, 0], [300, 200, 100, 0], [0, 200, 260, 0]])
def test_offsets_that_decrease_stay_inside(H, offsets):
    """Sequences found by a search that offsets in no order mislead: only rows of the batch are written, here and in the pages."""
    from dsmoe.mla import mla_cache_append
    x, scale = _batch([60, 200, 1], [300, 260, 64], 16, seed=44, shape=dict(SMALL, H=H), behind=40)
    g = _gpu(x)
    g["offsets"] = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    guard = torch.full((301 + 64, H, 16), 7.0, dtype=torch.bfloat16, device=DEV)
    for kw in (dict(), dict(max_q=1)):
        _call(g, scale, out=guard[32:-32], **kw)
        assert (guard[:32] == 7).all() and (guard[-32:] == 7).all()
    before = g["kv_pages"].clone()
    mla_cache_append(torch.randn(301, 16, device=DEV), torch.randn(301, 16, device=DEV), g["kv_pages"], g["pe_pages"], g["table"],
                     g["kv_lens"], g["offsets"])
    used = torch.zeros(before.shape[0], dtype=torch.bool)
    used[x["table"][x["table"] >= 0].long()] = True
    assert torch.equal(g["kv_pages"].cpu()[~used], before.cpu()[~used])


def test_tiny_values_keep_their_weight():
    """Thousands of keys with values of 1e-36 and 2^-14 of the weight each, beside one with ordinary values: as many together
    as half of its."""
    x, scale = _batch([64], [8192], 64, seed=45, shape=MID)
    pages = x["table"][0].long()
    x["kv_pages"][pages] = (x["kv_pages"][pages].float() * 1e-36).bfloat16()
    x["kv_pages"][pages[0], 0] = torch.randn(192, generator=torch.Generator().manual_seed(1)).bfloat16()
    x["q_nope"].zero_()
    x["q_pe"].fill_(1.0)
    x["pe_pages"].zero_()
    x["pe_pages"][pages[0], 0] = 14 * 0.6931 / (24 * scale)
    _check(_call(_gpu(x), scale), x, scale)


@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("n", [9, 150])
def test_not_finite_rows_reach_those_that_see_them(what, n):
    """In a cached row: NaN in the tokens that see it, the others' bits unchanged; behind a sequence's length, on unused
    pages and in another sequence: nothing."""
    x, scale = _batch([n, 1, 4], [n + 51, 200, 4], 16, seed=13, shape=SMALL)
    g = _gpu(x)
    clean = _call(g, scale)
    for j in (0, 30, 52, 55, n + 43, n + 50):        # sequence 0's new tokens stand at 51 .. n + 50
        bad = dict(g, kv_pages=g["kv_pages"].clone())
        bad["kv_pages"][int(x["table"][0, j // 16]), j % 16, 3] = what
        got = _call(bad, scale)
        sees = torch.arange(n + 5, device=DEV) + 51 >= j
        sees[n:] = False
        assert torch.isnan(got[sees]).any(-1).all() and torch.equal(got[~sees], clean[~sees]), j
    used = torch.zeros(g["kv_pages"].shape[:2], dtype=torch.bool)
    for b, kv in enumerate((n + 51, 200, 4)):
        for j in range(kv):
            used[int(x["table"][b, j // 16]), j % 16] = True
    bad = dict(g, kv_pages=g["kv_pages"].clone(), pe_pages=g["pe_pages"].clone())
    bad["kv_pages"][~used.to(DEV)] = what
    bad["pe_pages"][~used.to(DEV)] = what
    assert torch.equal(_call(bad, scale), clean)
    bad = dict(g, q_nope=g["q_nope"].clone())
    bad["q_nope"][3, 2, 1] = float("nan")
    got = _call(bad, scale)
    assert torch.isnan(got[3, 2]).all()
    got[3, 2] = clean[3, 2]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("shape,page", [(MID, 64), (WIDE, 16), (ODD, 5), (dict(SMALL, R=8, Dr=8), 1), (dict(SMALL, R=252, Dr=3), 16)])
def test_append(dtype, norm, shape, page):
    new, kv = [1, 40, 0, 3, 1], [100, 40, 7, 2, 64]      # sequence 3: one token before position 0
    x, _ = _batch(new, kv, page, seed=page, shape=shape, behind=4)
    x["table"][4, 63 // page] = -1                       # and the last one's page is not there
    g = torch.Generator().manual_seed(1)
    c = (torch.randn(49, shape["R"], generator=g) * 3).to(dtype)
    pe = torch.randn(49, shape["Dr"], generator=g).to(dtype)
    w = (1 + 0.1 * torch.randn(shape["R"], generator=g)) if norm else None
    kv_ref, pe_ref, written = append_ref(c, pe, x["kv_pages"], x["pe_pages"], x["table"], x["kv_lens"], x["offsets"], w)
    y = _gpu(x)
    from dsmoe.mla import mla_cache_append
    mla_cache_append(c.to(DEV), pe.to(DEV), y["kv_pages"], y["pe_pages"], y["table"], y["kv_lens"], y["offsets"],
                     norm_weight=None if w is None else w.to(DEV))
    for got, ref, before in ((y["kv_pages"], kv_ref, x["kv_pages"]), (y["pe_pages"], pe_ref, x["pe_pages"])):
        got = got.cpu()
        assert torch.equal(got[~written], before[~written])
        err = (got.double() - ref).abs()[written]
        assert (err <= ref.abs()[written] * (2.0 ** -8 + (shape["R"] + 8) * 2.0 ** -24)).all()
    assert int(written.sum()) == 1 + 40 + 2


def test_append_into_views_and_from_views():
    """Halves of one pool with a gap, rows that are halves of one projection, a column-major tensor, a bf16 norm weight."""
    from dsmoe.mla import mla_cache_append
    x, _ = _batch([3, 17], [30, 17], 16, seed=2, shape=MID)
    g = _gpu(x)
    rows = torch.randn(20, 192 + 24, device=DEV).bfloat16()
    w = torch.randn(192, device=DEV).bfloat16()
    plain = [g["kv_pages"].clone(), g["pe_pages"].clone()]
    mla_cache_append(rows[:, :192].contiguous(), rows[:, 192:].contiguous(), *plain, g["table"], g["kv_lens"], g["offsets"],
                     norm_weight=w.float())
    pool = torch.zeros(g["kv_pages"].shape[0], 18, 224, dtype=torch.bfloat16, device=DEV)
    pool[:, :16, :192], pool[:, :16, 192:216] = g["kv_pages"], g["pe_pages"]
    mla_cache_append(rows[:, :192], rows[:, 192:].T.contiguous().T, pool[:, :16, :192], pool[:, :16, 192:216], g["table"],
                     g["kv_lens"], g["offsets"], norm_weight=w)
    assert torch.equal(pool[:, :16, :192], plain[0]) and torch.equal(pool[:, :16, 192:216], plain[1])
    assert (pool[:, 16:] == 0).all() and (pool[..., 216:] == 0).all()


@pytest.mark.parametrize("chunks", [[1] * 12, [200, 1, 1, 90, 1], [33, 32, 31]])
def test_a_prompt_in_chunks_is_the_contiguous_attention(chunks):
    """append, then attend, chunk after chunk, beside a second sequence: the rows of one causal attention over the whole."""
    from dsmoe.mla import mla_cache_append
    S, other = sum(chunks), 7
    x, scale = _batch([S, other], [S, other], 16, seed=S, shape=MID)
    g = _gpu(x)
    c = torch.randn(S + other, 192, device=DEV).bfloat16()
    pe = torch.randn(S + other, 24, device=DEV).bfloat16()
    ref = [torch.as_tensor(mla_attention_oracle(g["q_nope"][r].transpose(0, 1)[None].cpu(), g["q_pe"][r].transpose(0, 1)[None].cpu(),
                                                c[r][None].cpu(), pe[r][None].cpu(), x["w_k"], x["w_v"], scale, is_causal=True))[0]
           for r in (slice(0, S), slice(S, S + other))]
    done = 0
    for n in chunks:
        rows = torch.cat([torch.arange(done, done + n), torch.arange(S, S + other)]).to(DEV)
        done += n
        b = dict(g, kv_lens=torch.tensor([done, other], dtype=torch.int32, device=DEV),
                 offsets=torch.tensor([0, n, n + other], dtype=torch.int32, device=DEV), q_nope=g["q_nope"][rows], q_pe=g["q_pe"][rows])
        mla_cache_append(c[rows], pe[rows], b["kv_pages"], b["pe_pages"], b["table"], b["kv_lens"], b["offsets"])
        got = _call(b, scale, max_q=max(n, other), max_kv=done).cpu().double()
        want = torch.cat([ref[0][done - n:done], ref[1]])
        assert (got - want).abs().max() <= 2e-2 * want.abs().max()


def test_captured_calls_replay_on_other_lengths_pages_and_values():
    """append and attend in a graph; between replays eager calls of the same operators on the same stream."""
    from dsmoe.mla import mla_cache_append
    x, scale = _batch([4, 61, 0], [70, 70, 64], 16, seed=21, shape=MID)
    g = _gpu(x)
    c, pe = torch.randn(65, 192, device=DEV).bfloat16(), torch.randn(65, 24, device=DEV).bfloat16()
    out = torch.empty(65, 12, 64, dtype=torch.bfloat16, device=DEV)

    def step(x, c, pe, out):
        mla_cache_append(c, pe, x["kv_pages"], x["pe_pages"], x["table"], x["kv_lens"], x["offsets"])
        return _call(x, scale, out=out)
    step(g, c, pe, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(g, c, pe, out)
    for new, kv in (([4, 61, 0], [70, 70, 64]), ([1, 1, 63], [9, 71, 64]), ([0, 65, 0], [1, 68, 2]), ([22, 21, 22], [40, 40, 30])):
        g["kv_lens"].copy_(torch.tensor(kv))
        g["offsets"].copy_(torch.tensor([0, *new]).cumsum(0))
        g["table"].copy_(g["table"].flip(1) if new[0] == 1 else g["table"])
        c.normal_()
        e = {k: v.clone() for k, v in g.items()}
        want = step(e, c, pe, torch.empty_like(out))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(g["kv_pages"], e["kv_pages"])


def test_captured_chunks_replay_and_streams():
    """Batches with K and V built: captured and replayed on other lengths, strided inputs with equal bits, two streams at once."""
    x, scale = _batch([100, 61, 0], [170, 70, 64], 16, seed=51, shape=MID)
    g = _gpu(x)
    out = torch.empty(161, 12, 64, dtype=torch.bfloat16, device=DEV)
    _call(g, scale, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _call(g, scale, out=out)
    for new, kv in (([100, 61, 0], [170, 70, 64]), ([1, 60, 100], [9, 71, 164]), ([0, 161, 0], [1, 170, 2]), ([40, 60, 61], [40, 80, 61])):
        g["kv_lens"].copy_(torch.tensor(kv))
        g["offsets"].copy_(torch.tensor([0, *new]).cumsum(0))
        g["q_nope"].normal_()
        want = _call({k: v.clone() for k, v in g.items()}, scale)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    v = dict(g)
    q = torch.cat([g["q_nope"], g["q_pe"]], -1).transpose(0, 1).contiguous().transpose(0, 1)
    v["q_nope"], v["q_pe"] = q[..., :48], q[..., 48:]
    pool = torch.cat([g["kv_pages"], g["pe_pages"]], -1)
    v["kv_pages"], v["pe_pages"] = pool[..., :192], pool[..., 192:]
    w = torch.cat([g["w_k"], g["w_v"]], 1)
    v["w_k"], v["w_v"] = w[:, :48], w[:, 48:]
    assert torch.equal(_call(v, scale), want)
    y, _ = _batch([150, 3], [900, 33], 16, seed=52, shape=MID)
    h, side = _gpu(y), torch.cuda.Stream()
    other = _call(h, scale)
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(side):
            b = _call(h, scale)
        a = _call(g, scale)
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, other)


def test_captured_as_a_threads_first_call():
    """Both kinds of sequences in a call that a thread captures before it ever ran one."""
    import threading
    x, scale = _batch([2, 70, 1], [40, 170, 9], 16, seed=47, shape=MID)
    g = _gpu(x)
    out, want, errors = torch.empty(73, 12, 64, dtype=torch.bfloat16, device=DEV), _call(g, scale), []
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()

    def run():
        try:
            with torch.no_grad(), torch.cuda.graph(graph):
                _call(g, scale, out=out)
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    t = threading.Thread(target=run)
    t.start()
    t.join()
    assert not errors, errors
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_compiled_with_a_graph_break():
    from dsmoe.mla import mla_cache_append
    x, scale = _batch([4, 61], [70, 70], 16, seed=46, shape=MID)
    a, b = _gpu(x), _gpu(x)
    c, pe = torch.randn(65, 192, device=DEV).bfloat16(), torch.randn(65, 24, device=DEV).bfloat16()

    def f(x, c, pe):
        mla_cache_append(c, pe, x["kv_pages"], x["pe_pages"], x["table"], x["kv_lens"], x["offsets"])
        return _call(x, scale) * 2
    assert torch.equal(torch.compile(f, backend="eager")(a, c, pe), f(b, c, pe))
    assert torch.equal(a["kv_pages"], b["kv_pages"])


def test_two_streams_at_once():
    x, scale = _batch([3, 100], [300, 700], 16, seed=23, shape=MID)
    y, _ = _batch([70, 1], [900, 33], 16, seed=24, shape=MID)
    a, b = _gpu(x), _gpu(y)
    want = _call(a, scale), _call(b, scale)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(5):
        with torch.cuda.stream(s1):
            got.append((_call(a, scale), want[0]))
        with torch.cuda.stream(s2):
            got.append((_call(b, scale), want[1]))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in got)


def test_float32_queries_and_weights_under_autocast():
    x, scale = _batch([2, 1], [40, 50], 16, seed=25, shape=SMALL)
    g = _gpu(x)
    f = dict(g, **{k: g[k].float() for k in ("q_nope", "q_pe", "w_k", "w_v")})
    with pytest.raises(ValueError, match="autocast"):
        _call(f, scale)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = _call(f, scale)
    assert got.dtype == torch.float32 and torch.equal(got, _call(g, scale).float())


def test_refusals():
    from dsmoe.mla import mla_attention_paged, mla_cache_append
    x, scale = _batch([2, 1], [40, 50], 16, seed=26, shape=SMALL)
    g = _gpu(x)
    for change, text in (
            (dict(kv_pages=g["kv_pages"].float()), "bfloat16"), (dict(table=g["table"].long()), "int32"),
            (dict(kv_lens=g["kv_lens"][:1]), "block_table"), (dict(offsets=g["offsets"][:2]), "q_offsets"),
            (dict(pe_pages=g["pe_pages"][:, :8]), "kv_pages"), (dict(w_k=g["w_k"][:3]), "inconsistent"),
            (dict(q_pe=g["q_pe"][..., :8]), "inconsistent"), (dict(q_nope=g["q_nope"].half()), "bf16 or fp32"),
            (dict(kv_pages=g["kv_pages"].transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
            (dict(q_nope=g["q_nope"][0]), "three dimensions")):
        with pytest.raises(ValueError, match=text):
            _call(dict(g, **change), scale)
    with pytest.raises(ValueError, match="out must"):
        _call(g, scale, out=torch.empty(3, 4, 17, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(RuntimeError, match="no backward"):
        _call(dict(g, q_nope=g["q_nope"].clone().requires_grad_(True)), scale)
    with torch.no_grad():
        _call(dict(g, q_nope=g["q_nope"].clone().requires_grad_(True)), scale)
    c, pe = torch.zeros(3, 16, device=DEV), torch.zeros(3, 16, device=DEV)
    rest = [g[k] for k in ("kv_pages", "pe_pages", "table", "kv_lens", "offsets")]
    for bad, text in (((c[:, :8], pe), "width"), ((c, pe[:2]), "width"), ((c.half(), pe.half()), "dtype"), ((c, pe.bfloat16()), "one dtype")):
        with pytest.raises(ValueError, match=text):
            mla_cache_append(*bad, *rest)
    with pytest.raises(ValueError, match="norm_weight"):
        mla_cache_append(c, pe, *rest, norm_weight=c[0, :5])
    torch.cuda.synchronize()
