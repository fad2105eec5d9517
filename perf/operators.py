"""The serving and routing operators that are timed beside their plain forms, with inputs and float64 results.

* ``append``: new latent rows normed and written into the pages of a latent cache (``dsmoe.mla.mla_cache_append``).
* ``attend``: MLA attention of the new tokens over that cache (``dsmoe.mla.mla_attention_paged``).
* ``route``: routing to experts from logits, and with ``train`` its gradient (``dsmoe.ops.route_experts``).

``listed()`` are the named cases and ``draw(rng)`` gives another one of the same ranges; ``prepare`` makes inputs, ``run``
does one pass (in elementary torch operations, or with ``own`` through the framework), ``exact`` gives its results in
float64, ``work`` the bytes and operations it cannot do without."""
import random
import sys

import torch

own = False

if "deepseek-v3-lite_amd" not in sys.path:
    sys.path.insert(0, "deepseek-v3-lite_amd")

EPS = 1e-6
DEV = "cuda"


# ---------------------------------------------------------------------------- cases
# Attention shapes (heads, latent rank, query/key width without and with the rotary part, value width): those of the
# model configurations that tests and benchmark use, and the wide one of the attention's tests.
_SMALL = dict(H=4, R=16, Dn=16, Dr=16, Dv=16)
_MID = dict(H=12, R=192, Dn=48, Dr=24, Dv=64)
_WIDE = dict(H=32, R=256, Dn=128, Dr=64, Dv=128)


def _cache(op, shape, seqs, new, past, decoding, page, ragged, **more):
    """seqs sequences with `new` new tokens after `past` cached ones: the first sequence exactly so, the others ragged,
    each of them a decoding one (a single new token) with probability `decoding`."""
    return dict(op=op, seqs=seqs, new=new, past=past, decoding=decoding, page=page, ragged=ragged, **shape, **more)


def _route(T, E, k, score, bias, groups, keep, normalise, train):
    return dict(op="route", T=T, E=E, k=k, score=score, bias=bias, groups=groups, keep=keep, normalise=normalise, train=train)


def listed():
    return [
        # one decoded token for each of 48 users: latency
        dict(name="append_decode", **_cache("append", _MID, 48, 1, 900, 0.0, 64, 1, norm=True)),
        # prompt chunks of some users beside decoding ones, rows normed by the caller, small pages
        dict(name="append_chunks", **_cache("append", _WIDE, 24, 1500, 2500, 0.3, 16, 2, norm=False)),
        # one user's next token over a short context: the smallest call
        dict(name="attend_one", **_cache("attend", _MID, 1, 1, 299, 0.0, 64, 3)),
        # a serving batch in its decode phase, ragged contexts
        dict(name="attend_decode", **_cache("attend", _MID, 64, 1, 2047, 0.0, 64, 4)),
        # long contexts, wide heads: the cache's bytes
        dict(name="attend_decode_long", **_cache("attend", _WIDE, 12, 1, 32700, 0.0, 64, 5)),
        # a scheduler's mixed step: chunks of prompts beside decoding users, odd pages
        dict(name="attend_mixed", **_cache("attend", _MID, 20, 500, 1400, 0.7, 48, 6)),
        # the second chunk of two long prompts: matrix products
        dict(name="attend_prefill", **_cache("attend", _WIDE, 2, 2048, 4096, 0.0, 128, 7)),
        # the router of a decode step of 64 users
        dict(name="route_decode", **_route(64, 64, 6, "sigmoid", True, 8, 3, True, False)),
        # prefill of 8192 tokens with many fine experts in groups
        dict(name="route_prefill", **_route(8192, 256, 8, "sigmoid", True, 8, 4, True, False)),
        # softmax scores kept as they are, an odd token count and no groups
        dict(name="route_softmax", **_route(5001, 64, 6, "softmax", False, 1, 1, False, False)),
        # a micro batch's router with its gradient
        dict(name="route_train_small", **_route(1000, 16, 4, "sigmoid", True, 4, 2, True, True)),
        # the training step of bench.py, with softmax scores whose gradient reaches every expert
        dict(name="route_train", **_route(16384, 160, 6, "softmax", True, 8, 3, False, True)),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "route", "route", "route"])
    ragged = rng.randrange(1, 1 << 20)
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        E = groups * _log_int(rng, 4, 256 // groups)
        keep = rng.randint((groups + 1) // 2, groups)
        k = rng.randint(1, min(8, E // groups * keep))
        return _route(_log_int(rng, 1, 16384), E, k, rng.choice(["sigmoid", "softmax"]), rng.random() < 0.7, groups, keep,
                      rng.random() < 0.6, rng.random() < 0.4)
    shape = rng.choice([_SMALL, _MID, _MID, _WIDE])
    page = rng.choice([1, 16, 37, 64, 64, 128])
    if op == "append":
        return _cache(op, shape, _log_int(rng, 1, 64), _log_int(rng, 1, 1024), _log_int(rng, 1, 2048), rng.choice([0.0, 0.5]), page,
                      ragged, norm=rng.random() < 0.5)
    form = rng.choice(["decode", "mixed", "prefill"])
    if form == "decode":
        return _cache(op, shape, _log_int(rng, 1, 64), 1, _log_int(rng, 1, 4096), 0.0, page, ragged)
    if form == "mixed":
        return _cache(op, shape, _log_int(rng, 1, 16), _log_int(rng, 2, 512), _log_int(rng, 1, 2048), 0.6, page, ragged)
    return _cache(op, shape, rng.choice([1, 2]), _log_int(rng, 64, 1500), _log_int(rng, 1, 2048), 0.0, page, ragged)


def _lengths(case):
    """New tokens and lengths (with them) of every sequence of a case."""
    r = random.Random(case["ragged"])
    new, kv = [case["new"]], [case["past"] + case["new"]]
    for _ in range(case["seqs"] - 1):
        n = 1 if r.random() < case["decoding"] else r.randint((case["new"] + 1) // 2, case["new"])
        new.append(n)
        kv.append(r.randint(case["past"] // 4, case["past"]) + n)
    return new, kv


# ---------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)

    s = dict(case=case)
    if case["op"] == "route":
        T, E = case["T"], case["E"]
        s["logits"] = normal(T, E, dtype=torch.float32)
        s["bias"] = normal(E, std=0.05, dtype=torch.float32) if case["bias"] else None
        if case["train"]:
            s["logits"].requires_grad_(True)
            s["dw"] = normal(T, case["k"], dtype=torch.float32)
        return s
    # the pages: handed out in no order, some of them to nobody; entries of a table past a sequence's pages are -1
    new, kv = _lengths(case)
    page, H, R, Dn, Dr, Dv = (case[n] for n in ("page", "H", "R", "Dn", "Dr", "Dv"))
    need = [-(-n // page) for n in kv]
    order = torch.randperm(sum(need) + 7, generator=g, device=DEV).cpu().tolist()
    table = torch.full((len(kv), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    offsets = torch.tensor([0, *new]).cumsum(0)
    T = int(offsets[-1])
    s["table"], s["kv_lens"] = table.to(DEV), torch.tensor(kv, dtype=torch.int32, device=DEV)
    s["offsets"] = offsets.to(torch.int32).to(DEV)
    s["max_q"], s["max_kv"] = max(new), max(kv)
    s["kv_pages"], s["pe_pages"] = normal(len(order), page, R), normal(len(order), page, Dr)
    if case["op"] == "append":
        s["ctx_kv"], s["ctx_pe"] = normal(T, R, std=3.0), normal(T, Dr)
        s["norm"] = (1.0 + 0.1 * torch.randn(R, generator=g, device=DEV)) if case["norm"] else None
        return s
    # queries as one projection leaves them, split per head, and the per-head views of one up-projection weight
    q = normal(T, H, Dn + Dr)
    w = normal(H, Dn + Dv, R, std=R ** -0.5)
    s["q_nope"], s["q_pe"] = q[..., :Dn], q[..., Dn:]
    s["w_k"], s["w_v"] = w[:, :Dn], w[:, Dn:]
    s["scale"] = (Dn + Dr) ** -0.5
    return s


# ---------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    if case["op"] == "route":
        return _plain_route(state, case)
    return _plain_append(state) if case["op"] == "append" else _plain_attend(state)


def _own(s, case):
    from dsmoe import mla, ops
    if case["op"] == "append":
        mla.mla_cache_append(s["ctx_kv"], s["ctx_pe"], s["kv_pages"], s["pe_pages"], s["table"], s["kv_lens"], s["offsets"],
                             norm_weight=s["norm"], norm_eps=EPS)
        return s["kv_pages"], s["pe_pages"]
    if case["op"] == "attend":
        return mla.mla_attention_paged(s["q_nope"], s["q_pe"], s["kv_pages"], s["pe_pages"], s["table"], s["kv_lens"],
                                       s["offsets"], s["w_k"], s["w_v"], s["scale"], max_q=s["max_q"], max_kv=s["max_kv"])
    w, idx, counts = ops.route_experts(s["logits"], case["k"], s["bias"], score=case["score"], n_groups=case["groups"],
                                       topk_groups=case["keep"], normalise=case["normalise"], route_scale=2.5)
    if not case["train"]:
        return w, idx, counts
    return w.detach(), idx, counts, torch.autograd.grad(w, s["logits"], s["dw"])[0]


def _plain_append(s):
    T, page = s["ctx_kv"].shape[0], s["kv_pages"].shape[1]
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(s["offsets"], t, right=True) - 1
    pos = s["kv_lens"][b] - s["offsets"][b + 1] + t
    at = (s["table"][b, pos // page].long(), pos % page)
    c = s["ctx_kv"].float()
    if s["norm"] is not None:
        c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS) * s["norm"]
    s["kv_pages"][at] = c.to(torch.bfloat16)
    s["pe_pages"][at] = s["ctx_pe"]
    return s["kv_pages"], s["pe_pages"]


def _plain_attend(s):
    page, off = s["kv_pages"].shape[1], s["offsets"].long()
    T, B = s["q_nope"].shape[0], off.numel() - 1
    # the batch padded to its longest sequence and chunk
    j = torch.arange(s["max_kv"], device=DEV)
    pages = s["table"][:, j // page].long().clamp(min=0)
    c, pe = s["kv_pages"][pages, j % page].float(), s["pe_pages"][pages, j % page].float()        # (B, kv, R), (B, kv, Dr)
    i = torch.arange(s["max_q"], device=DEV)
    tok = (off[:-1, None] + i).clamp(max=T - 1)
    qn, qp = s["q_nope"][tok].float().transpose(1, 2), s["q_pe"][tok].float().transpose(1, 2)     # (B, H, q, D)
    k = torch.matmul(c[:, None], s["w_k"].float().transpose(1, 2).contiguous())                  # (B, H, kv, Dn)
    v = torch.matmul(c[:, None], s["w_v"].float().transpose(1, 2).contiguous())
    scores = torch.matmul(qn, k.transpose(2, 3)) + torch.matmul(qp, pe[:, None].transpose(2, 3))
    pos = (s["kv_lens"] - (off[1:] - off[:-1]))[:, None] + i
    scores = torch.where(j <= pos[:, None, :, None], scores * s["scale"], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)                                              # (B, H, q, Dv)
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(off, t, right=True) - 1
    return o[b, :, t - off[b]].to(torch.bfloat16)


def _scores(logits, score):
    """Scores in 64 bits: what the choice rests on is rounded to 32 from them, once."""
    x = logits.double()
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_route(s, case):
    T, E, k, G, keep = (case[n] for n in ("T", "E", "k", "groups", "keep"))
    sc = _scores(s["logits"].detach(), case["score"])
    s32 = sc.float()
    c = s32 + s["bias"] if s["bias"] is not None else s32
    if G > 1:
        top = torch.sort(c.view(T, G, E // G), dim=-1, descending=True).values
        best = torch.sort(top[..., :2].sum(-1), dim=-1, descending=True, stable=True).indices[:, :keep]
        stays = torch.zeros(T, G, dtype=torch.bool, device=DEV).scatter_(1, best, True)
        c = torch.where(stays[..., None], c.view(T, G, E // G), float("-inf")).view(T, E)
    idx = torch.sort(c, dim=-1, descending=True, stable=True).indices[:, :k]
    sel = s32.gather(1, idx)
    total = sel.sum(-1, keepdim=True).clamp(min=1e-10) if case["normalise"] else 1.0
    w = sel / total * 2.5
    counts = torch.zeros(E, dtype=torch.int32, device=DEV).index_add_(0, idx.reshape(-1), torch.ones(T * k, dtype=torch.int32, device=DEV))
    if not case["train"]:
        return w, idx.to(torch.int32), counts
    ds = s["dw"] * 2.5 / total
    if case["normalise"]:
        ds = ds - (ds * sel).sum(-1, keepdim=True) / total
    if case["score"] == "sigmoid":
        dl = torch.zeros_like(s32).scatter_(1, idx, ds * sel * (1.0 - sel))
    else:
        dl = s32 * (torch.zeros_like(s32).scatter_(1, idx, ds) - (ds * sel).sum(-1, keepdim=True))
    return w, idx.to(torch.int32), counts, dl


# ---------------------------------------------------------------------------- work, exact results
def work(case):
    if case["op"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        nbytes = 4 * T * E + 8 * T * k + 8 * E
        if case["train"]:
            nbytes += 4 * T * k + 4 * T * E
        return {"bytes": nbytes, "flops": 4 * T * E}
    new, kv = _lengths(case)
    T, R, Dr = sum(new), case["R"], case["Dr"]
    if case["op"] == "append":
        return {"bytes": 4 * T * (R + Dr) + 4 * (2 * len(kv) + 1) + 4 * sum(new), "flops": 4 * T * R if case["norm"] else 0}
    H, Dn, Dv = case["H"], case["Dn"], case["Dv"]
    up = 2 * R * (Dn + Dv)
    flops = 0
    for n, m in zip(new, kv):
        pairs = n * (m - n) + n * (n + 1) // 2
        # through the latent rows, or with keys and values of every head: the cheaper of the two
        flops += H * min(n * up + pairs * 2 * (2 * R + Dr), m * up + pairs * 2 * (Dn + Dr + Dv))
    nbytes = 2 * sum(kv) * (R + Dr) + 2 * T * H * (Dn + Dr + Dv) + 2 * H * (Dn + Dv) * R
    return {"bytes": nbytes, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(s, case)
    new, kv = _lengths(case)
    page = case["page"]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    if case["op"] == "append":
        pools = [s["kv_pages"].double(), s["pe_pages"].double()]
        for b, (n, m) in enumerate(zip(new, kv)):
            rows = slice(starts[b], starts[b + 1])
            c = s["ctx_kv"][rows].double()
            if s["norm"] is not None:
                c = c / torch.sqrt(c.square().sum(1, keepdim=True) / case["R"] + EPS) * s["norm"].double()
            pos = torch.arange(m - n, m, device=DEV)
            slot = s["table"][b].long()[pos // page] * page + pos % page
            for pool, new_rows in zip(pools, (c, s["ctx_pe"][rows].double())):
                pool.view(-1, pool.shape[-1])[slot] = new_rows
        return tuple(pools)
    out = []
    for b, (n, m) in enumerate(zip(new, kv)):
        pages = s["table"][b, :-(-m // page)].long()
        c, pe = (x[pages].reshape(-1, x.shape[-1])[:m].double() for x in (s["kv_pages"], s["pe_pages"]))
        rows = slice(starts[b], starts[b + 1])
        hidden = torch.arange(m, device=DEV)[None] > torch.arange(m - n, m, device=DEV)[:, None]
        heads = []
        for h in range(case["H"]):
            # through the latent rows: (q W_k) . c and (sum p c) W_v^T
            z = (s["q_nope"][rows, h].double() @ s["w_k"][h].double()) @ c.T + s["q_pe"][rows, h].double() @ pe.T
            p = torch.softmax((z * s["scale"]).masked_fill(hidden, float("-inf")), dim=-1)
            heads.append((p @ c) @ s["w_v"][h].double().T)
        out.append(torch.stack(heads, 1))
    return torch.cat(out)


def _exact_route(s, case):
    """The choice is defined on scores rounded to 32 bits (plus the bias in 32 bits); weights and gradients in 64."""
    T, E, k, G = (case[n] for n in ("T", "E", "k", "groups"))
    x = s["logits"].detach().double().requires_grad_(case["train"])
    full = torch.sigmoid(x) if case["score"] == "sigmoid" else torch.softmax(x, dim=-1)
    c = full.detach().float()
    if s["bias"] is not None:
        c = c + s["bias"]
    ids = torch.arange(E, device=DEV)
    if G > 1:
        pairs = c.view(T, G, E // G).topk(min(2, E // G), dim=-1).values.sum(-1)
        # a group stays where fewer than `keep` others come before it
        before = (pairs[:, None, :] > pairs[:, :, None]) | ((pairs[:, None, :] == pairs[:, :, None]) & (ids[:G] < ids[:G, None]))
        gone = (before.sum(-1) >= case["keep"]).repeat_interleave(E // G, dim=1)
        c = c.masked_fill(gone, float("-inf"))
    idx = torch.empty(T, k, dtype=torch.int64, device=DEV)
    for j in range(k):
        top = c == c.amax(-1, keepdim=True)
        idx[:, j] = torch.where(top, ids, E).amin(-1)
        c = c.scatter(1, idx[:, j:j + 1], float("-inf"))
    w = full.gather(1, idx) * 2.5
    if case["normalise"]:
        w = w / (w.sum(-1, keepdim=True) / 2.5).clamp(min=1e-10)
    counts = torch.bincount(idx.reshape(-1), minlength=E).to(torch.int32)
    got = (w.detach(), idx.to(torch.int32), counts)
    return got + (torch.autograd.grad(w, x, s["dw"].double())[0],) if case["train"] else got
