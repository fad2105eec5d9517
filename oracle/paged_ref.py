"""CPU restatement of the paged latent cache and its attention — TEST INFRASTRUCTURE ONLY.

Parity oracle for ``dsmoe.mla.mla_cache_append`` and ``dsmoe.mla.mla_attention_paged``
(csrc/mla_cache.hip, csrc/mla_paged.hip), in float64 from the definition: no counterpart in the reference,
whose cache is one contiguous tensor per batch row (models/mla.py:95-125); the attention of one sequence is
``mla_ref.mla_attention_oracle`` with the causal mask, which the tests pin it against.

Sequence b's new tokens are the rows offsets[b] .. offsets[b + 1] - 1 and stand at the last positions of its
kv_lens[b]; position p lies on page table[b][p // page_size].  A token without a place is not written; a
position without one is not seen; a token that sees none gives zeros.
"""
from __future__ import annotations

import torch


def _sequences(table, kv_lens, offsets, T):
    for b, kv in enumerate(kv_lens.tolist()):
        t0, t1 = (min(max(int(o), 0), T) for o in offsets[b:b + 2])
        n, kv = max(t1 - t0, 0), max(kv, 0)
        yield b, t0, n, kv - n, kv


def _slot(table, b, pos, pages, page_size):
    """(page, row) of a position, or None."""
    if pos < 0 or pos // page_size >= table.shape[1]:
        return None
    page = int(table[b, pos // page_size])
    return (page, pos % page_size) if 0 <= page < pages else None


def append_ref(ctx_kv, ctx_pe, kv_pages, pe_pages, table, kv_lens, offsets, norm_weight=None, eps=1e-6):
    """The pools after the call, in float64 (unrounded new rows), and a mask of the rows written."""
    c = ctx_kv.double()
    if norm_weight is not None:
        c = c / torch.sqrt((c * c).mean(1, keepdim=True) + eps) * norm_weight.double()
    kv, pe = kv_pages.double().clone(), pe_pages.double().clone()
    written = torch.zeros(kv.shape[:2], dtype=torch.bool)
    for b, t0, n, first, _ in _sequences(table, kv_lens, offsets, ctx_kv.shape[0]):
        for i in range(n):
            at = _slot(table, b, first + i, kv.shape[0], kv.shape[1])
            if at is not None:
                kv[at], pe[at], written[at] = c[t0 + i], ctx_pe[t0 + i].double(), True
    return kv, pe, written


def attend_ref(q_nope, q_pe, kv_pages, pe_pages, table, kv_lens, offsets, w_k, w_v, scale):
    """(out, spread, size) in float64: out (T, H, Dv), NaN in rows behind the last sequence; spread = sum_j p_j |v_j|
    (T, H, Dv) and size (T, H), the largest sum of absolute terms of a row's scores, for error bounds."""
    T, H, _ = q_nope.shape
    Dv = w_v.shape[1]
    out = torch.full((T, H, Dv), float("nan"), dtype=torch.float64)
    spread, size = torch.zeros_like(out), torch.zeros(T, H, dtype=torch.float64)
    qn, qp, wk, wv = (t.double() for t in (q_nope, q_pe, w_k, w_v))
    P, page = kv_pages.shape[:2]
    for b, t0, n, first, kv in _sequences(table, kv_lens, offsets, T):
        if n == 0:
            continue
        slots = [(j, _slot(table, b, j, P, page)) for j in range(min(kv, table.shape[1] * page))]
        seen = [(j, s) for j, s in slots if s is not None]
        rows = slice(t0, t0 + n)
        if not seen:
            out[rows] = 0.0
            continue
        pos = torch.tensor([j for j, _ in seen])
        pg, ip = torch.tensor([s[0] for _, s in seen]), torch.tensor([s[1] for _, s in seen])
        c, pe = kv_pages[pg, ip].double(), pe_pages[pg, ip].double()
        visible = pos[None] <= first + torch.arange(n)[:, None]
        for h in range(H):
            k, v = c @ wk[h].T, c @ wv[h].T
            z = ((qn[rows, h] @ k.T + qp[rows, h] @ pe.T) * scale).masked_fill(~visible, float("-inf"))
            top = torch.nan_to_num(z, nan=0.0, neginf=-1e300).amax(1, keepdim=True)
            p = torch.where(visible, torch.exp(z - top), 0.0)
            l = p.sum(1, keepdim=True)
            p = torch.where(l == 0, p, p / l)
            for i in range(n):
                on = visible[i]
                out[t0 + i, h] = p[i, on] @ v[on]
                spread[t0 + i, h] = p[i, on] @ v[on].abs()
            terms = (qn[rows, h].abs() @ wk[h].abs()) @ c.abs().T + qp[rows, h].abs() @ pe.abs().T
            size[rows, h] = (abs(scale) * terms * visible).amax(1)
    return out, spread, size
