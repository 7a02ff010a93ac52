"""Plain PyTorch reference of the 4-bit products and of the balanced choice of experts (ops/int4.py, ops/experts.py)."""
from __future__ import annotations

import torch

from . import reference as ref


def dequant(codes, scale, zero, group):
    """codes [..., rows, K / 2] (even k in the low half of a byte), scale [..., rows, K / group] -> fp32 [..., rows, K]."""
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    z = 8.0 if zero is None else zero.float().repeat_interleave(group, -1)
    return (q - z) * scale.float().repeat_interleave(group, -1)


def product(x, w, residual=None, out_f32=False, swiglu=False):
    """x [T, K], w fp32 [rows, K] (gate rows, then up rows with swiglu)."""
    y = x.float() @ w.t()
    if swiglu:
        g, u = y.chunk(2, -1)
        y = torch.nn.functional.silu(g) * u
    if residual is not None:
        y = y + residual.float()
    return y if out_f32 else y.to(torch.bfloat16)


def grouped_product(x, w, counts, offsets, swiglu, src_row, out):
    """Rows offsets[e] .. + counts[e] of `out` from rows of x (by src_row, or the same ones); the others stay."""
    ends = [(e, o, o + c) for e, (c, o) in enumerate(zip(counts.tolist(), offsets.tolist())) if c]
    for e, a, b in ends:
        named = src_row[max(a, 0):max(b, 0)] if src_row is not None else None
        if a < 0 or b < a or b > out.shape[0] or (named is not None and bool(((named < 0) | (named >= x.shape[0])).any())):
            raise ValueError(f"int4 grouped_linear: index out of range at expert {e}")
    for e, a, b in ends:
        rows = x[a:b] if src_row is None else x[src_row[a:b].long()]
        out[a:b] = product(rows, w[e], swiglu=swiglu)
    return out


def select_balanced(logits, top, bias, groups, keep, score, group_best, renorm, scale):
    """(ids int32 [T, top], weights fp32 [T, top]); see ops/experts.py."""
    T, E = logits.shape
    z = logits.double()
    z = torch.where(z == z, z, torch.full_like(z, -3e38)).clamp(-3e38, 3e38)
    s = torch.sigmoid(z) if score == "sigmoid" else torch.softmax(z, 1)
    c = s if bias is None else s + torch.where(bias == bias, bias, torch.full_like(bias, -3e38)).clamp(-3e38, 3e38).double()
    if keep < groups:
        per = E // groups
        worth = c.view(T, groups, per).sort(dim=2, descending=True).values[:, :, :min(group_best, per)].sum(2)
        best = worth.sort(dim=1, descending=True, stable=True).indices[:, :keep]
        kept = torch.zeros(T, groups, dtype=torch.bool, device=z.device).scatter_(1, best, True)
        c = c.masked_fill(~kept.repeat_interleave(per, 1), -float("inf"))
    ids = c.sort(dim=1, descending=True, stable=True).indices[:, :top]
    w = s.gather(1, ids) * scale
    if renorm:
        w = w / (s.gather(1, ids).sum(1, keepdim=True) + 1e-20)
    return ids.to(torch.int32), w.float()


def route_balanced(logits, top, bias, groups, keep, score, group_best, renorm, scale, e_first, e_count):
    ids, w = select_balanced(logits, top, bias, groups, keep, score, group_best, renorm, scale)
    counts, offsets, row_of, src = ref.router_plan(ids, logits.shape[1], e_first, e_count)
    src_token = src.new_zeros(row_of.shape)      # (of every pair, as on the GPU: a product's result has as many rows)
    src_token[:int(offsets[-1])] = src[:int(offsets[-1])]
    return ids, w, counts, offsets, row_of, src_token
