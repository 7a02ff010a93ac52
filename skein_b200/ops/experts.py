"""Choice of experts with a balance bias, and the expert-sorted layout that the experts' products read.

`route_balanced` is the router of models whose load is balanced by a bias on the scores instead of a loss: the bias decides who is chosen, the weights
come from the scores without it. It takes up to 512 experts; `ops.route`, `ops.latent.route_grouped` and `ops.prenorm.route` are the routers without
a bias, up to 64 experts, with the router's product in the call. On CPU tensors the reference in reference_int4.py runs.
"""
from __future__ import annotations

import torch

from . import _lib, reference_int4 as ri

MAX_EXPERTS, MAX_TOP, MAX_GROUPS = 512, 16, 64
SCORES = ("softmax", "sigmoid")
ONE_LAUNCH = 256       # tokens up to which one kernel does it all, without scratch


def route_balanced(logits, top, bias=None, groups=1, keep=1, score="sigmoid", group_best=2, renorm=True, scale=1.0, e_first=0, e_count=None):
    """Experts of every token from its router logits [T, E] (fp32 or bf16, rows may be strided), and the expert-sorted layout.

    s is the sigmoid or the softmax of the logits, c = s + bias (fp32 [E]). With groups > keep, the experts are `groups` equal groups of neighbours, a
    group is worth the sum of its `group_best` (1 or 2) largest c, and the `keep` best groups are eligible. The `top` largest c are chosen in descending
    order, ties to the lower index; their weights are scale * s, divided by the sum of the chosen s (+ 1e-20) with renorm. Scores and choices are 64-bit;
    logits and biases that are not numbers count as the lowest, infinite ones as +-3e38.

    Returns (ids int32 [T, top], weights fp32 [T, top], counts [E], offsets [E + 1], row_of [T * top], src_token [T * top]) as `ops.route` does: pair
    (t, j) sits at row_of[t * top + j] of the expert-sorted rows (-1: an expert outside e_first .. + e_count), src_token is its inverse; rows of
    src_token from offsets[E] on are unset. On a GPU the six lie in one allocation, which lives as long as any of them, and a call takes at most
    227,328 tokens (148 tiles of 1536)."""
    dtype = logits.dtype
    if logits.dim() != 2 or dtype not in (torch.float32, torch.bfloat16) or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("route_balanced: logits must be [tokens, experts] fp32 or bf16 with contiguous rows")
    T, E = logits.shape
    e_count = E - e_first if e_count is None else e_count
    if not 1 <= E <= MAX_EXPERTS or not 1 <= groups <= MAX_GROUPS or E % groups or not 1 <= keep <= groups:
        raise ValueError(f"route_balanced: {E} experts in {groups} groups of which {keep} are kept (at most {MAX_EXPERTS} experts, {MAX_GROUPS} groups)")
    if not 1 <= top <= min(MAX_TOP, keep * (E // groups)):
        raise ValueError(f"route_balanced: top {top} of {keep * (E // groups)} eligible experts (at most {MAX_TOP})")
    if score not in SCORES or group_best not in (1, 2):
        raise ValueError(f"route_balanced: score is one of {SCORES}, group_best 1 or 2")
    if e_first < 0 or e_count < 0 or e_first + e_count > E:
        raise ValueError("route_balanced: experts e_first .. e_first + e_count lie outside the router's")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (E,) or not bias.is_contiguous() or bias.device != logits.device):
        raise ValueError("route_balanced: bias must be fp32 [experts] on the logits' device")
    if not logits.is_cuda:
        return ri.route_balanced(logits, top, bias, groups, keep, score, group_best, renorm, scale, e_first, e_count)
    dev, n = logits.device, T * top
    with _lib.on_device(logits):
        L = _lib.lib()
        need = L.skein_route_balanced_scratch(T, E) if T > ONE_LAUNCH else 0
        if need < 0:
            raise ValueError(f"route_balanced: {T} tokens are more than one call takes")
        scratch = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        buf = torch.empty(4 * n + 2 * E + 1, dtype=torch.int32, device=dev)      # all results: an allocation costs more than a view
        at = buf.data_ptr()
        rc = L.skein_route_balanced(
            logits.data_ptr(), logits.stride(0), dtype == torch.bfloat16, None if bias is None else bias.data_ptr(), T, E, top, groups, keep, group_best,
            renorm, score == "sigmoid", scale, e_first, e_count, at, at + 4 * n, at + 8 * n, at + 8 * n + 4 * E, at + 8 * n + 8 * E + 4,
            at + 12 * n + 8 * E + 4, scratch.data_ptr() if need else None, _lib.stream_on(dev))
    _lib.check(rc, "route_balanced")
    _lib.count_launch(2 if need else 1)
    ids, w, counts, offsets, row_of, src_token = buf.split_with_sizes((n, n, E, E + 1, n, n))
    return ids.view(T, top), w.view(torch.float32).view(T, top), counts, offsets, row_of, src_token
