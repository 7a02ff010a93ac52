"""4-bit weights and the balanced choice of experts on the CPU: packing, references, refusals."""
import pytest
import torch

from skein_b200.ops import experts, int4, reference as ref, reference_int4 as ri

GEN = torch.Generator().manual_seed(5)


def parts(lead, rows, K, group, zeros, scales=torch.float16):
    codes = torch.randint(0, 256, (*lead, rows, K // 2), generator=GEN, dtype=torch.uint8)
    scale = (torch.rand(*lead, rows, K // group, generator=GEN) + 0.1).to(scales)
    zero = torch.randint(0, 16, (*lead, rows, K // group), generator=GEN, dtype=torch.uint8) if zeros else None
    return codes, scale, zero


@pytest.mark.parametrize("lead, rows, K, group, pair, zeros", [
    ((), 1, 32, 32, False, False), ((), 50, 96, 32, False, True), ((3,), 22, 256, 128, True, False), ((2,), 34, 192, 64, True, True),
    ((), 16, 128, 64, False, False), ((1,), 2, 128, 128, True, True),
    ((2,), 16 * 17 + 5, 160, 32, False, True), ((), 2 * 8 * 8, 256, 64, True, False), ((3,), 2 * 77, 96, 32, True, True)])
def test_packing_keeps_every_code_scale_and_zero(lead, rows, K, group, pair, zeros):
    given = parts(lead, rows, K, group, zeros)
    w = int4.pack_weight(*given, pair=pair)
    for a, b in zip(given, w.parts()):
        assert (a is None and b is None) or torch.equal(a, b)
    assert w.shape == (*lead, rows, K) and w.features == (rows // 2 if pair else rows)


def test_place_of_a_code():
    """csrc/kernels/int4.cuh: code of row 16 s + 8 half + g, k = 128 b + 64 j + 32 h + 8 t + i."""
    codes, scale, zero = parts((), 40, 384, 64, True)
    w = int4.pack_weight(codes, scale, zero)
    assert w.data.shape == (1, 1, 3, 8 * (1024 + 64 + 32))
    for row, k in ((0, 0), (7, 9), (8, 0), (39, 383), (17, 200), (26, 127), (33, 256 + 77)):
        s, half, g = row // 16, row % 16 // 8, row % 8
        b, j, h, t, i = k // 128, k % 128 // 64, k % 64 // 32, k % 32 // 8, k % 8
        step = w.data[0, 0, b]
        word = int(step[:8192].view(torch.int32)[((s * 2 + j) * 32 + t * 8 + g) * 4 + 2 * half + h]) & 0xffffffff
        assert word >> (4 * (i // 2) + 16 * (i % 2)) & 15 == int(codes[row, k // 2]) >> (4 * (k % 2)) & 15
        at = ((s * 8 + g) * 2 + k % 128 // 64) * 2 + half
        assert step[8192:8704].view(torch.float16)[at] == scale[row, k // 64] and step[8704:][at] == zero[row, k // 64]


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantised_weight_is_within_half_a_step(symmetric, group):
    w = torch.randn(24, 256, generator=GEN)
    w[3] = 0
    q = int4.quantize_weight(w, group, symmetric)
    # half a step, plus the rounding of the scale to bf16 (2^-9 of a scale, over at most 15 steps); a zero that is rounded moves the range by half a step
    step = q.parts()[1].float().repeat_interleave(group, -1)
    most = step * (0.5 + 15 * 2.0 ** -9 + (0 if symmetric else 0.5))
    assert bool(((q.dequant() - w).abs() <= most).all()) and bool((q.dequant()[3] == 0).all())


@pytest.mark.parametrize("rows, T, pair", [(5, 0, False), (5, 3, False), (12, 7, True)])
def test_cpu_products(rows, T, pair):
    codes, scale, zero = parts((), rows, 64, 32, True, torch.bfloat16)
    w = int4.pack_weight(codes, scale, zero, pair=pair)
    x = torch.randn(T, 64, generator=GEN).bfloat16()
    full = ri.dequant(codes, scale, zero, 32)
    if pair:
        assert torch.equal(int4.swiglu_linear(x, w), ref.swiglu_linear(x, full))
        return
    assert torch.equal(int4.linear(x, w), ref.linear(x, full))
    r = torch.randn(T, rows, generator=GEN)
    assert torch.equal(int4.linear(x, w, residual=r, out_f32=True), ref.linear(x, full, r, True))


def test_cpu_experts_read_their_rows():
    codes, scale, zero = parts((4,), 6, 64, 64, False)
    w = int4.pack_weight(codes, scale, zero)
    x = torch.randn(5, 64, generator=GEN).bfloat16()
    ids = torch.tensor([[0, 3], [3, 1], [1, 0], [3, 0], [0, 1]], dtype=torch.int32)
    counts, offsets, row_of, src = ref.router_plan(ids, 4)
    y = int4.grouped_linear(x, w, counts, offsets, src_row=src)
    assert torch.equal(y, int4.grouped_linear(x[src.long()], w, counts, offsets))
    assert torch.equal(y, ref.grouped_linear(x[src.long()], w.dequant(), counts, offsets))
    kept = torch.full((10, 6), 7.0, dtype=torch.bfloat16)
    int4.grouped_linear(x[src.long()], w, counts * 0, offsets, out=kept)
    assert bool((kept == 7).all())


def test_weight_refusals():
    codes, scale, zero = parts((), 8, 128, 64, True)
    good = int4.pack_weight(codes, scale, zero)
    bad = [lambda: int4.pack_weight(codes.int(), scale), lambda: int4.pack_weight(codes, scale.float()), lambda: int4.pack_weight(codes, scale[:, :1].repeat(1, 8)),
           lambda: int4.pack_weight(codes, scale[:4]), lambda: int4.pack_weight(codes, scale, zero + 16), lambda: int4.pack_weight(codes, scale, zero[:, :1]),
           lambda: int4.pack_weight(codes[:7], scale[:7], pair=True), lambda: int4.quantize_weight(torch.zeros(4, 100)),
           lambda: int4.quantize_weight(torch.zeros(4, 128), group=16), lambda: good.copy_(int4.pack_weight(codes, scale))]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_product_refusals():
    codes, scale, zero = parts((2,), 8, 64, 64, False)
    many, one, pair = int4.pack_weight(codes, scale), int4.pack_weight(codes[0], scale[0]), int4.pack_weight(codes[0], scale[0], pair=True)
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    n = torch.tensor([2, 2], dtype=torch.int32)
    bad = [lambda: int4.linear(x, many), lambda: int4.linear(x, pair), lambda: int4.swiglu_linear(x, one), lambda: int4.linear(x.float(), one),
           lambda: int4.linear(x[:, :32], one), lambda: int4.linear(torch.zeros(64, 4, dtype=torch.bfloat16).t(), one),
           lambda: int4.linear(x, one, out=torch.zeros(4, 8)), lambda: int4.linear(x, one, out=torch.zeros(1, 8, dtype=torch.bfloat16).expand(4, 8)),
           lambda: int4.linear(x, one, residual=torch.zeros(4, 8)), lambda: int4.linear(x, one, residual=torch.zeros(8, 4, dtype=torch.bfloat16).t()),
           lambda: int4.grouped_linear(x, one, n, n), lambda: int4.grouped_linear(x, many, n.long(), n), lambda: int4.grouped_linear(x, many, n[:1], n),
           lambda: int4.grouped_linear(x, many, n, n, swiglu=True), lambda: int4.grouped_linear(x, many, n, n, src_row=n.long())]
    bad += [lambda: int4.linear(x, one, out=x[:, :8]), lambda: int4.grouped_linear(x, many, n, n, out=x[:, :8])]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def _select_one(z, bias, top, groups, keep, score, best, renorm, scale):
    """One token, from the definition."""
    z = [-3e38 if v != v else max(-3e38, min(3e38, v)) for v in z]
    t = torch.tensor(z, dtype=torch.float64)
    s = (torch.sigmoid(t) if score == "sigmoid" else torch.softmax(t, 0)).tolist()
    c = [a + b for a, b in zip(s, bias)]
    per = len(z) // groups
    worth = [sum(sorted(c[g * per:(g + 1) * per], reverse=True)[:best]) for g in range(groups)]
    kept = sorted(range(groups), key=lambda g: (-worth[g], g))[:keep]
    ids = sorted((e for e in range(len(z)) if e // per in kept), key=lambda e: (-c[e], e))[:top]
    tot = sum(s[e] for e in ids) + 1e-20
    return ids, [s[e] * scale / (tot if renorm else 1) for e in ids]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E, top, groups, keep, best", [(1, 1, 1, 1, 2), (8, 2, 1, 1, 1), (24, 5, 4, 2, 2), (24, 5, 4, 2, 1), (6, 2, 6, 3, 2)])
def test_balanced_choice_on_the_cpu(score, E, top, groups, keep, best):
    z = torch.randn(9, E, generator=GEN)
    z[0, E // 2] = float("nan")
    z[1] = -float("inf")
    z[2, :] = z[2, 0]
    bias = torch.randn(E, generator=GEN) * 0.2
    for b in (None, bias):
        ids, w, counts, offsets, row_of, src = experts.route_balanced(z, top, bias=b, groups=groups, keep=keep, score=score, group_best=best, scale=2.5)
        for t in range(9):
            want = _select_one(z[t].tolist(), [0.0] * E if b is None else b.double().tolist(), top, groups, keep, score, best, True, 2.5)
            assert ids[t].tolist() == want[0]
            assert torch.allclose(w[t].double(), torch.tensor(want[1], dtype=torch.float64), rtol=2.0 ** -23, atol=0)
        assert torch.equal(src[row_of.long()], torch.arange(9 * top, dtype=torch.int32) // top) and int(counts.sum()) == int(offsets[-1]) == 9 * top


def test_router_refusals():
    z = torch.zeros(3, 16)
    ok = dict(top=2)
    bad = [dict(top=0), dict(top=17), dict(top=5, groups=4, keep=1), dict(top=2, groups=5), dict(top=2, groups=4, keep=5), dict(top=2, score="tanh"),
           dict(top=2, group_best=3), dict(top=2, bias=torch.zeros(15)), dict(top=2, bias=torch.zeros(16, dtype=torch.float64)), dict(top=2, e_first=10, e_count=7)]
    experts.route_balanced(z, **ok)
    for kw in bad:
        with pytest.raises(ValueError):
            experts.route_balanced(z, **kw)
    for logits in (z.half(), z.t(), torch.zeros(2, 513), z[0]):
        with pytest.raises(ValueError):
            experts.route_balanced(logits, 2)
