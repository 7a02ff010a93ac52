"""4-bit products and the balanced choice of experts on the GPU, against 64 bits."""
import pytest
import torch

from skein_b200 import ops
from skein_b200.ops import experts, int4, reference_int4 as ri

pytestmark = pytest.mark.gpu
DEV = "cuda"


def weight(lead, rows, K, group, zeros, scales, pair, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 256, (*lead, rows, K // 2), generator=gen, device=DEV, dtype=torch.uint8)
    scale = (torch.rand(*lead, rows, K // group, generator=gen, device=DEV) * 0.02 + 0.005).to(scales)
    zero = torch.randint(0, 16, (*lead, rows, K // group), generator=gen, device=DEV, dtype=torch.uint8) if zeros else None
    return int4.pack_weight(codes, scale, zero, pair=pair), ri.dequant(codes, scale, zero, group).double()


def acts(rows, K, seed=1):
    return torch.randn(rows, K, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).bfloat16()


def within(y, x, w, pair=False, residual=None, half_step=2.0 ** -8):
    """|y - exact| against the bound of the arithmetic: K sums in 32 bits, each off by at most a step (2^-23, the tensor cores cut off) of the sum of
    magnitudes, and one rounding of the result. A pair adds what its two sums' errors do through silu (slope at most 1.1) and the error of a
    fast exponential (2^-20)."""
    x = x.double()
    K = x.shape[1]
    exact, size = x @ w.t(), x.abs() @ w.abs().t()
    d = K * 2.0 ** -23 * size
    if pair:
        g, u = exact.chunk(2, 1)
        dg, du = d.chunk(2, 1)
        s = g * torch.sigmoid(g)
        exact = s * u
        d = 1.1 * dg * (u.abs() + du) + s.abs() * du + 2.0 ** -20 * exact.abs()
    if residual is not None:
        exact = exact + residual.double()
        d = d + 2.0 ** -24 * exact.abs()
    off = (y.double() - exact).abs() - d - half_step * (exact.abs() + d)
    assert bool((off <= 0).all()), (float(off.max()), int((off > 0).sum()))


SIZES = [  # rows, features, K, group, zeros, scales
    (1, 16, 128, 128, False, torch.bfloat16), (1, 1, 32, 32, True, torch.float16), (3, 17, 96, 32, True, torch.bfloat16), (8, 130, 384, 64, True, torch.float16),
    (9, 200, 1408, 128, False, torch.bfloat16), (16, 64, 4096, 128, True, torch.float16), (17, 48, 256, 32, False, torch.bfloat16), (33, 1000, 512, 64, False, torch.bfloat16),
    (64, 256, 3584, 128, True, torch.bfloat16), (100, 129, 640, 128, False, torch.float16), (257, 384, 1056, 32, True, torch.float16), (130, 513, 2048, 64, True, torch.bfloat16)]


@pytest.mark.parametrize("rows, features, K, group, zeros, scales", SIZES)
def test_linear(rows, features, K, group, zeros, scales):
    w, full = weight((), features, K, group, zeros, scales, False)
    assert torch.equal(w.dequant().double(), full)
    x = acts(rows, K)
    within(int4.linear(x, w), x, full)
    within(int4.linear(x, w, out_f32=True), x, full, half_step=2.0 ** -24)
    r = torch.randn(rows, features, device=DEV)
    within(int4.linear(x, w, residual=r, out_f32=True), x, full, residual=r, half_step=2.0 ** -24)
    rb = r.bfloat16()
    keep = rb.clone()
    assert int4.linear(x, w, residual=rb, out=rb) is rb
    within(rb, x, full, residual=keep)


KERNELS = [(0, 0), (16, 1), (16, 2), (16, 8), (32, 1), (32, 4), (64, 1), (64, 8), (128, 1), (128, 2), (128, 8)]


@pytest.mark.parametrize("cfg", KERNELS)
@pytest.mark.parametrize("rows, features, K, group, zeros, scales", [SIZES[1], SIZES[2], SIZES[3], SIZES[6], SIZES[10], SIZES[11]])
def test_every_kernel_takes_every_size(rows, features, K, group, zeros, scales, cfg):
    w, full = weight((), features, K, group, zeros, scales, False)
    x = acts(rows, K)
    within(int4.linear(x, w, out_f32=True, _cfg=cfg), x, full, half_step=2.0 ** -24)
    w, full = weight((3,), 2 * features, K, group, zeros, scales, True)
    cnt = torch.tensor([rows, 0, 2 * rows], dtype=torch.int32, device=DEV)
    off = torch.tensor([0, rows, rows, 3 * rows], dtype=torch.int32, device=DEV)
    src = torch.randint(0, rows, (3 * rows,), device=DEV, dtype=torch.int32)
    y = int4.grouped_linear(x, w, cnt, off, swiglu=True, src_row=src, _cfg=cfg)
    within(y[:rows], x[src[:rows].long()], full[0], True)
    within(y[rows:], x[src[rows:].long()], full[2], True)
    ops.workspace().check_status()


@pytest.mark.parametrize("rows, features, K, group, zeros, scales", SIZES)
def test_swiglu_linear(rows, features, K, group, zeros, scales):
    w, full = weight((), 2 * features, K, group, zeros, scales, True)
    x = acts(rows, K)
    within(int4.swiglu_linear(x, w), x, full, pair=True)


@pytest.mark.parametrize("rows", [1, 7, 40, 150])
def test_strides_and_alignment(rows):
    w, full = weight((), 96, 256, 64, True, torch.bfloat16, False)
    wide = acts(rows, 600)
    for first in (0, 8, 1, 3):             # on and off 16-byte boundaries
        x = wide[:, first:first + 256]
        out = torch.full((rows, 200), 5.0, device=DEV, dtype=torch.bfloat16)
        int4.linear(x, w, out=out[:, 50:146])
        within(out[:, 50:146], x, full)
        assert bool((out[:, :50] == 5).all()) and bool((out[:, 146:] == 5).all())
    odd = acts(rows, 257)[:, :256]         # rows of 514 bytes
    within(int4.linear(odd, w), odd, full)
    within(int4.linear(wide[:1, :256].expand(rows, 256), w), wide[:1, :256].expand(rows, 256), full)


def test_long_rows():
    """Rows that the kernel of few rows has no place for go to the other one, or are refused where that cannot read them."""
    K = int4.MAX_ROW + 32768
    w, full = weight((2,), 48, K, 128, True, torch.bfloat16, False)
    wide = acts(3, K + 8)
    x = wide[:, :K]
    cnt, off = torch.tensor([1, 2], dtype=torch.int32, device=DEV), torch.tensor([0, 1, 3], dtype=torch.int32, device=DEV)
    y = int4.grouped_linear(x, w, cnt, off)
    within(y[:1], x[:1], full[0])
    within(y[1:], x[1:], full[1])
    with pytest.raises(ValueError, match="16-byte"):
        int4.grouped_linear(wide[:, 1:K + 1], w, cnt, off)
    w, full = weight((), 48, int4.MAX_ROW, 128, True, torch.bfloat16, False)
    within(int4.linear(wide[:, 1:int4.MAX_ROW + 1], w), wide[:, 1:int4.MAX_ROW + 1], full)
    w, full = weight((), 16, K, 128, True, torch.bfloat16, False)
    odd = wide.view(-1)[:2 * K + 1].as_strided((1, K), (K + 1, 1))      # the stride of one row says nothing
    within(int4.linear(odd, w), odd, full)
    ops.workspace().check_status()


@pytest.mark.parametrize("rows", [4, 40])
def test_a_row_that_is_no_number_stays_alone(rows):
    w, full = weight((), 64, 256, 128, False, torch.bfloat16, False)
    x = acts(rows, 256)
    x[1, 5], x[2, 255] = float("nan"), float("inf")
    y = int4.linear(x, w)
    assert bool(y[1].isnan().all()) and not bool(y[2].isfinite().any())
    others = [r for r in range(rows) if r not in (1, 2)]
    within(y[others], x[others], full)


EXPERTS = [  # counts, features, K, group, zeros, scales, pair
    ([1], 32, 128, 128, False, torch.bfloat16, False), ([0, 1, 0, 1], 64, 256, 64, True, torch.float16, True), ([3, 0, 9, 20, 1, 0], 40, 384, 128, False, torch.bfloat16, False),
    ([0, 0, 50, 0], 24, 160, 32, True, torch.bfloat16, True), ([130, 1, 0, 77], 136, 512, 128, True, torch.float16, False), ([200, 3, 260], 72, 256, 64, False, torch.bfloat16, True),
    ([1, 0, 2] * 30, 48, 128, 64, False, torch.float16, False), ([0, 0], 16, 128, 128, False, torch.bfloat16, True)]


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("hint", [None, 1, 10 ** 6])
@pytest.mark.parametrize("counts, features, K, group, zeros, scales, pair", EXPERTS)
def test_grouped_linear(counts, features, K, group, zeros, scales, pair, hint, gather):
    E, spare = len(counts), 3
    w, full = weight((E,), features * (2 if pair else 1), K, group, zeros, scales, pair)
    n = sum(counts)
    cnt = torch.tensor(counts, dtype=torch.int32, device=DEV)
    off = torch.cat((cnt.new_zeros(1), cnt.cumsum(0))).to(torch.int32)
    tokens = max(1, n // 2)
    x = acts(tokens if gather else n + spare, K)
    src = torch.randint(0, tokens, (n + spare,), device=DEV, dtype=torch.int32) if gather else None
    out = torch.full((n + spare, features), 3.0, device=DEV, dtype=torch.bfloat16)
    int4.grouped_linear(x, w, cnt, off, swiglu=pair, src_row=src, out=out, rows_hint=hint)
    rows = x[src.long()] if gather else x
    for e in range(E):
        a, b = int(off[e]), int(off[e + 1])
        if a < b:
            within(out[a:b], rows[a:b], full[e], pair)
    assert bool((out[n:] == 3).all())
    ops.workspace().check_status()


def test_rows_outside_are_reported():
    w, _ = weight((2,), 32, 128, 128, False, torch.bfloat16, False)
    x = acts(4, 128)
    n = torch.tensor([2, 2], dtype=torch.int32, device=DEV)
    off = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    for counts, offsets, src in ((n, off, torch.tensor([0, 4, 1, 2], dtype=torch.int32, device=DEV)), (n, off, torch.tensor([0, -1, 1, 2], dtype=torch.int32, device=DEV)),
                                 (n + 1, off, None), (n, off - 1, None)):
        int4.grouped_linear(x, w, counts, offsets, src_row=src)
        with pytest.raises(RuntimeError, match="out of range"):
            ops.workspace().check_status()
    int4.grouped_linear(x, w, n, off)
    ops.workspace().check_status()


@pytest.mark.parametrize("rows", [1, 12, 80])
def test_captured_products_follow_their_inputs(rows):
    w, full = weight((4,), 64, 256, 128, False, torch.bfloat16, True)
    x, cnt, off = acts(rows, 256), torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(5, dtype=torch.int32, device=DEV)
    cnt[0], off[1:] = rows, rows
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        int4.grouped_linear(x, w, cnt, off, swiglu=True)
        with torch.cuda.graph(graph, stream=side):
            y = int4.grouped_linear(x, w, cnt, off, swiglu=True)
    torch.cuda.current_stream().wait_stream(side)
    for e in (0, 3, 1):
        x.copy_(acts(rows, 256, seed=e + 7))
        cnt.zero_()
        cnt[e] = rows
        off.copy_(torch.cat((cnt.new_zeros(1), cnt.cumsum(0))))
        graph.replay()
        within(y, x, full[e], True)


def test_same_bits_twice_and_on_two_streams():
    w, full = weight((), 512, 2048, 128, True, torch.bfloat16, False)
    for rows in (2, 14, 60, 300):
        x = acts(rows, 2048)
        y = int4.linear(x, w, out_f32=True)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append([int4.linear(x, w, out_f32=True) for _ in range(3)])
        torch.cuda.synchronize()
        assert all(torch.equal(y, z) for g in got for z in g)


@pytest.mark.parametrize("cfg, rows, features, K, group", [((16, 1), 16, 128 * 301, 256, 64), ((32, 1), 40, 128 * 150, 128, 32), ((64, 1), 129, 128 * 101, 384, 128),
                                                           ((128, 1), 400, 128 * 41, 128, 64), ((128, 1), 300, 128 * 60, 256, 32), (None, 500, 9000, 192, 64), (None, 17, 40000, 128, 128)])
def test_more_tiles_than_places(cfg, rows, features, K, group):
    """Every CTA walks several tiles: what one leaves (accumulators, slots, stages) the next finds in order."""
    w, full = weight((), features, K, group, True, torch.float16, False)
    x = acts(rows, K)
    within(int4.linear(x, w, out_f32=True, _cfg=cfg), x, full, half_step=2.0 ** -24)
    w, full = weight((), 2 * (features // 3), K, group, False, torch.bfloat16, True)
    within(int4.swiglu_linear(x, w, _cfg=cfg), x, full, True)
    ops.workspace().check_status()


@pytest.mark.parametrize("cfg", [None, (16, 1), (128, 1), (0, 0)])
def test_many_uneven_experts(cfg):
    gen = torch.Generator(device=DEV).manual_seed(8)
    counts = torch.randint(0, 40, (90,), generator=gen, device=DEV, dtype=torch.int32)
    counts[::7] = 0
    off = torch.cat((counts.new_zeros(1), counts.cumsum(0))).to(torch.int32)
    n = int(off[-1])
    w, full = weight((90,), 300, 160, 32, True, torch.bfloat16, False)
    x, src = acts(64, 160), torch.randint(0, 64, (n,), generator=gen, device=DEV, dtype=torch.int32)
    y = int4.grouped_linear(x, w, counts, off, src_row=src, _cfg=cfg)
    expert = torch.repeat_interleave(torch.arange(90, device=DEV), counts.long())
    for e in range(90):
        mine = expert == e
        if bool(mine.any()):
            within(y[mine], x[src[mine].long()], full[e])
    ops.workspace().check_status()


@pytest.mark.parametrize("tiles, last", [(2 * 296 + 1, 5), (2 * 296 + 4, 128), (2 * 296 + 296, 77), (4 * 296 + 40, 1), (2 * 296 + 300, 128)])
def test_a_last_round_is_shared(tiles, last):
    """Tiles that do not fill a round of the GPU's places, with and without CTAs that share them, an odd one and one of few rows among them."""
    features, K = 128 * (tiles - 1) + last, 1088
    w, full = weight((), features, K, 64, True, torch.bfloat16, False)
    x = acts(14, K)
    y = int4.linear(x, w, out_f32=True, _cfg=(16, 0))
    within(y, x, full, half_step=2.0 ** -24)
    assert torch.equal(y, int4.linear(x, w, out_f32=True, _cfg=(16, 0)))
    r = torch.randn(14, features, device=DEV).bfloat16()
    within(int4.linear(x, w, residual=r, _cfg=(16, 0)), x, full, residual=r)
    del w, full
    w, full = weight((), 2 * (features // 2), K, 32, False, torch.float16, True)
    within(int4.swiglu_linear(x, w, _cfg=(16, 0)), x, full, True)
    ops.workspace().check_status()


@pytest.mark.parametrize("tile", [16, 32, 64, 128])
@pytest.mark.parametrize("E, features, K, group, zeros, pair", [(60, 650, 1024, 128, False, False), (100, 392, 416, 32, True, True), (1024, 130, 192, 64, True, False),
                                                                (7, 5400, 320, 64, False, True), (40, 1030, 2176, 128, True, False)])
def test_gathered_rows_of_many_tiles(E, features, K, group, zeros, pair, tile):
    """An odd number of weight tiles per expert, experts that are empty, of one row and of several row tiles, rows named twice, rows of x that lie apart; a row
    that is no number stays alone, though its place in shared memory is used again."""
    gen = torch.Generator(device=DEV).manual_seed(E)
    counts = torch.randint(0, 30, (E,), generator=gen, device=DEV, dtype=torch.int32)
    counts[::5], counts[1], counts[-1] = 0, 1, 150
    off = torch.cat((counts.new_zeros(1), counts.cumsum(0))).to(torch.int32)
    n = int(off[-1])
    w, full = weight((E,), features * (2 if pair else 1), K, group, zeros, torch.bfloat16, pair)
    x = acts(50, K + 24)[:, 8:8 + K]
    x[7] = float("nan")
    src = torch.randint(0, 50, (n,), generator=gen, device=DEV, dtype=torch.int32)
    src[torch.randint(0, n, (n // 3,), generator=gen, device=DEV)] = 5
    y = int4.grouped_linear(x, w, counts, off, swiglu=pair, src_row=src, _cfg=(tile, 1))
    expert = torch.repeat_interleave(torch.arange(E, device=DEV), counts.long())
    lost = src == 7
    assert bool(lost.any()) and bool(y[lost].isnan().all())
    for e in list(range(0, E, max(1, E // 40))) + [E - 1]:
        mine = (expert == e) & ~lost
        if bool(mine.any()):
            within(y[mine], x[src[mine].long()], full[e], pair)
    assert bool(y[~lost].isfinite().all())
    ops.workspace().check_status()


@pytest.mark.parametrize("cfg", [(0, 0), (16, 1), (64, 1)])
def test_experts_beyond_31_bits(cfg):
    """The last expert's codes lie more than 2^31 bytes into the weight."""
    one, full = weight((1,), 512, 8192, 128, False, torch.bfloat16, False)
    E = (1 << 31) // one.data[0].numel() + 2
    if E > int4.MAX_EXPERTS:
        E = int4.MAX_EXPERTS
    data = torch.zeros(E, *one.data.shape[1:], dtype=torch.uint8, device=DEV)
    data[-1].copy_(one.data[0])
    assert (E - 1) * one.data[0].numel() >= 1 << 31
    w = int4.Int4Weight(data, (E, 512, 8192), 128, False, torch.bfloat16, False)
    x = acts(20, 8192)
    counts = torch.zeros(E, dtype=torch.int32, device=DEV)
    counts[-1] = 20
    y = int4.grouped_linear(x, w, counts, torch.zeros_like(counts), _cfg=cfg)
    within(y, x, full[0])


def test_two_graphs_at_once():
    """Captured products and routers share nothing: replayed at once on two streams they give what they give one after another."""
    x = [acts(48, 512, seed=s) for s in (1, 2)]
    w, _ = weight((16,), 2 * 192, 512, 64, True, torch.bfloat16, True)
    d, _ = weight((), 4096, 2048, 128, False, torch.bfloat16, False)
    wide = [acts(30, 2048, seed=s) for s in (3, 4)]
    wg = torch.randn(16, 512, device=DEV).bfloat16()
    graphs, outs = [], []
    for i in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            def step():
                logits = x[i].float() @ wg.float().t()
                ids, rw, counts, offsets, row_of, src = experts.route_balanced(logits, 2)
                return int4.grouped_linear(x[i], w, counts, offsets, swiglu=True, src_row=src), int4.linear(wide[i], d, out_f32=True), ids, row_of
            step()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(step())
        graphs.append((g, side))
        torch.cuda.synchronize()
    for g, _ in graphs:
        g.replay()
        torch.cuda.synchronize()
    want = [[t.clone() for t in o] for o in outs]
    for o in outs:
        for t in o:
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for g, side in graphs:
            with torch.cuda.stream(side):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, outs):
        for s, t in zip(a, b):
            assert torch.equal(s, t)


# ---- choice of experts ------------------------------------------------------------------------------------------------
ROUTES = [  # tokens, experts, top, groups, keep, group_best, score, renorm
    (1, 1, 1, 1, 1, 2, "softmax", True), (1, 128, 8, 1, 1, 2, "softmax", True), (5, 33, 4, 1, 1, 1, "sigmoid", False), (64, 64, 6, 8, 4, 2, "sigmoid", True),
    (200, 120, 8, 8, 2, 1, "softmax", True), (256, 256, 8, 8, 4, 2, "sigmoid", True), (257, 40, 3, 5, 2, 2, "sigmoid", True), (300, 512, 16, 64, 8, 2, "softmax", False),
    (31, 512, 16, 1, 1, 2, "sigmoid", True), (4096, 256, 8, 8, 4, 2, "sigmoid", True), (9000, 8, 2, 1, 1, 2, "softmax", True), (1000, 6, 2, 6, 3, 2, "sigmoid", True)]


def plan_of(ids, E, e_first, e_count):
    flat = ids.reshape(-1).long()
    mine = (flat >= e_first) & (flat < e_first + e_count)
    counts = torch.bincount(flat[mine], minlength=E).to(torch.int32)
    offsets = torch.cat((counts.new_zeros(1), counts.cumsum(0))).to(torch.int32)
    order = torch.where(mine, flat, torch.full_like(flat, E)).sort(stable=True).indices[:int(mine.sum())]
    row_of = torch.full_like(flat, -1)
    row_of[order] = torch.arange(order.numel(), device=flat.device)
    return counts, offsets, row_of.to(torch.int32), (order // ids.shape[1]).to(torch.int32)


def check_route(z, top, bias, groups, keep, best, score, renorm, scale=1.0, e_first=0, e_count=None):
    E = z.shape[1]
    got = experts.route_balanced(z, top, bias=bias, groups=groups, keep=keep, score=score, group_best=best, renorm=renorm, scale=scale, e_first=e_first,
                                 e_count=e_count)
    ids, w = ri.select_balanced(z, top, bias, groups, keep, score, best, renorm, scale)
    assert torch.equal(got[0], ids)
    # one rounding of a 64-bit value on either side
    assert torch.allclose(got[1].double(), w.double(), rtol=2.0 ** -23, atol=1e-40)
    want = plan_of(ids, E, e_first, E - e_first if e_count is None else e_count)
    for a, b in zip(got[2:5], want[:3]):
        assert torch.equal(a, b)
    assert torch.equal(got[5][:want[3].numel()], want[3])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T, E, top, groups, keep, best, score, renorm", ROUTES)
def test_route_balanced(T, E, top, groups, keep, best, score, renorm, dtype):
    gen = torch.Generator(device=DEV).manual_seed(T + E)
    z = torch.randn(T, E, generator=gen, device=DEV).to(dtype)
    bias = torch.randn(E, generator=gen, device=DEV) * 0.1
    for b in (None, bias):
        check_route(z, top, b, groups, keep, best, score, renorm, 2.5)
    if E > 2:
        check_route(z, top, bias, groups, keep, best, score, renorm, 1.0, E // 3, E // 2)
    wide = torch.randn(T, E + 5, generator=gen, device=DEV).to(dtype)
    check_route(wide[:, 3:3 + E], top, bias, groups, keep, best, score, renorm)


@pytest.mark.parametrize("T", [16, 600])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_of_masked_and_equal_logits(T, score):
    z = torch.randn(T, 48, device=DEV)
    z[0] = 0
    z[1] = -float("inf")
    z[2, 5:] = -float("inf")
    z[3] = float("nan")
    z[4, ::2] = float("nan")
    z[5, 7] = float("inf")
    z[6] = torch.finfo(torch.float32).min
    z[7] = torch.finfo(torch.float32).max
    z[8] = z[8].bfloat16().float().round()
    z[9, 40] = -float("inf")
    off = torch.zeros(48, device=DEV)
    off[3], off[11] = -float("inf"), float("inf")
    for bias in (None, off):
        for groups, keep in ((1, 1), (6, 2), (48, 7)):
            check_route(z, 7, bias, groups, keep, 2, score, True)


def test_route_of_no_tokens():
    got = experts.route_balanced(torch.empty(0, 12, device=DEV), 3)
    assert got[0].shape == (0, 3) and bool((got[2] == 0).all()) and bool((got[3] == 0).all()) and got[4].numel() == 0


@pytest.mark.parametrize("T", [40, 700])
def test_captured_route_follows_its_logits(T):
    z = torch.randn(T, 64, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        experts.route_balanced(z, 6, groups=8, keep=4)
        with torch.cuda.graph(graph, stream=side):
            got = experts.route_balanced(z, 6, groups=8, keep=4)
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(3):
        z.copy_(torch.randn(T, 64, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV))
        graph.replay()
        ids, _ = ri.select_balanced(z, 6, None, 8, 4, "sigmoid", 2, True, 1.0)
        assert torch.equal(got[0], ids)
        for a, b in zip(got[2:], plan_of(ids, 64, 0, 64)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 50, 400])
def test_layer_of_experts(T):
    """Router, gate / up by the router's layout, down, combine with the residual: a layer as it is used."""
    H, I, E, top = 256, 128, 12, 3
    gen = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn(T, H, generator=gen, device=DEV).bfloat16()
    wg = torch.randn(E, H, generator=gen, device=DEV).bfloat16()
    bias = torch.randn(E, generator=gen, device=DEV) * 0.1
    up, up_full = weight((E,), 2 * I, H, 64, True, torch.bfloat16, True, seed=2)
    down, down_full = weight((E,), H, I, 32, False, torch.float16, False, seed=3)
    logits = ops.linear(x, wg, out_f32=True)
    ids, w, counts, offsets, row_of, src = experts.route_balanced(logits, top, bias=bias, groups=4, keep=2, scale=2.0)
    h = int4.grouped_linear(x, up, counts, offsets, swiglu=True, src_row=src)
    y = int4.grouped_linear(h, down, counts, offsets)
    out, _ = ops.reduce_residual_rmsnorm(x, y[None], None, 1e-5, row_idx=row_of.view(T, top), row_w=w)
    ops.workspace().check_status()
    ids_want, w_want = ri.select_balanced(logits, top, bias, 4, 2, "sigmoid", 2, True, 2.0)
    assert torch.equal(ids, ids_want)
    want, size = x.double(), torch.zeros(T, H, dtype=torch.float64, device=DEV)
    for j in range(top):
        for t in range(T):
            e = int(ids[t, j])
            g, u = (x[t].double() @ up_full[e].t()).chunk(2)
            a = g * torch.sigmoid(g) * u
            v = a @ down_full[e].t()
            want[t] += w_want[t, j].double() * v
            # h is rounded (2^-8 of each product of the sum), y and the result are
            size[t] += w_want[t, j].double() * ((a.abs() @ down_full[e].abs().t()) * 2.0 ** -8 * 1.01 + v.abs() * 2.0 ** -8 * 1.01)
    off = (out.double() - want).abs() - size - 2.0 ** -8 * (want.abs() + size) - 1e-4 * size
    assert bool((off <= 0).all()), float(off.max())
