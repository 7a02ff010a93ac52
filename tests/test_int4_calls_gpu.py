"""Calls of the 4-bit products with unusual operands on the GPU, against 64 bits."""
import pytest
import torch

from skein_b200 import ops
from skein_b200.ops import experts, int4, reference_int4 as ri

pytestmark = pytest.mark.gpu
DEV = "cuda"


def weight(lead, rows, K, group, zeros=True, scales=torch.bfloat16, pair=False, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 256, (*lead, rows, K // 2), generator=gen, device=DEV, dtype=torch.uint8)
    scale = (torch.rand(*lead, rows, K // group, generator=gen, device=DEV) * 0.02 + 0.005).to(scales)
    zero = torch.randint(0, 16, (*lead, rows, K // group), generator=gen, device=DEV, dtype=torch.uint8) if zeros else None
    return int4.pack_weight(codes, scale, zero, pair=pair), ri.dequant(codes, scale, zero, group).double()


def acts(rows, K, seed=1):
    return torch.randn(rows, K, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).bfloat16()


def unit(y, x, w, group, half_step=2.0 ** -24):
    """|y - exact| over what the order of the sums allows. A group's sum is a chain of at most `group` additions, each off by at most a step (2^-23, the
    tensor cores cut off) of the sum of its magnitudes. The groups' sums meet their scales in one rounding each (2^-24 of the running sum, which is at most
    the sum of all magnitudes), and the parts of K (at most 16) in one each. Then comes the rounding of the result."""
    exact, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    d = (group * 2.0 ** -23 + (x.shape[1] // group + 16) * 2.0 ** -24) * size
    return (y.double() - exact).abs() / (d + half_step * (exact.abs() + d))


@pytest.mark.parametrize("rows", [9, 40, 300])
def test_rows_off_16_bytes_give_the_bits_of_aligned_ones(rows):
    """They are laid out anew and take the kernel that aligned rows take, experts' and named rows too."""
    wide = acts(rows, 600)
    for first in (1, 4):
        x = wide[:, first:first + 256]
        w, full = weight((), 96, 256, 64)
        y = int4.linear(x, w, out_f32=True)
        assert torch.equal(y, int4.linear(x.contiguous(), w, out_f32=True)) and float(unit(y, x, full, 64).max()) <= 1
        w, _ = weight((), 96, 256, 64, pair=True)
        assert torch.equal(int4.swiglu_linear(x, w), int4.swiglu_linear(x.contiguous(), w))
        w, _ = weight((3,), 96, 256, 32, pair=True)
        cnt = torch.tensor([rows // 2, 0, rows - rows // 2], dtype=torch.int32, device=DEV)
        off = torch.tensor([0, rows // 2, rows // 2, rows], dtype=torch.int32, device=DEV)
        src = torch.randint(0, rows, (rows,), device=DEV, dtype=torch.int32)
        for named in (None, src):
            assert torch.equal(int4.grouped_linear(x, w, cnt, off, swiglu=True, src_row=named), int4.grouped_linear(x.contiguous(), w, cnt, off, swiglu=True, src_row=named))
    ops.workspace().check_status()


def test_captured_rows_off_16_bytes_follow_their_input():
    """The copy belongs to the graph."""
    w, full = weight((), 128, 384, 128)
    wide = acts(50, 400)
    x = wide[:, 3:387]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        int4.linear(x, w, out_f32=True)
        with torch.cuda.graph(graph, stream=side):
            y = int4.linear(x, w, out_f32=True)
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(3):
        wide.copy_(acts(50, 400, seed=20 + seed))
        graph.replay()
        assert float(unit(y, x, full, 128).max()) <= 1


ORDERS = [  # rows, features, K, group: long sums, where an allowance for a chain over all of K would let whole groups go missing
    (1, 40, 98304, 128), (2, 33, 65536, 64), (3, 64, 14336, 128), (5, 70, 28672, 32), (8, 130, 8192, 128), (13, 300, 14336, 64), (40, 129, 16384, 128), (100, 64, 32768, 128),
    (130, 200, 14336, 32)]


@pytest.mark.parametrize("rows, features, K, group", ORDERS)
def test_long_sums(rows, features, K, group):
    w, full = weight((), features, K, group)
    x = acts(rows, K)
    y = int4.linear(x, w, out_f32=True)
    assert float(unit(y, x, full, group).max()) <= 1
    # what the bound is worth: without the last group most results are out of it
    short = x.clone()
    short[:, K - group:] = 0
    assert float((unit(int4.linear(short, w, out_f32=True), x, full, group) > 1).float().mean()) > 0.5
    w, full = weight((2,), features, K, group, zeros=False, scales=torch.float16)
    cnt, off = torch.tensor([rows - rows // 3, rows // 3], dtype=torch.int32, device=DEV), torch.tensor([0, rows - rows // 3, rows], dtype=torch.int32, device=DEV)
    y = int4.grouped_linear(x, w, cnt, off)
    for e, part in ((0, slice(0, rows - rows // 3)), (1, slice(rows - rows // 3, rows))):
        if part.start < part.stop:
            assert float(unit(y[part], x[part], full[e], group, 2.0 ** -8).max()) <= 1
    ops.workspace().check_status()


@pytest.mark.parametrize("team", [1, 4, 8, 16])
@pytest.mark.parametrize("rows, features, K, group", [(1, 16, 2048, 64), (7, 200, 2176, 128), (8, 1000, 2048, 32), (11, 150, 384, 128), (11, 96, 2176, 64), (19, 40, 640, 32), (30, 300, 1408, 128),
                                                      (13, 70, 8192, 128), (29, 33, 16384, 64)])
def test_teams_of_few_rows(rows, features, K, group, team):
    """Every size of a team, with tiles of fewer than eight rows where a team's shared memory holds no more (K of 1408 with one warp, 8192 with four,
    16384 with eight and sixteen), a last tile that is not full, and experts of unequal rows."""
    steps = -(-K // 128)
    row = steps * 256 + 64
    if team > steps or 16 // team * row > 184 * 1024:
        pytest.skip("a team of more warps than steps, or without room for a row")
    w, full = weight((), features, K, group)
    x = acts(rows, K)
    y = int4.linear(x, w, out_f32=True, _cfg=(0, team))
    assert float(unit(y, x, full, group).max()) <= 1
    w, full = weight((4,), features, K, group, scales=torch.float16)
    counts = [rows // 2, 0, 1, rows]
    cnt = torch.tensor(counts, dtype=torch.int32, device=DEV)
    off = torch.cat((cnt.new_zeros(1), cnt.cumsum(0))).to(torch.int32)
    src = torch.randint(0, rows, (sum(counts),), generator=torch.Generator(device=DEV).manual_seed(4), device=DEV, dtype=torch.int32)
    y = int4.grouped_linear(x, w, cnt, off, src_row=src, _cfg=(0, team))
    for e in range(4):
        part = slice(int(off[e]), int(off[e + 1]))
        if counts[e]:
            assert float(unit(y[part], x[src[part].long()], full[e], group, 2.0 ** -8).max()) <= 1
    ops.workspace().check_status()


@pytest.mark.parametrize("cfg", [(16, 8), (32, 2), (64, 4), (128, 2)])
def test_rows_of_several_experts_are_reported(cfg):
    """Tiles that share their K have one place each: experts that claim the same rows make more tiles than places, which is told at once, not waited for."""
    w, full = weight((4,), 200, 2048, 128)
    x = acts(260, 2048)
    cnt, off = torch.full((4,), 260, dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    src = torch.arange(260, dtype=torch.int32, device=DEV)
    for named in (None, src):
        int4.grouped_linear(x, w, cnt, off, src_row=named, _cfg=cfg)
        with pytest.raises(RuntimeError, match="out of range"):
            ops.workspace().check_status()
    cnt = torch.tensor([200, 0, 60, 0], dtype=torch.int32, device=DEV)
    off = torch.tensor([0, 7, 200, 0], dtype=torch.int32, device=DEV)
    y = int4.grouped_linear(x, w, cnt, off, _cfg=cfg)
    assert float(unit(y[:200], x[:200], full[0], 128, 2.0 ** -8).max()) <= 1 and float(unit(y[200:], x[200:], full[2], 128, 2.0 ** -8).max()) <= 1
    ops.workspace().check_status()


@pytest.mark.parametrize("cfg", [None, (0, 0), (16, 1), (16, 4), (128, 1)])
def test_subnormal_fp16_scales(cfg):
    """Scales below 2^-14, where fp16 has fewer bits, are taken as they are."""
    gen = torch.Generator(device=DEV).manual_seed(3)
    codes = torch.randint(0, 256, (64, 128), generator=gen, device=DEV, dtype=torch.uint8)
    scale = (torch.randint(1, 1024, (64, 4), generator=gen, device=DEV).float() * 2.0 ** -24).half()
    w, full = int4.pack_weight(codes, scale), ri.dequant(codes, scale, None, 64).double()
    assert bool((scale > 0).all()) and float(scale.max()) < 2.0 ** -14
    x = acts(11, 256)
    assert float(unit(int4.linear(x, w, out_f32=True, _cfg=cfg), x, full, 64).max()) <= 1


@pytest.mark.parametrize("T, first, count", [(0, 0, 4), (5, 0, 4), (5, 1, 2), (5, 4, 0), (400, 3, 1)])
def test_a_layer_of_some_or_no_tokens_and_experts(T, first, count):
    w, full = weight((4,), 32, 256, 128)
    x = acts(T, 256)
    z = torch.randn(T, 4, generator=torch.Generator().manual_seed(7))
    ids, p, counts, offsets, row_of, src = experts.route_balanced(z.to(DEV), 2, e_first=first, e_count=count)
    assert ids.shape == p.shape == (T, 2) and counts.shape == (4,) and offsets.shape == (5,) and row_of.shape == src.shape == (2 * T,)
    out = torch.full((2 * T, 32), 5.0, device=DEV, dtype=torch.bfloat16)
    int4.grouped_linear(x, w, counts, offsets, src_row=src, out=out)
    n = int(offsets[-1])
    assert n == int(((ids >= first) & (ids < first + count)).sum()) and bool((out[n:] == 5).all())
    for e in range(first, first + count):
        part = slice(int(offsets[e]), int(offsets[e + 1]))
        if part.start < part.stop:
            assert float(unit(out[part], x[src[part].long()], full[e], 128, 2.0 ** -8).max()) <= 1
    ops.workspace().check_status()
