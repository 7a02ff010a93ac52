"""Calls of the 4-bit products with unusual operands on the GPU, against 64 bits."""
import pytest
import torch

from skein_b200 import ops
from skein_b200.ops import int4, reference_int4 as ri

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
