"""Calls of the 4-bit products and of the balanced router that share memory, are copied or name rows that are not there, on the CPU."""
import copy
import io
import random

import pytest
import torch

from skein_b200.ops import experts, int4


def small(lead=(), rows=16, K=64, pair=False, seed=0):
    gen = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (*lead, rows, K // 2), generator=gen, dtype=torch.uint8)
    return int4.pack_weight(codes, torch.rand(*lead, rows, K // 64, generator=gen).bfloat16(), pair=pair)


def test_meeting_matrices_are_found():
    """Against the bytes themselves, over every kind of pair: columns and rows of one buffer, single and repeated rows, rows of other distances, two types."""
    rng, found = random.Random(3), [0, 0]
    buf = torch.zeros(400, dtype=torch.bfloat16)

    def matrix():
        rows, wide = rng.choice((1, 2, 3, 7)), rng.randint(1, 12)
        step = rng.choice((0, 12, 12, 24, 24, 31)) if rng.random() < 0.8 else rng.randint(wide, 40)
        t, first = (buf, rng.randint(0, 60)) if rng.random() < 0.7 else (buf.view(torch.float32), rng.randint(0, 30))
        step = step if t is buf else step // 2
        return t.as_strided((rows, wide), (step, 1), first + (rng.randint(0, 60) if t is buf else 0))

    def bytes_of(t):
        size = t.element_size()
        return {t.data_ptr() + (r * t.stride(0) + c) * size + i for r in range(t.shape[0]) for c in range(t.shape[1]) for i in range(size)}
    for _ in range(4000):
        a, b = matrix(), matrix()
        want = bool(bytes_of(a) & bytes_of(b))
        assert int4._meet(a, b) == int4._meet(b, a) == want, (a.shape, a.stride(), a.storage_offset(), a.dtype, b.shape, b.stride(), b.storage_offset(), b.dtype)
        found[want] += 1
    assert min(found) > 500
    assert not int4._meet(buf[:0].view(0, 4), buf[:8].view(2, 4)) and not int4._meet(buf[:8].view(2, 4), buf[:0].view(2, 0))


def test_out_on_rows_of_x_is_refused():
    one, many, pair = small(rows=16), small((2,), rows=16), small(rows=32, pair=True)
    n, first = torch.tensor([2, 2], dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32)
    buf = torch.zeros(6, 200, dtype=torch.bfloat16)
    flat = torch.zeros(8, 64, dtype=torch.bfloat16)
    for x, out in ((buf[:4, :64], buf[:4, 8:24]), (buf[:4, :64], buf[1:5, :16]), (buf[:4, 60:124], buf[2:, 50:66]), (buf[1:5, 40:104], buf[:4, 30:46]),
                   (flat[:4], flat.view(-1)[192 + 63:].as_strided((4, 16), (16, 1))), (flat[::2], flat.view(16, 32)[1::4, 16:])):
        for call in (lambda: int4.linear(x, one, out=out), lambda: int4.swiglu_linear(x, pair, out=out), lambda: int4.grouped_linear(x, many, n, first, out=out)):
            with pytest.raises(ValueError, match="lies on x"):
                call()
    # as a result of other rows, with the rows named
    with pytest.raises(ValueError, match="lies on x"):
        int4.grouped_linear(flat[:1], many, n, first, src_row=torch.zeros(4, dtype=torch.int32), out=flat.view(-1)[32:].as_strided((4, 16), (16, 1)))


def test_out_beside_x_is_taken():
    one = small(rows=16)
    buf = torch.randn(9, 200, generator=torch.Generator().manual_seed(1)).bfloat16()
    want = int4.linear(buf[:4, :64].clone(), one)
    for x, out in ((buf[:4, :64], buf[:4, 64:80]), (buf[:4, :64], buf[4:8, :16]), (buf[:4, :64], buf.view(-1)[800:].as_strided((4, 16), (16, 1))), (buf[:4, :64], buf[:4, 184:])):
        assert torch.equal(int4.linear(x, one, out=out), want) and torch.equal(out, want)
    rows = torch.zeros(8, 64, dtype=torch.bfloat16)
    rows[::2] = buf[:4, :64]
    assert torch.equal(int4.linear(rows[::2], one, out=rows[1::2, 5:21]), want)


def test_a_residual_is_out_or_beside_it():
    one = small(rows=16)
    x = torch.randn(4, 64, generator=torch.Generator().manual_seed(2)).bfloat16()
    buf = torch.randn(9, 40, generator=torch.Generator().manual_seed(3)).bfloat16()
    for r, out in ((buf[1:5, :16], buf[:4, :16]), (buf[:4, 5:21], buf[:4, :16]), (buf[:4, 30:].as_strided((4, 16), (40, 1)), buf[1:5, :16])):
        with pytest.raises(ValueError, match="residual"):
            int4.linear(x, one, out=out, residual=r)
    with pytest.raises(ValueError, match="residual"):      # one row
        int4.linear(x[:1], one, out=buf[:1, :16], residual=buf[:1, 15:31])
    keep = buf.clone()
    want = int4.linear(x, one, residual=keep[:4, 16:32].contiguous())
    assert torch.equal(int4.linear(x, one, out=buf[:4, :16], residual=buf[:4, 16:32]), want)
    assert torch.equal(int4.linear(x, one, out=buf[:4, 16:32], residual=buf[:4, 16:32]), want)
    wide = torch.randn(4, 16)
    assert torch.equal(int4.linear(x[:1], one, out=wide[:1], residual=wide[:1].as_strided((1, 16), (3, 1)), out_f32=True), wide[:1])


def test_a_copied_or_pickled_weight_has_its_own_address():
    w = small((2,), 16, 128)
    file = io.BytesIO()
    torch.save(w, file)
    file.seek(0)
    for other in (copy.deepcopy(w), torch.load(file, weights_only=False)):
        assert other.data.data_ptr() != w.data.data_ptr() and other.ptr == other.data.data_ptr()
        assert torch.equal(other.dequant(), w.dequant()) and other.device == w.device and other.matrices == 2
    moved = copy.copy(w)
    moved.data = w.data.to("meta")
    assert moved.device.type == "meta" and not moved.is_cuda and w.device.type == "cpu"


def test_a_weight_made_from_other_storage_is_checked():
    w = small((3,), 32, 128, pair=True)
    make = lambda data, shape=w.shape, group=64, pair=True, scales=torch.bfloat16, zeros=False: int4.Int4Weight(data, shape, group, pair, scales, zeros)      # noqa: E731
    buf = torch.zeros(w.nbytes() + 64, dtype=torch.uint8)
    first = -buf.data_ptr() % 16
    at = buf[first + 16:first + 16 + w.nbytes()].view(w.data.shape)
    at.copy_(w.data)
    assert torch.equal(make(at).dequant(), w.dequant())
    bad = [dict(data=buf[first + 8:first + 8 + w.nbytes()].view(w.data.shape)), dict(data=w.data[:2]), dict(data=w.data.to(torch.int8)), dict(data=w.data, shape=(3, 32, 256)),
           dict(data=w.data, shape=(3, 200, 128)), dict(data=w.data, group=32), dict(data=w.data, group=48), dict(data=w.data, zeros=True), dict(data=w.data, shape=(3, 31, 128)),
           dict(data=w.data.expand(3, 1, 1, -1)[:1].expand(3, 1, 1, w.data.shape[-1])), dict(data=w.data, scales=torch.float32), dict(data=w.data, shape=(32, 128))]
    for kw in bad:
        with pytest.raises(ValueError):
            make(**kw)


@pytest.mark.parametrize("first", [0, 1, 2, 4, 7])
def test_codes_may_begin_at_any_byte(first):
    gen = torch.Generator().manual_seed(9)
    codes, scale = torch.randint(0, 256, (2, 6, 48), generator=gen, dtype=torch.uint8), torch.rand(2, 6, 3, generator=gen).bfloat16()
    buf = torch.empty(first + codes.numel(), dtype=torch.uint8)
    part = buf[first:].view(codes.shape)
    part.copy_(codes)
    assert torch.equal(int4.pack_weight(part, scale).data, int4.pack_weight(codes, scale).data)
    assert torch.equal(int4.pack_weight(part[1], scale[1]).dequant(), int4.pack_weight(codes, scale).dequant()[1])


def test_rows_outside_are_refused():
    """What a GPU call reports in the workspace's status."""
    w = small((2,), 16, 64)
    x, out = torch.ones(4, 64, dtype=torch.bfloat16), torch.full((4, 16), 3.0, dtype=torch.bfloat16)
    n, first = torch.tensor([2, 2], dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32)
    src = torch.tensor([0, 3, 1, 2], dtype=torch.int32)
    for counts, offsets, rows in ((n, first, src - 1), (n, first, src + 1), (n + 1, first, None), (n, first - 1, None), (n, first + 1, src), (n - 3, first, None)):
        with pytest.raises(ValueError, match="out of range"):
            int4.grouped_linear(x, w, counts, offsets, src_row=rows, out=out)
    assert bool((out == 3).all())
    unset = torch.tensor([1, 2, -7, 90], dtype=torch.int32)              # rows that no expert covers
    int4.grouped_linear(x, w, torch.tensor([2, 0], dtype=torch.int32), torch.tensor([0, -5], dtype=torch.int32), src_row=unset, out=out)
    assert bool((out[2:] == 3).all()) and not bool((out[:2] == 3).any())


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_weights_that_are_not_finite_are_not_quantised(value, symmetric):
    w = torch.randn(2, 3, 128, generator=torch.Generator().manual_seed(4))
    int4.quantize_weight(w, 64, symmetric)
    w[1, 2, 70] = value
    with pytest.raises(ValueError, match="finite"):
        int4.quantize_weight(w, 64, symmetric)


@pytest.mark.parametrize("T, first, count", [(0, 0, 4), (5, 0, 4), (5, 1, 2), (5, 4, 0)])
def test_a_layer_of_some_or_no_tokens_and_experts(T, first, count):
    """The layout has an entry for every pair, whatever experts are this rank's: a layer's shapes are the GPU's."""
    x = torch.randn(T, 64, generator=torch.Generator().manual_seed(6)).bfloat16()
    ids, p, counts, offsets, row_of, src = experts.route_balanced(torch.randn(T, 4, generator=torch.Generator().manual_seed(7)), 2, e_first=first, e_count=count)
    assert ids.shape == p.shape == (T, 2) and counts.shape == (4,) and offsets.shape == (5,) and row_of.shape == src.shape == (2 * T,)
    y = int4.grouped_linear(x, small((4,), 16, 64), counts, offsets, src_row=src)
    assert y.shape == (2 * T, 16)
    mine = (ids.reshape(-1) >= first) & (ids.reshape(-1) < first + count)
    assert int(offsets[-1]) == int(mine.sum()) and torch.equal(row_of >= 0, mine)
    assert torch.equal(src[row_of[mine].long()], (torch.arange(2 * T, dtype=torch.int32) // 2)[mine])
