"""Scores of the balanced router that lie a few units in the last place apart, against the choice in 64 bits by the definition."""
import pytest
import torch

from skein_b200.ops import experts, reference_int4 as ri

pytestmark = pytest.mark.gpu
DEV = "cuda"


def close_logits():
    """fp32 logits whose sigmoids are 1 to some 30 units in the last place apart, or equal (from 36.75 on 1 + exp(-z) rounds to 1)."""
    near = []
    for z in (21.5, 24.0, 27.25, 30.0):
        v = torch.tensor(z)
        for _ in range(6):
            near.append(float(v))
            v = torch.nextafter(v, torch.tensor(100.0))
    return near + [33 + i / 4 for i in range(24)]


def case(T, E, seed):
    gen = torch.Generator().manual_seed(seed)
    values = torch.tensor(close_logits())
    return values[torch.randint(0, len(values), (T, E), generator=gen)]


@pytest.mark.parametrize("T", [3, 70, 300])
@pytest.mark.parametrize("E, top, groups, keep, best", [(16, 4, 1, 1, 2), (64, 8, 8, 3, 2), (100, 16, 1, 1, 2), (120, 6, 60, 30, 1), (256, 8, 8, 4, 2), (250, 16, 1, 1, 2), (512, 16, 1, 1, 2),
                                                        (512, 12, 64, 20, 2)])
def test_close_scores_are_told_apart(T, E, top, groups, keep, best):
    z = case(T, E, T + E)
    z[0] = 35.0                         # one larger score, at a higher index of another lane, of the same lane, behind the others
    z[0, E // 2] = 36.0
    z[1] = 34.0
    z[1, E - 1] = 35.0
    z[2] = 21.5
    z[2, min(E - 1, 40)] = 21.500001907348633
    bias = torch.zeros(E)
    bias[::3] = 2.0 ** -52              # (scores lie in [0.5, 1]: one or two units in the last place)
    for b in (None, bias):
        got = experts.route_balanced(z.to(DEV), top, bias=None if b is None else b.to(DEV), groups=groups, keep=keep, score="sigmoid", group_best=best, renorm=False)
        ids, w = ri.select_balanced(z, top, b, groups, keep, "sigmoid", best, False, 1.0)
        assert torch.equal(got[0].cpu(), ids)
        assert torch.allclose(got[1].cpu(), w, rtol=2.0 ** -23, atol=0)
        same = experts.route_balanced(z, top, bias=b, groups=groups, keep=keep, score="sigmoid", group_best=best, renorm=False)      # on the CPU
        assert torch.equal(got[0].cpu(), same[0])
        for a, c in zip(got[2:], same[2:]):
            assert torch.equal(a.cpu(), c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E, top", [(40, 7), (128, 16), (256, 8), (512, 16)])
def test_equal_scores_go_to_the_lower_index(E, top, dtype):
    """Few different logits: most of a token's choices are ties, inside lanes and between them."""
    gen = torch.Generator().manual_seed(E)
    z = torch.randint(0, 3, (300, E), generator=gen).float()
    z[5] = 0
    z[6, :E // 2] = -1
    for score in experts.SCORES:
        got = experts.route_balanced(z.to(DEV, dtype), top, score=score)
        want = [sorted(range(E), key=lambda e: (-row[e], e))[:top] for row in z.tolist()]
        assert got[0].cpu().tolist() == want


@pytest.mark.parametrize("T", [2, 300])
def test_subnormal_numbers_count(T):
    """Weights, biases and logits below the smallest normal number of 32 bits."""
    z = torch.zeros(T, 24)
    z[:, 1:] = -86.0 - torch.arange(23) * 0.75
    ids, w, *_ = experts.route_balanced(z.to(DEV), 16, score="softmax", renorm=False)
    want = ri.select_balanced(z, 16, None, 1, 1, "softmax", 2, False, 1.0)
    assert torch.equal(ids.cpu(), want[0]) and bool((want[1][:, 4:] < 2.0 ** -126).all()) and bool((want[1] > 0).all())
    # (a rounding of 64 bits on either side: a step of the value, or of the subnormal numbers)
    assert torch.allclose(w.cpu().double(), want[1].double(), rtol=2.0 ** -23, atol=2.0 ** -149)
    z = torch.full((T, 24), -800.0)              # scores of 0: the bias alone decides
    bias = (torch.arange(24) % 7) * 2.0 ** -140
    ids = experts.route_balanced(z.to(DEV), 9, bias=bias.to(DEV))[0]
    assert torch.equal(ids.cpu(), ri.select_balanced(z, 9, bias, 1, 1, "sigmoid", 2, True, 1.0)[0])
    z = (torch.arange(24) % 5).float().repeat(T, 1) * 2.0 ** -140       # (sigmoids of 1/2, softmaxes of 1/24, whatever the logits)
    for score in experts.SCORES:
        assert experts.route_balanced(z.to(DEV), 9, score=score)[0].cpu().tolist() == [list(range(9))] * T


def test_as_many_tokens_as_a_call_takes():
    T = 148 * 1536
    z = torch.randn(T + 1, 3, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    ids, _, counts, offsets, row_of, src = experts.route_balanced(z[:T], 1)
    assert torch.equal(ids[:, 0].long(), z[:T].double().sigmoid().argmax(1)) and int(offsets[-1]) == T
    assert torch.equal(counts.long(), torch.bincount(ids[:, 0], minlength=3)) and torch.equal(src[row_of.long()], torch.arange(T, device=DEV, dtype=torch.int32))
    with pytest.raises(ValueError, match="more than one call takes"):
        experts.route_balanced(z, 1)
