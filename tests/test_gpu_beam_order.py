"""Order of beams whose keys are equal, or equal up to roundings: rows that start at
different offsets from a 16-byte boundary, logits of any size, cums of any size."""
import numpy as np
import pytest
import torch

import mflat_b200 as M
import select_ref as R
from test_gpu_beam import check, gen, select

pytestmark = pytest.mark.gpu


def equal_beams(b, w, row, cum):
    """b sequences of w beams alike, from b rows of logits."""
    x = row[:, None, :].expand(b, w, row.shape[1]).contiguous().cuda()
    return x, torch.full((b, w), cum).cuda()


def expect_equal_beams(x, cum, k):
    """By logit, then beam, then token: what the rule leaves of equal rows and cums."""
    out, _ = select(x, cum, k)
    torch.cuda.synchronize()
    w = x.shape[1]
    for i, row in enumerate(R.f64(x[:, 0])):
        token = np.tile(R.best(row, k), w)          # the lowest beams' k best hold all
        beam = np.repeat(np.arange(w), k)
        order = np.lexsort((token, beam, -row[token]))[:k]
        np.testing.assert_array_equal(out[0][i].cpu().numpy(), beam[order])
        np.testing.assert_array_equal(out[1][i].cpu().numpy(), token[order])


# (an odd vocabulary: neighbouring rows start 4 bytes further from a boundary each)
@pytest.mark.parametrize("size", [(64, 8, 50_257), (64, 4, 50_257), (16, 5, 50_001), (2, 4, 128_001), (40, 3, 9001)],
                         ids=lambda s: "b%d_w%d_v%d" % s)
@pytest.mark.parametrize("cum", [0.0, -7.3, -3e12])
def test_equal_beams_at_different_offsets(size, cum):
    b, w, v = size
    g = gen(("offsets", size, cum))
    # 16-bit values a step of 2^-6 apart: no two of them meet in 64 bits even at -3e12
    row = (torch.randn(b, v, generator=g) * 64).round() / 64
    for at in range(8192, v, 8192):     # larger ones where a row's offset moves the cuts
        row[:, at - 2] = 4 + torch.rand(b, generator=g).mul(64).round() / 64
    x, c = equal_beams(b, w, row, cum)
    expect_equal_beams(x, c, 2 * w)


@pytest.mark.parametrize("shift,spread", [(6e5, 4), (-6e5, 4), (3e7, 16)])
def test_equal_beams_of_large_logits(shift, spread):
    """Beyond the sizes that fp32 sums take.  Few terms weigh much, so that the last digits
    of their sum reach the key."""
    b, w, v = 64, 8, 50_257
    row = spread * torch.randn(b, v, generator=gen(("large", shift))) + shift
    x, c = equal_beams(b, w, row, 0.0)
    expect_equal_beams(x, c, 16)


def test_equal_beams_with_infinite_logits():
    b, w, v = 4, 4, 9001
    row = torch.randn(b, v, generator=gen("infinite"))
    row[:, 77] = row[:, 4000] = row[:, 8999] = float("inf")
    x, c = equal_beams(b, w, row, -2.0)
    out, _ = select(x, c, 12)
    # three a beam, with a third of the probability each
    place = torch.arange(12)
    assert torch.equal(out[0].cpu().long(), (place // 3).expand(b, 12))
    assert torch.equal(out[1].cpu().long(), torch.tensor([77, 4000, 8999])[place % 3].expand(b, 12))


@pytest.mark.parametrize("low", [-1e9, -1e30, -3.402823466e38])
def test_first_step_with_the_other_beams_far_below(low):
    """All beams alike and all but one out of the way: the usual first step."""
    x = torch.randn(3, 1, 30_011, generator=gen(("first", low))).expand(3, 8, 30_011).contiguous().cuda()
    cum = torch.full((3, 8), low)
    cum[:, 2] = 0.0
    out = check(x, cum.cuda(), 16)
    assert (out[0].cpu() == 2).all()


LOW = -3.402823466e38


@pytest.mark.parametrize("cum,scale", [(-1e12, 1e-3), (-1e15, 1.0), (-1e30, 1.0), (LOW, 3.0), (1e20, 1.0), (-5.0, 1e-18)])
@pytest.mark.parametrize("v,kind", [(40, "fp32"), (30_011, "fp32"), (30_011, "bf16"), (9001, "fp16")])
def test_keys_of_different_logits_that_are_equal_in_64_bits(cum, scale, v, kind):
    """Ties go to the lowest beam, then token, whatever the logits are."""
    if kind == "fp16":
        scale = max(scale, 1e-3)
    b, w = 4, 4
    x = scale * torch.randn(b, w, v, generator=gen(("own", cum, scale, v)))
    x[1, 1:] = x[1, :1]                         # a sequence of equal beams
    x[2, 0, 7:] = -float("inf")                 # a beam that has fewer than are asked for
    x[3, 1, ::2], x[3, 2] = float("nan"), 0.0
    x = x.to(R.TYPES[kind])
    c = torch.full((b, w), cum)
    done = torch.zeros(b, w, dtype=torch.uint8)
    done[0, 1] = done[2, 0] = done[3, 3] = 1
    for beams, k in [(1, 1), (1, 3), (1, 20), (w, 3), (w, 20), (w, 128)]:
        xs, cs, ds = (t[:, :beams].contiguous().cuda() for t in (x, c, done))
        check(xs, cs, k)
        check(xs, cs, k, ds, eos=v // 2)


def test_beams_at_the_lowest_cum_fill_up():
    """Few tokens allowed in the one beam that is alive: the others' fill the places."""
    x = torch.full((2, 4, 20_003), -float("inf"))
    x[:, 0, [5, 900]] = torch.tensor([1.0, 2.0])
    x[:, 1:, 100:] = torch.randn(2, 3, 19_903, generator=gen("fill"))
    cum = torch.full((2, 4), LOW)
    cum[:, 0] = -1.0
    out = check(x.cuda(), cum.cuda(), 8)
    assert out[1][0].tolist() == [900, 5, 100, 101, 102, 103, 104, 105]


def test_more_equal_keys_than_a_list_holds():
    x = torch.randn(1, 1, 40_009, generator=gen("many equal")).expand(1, 64, 40_009).contiguous()
    check(x.cuda(), torch.full((1, 64), -1e30).cuda(), 128)


def test_zeros():
    for v in (50, 20_011):
        check(torch.zeros(2, 3, v).cuda(), torch.zeros(2, 3).cuda(), 9)
        check(torch.zeros(2, 3, v).bfloat16().cuda(), torch.tensor([[0.0, 1.0, 1.0]] * 2).cuda(), 9)


@pytest.mark.parametrize("v", [1, 2, 3, 30])
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_equal_beams_with_fewer_candidates_than_choices(v, kind):
    for w, k in [(3, 3 * v + 1), (8, 128), (21, min(128, 21 * v))]:
        g = gen(("few", v, kind, w))
        x = (3 * torch.randn(6, 1, v, generator=g)).to(R.TYPES[kind]).expand(6, w, v).contiguous()
        for shift in (0.0, -1e6, 53.3):
            c = torch.randn(6, 1, generator=g).expand(6, w) + shift
            check(x.cuda(), c.contiguous().cuda(), k)
            done = (torch.rand(6, w, generator=g) < 0.3).to(torch.uint8)
            check(x.cuda(), c.contiguous().cuda(), k, done.cuda(), eos=v - 1)


def test_reorder_of_the_most_outer_rows():
    """2^31 - 1 outer rows of two beams of a byte each."""
    outer = 2 ** 31 - 1
    x = torch.zeros(outer, 2, dtype=torch.uint8, device="cuda")
    x[:, 1] = 7
    x[::1001, 0] = 3
    parents = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    M.beam_reorder_device(x.data_ptr(), parents.data_ptr(), outer, 1, 2, 1)
    torch.cuda.synchronize()
    assert bool((x[:, 0] == 7).all())
    assert bool((x[::1001, 1] == 3).all()) and int(torch.count_nonzero(x[:, 1])) == -(-outer // 1001)
