"""Beam selection and reordering on the GPU against the 64-bit definition
(select_ref.beam): parents and tokens equal, scores to fp32's last digits."""
import itertools
import zlib

import numpy as np
import pytest
import torch

import mflat_b200 as M
import select_ref as R

pytestmark = pytest.mark.gpu

# A score is cum + x - log of the row's sum, rounded once.
S_REL = 2.0 ** -24 * 1.001


def log_sum_bound(x):
    """Error of the logarithm of a row's sum, that is, the relative error of the sum of
    fp32 terms 2^t, t = x log2(e) - ref: the exponential's 2^-22; t's rounding, half a
    step 2^-24 |t| in t and so 2^-24 |x - m| in the term, where |x - m| weighted by the
    terms averages at most ln(vocab), or for t in (0, 9] 2^-24 times 9 ln 2; log2(e) in fp32, 2^-26 |x|, |x| <= |m| + |x - m|;
    and at most 13 additions in a row in fp32, 2^-24 each."""
    m = x.double().nan_to_num(nan=0.0, posinf=0.0, neginf=0.0).abs().max().item() if x.numel() else 0.0
    ln_v = np.log(x.shape[-1]) + 1
    return 2.0 ** -22 + (13 + 6.3) * 2.0 ** -24 + (2.0 ** -24 + 2.0 ** -26) * ln_v + 2.0 ** -26 * m


def gen(seed):
    return torch.Generator().manual_seed(zlib.crc32(repr(seed).encode()))


def select(x, cum, k, finished=None, eos=-1, ws=None, stream=0, out=None):
    kind = {v: n for n, v in R.TYPES.items()}[x.dtype]
    b, w, v = x.shape
    op = M.BeamSearch(w, v, k, dtype=kind, eos=eos)
    if out is None:
        out = (torch.full((b, k), -7, dtype=torch.int32, device="cuda"),
               torch.full((b, k), -7, dtype=torch.int32, device="cuda"), torch.full((b, k), 7.0, device="cuda"))
    if ws is None:
        ws = torch.randint(0, 255, (op.workspace_bytes(b),), dtype=torch.uint8, device="cuda")
    assert x.stride(0) == w * x.stride(1)
    op.select_device(x.data_ptr(), cum.data_ptr(), b, *(t.data_ptr() for t in out), stride=x.stride(1),
                     finished=finished.data_ptr() if finished is not None else 0, ws=ws.data_ptr(),
                     ws_bytes=ws.numel(), stream=stream)
    return out, ws


def check(x, cum, k, finished=None, eos=-1):
    out, ws = select(x, cum, k, finished, eos)
    torch.cuda.synchronize()
    p, t, s = (o.cpu().numpy() for o in out)
    rp, rt, rs = R.beam(x, cum, k, None if finished is None else finished.cpu().numpy(), eos)
    np.testing.assert_array_equal(p, rp)
    np.testing.assert_array_equal(t, rt)
    np.testing.assert_allclose(s, rs, rtol=S_REL, atol=log_sum_bound(x))
    return out


SIZES = [  # batch, beams, vocab, k
    (1, 1, 1, 1), (2, 1, 3, 2), (1, 2, 1, 4), (3, 3, 7, 6), (2, 4, 31, 9), (1, 4, 257, 8), (5, 5, 1000, 10),
    (2, 8, 4099, 16), (1, 16, 8191, 32), (1, 64, 300, 128), (1, 33, 2049, 66), (3, 2, 32000, 4), (1, 3, 50257, 128),
    (2, 1, 128_000, 100), (1, 2, 70_001, 1), (1, 1, 262_147, 2), (7, 6, 511, 12),
    (700, 3, 37, 4), (40, 8, 6007, 16),
]


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "b%d_w%d_v%d_k%d" % s)
def test_sizes_and_types(size, kind):
    b, w, v, k = size
    g = gen((size, kind))
    x = (3 * torch.randn(b, w, v, generator=g)).to(R.TYPES[kind]).cuda()
    cum = (-5 * torch.rand(b, w, generator=g)).cuda()
    check(x, cum, k)
    done = (torch.rand(b, w, generator=g) < 0.4).to(torch.uint8).cuda()
    check(x, cum, k, done, eos=v - 1)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_rows_with_strides_and_odd_bases(kind):
    g = gen(("strides", kind))
    for pad, off, v in itertools.product([0, 1, 5, 8], [0, 1, 3], [1000, 9001]):
        flat = torch.randn(2 * 3 * (v + pad) + off, generator=g).to(R.TYPES[kind]).cuda()
        x = flat[off:].view(2, 3, v + pad)[:, :, :v]
        check(x, torch.randn(2, 3, generator=g).cuda(), 7)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
def test_ties_go_to_the_lowest_beam_and_token(kind):
    g = gen(("ties", kind))
    for v, k in [(50, 20), (5000, 8), (5000, 128), (40_000, 16)]:
        x = torch.randint(0, 3, (2, 4, v), generator=g).to(R.TYPES[kind]).cuda()
        check(x, torch.rand(2, 4, generator=g).cuda(), k)       # thousands of equal logits in a row
        cum = torch.zeros(2, 4).cuda()
        x[:, 1:] = x[:, :1]
        check(x, cum, k)                        # and equal beams
        x[:] = 1.5
        check(x, cum, k)                        # nothing but ties


def test_a_row_that_holds_all_the_best():
    """Every candidate in one beam, at one end of the vocabulary, or spread thinly."""
    for v in (3000, 33_333):
        x = torch.zeros(1, 4, v)
        x[0, 2, -200:] = 20 + torch.arange(200) / 64
        check(x.cuda(), torch.zeros(1, 4).cuda(), 128)
        x = torch.zeros(1, 4, v)
        x[0, 1, ::97] = 5 + torch.arange(len(range(0, v, 97))) / 1024
        check(x.cuda(), torch.zeros(1, 4).cuda(), 30)
        x = torch.arange(v).float().expand(1, 4, v) / 512         # ascending: the last are the best
        check(x.contiguous().cuda(), torch.tensor([[0.0, -1e-7, 1e-7, -2e-7]]).cuda(), 40)
        check(-x.contiguous().cuda(), torch.tensor([[0.0, -1e-7, 1e-7, -2e-7]]).cuda(), 40)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
def test_values_that_leave_little_or_nothing(kind):
    low, inf, nan = torch.finfo(R.TYPES[kind]).min, float("inf"), float("nan")
    g = gen(("values", kind))
    for v in (9, 9000):
        x = torch.randn(8, 3, v, generator=g)
        x[0] = -inf                             # a sequence with nothing
        x[1, 0], x[1, 1] = -inf, nan
        x[2, :, 3:] = -inf                      # fewer candidates than k
        x[3] = low
        x[4, 1, 5:] = low
        x[5, 0, 2], x[5, 0, 7] = inf, inf
        x[6, :, ::2] = nan
        x[7, 2] = -0.0
        x = x.to(R.TYPES[kind]).cuda()
        cum = torch.randn(8, 3, generator=g)
        cum[4, 0], cum[5, 2], cum[6, 1] = -inf, nan, inf
        check(x, cum.cuda(), 12)
        done = torch.zeros(8, 3, dtype=torch.uint8)
        done[0, 1] = done[2, 0] = done[4, 0] = done[7, 2] = 1
        check(x, cum.cuda(), 12, done.cuda(), eos=1)
        check(x, cum.cuda(), 2, done.cuda(), eos=0)


def test_beams_closer_than_fp32_are_ordered_in_64_bits():
    """Beams whose keys differ by less than fp32 sums can tell."""
    g = gen("near")
    for v in (64, 5000, 40_000):
        x = torch.randn(4, 4, v, generator=g)
        x[:, 1:] = x[:, :1]                     # equal rows: the cums decide
        cum = torch.full((4, 4), -3.0)
        for w in range(4):                      # one step of fp32 apart, in both directions
            cum[:, w] += (w % 3) * 2.4e-7
        check(x.cuda(), cum.cuda(), 24)
        x[:, 2, v // 2] += 1e-4                 # sums that differ in their last digits
        x[:, 3, v // 3] -= 1e-5
        check(x.cuda(), cum.cuda(), 24)


def test_cums_far_from_zero():
    g = gen("far")
    x = (4 * torch.randn(3, 5, 2000, generator=g)).cuda()
    check(x, (-1e4 + torch.rand(3, 5, generator=g)).cuda(), 20)
    check(x, (1e6 * torch.randn(3, 5, generator=g)).cuda(), 20)
    check(300 * x, torch.randn(3, 5, generator=g).cuda(), 20)       # spread over thousands


def test_rows_whose_largest_logits_come_late():
    """References of sums that grow along the row, by little and by much."""
    g = gen("late")
    for v in (5000, 70_000, 262_144):
        x = torch.randn(1, 3, v, generator=g)
        x[0, 0] += torch.linspace(0, 12, v)
        x[0, 1] += torch.linspace(-300, 60, v)
        x[0, 2, -3:] += 45
        for kind in ("fp32", "bf16"):
            check(x.to(R.TYPES[kind]).cuda(), torch.tensor([[0.0, 1.0, 2.0]]).cuda(), 12)


def test_scores_over_the_cums():
    g = gen("over")
    x, cum = torch.randn(4, 5, 3000, generator=g).cuda(), torch.randn(4, 5, generator=g).cuda()
    want, ws = select(x, cum, 5)
    want = [t.clone() for t in want]
    got = [torch.empty_like(want[0]), torch.empty_like(want[1]), cum]
    for _ in range(3):
        cum.copy_(torch.randn(4, 5, generator=g))
        want, _ = select(x, cum.clone(), 5)
        select(x, cum, 5, ws=ws, out=got)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_results_do_not_depend_on_the_call_before():
    g = gen("again")
    x = torch.randn(2, 4, 20_000, generator=g).cuda()
    y = (5 + torch.randn(2, 4, 20_000, generator=g)).cuda()
    cum = torch.zeros(2, 4).cuda()
    first, ws = select(x, cum, 8)
    first = [t.clone() for t in first]
    select(y, cum, 8, ws=ws)
    again, _ = select(x, cum, 8, ws=ws)
    for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_no_batch():
    M.BeamSearch(4, 100, 8).select_device(0, 0, 0, 0, 0, 0)


# --------------------------------------------------------------- reordering
@pytest.mark.parametrize("beams", [1, 2, 3, 4, 5, 8, 9, 16, 17, 40, 64])
@pytest.mark.parametrize("row", [1, 2, 6, 24, 100, 4096, 5008])
def test_reorder(beams, row):
    g = gen((beams, row))
    for outer, batch in [(1, 1), (3, 2)]:
        x = torch.randint(0, 255, (outer, batch, beams, row), generator=g, dtype=torch.uint8)
        parents = torch.randint(-2, beams + 2, (batch, beams), generator=g, dtype=torch.int32)
        y = x.cuda()
        M.beam_reorder_device(y.data_ptr(), parents.cuda().data_ptr(), outer, batch, beams, row)
        torch.cuda.synchronize()
        assert torch.equal(y.cpu(), R.reorder(x, parents.tolist()))


@pytest.mark.parametrize("beams", [2, 4, 7, 20])
def test_reorder_parts_of_a_cache(beams):
    """[layer][batch][beam][head][slot][dim] with only the first slots in use, parents as
    the first columns of a wider table; what lies between stays."""
    g = gen(("cache", beams))
    for used, dim, kind in itertools.product([1, 9, 16], [20, 64], [torch.bfloat16, torch.float32]):
        x = torch.randn(5, 3, beams, 2, 16, dim, generator=g).to(kind)
        table = torch.randint(0, beams, (3, 2 * beams), generator=g, dtype=torch.int32)
        y, line = x.cuda(), dim * x.element_size()
        M.beam_reorder_device(y.data_ptr(), table.cuda().data_ptr(), 5, 3, beams, used * line, segments=2,
                              segment_stride=16 * line, parent_stride=2 * beams)
        want = x.clone()
        want[:, :, :, :, :used] = R.reorder(x, table[:, :beams].tolist())[:, :, :, :, :used]
        assert torch.equal(y.cpu(), want)


def test_reorder_of_many_outer_rows_and_of_none():
    g = gen("outer")
    x = torch.randint(0, 2 ** 30, (30_000, 3, 2, 8), generator=g, dtype=torch.int32)
    parents = torch.tensor([[1, 0], [0, 0], [0, 1]], dtype=torch.int32)
    y, q = x.cuda(), parents.cuda()
    M.beam_reorder_device(y.data_ptr(), q.data_ptr(), 30_000, 3, 2, 32)
    assert torch.equal(y.cpu(), R.reorder(x, parents.tolist()))
    M.beam_reorder_device(0, 0, 0, 3, 2, 32)
    M.beam_reorder_device(0, 0, 3, 3, 2, 0)
