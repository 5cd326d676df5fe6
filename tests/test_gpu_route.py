"""Routing to experts on the GPU against the 64-bit definition (select_ref.route): ids
and lists equal, weights and gradients within bounds that follow from their
arithmetic."""
import itertools
import zlib

import numpy as np
import pytest
import torch

import mflat_b200 as M
import select_ref as R

pytestmark = pytest.mark.gpu

# Relative error of a weight: expf and a division (2^-22 each), the softmax's sum --
# terms off by 2^-22 + |d| 2^-23 at distance d below the maximum, d weighted by its own
# probability (at most ln E + 1 < 8), ten levels of a tree of additions -- and the scale.
W_REL = 2 * 2.0 ** -22 + 2.0 ** -22 + 8 * 2.0 ** -23 + 12 * 2.0 ** -24
TINY = 2.0 ** -125      # below it fp32 loses digits


def gen(seed):
    return torch.Generator().manual_seed(zlib.crc32(repr(seed).encode()))


def dev(t):
    return None if t is None else t.cuda()


def ptr(t):
    return 0 if t is None else t.data_ptr()


def run(x, k, score, bias=None, mask=None, lists=True, stream=0, stride=None, **kw):
    names = {"kept": "groups_kept", "top": "group_top"}
    kind = {v: n for n, v in R.TYPES.items()}[x.dtype]
    t, n = x.shape
    r = M.Router(n, k, score=score, dtype=kind, **{names.get(a, a): v for a, v in kw.items()})
    ids = torch.full((t, k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((t, k), -7.0, device="cuda")
    start = torch.full((n + 1,), -7, dtype=torch.int32, device="cuda")
    slots = torch.full((t * k,), -7, dtype=torch.int32, device="cuda")
    ws = torch.empty(max(1, r.workspace_bytes(t)), dtype=torch.uint8, device="cuda")
    r.route_device(x.data_ptr(), t, ids.data_ptr(), w.data_ptr(), stride=stride or x.stride(0), bias=ptr(bias),
                   mask=ptr(mask), start=ptr(start) if lists else 0, slots=ptr(slots) if lists else 0,
                   ws=ptr(ws), ws_bytes=ws.numel(), stream=stream)
    torch.cuda.synchronize()
    return ids.cpu().numpy(), w.cpu().numpy(), start.cpu().numpy(), slots.cpu().numpy()


def check(x, k, score, bias=None, mask=None, **kw):
    ids, w, start, slots = run(x, k, score, bias, mask, **kw)
    ref = {a: v for a, v in kw.items() if a not in ("lists", "stream", "stride")}
    rid, rw = R.route(x, k, score, bias, None if mask is None else mask.cpu().numpy(), **ref)
    np.testing.assert_array_equal(ids, rid)
    np.testing.assert_allclose(w, rw, rtol=W_REL, atol=TINY * max(1.0, abs(kw.get("scale", 1.0))))
    rs, ro = R.lists(rid, x.shape[1])
    np.testing.assert_array_equal(start, rs)
    np.testing.assert_array_equal(slots[:len(ro)], ro)
    assert (slots[len(ro):] == -7).all()        # left as they were
    return ids, w


SIZES = [  # tokens, experts, k
    (1, 1, 1), (3, 2, 2), (5, 5, 3), (70, 8, 2), (33, 13, 4), (129, 16, 16), (64, 17, 5), (257, 32, 32),
    (40, 60, 4), (100, 64, 6), (31, 100, 8), (513, 128, 8), (77, 255, 7), (640, 256, 8), (19, 257, 8),
    (65, 512, 10), (9, 1000, 31), (12, 1024, 32), (2100, 96, 3),
]


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "t%d_e%d_k%d" % s)
def test_sizes_and_types(size, kind):
    t, n, k = size
    g = gen((size, kind))
    for i, (score, with_bias, renorm) in enumerate(itertools.product(["softmax", "sigmoid"], [0, 1], [False, True])):
        x = (2 * torch.randn(t, n, generator=g)).to(R.TYPES[kind]).cuda()
        bias = (0.1 * torch.randn(n, generator=g)).cuda() if with_bias else None
        mask = (torch.rand(t, generator=g) < 0.8).to(torch.uint8).cuda() if i % 2 else None
        check(x, k, score, bias, mask, renormalise=renorm, scale=1.0 + i)


GROUPS = [  # tokens, experts, groups, kept, top, k
    (50, 256, 8, 4, 2, 8), (50, 256, 8, 1, 1, 8), (40, 160, 8, 3, 2, 6), (33, 64, 2, 1, 2, 8), (33, 64, 32, 5, 2, 4),
    (20, 60, 4, 2, 1, 4), (20, 16, 4, 2, 2, 3), (20, 8, 8, 3, 2, 2), (10, 1024, 16, 4, 2, 8), (9, 7, 7, 7, 1, 7),
    (30, 96, 3, 2, 2, 5), (12, 512, 4, 2, 1, 8),
]


@pytest.mark.parametrize("case", GROUPS, ids=lambda c: "t%d_e%d_g%d_%d_%d_k%d" % c)
def test_groups(case):
    t, n, groups, kept, top, k = case
    g = gen(case)
    for score, with_bias in itertools.product(["softmax", "sigmoid"], [0, 1]):
        for kind in ("fp32", "bf16"):
            x = torch.randn(t, n, generator=g).to(R.TYPES[kind]).cuda()
            bias = (0.2 * torch.randn(n, generator=g)).cuda() if with_bias else None
            check(x, k, score, bias, renormalise=True, scale=2.5, groups=groups, kept=kept, top=top)


def test_rows_with_strides_and_odd_bases():
    g = gen("strides")
    for kind, pad, off in itertools.product(["fp32", "bf16"], [1, 3, 8], [0, 1, 4]):
        wide = torch.randn(37, 64 + pad, generator=g).to(R.TYPES[kind]).cuda()
        flat = torch.cat([torch.zeros(off, dtype=wide.dtype, device="cuda"), wide.reshape(-1)])
        x = flat[off:].view(37, 64 + pad)[:, :64]
        assert x.stride(0) == 64 + pad
        check(x, 6, "softmax", renormalise=True)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_values_that_leave_little_or_nothing(kind, score):
    n, low, inf = 24, torch.finfo(R.TYPES[kind]).min, float("inf")
    rows = torch.zeros(10, n)
    rows[0] = -inf                              # nothing to choose
    rows[1] = low                               # all at the type's lowest value
    rows[2], rows[2, 5] = low, 1.0
    rows[3], rows[3, 7] = -inf, 0.5             # one choice, k asks for more
    rows[4, 3], rows[4, 9] = float("nan"), float("nan")
    rows[5, 11], rows[5, 20] = inf, inf
    rows[6] = float("nan")
    rows[7] = torch.arange(n) // 4              # ties
    rows[8] = -80.0                             # scores near the end of fp32
    rows[9, ::2] = -0.0                         # both zeros are one value
    x = rows.to(R.TYPES[kind]).cuda()
    bias = torch.linspace(-0.3, 0.3, n).cuda()
    odd = bias.clone()
    odd[2], odd[4] = -inf, float("nan")
    for b, renorm in itertools.product([None, bias, odd, torch.zeros(n).cuda()], [False, True]):
        check(x, 5, score, b, renormalise=renorm)
        check(x, 5, score, b, renormalise=renorm, groups=6, kept=2, top=2)


@pytest.mark.parametrize("n", [64, 200, 256, 512, 1024])
def test_wide_rows_of_equals_and_of_strange_values(n):
    """More equal logits than a warp ranks, and -inf, NaN and infinities among them."""
    inf, nan = float("inf"), float("nan")
    g = gen(("wide", n))
    x = torch.zeros(12, n)
    x[1] = 3.0
    x[2] = torch.randint(0, 2, (n,), generator=g).float()
    x[3, ::3] = -inf
    x[4, 1::2] = nan
    x[5, n // 2:] = -inf
    x[6] = -inf
    x[6, n - 1] = 1.0
    x[7, 5], x[7, n - 2] = inf, inf
    x[8:] = torch.randn(4, n, generator=g)
    x[9, ::7] = nan
    bias = 0.1 * torch.randn(n, generator=g)
    bias[::5], bias[3], bias[n // 2] = nan, -inf, inf
    x, bias = x.cuda(), bias.cuda()
    for score, b in itertools.product(["softmax", "sigmoid"], [None, bias, torch.zeros(n).cuda()]):
        for k in (1, 8, 32):
            check(x, k, score, b, renormalise=k == 8)
        for groups, kept, top in [(8, 3, 2), (8, 8, 1), (4, 1, 2)]:
            check(x, 4, score, b, groups=groups, kept=kept, top=top)


def test_far_logits_keep_their_quotients():
    """sigmoid scores that underflow fp32 still divide: weights from exponents."""
    x = torch.tensor([[-200.0, -201.0, -203.0, -400.0], [300.0, 250.0, -250.0, 0.0]]).cuda()
    check(x, 3, "sigmoid", renormalise=True)
    check(x, 3, "softmax", renormalise=True)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_scores_closer_than_fp32_are_ordered_in_64_bits(score):
    """Biases that bring the sums of many experts within 1e-9 of one another."""
    g = gen(("near", score))
    x = torch.randn(200, 64, generator=g)
    base = torch.randn(1, 64, generator=g)
    x = torch.where(torch.rand(200, 1, generator=g) < 0.7, base, x)     # most tokens share their logits
    _, s = R.scores(base[0].double().numpy(), score)
    bias = torch.from_numpy(0.75 - s).float()       # s + bias differs from 0.75 by the bias's rounding only
    xs, bs = x.cuda(), bias.cuda()
    check(xs, 8, score, bs)
    check(xs, 8, score, bs, groups=8, kept=3, top=2)
    check(xs, 8, score, 100 + bs)                   # large biases: the tolerance grows with them
    check(xs, 8, score, bs * 0 + 0.5)               # equal biases: ties wherever the logits tie


def test_many_tokens_and_lists():
    g = gen("many")
    for t, n, k in [(4096, 64, 8), (20_000, 16, 2), (3001, 256, 8)]:
        x = (torch.randn(t, n, generator=g) + 0.5 * torch.randn(n, generator=g)).bfloat16().cuda()
        mask = (torch.rand(t, generator=g) < 0.9).to(torch.uint8).cuda()
        check(x, k, "softmax", None, mask, renormalise=True)
    x = torch.zeros(2500, 40).cuda()                # every token chooses the same experts
    check(x, 4, "sigmoid")


def test_more_tokens_than_16_bit_counts_hold():
    """Tiles are cut at 65,535 tokens; one expert takes nearly all of them."""
    t, n = 9_800_000, 3
    x = torch.zeros(t, n, device="cuda")
    x[:, 1] = 1.0
    x[::1000, 2] = 2.0
    r = M.Router(n, 1)
    ids = torch.empty(t, 1, dtype=torch.int32, device="cuda")
    w = torch.empty(t, 1, device="cuda")
    start = torch.empty(n + 1, dtype=torch.int32, device="cuda")
    slots = torch.empty(t, dtype=torch.int32, device="cuda")
    ws = torch.empty(r.workspace_bytes(t), dtype=torch.uint8, device="cuda")
    r.route_device(x.data_ptr(), t, ids.data_ptr(), w.data_ptr(), start=start.data_ptr(), slots=slots.data_ptr(),
                   ws=ws.data_ptr(), ws_bytes=ws.numel())
    want = x.argmax(1)
    assert torch.equal(ids[:, 0].long(), want)
    assert start.tolist() == [0, 0, t - t // 1000, t]
    assert torch.equal(slots.long(), torch.sort(want, stable=True).indices)


def test_no_tokens_gives_empty_lists():
    r = M.Router(10, 2)
    start = torch.full((11,), 5, dtype=torch.int32, device="cuda")
    r.route_device(0, 0, 0, 0, start=start.data_ptr())
    assert (start.cpu() == 0).all()
    r.route_device(0, 0, 0, 0)
    r.backward_device(0, 0, 0, 0, 0)


def test_without_lists():
    x = torch.randn(100, 32, generator=gen("nolists")).cuda()
    ids, w, start, slots = run(x, 4, "softmax", lists=False)
    np.testing.assert_array_equal(ids, R.route(x, 4, "softmax")[0])
    assert (start == -7).all() and (slots == -7).all()


# --------------------------------------------------------------- backward
def backward(x, ids, g, score, out=None, grad_stride=0, **kw):
    kind = {v: n for n, v in R.TYPES.items()}[x.dtype]
    r = M.Router(x.shape[1], ids.shape[1], score=score, dtype=kind, **kw)
    out = torch.full_like(x, 3.0) if out is None else out
    r.backward_device(x.data_ptr(), x.shape[0], ids.data_ptr(), g.data_ptr(), out.data_ptr(),
                      stride=x.stride(0), grad_stride=grad_stride or out.stride(0))
    torch.cuda.synchronize()
    return out


def check_grad(x, ids, g, score, kind, **kw):
    out = R.f64(backward(x, ids, g, score, **kw))
    ref, size = R.route_grad(x, ids.cpu().numpy(), g, score, **kw)
    # a weight's error, the sum over k <= 32 products and the factor 1 - s, relative to the
    # terms' sizes (twice: the sum and what it is taken from); then one rounding to the type
    bound = 2 * (2 * W_REL + 36 * 2.0 ** -24) * size + R.HALF[kind] * np.abs(ref) + \
        (2.0 ** -25 if kind == "fp16" else TINY)
    assert (np.abs(out - ref) <= bound).all(), np.max(np.abs(out - ref) - bound)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("size", [s for s in SIZES if s[0] < 600], ids=lambda s: "t%d_e%d_k%d" % s)
def test_backward(size, kind):
    t, n, k = size
    gr = gen(("grad", size, kind))
    for score, renorm in itertools.product(["softmax", "sigmoid"], [False, True]):
        x = (1.5 * torch.randn(t, n, generator=gr)).to(R.TYPES[kind]).cuda()
        ids = torch.topk(x.float(), k, dim=-1).indices.to(torch.int32)
        g = torch.randn(t, k, generator=gr).cuda()
        check_grad(x, ids, g, score, kind, renormalise=renorm, scale=1.7)


def test_backward_padding_repeats_and_strange_entries():
    gr = gen("odd ids")
    x = torch.randn(40, 30, generator=gr).cuda()
    x[5] = float("-inf")
    x[6, ::2] = float("nan")
    ids = torch.randint(-3, 34, (40, 6), generator=gr, dtype=torch.int32).cuda()
    ids[7] = 4                                  # the same expert throughout
    ids[8] = -1
    g = torch.randn(40, 6, generator=gr)
    g[8] = float("nan")                         # behind -1: not read into anything
    g = g.cuda()
    for score, renorm in itertools.product(["softmax", "sigmoid"], [False, True]):
        check_grad(x, ids, g, score, "fp32", renormalise=renorm, scale=0.5)


def test_backward_over_the_logits_and_into_strides():
    gr = gen("inplace")
    for kind in ("fp32", "bf16"):
        wide = torch.randn(50, 71, generator=gr).to(R.TYPES[kind]).cuda()
        x = wide[:, :64]
        ids = torch.topk(x.float(), 4, dim=-1).indices.to(torch.int32)
        g = torch.randn(50, 4, generator=gr).cuda()
        want = backward(x, ids, g, "softmax")
        out = torch.full((50, 80), 3.0, dtype=x.dtype, device="cuda")
        backward(x, ids, g, "softmax", out=out[:, :64])
        assert torch.equal(out[:, :64], want) and (out[:, 64:] == 3.0).all()
        rest = wide[:, 64:].clone()
        backward(x, ids, g, "softmax", out=x)
        assert torch.equal(x, want) and torch.equal(wide[:, 64:], rest)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
def test_backward_against_differences(score, renorm):
    """The forward pass's own weights, moved one logit at a time in 64 bits by the
    definition; and the kernel's gradient against those quotients."""
    gr = gen(("fd", score, renorm))
    x = torch.randn(6, 12, generator=gr)
    rid, _ = R.route(x, 4, score, renormalise=renorm, scale=1.3)
    ids = torch.from_numpy(rid).to(torch.int32)
    g = torch.randn(6, 4, generator=gr)
    got = R.f64(backward(x.cuda(), ids.cuda(), g.cuda(), score, renormalise=renorm, scale=1.3))

    def loss(v, t):
        xi, s = R.scores(v, score)
        w = 1.3 * (R.quotients(xi[rid[t]], score) if renorm else s[rid[t]])
        return float(w @ g[t].double().numpy())

    h = 1e-5        # error of a central difference: h^2 / 6 of a third derivative of order 1, 2^-53 / h
    for t in range(6):
        for e in range(12):
            v = x[t].double().numpy()
            up, down = v.copy(), v.copy()
            up[e] += h
            down[e] -= h
            assert abs((loss(up, t) - loss(down, t)) / (2 * h) - got[t, e]) < 1e-5
