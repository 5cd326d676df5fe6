"""Eviction from a key/value cache on the GPU against the 64-bit definition
(select_ref.evict): kept slots, positions, rows and accumulated weights all equal."""
import itertools
import zlib

import numpy as np
import pytest
import torch

import mflat_b200 as M
import select_ref as R

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(zlib.crc32(repr(seed).encode()))


def make(g, b, h, cap, lens, dim=8, kind=torch.bfloat16, spread=1):
    acc = torch.rand(b, h, cap, generator=g)
    pos = torch.stack([torch.randperm(cap, generator=g) for _ in range(b * h)]).view(b, h, cap)
    for i, n in enumerate(lens):        # live positions are 0 .. n - 1 in some order
        for j in range(h):
            if n > 0:
                pos[i, j, :n] = torch.randperm(n, generator=g)
    pos = (pos * spread).to(torch.int32)
    keys = torch.randn(b, h, cap, dim, generator=g).to(kind)
    values = torch.randn(b, h, cap, 2 * dim, generator=g).to(kind)
    return acc, pos, keys, values


def run(lens, seen, acc, pos, keys, values, budget, recent=0, sink=0, weights=None, group=1, rows=None,
        in_place=False, layout="bhs", stream=0, weight_stride=None, queries=None):
    """(lens, acc, pos, keys, values) after the call, on the CPU."""
    b, h, cap = acc.shape
    kind = {v: n for n, v in R.TYPES.items()}[weights.dtype] if weights is not None else "fp32"
    lens, seen = torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(seen, dtype=torch.int32).cuda()
    acc, pos = acc.cuda(), pos.cuda()
    kb, vb = keys.shape[-1] * keys.element_size(), values.shape[-1] * values.element_size()
    strides = {}
    if layout == "bsh":                 # [sequence][slot][head][row]
        keys, values = keys.transpose(1, 2).contiguous(), values.transpose(1, 2).contiguous()
        strides = {"key_stride": (cap * h * kb, kb, h * kb), "value_stride": (cap * h * vb, vb, h * vb)}
    keys, values = keys.cuda(), values.cuda()
    op = M.CacheEviction(h, group, cap, budget, kb, vb, recent=recent, sink=sink, dtype=kind, **strides)
    ws = torch.randint(0, 255, (op.workspace_bytes(b),), dtype=torch.uint8, device="cuda")
    out_lens = torch.full((b,), -7, dtype=torch.int32, device="cuda")
    out_acc = acc if in_place else torch.full_like(acc, -7.0)
    out_pos = pos if in_place else torch.full_like(pos, -7)
    w = weights.cuda() if weights is not None else None
    r = torch.tensor(rows, dtype=torch.int32).cuda() if rows is not None else None
    q = queries if queries is not None else (w.shape[2] if w is not None else 0)
    torch.cuda.synchronize()
    op.evict_device(b, lens.data_ptr(), seen.data_ptr(), acc.data_ptr(), pos.data_ptr(), keys.data_ptr(),
                    values.data_ptr(), out_lens.data_ptr(), out_acc=0 if in_place else out_acc.data_ptr(),
                    out_pos=0 if in_place else out_pos.data_ptr(),
                    weights=w.data_ptr() if w is not None else 0, queries=q, weight_stride=weight_stride,
                    rows=r.data_ptr() if r is not None else 0, ws=ws.data_ptr(), ws_bytes=ws.numel(), stream=stream)
    torch.cuda.synchronize()
    if layout == "bsh":
        keys, values = keys.transpose(1, 2), values.transpose(1, 2)
    return [t.cpu() for t in (out_lens, out_acc, out_pos, keys, values)]


def check(lens, seen, acc, pos, keys, values, budget, recent=0, sink=0, weights=None, group=1, rows=None, **kw):
    got = run(lens, seen, acc, pos, keys, values, budget, recent, sink, weights, group, rows, **kw)
    in_place = kw.get("in_place", False)
    rl, total, source = R.evict(lens, seen, acc, pos.numpy(), budget, recent, sink, weights, rows, group)
    np.testing.assert_array_equal(got[0].numpy(), rl)
    for (i, j), at in source.items():
        m = len(at)
        np.testing.assert_array_equal(got[1][i, j, :m].numpy(), total[i, j, at])
        np.testing.assert_array_equal(got[2][i, j, :m].numpy(), pos[i, j, at].numpy())
        for now, before in ((got[3], keys), (got[4], values)):
            assert torch.equal(now[i, j, :m], before[i, j, at])
            assert torch.equal(now[i, j, m:], before[i, j, m:])       # left as they were
        if in_place:
            assert torch.equal(got[2][i, j, m:], pos[i, j, m:])
            assert torch.equal(got[1][i, j, m:].nan_to_num(), acc[i, j, m:].nan_to_num())
        else:
            assert (got[1][i, j, m:] == -7).all() and (got[2][i, j, m:] == -7).all()
    return got


SIZES = [  # batch, heads, group, queries, capacity, lens, budget, recent, sink
    (1, 1, 1, 1, 1, [1], 1, 0, 0), (2, 1, 2, 1, 5, [5, 0], 3, 1, 1), (3, 2, 1, 3, 9, [9, 1, 4], 4, 0, 0),
    (2, 2, 4, 1, 70, [65, 64], 64, 8, 4), (4, 1, 1, 2, 300, [300, 299, 17, 0], 100, 50, 50),
    (1, 3, 2, 1, 1025, [1025], 1024, 0, 1), (2, 2, 1, 7, 2000, [2000, 1500], 37, 10, 4),
    (1, 2, 3, 5, 4099, [4098], 4000, 100, 0), (1, 1, 1, 1, 9000, [9000], 1, 0, 0), (1, 2, 2, 2, 8193, [8000], 4096, 0, 0),
    (3, 8, 4, 1, 130, [129, 130, 128], 128, 16, 4),
    (150, 8, 2, 1, 41, [(7 * i) % 42 for i in range(150)], 20, 5, 1),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", SIZES, ids=lambda c: "b%d_h%d_g%d_q%d_c%d_m%d" % (c[:5] + (c[6],)))
def test_sizes_and_types(case, kind, in_place):
    b, h, group, q, cap, lens, budget, recent, sink = case
    g = gen((case, kind))
    data = make(g, b, h, cap, lens)
    w = torch.softmax(2 * torch.randn(b, h * group, q, cap, generator=g), -1).to(R.TYPES[kind])
    for i, n in enumerate(lens):
        w[i, :, :, n:] = float("nan")           # behind the length: never read
        data[0][i, :, n:] = float("inf")
    check(lens, lens, *data, budget, recent, sink, w, group, in_place=in_place)


def test_nothing_to_add_and_nothing_to_move():
    g = gen("plain")
    data = make(g, 2, 2, 50, [50, 20])
    check([50, 20], [50, 20], *data, 30, 4, 2)
    check([50, 20], [50, 20], *data, 50, 4, 2)
    w = torch.rand(2, 2, 0, 50)
    check([50, 20], [50, 20], *data, 30, 4, 2, w)
    one = make(g, 1, 1, 6, [6])
    check([6], [6], *one, 6)


def test_lengths_outside_the_cache_are_cut_to_it():
    g = gen("lens")
    acc, pos, keys, values = make(g, 3, 1, 40, [40, 0, 40])
    rl, total, source = R.evict([99, -3, 40], [40] * 3, acc, pos.numpy(), 25, 0, 0)
    got = run([99, -3, 40], [40] * 3, acc, pos, keys, values, 25)
    np.testing.assert_array_equal(got[0].numpy(), [25, 0, 25])
    np.testing.assert_array_equal(got[2][0, 0, :25].numpy(), pos[0, 0, source[0, 0]].numpy())
    assert (got[2][1] == -7).all()


def test_ties_stay_at_the_lowest_slots():
    g = gen("ties")
    for cap, budget in [(100, 33), (3000, 2900), (5000, 64)]:
        acc, pos, keys, values = make(g, 2, 2, cap, [cap, cap])
        acc = torch.randint(0, 3, acc.shape, generator=g).float()
        check([cap, cap], [cap, cap], acc, pos, keys, values, budget)
        check([cap, cap], [cap, cap], acc * 0, pos, keys, values, budget, recent=budget // 2)
        check([cap, cap], [cap, cap], -acc, pos, keys, values, budget, sink=3)


def test_protected_entries():
    g = gen("held")
    acc, pos, keys, values = make(g, 1, 2, 200, [200])
    acc[:] = 1 + pos                            # the protected recent are heavy, the sinks light
    check([200], [200], acc, pos, keys, values, 20, 10, 10)
    check([200], [200], -acc, pos, keys, values, 20, 10, 10)
    check([200], [1000], acc, pos, keys, values, 20, 10, 10)        # none is recent
    check([200], [5], acc, pos, keys, values, 20, 20, 0)            # all are: the lowest slots stay
    check([200], [2 ** 31 - 1], acc, pos, keys, values, 20, 20, 0)
    check([200], [-2 ** 31], acc, pos, keys, values, 20, 20, 0)


def test_strange_weights():
    g = gen("strange")
    acc, pos, keys, values = make(g, 1, 1, 64, [64])
    nan, inf = float("nan"), float("inf")
    acc[0, 0, 3], acc[0, 0, 10], acc[0, 0, 40], acc[0, 0, 50] = nan, inf, -inf, 3e38
    acc[0, 0, 60:] = -acc[0, 0, 60:]
    for budget in (1, 2, 3, 10, 61, 62, 63):
        got = run([64], [64], acc, pos, keys, values, budget)
        _, total, source = R.evict([64], [64], acc, pos.numpy(), budget, 0, 0)
        np.testing.assert_array_equal(got[2][0, 0, :budget].numpy(), pos[0, 0, source[0, 0]].numpy())
    w = torch.rand(1, 1, 2, 64, generator=g)
    w[0, 0, 0, 5], w[0, 0, 1, 5] = inf, -inf
    got = run([64], [64], acc, pos, keys, values, 62, weights=w)
    assert np.isin(pos[0, 0, [3, 5]].numpy(), got[2][0, 0, :62].numpy()).sum() == 0


def test_valid_query_rows():
    """A padded batch: rows behind the valid ones hold anything."""
    g = gen("rows")
    data = make(g, 3, 2, 90, [90, 80, 90])
    w = torch.rand(3, 4, 5, 90, generator=g)
    w[0, :, 2:], w[1, :, 0:] = float("nan"), float("nan")
    check([90, 80, 90], [90, 80, 90], *data, 40, 4, 1, w, 2, rows=[2, 0, 5])
    check([90, 80, 90], [90, 80, 90], *data, 40, 4, 1, w[:, :, :2].contiguous(), 2, rows=[2, -4, 99])


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32, torch.uint8])
@pytest.mark.parametrize("dim", [1, 3, 8, 20, 64])
@pytest.mark.parametrize("layout", ["bhs", "bsh"])
def test_rows_of_any_size_and_layout(layout, dim, kind):
    g = gen((layout, dim))
    acc, pos, keys, values = make(g, 2, 3, 150, [150, 120], dim, torch.float32)
    keys, values = (keys * 50).to(kind), (values * 50).to(kind)
    check([150, 120], [150, 120], acc, pos, keys, values, 70, 5, 2, layout=layout)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_weights_with_strides(kind):
    g = gen(("w strides", kind))
    data = make(g, 2, 2, 77, [77, 60])
    big = torch.rand(2, 3, 4, 101, generator=g).to(R.TYPES[kind])       # [b][query][head][slot]
    w = big.permute(0, 2, 1, 3)[..., :77]
    rl = check([77, 60], [77, 60], *data, 30, 0, 0, w.contiguous(), 2)
    got = run([77, 60], [77, 60], *data, 30, weights=big, group=2, queries=3,
              weight_stride=(3 * 4 * 101, 101, 4 * 101))
    for a, b in zip(rl, got):
        assert torch.equal(a, b)


def test_weights_shared_by_all_heads():
    """A stride of 0: one row of weights for every query head."""
    g = gen("shared")
    for cap in (60, 61):
        data = make(g, 2, 2, cap, [cap, 50])
        w = torch.rand(2, 1, 1, cap, generator=g)
        want = check([cap, 50], [cap, 50], *data, 30, 0, 0, w.expand(2, 6, 1, cap).contiguous(), 3)
        got = run([cap, 50], [cap, 50], *data, 30, weights=w, group=3, queries=1, weight_stride=(cap, 0, 0))
        for a, b in zip(want, got):
            assert torch.equal(a, b)


def test_a_value_buffer_alone_and_none():
    g = gen("values only")
    acc, pos, keys, values = make(g, 1, 2, 60, [60])
    lens = torch.tensor([60], dtype=torch.int32).cuda()
    out = torch.zeros(1, dtype=torch.int32).cuda()
    _, _, source = R.evict([60], [60], acc, pos.numpy(), 20, 0, 0)
    for vb in (32, 0):
        a, p, v = acc.cuda(), pos.cuda(), values.cuda()
        op = M.CacheEviction(2, 1, 60, 20, 0, vb)
        ws = torch.empty(op.workspace_bytes(1), dtype=torch.uint8, device="cuda")
        op.evict_device(1, lens.data_ptr(), lens.data_ptr(), a.data_ptr(), p.data_ptr(), 0, v.data_ptr() if vb else 0,
                        out.data_ptr(), ws=ws.data_ptr(), ws_bytes=ws.numel())
        for j in range(2):
            at = source[0, j]
            np.testing.assert_array_equal(p.cpu()[0, j, :20].numpy(), pos[0, j, at].numpy())
            assert torch.equal(v.cpu()[0, j, :20], values[0, j, at if vb else slice(0, 20)])


@pytest.mark.parametrize("cap", [40_000, 150_001, 196_608, 196_609, 300_003, 393_216, 393_217, 500_000])
def test_long_caches(cap):
    g = gen(("long", cap))
    acc, pos, keys, values = make(g, 1, 2, cap, [cap - 3], dim=2)
    w = torch.rand(1, 2, 1, cap, generator=g)
    for budget in (100, cap // 2, cap - 4):
        check([cap - 3], [cap - 3], acc, pos, keys, values, budget, 10, 4, w)


@pytest.mark.parametrize("cap", [196_608, 393_216, 400_000])
def test_long_caches_whose_lower_half_leaves(cap):
    """As many moves as there can be, all of a block's slots holes or tails."""
    g = gen(("half", cap))
    acc, pos, keys, values = make(g, 1, 1, cap, [cap], dim=2)
    acc[:] = torch.arange(cap) / cap
    check([cap], [cap], acc, pos, keys, values, cap // 2, 0, 0)
    check([cap], [cap], -acc, pos, keys, values, cap // 2, 0, 0)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes in one stride."""
    cap, dim = 40, 16
    stride = (1 << 32) + 4096
    raw = torch.zeros(stride + cap * dim * 2, dtype=torch.uint8, device="cuda")
    g = gen("wide")
    acc, pos, keys, _ = make(g, 2, 1, cap, [cap, cap], dim)
    for i in range(2):
        raw[i * stride:i * stride + cap * dim * 2] = keys[i].reshape(-1).view(torch.uint8).cuda()
    lens = torch.tensor([cap, cap], dtype=torch.int32).cuda()
    out = torch.zeros(2, dtype=torch.int32).cuda()
    a, p = acc.cuda(), pos.cuda()
    op = M.CacheEviction(1, 1, cap, 15, dim * 2, 0, key_stride=(stride, cap * dim * 2, dim * 2))
    ws = torch.empty(op.workspace_bytes(2), dtype=torch.uint8, device="cuda")
    op.evict_device(2, lens.data_ptr(), lens.data_ptr(), a.data_ptr(), p.data_ptr(), raw.data_ptr(), 0, out.data_ptr(),
                    ws=ws.data_ptr(), ws_bytes=ws.numel())
    _, _, source = R.evict([cap, cap], [cap, cap], acc, pos.numpy(), 15, 0, 0)
    for i in range(2):
        now = raw[i * stride:i * stride + cap * dim * 2].cpu().view(torch.bfloat16).view(cap, dim)
        assert torch.equal(now[:15], keys[i, 0, source[i, 0]])
        assert torch.equal(now[15:], keys[i, 0, 15:])


def test_no_batch():
    M.CacheEviction(1, 1, 4, 2, 8, 8).evict_device(0, 0, 0, 0, 0, 0, 0, 0)
