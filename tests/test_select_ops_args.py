"""Refusals of the selection operators, without a device: every size, type, stride,
pointer and workspace outside the stated limits comes back as a status before
anything is enqueued."""
import ctypes

import numpy as np
import pytest

import mflat_b200 as M

NULL, BAD = 1, 2
P = 1 << 20         # an aligned address that no refused call reads


def status(fn, *a, **kw):
    with pytest.raises(M.MflatError) as e:
        fn(*a, **kw)
    return e.value.status


def route(r, **kw):
    a = dict(logits=P, tokens=4, ids=P, weights=P)
    a.update(kw)
    return status(r.route_device, **a)


@pytest.mark.parametrize("bad", [
    dict(experts=0), dict(experts=1025, k=4), dict(experts=-5), dict(k=0), dict(k=33), dict(k=9), dict(score=2),
    dict(score=-1), dict(dtype=3), dict(dtype=-1), dict(groups=0), dict(groups=3), dict(groups=33, experts=66, k=2),
    dict(groups=4, groups_kept=0), dict(groups=4, groups_kept=5), dict(group_top=0), dict(group_top=3)])
def test_router_specs(built_lib, bad):
    spec = dict(experts=8, k=2)
    spec.update(bad)
    r = M.Router(**spec)
    assert route(r) == BAD
    assert status(r.backward_device, P, 4, P, P, P) == BAD
    assert r.workspace_bytes(4) == 0


def test_route_arguments(built_lib):
    r = M.Router(64, 4, dtype="bf16")
    for name in ("logits", "ids", "weights"):
        assert route(r, **{name: 0}) == NULL
    assert route(r, start=P) == NULL and route(r, slots=P) == NULL      # both lists or neither
    assert route(r, tokens=-1) == BAD and route(r, tokens=2 ** 30) == BAD
    assert route(r, stride=63) == BAD and route(r, stride=-64) == BAD
    assert route(r, logits=P + 1) == BAD
    for name in ("ids", "weights", "bias"):
        assert route(r, **{name: P + 2}) == BAD
    assert route(r, start=P + 1, slots=P) == BAD and route(r, start=P, slots=P + 2) == BAD
    need = r.workspace_bytes(100_000)
    if need:
        lists = dict(tokens=100_000, start=P, slots=P)
        assert route(r, **lists) == BAD
        assert route(r, ws=P, ws_bytes=need - 1, **lists) == BAD
        assert route(r, ws=P + 16, ws_bytes=need, **lists) == BAD
    for i in (0, 2, 3, 4):
        a = [P, 4, P, P, P]
        a[i] = 0
        assert status(r.backward_device, *a) == NULL
    assert status(r.backward_device, P, -1, P, P, P) == BAD
    assert status(r.backward_device, P, 4, P, P, P, stride=60) == BAD
    assert status(r.backward_device, P, 4, P, P, 2 * P, grad_stride=60) == BAD
    assert status(r.backward_device, P, 4, P, P, P, stride=64, grad_stride=80) == BAD    # over the logits
    assert status(r.backward_device, P, 4, P + 1, P, 2 * P) == BAD
    assert status(r.backward_device, P, 4, P, P, P + 1) == BAD
    assert built_lib.mflat_route_device(None, P, 0, 1, 0, 0, P, P, 0, 0, 0, 0, -1, 0) == NULL
    assert built_lib.mflat_route_backward_device(None, P, 0, 1, P, P, P, 0, -1, 0) == NULL
    assert built_lib.mflat_route_workspace_bytes(None, 5) == 0
    assert route(M.Router(8, 2, device=10_000)) in (BAD, 6)             # no such device


@pytest.mark.parametrize("bad", [
    dict(beams=0), dict(beams=65), dict(vocab=0), dict(vocab=-1), dict(k=0), dict(k=129), dict(dtype=3),
    dict(eos=-2), dict(eos=100)])
def test_beam_specs(built_lib, bad):
    spec = dict(beams=4, vocab=100, k=8)
    spec.update(bad)
    b = M.BeamSearch(**spec)
    assert b.workspace_bytes(2) == 0
    assert status(b.select_device, P, P, 2, P, P, P, ws=P, ws_bytes=1 << 30) == BAD


def test_beam_arguments(built_lib):
    b = M.BeamSearch(4, 1000, 8, dtype="fp16")
    need = b.workspace_bytes(3)
    ok = dict(logits=P, cum=P, batch=3, parents=P, tokens=P, scores=2 * P, ws=P, ws_bytes=need)
    for name in ("logits", "cum", "parents", "tokens", "scores"):
        assert status(b.select_device, **{**ok, name: 0}) == NULL
        assert status(b.select_device, **{**ok, name: P + 1}) == BAD
    assert status(b.select_device, **{**ok, "batch": -1}) == BAD
    assert status(b.select_device, **{**ok, "batch": 2 ** 30, "ws_bytes": 1 << 62}) == BAD
    assert status(b.select_device, **{**ok, "stride": 999}) == BAD
    assert status(b.select_device, **{**ok, "finished": P}) == BAD      # finished beams without an eos
    assert status(b.select_device, **{**ok, "scores": P, "cum": P}) == BAD      # over the cums, with k != beams
    if need:
        assert status(b.select_device, **{**ok, "ws": 0}) == BAD
        assert status(b.select_device, **{**ok, "ws": P + 8}) == BAD
        assert status(b.select_device, **{**ok, "ws_bytes": need - 1}) == BAD
    assert built_lib.mflat_beam_select_device(None, P, 0, P, 0, 1, P, P, P, P, 1 << 20, -1, 0) == NULL
    assert built_lib.mflat_beam_workspace_bytes(None, 5) == 0


def test_reorder_arguments(built_lib):
    f, ok = M.beam_reorder_device, dict(states=P, parents=P, outer=2, batch=3, beams=4, segment_bytes=64)
    assert status(f, **{**ok, "states": 0}) == NULL and status(f, **{**ok, "parents": 0}) == NULL
    for name, v in [("beams", 0), ("beams", 65), ("outer", -1), ("batch", -1), ("segments", -1), ("segment_bytes", -1),
                    ("parent_stride", 3), ("row_stride", 63), ("outer_stride", 12 * 64 - 1), ("parents", P + 2)]:
        assert status(f, **{**ok, name: v}) == BAD, name
    assert status(f, **{**ok, "segments": 2, "segment_stride": 63}) == BAD
    assert status(f, **{**ok, "segments": 2, "segment_stride": 128, "row_stride": 191}) == BAD
    assert status(f, **{**ok, "segments": 2, "segment_stride": -128}) == BAD
    assert status(f, **{**ok, "segments": 2 ** 31 - 1, "segment_stride": 2 ** 62}) == BAD
    assert status(f, **{**ok, "row_stride": -64}) == BAD
    assert status(f, **{**ok, "segment_bytes": 2 ** 62}) == BAD


@pytest.mark.parametrize("bad", [
    dict(heads=0), dict(group=0), dict(capacity=0), dict(capacity=2 ** 30 + 1), dict(budget=0), dict(budget=101), dict(recent=-1), dict(sink=-1),
    dict(recent=30, sink=21), dict(recent=2 ** 31 - 1, sink=2 ** 31 - 1), dict(dtype=5), dict(key_bytes=-1),
    dict(value_bytes=-16)])
def test_cache_specs(built_lib, bad):
    spec = dict(heads=2, group=4, capacity=100, budget=50, key_bytes=16, value_bytes=16)
    spec.update(bad)
    c = M.CacheEviction(**spec)
    assert c.workspace_bytes(2) == 0
    assert status(c.evict_device, 2, P, P, P, P, P, P, 2 * P, ws=P, ws_bytes=1 << 30) == BAD


def test_cache_arguments(built_lib):
    c = M.CacheEviction(2, 4, 100, 50, 16, 16, dtype="bf16")
    need = c.workspace_bytes(3)
    ok = dict(batch=3, lens=P, seen=P, acc=P, pos=P, keys=P, values=P, out_lens=2 * P, weights=P, queries=1, ws=P,
              ws_bytes=need)
    for name in ("lens", "seen", "acc", "pos", "out_lens", "keys", "values"):
        assert status(c.evict_device, **{**ok, name: 0}) == NULL
    for name in ("lens", "seen", "acc", "pos", "out_lens", "out_acc", "out_pos", "weights", "rows"):
        assert status(c.evict_device, **{**ok, name: P + 1}) == BAD, name
    assert status(c.evict_device, **{**ok, "out_lens": P}) == BAD       # the lengths themselves
    assert status(c.evict_device, **{**ok, "batch": -1}) == BAD
    assert status(c.evict_device, **{**ok, "batch": 40_000, "ws_bytes": 1 << 62}) == BAD
    assert status(c.evict_device, **{**ok, "queries": -1}) == BAD
    assert status(c.evict_device, **{**ok, "queries": 2 ** 30}) == BAD
    assert status(c.evict_device, **{**ok, "weight_stride": (1, 1, -1)}) == BAD
    if need:
        assert status(c.evict_device, **{**ok, "ws": 0}) == BAD
        assert status(c.evict_device, **{**ok, "ws": P + 4}) == BAD
        assert status(c.evict_device, **{**ok, "ws_bytes": need - 1}) == BAD
    for stride in [(3200, 1600, 15), (3200, 15, 16), (15, 1600, 16), (-3200, 1600, 16), (0, 1600, 16), (3199, 1600, 16),
                   (3200, 1599, 16), (3200, 16, 31), (1 << 62, 1600, 16)]:
        short = M.CacheEviction(2, 4, 100, 50, 16, 16, key_stride=stride)
        assert status(short.evict_device, **ok) == BAD, stride
        short = M.CacheEviction(2, 4, 100, 50, 16, 16, value_stride=stride)
        assert status(short.evict_device, **ok) == BAD, stride
    assert built_lib.mflat_cache_evict_device(None, 1, P, P, 0, 0, None, *[P] * 9, 1 << 20, -1, 0) == NULL
    assert built_lib.mflat_cache_workspace_bytes(None, 5) == 0


def test_specs_match_the_header(built_lib):
    """Sizes of the binding's structures as a C compiler lays the header's out."""
    import os
    import subprocess
    import tempfile
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with tempfile.TemporaryDirectory() as d:
        src = os.path.join(d, "s.c")
        with open(src, "w") as f:
            f.write('#include <stdio.h>\n#include "mflat.h"\nint main(void) { printf("%zu %zu %zu %zu %zu", '
                    'sizeof(mflat_router_t), sizeof(mflat_beam_t), sizeof(mflat_cache_t), '
                    'offsetof(mflat_cache_t, key_bytes), offsetof(mflat_router_t, scale)); return 0; }\n')
        subprocess.run(["gcc", "-I", os.path.join(root, "include"), src, "-o", os.path.join(d, "s")], check=True)
        out = subprocess.run([os.path.join(d, "s")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in out] == [ctypes.sizeof(M.RouterSpec), ctypes.sizeof(M.BeamSpec), ctypes.sizeof(M.CacheSpec),
                                     M.CacheSpec.key_bytes.offset, M.RouterSpec.scale.offset]


def test_refusals_are_logged(built_lib):
    seen = []
    handler = M.LOG_HANDLER(lambda level, msg, user: seen.append((level, msg.decode())))
    built_lib.mflat_set_log_handler(handler, None)
    try:
        assert status(M.BeamSearch(65, 10, 2).select_device, P, P, 1, P, P, P) == BAD
    finally:
        built_lib.mflat_set_log_handler(M.LOG_HANDLER(0), None)
    assert seen == [(2, "beam select: beams=65 outside [1, 64]")]
