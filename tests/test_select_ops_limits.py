"""Sizes at the ends of the stated ranges, and arguments that share memory, without a
device: workspaces that grow with the work, and refusals before anything is enqueued."""
import pytest

import mflat_b200 as M
from test_select_ops_args import BAD, P, route, status

NOWHERE = 10_000        # a device that is not there: a call that passes its checks ends at it


def reasons(built_lib, fn, *a, **kw):
    """What the log says of a refused call."""
    seen = []
    handler = M.LOG_HANDLER(lambda level, msg, user: seen.append(msg.decode()))
    built_lib.mflat_set_log_handler(handler, None)
    try:
        status(fn, *a, **kw)
    finally:
        built_lib.mflat_set_log_handler(M.LOG_HANDLER(0), None)
    return " ".join(seen)


@pytest.mark.parametrize("experts", [2, 300])
def test_router_workspace_up_to_the_last_token(built_lib, experts):
    """Ranks of 2 bytes a choice, counts of 2 bytes for each tile of up to 65,535 tokens."""
    r = M.Router(experts, 1)

    def need(t):
        per = min(65_535, -(-t // 148))
        tiles = -(-t // per)
        return sum((n + 255) // 256 * 256 for n in (2 * t, 2 * tiles * (experts + experts % 2)))

    for t in (1000, 148 * 65_535, 148 * 65_535 + 1, 2 ** 30, *(2 ** 31 - 1 - i for i in (0, 1, 7, 100, 146, 147, 148))):
        assert r.workspace_bytes(t) == need(t), t
        assert route(r, tokens=t, start=P, slots=P, ws=P, ws_bytes=need(t) - 1) == BAD


@pytest.mark.parametrize("other", ["lens", "seen", "rows"])
def test_new_lengths_apart_from_what_is_read(built_lib, other):
    """A sequence's new length is written while its other heads still read the old ones."""
    c = M.CacheEviction(2, 4, 100, 50, 16, 16, device=NOWHERE)
    ok = dict(batch=3, lens=4 * P, seen=5 * P, rows=6 * P, acc=P, pos=P, keys=P, values=P, out_lens=2 * P, weights=P,
              queries=1, ws=P, ws_bytes=1 << 30)
    for at in (2 * P - 8, 2 * P, 2 * P + 8):
        assert "out_lens" in reasons(built_lib, c.evict_device, **{**ok, other: at})
    for at in (2 * P - 12, 2 * P + 12):         # next to it
        assert "device" in reasons(built_lib, c.evict_device, **{**ok, other: at})


def test_more_rows_of_weights_than_the_kernels_count(built_lib):
    """Row numbers stay below 2^31 in steps past the last row too."""
    for group, queries, fits in [(1, 2 ** 30, True), (4, 2 ** 28, True), (1, 2 ** 30 + 1, False), (1, 2 ** 31 - 1, False),
                                 (3, (2 ** 31 - 1) // 3, False), (2 ** 31 - 1, 1, False)]:
        c = M.CacheEviction(1, group, 100, 50, 16, 16, device=NOWHERE)
        # (strides of 0: all rows are one)
        why = reasons(built_lib, c.evict_device, 1, P, P, P, P, P, P, 2 * P, weights=P, queries=queries,
                      weight_stride=(0, 0, 0), ws=P, ws_bytes=1 << 30)
        assert ("device" if fits else "queries") in why
