"""Sizes at the ends of the stated ranges, and arguments that share memory, without a
device: workspaces that grow with the work, and refusals before anything is enqueued."""
import pytest

import mflat_b200 as M
from test_select_ops_args import BAD, P, route, status


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
