"""Cuts between groups whose sums are a few fp32 roundings apart."""
import numpy as np
import pytest
import torch

import select_ref as R
from test_gpu_route import check, gen, run

pytestmark = pytest.mark.gpu


def near(t, size, seed):
    """Two groups a token: the first two experts' scores lie within 5e-8 of 1/2, which is
    half a step at 2^23, so that s + 2^23, and then the sum of two, round up or down by
    half a step each on differences that fp32 scores miss."""
    g = gen(("cuts", size, seed))
    x = torch.full((t, 2 * size), -3.0)
    for group in range(2):
        x[:, group * size:group * size + 2] = 2e-7 * (2 * torch.rand(t, 2, generator=g) - 1)
    bias = torch.full((2 * size,), -1.0)
    bias[0] = bias[size] = 2.0 ** 23
    bias[1] = bias[size + 1] = 0.0
    return x, bias


@pytest.mark.parametrize("size", [2, 3, 4, 16, 20, 32])
def test_group_sums_round_once_more(size):
    """Sums of two large scores: each term is rounded, and their sum."""
    x, bias = near(20_000, size, 0)
    s = 1 / (1 + np.exp(-x.double().numpy()))
    sums = s[:, [0, size]] + s[:, [1, size + 1]]
    clear = np.abs(sums[:, 0] - sums[:, 1]) > 1e-8         # (2^23 + s has steps of 1.9e-9 in 64 bits)
    x = x[torch.from_numpy(clear)]
    ids, _, _, _ = run(x.cuda(), 2, "sigmoid", bias.cuda(), groups=2, kept=1, top=2)
    first = np.where(sums[clear, 0] > sums[clear, 1], 0, size)
    np.testing.assert_array_equal(np.sort(ids, 1), np.stack([first, first + 1], 1))


@pytest.mark.parametrize("scale", [1.0, 100.0])
@pytest.mark.parametrize("n,groups", [(64, 8), (60, 5), (256, 8)])
def test_group_sums_a_few_roundings_apart(scale, n, groups):
    """Biases that bring every group's two best to the same sum, up to their roundings."""
    g = gen(("sums", scale, n, groups))
    x = torch.randn(1, n, generator=g).expand(300, n).clone()
    x += 2e-7 * torch.randn(300, n, generator=g)
    _, s = R.scores(x[0].double().numpy(), "sigmoid")
    bias = torch.from_numpy(scale * 0.75 - s).float()
    check(x.cuda(), 6, "sigmoid", bias.cuda(), groups=groups, kept=groups // 2, top=2)
