"""GPU tests of the routed experts (cuda-zkml_amd/csrc/experts.hip) at sizes where
other kernels, or more blocks, take part than at small ones: sorts up to the most
pairs there may be, rows that pass the caches."""
import numpy as np
import pytest

import zkml_amd as z
from test_gpu_experts import expected, say, sort

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return z.Context(0)


@pytest.mark.parametrize("pairs,experts", [(1 << 20, 1024), ((1 << 22) - 1, 8), (1 << 22, 1), (1 << 22, 1024)])
def test_sort_of_many_pairs(ctx, pairs, experts):
    rng = np.random.default_rng([pairs, experts])
    e = rng.integers(0, experts, pairs)
    e[rng.random(pairs) < 0.1] = -1
    say("[experts sort]", pairs, experts)
    for got, want in zip(sort(ctx, e, experts), expected(e, experts)):
        assert np.array_equal(got, want)


@pytest.mark.parametrize("pairs", [640, 8192, 30000])
@pytest.mark.parametrize("each", [1, 2, 31, 63, 64, 65, 200])
def test_sort_of_neighbours_with_the_same_expert(ctx, pairs, each):
    """The running counts of a wave: 64 pairs at a time share a count, take one each,
    or anything between, and the next 64 go on from there."""
    e = np.arange(pairs) // each % 7
    e[::11] = 3
    say("[experts sort]", pairs, each)
    for got, want in zip(sort(ctx, e, 7), expected(e, 7)):
        assert np.array_equal(got, want)
