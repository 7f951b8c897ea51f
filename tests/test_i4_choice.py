"""Host tests of the rule that names a 4-bit product's kernel: the sizes that the GPU
tests run are held to the kernels they are meant for, and no kernel that the rule can
name is without a size (cuda-zkml_amd/csrc/i4_matmul.hip: choose_i4)."""
import numpy as np
import pytest

import zkml_amd as z
from i4_sizes import GROUPED, PLAIN, listed


def kernel(rows, n_out, n_in, experts=0, group=128, pad=0, address=0):
    name = z.lib().zk_debug_i4_kernel(rows, n_out, n_in, n_in + pad, address, group, experts)
    return name and name.decode()


@pytest.mark.parametrize("name,rows,n_out,n_in", listed(PLAIN))
def test_plain_sizes_reach_their_kernel(name, rows, n_out, n_in):
    assert kernel(rows, n_out, n_in) == name


@pytest.mark.parametrize("name,rows,n_out,n_in,experts", listed(GROUPED))
def test_grouped_sizes_reach_their_kernel(name, rows, n_out, n_in, experts):
    assert kernel(rows, n_out, n_in, experts) == name


@pytest.mark.parametrize("grouped,sizes", [(False, PLAIN), (True, GROUPED)])
def test_every_kernel_has_a_size(grouped, sizes):
    rng = np.random.default_rng(1)
    named = set()
    for _ in range(20000):
        rows, n_out, n_in = (int(2 ** rng.uniform(0, 14)) for _ in range(3))
        experts = int(2 ** rng.uniform(0, 9)) if grouped else 0
        named.add(kernel(rows, n_out, n_in // 16 * 16 if rng.random() < 0.5 else n_in, experts,
                         int(rng.choice([32, 64, 128, 256])), int(rng.integers(0, 17)), int(rng.integers(0, 16))))
    assert named == set(sizes)


def test_odd_rows_leave_the_largest_tiles():
    assert kernel(2049, 7535, 672) == "stages 256x256"
    for more in (dict(pad=3), dict(address=1), dict(pad=1 << 23)):
        assert kernel(2049, 7535, 672, **more) != "stages 256x256"
    assert kernel(2049, 7535, 673) != "stages 256x256"


def test_a_launch_holds_the_tiles():
    """At most 2^22 blocks a launch: the widest layers leave the smallest tiles."""
    for n_in in (64, 4096):
        for rows in (1, 4, 5, 16):
            sizes = [int(s) for s in kernel(rows, 1 << 26, n_in).split()[-1].split("x")]
            assert -(-rows // sizes[0]) * (2**26 // sizes[1]) <= 1 << 22
    # grouped: one tile for each expert beside the whole ones
    for experts, rows, n_out in ((2, 14, 53232046), (1000, 1000, 1 << 16), (60000, 60000, 2048), (8, 64, 1 << 24)):
        sizes = [int(s) for s in kernel(rows, n_out, 11296, experts, 64).split()[-1].split("x")]
        assert (rows // sizes[0] + min(experts + 1, rows)) * -(-n_out // sizes[1]) <= 1 << 22


def test_sizes_out_of_range():
    assert kernel(1 << 31, 4, 4) is None and kernel(4, (1 << 26) + 1, 4) is None and kernel(4, 4, (1 << 24) + 1) is None
    assert kernel(4, 4, 4, experts=-1) is None and kernel(0, 4, 4) is None
