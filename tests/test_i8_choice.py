"""Host tests of the rule that names a product's kernel: the sizes that the GPU
tests run are held to the kernels they are meant for, and no kernel that the rule
can name is without a size (cuda-zkml_amd/csrc/i8_matmul.hip: choose_kernel)."""
import numpy as np
import pytest

import zkml_amd as z
from i8_sizes import GROUPED, PLAIN, listed


def kernel(rows, n_out, n_in, experts=0, pad=0, address=0):
    name = z.lib().zk_debug_i8_kernel(rows, n_out, n_in, n_in + pad, n_in + pad, address, experts)
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
                         int(rng.integers(0, 17)), int(rng.integers(0, 16))))
    assert named <= set(sizes) and named >= {k for k in sizes if not k.startswith("ring 256")}


def test_rows_at_odd_addresses_leave_the_ring():
    assert kernel(4000, 4090, 2064).startswith("ring")
    assert kernel(4000, 4090, 2064, address=8).startswith("odd")
    assert kernel(4000, 4090, 2064, pad=4).startswith("odd")


def test_sizes_out_of_range():
    assert kernel(1 << 31, 4, 4) is None and kernel(4, 1 << 31, 4) is None and kernel(4, 4, 131072) is None
    assert kernel(4, 4, 4, experts=-1) is None
