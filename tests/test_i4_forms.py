"""Host tests: the sizes of i4_forms take the kernels that they are meant for, and the
rule (cuda-zkml_amd/csrc/i4_matmul.hip: choose_i4) names no form that has none."""
import subprocess
import sys

import numpy as np
import pytest

import zkml_amd as z
from i4_forms import FORMS, GROUPS


def kernel(rows, n_out, n_in, odd, group, experts):
    name = z.lib().zk_debug_i4_kernel(rows, n_out, n_in, n_in + odd, odd, group, experts)
    return name and name.decode()


@pytest.mark.parametrize("name,odd,group,rows,n_out,n_in,experts", FORMS)
def test_sizes_reach_their_kernel(name, odd, group, rows, n_out, n_in, experts):
    assert kernel(rows, n_out, n_in, odd, group, experts) == name


def test_every_form_has_a_size():
    listed = {(name, odd, group, experts > 0) for name, odd, group, _, _, _, experts in FORMS}
    rng, named = np.random.default_rng(2), set()
    for _ in range(30000):
        rows, n_out, n_in = (int(2 ** rng.uniform(0, 13.5)) for _ in range(3))
        experts = int(2 ** rng.uniform(0, 7)) if rng.random() < 0.5 else 0
        odd = int(rng.integers(0, 2))
        if not odd:
            n_in = max(16, n_in // 16 * 16)
        named |= {(kernel(rows, n_out, n_in, odd, g, experts), odd, g, experts > 0) for g in GROUPS}
    assert named <= listed


def test_groups_out_of_range():
    """A group that no product takes has no kernel, and ends no process."""
    code = ("import sys; sys.path[:0] = sys.argv[1:]; import zkml_amd as z; "
            "assert all(z.lib().zk_debug_i4_kernel(4, 4, 64, 64, 0, g, e) is None "
            "for g in (0, -1, -128, 1, 96, 129) for e in (0, 3))")
    assert subprocess.run([sys.executable, "-c", code, *sys.path]).returncode == 0
