"""What the token operators' kernels load back from the stack, by ptxas' report of the last build: no more than it is now."""
import re

import pytest

from d2conv3d_b200 import build

# bytes a thread loads back at most.  What spills: the forward with two parts of 128 channels (scores, weights and their rests at a time);
# layer norm of 32 channels a thread one at a time (rows) or in pairs of positions (volumes); otherwise a handful of set-up values
MOST = {"fwd_tc_kernel": (8, 456), "bwd_tc_kernel": (16, 160), "few_kernel": (36, 0), "fwd_kernel": (9, 0), "bwd_q_kernel": (9, 88),
        "bwd_kv_kernel": (9, 24), "combine_kernel": (6, 0), "norm_rows_fwd_kernel": (36, 0), "norm_rows_bwd_kernel": (36, 392),
        "norm_volume_kernel": (120, 252), "rotary_kernel": (18, 60)}


@pytest.mark.parametrize("kernel", MOST)
def test_spills_stay_small(kernel):
    variants, most = MOST[kernel]
    found = {name: r for name, r in build.ptxas_report().items() if re.search(rf"\d{kernel}I", name)}
    if not found:
        pytest.skip("the library was not built here")
    assert len(found) == variants, sorted(found)
    assert all(loads <= most for _, _, _, loads in found.values()), {n: r for n, r in found.items() if r[3] > most}


def test_only_the_widest_forward_spills_its_tiles():
    found = {name: r[3] for name, r in build.ptxas_report().items() if "fwd_tc_kernel" in name}
    if not found:
        pytest.skip("the library was not built here")
    assert sum(loads > 104 for loads in found.values()) <= 1, found
