"""CPU: registers and LDS of the paged-cache operators' kernels, from the built code objects: those
whose time is latency or one pass over memory spill nothing, and as many blocks of the 4-bit walk
fit a CU's LDS as its grid counts on."""
import re

import pytest

from test_kernel_resources import kernels  # noqa: F401  (the fixture)


@pytest.mark.parametrize("name", ["int4_gather_kernel", "int4_join_kernel", "kv_append_pair_kernel", "packed_f32_combine_kernel",
                                  r"kv_append_kernelILi\dELi\dELb1E", "kv_append_kernelILi0E",
                                  r"prefill_kernelILi\d+ELi\d+ELb\dELb\dENS_10PackedArgs"])
def test_no_spills(kernels, name):  # noqa: F811
    mine = {n: k[".vgpr_spill_count"] for n, k in kernels.items() if re.search(name, n)}
    assert mine
    assert not {n: v for n, v in mine.items() if v}


def test_blocks_of_the_4_bit_walk_fit_a_cu(kernels):  # noqa: F811
    seen = 0
    for n, k in kernels.items():
        m = re.search(r"int4_walk_kernelILi\dELi(\d+)ELi(\d)E", n)
        if not m:
            continue
        seen += 1
        dim, groups = map(int, m.groups())
        blocks = 1 if dim > 128 else 3 if groups == 1 or dim == 64 else 2
        lds = -(-k[".group_segment_fixed_size"] // 1280) * 1280   # what a block is given
        assert blocks * lds <= 160 * 1024, n
        # four waves a block, one on each SIMD of 512 registers a lane
        assert blocks * (-(-k[".vgpr_count"] // 8) * 8) <= 512, n
    assert seen == 16
