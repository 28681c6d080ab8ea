"""What the 4-bit attention kernels keep in scratch memory, read from the library that was built here."""
import os
import re

import pytest

from tests.test_host_support import READELF, ROOT, _kernel_metadata


def test_attention_kernels_spill_at_two_blocks_of_head_dim_256_only(tmp_path):
    library = os.path.join(ROOT, "tvm_amd", "lib", "libtvmkv.so")
    if not (os.path.exists(READELF) and os.path.exists(library)):
        pytest.skip("needs the built library and llvm-readelf")
    kernels = [k for k in _kernel_metadata(library, tmp_path) if "mxfp4" in k[0]]
    assert len(kernels) == 33 + 8  # eleven pairs of head dim and row blocks, prefill and two of decode; append and read
    spills = {k[0]: k[1] for k in kernels if k[1] or k[2]}
    assert all(re.search(r"mxfp4_attn_kernelILi256ELi2E", name) for name in spills)
    assert max(spills.values(), default=0) <= 22
