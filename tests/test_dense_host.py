"""The host's half of the operators of a layer's dense half, without a GPU."""
import glob
import os
import re

import pytest

from apt_b200 import _lib

lib = _lib.lib
TYPES = {_lib.F32: 4, _lib.BF16: 2, _lib.F16: 2}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,out_dim,groups", [(20000, 8192, 8192, 1), (66000, 4096, 4096, 3), (1_060_000, 1024, 1024, 4), (500_000, 1000, 264, 4096), (1, 8, 8, 1)])
def test_a_grouped_product_takes_a_bounded_workspace(rows, dim, out_dim, groups, dtype):
    """Three tiles of sums a block at most, and the plan; rows of whole 16-byte slices are not copied."""
    tile = 128 * (128 if dtype == _lib.F32 else 256) * 4
    for backward in (0, 1):
        assert lib.apt_grouped_linear_workspace_bytes(dtype, rows, dim, out_dim, groups, backward) <= 148 * (3 * tile + 2048) + 4096


def test_what_a_device_is_told_is_told_to_every_device():
    """A kernel's shared memory is a setting of the device: asked for once a process, it fails on the second GPU, and an error stays for good."""
    sources = glob.glob(os.path.join(os.path.dirname(_lib.__file__), "csrc", "*.cu*"))
    calls = [(os.path.basename(f), text[max(0, m.start() - 200):m.start()]) for f in sources for text in [open(f).read()]
             for m in re.finditer(r"cudaFuncSetAttribute\(", text)]
    assert len(calls) >= 4
    for name, before in calls:
        assert re.search(r"!\w+\[dev\]\)", before), name
