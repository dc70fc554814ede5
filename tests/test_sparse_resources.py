"""Scratch budget of the sparse layer's and Newton-Schulz kernels, read from the
compiled code objects (CPU only): an accumulator that leaves the registers
keeps its values and costs several times the kernel's time."""
import os
import shutil
from concurrent.futures import ThreadPoolExecutor

import pytest

from neuralscript_amd import build
from test_kernel_resources import _kernel_metadata

SOURCES = {"moe_topk.hip": ("route_row_kernel", "route_grad_row_kernel", "few_kernel", "few_outer_kernel"),
           "moe_small.hip": ("small_kernel",), "moe_split.hip": ("split_kernel",),
           "newton.hip": ("ns_gemm_kernel", "ns_mid_kernel", "ns_few_kernel", "ns_fused_kernel")}

pytestmark = pytest.mark.skipif(shutil.which("hipcc") is None, reason="hipcc not installed")


def test_sparse_kernels_use_no_scratch(tmp_path):
    with ThreadPoolExecutor(max_workers=3) as ex:
        rows = dict(zip(SOURCES, ex.map(lambda s: _kernel_metadata(os.path.join(build.CSRC, s), str(tmp_path)), SOURCES)))
    for src, names in SOURCES.items():
        for want in names:
            assert any(want in name for name, _, _ in rows[src]), want
        bad = [(name, scratch) for name, scratch, _ in rows[src] if scratch > 0]
        assert not bad, f"{src}: kernels with a private (scratch) segment: {bad}"
