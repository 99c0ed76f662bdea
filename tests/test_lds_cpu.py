"""Shared memory as the sources declare it."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda_gpt2_inference_amd", "csrc")
SINGLY = {"pages.hip", "kvattn.hip"}     # read and written an element at a time


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.hip"))), ids=os.path.basename)
def test_arrays_of_dynamic_size_are_aligned_for_16_bytes(path):
    """What is read 16 bytes at a time begins on such a boundary, whatever static arrays lie before it."""
    with open(path) as f:
        found = re.findall(r"extern __shared__ ([^;]*?)\w+\[\];", f.read())
    for declared in found:
        assert os.path.basename(path) in SINGLY or "__align__(16)" in declared or declared.strip() in ("uint4", "U32x4"), declared
