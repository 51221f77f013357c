"""Registers of the kernels that are bound by them: none of the products in 8 bits keeps any of its values in memory."""
import os
import re
import subprocess

import pytest

from fgms_amd import build


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="needs hipcc")
def test_products_in_eight_bits_stay_in_registers(tmp_path):
    listing = tmp_path / "int8.lst"
    subprocess.run([build.HIPCC] + build.HIP_FLAGS + ["--cuda-device-only", "-S", os.path.join(build.CSRC, "fgms_int8_linear.hip"), "-o", str(listing)],
                   check=True, capture_output=True)
    text = listing.read_text()
    kernels = re.findall(r"\.amdhsa_kernel (\S+)", text)
    scratch = [int(n) for n in re.findall(r"\.amdhsa_private_segment_fixed_size (\d+)", text)]
    assert len(kernels) == len(scratch) >= 24
    assert not any(scratch), dict(zip(kernels, scratch))
