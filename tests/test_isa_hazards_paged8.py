"""The static checks of test_isa_hazards.py (LDS-DMA destinations, scratch memory) on the kernels of the paged cache in 8 bits and of the rotary
positions."""
import os
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from flame_amd import build as fb
from tests import test_isa_hazards as hazards


@pytest.fixture(scope="module")
def text(tmp_path_factory):
    if shutil.which(fb.HIPCC) is None and not os.path.exists(fb.HIPCC):
        pytest.skip("hipcc not available")
    tmp = tmp_path_factory.mktemp("isa")
    flags = [f for f in fb.FLAGS if f not in ("-shared", "-fPIC")]

    def compiled(name):
        out = tmp / (name + ".s")
        subprocess.run([fb.HIPCC, *flags, "-S", "--cuda-device-only", os.path.join(fb.CSRC, name), "-o", str(out)], check=True, stdout=subprocess.DEVNULL,
                       stderr=subprocess.DEVNULL)
        return out.read_text()

    with ThreadPoolExecutor(2) as pool:
        return "\n".join(pool.map(compiled, ["flame_paged8.hip", "flame_rotary.hip"]))


def test_lds_dma_destinations(text):
    hazards.test_every_lds_dma_finds_its_destination_in_m0(text)


def test_no_scratch_and_no_packed_fp32(text):
    kernels = re.findall(r"^(_ZN5fattn\w*kernel\w+):.*?\.amdhsa_private_segment_fixed_size (\d+)", text, re.S | re.M)
    assert len(kernels) >= 40
    for name, bytes_ in kernels:
        assert int(bytes_) == 0, name
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)
