"""The static checks of test_isa_hazards.py (hand-emitted MFMAs, LDS-DMA destinations) on the kernels of packed sequences and of
the paged cache."""
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
        return "\n".join(pool.map(compiled, ["flame_packed.hip", "flame_paged.hip"]))


def test_results_of_hand_emitted_mfmas(text):
    """The check goes by the names of the dense kernels and wants nine of them: the three dK/dV kernels here under such names."""
    kernels = re.findall(r"^_ZN5fattn22bwd_dkdv_packed_kernel\w+:.*?\.end_amdhsa_kernel", text, re.S | re.M)
    assert len(kernels) == 3
    hazards.test_hand_emitted_mfma_results_are_not_touched_too_early(
        "\n".join(k.replace("_ZN5fattn22bwd_dkdv_packed_kernel", "_ZN5fattn15bwd_dkdv_kernel%d" % i) for i in range(3) for k in kernels))


def test_operands_of_hand_emitted_mfmas(text):
    hazards.test_operands_of_hand_emitted_mfmas_are_not_written_just_before(text)


def test_lds_dma_destinations(text):
    hazards.test_every_lds_dma_finds_its_destination_in_m0(text)


def test_next_to_no_scratch(text):
    """Scratch memory per wavefront limits how many workgroups the device keeps resident."""
    for name in re.findall(r"^(_ZN5fattn\w*(?:packed|paged)\w*kernel\w+):", text, re.M):
        body = re.search(r"^%s:.*?\.end_amdhsa_kernel" % re.escape(name), text, re.S | re.M).group(0)
        assert int(re.search(r"\.amdhsa_private_segment_fixed_size (\d+)", body).group(1)) <= 32, name      # a few registers of a tail
