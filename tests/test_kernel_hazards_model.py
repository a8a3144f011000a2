"""What the compiler made of the kernels of RMS norm, dropout and the adapters: no packed fp32 arithmetic, nothing that spills but for the widest rows of the norm's backward pass (no GPU needed)."""
import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from float8_experimental_amd import _build

UNITS = ["f8mi_rms_norm.hip", "f8mi_dropout.hip", "f8mi_adapter_rows.hip", "f8mi_adapters.hip"]


@pytest.fixture(scope="module")
def listings(tmp_path_factory):
    d = str(tmp_path_factory.mktemp("asm"))

    def asm(unit):
        out = os.path.join(d, unit[:-4] + ".s")
        subprocess.run([_build.HIPCC, *_build.FLAGS, "--cuda-device-only", "-S", os.path.join(_build.CSRC, unit), "-o", out], check=True, stderr=subprocess.DEVNULL)
        with open(out) as f:
            return f.read()

    with ThreadPoolExecutor(max_workers=4) as ex:
        return dict(zip(UNITS, ex.map(asm, UNITS)))


@pytest.mark.parametrize("unit", UNITS)
def test_nothing_spills(listings, unit):
    """But rows of three pieces a lane and more, backward: 1024 lanes leave each of them 128 registers, and the addresses of a row go."""
    sizes = dict(re.findall(r"\.amdhsa_kernel (\S+).*?_private_segment_fixed_size (\d+)", listings[unit], re.S))
    spilled = {name: int(size) for name, size in sizes.items() if int(size)}
    assert sizes and all(re.search(r"rms_norm_backward_kernelILi\dELi\dELi1024ELi[345]E", name) and size <= 128 for name, size in spilled.items()), spilled


@pytest.mark.parametrize("unit", UNITS)
def test_no_packed_fp32_arithmetic(listings, unit):
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", listings[unit])


def test_products_run_on_the_matrix_cores(listings):
    text = listings["f8mi_adapters.hip"]
    for instruction in ("v_mfma_f32_16x16x32_bf16", "v_mfma_f32_16x16x32_f16", "v_mfma_f32_16x16x4_f32", "ds_read_b64_tr_b16"):
        assert instruction in text
