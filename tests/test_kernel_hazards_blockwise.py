"""The products with block scales are built from hand-written matrix instructions, whose wait states the compiler does not insert.  These
tests compile their units to assembly (no GPU needed) and check on what was emitted: the distance of accumulator reads, that nothing
writes an operand or a scale just before the instruction that reads it, M0 before every load into LDS, and that nothing spills.
"""
import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from float8_experimental_amd import _build

LARGE = ["f8mi_block_gemm_large.hip", "f8mi_block_gemm_large_odd.hip", "f8mi_block_gemm_large_tr.hip"]
MID = ["f8mi_block_gemm.hip"]
OTHERS = ["f8mi_block_gemm_few.hip", "f8mi_block_cast.hip", "f8mi_layer_norm.hip", "f8mi_grad_clip.hip"]
MIN_MFMAS = 8         # MFMAs issued after the one that writes an accumulator, before it is read ...
MIN_WAIT_STATES = 18  # ... or this many wait states
VALU_TO_MFMA = 2      # wait states between a vector instruction and the MFMA that reads its result


def _asm(unit, out_dir):
    out = os.path.join(out_dir, unit[:-4] + ".s")
    subprocess.run([_build.HIPCC, *_build.FLAGS, "--cuda-device-only", "-S", os.path.join(_build.CSRC, unit), "-o", out], check=True, stderr=subprocess.DEVNULL)
    with open(out) as f:
        return f.read()


@pytest.fixture(scope="module")
def listings(tmp_path_factory):
    d = str(tmp_path_factory.mktemp("asm"))
    units = LARGE + MID + OTHERS
    with ThreadPoolExecutor(max_workers=4) as ex:
        return dict(zip(units, ex.map(lambda u: _asm(u, d), units)))


def _code(text):
    lines = [line.strip() for line in text.split("\n")]
    return [line for line in lines if line and not line.startswith((";", ".", "//")) and not line.endswith(":")]


def _kernels(text):
    return [part for part in re.split(r"\.Lfunc_end\d+:", text) if "s_endpgm" in part]


def _vgprs(operand):
    m = re.match(r"v\[(\d+):(\d+)\]", operand) or re.match(r"v(\d+)()$", operand)
    return set() if m is None else set(range(int(m.group(1)), int(m.group(2) or m.group(1)) + 1))


def _nops(line):
    m = re.match(r"s_nop (\d+)", line)
    return 0 if m is None else int(m.group(1)) + 1


def test_the_parsing_sees_hazards():
    """A planted listing of each kind is told from a sound one."""
    mfma = "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[0:7], v[8:15], a[0:3], v20, v21 op_sel_hi:[0,0,0]"
    assert _early_operands(["v_lshrrev_b32 v20, 8, v30", "s_nop 0", mfma]) and not _early_operands(["v_lshrrev_b32 v20, 8, v30", "s_nop 1", mfma])
    assert _early_operands(["v_mov_b32 v3, v1", mfma]) and not _early_operands(["v_mov_b32 v31, v1", mfma])
    assert _early_reads([mfma, "s_nop 3", "v_accvgpr_read_b32 v1, a2"]) and not _early_reads([mfma, "s_nop 15", "s_nop 1", "v_accvgpr_read_b32 v1, a2"])


def _early_operands(code):
    bad = []
    for i, line in enumerate(code):
        if not line.startswith("v_mfma"):
            continue
        uses = set().union(*(_vgprs(t.strip().split()[0]) for t in line.split(None, 1)[1].split(",")[1:]))
        states = 0
        for before in reversed(code[max(0, i - 4):i]):
            if states >= VALU_TO_MFMA:
                break
            if before.startswith("v_") and not before.startswith("v_mfma") and _vgprs(before.split(None, 1)[1].split(",")[0].strip()) & uses:
                bad.append((before, line))
            states += _nops(before) or 1
    return bad


def _early_reads(code):
    bad, written, n = [], {}, 0
    for i, line in enumerate(code):
        m = re.match(r"v_mfma_\S+ a\[(\d+):(\d+)\]", line)
        if m:
            n += 1
            written.update({r: (n, i) for r in range(int(m.group(1)), int(m.group(2)) + 1)})
            continue
        m = re.match(r"v_accvgpr_read_b32 v\d+, a(\d+)", line)
        if m:
            at, where = written[int(m.group(1))]
            if n - at < MIN_MFMAS and sum(map(_nops, code[where + 1:i])) < MIN_WAIT_STATES:
                bad.append(line)
    return bad


@pytest.mark.parametrize("unit", LARGE)
def test_large_tiles_read_accumulators_late_and_keep_them_in_place(listings, unit):
    kernels = _kernels(listings[unit])
    assert len(kernels) >= 4
    for kernel in kernels:
        code = _code(kernel)
        assert sum(line.startswith("v_accvgpr_read") for line in code) == 256 and not any(line.startswith(("v_accvgpr_write", "v_accvgpr_mov")) for line in code)
        assert sum(line.startswith("v_mfma_scale") for line in code) == sum(line.startswith("v_mfma") for line in code) > 64 * 2
        assert not _early_reads(code)


@pytest.mark.parametrize("unit", LARGE + MID + ["f8mi_block_gemm_few.hip"])
def test_no_vector_instruction_writes_an_operand_or_a_scale_just_before_its_mfma(listings, unit):
    code = _code(listings[unit])
    assert sum(line.startswith("v_mfma_scale") for line in code) > 0
    assert not _early_operands(code)


@pytest.mark.parametrize("unit", LARGE + MID)
def test_every_load_into_lds_sets_m0_with_the_wait_state_it_needs(listings, unit):
    code, n = _code(listings[unit]), 0
    for i, line in enumerate(code):
        if line.startswith("global_load_lds_"):
            n += 1
            assert code[i - 1].startswith("s_nop") and code[i - 2].startswith("s_mov_b32 m0,"), code[i - 2:i + 1]
    assert n >= len(_kernels(listings[unit])) * 16


@pytest.mark.parametrize("unit", LARGE + MID + OTHERS)
def test_nothing_spills(listings, unit):
    """But for the widest rows of layer norm's backward pass, whose column sums leave few registers: some addresses, once a row."""
    sizes = dict(re.findall(r"\.amdhsa_kernel (\S+).*?_private_segment_fixed_size (\d+)", listings[unit], re.S))
    spilled = {name: int(size) for name, size in sizes.items() if int(size)}
    assert sizes and all("layer_norm_backward_kernel" in name and "Li1024E" in name and size <= 96 for name, size in spilled.items()), spilled


@pytest.mark.parametrize("unit", LARGE + MID + OTHERS)
def test_no_packed_fp32_arithmetic(listings, unit):
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", listings[unit])
