"""The device assembly of attention_masked, rotary and linear_f16 under the scans of mfma_hazards: no MFMA
result is read through a branch sooner than the compiler pads such reads inside a block, no inline asm
reads a fresh result, and no kernel keeps arrays in scratch memory."""

import re
import shutil
from pathlib import Path

import pytest

from tests import mfma_hazards
from tessery_amd import _build

SOURCES = ("attention_masked.hip", "linear_f16.hip", "rotary.hip")

pytestmark = pytest.mark.skipif(shutil.which("hipcc") is None and
                                not Path("/opt/rocm/bin/hipcc").exists(),
                                reason="hipcc is needed to build the device assembly")


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    out = tmp_path_factory.mktemp("asm")
    return {s: mfma_hazards.device_assembly(_build.CSRC / s, out / (s + ".s")) for s in SOURCES}


def test_no_mfma_result_read_early_through_a_branch(assembly):
    rule, cross, short = mfma_hazards.scan(list(assembly.values()))
    assert "v_mfma_f32_32x32x16_f16" in rule and "v_mfma_f32_32x32x2_f32" in rule
    assert len(cross) > 50  # the scores behind the masking branch
    assert short == [], short[:5]


def test_inline_asm_reads_no_fresh_valu_result(assembly):
    assert mfma_hazards.inline_asm_hazards(list(assembly.values())) == []


def test_no_kernel_uses_scratch(assembly):
    sizes = {s: [int(n) for n in re.findall(r"^\s*\.amdhsa_private_segment_fixed_size (\d+)",
                                            assembly[s], re.M)] for s in SOURCES}
    assert {s: v for s, v in sizes.items() if any(v)} == {}
