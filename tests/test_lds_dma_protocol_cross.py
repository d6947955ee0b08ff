"""The LDS-DMA protocol (M0 written by SALU one wait state before each copy, no
freshly written SGPR base) on the compiled cross attention kernels, whose
copies take their base from SGPRs."""

import re
from pathlib import Path

import pytest
from test_lds_dma_protocol import CSRC, HIPCC
from test_lds_dma_protocol import test_compiled_lds_dmas_follow_the_protocol as check

pytestmark = pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not available")


@pytest.mark.parametrize("stem", ["cross_attention", "cross_attention_bwd"])
def test_cross_attention_lds_dmas_follow_the_protocol(stem, tmp_path):
    check(stem, tmp_path)


def test_cross_attention_copies_wait_five_states():
    text = (CSRC / "cross_attention.h").read_text()
    asm = re.findall(r'asm\s+volatile\s*\(\s*"([^"]*)"', text)
    assert [a for a in asm if a] == [r"s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1"]
