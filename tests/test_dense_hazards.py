"""The order of inline-asm MFMA statements in the compiled dense attention over cached rows (see test_attention_hazards)."""
import os
import re
import subprocess

import pytest

from arcagi2_flashnext_dots3_amd import build
from tests.test_attention_hazards import branch_hazards, hazards


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="no hipcc")
def test_compiled_order_of_asm_statements(tmp_path):
    out = tmp_path / "chunk.s"
    subprocess.run([build.HIPCC, *build.FLAGS, "--cuda-device-only", "-S", os.path.join(build.CSRC, "spmla_chunk.hip"), "-o", str(out)],
                   check=True, capture_output=True)
    text = out.read_text().split("\n")
    starts = [i for i, l in enumerate(text) if re.match(r"_ZN5spmla5chunk11wide_kernelI\S+:", l)]
    assert len(starts) == 4
    for s in starts:
        end = next(i for i in range(s, len(text)) if ".Lfunc_end" in text[i])
        body = text[s:end]
        assert sum("v_mfma_f32_32x32x16_" in l for l in body) == 36 + 32
        assert not hazards(body), text[s]
        assert not branch_hazards(body), text[s]
