"""CPU: the device code of the transformer-layer operators as the Makefile builds it."""
import os
import re
import shutil

import pytest

from tests.test_build_flags import CSRC, _compile_to_asm


def _sources():
    mk = open(os.path.join(CSRC, "Makefile")).read()
    return re.search(r"^LAYER_SRCS\s*:=\s*(.+)$", mk, re.M).group(1).split()


@pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"), reason="hipcc not installed")
@pytest.mark.parametrize("src", _sources())
def test_no_packed_fp32_instructions(src, tmp_path):
    asm = _compile_to_asm(os.path.join(CSRC, src), tmp_path / (src + ".s"))
    assert "gfx950" in asm
    hits = re.findall(r"v_pk_(?:add|mul|fma)_f32", asm)
    assert not hits, "%d packed-fp32 instructions in %s" % (len(hits), src)
