"""The tile kernels of the weight product issue their LDS reads from assembly, like the GEMM kernels: the same walk over their
compiled form finds no register that is touched while a read into it is in flight, and nothing is spilled inside the loop.
Needs hipcc, no GPU."""
import os
import re
import shutil
import subprocess

import pytest

from dion_amd import _build
from test_isa_inflight_registers import walk


@pytest.mark.skipif(shutil.which("hipcc") is None, reason="hipcc not on PATH")
def test_tile_kernels_keep_their_reads_apart(tmp_path):
    out = tmp_path / "linear.s"
    cmd = ["hipcc", *[f for f in _build.HIPCC_FLAGS if f != "-fPIC"], "-S", "--cuda-device-only",
           os.path.join(_build.CSRC, "linear.hip"), "-o", str(out)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=900)
    text = out.read_text().split("\n")
    starts = [i for i, line in enumerate(text) if re.match(r"_ZN4dion\d+lin_tile_kernel\S*:", line)]
    assert len(starts) == 48
    transposing = 0
    for i in starts:
        body = text[i + 1:next(j for j in range(i, len(text)) if "s_endpgm" in text[j]) + 1]
        n_reads, hazards = walk(body)
        assert n_reads > 0 and not hazards, (text[i], hazards[:5])
        transposing += any("ds_read_b64_tr" in line for line in body)
        mfma = [j for j, line in enumerate(body) if "v_mfma" in line]
        loop = body[mfma[0]:mfma[-1] + 1]
        assert not [line for line in loop if "scratch_" in line or "s_load" in line], text[i]
    assert transposing == 12
