"""The tile kernels of the gated projections, like those of the weight product: no register is touched while an LDS read into it is in
flight, and nothing is spilled, in the loop or around it.  The norm kernels of up to 8192 columns keep their rows in
registers.  Needs hipcc, no GPU."""
import os
import re
import shutil
import subprocess

import pytest

from dion_amd import _build
from test_isa_inflight_registers import walk

NEEDS_HIPCC = pytest.mark.skipif(shutil.which("hipcc") is None, reason="hipcc not on PATH")


def assembly(source, tmp_path):
    out = tmp_path / (source + ".s")
    cmd = ["hipcc", *[f for f in _build.HIPCC_FLAGS if f != "-fPIC"], "-S", "--cuda-device-only", os.path.join(_build.CSRC, source), "-o",
           str(out), "-Rpass-analysis=kernel-resource-usage"]
    usage = subprocess.run(cmd, check=True, capture_output=True, text=True, timeout=900).stderr
    scratch, name = {}, None
    for line in usage.split("\n"):
        m = re.search(r"Function Name: (\S+)", line)
        name = m.group(1) if m else name
        m = re.search(r"ScratchSize \[bytes/lane\]: (\d+)", line)
        if m:
            scratch[name] = int(m.group(1))
    return out.read_text().split("\n"), scratch


@NEEDS_HIPCC
def test_tile_kernels_keep_their_reads_apart(tmp_path):
    text, scratch = assembly("gated.hip", tmp_path)
    starts = [i for i, line in enumerate(text) if re.match(r"_ZN4dion\d+lin_tile_kernel\S*:", line)]
    assert len(starts) == 63
    transposing = 0
    for i in starts:
        if re.search(r"E(Lb[01]E){2}Li[1245]E", text[i]):  # (the gelu's has the most registers in use: the others' loops are its)
            continue
        body = text[i + 1:next(j for j in range(i, len(text)) if "s_endpgm" in text[j]) + 1]
        n_reads, hazards = walk(body)
        assert n_reads > 0 and not hazards, (text[i], hazards[:5])
        transposing += any("ds_read_b64_tr" in line for line in body)
        mfma = [j for j, line in enumerate(body) if "v_mfma" in line]
        assert not [line for line in body[mfma[0]:mfma[-1] + 1] if "scratch_" in line or "s_load" in line], text[i]
    assert transposing == 6
    assert not {k: v for k, v in scratch.items() if v > 0}


@NEEDS_HIPCC
def test_rows_of_layer_norm_stay_in_registers(tmp_path):
    _text, scratch = assembly("layer_norm.hip", tmp_path)
    held = {k: v for k, v in scratch.items() if "norm_forward_kernel" in k or re.search(r"norm_backward_kernelI..Li\d+ELi8E", k)}
    assert len(held) >= 120 and not {k: v for k, v in held.items() if v > 0}
