"""What the compiler makes of the adapters' kernels: matrix instructions do not look at EXEC, so none may stand where lanes are masked off."""
import os
import re
import subprocess

import pytest

from rwkvstic_amd import build as B


def test_no_matrix_instruction_behind_a_mask(tmp_path):
    if not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("no hipcc")
    out = str(tmp_path / "lora.s")
    flags = [f for f in B.FLAGS if f not in ("-fPIC", "-shared")]
    subprocess.run([B.hipcc(), *flags, "--cuda-device-only", "-S", "-o", out, os.path.join(B.CSRC, "rwkv_lora.hip")], check=True, stderr=subprocess.DEVNULL)
    kernel, masked, found, matrix = None, False, set(), 0
    for line in open(out):
        start = re.match(r"(_Z\w+):", line)
        if start:
            kernel, masked = start[1], False
        words = re.split(r"[\s,]+", line.split(";")[0].strip())
        if kernel is None or not words[0] or words[0].startswith("."):
            continue
        to_exec = len(words) > 1 and words[1] == "exec"
        if re.match(r"s_(and|andn2|xor)_saveexec", words[0]) or (to_exec and re.match(r"s_(and|andn2|xor)_b64$", words[0])):
            masked = True
        elif to_exec and words[0] in ("s_or_b64", "s_mov_b64") or words[0].startswith("s_or_saveexec"):
            masked = False
        elif words[0].startswith("v_mfma"):
            matrix += 1
            if masked:
                found.add(kernel)
    assert matrix > 0 and not found, sorted(found)
