"""Inline asm in the kernels names the scalar registers that it writes itself."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tokenvector", "inference_amd", "csrc")
STATEMENT = re.compile(r"\basm\s+(?:volatile\s*)?\((.*?)\);", re.S)
WRITES = re.compile(r"\bs_\w+\s+(m0|vcc|exec|s\d+|s\[\d+:\d+\])\b")


def test_written_registers_are_clobbers():
    """A fixed register that an instruction in asm writes, and the compiler may hold
    a value in, is on the statement's clobber list."""
    written = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip"))):
        for statement in STATEMENT.findall(open(path).read()):
            parts = statement.rsplit(":", 1)
            for register in WRITES.findall(parts[0]):
                written += 1
                assert f'"{register}"' in parts[-1], f"{os.path.basename(path)}: {register} in {statement[:60]}"
    assert written >= 3
