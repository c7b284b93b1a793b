"""Buffer loads keep what their bounds check has to see where it looks."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tokenvector", "inference_amd", "csrc")
CALL = re.compile(r"\b__builtin_amdgcn_raw_\w*buffer_(?:load|store)\w*\s*\(")


def _arguments(text, at):
    """The arguments of the call whose opening bracket is before `at`."""
    depth, start, out = 1, at, []
    while depth:
        c = text[at]
        depth += (c in "([{") - (c in ")]}")
        if (c == "," and depth == 1) or depth == 0:
            out.append(text[start:at].strip())
            start = at + 1
        at += 1
    return out


def test_offsets_are_in_the_checked_operand():
    """The check of a raw buffer access against the buffer's size takes in the vector
    offset and not the scalar one, so an access that relies on it (rows past an
    operand's last) has its whole offset in the former and 0 in the latter: the last
    but two arguments."""
    calls = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip"))):
        text = open(path).read()
        for m in CALL.finditer(text):
            calls += 1
            args = _arguments(text, m.end())
            scalar = args[-3] if "lds" in m.group() else args[-2]
            assert scalar == "0", f"{os.path.basename(path)}: scalar offset {scalar}"
    assert calls >= 1
