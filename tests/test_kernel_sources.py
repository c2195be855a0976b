"""The kernels' sources, read without a GPU: waits that the compiler does not
add inside an inline asm block."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "vllm-xpu-kernels_amd", "csrc")
FILES = sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.h")))


def _asm_blocks(text):
    """The instructions of every asm statement, in order."""
    for m in re.finditer(r'\basm\s*(?:volatile)?\s*\(\s*((?:"(?:[^"\\]|\\.)*"\s*)+)', text):
        body = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', m.group(1)))
        yield [i.strip() for i in re.split(r"\\n|;", body.replace("\\t", " ")) if i.strip()]


def _writes_m0(ins):
    return re.match(r"s_\w+ m0\b", ins) is not None


def _copies_to_lds(ins):
    return re.match(r"(global|buffer|scratch)_load_(lds_|.*\blds\b)", ins) is not None


@pytest.mark.parametrize("path", FILES, ids=os.path.basename)
def test_m0_is_written_one_wait_state_before_a_copy_to_lds_reads_it(path):
    """gfx9: a scalar write of M0 and a load to LDS, which takes its address from
    M0, need an instruction between them.  The compiler places it where it
    writes both, not inside an asm block."""
    with open(path) as f:
        blocks = list(_asm_blocks(f.read()))
    for b in blocks:
        for a, c in zip(b, b[1:]):
            assert not (_writes_m0(a) and _copies_to_lds(c)), f"{a} / {c}"


def test_copies_to_lds_are_found():
    """The test above reads what it means to read."""
    found = sum(_copies_to_lds(i) for p in FILES for b in _asm_blocks(open(p).read()) for i in b)
    assert found >= 12
    bad = r'asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dword %0, off" :: "v"(g));'
    (b,) = _asm_blocks(bad)
    assert _writes_m0(b[0]) and _copies_to_lds(b[1])
