"""Rules that the attention kernels' inline assembly keeps, looked up in the
source: what the compiler is not told, no test of results shows reliably."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sym_amd", "csrc")


def statements():
    """(file, text) of every asm statement."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip"))):
        text = open(path).read()
        for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(", text):
            depth, i, quoted = 1, m.end(), False
            while depth:
                c = text[i]
                if c == '"' and text[i - 1] != "\\":
                    quoted = not quoted
                elif not quoted:
                    depth += (c == "(") - (c == ")")
                i += 1
            yield os.path.basename(path), text[m.start():i]


def test_what_assembly_writes_is_named():
    writes = [(f, s) for f, s in statements() if re.search(r"s_mov_b32 m0\b", s)]
    assert len(writes) >= 3
    for f, s in writes:
        assert '"m0"' in s.split(":")[-1], (f, s)


def test_a_bare_barrier_waits_for_shared_memory():
    """A wave that passes it may have its loads take the place of what another reads."""
    found = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "k_attend*")) + glob.glob(os.path.join(CSRC, "k_rotate*"))):
        text = open(path).read()
        for m in re.finditer(r"__builtin_amdgcn_s_barrier\(\)", text):
            found += 1
            before = text[text.rindex("{", 0, m.start()):m.start()]
            assert "shared_done();" in before or "lgkmcnt(0)" in before, path
    assert found >= 1
