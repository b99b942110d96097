"""Barriers in shared memory are laid out one array behind another; each is initialised once, over its own length."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "gemma4-webgpu_b200" / "csrc"
DECL = re.compile(r"uint64_t\* (\w+) = (\w+)(?: \+ ([\w:]+))?;")
LOOP = re.compile(r"for \(int (\w+) = 0; \1 < ([\w:]+); \1\+\+\) (\{.*?\n    \}|[^;]*;)", re.S)


def _lengths(text):
    """Length of every array in a chain that starts at `bars`, by what the next one adds to it; the last one has none."""
    out, chain = {}, {"bars"}
    for name, of, n in DECL.findall(text):
        if of in chain:
            chain.add(name)
            if n is not None and of != "bars":
                out[of] = n.replace("C::", "") if n else None
    return out


@pytest.mark.parametrize("name", ["g4a_chunk_tc.cu", "g4a_mass.cu"])
def test_barriers_are_initialised_over_their_own_length(name):
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    lengths = _lengths(text)
    assert len(lengths) > 8
    seen = {}
    for var, n, body in LOOP.findall(text):
        for array in re.findall(r"mbar_init\(&(\w+)\[" + var + r"\]", body):
            seen.setdefault(array, []).append(n.replace("C::", ""))
    single = re.findall(r"mbar_init\((\w+),", text)
    pairs = re.findall(r"mbar_init\(&(\w+)\[(\d)\]", text)
    for array, n in lengths.items():
        if array in seen:
            assert seen[array] == [n], (array, seen[array], n)
        elif n == "1":
            assert single.count(array) == 1, array
        else:
            assert [i for a, i in pairs if a == array] == [str(i) for i in range(int(n))], array
