"""The error word's codes: what a kernel whose wait gave up leaves there is none of the codes of a batch that contradicts
itself, so a report names what happened."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quixicore-cpu_b200", "csrc")


def test_stalls_and_batches_have_codes_of_their_own():
    stalls, named, first = set(), {}, []
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith((".cu", ".cuh")):
            continue
        with open(os.path.join(CSRC, name)) as f:
            text = f.read()
        stalls |= {int(n) for n in re.findall(r"report_error\([^;]*?,\s*(\d+)\)", text)}
        stalls |= {int(n) for n in re.findall(r"\b(?:role|gave_up) = (\d+);", text)}
        first += re.findall(r"kErrorFirstBatch = (\d+);", text)
        named.update(re.findall(r"constexpr int (kError(?:Sequence|Block)) = ([^;]+);", text))
    assert {1, 11, 16, 41, 44, 61, 66} <= stalls and len(first) == 1
    codes = {eval(v.replace("sm100::", ""), {"kErrorFirstBatch": int(first[0])}) for v in named.values()}
    assert len(codes) == 2 and min(codes) == int(first[0]) > max(stalls)
