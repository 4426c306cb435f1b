"""CPU test of the ids that the paged kernels' bounded waits leave in the status word: one per thing waited for."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-attention-v100_b200", "csrc")
WAIT = re.compile(r"\b(?:rolled_wait|rolled_wait_warp|mbar_wait|mbar_wait_warp)\(")


def _waits(name):
    """{id: what is waited for} of a file; an id is a number at the call's end."""
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    found = {}
    for m in WAIT.finditer(text):
        depth, args, last, i = 0, [], m.end(), m.end()
        while depth >= 0:
            depth += (text[i] in "([{") - (text[i] in ")]}")
            if depth < 0 or (depth == 0 and text[i] == ","):
                args.append(text[last:i].strip())
                last = i + 1
            i += 1
        assert len(args) == 4 and args[2].endswith("abort_word"), args
        assert args[3].isdigit(), args
        found.setdefault(int(args[3]), set()).add(args[0])
    return found


@pytest.mark.parametrize("kernel,least", [("paged_few_kernel.cuh", 22), ("paged_many_kernel.cuh", 15)])
def test_an_id_names_one_wait(kernel, least):
    waits, shared = _waits(kernel), _waits("paged_work.cuh")  # (what both kernels call)
    assert len(waits) >= least and len(shared) == 1
    assert [(i, w) for i, w in sorted(waits.items()) if len(w) > 1] == []
    assert not set(waits) & set(shared)
    assert max(waits) < 256 and min(waits) > 0  # (a byte of the status word)
