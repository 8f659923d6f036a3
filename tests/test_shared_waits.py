"""How the waits of attention over shared keys end that something never comes for."""

import os
import re

import pytest

from freetoken_b200.kernels import library, ops


def test_lanes_of_a_warp_give_up_together():
    """Every wait is voted on, at once or (the issuing warp's) at the end of the key tile, with no way out before that."""
    with open(os.path.join(library.CSRC, "shared_attention_tc.cuh")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    seen = 0
    for m in re.finditer(r"mbar_wait\(", text):
        before = text[max(text.rindex(";", 0, m.start()), text.rindex("{", 0, m.start())):m.start()]
        seen += 1
        if "__all_sync(" in before:
            continue
        rest = text[m.end():text.index("ok = all_of_warp(fine)", m.end())]
        assert "fine = false;" in rest[:200] and not re.search(r"\b(break|return|continue)\b", rest), text[m.start() - 80:m.end() + 60]
    for issue in re.finditer(r"elect_one\(\)\) ([^\n]*)", text):
        assert issue.group(1).startswith("if (fine)")
    assert seen == 5


@pytest.mark.gpu
@pytest.mark.parametrize("code", [801, 809])
def test_the_status_word_is_read_and_cleared(code):
    """Written from the host: no wait is made to run out."""
    assert ops.read_status() == 0
    ops.debug_set_status(6, code)
    with pytest.raises(ops.KernelError, match=f"status {code}"):
        ops.check_status()
    assert ops.read_status() == 0
