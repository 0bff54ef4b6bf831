"""Every kernel that follows tables to memory checks its indices in the bounds build: seen in its source, since a sound call
cannot show a check that is missing."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oxide_infer_b200", "csrc")


def _kernel(source, name):
    """The kernel's text, from its name to the closing brace in the first column."""
    with open(os.path.join(CSRC, source)) as f:
        text = f.read()
    at = re.search(r"^" + name + r"\(", text, re.M)
    assert at, name
    return text[at.start():text.index("\n}\n", at.start())]


@pytest.mark.parametrize("source,name,least", [
    ("append_q8.cu", "append_q8_step_kernel", 2),  # the token's row, the slots that move to a larger scale
    ("append_q8.cu", "append_q8_wave_kernel", 3),  # the window's rows, the rows behind it, the slots
    ("decode_attn_q8.cu", "decode_attn_q8_kernel", 2),  # copied groups, partial results
    ("decode_attn.cu", "decode_attn_kernel", 3),  # copied groups, the appended row, partial results
    ("prefill_attn.cu", "prefill_attn_kernel", 4),  # partial results, output rows, 8-bit groups, paged groups
])
def test_table_driven_accesses_are_checked(source, name, least):
    assert _kernel(source, name).count("OXI_IN_BOUNDS(") >= least
