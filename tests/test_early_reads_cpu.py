"""What kernels may read before they wait for the kernel that precedes them in the stream, from their source.

A kernel that is launched as a programmatic dependent runs up to its pdl_wait() while earlier kernels still write: in front of
the wait it may read the step's inputs (positions, lengths, pointer and block tables), but nothing that another entry point
produces.  A wrong order cannot be shown by running it: the result then depends on how kernels happen to overlap."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oxide_infer_b200", "csrc")


def _before_the_wait(source, kernel):
    with open(os.path.join(CSRC, source)) as f:
        text = f.read()
    at = re.search(r"^" + kernel + r"\(const \w+ p\)( \{)?$", text, re.M)
    assert at, kernel
    body = text[at.end():]
    return re.sub(r"//[^\n]*", "", body[:body.index("pdl_wait();")])


def _reads(code):
    """Members of the parameter struct that are indexed or dereferenced."""
    return set(re.findall(r"\bp\.((?:\w+\.)*\w+)\s*\[", code)) | set(re.findall(r"\*\s*p\.((?:\w+\.)*\w+)", code))


def test_the_merge_reads_only_the_steps_inputs_before_it_waits():
    # oxi_project_append writes the gate that the merge applies; partial results come from the streaming kernel
    assert _reads(_before_the_wait("decode_attn.cu", "decode_merge_kernel")) == {"seq_lens", "k_ptrs", "v_ptrs"}
