"""A kernel file that has a word in bounds_errors() checks indices: a word
that nothing can set would call any run clean."""
import os
import re

import pytest

CUDA = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "test1_b200", "csrc", "cuda")


def _body(source, name):
    """The text of a function, from its name to the brace that closes it."""
    at = source.index(name + "(")
    first = source.index("{", source.index(")", at))
    depth, i = 0, first
    while True:
        depth += {"{": 1, "}": -1}.get(source[i], 0)
        i += 1
        if depth == 0:
            return source[first:i]


@pytest.mark.parametrize("file,functions", [
    ("answer_loss.cu", ["join_units", "write_totals", "for_units", "for_fours", "pairs_phase", "lengths_phase",
                        "policy_grad_phase"]),
    ("logprob.cu", ["logprob_pack_kernel", "logprob_join_kernel", "logprob_planes_kernel", "logprob_few_kernel"]),
    ("vocab_gemm.cuh", ["vocab_kernel"]),
])
def test_index_checks(file, functions):
    source = re.sub(r"//[^\n]*", "", open(os.path.join(CUDA, file)).read())
    for name in functions:
        assert "T1_OOB(" in _body(source, name), f"{file}: {name} checks no index"
