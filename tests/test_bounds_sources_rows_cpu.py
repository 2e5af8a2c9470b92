"""The kernels on rows of logits and lists of tokens check their indices against
what was allocated, so that the bounds-checked build's silence says something."""
import os
import re

import pytest

from test_bounds_sources_cpu import CUDA, _body


def _source(file):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CUDA, file)).read())


@pytest.mark.parametrize("file,functions", [
    ("row_select.cu", ["void fetch", "void add_to", "Scan scan_stretch", "scan_bins_kernel", "void order_list", "void finish_row",
                       "scan_list_kernel"]),
    ("distillation.cu", ["loss_kernel", "scale_kernel"]),
    ("logprob.cu", ["list_kernel"]),
])
def test_functions_check_indices(file, functions):
    source = _source(file)
    for name in functions:
        assert "T1_OOB(" in _body(source, name), f"{file}: {name} checks no index"


@pytest.mark.parametrize("file,sizes", [
    # global memory read and written, workspaces, shared memory by its size
    ("row_select.cu", ["p.elements", "p.outputs", "p.all_segments", "p.list_slots", "p.rows", "p.V", "held_bytes()", "kBins",
                       "kBatch", "kListSlots", "kMostCtas"]),
    ("distillation.cu", ["p.entries", "p.rows", "p.blocks", "entries"]),
])
def test_checks_are_against_what_was_allocated(file, sizes):
    source = _source(file)
    for size in sizes:
        assert re.search(r"T1_OOB\([^;{}]*, " + re.escape(size) + r"\)", source), f"{file}: no index is checked against {size}"
