"""What the layer norm kernels have to do in order, read from their source: an access out of order need not show in any
result, since the blocks of a cluster usually start together."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quabla_b200", "csrc")


def code(name):
    """A source file without its comments."""
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def body(text, start):
    """The block in braces that follows `start`."""
    at = text.index("{", text.index(start))
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i + 1]
    raise AssertionError(f"no end of {start}")


def test_only_the_row_sums_reach_into_another_blocks_shared_memory():
    remote = [name for name in sorted(os.listdir(CSRC)) if re.search(r"map_shared_rank|\bmapa\b|shared::cluster", code(name))
              and name.startswith("norm")]
    assert remote == ["norm_kernels.cuh"]
    text = code("norm_kernels.cuh")
    assert text.count("map_shared_rank") == body(text, "struct RowSum").count("map_shared_rank") == 1


def test_row_sums_arrive_when_they_are_made_and_wait_when_they_meet():
    sums = body(code("norm_kernels.cuh"), "struct RowSum")
    made = body(sums, "group(threadIdx.x / shape.threads_per_row)")
    assert "barrier_arrive" in made and "barrier_wait" not in made
    assert "barrier_wait" in body(sums, "void meet()")


@pytest.mark.parametrize("kernel", ["norm_forward_kernel", "norm_backward_kernel"])
def test_a_clusters_blocks_meet_before_the_first_sum(kernel):
    rows = body(code("norm_kernels.cuh"), f"\n{kernel}(")
    made, met = rows.index("row_sum(shared, shape)"), [m.start() for m in re.finditer(r"row_sum\.meet\(\)", rows)]
    sums = [m.start() for m in re.finditer(r"row_sum\((?!shared)", rows)]
    assert len(met) == 1 and sums and made < met[0] < min(sums)
    # In the kernel's outermost block, and nothing leaves the kernel before it: every thread takes part.
    before = rows[:met[0]]
    assert before.count("{") - before.count("}") == 1
    assert not re.search(r"\breturn\b", before[:before.index("auto fetch")])


def test_one_rows_stride_forms_no_address():
    # Groups and turns without a row still name a source in their copies of no bytes: with one row that is the row itself.
    text = code("norm.cu")
    assert "rows > 1 ? (long long)stride : 0" in body(text, "qb::RowArray rows_of(")
    calls = re.findall(r"rows_of\(d_[^)]*\)", text)
    assert calls and all(call.endswith(", rows)") for call in calls)
