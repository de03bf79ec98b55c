"""What the rows' warps of prompt attention look at of a unit.  Read from the sources: what an early look returns is a matter of time on a GPU."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tensorwarp_b200", "csrc")


def test_rows_look_at_a_units_values_behind_its_scores():
    """A half that a tile did not have comes to the next tile ahead of the conversion, where a phase of `unit_full` may be taken for the one after the
    next: the scores of the unit are waited for first, and the values are given up (the factors' arrival) afterwards."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "twm_cache8_prompt.cuh")).read())
    rows = text[text.index("for (int j = 0; j < w.n; ++j, ++n) {"):]
    looks = [m.start() for m in re.finditer(r"unit_full\[", rows)]
    assert len(looks) == 1
    assert rows.index("tc::wait_uniform(&s_full[x][n & 1]") < looks[0] < rows.index("mbar_arrive(&p_full[x][n & 1])")
