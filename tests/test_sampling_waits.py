"""What sampling's threads share between the passes of top-k and top-p.  Read from the sources: a warp that reads late what the next pass has
reset would wait at another barrier than the rest, so none is made to on a GPU."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tensorwarp_b200", "csrc")
BARRIER = r"__syncthreads\(\)|cluster_sync_all\(\)|\bjoin\(\)|\bscan\("


def block(text, at):
    """The braces that open behind `at`, with all in them."""
    at = text.index("{", at)
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return text[at:i + 1]


def test_a_pass_ends_with_a_barrier_behind_what_it_read():
    """`find` resets its bin ahead of its first barrier, so every way from a pass's last look at it to the next pass has a barrier."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "twm_sample.cuh")).read())
    find = block(text, text.index("auto find = "))
    assert find.index("sh.found_bin = BINS") < find.index("__syncthreads()") and find.rstrip("} \n;").endswith("__syncthreads()")
    loop = block(text, text.index("for (int what = "))
    narrowing = loop[loop.index("while (left > FEW"):]
    rest = narrowing[len(block(narrowing, 0)) + narrowing.index("{"):]
    equal, listed = block(rest, rest.index("if (left > FEW)")), block(rest, rest.index("else {"))
    assert "found_" in narrowing[:narrowing.index(rest)] and "found_" not in rest
    assert re.search(BARRIER, equal) and re.search(BARRIER, listed)
    # in the loop itself the counts are joined ahead of the next look
    body = block(narrowing, 0)
    assert re.search(r"\bjoin\(\);.*\bfind\(", body, re.S)
    # ahead of the loop: what the first look left is read in front of the barrier at the ends of its bin
    ahead = loop[:loop.index("while (left > FEW")]
    look = ahead[ahead.rindex("const int bin = (int)sh.found_bin"):]
    last = max(look.rindex(name) for name in ("sh.found_bin", "sh.found_count", "sh.found_over", "sh.found_over_mass"))
    assert re.search(BARRIER, look[last:])
