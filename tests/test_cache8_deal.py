"""How attention over the cache held in 8 bits deals out its units, on the CPU: the kernels' own source, a thread a lane."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def part(name, first, last):
    text = open(os.path.join(ROOT, "tensorwarp_b200", "csrc", name)).read()
    return text[text.index(first):text.index(last)]


def test_runs_of_units(tmp_path):
    source = part("twm_cache8.cuh", "struct Cache {", "__device__ __forceinline__ void unpack8") + part("twm_cache8_attn.cuh", "struct __align__(16) Join", "// The same where every")
    assert not re.search(r"\basm\b", source)
    (tmp_path / "deal.h").write_text(source)
    exe = str(tmp_path / "deal_check")
    r = subprocess.run(["g++", "-std=c++20", "-O1", "-pthread", f'-DDEAL="{tmp_path}/deal.h"', os.path.join(ROOT, "tests", "cpp", "deal_check.cpp"), "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr
