"""What the serving operators' second kernel does with what a call leaves whose wait ran out: the spans that it reads are
bounded (here, without a GPU) and its rows are NaN (with one)."""
import os
import subprocess

import pytest

from huggingfaceeacp_b200 import build

CSRC = os.path.join(build.PKG, "csrc")

SPANS = """
#include "key_span.cuh"
#include <climits>
#include <initializer_list>
#include <cstdio>
using namespace hfk;
int main()
{
    const int words[] = {INT_MIN, -kFew, -2, -1, 0, 1, 147, 148, 295, 296, kFew - 1, kFew, kFew | 1, kFew | 295, kFew | 296, INT_MAX};
    int wrong = 0;
    for (int ctas : {1, 148, 296})
        for (int x : words)
            for (int y : words)
            {
                const KeySpan s = key_span(x, y, ctas);
                bool fits = false; // one of the pairs that a CTA can leave
                for (int first = 0; first < ctas; ++first)
                    fits = fits || ((x == first || x == (kFew | first)) && y >= first && y < ctas);
                wrong += s.there != fits;
                wrong += s.there && (s.first < 0 || s.last >= ctas || s.first > s.last || s.few != (x >= kFew));
            }
    std::printf("%d\\n", wrong);
    return wrong != 0;
}
"""


def test_spans_that_no_cta_left_are_not_followed(tmp_path):
    source, program = str(tmp_path / "spans.cpp"), str(tmp_path / "spans")
    with open(source, "w") as f:
        f.write(SPANS)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", source, "-o", program], check=True)
    result = subprocess.run([program], capture_output=True, text=True)
    assert result.returncode == 0, result.stdout


@pytest.mark.gpu
def test_the_join_of_a_failed_call_is_nan(tmp_path):
    program = str(tmp_path / "join")
    subprocess.run([build.NVCC, *build.ARCH, "-std=c++17", "-O1", f"-I{build.INCLUDE}", f"-I{CSRC}",
                    os.path.join(os.path.dirname(os.path.abspath(__file__)), "join_harness.cu"), "-o", program], check=True)
    result = subprocess.run([program], capture_output=True, text=True, timeout=120)
    assert result.returncode == 0, result.stdout + result.stderr
