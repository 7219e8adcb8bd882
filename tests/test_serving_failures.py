"""What the serving operators do once a wait has run out: copies in flight are waited for, the spans that the second kernel
reads are bounded (without a GPU), and its rows are NaN (with one)."""
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
                wrong += !s.there && s.first <= s.last;
            }
    std::printf("%d\\n", wrong);
    return wrong != 0;
}
"""


def test_spans_that_no_cta_left_are_not_followed(tmp_path):
    result = _host_program(tmp_path, SPANS)
    assert result.returncode == 0, result.stdout


PHASES = """
#include "phases.cuh"
#include <cstdio>
using namespace hfk;
int main()
{
    int wrong = 0;
    for (int begun = 1; begun < 9; ++begun)
        for (int over = begun - 1; over <= begun; ++over) // the last use in flight, then over
        {
            const bool returns = (unsigned) (over & 1) != last_parity(begun); // the current phase has the other parity
            wrong += returns != (over == begun);
        }
    std::printf("%d\\n", wrong);
    return wrong != 0;
}
"""


def _host_program(tmp_path, text):
    source, program = str(tmp_path / "program.cpp"), str(tmp_path / "program")
    with open(source, "w") as f:
        f.write(text)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", source, "-o", program], check=True)
    return subprocess.run([program], capture_output=True, text=True)


def test_a_failed_call_waits_for_the_last_copy_of_queries(tmp_path):
    """A CTA may not end while a copy into its shared memory is in flight: the wait names that copy's phase."""
    result = _host_program(tmp_path, PHASES)
    assert result.returncode == 0, result.stdout
    with open(os.path.join(CSRC, "attention_mma.cuh")) as f:
        assert "mbar_wait(&h.query, last_parity(put_queries))" in f.read()


def _device_program(tmp_path, source, *flags):
    program = str(tmp_path / "program")
    subprocess.run([build.NVCC, *build.ARCH, "-std=c++17", "-O1", *flags, f"-I{build.INCLUDE}", f"-I{CSRC}",
                    os.path.join(os.path.dirname(os.path.abspath(__file__)), source), "-o", program], check=True)
    return subprocess.run([program], capture_output=True, text=True, timeout=120)


@pytest.mark.gpu
def test_the_join_of_a_failed_call_is_nan(tmp_path):
    result = _device_program(tmp_path, "join_harness.cu")
    assert result.returncode == 0, result.stdout + result.stderr


@pytest.mark.gpu
def test_a_wait_without_an_arrival_ends(tmp_path):
    """However its lanes wait, it returns and sets the error word; what has come is not kept waiting."""
    result = _device_program(tmp_path, "wait_harness.cu", "-DHFK_WAIT_TICKS=0")
    assert result.returncode == 0, result.stdout + result.stderr
