"""The order that programmatic launches need, read from the serving operators' kernels (CPU only)."""
import os
import re

import pytest

from huggingfaceeacp_b200 import build

CSRC = os.path.join(build.PKG, "csrc")
FILES = ["attention_few.cuh", "attention_limbs.cuh", "attention_mma.cuh", "attention_short.cuh", "pages.cuh"]
READS = r"bounded_offset|sequence_of|load8|\.begin\(|prompt_place|open_book|\bb\.copies|\bw\.\w+\[|\bc\.spans|g_operator_error"


def _kernels(text):
    """(name, body) of every __global__ function."""
    for found in re.finditer(r"__global__ void[^{;]*?\b(\w+)\(const[^{;]*\n{", text):
        yield found.group(1), text[found.end():text.index("\n}\n", found.end())]


@pytest.mark.parametrize("file", FILES)
def test_kernels_wait_before_they_read_what_an_earlier_one_wrote(file):
    with open(os.path.join(CSRC, file)) as f:
        kernels = dict(_kernels(f.read()))
    assert kernels
    for name, body in kernels.items():
        wait, read = body.find("pdl_wait();"), re.search(READS, body)
        assert wait >= 0 and read, name
        assert wait < read.start(), f"{name} reads before it waits: {body[read.start():read.start() + 40]}"
        assert body.find("pdl_trigger();") < 0 or wait < body.find("pdl_trigger();"), name
