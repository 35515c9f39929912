"""The paged kernels' sources: no instruction of theirs is written in inline
assembly.  The compiler makes a vector instruction wait for the matrix products
whose results it reads only where it chose the instruction itself."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xwfes_amd", "csrc")


@pytest.mark.parametrize("name", ["k_paged.hip", "paged_dev.h", "paged.hip", "paged.h"])
def test_no_instructions_in_inline_assembly(name):
    with open(os.path.join(CSRC, name)) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    found = re.findall(r"\basm\b(?:\s+volatile)?\s*\(\s*((?:\"[^\"]*\"\s*)+)", code)
    assert len(found) == len(re.findall(r"\basm\b", code))
    assert not [x for x in found if re.sub(r"[\"\s]", "", x)]
