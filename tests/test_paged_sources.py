"""The paged kernels are launched to start while the kernel before them in the
stream still runs. What that one wrote is visible after griddepcontrol.wait and
not promised to be otherwise, so every kernel has to wait, unconditionally."""
import glob
import os
import re

import pytest

from helpers import ROOT

SOURCES = sorted(glob.glob(os.path.join(ROOT, "lfm3-gufo-extension_b200", "csrc",
                                        "paged_*.cu")))


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_every_kernel_waits_for_the_one_before(path):
    text = open(path).read()
    # a kernel's body: from its opening brace to the next "}" in column 0
    kernels = re.findall(r"__global__.*?\)\s*\{\n(.*?)\n\}", text, re.S)
    assert len(kernels) == text.count("__global__")
    for body in kernels:
        waits = re.findall(r"^( *)grid_dependency_wait\(\);", body, re.M)
        assert waits == ["  "], waits  # one, a statement of the body itself
        # (no condition without braces in front of it)
        before = body[:body.index("grid_dependency_wait();")].rstrip()
        assert before == "" or before[-1] in ";}" or before.splitlines()[-1] \
            .lstrip().startswith("//"), before[-80:]
