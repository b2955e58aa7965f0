"""Every launch of the attention operators may begin beside the one before it.  A read that says its data are constant while the grid
lives (__ldg, ld.global.nc, a const __restrict__ pointer) may then be moved in front of the wait for that launch: there is none."""
import glob
import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "miori_b200", "csrc")


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "attention*")) + [os.path.join(CSRC, "pages.cu")]), ids=os.path.basename)
def test_no_read_is_called_constant(path):
    code = re.sub(r"//[^\n]*", "", open(path).read())
    assert "griddepcontrol" not in code  # the waits are those of common.cuh
    assert not re.search(r"__ldg|ld\.global\.nc|__restrict__", code)
