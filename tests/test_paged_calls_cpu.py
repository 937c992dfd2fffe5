"""What the sources of the paged cache's kernels keep to."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_kernels_that_begin_early_read_nothing_as_constant():
    """They are launched before the kernel in front has ended, which may write what they read: ld.global.nc is for what nobody writes meanwhile."""
    files = glob.glob(os.path.join(ROOT, "vkllama_b200", "csrc", "paged*.cu*"))
    assert len(files) >= 7
    for f in files:
        with open(f) as t:
            code = re.sub(r"//[^\n]*", "", t.read())
        assert not re.search(r"__ldg\b|\bldg_stream\b|ld\.global\.nc|__restrict__", code), f
