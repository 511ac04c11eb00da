"""What the operators on rows of logits refuse or take at the ends of their
arguments, and what their source has to keep, as far as no device is needed."""
import os
import re

from conftest import PKG


def test_dynamic_shared_memory_is_aligned_for_16_byte_accesses():
    """Lists and slices there are read 16 bytes at a time; an array declared with a smaller type's alignment may start 8 bytes off."""
    source = open(os.path.join(PKG, "csrc", "logits_kernels.cu")).read()
    arrays = re.findall(r"extern __shared__ ([^;]*);", source)
    assert len(arrays) >= 7
    assert [a for a in arrays if not a.startswith(("uint4 ", "__align__(16) "))] == []
