"""What the fp4 kernels' sources and the compiler's assembly of them have to keep, where correctness depends on it."""
import os
import re

from kubernetes_amd.native import build as nb

SOURCE = os.path.join(nb.SRC_DIR, "hip", "kamd_mxfp4.hip")


def test_lds_arrays_state_their_alignment():
    """Arrays of bytes in LDS are read and written by words, 8 and 16 bytes: their declarations have to say so, the type
    does not."""
    with open(SOURCE) as f:
        arrays = [line.strip() for line in f if re.search(r"__shared__.*\[.*\];", line)]
    assert len(arrays) >= 4
    for line in arrays:
        m = re.search(r"aligned\((\d+)\)", line)
        assert m and int(m.group(1)) >= 8, line
