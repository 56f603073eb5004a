"""The order in which kernels take tensor memory and let the next kernel start, read from their sources."""

import glob
import os
import re

import axonn_b200


def _kernels():
    """(file, line, text) of every ``__global__`` function, comments taken out."""
    csrc = os.path.join(os.path.dirname(os.path.abspath(axonn_b200.__file__)), "csrc")
    for path in sorted(glob.glob(os.path.join(csrc, "*.cu"))):
        with open(path) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        starts = [m.start() for m in re.finditer(r"\b__global__\b", text)] + [len(text)]
        for a, b in zip(starts, starts[1:]):
            yield os.path.basename(path), text.count("\n", 0, a) + 1, text[a:b]


def test_the_next_kernel_starts_when_the_tensor_memory_is_taken():
    """A block whose other warps let the next kernel start before one warp has allocated may find the memory gone to it: a barrier of the
    block stands between the two."""
    both = 0
    for name, line, text in _kernels():
        alloc, ahead = re.search(r"\btmem_alloc(_pair)?\(", text), text.find("pdl_launch_next()")
        if alloc is None or ahead < 0:
            continue
        both += 1
        assert "__syncthreads()" in text[alloc.start():ahead], f"{name}:{line} lets the next kernel start before its tensor memory is allocated"
    assert both >= 4
