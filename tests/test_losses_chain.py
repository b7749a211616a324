"""The kernels of the losses over the class axis are launched while the kernel before them still runs: what they read behind
their wait must come from ordinary loads, never from read-only ones, which promise that memory does not change while
the kernel lives."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "graph_rws_b200", "csrc")


def _sources():
    """The files whose kernels wait for the kernel before them, without comments."""
    found = {}
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        with open(path) as f:
            text = re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)
        if "wait_for_previous()" in text:
            found[os.path.basename(path)] = text
    return found


def test_dependent_kernels_read_with_ordinary_loads():
    sources = _sources()
    assert {"class_loss.cuh", "class_product.cuh", "linear_ce.cu", "distill.cu"} <= set(sources)
    for name, text in sources.items():
        bad = re.findall(r"__ldg\b|\.global\.nc\b|\bconst\s+\w+\s*\*\s*__restrict__\s*\w*", text)
        assert not bad, (name, bad)


def test_every_kernel_of_a_chain_waits():
    """Each may rely on all before it only if each waits."""
    for name, text in _sources().items():
        kernels = re.findall(r"__global__\s+void\b[^{;]*\{(.*?)\n\}", text, flags=re.S)
        assert kernels or name.endswith(".cuh")
        for body in kernels:
            assert "wait_for_previous()" in body, (name, body[:200])
