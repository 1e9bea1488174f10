"""Loads of data that the preceding kernel of the stream writes are coherent.

Under programmatic dependent launch a kernel is resident while its predecessor
still writes; the non-coherent load path (``ld.global.nc``, which the compiler
also takes for ``const T* __restrict__`` inputs) is only for data that nobody
writes while the kernel is resident.  No run shows the difference reliably, so
the sources are read.
"""

import os
import re

from conftest import ROOT

CSRC = os.path.join(ROOT, "rotalabs_accel_b200", "csrc")


def _source(name):
    return open(os.path.join(CSRC, name)).read()


def test_only_weights_are_read_through_the_non_coherent_path():
    uses = []
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".cu", ".cuh")):
            code = re.sub(r"//[^\n]*", "", _source(name))
            for m in re.finditer(r"\.nc\b|__ldg\s*\(", code):
                function = re.findall(r"\b(rla_\w+|\w+)\s*\([^()]*\)\s*\{", code[:m.start()])[-1]
                uses.append((name, function))
    assert uses == [("rla_common.cuh", "rla_ldg_stream")]
    for name in ("rla_skinny.cu", "rla_moe.cu", "rla_rows.cu"):      # ... and that one reads weights only
        for arg in re.findall(r"rla_ldg_stream\(([^)]*)\)", _source(name)):
            assert arg.startswith("wrow"), (name, arg)


def test_rows_of_dependent_launches_are_not_restrict():
    """The row kernels launched with the attribute and their activations."""
    signature = re.search(r"__global__ void rmsnorm_rows_kernel\((.*?)\)\s*\{", _source("rla_misc.cu"), re.S).group(1)
    assert re.search(r"const __half\* x\b", signature), signature
    assert "__restrict__" not in _source("rla_rows.cu") and "__restrict__" not in _source("rla_moe.cu")
