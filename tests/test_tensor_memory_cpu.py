"""Nobody holds Tensor Memory while waiting for another CTA of the split product.

tcgen05.alloc has no limit, so a CTA that keeps its columns until its cluster
has met can close a circle of waits with a kernel of another stream.  Such a
circle is never provoked on a GPU: the order is read from the source.
"""

import os
import re

from conftest import ROOT


def test_columns_go_back_before_the_cluster_meets():
    text = open(os.path.join(ROOT, "rotalabs_accel_b200", "csrc", "rla_w8a8.cu")).read()
    code = re.sub(r"//[^\n]*", "", text)
    start = code.index("w8a8_split_kernel(const __grid_constant__")
    body = code[start:code.index("struct W8Order")]
    waits = [m.start() for m in re.finditer(r"rla_cluster_(?:sync|wait)\(", body)]
    frees = [m.start() for m in re.finditer(r"rla_tmem_dealloc\(", body)]
    assert waits and frees and max(frees) < min(waits)
    # the CTA pair shares its SMs with nobody
    size = re.search(r"constexpr int kW8PairSmem = (\d+) \* 1024;", code)
    assert int(size.group(1)) == 227
