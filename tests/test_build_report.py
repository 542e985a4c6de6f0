"""What the build asks of the compiler's resource report."""

import pytest

from flaxchat_amd import build

REPORT = """csrc/a.hip:10:1: remark: Function Name: k_walk<1> [-Rpass-analysis=kernel-resource-usage]
   10 | __global__ void k_walk(Args a) {
csrc/a.hip:10:1: remark:     TotalSGPRs: 106 [-Rpass-analysis=kernel-resource-usage]
csrc/a.hip:10:1: remark:     SGPRs Spill: N [-Rpass-analysis=kernel-resource-usage]
csrc/a.hip:10:1: remark:     VGPRs Spill: 3 [-Rpass-analysis=kernel-resource-usage]
csrc/a.hip:40:1: remark: Function Name: k_other [-Rpass-analysis=kernel-resource-usage]
csrc/a.hip:40:1: remark:     SGPRs Spill: 0 [-Rpass-analysis=kernel-resource-usage]
"""


def test_scalar_spills_are_refused():
    build.check_scalar_spills("a.hip", REPORT.replace("Spill: N", "Spill: 0"))
    with pytest.raises(RuntimeError, match="k_walk<1>"):
        build.check_scalar_spills("a.hip", REPORT.replace("Spill: N", "Spill: 23"))
    with pytest.raises(RuntimeError, match="no resource report"):  # nothing to go by is no pass
        build.check_scalar_spills("a.hip", "warning: something else")


def test_the_paged_walks_are_checked():
    assert "fc_paged.hip" in build.NO_SCALAR_SPILLS and set(build.NO_SCALAR_SPILLS) <= set(build.SOURCES)
