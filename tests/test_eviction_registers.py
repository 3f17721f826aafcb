"""The eviction kernels hold a row in registers: the compiler's resource report has to agree (rows that spill to memory are
written, read and waited for again in every pass)."""

import os
import re
import subprocess

import build


def test_no_row_spills():
    source = os.path.join(build.CSRC, "ekv_evict.hip")
    command = [build.hipcc(), *build.HIPCC_FLAGS, "-Rpass-analysis=kernel-resource-usage", "--cuda-device-only", "-c", source,
               "-o", os.devnull]
    report = subprocess.run(command, capture_output=True, text=True, check=True).stderr
    name, spills = None, {}
    for line in report.splitlines():
        if found := re.search(r"Function Name: (\S+)", line):
            name = found.group(1)
        if found := re.search(r"VGPRs Spill: (\d+)", line):
            spills[name] = int(found.group(1))
    assert sum("select_kernel" in name for name in spills) >= 5 and len(spills) >= 7
    # two registers of the copy's addresses, where 64 are the bound; a row's scores and positions are 8 a round
    assert max(spills.values()) <= 2, spills
