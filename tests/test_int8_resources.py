"""The kernels of the 8-bit layers, compiled with the product's flags: registers, scratch memory and LDS hold what their launches
assume -- two 128 x 192 tiles to a CU, nothing spilled in a kernel that is not known to."""
import os
import re
import subprocess

import pytest

from test_kernel_resources import HIPCC, ROOT, product_flags

DECODER_ONLY = 2                                    # product_flags() ends with decoder.hip's own pair


def usage_of(source, tmp_path):
    flags = product_flags()
    assert flags[-DECODER_ONLY:] == ["-mllvm", "-disable-machine-licm"]
    r = subprocess.run([HIPCC] + flags[:-DECODER_ONLY] + ["-Rpass-analysis=kernel-resource-usage", "-c", "-o", str(tmp_path / "o.o"),
                                                          os.path.join(ROOT, "kaldi_amd", "csrc", source)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    usage, name = {}, None
    for line in r.stderr.splitlines():
        m = re.search(r"Function Name: (\S+)", line)
        if m:
            name = m.group(1)
            usage[name] = {}
            continue
        m = re.search(r"remark:.*?\s([A-Za-z][^:]*): (\d+)", line)
        if m and name:
            usage[name][m.group(1).strip()] = int(m.group(2))
    return usage


def spilled(usage):
    return {n for n, u in usage.items() if u["ScratchSize [bytes/lane]"] or u["VGPRs Spill"] or u["SGPRs Spill"]}


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_row_kernels(tmp_path):
    usage = usage_of("rownorm.hip", tmp_path)
    assert sum("RowKernel" in n for n in usage) > 60
    # f32 norm to codes of 16385 .. 32768 columns, 32 elements in each of 1024 threads: 3 registers in scratch memory (right, and slower)
    assert spilled(usage) <= {n for n in usage if re.search(r"RowKernelIfaLb1ELi4ELi1024ELi8E", n)}, spilled(usage)


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_product_kernels(tmp_path):
    usage = usage_of("affine_i8.hip", tmp_path)
    assert sum("TileKernel" in n for n in usage) == 5 * 2 * 3 and sum("SplitKernel" in n for n in usage) == 2 * 2 * 3
    assert not spilled(usage)
    for n, u in usage.items():
        if re.search(r"TileKernelILi128ELi192ELi2ELi4ELi2E", n):         # two workgroups of 8 waves to a CU
            assert u["VGPRs"] + u.get("AGPRs", 0) <= 128 and u["LDS Size [bytes/block]"] <= 80 * 1024, (n, u)
