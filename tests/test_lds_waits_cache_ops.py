"""The prompt attention that takes its rows' images by direct loads into LDS
orders them as the kernels of test_lds_waits.py do: at its one barrier a step's
image has arrived and the wave's reads of the step before it have returned.
Checked on the built library."""
import glob
import os
import re
import shutil

import pytest
from test_lds_waits import LLVM, _run

from rapidocrvl_amd import build

# k_cache_attn<head_dim, tree, shaped, images = true>
NAMES = [f"_ZN4pocr12k_cache_attnILi{hd}ELb0ELb{shaped}ELb1EEEvNS_9CacheAttnENS_8AttnPlanE" for hd in (64, 128) for shaped in (0, 1)]


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not os.path.exists(build.LIB):
        build.build()
    if not os.path.exists(os.path.join(LLVM, "llvm-objdump")):
        pytest.skip("no llvm-objdump")
    d = tmp_path_factory.mktemp("code")
    _run(os.path.join(LLVM, "llvm-objdump"), "--offloading", shutil.copy(build.LIB, d))
    out = {}
    for obj in glob.glob(os.path.join(d, "*gfx950")):
        if NAMES[0] not in _run(os.path.join(LLVM, "llvm-readelf"), "-sW", obj):
            continue
        text = _run(os.path.join(LLVM, "llvm-objdump"), "-d", "--no-show-raw-insn", "--disassemble-symbols=" + ",".join(NAMES), obj)
        for part in re.split(r"^[0-9a-f]+ <", text, flags=re.M)[1:]:
            name, body = part.split(">:", 1)
            out[name] = [ln.split("//")[0].strip() for ln in body.splitlines() if ln.strip()]
    return out


@pytest.mark.parametrize("name", NAMES)
def test_image_loads_arrive_and_reads_return(kernels, name):
    code = kernels[name]
    assert sum("load_lds" in i for i in code) >= 2  # the first step's and the next one's
    at = [i for i, ins in enumerate(code) if ins.startswith("s_barrier")]
    assert at
    for i in at:
        assert re.match(r"s_waitcnt\b.*lgkmcnt\(0\)", code[i - 1]), code[i - 1]
        # no direct load between the wait for the loads and the barrier
        wait = max(j for j in range(i) if re.match(r"s_waitcnt\b.*vmcnt\(0\)", code[j]))
        assert not any("load_lds" in c or c.startswith("s_cbranch") for c in code[wait:i])
