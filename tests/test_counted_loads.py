"""The build's check of kernels that wait for loads by their number: no scratch, whose loads would count among them."""
import os
import re

import pytest

from quant_flash_attn_amd import build, save_check


@pytest.mark.parametrize("name, scratch, found", [(save_check.COUNTING[0], 0, 0), (save_check.COUNTING[0], 16, 1), ("other_kernel", 16, 0)])
def test_no_scratch(tmp_path, name, scratch, found):
    path = tmp_path / "k.s"
    path.write_text(f"_Z3qfa{name}:\n\ts_endpgm\n\t\t.amdhsa_private_segment_fixed_size {scratch}\n")
    assert len(save_check.check(str(path))) == found


def test_the_library_as_built():
    """The loads of values that such a kernel counts are as many as its wait leaves on their way, and stand behind the loads of keys into LDS."""
    asm = build.assembly_path("qfa_paged_list.hip")
    if not os.path.exists(asm):
        pytest.skip("the library's assembly is not there: it stays in the build folder of the machine that built it")
    kernels = re.findall(r"^_Z\S*paged_list_few_kernel\S*:.*?^\s*s_endpgm", open(asm).read(), re.S | re.M)
    assert len(kernels) == 18
    for text in kernels:
        waits = {int(n) for n in re.findall(r"ASMSTART\n\s*s_waitcnt vmcnt\((\d+)\)\n", text)} - {0}
        assert len(waits) == 1
        events, own = [], False
        for line in text.splitlines():
            own = "ASMSTART" in line or (own and "ASMEND" not in line)
            if re.match(r"\s*buffer_load\S* .*lds", line):
                events.append("k")
            elif re.match(r"\s*global_load_dwordx4 (?!.* nt)", line):
                events.append("v")
            elif own and "vmcnt(" in line and "vmcnt(0)" not in line:
                events.append("w")
            elif re.match(r"\s*(scratch|flat)_", line):
                events.append("s")
        runs = re.findall(r"v+", "".join(events))
        assert "s" not in events and len(runs) >= 2 and {len(r) for r in runs} == waits and not re.search(r"(^|w)v", "".join(events))
