"""The build's check of kernels that wait for loads by their number: no scratch, whose loads would count among them."""
import pytest

from quant_flash_attn_amd import save_check


@pytest.mark.parametrize("name, scratch, found", [(save_check.COUNTING[0], 0, 0), (save_check.COUNTING[0], 16, 1), ("other_kernel", 16, 0)])
def test_no_scratch(tmp_path, name, scratch, found):
    path = tmp_path / "k.s"
    path.write_text(f"_Z3qfa{name}:\n\ts_endpgm\n\t\t.amdhsa_private_segment_fixed_size {scratch}\n")
    assert len(save_check.check(str(path))) == found
