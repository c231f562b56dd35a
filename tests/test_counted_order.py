"""The build's check of kernels that wait for loads by their number: how many requests lie behind the loads into LDS on every path, and what is waited for
before LDS is loaded again."""
import pytest

from quant_flash_attn_amd import save_check

KEYS, VALUE, SCALE = "buffer_load_dwordx4 v1, s[0:3], 0 offen lds", "global_load_dwordx4 v[4:7], v[2:3], off", "global_load_dword v8, v[2:3], off"
WAIT, READ = "s_waitcnt vmcnt(2)", "ds_read_b128 v[12:15], v9"


def asm(*lines):
    return [x for line in lines for x in ("\t;;#ASMSTART", "\t" + line, "\t;;#ASMEND")]


def found(tmp_path, *lines, name="_Z3" + save_check.COUNTING[0]):
    path = tmp_path / "k.s"
    path.write_text("\n".join([name + ":", *lines, "\ts_endpgm", "\t\t.amdhsa_private_segment_fixed_size 0", ""]))
    return save_check.check(str(path))


def loop(first=(KEYS, VALUE, VALUE), inside=(KEYS, VALUE, VALUE), reads_done="s_waitcnt lgkmcnt(0)", inline=True):
    done = asm(reads_done) if inline else ["\t" + reads_done]
    return [*("\t" + x for x in first), ".LBB0_1:", *asm(WAIT), "\t" + READ, *done, *("\t" + x for x in inside), "\ts_cbranch_scc1 .LBB0_1"]


@pytest.mark.parametrize("lines", [loop(), loop(inside=(KEYS, KEYS, VALUE, "v_add_u32_e32 v1, v2, v3", VALUE)), loop(inside=(KEYS, SCALE, VALUE, VALUE)), [], loop(first=(SCALE, KEYS, VALUE, VALUE))])
def test_in_order(tmp_path, lines):
    assert not found(tmp_path, *lines)


# on one path or another too few behind the keys, none, or what was read is not waited for by a statement (one of the compiler's may move)
@pytest.mark.parametrize("lines,what", [(loop(first=(KEYS, VALUE)), "behind"), (loop(inside=(KEYS, VALUE)), "behind"), (loop(inside=(VALUE, VALUE, KEYS)), "behind"),
                                        (loop(first=()), "behind"), (loop(inside=(KEYS, VALUE, KEYS, VALUE)), "behind"),
                                        (loop(reads_done="s_waitcnt lgkmcnt(1)"), "read"), (loop(reads_done="s_nop 0"), "read"), (loop(inline=False), "read")])
def test_out_of_order(tmp_path, lines, what):
    bad = found(tmp_path, *lines)
    assert bad and all(what in b for b in bad)
    assert not found(tmp_path, *lines, name="_Z3other_kernel")
