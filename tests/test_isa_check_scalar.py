"""The build-time check of scalar registers that a VALU instruction wrote and a memory access in inline assembly reads
(h3metal_amd/isa_check.py): 5 wait states, or a scalar instruction's value in between."""

from h3metal_amd.isa_check import VALU_TO_VMEM, scan

LOAD = """;;#ASMSTART
s_mov_b32 m0, s9
s_nop 0
buffer_load_dwordx4 v1, s[16:19], 0 offen lds
;;#ASMEND"""


def listing(*lines):
    return "\n".join(["kern:"] + list(lines))


def test_a_lane_value_in_a_descriptor_waits():
    assert VALU_TO_VMEM == 5
    for write in ("v_readlane_b32 s18, v3, 5", "v_readfirstlane_b32 s16, v3", "v_cmp_gt_u32_e64 s[18:19], v1, v2"):
        assert len(scan(listing(write, LOAD))) == 1  # two instructions in between
        assert len(scan(listing(write, "s_nop 1", LOAD))) == 1  # four
        assert scan(listing(write, "s_nop 2", LOAD)) == []
        assert scan(listing(write, *["v_add_f32 v9, v9, v9"] * 3, LOAD)) == []


def test_scalar_instructions_need_no_wait():
    assert scan(listing("v_readlane_b32 s4, v3, 5", "s_lshl_b32 s18, s4, 8", LOAD)) == []
    assert scan(listing("v_readlane_b32 s18, v3, 5", "s_lshl_b32 s18, s18, 8", LOAD)) == []
    assert scan(listing("v_readlane_b32 s20, v3, 5", "v_readlane_b32 s9, v3, 6", LOAD)) == []  # M0's is read by s_mov


def test_the_compilers_own_accesses_are_its_own():
    assert scan(listing("v_readlane_b32 s18, v3, 5", "buffer_load_dwordx4 v[0:3], v1, s[16:19], 0 offen")) == []
