"""The build's look at spilled vector registers, on listings."""

from __future__ import annotations

import pytest

from pocketlm_amd.build import masked_spills

# the end of a divergent region: lanes that did not take it are enabled by the s_or
REGION = """
_Z6kernelv:                             ; @_Z6kernelv
; %bb.0:
	s_and_saveexec_b64 s[0:1], s[22:23]
	s_cbranch_execz .LBB0_2
.LBB0_1:
	ds_write_b32 v1, v2
.LBB0_2:
{before}	s_or_b64 exec, exec, s[0:1]
{after}	s_endpgm
.Lfunc_end0:
"""
SPILL = "\tscratch_store_dwordx2 off, v[86:87], off offset:16 ; 8-byte Folded Spill\n"
RELOAD = "\tscratch_load_dwordx2 v[86:87], off, off offset:16 ; 8-byte Folded Reload\n"
SCALARS = "\tv_writelane_b32 v255, s89, 12\n"
OWN = "\tscratch_store_dword off, v3, off\n"  # a store of the program's


@pytest.mark.parametrize("before,after,count", [
    ("", "", 0), (SCALARS, "", 0), (OWN, "", 0), ("", SPILL, 0), (RELOAD, SPILL, 0), (SPILL, "", 1), (SCALARS + SPILL, "", 1),
    (SPILL + SCALARS + SPILL, SPILL, 2)])
def test_spills_while_lanes_are_off(before, after, count):
    found = masked_spills(REGION.format(before=before, after=after))
    assert len(found) == count
    assert all(f.startswith("_Z6kernelv: scratch_store_dwordx2") for f in found)


def test_saves_of_all_lanes():
    """A function's own save of a register, with every lane on, and a spill in a region of its own."""
    assert masked_spills("""
_Z4colds:
; %bb.0:
	s_or_saveexec_b64 s[16:17], -1
	scratch_store_dword off, v38, s32       ; 4-byte Folded Spill
	s_mov_b64 exec, s[16:17]
	s_and_saveexec_b64 s[0:1], vcc
	scratch_store_dword off, v4, s32        ; 4-byte Folded Spill
	s_cbranch_execz .LBB1_2
; %bb.1:
	scratch_store_dword off, v5, s32        ; 4-byte Folded Spill
.LBB1_2:
	s_or_b64 exec, exec, s[0:1]
	s_setpc_b64 s[30:31]
.Lfunc_end1:
""") == []
