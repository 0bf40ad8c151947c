"""What a build finds in the code that the compiler made."""


def test_build_rejects_spills_in_front_of_the_lanes_that_come_back():
    from optimus_dl_amd.build import check_masked_spills

    masked = "_Z1kv:\n\ts_and_saveexec_b64 s[2:3], s[14:15]\n\ts_cbranch_execz .LBB0_1\n; %bb.0:\n\tglobal_load_dword v2, v1, s[4:5]\n"
    spill, reload = "\tscratch_store_dword off, v9, off offset:80 ; 4-byte Folded Spill\n", "\tscratch_load_dword v9, off, off offset:80 ; 4-byte Folded Reload\n"
    back = "\ts_or_b64 exec, exec, s[2:3]\n"
    for moved in (spill, reload):
        assert len(check_masked_spills(masked + ".LBB0_1:\n\ts_mov_b32 s28, s30\n" + moved + back, "x.s")) == 1
        assert len(check_masked_spills(masked + ".LBB0_1:\n" + moved + moved + back, "x.s")) == 2
        assert check_masked_spills(masked + ".LBB0_1:\n" + back + moved, "x.s") == []
        # before the lanes are switched off, and for the lanes of the path alone
        assert check_masked_spills("_Z1kv:\n" + moved + masked + ".LBB0_1:\n" + back, "x.s") == []
        assert check_masked_spills(masked + moved + ".LBB0_1:\n" + back, "x.s") == []
    # another function's block is its own
    assert check_masked_spills("_Z1kv:\n.LBB0_1:\n" + spill + "_Z1lv:\n" + back, "x.s") == []
