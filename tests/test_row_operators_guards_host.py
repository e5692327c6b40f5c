"""What is checked of the row operators without a GPU: the device assembly."""
import glob
import os

import pytest

from compactwarprnntloss_amd.build import HERE, early_scalar_reads


def test_the_check_of_scalar_reads():
    early = ["v_cmp_le_f32 vcc, v56, v38", "v_addc_co_u32 v64, vcc, v64, v64, vcc"]
    assert [n for n, _ in early_scalar_reads("\n".join(early))] == [2]
    assert early_scalar_reads("\n".join([early[0], "\ts_nop 0 ; one", early[1]])) != []
    assert early_scalar_reads("\n".join([early[0], "\ts_nop 1", early[1]])) == []
    assert early_scalar_reads("\n".join([early[0], "v_mov_b32 v1, v2", "s_mov_b32 s0, 0", early[1]])) == []
    pair = "v_cmp_le_f32_e64 s[10:11], v1, v2"
    assert early_scalar_reads(pair + "\nv_cndmask_b32_e64 v1, 0, 1, s[10:11]") != []
    assert early_scalar_reads(pair + "\nv_add_f32 v1, s11, v2") != []
    assert early_scalar_reads(pair + "\nv_cndmask_b32_e64 v1, 0, 1, s[12:13]") == []
    assert early_scalar_reads(pair + "\ns_and_b64 s[0:1], s[10:11], exec") == []  # the scalar unit waits by itself


def test_no_kernel_reads_a_scalar_register_too_soon():
    listings = glob.glob(os.path.join(HERE, "build", "*-hip-amdgcn-amd-amdhsa-gfx950.s"))
    if not listings:
        pytest.skip("no device assembly beside the library (it is left by a build)")
    for path in listings:
        with open(path) as f:
            assert early_scalar_reads(f.read()) == [], os.path.basename(path)
