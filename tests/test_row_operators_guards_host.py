"""What is checked of the row operators without a GPU: the device assembly, refusals."""
import glob
import os

import pytest
import torch

import compactwarprnntloss_amd as pkg
from compactwarprnntloss_amd import _lib
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


def test_checks_of_the_step_rows():
    """cwr_join_rows(f, g, dtype, act, R, H, h, stream): refused before any HIP call."""
    call = _lib.load().cwr_join_rows
    p = [0x10000 * n for n in range(1, 4)]
    null, dtype, mode, shape, align, large = 1, 2, 3, 4, 6, 8
    assert call(None, p[1], 0, 0, 5, 8, p[2], None) == null and call(p[0], None, 0, 0, 5, 8, p[2], None) == null
    assert call(p[0], p[1], 0, 0, 5, 8, None, None) == null
    assert call(p[0], p[1], 4, 0, 5, 8, p[2], None) == dtype and call(p[0], p[1], 0, 3, 5, 8, p[2], None) == mode
    assert call(p[0], p[1], 0, 0, -1, 8, p[2], None) == shape and call(p[0], p[1], 0, 0, 5, 0, p[2], None) == shape
    assert call(p[0] + 2, p[1], 0, 0, 5, 8, p[2], None) == align and call(p[0], p[1], 1, 0, 5, 8, p[2] + 1, None) == align
    assert call(p[0], p[1], 0, 0, 5, 1 << 30, p[2], None) == large and call(p[0], p[1], 0, 0, 1 << 33, 8, p[2], None) == large
    assert call(None, None, 0, 0, 0, 8, None, None) == 0


def test_lattice_tokens_refuses_tensors_of_several_devices():
    """A kernel on one device would read another's memory.  The checks look at a tensor's description only, so that
    stand-ins do where there is one device or none."""
    class Described:
        is_cuda, dtype = True, torch.int32

        def __init__(self, index, *shape):
            self.device, self.shape = torch.device("cuda", index), torch.Size(shape)

        def is_contiguous(self):
            return True

        def dim(self):
            return len(self.shape)

        def size(self, d):
            return self.shape[d]
    for devices in ((0, 1, 0), (0, 0, 1), (1, 0, 0)):
        lx, y, ly = (Described(i, *shape) for i, shape in zip(devices, ((2,), (2, 3), (2,))))
        with pytest.raises(RuntimeError, match="device of lx"):
            pkg.lattice_tokens(lx, y, ly, 4, 8)
