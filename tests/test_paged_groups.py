"""How many workgroups a launch over pages may have (undertow_amd/csrc/
ut_paged_plan.h), on the CPU; and that appends beyond that are refused."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "undertow_amd" / "csrc"


def test_an_axis_of_a_launch_has_fewer_than_2_32_threads(tmp_path):
    (tmp_path / "g.cpp").write_text('#include "ut_paged_plan.h"\nextern "C" int64_t most(int64_t t) { return ut::most_groups(t); }\n')
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(CSRC), "-o", str(tmp_path / "g.so"),
                    str(tmp_path / "g.cpp")], check=True)
    lib = C.CDLL(str(tmp_path / "g.so"))
    lib.most.restype, lib.most.argtypes = C.c_int64, [C.c_int64]
    for t in (64, 256, 512, 576, 1023, 1024):
        n = lib.most(t)
        assert n * t < 2**32 and (n == 2**22 or (n + 1) * t >= 2**32), t


@pytest.mark.gpu
def test_appends_beyond_a_launch_are_refused(ctx):
    """Before anything is launched: the memory need not be there."""
    import undertow_amd as U
    lib, rt = U.lib(), U.runtime
    import torch
    x = torch.zeros(4096, device="cuda")
    table = torch.zeros(4, dtype=torch.int32, device="cuda")
    for fmt, most in ((U.KV_I8, 2**22 - 1), (U.KV_BF16, 2**22), (U.KV_F16X2, 2**22)):
        kv = rt.MlaPages(pages=x.data_ptr(), n_pages=4, page=1, latent=8, rope=8, fmt=fmt, scales=x.data_ptr())
        n = most + 1
        code = lib.ut_mla_paged_append(ctx.handle, C.byref(kv), table.data_ptr(), n, n, table.data_ptr(), 1, n, x.data_ptr(), x.data_ptr())
        assert code == rt.UT_ERR_SHAPE, fmt
    ctx.synchronize()
