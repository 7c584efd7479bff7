"""What the 8-bit cache's Python side, its rows read back and attention with a
window turn down before the library is called (CPU), and what the library
itself does without a context."""
import torch

import paged8_ref as R8
import undertow_amd as U
from test_paged_api import Ctx, code, dev
from undertow_amd.runtime import UT_ERR_ARG, UT_ERR_SHAPE, PagedCache


def i8(*s):
    return dev(*s, dtype=torch.int8)


def i32(*s):
    return dev(*s, dtype=torch.int32)


def bf(*s):
    return dev(*s, dtype=torch.bfloat16)


def test_pools_that_are_none():
    assert code(lambda: PagedCache(Ctx(), i8(4, 16, 576))) == UT_ERR_ARG  # no scales
    assert code(lambda: PagedCache(Ctx(), bf(4, 16, 576), scales=dev(4, 16, 2))) == UT_ERR_ARG
    assert code(lambda: PagedCache(Ctx(), i8(4, 16, 575), scales=dev(4, 16, 2))) == UT_ERR_SHAPE
    assert code(lambda: PagedCache(Ctx(), i8(4), scales=dev(4, 16, 2))) == UT_ERR_SHAPE
    for s in (dev(4, 16), dev(4, 16, 1), dev(3, 16, 2), dev(4, 2, 16)):
        assert code(lambda: PagedCache(Ctx(), i8(4, 16, 576), scales=s)) == UT_ERR_SHAPE
    for s in (bf(4, 16, 2), dev(4, 16, 4)[..., ::2], torch.zeros((4, 16, 2))):
        assert code(lambda: PagedCache(Ctx(), i8(4, 16, 576), scales=s)) == UT_ERR_ARG
    c = PagedCache(Ctx(), i8(4, 16, 576), scales=dev(4, 16, 2))
    assert c.fmt == U.KV_I8 and c.dtype == torch.bfloat16 and c._kv.scales == c.scales.data_ptr()


def test_rows_read_back_that_do_not_fit():
    c = PagedCache(Ctx(), i8(4, 16, 576), scales=dev(4, 16, 2))
    t, n = i32(2, 4), i32(2)
    assert code(lambda: c.read(t, n, 3, dtype=torch.float16)) == UT_ERR_ARG
    assert code(lambda: c.read(i32(2), n, 3)) == UT_ERR_SHAPE
    assert code(lambda: c.read(t, i32(3), 3)) == UT_ERR_SHAPE
    assert code(lambda: c.read(t, n, 3, starts=i32(3))) == UT_ERR_SHAPE
    assert code(lambda: c.read(t, n, 3, starts=dev(2))) == UT_ERR_ARG
    assert code(lambda: c.read(t, n, 3, out=(dev(2, 3, 512),))) == UT_ERR_SHAPE
    assert code(lambda: c.read(t, n, 3, out=(dev(2, 3, 512), dev(2, 3, 32)))) == UT_ERR_SHAPE
    assert code(lambda: c.read(t, n, 3, out=(bf(2, 3, 512), bf(2, 3, 64)))) == UT_ERR_ARG
    assert code(lambda: c.read(t, n, 3, out=(dev(2, 3, 1024)[..., ::2], dev(2, 3, 64)))) == UT_ERR_ARG


def test_windows_over_batches_that_do_not_fit():
    c = PagedCache(Ctx(), bf(4, 16, 576))
    good = (i32(2, 4), i32(2), bf(2, 1, 16, 512), bf(2, 1, 16, 64))
    for at, t, want in ((0, i32(2), UT_ERR_SHAPE), (1, i32(3), UT_ERR_SHAPE), (2, bf(2, 16, 512), UT_ERR_SHAPE),
                        (2, dev(2, 1, 16, 512), UT_ERR_ARG), (3, bf(2, 1, 16, 32), UT_ERR_SHAPE)):
        args = list(good)
        args[at] = t
        assert code(lambda: c.attend_window(*args, 0.1, 8)) == want, (at, t.shape)
    assert code(lambda: c.attend_window(*good, 0.1, 8, out=dev(2, 1, 16, 512))) == UT_ERR_ARG


def test_the_library_turns_down_a_missing_context():
    L = U.lib()
    assert L.ut_mla_paged_read(None, None, None, 0, 0, None, 0, 0, None, 0, None, None) == UT_ERR_ARG
    assert L.ut_mla_window_attend(None, None, None, 0, 0, None, 0, 0, 0, None, None, 0.0, 1, 0, None) == UT_ERR_ARG


def test_the_oracle_rounds_to_the_nearest_code():
    x = torch.randn((50, 80), generator=torch.Generator().manual_seed(1))
    x[3] = 0.0
    codes, scales = R8.quantised(x, 64)
    y = R8.values8(codes, scales, 64)
    for lo, hi in ((0, 64), (64, 80)):
        top = x[:, lo:hi].double().abs().amax(-1, keepdim=True)
        # half a code step, and the scale's own rounding
        assert ((y - x.double())[:, lo:hi].abs() <= top / 254.0 + top * 2.0 ** -24).all()
        assert torch.equal(codes[:, lo:hi].abs().amax(-1), torch.where(top[:, 0] > 0, 127, 0).to(torch.int8))
