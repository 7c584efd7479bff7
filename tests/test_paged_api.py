"""What the paged cache's Python side turns down before the library is called
(CPU: the checks need no device, so tensors stand in for device ones)."""
import pytest
import torch

import undertow_amd as U
from undertow_amd.runtime import UT_ERR_ARG, UT_ERR_SHAPE, PagedCache


class OnDevice(torch.Tensor):
    """A CPU tensor that says it lies on cuda:0."""

    def get_device(self):
        return 0


def dev(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnDevice)


class Ctx:
    device, handle = 0, None

    def check(self, rc):
        raise AssertionError("the library was reached")


@pytest.fixture
def cache():
    return PagedCache(Ctx(), dev(4, 16, 576, dtype=torch.bfloat16), mean=dev(4, 576, dtype=torch.int8),
                      mean_scale=dev(4))


def code(f):
    with pytest.raises(U.UtError) as e:
        f()
    return e.value.code


def test_pools_that_are_none():
    bf = lambda *s: dev(*s, dtype=torch.bfloat16)
    assert code(lambda: PagedCache(Ctx(), dev(4, 16, 576))) == UT_ERR_ARG
    assert code(lambda: PagedCache(Ctx(), bf(4, 16, 575))) == UT_ERR_SHAPE
    assert code(lambda: PagedCache(Ctx(), bf(4))) == UT_ERR_SHAPE
    assert code(lambda: PagedCache(Ctx(), dev(4, 16, 576, dtype=torch.float16))) == UT_ERR_SHAPE
    assert code(lambda: PagedCache(Ctx(), bf(8, 16, 576)[::2])) == UT_ERR_ARG
    assert code(lambda: PagedCache(Ctx(), torch.zeros((4, 16, 576), dtype=torch.bfloat16))) == UT_ERR_ARG
    assert code(lambda: PagedCache(Ctx(), bf(4, 16, 576), mean=dev(4, 576, dtype=torch.int8))) == UT_ERR_ARG
    assert code(lambda: PagedCache(Ctx(), bf(4, 16, 576), mean=dev(3, 576, dtype=torch.int8),
                                   mean_scale=dev(3))) == UT_ERR_SHAPE


def test_a_format_that_is_none():
    for fmt in (2, -1, "bf16", None):
        assert code(lambda: PagedCache.empty(Ctx(), 4, fmt=fmt)) == UT_ERR_ARG


def test_batches_that_do_not_fit(cache):
    i32 = lambda *s: dev(*s, dtype=torch.int32)
    bf = lambda *s: dev(*s, dtype=torch.bfloat16)
    qa, qr = bf(2, 1, 16, 512), bf(2, 1, 16, 64)
    good = (i32(2, 4), i32(2), qa, qr)

    def calls(table, lens, qa, qr):
        yield lambda: cache.attend(table, lens, qa, qr, 0.1)
        yield lambda: cache.attend_pages(table, lens, qa, qr, 0.1, i32(2, 1, 3))
        yield lambda: cache.select(table, lens, qa, qr, 3)

    for at, t, want in ((0, i32(2), UT_ERR_SHAPE), (0, i32(0, 4), UT_ERR_SHAPE), (0, dev(2, 4), UT_ERR_ARG),
                        (0, i32(4, 2).T, UT_ERR_ARG), (0, i32(1, 4).expand(2, 4), UT_ERR_ARG),
                        (1, i32(3), UT_ERR_SHAPE), (1, dev(2, dtype=torch.int64), UT_ERR_ARG),
                        (1, i32(4)[::2], UT_ERR_ARG), (1, torch.zeros(2, dtype=torch.int32), UT_ERR_ARG),
                        (2, bf(2, 16, 512), UT_ERR_SHAPE), (2, bf(3, 1, 16, 512), UT_ERR_SHAPE),
                        (2, dev(2, 1, 16, 512), UT_ERR_ARG), (2, bf(2, 1, 16, 1024)[..., :512], UT_ERR_ARG),
                        (3, bf(2, 1, 16, 32), UT_ERR_SHAPE), (3, bf(2, 1, 8, 64), UT_ERR_SHAPE)):
        args = list(good)
        args[at] = t
        for f in calls(*args):
            assert code(f) == want, (at, t.shape)
    assert code(lambda: cache.attend(*good, 0.1, out=dev(2, 1, 16, 512))) == UT_ERR_ARG
    assert code(lambda: cache.attend(*good, 0.1, out=bf(2, 1, 16, 64))) == UT_ERR_SHAPE
    assert code(lambda: cache.attend_pages(*good, 0.1, i32(2, 3))) == UT_ERR_SHAPE
    assert code(lambda: cache.attend_pages(*good, 0.1, i32(2, 2, 3))) == UT_ERR_SHAPE
    assert code(lambda: cache.select(*good, 3, weights=dev(2, 16))) == UT_ERR_SHAPE
    assert code(lambda: cache.select(*good, 3, out=i32(2, 1, 4))) == UT_ERR_SHAPE
    assert code(lambda: cache.append(good[0], good[1], dev(2, 512), dev(2, 64))) == UT_ERR_SHAPE
    assert code(lambda: cache.append(good[0], good[1], dev(2, 3, 512), dev(2, 2, 64))) == UT_ERR_SHAPE
    assert code(lambda: cache.append(good[0], good[1], bf(2, 1, 512), bf(2, 1, 64))) == UT_ERR_ARG


def test_the_library_turns_down_a_missing_context():
    L = U.lib()
    assert L.ut_mla_paged_append(None, None, None, 0, 0, None, 0, 0, None, None) == UT_ERR_ARG
    assert L.ut_mla_paged_attend(None, None, None, 0, 0, None, 0, 0, 0, None, None, 0.0, None) == UT_ERR_ARG
    assert L.ut_mla_page_select(None, None, None, 0, 0, None, 0, 0, 0, None, None, None, 0, 0, 0, None) == UT_ERR_ARG
    assert L.ut_mla_sparse_attend(None, None, None, 0, 0, None, 0, 0, 0, None, None, 0.0, None, 0, None) == UT_ERR_ARG
