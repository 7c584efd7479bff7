"""Attention over the paged cache with a window and a few first positions on
the GPU against 64 bits, over pages of each format.  Tolerances stand at
paged8_ref.close."""
import math

import pytest
import torch

import paged8_ref as R8
from test_gpu_paged import SCALE

pytestmark = pytest.mark.gpu
FMTS = ["bf16", "f16x2", "i8"]


def unnamed(pool, M, window, sinks):
    """The pool's table with the pages that no row of a call sees named by ids
    that exist nowhere, and everything in those pages NaN."""
    table = pool.table.clone()
    for b, n in enumerate(pool.lens):
        at = [R8.positions(n - M + j + 1, window, sinks) for j in range(M)]
        seen = set((torch.cat(at) // pool.page).tolist())
        for k in range(-(-n // pool.page)):
            if k not in seen:
                (pool.scales if hasattr(pool, "scales") else pool.pages)[table[b, k].long()] = math.nan
                table[b, k] = -1 if k % 2 else 2**31 - 1
    return table


def window_case(ctx, fmt, lens, M, H, window, sinks, L=512, P=64, page=64, width=None, seed=1):
    pool = R8.pool(fmt, seed, lens, page, L, P, width)
    qabs, qrope = pool.queries(M, H)
    table = unnamed(pool, M, window, sinks)
    got = pool.cuda(ctx=ctx).attend_window(table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE, window, sinks)
    ctx.synchronize()  # no page that is not named was asked for
    R8.check(pool, fmt, got, qabs, qrope, SCALE, window=window, sinks=sinks)
    return pool, qabs, qrope, got


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,H,page,window,sinks", [
    ([1], 1, 128, 64, 1, 0), ([2, 0, 1], 1, 128, 16, 1, 1), ([300, 64, 65, 63, 1, 0], 1, 128, 64, 64, 4),
    ([500], 1, 128, 64, 7, 0), ([500], 1, 128, 64, 33, 33), ([130, 1, 0, 77], 4, 128, 32, 16, 2),
    ([300, 200, 1, 0], 3, 32, 64, 31, 64), ([257, 3, 600], 2, 64, 128, 100, 1), ([100, 31, 1001], 1, 16, 16, 96, 32),
    ([140, 1, 229], 2, 16, 8, 40, 9), ([333, 12], 1, 20, 64, 2000, 5), ([190], 3, 1, 32, 1, 0), ([190], 3, 1, 32, 1, 3),
    ([200, 45, 5], 1, 96, 256, 32, 1000), ([70, 12, 0, 9], 2, 48, 1, 5, 3), ([1500, 9, 1], 1, 128, 1024, 77, 40),
    ([400, 399, 385, 384, 383, 353, 352], 2, 128, 32, 64, 32)])
def test_window(ctx, fmt, lens, M, H, page, window, sinks):
    window_case(ctx, fmt, lens, M, H, window, sinks, page=page)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,H,L,P,page,window,sinks", [
    ([1, 0, 140, 65], 1, 4, 64, 16, 16, 20, 3), ([17, 64, 130], 3, 4, 64, 16, 64, 64, 0), ([33, 5], 2, 8, 16, 8, 4, 3, 1),
    ([100], 1, 3, 1000, 24, 32, 50, 70), ([60, 300], 1, 2, 512, 128, 16, 100, 30), ([5000, 0, 70], 1, 5, 136, 8, 64, 3000, 64)])
def test_window_other_widths(ctx, fmt, lens, M, H, L, P, page, window, sinks):
    window_case(ctx, fmt, lens, M, H, window, sinks, L, P, page)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,H,window,sinks,width", [
    ([9001], 1, 128, 4096, 4, None), ([5000, 17, 3000], 2, 128, 1000, 1, None), ([6001] * 5, 1, 16, 2048, 64, None),
    ([4000, 0, 2000, 1], 1, 64, 999, 0, None), ([12000], 4, 32, 5000, 128, None), ([5, 900, 31] * 30, 1, 16, 200, 4, 9000),
    ([(37 * k) % 900 for k in range(300)], 1, 16, 100, 4, None), ([2000] + [100] * 70, 1, 128, 700, 4, 8192)])
def test_window_cut_into_ranges(ctx, fmt, lens, M, H, window, sinks, width):
    window_case(ctx, fmt, lens, M, H, window, sinks, width=None if width is None else width // 64)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,H,window,sinks,width", [
    ([600, 40, 333], 128, 256, 64, 4, 4096), ([700], 300, 128, 100, 0, 8192), ([1500, 700], 40, 128, 513, 33, 2048),
    ([140, 200], 140, 16, 5, 1, 300)])
def test_window_prompt_rows(ctx, fmt, lens, M, H, window, sinks, width):
    window_case(ctx, fmt, lens, M, H, window, sinks, width=width // 64)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,H,L,P,page,window,sinks", [
    (3, 128, 512, 64, 64, 20, 2), (3, 16, 512, 64, 16, 70, 0), (40, 32, 512, 64, 32, 9, 1), (3, 4, 64, 16, 16, 20, 2)])
def test_what_a_row_does_not_see_does_not_reach_it(ctx, fmt, M, H, L, P, page, window, sinks):
    """NaN at positions that some rows of a call see and others do not, in
    front of a window as behind the end: the rows that see one are NaN, the
    others as without."""
    lens = [197, 164, 230]
    pool = R8.pool(fmt, 3, lens, page, L, P)
    qabs, qrope = [t.cuda() for t in pool.queries(M, H)]
    args = pool.table.cuda(), pool.lens32().cuda(), qabs, qrope, SCALE, window, sinks
    clean = pool.cuda(ctx=ctx).attend_window(*args)
    odd = {}
    for b, n in enumerate(lens):
        first = n - M + 1 - window  # the first row's window begins here
        odd[b] = [(n - 1, first), (first + 1, sinks), (n - M + 1,)][b]
        for t in odd[b]:
            x = torch.full((1, L + P), math.nan)
            if fmt != "i8":
                x[:, 1::2] = math.inf
            pool.put(b, t, x)
    got = pool.cuda(ctx=ctx).attend_window(*args)
    ctx.synchronize()
    some = 0
    for b, n in enumerate(lens):
        for j in range(M):
            at = set(R8.positions(n - M + j + 1, window, sinks).tolist())
            if at & set(odd[b]):
                assert not torch.isfinite(got[b, j]).any()
            else:
                assert torch.equal(got[b, j], clean[b, j])
                some += 1
    assert some


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("H,L,P", [(128, 512, 64), (16, 512, 64), (4, 64, 16)])
def test_a_window_that_holds_everything_is_attention(ctx, fmt, H, L, P):
    """Windows and first positions up to the widest numbers."""
    pool = R8.pool(fmt, 7, [300, 64, 0, 7], 16, L, P)
    qabs, qrope = [t.cuda() for t in pool.queries(2, H)]
    cache, args = pool.cuda(ctx=ctx), (pool.table.cuda(), pool.lens32().cuda(), qabs, qrope, SCALE)
    for window, sinks in ((300, 0), (2**31 - 1, 0), (2**62, 2**62), (1, 2**40)):
        out = cache.attend_window(*args, window, sinks)
        ctx.synchronize()
        R8.check(pool, fmt, out, qabs, qrope, SCALE)


def test_a_bad_page_in_the_window_is_reported(ctx):
    import undertow_amd as U
    pool = R8.pool("bf16", 9, [300, 300, 300], 16, 512, 64)
    qabs, qrope = [t.cuda() for t in pool.queries(1, 16)]
    table = pool.table.clone()
    table[:, 2:15] = -1  # neither first positions nor the window's
    cache, lens = pool.cuda(ctx=ctx), pool.lens32().cuda()
    want = cache.attend_window(table.cuda(), lens, qabs, qrope, SCALE, 50, 20)
    ctx.synchronize()
    table[1, 16] = pool.n_pages
    got = cache.attend_window(table.cuda(), lens, qabs, qrope, SCALE, 50, 20)
    with pytest.raises(U.UtError) as e:
        ctx.synchronize()
    assert e.value.code == U.runtime.UT_ERR_BAD_PAGE
    assert torch.equal(got[::2], want[::2])


def test_a_captured_window_slides(ctx):
    """One call captured, replayed as the lengths grow past the window and
    tables give pages back: every replay has the eager call's bits."""
    import undertow_amd as U
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c = U.Context(0)
        pool = R8.pool("bf16", 15, [900, 400, 650], 16, 512, 64)
        qabs, qrope = [t.cuda() for t in pool.queries(2, 128)]
        cache, table = pool.cuda(ctx=c), pool.table.cuda()
        lens = torch.tensor([30, 1, 200], dtype=torch.int32, device="cuda")
        call = lambda: cache.attend_window(table, lens, qabs, qrope, SCALE, 128, 4)
        call()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = call()
        for k in range(5):
            lens += 77
            for b, n in enumerate(lens.tolist()):
                table[b, 1:max(1, (n - 1 - 128) // 16)] = -1
            got.zero_()
            graph.replay()
            s.synchronize()
            first, want = got.clone(), call()
            c.synchronize()
            assert torch.equal(first, want)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("H", [16, 50, 128])
@pytest.mark.parametrize("window", [None, 60])
def test_prompt_rows_end_where_each_does(ctx, fmt, H, window):
    """Rows of a prompt before a value that is not finite have the bits that
    they have without it, and are right; rows from it on are not finite."""
    lens, M = [390, 70, 300], 300
    pool = R8.pool(fmt, 43, lens, 64, 512, 64, 128)
    qabs, qrope = pool.queries(M, H)
    args = pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE

    def run():
        cache = pool.cuda(ctx=ctx)
        got = cache.attend(*args) if window is None else cache.attend_window(*args, window, 3)
        ctx.synchronize()
        return got

    good = run()
    R8.check(pool, fmt, good, qabs, qrope, SCALE, window=window, sinks=3 if window else 0)
    for b, n in enumerate(lens):
        at = pool.where(b, torch.tensor([n - 33]))
        (pool.scales if fmt == "i8" else pool.pages)[at] = math.nan
    bad = run()
    assert torch.equal(bad[:, :M - 33], good[:, :M - 33])
    assert bad[:, M - 33:].isnan().any(-1).all()
