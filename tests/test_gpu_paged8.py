"""The paged latent cache in 8 bits on the GPU against 64 bits: append and
summaries, rows read back, attention over all and over listed pages, and a run
of them together.  Tolerances stand at paged8_ref.close."""
import math

import pytest
import torch

import paged8_ref as R8
import paged_ref as R
from test_gpu_paged import SCALE

pytestmark = pytest.mark.gpu


def attend_case(ctx, lens, M, H, L=512, P=64, page=64, width=None, seed=1, spread=None):
    pool = R8.Pool8(seed, lens, page, L, P, width)
    if spread is not None:  # positions of very different sizes
        for b, n in enumerate(lens):
            x = pool.randn(n, L + P)
            x[:, :L] *= torch.exp2(torch.randint(-spread, spread + 1, (n, 1), generator=pool.g))
            pool.put(b, 0, x)
    qabs, qrope = pool.queries(M, H)
    if spread is not None:
        qabs *= 2.0 ** -spread
    got = pool.cuda(ctx=ctx).attend(pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE)
    ctx.synchronize()
    R8.check(pool, "i8", got, qabs, qrope, SCALE)
    return pool, qabs, qrope, got


# ------------------------------------------------------------- attention
@pytest.mark.parametrize("lens,M,H,page", [
    ([1], 1, 128, 64), ([2, 0, 1], 1, 128, 16), ([31, 32, 33, 63, 64, 65], 1, 128, 64),
    ([500], 1, 128, 64), ([130, 1, 0, 77], 4, 128, 32), ([3, 2, 1, 0, 64, 65, 66], 3, 32, 64),
    ([257, 3, 600], 2, 64, 128), ([100, 31, 1001], 1, 16, 16), ([40, 1, 129], 2, 16, 8),
    ([333, 12], 1, 20, 64), ([90], 3, 1, 32), ([200, 45, 5], 1, 96, 256), ([70, 12, 0, 9], 2, 48, 1),
    ([1500, 9, 1], 1, 128, 1024), ([260, 140, 33], 1, 160, 64), ([21, 40], 1, 32, 4)])
def test_attend(ctx, lens, M, H, page):
    attend_case(ctx, lens, M, H, page=page)


@pytest.mark.parametrize("lens,M,H,L,P,page", [
    ([1, 0, 40, 65], 1, 4, 64, 16, 16), ([17, 64, 130], 3, 4, 64, 16, 64), ([33, 5], 2, 8, 16, 8, 4),
    ([100], 1, 3, 1000, 24, 32), ([60, 3], 1, 2, 512, 128, 16), ([5000, 0, 70], 1, 5, 136, 8, 64)])
def test_attend_other_widths(ctx, lens, M, H, L, P, page):
    attend_case(ctx, lens, M, H, L, P, page)


@pytest.mark.parametrize("lens,M,H,width", [
    ([9001], 1, 128, None), ([5000, 17, 3000], 2, 128, None), ([6001] * 5, 1, 16, None), ([4000, 0, 2000, 1], 1, 64, None),
    ([12000], 4, 32, None), ([1, 0, 33, 64, 100, 0], 2, 32, 9000), ([40], 1, 128, 9000), ([5, 90, 31] * 30, 1, 16, 9000),
    ([(37 * k) % 90 for k in range(700)], 1, 16, None), ([2000] + [100] * 70, 1, 128, 8192)])
def test_attend_cut_into_ranges(ctx, lens, M, H, width):
    attend_case(ctx, lens, M, H, width=None if width is None else width // 64)


@pytest.mark.parametrize("units", [1, 2, 3, 4])
@pytest.mark.parametrize("M,H", [(1, 16), (1, 50), (1, 64), (2, 16), (1, 128), (2, 128)])
def test_attend_of_a_few_long_sequences(ctx, units, M, H):
    attend_case(ctx, [7001, 3100, 9, 5000][:units], M, H)


@pytest.mark.parametrize("units", [60, 200, 600])  # each is found in another way
@pytest.mark.parametrize("kind", ["all", "window", "listed"])
def test_attend_of_many_sequences_in_a_wide_table(ctx, units, kind):
    M = 1 if kind != "listed" else 2
    lens = [(97 * k) % 331 if k % 7 else 0 for k in range(units // M)]
    pool = R8.Pool8(17, lens, 64, 512, 64, 128)
    qabs, qrope = pool.queries(M, 16)
    where = pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE
    cache, more = pool.cuda(ctx=ctx), {}
    if kind == "all":
        got = cache.attend(*where)
    elif kind == "window":
        more = dict(window=150, sinks=33)
        got = cache.attend_window(*where, **more)
    else:
        sel = torch.stack([torch.randperm(8, generator=pool.g)[:5] - 1 for _ in range(units)]).int().view(-1, M, 5)
        # places that lists are seldom filled to
        more = dict(sel=torch.cat([sel, torch.full((len(lens), M, 35), -1, dtype=torch.int32)], -1))
        got = cache.attend_pages(*where, more["sel"].cuda())
    ctx.synchronize()
    R8.check(pool, "i8", got, qabs, qrope, SCALE, **more)


@pytest.mark.parametrize("lens,M,H,width", [
    ([600, 40, 333], 128, 256, 4096), ([700], 300, 128, 8192), ([1500, 700], 40, 128, 2048), ([140, 200], 140, 16, 300)])
def test_attend_prompt_rows(ctx, lens, M, H, width):
    attend_case(ctx, lens, M, H, width=width // 64)


@pytest.mark.parametrize("lens", [[300, 64, 5], [5000, 64]])
@pytest.mark.parametrize("H,L,P,spread", [(128, 512, 64, 3), (16, 512, 64, 12), (128, 512, 64, 20), (4, 64, 16, 12)])
def test_attend_positions_of_very_different_sizes(ctx, lens, H, L, P, spread):
    """Scales up to 2^40 apart: a large position of small weight does not
    drown the small ones that have it, nor the other way round."""
    attend_case(ctx, lens, 2, H, L, P, spread=spread)


@pytest.mark.parametrize("lens", [[300, 40], [6000, 700, 3]])  # whole, and cut into ranges
@pytest.mark.parametrize("size", [-100, -60, 60, 100])
@pytest.mark.parametrize("H,L,P", [(128, 512, 64), (4, 64, 16)])
def test_attend_tiny_and_huge_values(ctx, lens, size, H, L, P):
    """Latent values of 2^size and queries of 2^-size: the context has the
    values' size whatever that is."""
    pool = R8.Pool8(41, lens, 64, L, P)
    for b, n in enumerate(lens):
        x = pool.randn(n, L + P)
        x[:, :L] *= 2.0 ** size
        pool.put(b, 0, x)
    qabs, qrope = pool.queries(1, H)
    qabs *= 2.0 ** -size
    got = pool.cuda(ctx=ctx).attend(pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE)
    ctx.synchronize()
    # tolerances relative to the values' size: everything is taken times 2^-size
    for b, n in enumerate(lens):
        kv = pool.rows(b, torch.arange(n)).cuda()
        q = torch.cat([qabs[b, 0], qrope[b, 0]], -1).double().cuda()
        out, spread, mass = R.attend(kv, q, L, SCALE)
        down = 2.0 ** -size
        R8.close("i8", (got[b, 0].double() * down), out * down, spread * down, mass * down,
                 R8.score_step(kv, q, L, SCALE)[:, None].cpu(), R8.largest(kv, q, L, SCALE).cpu() * down)


@pytest.mark.parametrize("H,L,P", [(128, 512, 64), (16, 512, 64), (4, 64, 16)])
def test_attend_extreme_scores(ctx, H, L, P):
    """Queries whose scores reach hundreds, queries of zeros, tiny and huge ones."""
    pool = R8.Pool8(5, [300, 77], 64, L, P)
    qabs, qrope = pool.queries(2, H)
    qabs[0, 0] *= 30.0
    qrope[0, 1] *= 100.0
    qabs[1, 0], qrope[1, 0, :, 1:] = 0.0, 0.0
    qabs[1, 1, ::2] *= 1e-30
    qrope[1, 1, 1::2] *= 1e-37
    got = pool.cuda(ctx=ctx).attend(pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE)
    ctx.synchronize()
    for b, n in enumerate(pool.lens):
        for j in range(2):
            kv = pool.rows(b, torch.arange(n - 1 + j))
            q = torch.cat([qabs[b, j], qrope[b, j]], -1).double()
            want, spread, mass = R.attend(kv, q, L, SCALE)
            # f32 scores of size s carry s 2^-23 or so, beside the queries' steps
            size = (q @ kv.T * SCALE).abs().max()
            step = R8.score_step(kv, q, L, SCALE)[:, None] + float(size) * 2.0 ** -21
            R8.close("i8", got[b, j], want, spread, mass, step, R8.largest(kv, q, L, SCALE))


@pytest.mark.parametrize("H,L,P", [(128, 512, 64), (16, 512, 64), (4, 64, 16)])
def test_what_a_row_does_not_see_does_not_reach_it(ctx, H, L, P):
    """NaN at the last position: its row is NaN, the rows before it are as
    without; a query that is not finite makes its head's context NaN alone."""
    pool = R8.Pool8(3, [97, 64, 130], 32, L, P)
    qabs, qrope = pool.queries(3, H)
    args = pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda()
    clean = pool.cuda(ctx=ctx).attend(*args, SCALE)
    for b, n in enumerate(pool.lens):
        x = torch.full((1, L + P), 0.5)
        x[0, 3 if b else L + 3] = math.inf if b == 1 else math.nan
        pool.put(b, n - 1, x)
    got = pool.cuda(ctx=ctx).attend(*args, SCALE)
    assert torch.equal(got[:, :-1], clean[:, :-1])
    assert not torch.isfinite(got[:, -1]).any()
    qabs[0, 0, 1, 7], qrope[0, 1, 2, 3] = math.nan, math.inf
    odd = pool.cuda(ctx=ctx).attend(*args[:2], qabs.cuda(), qrope.cuda(), SCALE)
    assert not torch.isfinite(odd[0, 0, 1]).any() and not torch.isfinite(odd[0, 1, 2]).any()
    odd[0, 0, 1], odd[0, 1, 2] = got[0, 0, 1], got[0, 1, 2]
    assert torch.equal(odd[:, :-1], got[:, :-1])


@pytest.mark.parametrize("lens,M,H,page,top_k", [
    ([500, 33, 0], 1, 128, 64, 4), ([130, 90], 2, 16, 16, 6), ([3000, 2000, 5], 2, 128, 64, 20), ([70, 65], 1, 128, 8, 9),
    ([200], 3, 20, 32, 12), ([300, 41], 2, 64, 128, 2)])
@pytest.mark.parametrize("L,P", [(512, 64), (64, 16)])
def test_attend_listed_pages(ctx, lens, M, H, page, top_k, L, P):
    pool = R8.Pool8(11, lens, page, L, P)
    B, W = pool.table.shape
    qabs, qrope = pool.queries(M, H)
    sel = torch.full((B, M, top_k), -1, dtype=torch.int32)
    for b in range(B):
        for j in range(M):
            ids = torch.randperm(W + 2, generator=pool.g)[:top_k] - 1  # any order, some behind the end, -1 among them
            sel[b, j, :len(ids)] = ids.int()
    table = pool.table.clone()
    got = pool.cuda(ctx=ctx).attend_pages(table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE, sel.cuda())
    ctx.synchronize()
    R8.check(pool, "i8", got, qabs, qrope, SCALE, sel=sel)


def test_select_takes_the_summaries_alone(ctx):
    """A selection over 8-bit pages is the one over bf16 pages of the same summaries."""
    import undertow_amd as U
    pool = R8.Pool8(13, [900, 33, 0, 500], 16, 512, 64)
    for b in range(4):
        pool.table[b, -(-pool.lens[b] // 16):] = -1
    mean = torch.randint(-127, 128, (pool.n_pages, 576), generator=pool.g).to(torch.int8).cuda()
    scale = torch.rand(pool.n_pages, generator=pool.g).cuda()
    qabs, qrope = [t.cuda() for t in pool.queries(2, 128)]
    args = pool.table.cuda(), pool.lens32().cuda(), qabs, qrope, 9
    want = U.PagedCache(ctx, torch.zeros(pool.pages.shape, dtype=torch.bfloat16, device="cuda"), mean=mean, mean_scale=scale).select(*args)
    assert torch.equal(pool.cuda(ctx=ctx, mean=mean, mean_scale=scale).select(*args), want)
    assert (want[0] >= 0).all()


# ---------------------------------------------------------------- append
def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("lens,M,L,P,page,summaries", [
    ([1], 1, 512, 64, 64, True), ([64, 65, 1, 300], 1, 512, 64, 64, True), ([130, 0, 17, 3], 4, 512, 64, 16, True),
    ([777, 900], 700, 512, 64, 64, True), ([40, 41], 3, 64, 16, 8, True), ([9, 30], 5, 1000, 24, 1, True),
    ([100, 2000], 90, 16, 8, 1024, True), ([50, 0, 3], 8, 512, 64, 32, False), ([33, 70], 2, 8, 1016, 16, True)])
def test_append(ctx, lens, M, L, P, page, summaries):
    """Codes, scales and summaries are the definition's to the bit; every
    other row and summary is as it was."""
    pool = R8.Pool8(17, lens, page, L, P)
    B = len(lens)
    x = pool.randn(B, M, L + P)
    x[:, M // 2, :L] = 0.0  # a part of zeros
    # quotients halfway between codes: half to even
    x[:, 0, :8] = torch.tensor([127.0, 0.5, 1.5, -2.5, -0.5, 126.5, 63.5, -126.5])
    x[:, 0, 8:L].clamp_(-3.0, 3.0)
    x[:, -1] *= torch.exp2(torch.randint(-60, 60, (B, 1), generator=pool.g))
    g = torch.Generator().manual_seed(2)
    mean = torch.randint(-127, 128, (pool.n_pages, L + P), generator=g).to(torch.int8)
    mean_scale = torch.rand(pool.n_pages, generator=g)
    cache = pool.cuda(ctx=ctx, **(dict(mean=mean.cuda(), mean_scale=mean_scale.cuda()) if summaries else {}))
    cache.append(pool.table.cuda(), pool.lens32().cuda(), x[..., :L].contiguous().cuda(), x[..., L:].contiguous().cuda())
    ctx.synchronize()
    for b, n in enumerate(lens):
        new = min(M, n)
        if not new:
            continue
        pool.put(b, n - new, x[b, M - new:])
        for k in range((n - new) // page, (n - 1) // page + 1):
            p = int(pool.table[b, k])
            mean[p], mean_scale[p] = R.summary(pool.rows(b, torch.arange(k * page, min(n, (k + 1) * page))))
    assert torch.equal(cache.pages.cpu(), pool.pages) and same_bits(cache.scales.cpu(), pool.scales)
    if summaries:
        assert torch.equal(cache.mean.cpu(), mean) and torch.equal(cache.mean_scale.cpu(), mean_scale)


def test_append_of_values_that_are_not_finite(ctx):
    """A part with NaN or an infinity is NaN read back, the other part of its
    row is not touched by that; subnormal and huge rows keep their values."""
    pool = R8.Pool8(19, [7], 16, 512, 64)
    x = pool.randn(1, 7, 576)
    x[0, 0, 5], x[0, 1, 520], x[0, 2, 500] = math.nan, math.inf, -math.inf
    x[0, 3] *= 5e37
    x[0, 4] *= 1e-42
    x[0, 5, :512] = 0.0
    cache = pool.cuda(ctx=ctx)
    cache.append(pool.table.cuda(), pool.lens32().cuda(), x[..., :512].contiguous().cuda(), x[..., 512:].contiguous().cuda())
    lat, kr = cache.read(pool.table.cuda(), pool.lens32().cuda(), 7)
    ctx.synchronize()
    pool.put(0, 0, x[0])
    want = pool.rows(0, torch.arange(7)).float()
    got = torch.cat([lat, kr], -1)[0].cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    assert got[0, :512].isnan().all() and got[1, 512:].isnan().all() and got[2, :512].isnan().all()
    assert got[0, 512:].isfinite().all() and got[1, :512].isfinite().all() and got[3:].isfinite().all()


# ------------------------------------------------------------------ read
@pytest.mark.parametrize("fmt", ["i8", "bf16", "f16x2"])
@pytest.mark.parametrize("lens,rows,starts,L,P,page", [
    ([1], 1, None, 512, 64, 64), ([64, 0, 65, 300], 70, None, 512, 64, 64), ([130, 17, 3], 40, [100, -5, 2], 512, 64, 16),
    ([40, 41], 3, [40, 39], 64, 16, 8), ([30, 9], 5, [-(2**31), 2**31 - 1], 1000, 24, 1), ([2000], 1999, [1], 16, 8, 1024),
    ([33, 70], 45, [1, 30], 8, 1016, 16)])
@pytest.mark.parametrize("bf16", [False, True])
def test_read(ctx, fmt, lens, rows, starts, L, P, page, bf16):
    """Every row that there is to the bit, zeros for those that there are not."""
    pool = R8.pool(fmt, 23, lens, page, L, P)
    t = torch.bfloat16 if bf16 else torch.float32
    s = None if starts is None else torch.tensor(starts, dtype=torch.int32)
    out = (torch.full((len(lens), rows, L), math.nan, dtype=t, device="cuda"),
           torch.full((len(lens), rows, P), math.nan, dtype=t, device="cuda"))
    got = pool.cuda(ctx=ctx).read(pool.table.cuda(), pool.lens32().cuda(), rows, starts=None if s is None else s.cuda(), dtype=t, out=out)
    ctx.synchronize()
    assert got[0] is out[0] and got[1] is out[1]
    got = torch.cat(got, -1).cpu()
    for b, n in enumerate(lens):
        at = torch.arange(rows) + (0 if s is None else int(s[b]))
        there = (at >= 0) & (at < n)
        want = torch.zeros((rows, L + P))
        if there.any():
            want[there] = pool.rows(b, at[there]).float()
        assert torch.equal(got[b], want.to(t))


def test_read_writes_its_rows_alone(ctx):
    """Behind the last row of the outputs nothing is written."""
    pool = R8.Pool8(29, [50, 20], 16, 512, 64)
    buf = [torch.full((2 * 13 * w + 64,), 7.0, device="cuda") for w in (512, 64)]
    pool.cuda(ctx=ctx).read(pool.table.cuda(), pool.lens32().cuda(), 13,
                            out=[x[:2 * 13 * w].view(2, 13, w) for x, w in zip(buf, (512, 64))])
    ctx.synchronize()
    assert all((x[-64:] == 7.0).all() for x in buf)


def test_read_of_more_than_the_caches_hold(ctx):
    """Rows that go past the L2s: the bits that they have a few at a time."""
    pool = R8.Pool8(41, [4300, 17, 4100, 2500], 64, 512, 64)
    cache, table, lens = pool.cuda(ctx=ctx), pool.table.cuda(), pool.lens32().cuda()
    for t in (torch.float32, torch.bfloat16):
        rows = 4200 if t == torch.float32 else 8400
        assert 4 * rows * 576 * t.itemsize > 2**25
        got = torch.cat(cache.read(table, lens, rows, dtype=t), -1)
        for at in range(0, rows, 1400):
            few = cache.read(table, lens, 1400, starts=torch.full((4,), at, dtype=torch.int32, device="cuda"), dtype=t)
            ctx.synchronize()
            assert torch.equal(got[:, at:at + 1400], torch.cat(few, -1))
        assert torch.equal(got[1, :17].cpu(), pool.rows(1, torch.arange(17)).float().to(t))


def test_positions_far_into_a_pool(ctx):
    """Pages beyond 2^32 bytes: the bits that the same rows have in a small pool."""
    import undertow_amd as U
    g = torch.Generator(device="cuda").manual_seed(5)
    rnd = lambda *d: torch.randn(d, device="cuda", generator=g)
    n, page, far = 700, 64, 2**33 // (64 * 576) + 30
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    new, q = (rnd(1, n, 512), rnd(1, n, 64)), (rnd(1, 2, 32, 512).bfloat16(), rnd(1, 2, 32, 64).bfloat16())
    sel = torch.tensor([[[0, 9, 3], [10, 2, 1]]], dtype=torch.int32, device="cuda")
    got = []
    for pages, first in ((30, 0), (far, far - 30)):
        cache = U.PagedCache.empty(ctx, pages, page, fmt=U.KV_I8)
        table = (first + 29 - torch.arange(11, dtype=torch.int32, device="cuda"))[None].contiguous()
        cache.append(table, lens, *new)
        got.append((*cache.read(table, lens, n), cache.attend(table, lens, *q, SCALE), cache.attend_pages(table, lens, *q, SCALE, sel),
                    cache.attend_window(table, lens, *q, SCALE, 100, 5), cache.mean[table[0].long()], cache.mean_scale[table[0].long()]))
        ctx.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert torch.equal(got[0][0][0].cpu(), R8.values8(*R8.quantised(torch.cat(new, -1)[0].cpu(), 512), 512)[:, :512].float())


# ------------------------------------------------- errors, streams, runs
@pytest.mark.parametrize("bad_page", [False, True])
def test_bad_lengths_and_pages_are_reported(ctx, bad_page):
    import undertow_amd as U
    pool = R8.Pool8(31, [100, 90, 80], 16, 512, 64, width=7)
    qabs, qrope = [t.cuda() for t in pool.queries(1, 16)]
    cache, lens, table = pool.cuda(ctx=ctx), pool.lens32().cuda(), pool.table.cuda()
    good = cache.read(table, lens, 80)
    ctx.synchronize()
    if bad_page:
        table[1, 4] = pool.n_pages
    else:
        lens[1] = -4
    lat, kr = pool.randn(3, 40, 512).cuda(), pool.randn(3, 40, 64).cuda()
    before = cache.pages.clone(), cache.scales.clone()
    for f in (lambda: [cache.attend(table, lens, qabs, qrope, SCALE)], lambda: cache.read(table, lens, 80),
              lambda: cache.append(table, lens, lat, kr)):
        got = f()
        with pytest.raises(U.UtError) as e:
            ctx.synchronize()
        assert e.value.code == U.runtime.UT_ERR_BAD_PAGE
        # the other sequences are as they should be: rows read back to the bit; contexts,
        # whose sums a length may cut elsewhere, in their tolerance
        if got and len(got) == 1:
            R8.check(pool, "i8", got[0], qabs.cpu(), qrope.cpu(), SCALE, only=(0, 2))
        elif got:
            assert all(torch.equal(a[::2], b[::2]) for a, b in zip(got, good))
    for b in (0, 2):
        n = pool.lens[b]
        at = tuple(t.cuda() for t in pool.where(b, torch.arange(n - 40, n)))
        c, s = R8.quantised(torch.cat([lat, kr], -1)[b].cpu(), 512)
        before[0][at], before[1][at] = c.cuda(), s.cuda()
    if not bad_page:
        assert torch.equal(cache.pages, before[0]) and same_bits(cache.scales, before[1])
    ctx.synchronize()


def test_refusals(ctx):
    """What the library itself turns down, before anything is launched."""
    import ctypes as C

    import undertow_amd as U
    lib, rt = U.lib(), U.runtime
    pages, scales = torch.zeros((4, 16, 576), dtype=torch.int8, device="cuda"), torch.zeros((4, 16, 2), device="cuda")
    table, lens = torch.zeros((2, 4), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    p = torch.zeros((2, 1, 16, 576), device="cuda").data_ptr()
    arg, shape = rt.UT_ERR_ARG, rt.UT_ERR_SHAPE

    def kv(**k):
        d = dict(pages=pages.data_ptr(), n_pages=4, page=16, latent=512, rope=64, fmt=U.KV_I8, scales=scales.data_ptr())
        return C.byref(rt.MlaPages(**{**d, **k}))

    def calls(cache, M=1, H=16, q=p, o=p):
        b = ctx.handle, cache, table.data_ptr(), 4, 4, lens.data_ptr(), 2, M
        yield lib.ut_mla_paged_attend(*b, H, q, p, 0.1, o)
        yield lib.ut_mla_window_attend(*b, H, q, p, 0.1, 5, 1, o)
        yield lib.ut_mla_sparse_attend(*b, H, q, p, 0.1, p, 2, o)
        yield lib.ut_mla_paged_append(*b, q, o)
        yield lib.ut_mla_paged_read(*b, None, rt.ROWS_F32, q, o)

    for k in (dict(scales=None), dict(scales=scales.data_ptr() + 8), dict(pages=None), dict(fmt=3), dict(n_pages=0)):
        assert all(c == arg for c in calls(kv(**k))), k
    for k in (dict(q=None), dict(o=None), dict(q=p + 4), dict(M=0)):
        assert all(c == arg for c in calls(kv(), **k)), k
    for k in (dict(page=24), dict(latent=508), dict(rope=1024)):
        assert all(c == shape for c in calls(kv(**k))), k
    b = ctx.handle, kv(), table.data_ptr(), 4, 4, lens.data_ptr(), 2, 1
    for window, sinks in ((0, 1), (-1, 0), (5, -1), (-(2**63), 0), (4, -(2**63))):
        assert lib.ut_mla_window_attend(*b, 16, p, p, 0.1, window, sinks, p) == arg
    for t in (2, -1):
        assert lib.ut_mla_paged_read(*b, None, t, p, p) == arg
    one = ctx.handle, kv(page=1), table.data_ptr(), 4, 4, lens.data_ptr(), 1, 2**31 - 1
    assert lib.ut_mla_paged_read(*one, None, 0, p, p) == shape
    ctx.synchronize()


@pytest.mark.parametrize("H,L,P", [(128, 512, 64), (16, 512, 64), (4, 64, 16)])
def test_captured_steps_follow_lengths(ctx, H, L, P):
    """One step captured (append, selection, attention over it, over all and
    in a window, the rows read back), replayed as the lengths grow with eager
    calls between: every replay gives the eager call's bits."""
    import undertow_amd as U
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c = U.Context(0)
        g = torch.Generator(device="cuda").manual_seed(3)
        rnd = lambda *d: torch.randn(d, device="cuda", generator=g)
        B, M = 3, 2
        cache = U.PagedCache.empty(c, 60, page=16, latent=L, rope=P, fmt=U.KV_I8)
        table = torch.arange(60, dtype=torch.int32, device="cuda").reshape(3, 20)
        lens = torch.tensor([150, 17, 31], dtype=torch.int32, device="cuda")
        starts = torch.tensor([140, 0, 29], dtype=torch.int32, device="cuda")
        cache.append(table, lens, rnd(B, 150, L), rnd(B, 150, P))
        lat, kr = rnd(B, M, L), rnd(B, M, P)
        q = rnd(B, M, H, L).bfloat16(), rnd(B, M, H, P).bfloat16()

        def step():
            cache.append(table, lens, lat, kr)
            sel = cache.select(table, lens, *q, 3, 1, 1)
            return (sel, cache.attend_pages(table, lens, *q, SCALE, sel), cache.attend(table, lens, *q, SCALE),
                    cache.attend_window(table, lens, *q, SCALE, 37, 3), *cache.read(table, lens, 12, starts))

        lens += M
        step()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = step()
        for k in range(4):
            lens += M
            starts += 1
            lat.copy_(rnd(B, M, L))
            for t in got:
                t.zero_()
            graph.replay()
            s.synchronize()
            first, pages = [t.clone() for t in got], cache.pages.clone()
            want = step()  # writes the same rows again
            assert all(torch.equal(a, b) for a, b in zip(first, want))
            assert torch.equal(pages, cache.pages)
            cache.attend(table[:1].expand(64, 20).contiguous(), lens[:1].expand(64).contiguous(), rnd(64, 1, H, L).bfloat16(),
                         rnd(64, 1, H, P).bfloat16(), SCALE)
            c.synchronize()


def test_two_contexts_at_once(ctx):
    """Two contexts on streams of their own over one pool: the bits of their calls alone."""
    import undertow_amd as U
    pool = R8.Pool8(37, [900, 333, 12], 32, 512, 64)
    qabs, qrope = [t.cuda() for t in pool.queries(2, 128)]
    cache, table, lens = pool.cuda(ctx=ctx), pool.table.cuda(), pool.lens32().cuda()
    want = cache.attend(table, lens, qabs, qrope, SCALE), cache.attend_window(table, lens, qabs, qrope, SCALE, 100, 4)
    torch.cuda.synchronize()
    runs = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            runs.append((s, U.PagedCache(U.Context(0), cache.pages, scales=cache.scales)))
    outs = []
    for _ in range(5):
        for s, c in runs:
            with torch.cuda.stream(s):
                outs.append((c.attend(table, lens, qabs, qrope, SCALE), c.attend_window(table, lens, qabs, qrope, SCALE, 100, 4)))
    for s, c in runs:
        c.ctx.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))


@pytest.mark.parametrize("H,L,P", [(128, 512, 64), (16, 512, 64), (4, 64, 16)])
def test_a_serving_run(ctx, H, L, P):
    """Prompts and steps, a rejected draft among them: what is read back is
    what attention sees, and the contiguous cache's attention over the rows
    read back agrees with it; so does a window that holds everything, and a
    move of the sequences to f16 pairs by reading and appending."""
    import undertow_amd as U
    g = torch.Generator(device="cuda").manual_seed(H)
    rnd = lambda *d: torch.randn(d, device="cuda", generator=g)
    B, page = 3, 16
    cache = U.PagedCache.empty(ctx, 64, page, L, P, U.KV_I8)
    pairs = U.PagedCache.empty(ctx, 64, page, L, P, U.KV_F16X2)
    table = torch.randperm(64, device="cuda", generator=g)[:60].reshape(B, 20).int()
    n = [0] * B
    for M in (100, 2, -1, 1, 3, 60):
        if M < 0:  # the last row of each was a wrong draft
            n = [a - 1 for a in n]
            continue
        n = [a + M - (7 * b if M == 100 else 0) for b, a in enumerate(n)]
        lens = torch.tensor(n, dtype=torch.int32, device="cuda")
        new = rnd(B, M, L + P)
        cache.append(table, lens, new[..., :L].contiguous(), new[..., L:].contiguous())
        R_ = min(M, 3)
        q = rnd(B, R_, H, L + P).bfloat16()
        qa, qr = q[..., :L].contiguous(), q[..., L:].contiguous()
        got = cache.attend(table, lens, qa, qr, SCALE)
        every = cache.attend_pages(table, lens, qa, qr, SCALE, cache.select(table, lens, qa, qr, 20, 1, 1))
        wide = cache.attend_window(table, lens, qa, qr, SCALE, 320, 2)
        near = cache.attend_window(table, lens, qa, qr, SCALE, 33, 2)
        lat, kr = cache.read(table, lens, max(n))
        pairs.append(table, lens, *cache.read(table, lens, max(n), starts=lens - max(n)))
        moved = pairs.attend(table, lens, qa.float(), qr.float(), SCALE)
        moved_near = pairs.attend_window(table, lens, qa.float(), qr.float(), SCALE, 33, 2)
        ctx.synchronize()
        for b in range(B):
            want = U.mla_attend(ctx, qa[b].float().contiguous(), qr[b].float().contiguous(), lat[b, :n[b]].contiguous(),
                                kr[b, :n[b]].contiguous(), n[b] - R_, SCALE)
            # weights to 2^-11, outputs to 2^-8, the contiguous cache's products to 1e-4 of the largest
            bar = (2.0 ** -8 + 2.0 ** -11 + 3e-4) * max(1.0, float(want.abs().max()))
            for x in (got, every, wide, moved):
                assert float((x[b].float() - want).abs().max()) <= bar
            assert float((near[b].float() - moved_near[b]).abs().max()) <= bar + 2.0 ** -8 * float(near[b].abs().max())
