"""The paged latent cache on the GPU against 64 bits: append and page
summaries, attention over ragged batches, page selection, attention over
selected pages, and a run of them together.

Tolerances.  bf16: an output is rounded once (half a step, 2^-8 of it at
most), and a softmax weight once in numerator and denominator alike, which
moves the context by at most 2^-8 sum_t p_t |v_t - out|; what is left is f32
arithmetic.  f16x2: stored values and queries keep 22 bits, the products of
two low parts are left out (2^-22 of a product), and sums run in f32 over
36 (scores) or T/16 (contexts) blocks: with |q k| summing to at most about 30
after scaling, a score is off by 30 (2^-21 + 6 2^-24) = 2.6e-5 at the very
most, a weight by twice that, and the context by that times its spread."""
import math

import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu
SCALE = 1.0 / math.sqrt(192.0)


def close(fmt, got, want, spread, mass):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    err = (got - want).abs()
    if fmt == "bf16":
        tol = 2.0 ** -8 * (want.abs() + spread) + 6e-5 * spread + 2.0 ** -20 * mass + 1e-30
    else:
        tol = 5.2e-5 * spread + 2.0 ** -20 * (mass + want.abs()) + 1e-30
    assert (err <= tol).all(), float((err / tol).max())


def reference(pool, qabs, qrope, scale=SCALE, sel=None):
    """(out, spread, mass), each [B, M, H, L]."""
    B, M, H, L = qabs.shape
    q = torch.cat([qabs, qrope], -1).double()
    parts = []
    for b, n in enumerate(pool.lens):
        for j, s in enumerate(R.seen(n, M)):
            pos = torch.arange(s)
            if sel is not None:
                pos = torch.cat([torch.arange(k * pool.page, (k + 1) * pool.page)
                                 for k in sel[b, j].tolist() if k >= 0] + [torch.zeros(0, dtype=torch.long)])
                pos = pos[pos < s]
            parts.append(R.attend(pool.rows(b, pos), q[b, j], L, scale))
    return [torch.stack([p[i] for p in parts]).reshape(B, M, H, L) for i in range(3)]


def attend_case(ctx, fmt, lens, M, H, L, P, page, seed=1, width=None):
    pool = R.Pool(seed, fmt, lens, page, L, P, width)
    qabs, qrope = pool.queries(M, H)
    cache = pool.cuda(ctx=ctx)
    got = cache.attend(pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE)
    ctx.synchronize()
    want = reference(pool, qabs, qrope)
    close(fmt, got, *want)
    for b, n in enumerate(lens):
        for j, s in enumerate(R.seen(n, M)):
            if s == 0:
                assert (got[b, j] == 0).all()
    return pool, cache, qabs, qrope, got


FMTS = ["bf16", "f16x2"]


# ------------------------------------------------------------- attention
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,H,page", [
    ([1], 1, 128, 64), ([2, 0, 1], 1, 128, 16), ([31, 32, 33, 63, 64, 65], 1, 128, 64),
    ([500], 1, 128, 64), ([130, 1, 0, 77], 4, 128, 32), ([3, 2, 1, 0, 64, 65, 66], 3, 32, 64),
    ([257, 3, 600], 2, 64, 128), ([100, 31, 1001], 1, 16, 16), ([40, 1, 129], 2, 16, 8),
    ([333, 12], 1, 20, 64), ([90], 3, 1, 32), ([200, 45, 5], 1, 96, 256), ([70, 12, 0, 9], 2, 48, 1),
    ([1500, 9, 1], 1, 128, 1024), ([260, 140, 33], 1, 160, 64)])
def test_attend(ctx, fmt, lens, M, H, page):
    attend_case(ctx, fmt, lens, M, H, 512, 64, page)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,H,L,P,page", [
    ([1, 0, 40, 65], 1, 4, 64, 16, 16), ([17, 64, 130], 3, 4, 64, 16, 64), ([33, 5], 2, 8, 16, 8, 4),
    ([100], 1, 3, 1000, 24, 32), ([60, 3], 1, 2, 512, 128, 16)])
def test_attend_other_widths(ctx, fmt, lens, M, H, L, P, page):
    attend_case(ctx, fmt, lens, M, H, L, P, page)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,H", [([9001], 1, 128), ([5000, 17, 3000], 2, 128), ([6001] * 5, 1, 16),
                                      ([4000, 0, 2000, 1], 1, 64), ([12000], 4, 32), ([140, 200], 140, 128),
                                      ([1000, 64, 30], 64, 16)])
def test_attend_long(ctx, fmt, lens, M, H):
    attend_case(ctx, fmt, lens, M, H, 512, 64, 64)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,H,L,P,page", [
    ([5000], 1, 4, 64, 16, 16), ([3000, 1, 777, 0], 2, 5, 128, 32, 4), ([2500, 64], 1, 6, 136, 8, 64),
    ([900] * 130, 1, 6, 72, 8, 32), ([65, 3, 200] * 200, 1, 5, 64, 16, 8), ([700, 130], 3, 7, 768, 256, 128)])
def test_attend_other_widths_long(ctx, fmt, lens, M, H, L, P, page):
    """Slices of a row joined, slices that are left empty, and none at all."""
    attend_case(ctx, fmt, lens, M, H, L, P, page)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,H,page", [
    ([1, 0, 33, 64, 100, 0], 2, 32, 16), ([40], 1, 128, 64), ([0, 0, 7], 1, 48, 8), ([5, 90, 31] * 30, 1, 16, 32),
    ([60, 1, 17], 4, 128, 128)])
def test_attend_short_in_a_wide_table(ctx, fmt, lens, M, H, page):
    """Lengths far below what the table holds: cut into ranges all the same."""
    attend_case(ctx, fmt, lens, M, H, 512, 64, page, width=9000 // page)


@pytest.mark.parametrize("fmt,H", [("bf16", 16), ("bf16", 64), ("bf16", 128), ("f16x2", 16)])
def test_attend_many_sequences(ctx, fmt, H):
    """More sequences than workgroups look up at once, most of them short."""
    lens = [(37 * k) % 90 for k in range(700)]
    attend_case(ctx, fmt, lens, 1, H, 512, 64, 16)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,H,page", [(3, 128, 64), (2, 16, 16), (4, 64, 32), (3, 4, 2)])
def test_a_later_row_does_not_reach_an_earlier_one(ctx, fmt, M, H, page):
    """NaN and infinities at the last position: its row is NaN, the rows
    before it are as without."""
    L, P = (512, 64) if H > 4 else (64, 16)
    pool = R.Pool(3, fmt, [97, 64, 130], page, L, P)
    qabs, qrope = pool.queries(M, H)
    args = pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE
    clean = pool.cuda(ctx=ctx).attend(*args)
    for b, n in enumerate(pool.lens):
        x = torch.full((1, L + P), math.nan)
        x[:, 1::2] = math.inf
        pool.put(b, n - 1, x)
    got = pool.cuda(ctx=ctx).attend(*args)
    assert torch.equal(got[:, :-1], clean[:, :-1])
    assert not torch.isfinite(got[:, -1]).any()


@pytest.mark.parametrize("fmt", FMTS)
def test_attend_extreme_scores(ctx, fmt):
    """One position far above the rest, then scores that fall from 200 to -200
    and rise again; a scale below zero and of zero."""
    pool = R.Pool(5, fmt, [300, 300], 64, 512, 64)
    u = torch.zeros(576)
    u[:8] = 1.0
    ramp = torch.linspace(200, -200, 300).abs() - 100
    pool.put(0, 0, pool.randn(300, 576) * 0.1 + ramp[:, None] * u / 8 * 0.5)
    pool.put(1, 0, pool.randn(300, 576) * 0.1)
    pool.put(1, 123, 30 * u[None])
    qabs, qrope = [torch.zeros_like(t) for t in pool.queries(1, 128)]
    qabs[..., :8] = 2.0
    cache = pool.cuda(ctx=ctx)
    for scale in (1.0, -1.0, 0.0):
        got = cache.attend(pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), scale)
        want, spread, mass = reference(pool, qabs, qrope, scale)
        # scores reach some hundreds, where f32's step is 2^-15 or less: weights to 2^-13
        close(fmt, got, want, spread + 2.0 ** -13 / 5e-5 * spread, mass)


def test_sequences_share_pages(ctx):
    pool = R.Pool(7, "bf16", [200, 200], 64, 512, 64)
    pool.table[1, :2] = pool.table[0, :2]
    qabs, qrope = pool.queries(1, 128)
    got = pool.cuda(ctx=ctx).attend(pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE)
    close("bf16", got, *reference(pool, qabs, qrope))


@pytest.mark.parametrize("fmt", FMTS)
def test_table_slices_and_out(ctx, fmt):
    pool = R.Pool(9, fmt, [150, 20, 64], 32, 512, 64, width=9)
    qabs, qrope = pool.queries(2, 32)
    wide = torch.full((6, 20), -5, dtype=torch.int32, device="cuda")
    wide[::2, 7:16] = pool.table.cuda()
    cache, lens = pool.cuda(ctx=ctx), pool.lens32().cuda()
    want = cache.attend(pool.table.cuda(), lens, qabs.cuda(), qrope.cuda(), SCALE)
    out = torch.full((4, 2, 32, 512), 7.0, dtype=cache.dtype, device="cuda")
    assert cache.attend(wide[::2, 7:16], lens, qabs.cuda(), qrope.cuda(), SCALE, out=out[:3]).data_ptr() == out.data_ptr()
    assert torch.equal(out[:3], want) and (out[3] == 7.0).all()


def test_a_pool_past_32_bits(ctx):
    """Pages whose first byte lies behind 4 GiB, and the pool's last."""
    import undertow_amd as U
    n = 2**32 // (64 * 1152) + 40
    pages = torch.zeros((n, 64, 576), dtype=torch.bfloat16, device="cuda")
    ids = [n - 1, n - 39, 0, n - 2, 5]
    pages[ids] = torch.randn((5, 64, 576), device="cuda").bfloat16()
    small = pages[ids].clone()
    q = torch.randn((1, 1, 128, 576), device="cuda").bfloat16()
    q = q[..., :512].contiguous(), q[..., 512:].contiguous()
    lens = torch.tensor([300], dtype=torch.int32, device="cuda")
    far = U.PagedCache(ctx, pages).attend(torch.tensor([ids], dtype=torch.int32, device="cuda"), lens, *q, SCALE)
    near = U.PagedCache(ctx, small).attend(torch.arange(5, dtype=torch.int32, device="cuda")[None], lens, *q, SCALE)
    assert torch.equal(far, near)
    lat, kr = torch.randn((1, 1, 512), device="cuda"), torch.randn((1, 1, 64), device="cuda")
    U.PagedCache(ctx, pages).append(torch.tensor([ids[::-1]], dtype=torch.int32, device="cuda"), lens, lat, kr)
    assert torch.equal(pages[n - 1, 43], torch.cat([lat, kr], -1)[0, 0].bfloat16())


# ------------------------------------------------------- selected pages
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,H,page,top_k", [
    ([400, 33, 0, 1], 2, 128, 16, 7), ([1000], 1, 128, 64, 5), ([700, 650], 3, 32, 32, 9),
    ([500, 20], 1, 16, 64, 3), ([300, 299], 1, 64, 8, 20), ([90, 200], 2, 4, 4, 11), ([2100, 70], 1, 48, 128, 4),
    ([50, 61], 2, 32, 2, 13), ([100, 900], 1, 128, 16, 300), ([1100, 5], 2, 16, 1024, 1),
    ([20, 33, 0, 70], 1, 64, 32, 150), ([9, 16] * 40, 2, 32, 16, 3)])
def test_attend_selected_pages(ctx, fmt, lens, M, H, page, top_k):
    """Entries in any order, gaps among them, pages behind the row's end, one
    listed twice, a row with none; pages that no row lists hold NaN."""
    L, P = (64, 16) if H == 4 else (512, 64)
    pool = R.Pool(11, fmt, lens, page, L, P)
    qabs, qrope = pool.queries(M, H)
    sel = torch.full((len(lens), M, top_k), -1, dtype=torch.int32)
    used = set()
    for b, n in enumerate(lens):
        for j, s in enumerate(R.seen(n, M)):
            ids = torch.randperm(-(-s // page), generator=pool.g)[:top_k - 1].int()
            at = torch.randperm(top_k, generator=pool.g)[:len(ids)].sort().values
            sel[b, j, at] = ids
            used |= {(b, int(k)) for k in ids}
    if lens[0] > 4 * page:
        sel[0, 0, 0], sel[0, 0, -1] = 1, 1  # counts twice
        sel[0, 0, 1] = 10**6
        used.add((0, 1))
    if len(lens) > 1:
        sel[1, -1] = -7
    for b, n in enumerate(lens):
        for k in range(-(-n // page)):
            if (b, k) not in used:
                pool.pages[pool.table[b, k].long()] = math.nan
    got = pool.cuda(ctx=ctx).attend_pages(pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE, sel.cuda())
    ctx.synchronize()
    close(fmt, got, *reference(pool, qabs, qrope, sel=sel))
    if len(lens) > 1:
        assert (got[1, -1] == 0).all()


def pages_in_order(pool, seed=0):
    """Summaries of every page that a sequence holds, from its stored rows."""
    mean = torch.full((pool.n_pages, pool.D), 99, dtype=torch.int8)
    scale = torch.full((pool.n_pages,), math.nan)
    for b, n in enumerate(pool.lens):
        for k in range(-(-n // pool.page)):
            at = pool.table[b, k].long()
            mean[at], scale[at] = R.summary(pool.rows(b, torch.arange(k * pool.page, min(n, (k + 1) * pool.page))))
    return mean, scale


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,H,page,top_k,first,last,weighted", [
    ([1000], 1, 128, 16, 9, 1, 1, False), ([64, 65, 0, 1, 700], 1, 128, 16, 5, 1, 2, False),
    ([900, 30], 3, 128, 8, 20, 0, 0, True), ([333, 332], 2, 16, 4, 31, 3, 4, False),
    ([640], 1, 7, 1, 100, 2, 2, True), ([500, 600], 2, 4, 8, 6, 5, 1, False),
    ([17000], 1, 32, 8, 64, 1, 2, False), ([800], 1, 160, 16, 3, 1, 1, True), ([4000], 2, 128, 2, 70, 1, 1, False)])
def test_select(ctx, fmt, lens, M, H, page, top_k, first, last, weighted):
    L, P = (64, 16) if H == 4 else (512, 64)
    pool = R.Pool(13, fmt, lens, page, L, P)
    mean, scale = pages_in_order(pool)
    # equal pages: the lower one first
    for b, n in enumerate(lens):
        if n > 12 * page:
            src = pool.table[b, 3].long()
            for k in (5, 8, 9):
                at = pool.table[b, k].long()
                mean[at], scale[at] = mean[src], scale[src]
    qabs, qrope = pool.queries(M, H)
    if H > 4:
        qabs[:, :, 1], qrope[:, :, 1] = 0, 0
        qabs[:, :, 2, 5] = math.nan
        qrope[:, :, 3, 1] = -math.inf
    w = pool.randn(len(lens), M, H) if weighted else None
    cache = pool.cuda(ctx=ctx, mean=mean.cuda(), mean_scale=scale.cuda())
    got = cache.select(pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), top_k, first, last,
                       weights=None if w is None else w.cuda())
    ctx.synchronize()
    q = torch.cat([qabs, qrope], -1).double()
    for b, n in enumerate(lens):
        for j, s in enumerate(R.seen(n, M)):
            k = -(-s // page)
            at = pool.table[b, :k].long()
            want = R.select(q[b, j], mean[at], scale[at], k, first, last, top_k, None if w is None else w[b, j])
            assert got[b, j].tolist() == want, (b, j)


@pytest.mark.parametrize("n_pages,top_k", [(1024, 1), (1025, 1024), (5000, 333), (40000, 64), (40000, 2000)])
def test_select_among_many_equal_pages(ctx, n_pages, top_k):
    """Scores of few different values: ties are cut at the lowest pages."""
    import undertow_amd as U
    g = torch.Generator(device="cuda").manual_seed(n_pages)
    pages = torch.zeros((n_pages, 1, 576), dtype=torch.bfloat16, device="cuda")
    mean = torch.zeros((n_pages, 576), dtype=torch.int8, device="cuda")
    level = torch.randint(0, 5, (n_pages,), device="cuda", generator=g)
    mean[:, 7] = level.to(torch.int8)
    cache = U.PagedCache(ctx, pages, mean=mean, mean_scale=torch.ones(n_pages, device="cuda"))
    q = torch.zeros((1, 1, 16, 512), dtype=torch.bfloat16, device="cuda")
    q[..., 7] = 1
    got = cache.select(torch.arange(n_pages, dtype=torch.int32, device="cuda")[None],
                       torch.tensor([n_pages], dtype=torch.int32, device="cuda"), q,
                       torch.zeros((1, 1, 16, 64), dtype=torch.bfloat16, device="cuda"), top_k, 0, 0)
    want = torch.sort(level, descending=True, stable=True).indices[:top_k].sort().values
    assert torch.equal(got[0, 0].long(), want)


def test_select_ranks_nan_last(ctx):
    import undertow_amd as U
    n = 40
    pages = torch.zeros((n, 16, 576), dtype=torch.bfloat16, device="cuda")
    mean = torch.ones((n, 576), dtype=torch.int8, device="cuda")
    scale = torch.linspace(1, 2, n, device="cuda")
    scale[::2] = math.nan
    cache = U.PagedCache(ctx, pages, mean=mean, mean_scale=scale)
    q = torch.ones((1, 1, 16, 512), dtype=torch.bfloat16, device="cuda")
    got = cache.select(torch.arange(n, dtype=torch.int32, device="cuda")[None],
                       torch.tensor([16 * n], dtype=torch.int32, device="cuda"), q,
                       torch.ones((1, 1, 16, 64), dtype=torch.bfloat16, device="cuda"), 23, 0, 0)
    assert got[0, 0].tolist() == sorted(list(range(1, n, 2)) + [0, 2, 4])


# --------------------------------------------------------------- append
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,L,P,page", [
    ([1, 64, 65, 200], 1, 512, 64, 64), ([5, 3, 0, 130], 4, 512, 64, 16), ([700, 500], 450, 512, 64, 64),
    ([33, 32], 2, 64, 16, 8), ([40], 40, 1000, 24, 16), ([9, 30], 12, 512, 64, 1), ([1000], 7, 8, 8, 1024),
    ([300, 2], 129, 512, 64, 128)])
@pytest.mark.parametrize("summaries", [True, False])
def test_append(ctx, fmt, lens, M, L, P, page, summaries):
    """New rows stand where they should, in the pool's type, every other row is
    untouched to the bit, and the touched pages' summaries are those of their
    stored rows."""
    pool = R.Pool(17, fmt, lens, page, L, P, fill=False)
    for b, n in enumerate(lens):
        pool.put(b, 0, pool.randn(max(0, n - M), L + P))
    x = pool.randn(len(lens), M, L + P) * torch.exp(4 * pool.randn(len(lens), M, 1))
    mean = torch.full((pool.n_pages, L + P), 99, dtype=torch.int8)
    scale = torch.full((pool.n_pages,), 99.0)
    more = dict(mean=mean.cuda(), mean_scale=scale.cuda()) if summaries else {}
    cache = pool.cuda(ctx=ctx, **more)
    cache.append(pool.table.cuda(), pool.lens32().cuda(), x[..., :L].contiguous().cuda(), x[..., L:].contiguous().cuda())
    ctx.synchronize()
    for b, n in enumerate(lens):
        k = min(n, M)
        pool.put(b, n - k, x[b, M - k:])
        for p in range(max(0, n - k) // page, -(-n // page) if k else 0):
            at = pool.table[b, p].long()
            mean[at], scale[at] = R.summary(pool.rows(b, torch.arange(p * page, min(n, (p + 1) * page))))
    assert torch.equal(cache.pages.cpu().view(torch.int16), pool.pages.view(torch.int16))
    if summaries:
        assert torch.equal(cache.mean.cpu(), mean)
        assert torch.equal(cache.mean_scale.cpu(), scale)


def test_append_values_past_f16(ctx):
    pool = R.Pool(19, "f16x2", [5], 16, 512, 64, fill=False)
    x = pool.randn(1, 5, 576)
    x[0, 1, :6] = torch.tensor([65504.0, 65519.0, 65520.0, -1e9, 3e38, 1e-30])
    x[0, 2, :3] = torch.tensor([math.inf, -math.inf, math.nan])
    x[0, 3] *= 1e-6
    cache = pool.cuda(ctx=ctx)
    cache.append(pool.table.cuda(), pool.lens32().cuda(), x[..., :512].contiguous().cuda(), x[..., 512:].contiguous().cuda())
    got = R.values("f16x2", cache.pages.cpu()[pool.where(0, torch.arange(5))])
    c = torch.where(x[0].isfinite(), x[0].double().clamp(-65504, 65504), x[0].double())
    nan = torch.isnan(c)
    assert torch.equal(torch.isnan(got), nan)
    inf = torch.isinf(c)
    assert torch.equal(got[inf], c[inf])
    ok = ~(nan | inf)
    assert ((got[ok] - c[ok]).abs() <= 2.0 ** -22 * c[ok].abs() + 2.0 ** -35).all()


# --------------------------------------------------------------- errors
def test_bad_pages_and_lengths_are_reported(ctx):
    """The bounds hold in every call: an error at the next synchronize, once,
    and the other sequences as without."""
    import undertow_amd as U
    pool = R.Pool(23, "bf16", [100, 90, 80], 16, 512, 64)
    mean, scale = pages_in_order(pool)
    qabs, qrope = [t.cuda() for t in pool.queries(1, 32)]
    lat, kr = torch.randn((3, 1, 512), device="cuda"), torch.randn((3, 1, 64), device="cuda")
    sel = torch.arange(4, dtype=torch.int32, device="cuda").repeat(3, 1, 1)
    for bad_page in (True, False):
        cache = pool.cuda(ctx=ctx, mean=mean.cuda(), mean_scale=scale.cuda())
        table, lens = pool.table.cuda(), pool.lens32().cuda()
        calls = [lambda: cache.attend(table, lens, qabs, qrope, SCALE),
                 lambda: cache.attend_pages(table, lens, qabs, qrope, SCALE, sel),
                 lambda: cache.select(table, lens, qabs, qrope, 4)]
        if not bad_page:  # a length beyond the table counts as the table's
            lens[1], table[1, 6] = 112, 0
        want = [f() for f in calls]
        ctx.synchronize()
        if bad_page:
            table[1] = torch.tensor([pool.n_pages, -1, 2**31 - 1, -2**31, pool.n_pages, -1, 7], device="cuda")
        else:
            lens[1] = 113
        for f, w in zip(calls, want):
            got = f()
            with pytest.raises(U.UtError) as e:
                ctx.synchronize()
            assert e.value.code == U.runtime.UT_ERR_BAD_PAGE
            assert torch.equal(got[::2], w[::2])
            ctx.synchronize()
        lens[1] = 86 if bad_page else -3
        before = cache.pages.clone()
        cache.append(table, lens, lat, kr)
        with pytest.raises(U.UtError) as e:
            ctx.synchronize()
        assert e.value.code == U.runtime.UT_ERR_BAD_PAGE
        for b, n in ((0, 100), (2, 80)):
            before[pool.where(b, torch.tensor(n - 1))] = torch.cat([lat, kr], -1)[b, 0].bfloat16()
        assert torch.equal(cache.pages.view(torch.int16), before.view(torch.int16))


def test_refusals(ctx):
    """What the library itself turns down, before anything is launched."""
    import ctypes as C

    import undertow_amd as U
    lib, rt = U.lib(), U.runtime
    pages = torch.zeros((4, 16, 576), dtype=torch.bfloat16, device="cuda")
    mean, scale = torch.zeros((4, 576), dtype=torch.int8, device="cuda"), torch.zeros(4, device="cuda")
    table, lens = torch.zeros((2, 4), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    f = torch.zeros((2, 1, 16, 576), device="cuda")
    p = f.data_ptr()

    def kv(**k):
        d = dict(pages=pages.data_ptr(), mean=mean.data_ptr(), mean_scale=scale.data_ptr(), n_pages=4, page=16,
                 latent=512, rope=64, fmt=U.KV_BF16)
        return C.byref(rt.MlaPages(**{**d, **k}))

    def batch(cache, **k):
        d = dict(ctx=ctx.handle, table=table.data_ptr(), stride=4, width=4, lens=lens.data_ptr(), B=2, M=1)
        d.update(k)
        return d["ctx"], cache, d["table"], d["stride"], d["width"], d["lens"], d["B"], d["M"]

    def calls(cache, **k):
        H = k.pop("H", 16)
        q, o = k.pop("q", p), k.pop("o", p)
        b = batch(cache, **k)
        yield lib.ut_mla_paged_attend(*b, H, q, p, 0.1, o)
        yield lib.ut_mla_sparse_attend(*b, H, q, p, 0.1, p, 2, o)
        yield lib.ut_mla_page_select(*b, H, q, p, None, 1, 1, 2, o)
        yield lib.ut_mla_paged_append(*b, q, o)

    arg, shape = rt.UT_ERR_ARG, rt.UT_ERR_SHAPE
    assert all(c == arg for c in calls(None)) and all(c == arg for c in calls(kv(), ctx=None))
    for k in (dict(pages=None), dict(fmt=2), dict(fmt=-1), dict(n_pages=0), dict(pages=pages.data_ptr() + 8)):
        assert all(c == arg for c in calls(kv(**k))), k
    for k in (dict(page=0), dict(page=24), dict(page=2048), dict(latent=0), dict(rope=0), dict(latent=508),
              dict(rope=20), dict(latent=1024), dict(n_pages=2**31)):
        assert all(c == shape for c in calls(kv(**k))), k
    for k in (dict(table=None), dict(lens=None), dict(stride=3), dict(width=0), dict(B=0), dict(M=0), dict(q=None),
              dict(q=p + 4), dict(o=None)):
        assert all(c == arg for c in calls(kv(), **k)), k
    for k in (dict(B=70000), dict(M=2**31), dict(width=2**30, stride=2**30), dict(width=2**27 - 63, stride=2**27)):
        assert all(c == shape for c in calls(kv(), **k)), k
    one = dict(page=1, pages=pages.data_ptr())  # within 32 bits, past what a launch spans
    assert list(calls(kv(**one), M=2**28, width=2**28, stride=2**28, B=1))[3] == shape
    assert list(calls(kv(**one), M=2**28, width=2**28, stride=2**28, B=1, H=1))[2] == shape
    assert lib.ut_mla_page_select(*batch(kv(**one), width=2**28, stride=2**28), 16, p, p, None, 1, 1, 2, p) == shape
    assert list(calls(kv(), H=0))[:3] == [arg] * 3 and list(calls(kv(), H=70000))[:3] == [shape] * 3
    assert list(calls(kv(), M=40000))[:3] == [shape] * 3 and list(calls(kv(), M=40000, H=1))[:3] == [shape] * 3
    b = batch(kv())
    assert lib.ut_mla_sparse_attend(*b, 16, p, p, 0.1, None, 2, p) == arg
    assert lib.ut_mla_sparse_attend(*b, 16, p, p, 0.1, p, 0, p) == arg
    assert lib.ut_mla_sparse_attend(*b, 16, p, p, 0.1, p, 2**27 - 63, p) == arg
    for first, last, k in ((-1, 1, 4), (1, -1, 4), (3, 2, 4), (0, 0, 0), (5, 0, 4), (2**62, 2**62, 4)):
        assert lib.ut_mla_page_select(*b, 16, p, p, None, first, last, k, p) == arg
    for k in (dict(mean=None), dict(mean_scale=None), dict(mean=None, mean_scale=None)):
        assert lib.ut_mla_page_select(*batch(kv(**k)), 16, p, p, None, 1, 1, 2, p) == arg
    assert lib.ut_mla_paged_append(*batch(kv(mean=None)), p, p) == arg
    ctx.synchronize()


# ------------------------------------------------- streams, graphs, runs
@pytest.mark.parametrize("H,L,P", [(128, 512, 64), (4, 64, 16)])
def test_captured_steps_follow_lengths(ctx, H, L, P):
    """One step captured (append, select, attention over the selection and
    over everything), replayed as the lengths grow and a page is added, with
    eager calls of other sizes between: every replay gives the eager call's
    bits."""
    import undertow_amd as U
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c = U.Context(0)
        g = torch.Generator(device="cuda").manual_seed(3)
        rnd = lambda *d: torch.randn(d, device="cuda", generator=g)
        B, M = 3, 2
        cache = U.PagedCache.empty(c, 60, page=16, latent=L, rope=P)
        table = torch.arange(60, dtype=torch.int32, device="cuda").reshape(3, 20)
        lens = torch.tensor([150, 17, 31], dtype=torch.int32, device="cuda")
        cache.append(table, lens, rnd(B, 150, L), rnd(B, 150, P))
        lat, kr = rnd(B, M, L), rnd(B, M, P)
        q = rnd(B, M, H, L).bfloat16(), rnd(B, M, H, P).bfloat16()

        def step():
            cache.append(table, lens, lat, kr)
            sel = cache.select(table, lens, *q, 3, 1, 1)
            return sel, cache.attend_pages(table, lens, *q, SCALE, sel), cache.attend(table, lens, *q, SCALE)

        lens += M
        step()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = step()
        for k in range(4):
            lens += M
            lat.copy_(rnd(B, M, L))
            for t in got:
                t.zero_()
            graph.replay()
            s.synchronize()
            first = [t.clone() for t in got]
            pages = cache.pages.clone()
            want = step()  # writes the same rows again
            assert all(torch.equal(a, b) for a, b in zip(first, want))
            assert torch.equal(pages, cache.pages)
            big = rnd(64, 1, H, L).bfloat16()  # grows the arena past what the graph took
            cache.attend(table[:1].expand(64, 20).contiguous(), lens[:1].expand(64).contiguous(), big,
                         rnd(64, 1, H, P).bfloat16(), SCALE)
            c.synchronize()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("H,L,P", [(128, 512, 64), (16, 512, 64), (4, 64, 16)])
def test_a_serving_run(ctx, fmt, H, L, P):
    """Prompts and then steps with a rejected draft: the cache's attention
    agrees with the contiguous cache's, the selection of every page with the
    whole, and a selection of few pages with attention over those."""
    import undertow_amd as U
    g = torch.Generator(device="cuda").manual_seed(H)
    rnd = lambda *d: torch.randn(d, device="cuda", generator=g)
    B, page = 3, 16
    cache = U.PagedCache.empty(ctx, 64, page, L, P, U.KV_BF16 if fmt == "bf16" else U.KV_F16X2)
    table = torch.randperm(64, device="cuda", generator=g)[:60].reshape(B, 20).int()
    hist = rnd(B, 320, L + P).bfloat16().float()  # what both formats hold exactly
    n = [0] * B

    def grow(k):
        nonlocal n
        n = [a + b for a, b in zip(n, k)]
        M = max(k)
        new = torch.zeros((B, M, L + P), device="cuda")
        for b in range(B):
            if k[b]:
                new[b, M - k[b]:] = hist[b, n[b] - k[b]:n[b]]
            # rows that are not new: what stands there already
            for j in range(M - k[b]):
                pos = n[b] - M + j
                if pos >= 0:
                    new[b, j] = hist[b, pos]
        lens = torch.tensor(n, dtype=torch.int32, device="cuda")
        cache.append(table, lens, new[..., :L].contiguous(), new[..., L:].contiguous())
        return lens, M

    for k in ([100, 37, 1], [2, 2, 2], "reject", [1, 1, 1], [3, 3, 3], [60, 60, 60]):
        if k == "reject":  # the last row of each was a wrong draft
            n = [a - 1 for a in n]
            continue
        lens, M = grow(k)
        M = min(M, 3)
        q = rnd(B, M, H, L + P).to(cache.dtype)
        qa, qr = q[..., :L].contiguous(), q[..., L:].contiguous()
        got = cache.attend(table, lens, qa, qr, SCALE)
        for b in range(B):
            rows = [j for j in range(M) if n[b] - M + j >= 0]
            base = n[b] - len(rows)
            want = U.mla_attend(ctx, qa[b, rows].float().contiguous(), qr[b, rows].float().contiguous(),
                                hist[b, :n[b], :L].contiguous(), hist[b, :n[b], L:].contiguous(), base, SCALE)
            # the contiguous cache keeps 16 bits of a product (1e-4), bf16 outputs and weights 2^-8 each
            tol = (1e-4 if fmt == "f16x2" else 2.0 ** -7) * max(1.0, float(want.abs().max()))
            assert float((got[b, rows].float() - want).abs().max()) <= tol
        every = cache.select(table, lens, qa, qr, 20, 1, 1)
        again = cache.attend_pages(table, lens, qa, qr, SCALE, every)
        bar = 2e-5 if fmt == "f16x2" else 2.0 ** -7
        assert float((again.float() - got.float()).norm()) <= bar * float(got.float().norm())
        few = cache.select(table, lens, qa, qr, 4, 1, 2)
        part = cache.attend_pages(table, lens, qa, qr, SCALE, few)
        ctx.synchronize()
        for b in range(B):
            for j in range(M):
                s = n[b] - M + j + 1
                if s <= 0:
                    assert (part[b, j] == 0).all() and (few[b, j] == -1).all()
                    continue
                ids = [k for k in few[b, j].tolist() if k >= 0]
                last = (s - 1) // page
                assert ids == sorted(set(ids)) and len(ids) == min(4, last + 1) and 0 in ids and last in ids
                pos = torch.cat([torch.arange(k * page, min(s, (k + 1) * page)) for k in ids]).cuda()
                want, spread, mass = R.attend(hist[b, pos].double(), q[b, j].double(), L, SCALE)
                close(fmt, part[b, j], want.cpu(), spread.cpu(), mass.cpu())


def test_calls_on_a_stream_of_their_own(ctx):
    """Two contexts on two streams over one pool at a time: the same bits."""
    import undertow_amd as U
    pool = R.Pool(29, "bf16", [900, 333, 12], 32, 512, 64)
    qabs, qrope = [t.cuda() for t in pool.queries(1, 128)]
    cache, table, lens = pool.cuda(ctx=ctx), pool.table.cuda(), pool.lens32().cuda()
    want = cache.attend(table, lens, qabs, qrope, SCALE)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        with torch.cuda.stream(s):
            c = U.PagedCache(U.Context(0), cache.pages)
            outs.append([c.attend(table, lens, qabs, qrope, SCALE) for _ in range(5)])
            c.ctx.synchronize()
    assert all(torch.equal(o, want) for v in outs for o in v)


def test_two_contexts_at_once(ctx):
    """Two contexts on streams of their own, over one pool, their calls under
    way at the same time: each has the bits of its calls alone."""
    import undertow_amd as U
    g = torch.Generator(device="cuda").manual_seed(8)
    rnd = lambda *d: torch.randn(d, device="cuda", generator=g)
    cache = U.PagedCache.empty(ctx, 300, page=16)
    table = torch.randperm(300, device="cuda", generator=g)[:264].reshape(3, 88).int()
    lens = torch.tensor([700, 90, 1300], dtype=torch.int32, device="cuda")
    cache.append(table, lens, rnd(3, 1300, 512), rnd(3, 1300, 64))
    ctx.synchronize()
    torch.cuda.synchronize()
    runs = []
    for k, M in enumerate((1, 4)):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            c = U.Context(0)
            mine = U.PagedCache(c, cache.pages, 512, 64, cache.mean, cache.mean_scale)
            q = rnd(3, M, 128, 512).bfloat16(), rnd(3, M, 128, 64).bfloat16()
            s.synchronize()
            runs.append((s, c, mine, q))

    def turn(s, c, mine, q):
        with torch.cuda.stream(s):
            sel = mine.select(table, lens, *q, 9)
            return sel, mine.attend(table, lens, *q, SCALE), mine.attend_pages(table, lens, *q, SCALE, sel)

    alone = []
    for x in runs:
        alone.append(turn(*x))
        x[1].synchronize()
    both = [[turn(*x) for x in runs] for _ in range(10)]
    for x in runs:
        x[1].synchronize()
    for pair in both:
        for got, want in zip(pair, alone):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_captured_calls_share_the_arena(ctx):
    """Two graphs of one context, the second captured with more working memory
    than the first, replayed in turn with eager calls between: each replay has
    the eager call's bits."""
    import undertow_amd as U
    g = torch.Generator(device="cuda").manual_seed(5)
    rnd = lambda *d: torch.randn(d, device="cuda", generator=g)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c = U.Context(0)
        cache = U.PagedCache.empty(c, 400, page=16)
        table = torch.randperm(400, device="cuda", generator=g).reshape(4, 100).int()
        lens = torch.tensor([1600, 3, 700, 1111], dtype=torch.int32, device="cuda")
        cache.append(table, lens, rnd(4, 1600, 512), rnd(4, 1600, 64))
        calls = []
        for rows, n in ((1, 1), (3, 4)):
            q = rnd(n, rows, 128, 512).bfloat16(), rnd(n, rows, 128, 64).bfloat16()
            calls.append((lambda t, x, q: lambda: cache.attend(t, x, *q, SCALE))(table[:n], lens[:n], q))
        graphs = []
        for f in calls:
            f()
            s.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                out = f()
            graphs.append((graph, out))
        for turn in range(4):
            lens -= turn
            want = [f().clone() for f in calls]
            for (graph, out), w in list(zip(graphs, want))[::1 if turn % 2 else -1]:
                out.zero_()
                graph.replay()
                s.synchronize()
                assert torch.equal(out, w)
