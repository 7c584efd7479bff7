"""Prompt-sized calls of the paged latent cache on the GPU: attention and page
selection against 64 bits, and what attention reserves."""
import pytest
import torch

import paged_ref as R
from test_gpu_paged import SCALE, close, pages_in_order

pytestmark = pytest.mark.gpu
FMTS = ["bf16", "f16x2"]


def check(pool, fmt, got, qabs, qrope, sel=None):
    """Every row of `got` against 64 bits; rows that see nothing are zeros."""
    B, M, H, L = qabs.shape
    for b, n in enumerate(pool.lens):
        kv = pool.rows(b, torch.arange(n)).cuda()
        q = torch.cat([qabs[b], qrope[b]], -1).double().cuda()
        for j, s in enumerate(R.seen(n, M)):
            x = kv[:s]
            if sel is not None:
                at = [torch.arange(k * pool.page, min(s, (k + 1) * pool.page)) for k in sel[b, j].tolist()
                      if 0 <= k and k * pool.page < s]
                x = kv[torch.cat(at).cuda()] if at else kv[:0]
            if len(x) == 0:
                assert (got[b, j] == 0).all()
                continue
            want, spread, mass = R.attend(x, q[j], L, SCALE)
            close(fmt, got[b, j], want.cpu(), spread.cpu(), mass.cpu())


def reserved(ctx, call):
    """(bytes that the context's arena grew by in a call, launches of the join)"""
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    ctx.enable_timing(True)
    call()
    joins = ctx.kernel_time("paged_join")[0]
    ctx.enable_timing(False)
    ctx.synchronize()
    return free - torch.cuda.mem_get_info()[0], joins


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("B,M,H,width", [(1, 512, 128, 8192), (1, 2048, 128, 4096), (3, 777, 128, 2000), (2, 1024, 32, 9000)])
def test_prompt_rows_reserve_nothing(ctx, fmt, B, M, H, width):
    """A call whose column groups alone fill the device leaves no parts: no
    memory for them and no join."""
    import undertow_amd as U
    pool = R.Pool(31, fmt, [80] * B, 64, 512, 64, width=width // 64)
    qabs, qrope = [t.cuda() for t in pool.queries(M, H)]
    c = U.Context(0)
    cache, table, lens = pool.cuda(ctx=c), pool.table.cuda(), pool.lens32().cuda()
    out = torch.empty_like(qabs)
    cache.attend(table[:, :2].contiguous(), lens, qabs[:, -1:, :16].contiguous(), qrope[:, -1:, :16].contiguous(), SCALE)
    assert reserved(c, lambda: cache.attend(table, lens, qabs, qrope, SCALE, out=out)) == (0, 0)
    assert (out[:, :M - 80] == 0).all()


@pytest.mark.parametrize("fmt,lens,M,H,width", [
    ("bf16", [600, 40, 333], 128, 256, 4096), ("f16x2", [500, 64], 64, 256, 2048),  # one range over all
    ("bf16", [700], 300, 128, 8192), ("f16x2", [300, 220], 150, 128, 2048),         # whole sequences
    ("bf16", [1500, 700], 40, 128, 2048), ("f16x2", [1100], 40, 64, 2048)])         # ranges and their join
def test_attend_prompt_rows(ctx, fmt, lens, M, H, width):
    pool = R.Pool(37, fmt, lens, 64, 512, 64, width=width // 64)
    qabs, qrope = pool.queries(M, H)
    got = pool.cuda(ctx=ctx).attend(pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE)
    ctx.synchronize()
    check(pool, fmt, got, qabs, qrope)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,H,width,at", [
    ([97, 64, 130], 40, 128, 192, 5), ([97, 64, 130], 64, 32, 4096, 33), ([300, 500, 20], 150, 128, 512, 70),
    ([600, 100], 128, 256, 4096, 100)])
def test_a_later_prompt_row_does_not_reach_an_earlier_one(ctx, fmt, lens, M, H, width, at):
    """NaN and infinities in one row of a prompt: that row and those behind it
    are NaN, the rows before it are as without."""
    pool = R.Pool(67, fmt, lens, 64, 512, 64, width=width // 64)
    qabs, qrope = pool.queries(M, H)
    args = pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE
    clean = pool.cuda(ctx=ctx).attend(*args)
    for b, n in enumerate(lens):
        x = torch.full((1, 576), float("nan"))
        x[:, 1::2] = float("inf")
        if n - M + at >= 0:
            pool.put(b, n - M + at, x)
    got = pool.cuda(ctx=ctx).attend(*args)
    ctx.synchronize()
    for b, n in enumerate(lens):
        if n - M + at >= 0:
            assert torch.equal(got[b, :at], clean[b, :at]) and torch.isfinite(clean[b]).all()
            assert not torch.isfinite(got[b, at:]).any()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,H,page,top_k", [
    ([700, 90], 130, 32, 64, 6), ([500], 300, 128, 16, 20), ([300, 40, 111], 100, 16, 8, 9), ([400, 399], 60, 64, 128, 3)])
def test_selected_pages_of_prompt_rows(ctx, fmt, lens, M, H, page, top_k):
    """Many rows of a sequence choose, with head weights, and attend to their
    choice: the choice as defined, the rest against 64 bits."""
    pool = R.Pool(71, fmt, lens, page, 512, 64)
    mean, scale = pages_in_order(pool)
    qabs, qrope = pool.queries(M, H)
    w = pool.randn(len(lens), M, H)
    cache = pool.cuda(ctx=ctx, mean=mean.cuda(), mean_scale=scale.cuda())
    where = pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda()
    sel = cache.select(*where, top_k, 1, 1, weights=w.cuda())
    got = cache.attend_pages(*where, SCALE, sel)
    ctx.synchronize()
    q = torch.cat([qabs, qrope], -1).double()
    for b, n in enumerate(lens):
        for j in list(range(0, M, 17)) + [M - 1]:
            k = -(-max(0, n - M + j + 1) // page)
            at = pool.table[b, :k].long()
            want = R.select(q[b, j], mean[at], scale[at], k, 1, 1, top_k, w[b, j])
            assert sel[b, j].tolist() == want, (b, j)
    check(pool, fmt, got, qabs, qrope, sel.cpu())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,H,width,warm", [
    ([600, 200], 128, 256, 4096, False), ([700], 300, 128, 8192, False), ([900, 30, 400], 2, 128, 4096, True)])
def test_captured_prompt_rows_follow_lengths(fmt, lens, M, H, width, warm):
    """One range, whole sequences (both captured at once: they reserve nothing)
    and ranges with their join, replayed as lengths shrink and grow again, with
    eager calls between: every replay has the eager call's bits."""
    import undertow_amd as U
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c = U.Context(0)
        pool = R.Pool(73, fmt, lens, 64, 512, 64, width=width // 64)
        q = [t.cuda() for t in pool.queries(M, H)]
        cache, table, n = pool.cuda(ctx=c), pool.table.cuda(), pool.lens32().cuda()
        out = torch.empty_like(q[0])
        if warm:
            cache.attend(table, n, *q, SCALE, out=out)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            cache.attend(table, n, *q, SCALE, out=out)
        for less in (0, 25, 125, 0, 500):
            n.copy_((pool.lens32().cuda() - less).clamp(min=0))
            out.fill_(7.0)
            graph.replay()
            s.synchronize()
            got = out.clone()
            assert torch.equal(got, cache.attend(table, n, *q, SCALE))
            c.synchronize()
            assert torch.isfinite(got).all()
