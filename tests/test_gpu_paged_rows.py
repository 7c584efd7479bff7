"""Prompt-sized calls of the paged latent cache's attention on the GPU: their
values against 64 bits, and what they reserve."""
import pytest
import torch

import paged_ref as R
from test_gpu_paged import SCALE, close

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
