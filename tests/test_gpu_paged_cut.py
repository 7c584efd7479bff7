"""Batches of paged attention that are cut into ranges although each sequence
has a workgroup: long tables over ragged lengths, on the GPU."""
import pytest
import torch

import paged_ref as R
from test_gpu_paged import SCALE
from test_gpu_paged_rows import check, reserved

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,B,M,H,width", [("bf16", 256, 1, 128, 4096), ("bf16", 64, 4, 128, 8192),
                                             ("bf16", 128, 2, 128, 8192), ("f16x2", 128, 1, 128, 8192)])
def test_a_long_sequence_among_short_ones_is_cut(ctx, fmt, B, M, H, width):
    """One sequence far longer than the rest spreads over the device: the call
    has parts to join, and every row its value."""
    lens = [(37 * k) % 90 for k in range(B)]
    lens[B // 3] = 1500
    pool = R.Pool(41, fmt, lens, 64, 512, 64, width=width // 64)
    qabs, qrope = pool.queries(M, H)
    cache, table, n = pool.cuda(ctx=ctx), pool.table.cuda(), pool.lens32().cuda()
    q = qabs.cuda(), qrope.cuda()
    out = torch.empty_like(q[0])
    assert reserved(ctx, lambda: cache.attend(table, n, *q, SCALE, out=out))[1] == 1
    check(pool, fmt, out, qabs, qrope)


@pytest.mark.parametrize("fmt,H", [("bf16", 16), ("bf16", 64), ("bf16", 128), ("f16x2", 16), ("f16x2", 128)])
@pytest.mark.parametrize("empty", [False, True])
def test_more_sequences_than_threads_are_cut(ctx, fmt, H, empty):
    """A range looks its sequence up over several turns of its workgroup, which
    also writes the first tiles down for the join; long runs of sequences
    without positions among them."""
    lens = [0 if empty and k % 300 > 30 else (37 * k) % 90 for k in range(700)]
    lens[650], lens[40] = 400, 300
    pool = R.Pool(59, fmt, lens, 64, 512, 64, width=9000 // 64)
    qabs, qrope = pool.queries(1, H)
    cache, table, n = pool.cuda(ctx=ctx), pool.table.cuda(), pool.lens32().cuda()
    q = qabs.cuda(), qrope.cuda()
    out = torch.full_like(q[0], 7.0)
    assert reserved(ctx, lambda: cache.attend(table, n, *q, SCALE, out=out))[1] == 1
    check(pool, fmt, out, qabs, qrope)


@pytest.mark.parametrize("fmt,H", [("bf16", 16), ("bf16", 128), ("f16x2", 16), ("f16x2", 128)])
@pytest.mark.parametrize("B,M", [(700, 1), (190, 3), (40, 2)])
def test_lists_of_many_rows_are_cut(ctx, fmt, H, B, M):
    """The same for rows with lists of their own, most places of them empty,
    some rows with none."""
    lens = [(37 * k) % 200 for k in range(B)]
    lens[B - 7] = 900
    pool = R.Pool(61, fmt, lens, 64, 512, 64, width=9000 // 64)
    qabs, qrope = pool.queries(M, H)
    sel = torch.full((B, M, 100), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for j, s in enumerate(R.seen(n, M)):
            ids = torch.randperm(-(-s // 64), generator=pool.g).int()
            if b % 9 != 5:
                sel[b, j, torch.randperm(100, generator=pool.g)[:len(ids)].sort().values] = ids
    cache, table, n = pool.cuda(ctx=ctx), pool.table.cuda(), pool.lens32().cuda()
    q = qabs.cuda(), qrope.cuda()
    out = torch.full_like(q[0], 7.0)
    assert reserved(ctx, lambda: cache.attend_pages(table, n, *q, SCALE, sel.cuda(), out=out))[1] == 1
    check(pool, fmt, out, qabs, qrope, sel)
