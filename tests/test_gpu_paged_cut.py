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
