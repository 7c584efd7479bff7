"""Attention over 8-bit pages whose positions differ in size by more than f32's
range holds, or have the smallest and largest sizes, against 64 bits.

Tolerances stand at paged8_ref.close; everything is taken times 2^-size, size
the largest of the sequence's positions, so that they are relative to it."""
import pytest
import torch

import paged8_ref as R8
import paged_ref as R
from test_gpu_paged import SCALE

pytestmark = pytest.mark.gpu
WIDTHS = [(128, 512, 64), (16, 512, 64), (4, 64, 16)]
ZERO = None  # a position whose latent values are zeros


def sized(seed, runs, scale, H, L, P):
    """A pool of sequences whose latent values have sizes runs[b] = [(positions,
    log2 of their size), ..], and queries.  Head 0's are zeros, so that all its
    weights are equal; latent queries meet the largest values at size 1, those
    beyond 2^100 are zeros (a query's own range)."""
    runs = [[(n * scale, s) for n, s in run] for run in runs]
    pool = R8.Pool8(seed, [sum(n for n, _ in run) for run in runs], 64, L, P)
    qabs, qrope = pool.queries(1, H)
    qrope[:, :, 0] = 0.0
    sizes = []
    for b, run in enumerate(runs):
        at, top = 0, max([s for _, s in run if s is not ZERO], default=0)
        for n, s in run:
            x = pool.randn(n, L + P)
            x[:, :L] *= 0.0 if s is ZERO else 2.0 ** s
            pool.put(b, at, x)
            at += n
        qabs[b] *= 2.0 ** -top if 0 < top <= 100 else 0.0 if top > 0 else 1.0
        sizes.append(top)
    qabs[:, :, 0] = 0.0
    return pool, qabs, qrope, sizes


def compare(pool, qabs, qrope, sizes, got, **near):
    L = pool.L
    for b, n in enumerate(pool.lens):
        kv = pool.rows(b, R8.positions(n, **near)).cuda()
        q = torch.cat([qabs[b, 0], qrope[b, 0]], -1).double().cuda()
        out, spread, mass = R.attend(kv, q, L, SCALE)
        down = 2.0 ** -sizes[b]
        R8.close("i8", got[b, 0].double() * down, out * down, spread * down, mass * down,
                 R8.score_step(kv, q, L, SCALE)[:, None].cpu(), R8.largest(kv, q, L, SCALE).cpu() * down)


def attend(ctx, pool, qabs, qrope, **near):
    cache, where = pool.cuda(ctx=ctx), (pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE)
    got = cache.attend_window(*where, near["window"], near["sinks"]) if near else cache.attend(*where)
    ctx.synchronize()
    return got


@pytest.mark.parametrize("scale", [1, 60])  # whole, and cut into ranges
@pytest.mark.parametrize("H,L,P", WIDTHS)
@pytest.mark.parametrize("run", [
    [(40, -60), (60, 70)], [(60, 70), (40, -60)], [(40, -100), (60, 20)], [(40, -100), (60, 100)], [(60, 100), (40, -100)],
    [(30, -100), (30, 0), (30, 100)], [(30, 0), (64, -100), (31, 90)]])
def test_sizes_further_apart_than_f32_holds(ctx, run, H, L, P, scale):
    """All positions keep their weight in the sum, whatever their size."""
    case = sized(61, [run, [(9, run[0][1])]], scale, H, L, P)
    compare(*case, attend(ctx, *case[:3]))


@pytest.mark.parametrize("scale", [1, 60])
@pytest.mark.parametrize("H,L,P", WIDTHS)
@pytest.mark.parametrize("size", [-110, -90, -80, -40, 0, 90])
def test_zeros_before_values_of_any_size(ctx, size, H, L, P, scale):
    """Positions of zero latent values weigh, and settle nothing about the
    others' size; a sequence of them alone has a context of zeros."""
    case = sized(62, [[(40, ZERO), (60, size)], [(70, ZERO)], [(3, size), (40, ZERO), (64, size)]], scale, H, L, P)
    got = attend(ctx, *case[:3])
    assert (got[1] == 0).all()
    compare(*case, got)


@pytest.mark.parametrize("H,L,P", WIDTHS)
def test_sizes_in_a_window(ctx, H, L, P):
    case = sized(63, [[(40, -100), (300, ZERO), (70, 100)], [(40, 80), (300, 0), (70, -90)]], 1, H, L, P)
    compare(*case, attend(ctx, *case[:3], window=90, sinks=35), window=90, sinks=35)


@pytest.mark.parametrize("scale", [1, 120])
@pytest.mark.parametrize("H,L,P", WIDTHS)
@pytest.mark.parametrize("size", [-115, 115])
def test_smallest_and_largest_sizes(ctx, size, H, L, P, scale):
    """Contexts of bf16's smallest normal numbers and of its largest."""
    case = sized(64, [[(70, size)], [(30, size)]], scale, H, L, P)
    compare(*case, attend(ctx, *case[:3]))


@pytest.mark.parametrize("scale", [1, 120])
@pytest.mark.parametrize("H", [128, 16])
def test_sums_of_the_largest_values(ctx, H, scale):
    """Many values near f32's largest, all of one sign: neither a part's context
    nor the parts' sum leaves the range that their mean lies in."""
    case = sized(65, [[(70, 122)], [(30, 0), (40, 122)]], scale, H, 512, 64)
    pool = case[0]
    pool.pages[..., :512] = pool.pages[..., :512].clamp(min=-127).abs()
    compare(*case, attend(ctx, *case[:3]))


@pytest.mark.parametrize("size", [-118, 0, 118])
def test_long_prompts_of_the_smallest_and_largest_sizes(ctx, size):
    """Rows whose sequence no other workgroup shares, and so no join, over
    thousands of positions of like weight."""
    M, H, n = 300, 128, 8400
    pool = R8.Pool8(66, [n], 64, 512, 64, fill=False)
    x = pool.randn(n, 576)
    x[:, :512] *= 2.0 ** size
    x[:, :512] += 2.0 ** (size + 1)  # means as large as the values
    pool.put(0, 0, x)
    qabs, qrope = pool.queries(M, H)
    qabs.zero_()
    qrope[:, :, 0] = 0.0
    got = pool.cuda(ctx=ctx).attend(pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE)
    ctx.synchronize()
    down = 2.0 ** -size
    for j in (0, 151, 299):
        kv = pool.rows(0, torch.arange(n - M + j + 1)).cuda()
        q = torch.cat([qabs[0, j], qrope[0, j]], -1).double().cuda()
        out, spread, mass = R.attend(kv, q, 512, SCALE)
        R8.close("i8", got[0, j].double() * down, out * down, spread * down, mass * down,
                 R8.score_step(kv, q, 512, SCALE)[:, None].cpu(), R8.largest(kv, q, 512, SCALE).cpu() * down)


@pytest.mark.parametrize("scale", [1, 60])
@pytest.mark.parametrize("H", [128, 16])
def test_scores_below_f32_before_others(ctx, H, scale):
    """Positions whose scores are -inf in f32 weigh nothing, and those behind
    them, far below 0 themselves, share the whole weight."""
    n, far = 100 * scale, 40 * scale
    pool = R8.Pool8(67, [n, 70], 64, 512, 64, fill=False)
    for b, m in enumerate((n, 70)):
        x = pool.randn(m, 576)
        size = torch.full((m, 1), 2.0 ** -100)
        size[:far if b == 0 else 33] = 2.0 ** 40
        x[:, :512] = x[:, :512].abs() * size
        x[:, 512:] = 1.0 + x[:, 512:] * 0.05
        pool.put(b, 0, x)
    qabs, qrope = pool.queries(1, H)
    qabs, qrope = -(qabs.abs() * 2.0 ** 100), -(qrope.abs() + 40.0)
    got = attend(ctx, pool, qabs, qrope)
    for b, m in enumerate((n, 70)):
        kv = pool.rows(b, torch.arange(far if b == 0 else 33, m)).cuda()
        q = torch.cat([qabs[b, 0], qrope[b, 0]], -1).double().cuda()
        assert float((q @ kv.T * SCALE).max()) < -150.0
        out, spread, mass = R.attend(kv, q, 512, SCALE)
        # f32 scores of size s carry s 2^-22 or so, beside the queries' steps
        step = R8.score_step(kv, q, 512, SCALE)[:, None].cpu() + float((q @ kv.T * SCALE).abs().max()) * 2.0 ** -21
        up = 2.0 ** 100
        R8.close("i8", got[b, 0].double() * up, out * up, spread * up, mass * up, step, R8.largest(kv, q, 512, SCALE).cpu() * up)


@pytest.mark.parametrize("order", [[0, 1, 2, 3, 4, 5], [5, 4, 3, 2, 1, 0], [2, 5, 0, -1, 4]])
@pytest.mark.parametrize("H", [128, 16])
def test_sizes_on_listed_pages(ctx, H, order):
    pool, qabs, qrope, sizes = sized(68, [[(64, -100), (64, ZERO), (64, 100), (64, 0), (64, -115), (30, 100)]], 1, H, 512, 64)
    sel = torch.tensor([[order]], dtype=torch.int32)
    got = pool.cuda(ctx=ctx).attend_pages(pool.table.cuda(), pool.lens32().cuda(), qabs.cuda(), qrope.cuda(), SCALE, sel.cuda())
    ctx.synchronize()
    at = torch.cat([torch.arange(64 * k, min(64 * k + 64, 350)) for k in order if k >= 0])
    kv = pool.rows(0, at).cuda()
    q = torch.cat([qabs[0, 0], qrope[0, 0]], -1).double().cuda()
    out, spread, mass = R.attend(kv, q, 512, SCALE)
    down = 2.0 ** -100
    R8.close("i8", got[0, 0].double() * down, out * down, spread * down, mass * down,
             R8.score_step(kv, q, 512, SCALE)[:, None].cpu(), R8.largest(kv, q, 512, SCALE).cpu() * down)
