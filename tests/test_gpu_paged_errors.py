"""Bad lengths and pages of the paged calls on the GPU: what is left alone and
what is reported."""
import pytest
import torch

import paged_ref as R
from test_gpu_paged import pages_in_order

pytestmark = pytest.mark.gpu
FMTS = ["bf16", "f16x2"]


def bad_page(ctx):
    import undertow_amd as U
    with pytest.raises(U.UtError) as e:
        ctx.synchronize()
    assert e.value.code == U.runtime.UT_ERR_BAD_PAGE
    ctx.synchronize()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("summaries", [True, False])
@pytest.mark.parametrize("rows,over", [(1, 1), (4, 1), (4, 3), (40, 7), (2, 1000), (3, 2**31 - 113)])
def test_append_past_the_table_writes_nothing(ctx, fmt, summaries, rows, over):
    """A sequence one position (and more) longer than its table: its pages and
    their summaries stay as they are to the bit, and the others' rows are
    written."""
    cap = 7 * 16
    pool = R.Pool(43, fmt, [100, cap, 80], 16, 512, 64)
    mean, scale = pages_in_order(pool)
    more = dict(mean=mean.cuda(), mean_scale=scale.cuda()) if summaries else {}
    cache = pool.cuda(ctx=ctx, **more)
    table, lens = pool.table.cuda(), pool.lens32().cuda()
    lens[1] = cap + over
    x = pool.randn(3, rows, 576)
    cache.append(table, lens, x[..., :512].contiguous().cuda(), x[..., 512:].contiguous().cuda())
    bad_page(ctx)
    for b in (0, 2):
        n = pool.lens[b]
        pool.put(b, n - rows, x[b])
        for k in range((n - rows) // 16, -(-n // 16)):
            at = pool.table[b, k].long()
            mean[at], scale[at] = R.summary(pool.rows(b, torch.arange(k * 16, min(n, (k + 1) * 16))))
    assert torch.equal(cache.pages.cpu().view(torch.int16), pool.pages.view(torch.int16))
    if summaries:
        assert torch.equal(cache.mean.cpu(), mean)
        assert torch.equal(cache.mean_scale.cpu().view(torch.int32), scale.view(torch.int32))


def test_an_expert_error_does_not_hide_a_page_error(ctx):
    """Both found before one synchronize: one each from two of them."""
    import undertow_amd as U
    c = U.Context(0)
    H = 64
    w = lambda o, i: U.QTensor(c, U.INT8, torch.ones((o, i), dtype=torch.int8).numpy(), torch.ones(o).numpy(), o, i)
    experts = U.ExpertTable(c, 1, H, 32)
    experts.set(0, w(32, H), w(32, H), w(H, 32))
    x, one = torch.ones((1, H), device="cuda"), torch.ones((1, 1), device="cuda")
    pool = R.Pool(47, "bf16", [20], 16, 64, 16)
    q = [t.cuda() for t in pool.queries(1, 4)]
    cache, table = pool.cuda(ctx=c), pool.table.cuda()
    for order in ((0, 1), (1, 0)):
        for k in order:
            if k == 0:
                experts.moe_experts(torch.tensor([[9]], dtype=torch.int32, device="cuda"), one, x)
            else:
                cache.attend(table, torch.tensor([33], dtype=torch.int32, device="cuda"), *q, 0.1)
        codes = []
        for _ in range(2):
            with pytest.raises(U.UtError) as e:
                c.synchronize()
            codes.append(e.value.code)
        assert sorted(codes) == sorted([U.runtime.UT_ERR_BAD_EXPERT, U.runtime.UT_ERR_BAD_PAGE])
        c.synchronize()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,M,H,L,P,page,top_k,width", [
    ([400, 333, 100], 2, 32, 512, 64, 16, 6, 25), ([900], 1, 128, 512, 64, 64, 40, 20),
    ([500, 480] * 20, 1, 16, 512, 64, 8, 300, 63), ([300, 200], 2, 4, 64, 16, 8, 5, 38)])
def test_pages_that_no_row_lists_need_not_be_there(ctx, fmt, lens, M, H, L, P, page, top_k, width):
    """A window's old pages given back, their entries made invalid: lists of
    later pages, with empty places and pages behind the row's end among them,
    read as with a whole table and report nothing."""
    pool = R.Pool(53, fmt, lens, page, L, P, width=width)
    qabs, qrope = [t.cuda() for t in pool.queries(M, H)]
    sel = torch.full((len(lens), M, top_k), -1, dtype=torch.int32)
    table = torch.full_like(pool.table, -1)
    for b, n in enumerate(lens):
        last = (n - M) // page
        ids = range(max(1, last - 3), last + 1)
        sel[b, :, 1:1 + len(ids)] = torch.tensor(ids, dtype=torch.int32)
        sel[b, :, -1] = width + 5
        table[b, list(ids)] = pool.table[b, list(ids)]
    cache, n = pool.cuda(ctx=ctx), pool.lens32().cuda()
    want = cache.attend_pages(pool.table.cuda(), n, qabs, qrope, 0.07, sel.cuda())
    ctx.synchronize()
    got = cache.attend_pages(table.cuda(), n, qabs, qrope, 0.07, sel.cuda())
    ctx.synchronize()
    assert torch.equal(got, want) and torch.isfinite(want).all()


def test_a_new_cache_is_zero_before_the_context_writes_to_it(ctx):
    """Made on torch's stream, behind work that it still has to do, for a
    context on a stream of its own: what the context appends stays."""
    import undertow_amd as U
    c = U.Context(0, bind_torch_stream=False)
    lat, kr = torch.randn((1, 40, 512), device="cuda"), torch.randn((1, 40, 64), device="cuda")
    table = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([40], dtype=torch.int32, device="cuda")
    U.PagedCache.empty(c, 3, 16).append(table, lens, lat, kr)  # the first call's set-up
    c.synchronize()
    x = torch.randn((8192, 8192), device="cuda")
    torch.cuda.synchronize()
    for _ in range(4):
        x = (x @ x) * 1e-4
    cache = U.PagedCache.empty(c, 3, 16)
    cache.append(table, lens, lat, kr)
    c.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(cache.pages.flatten(0, 1)[:40], torch.cat([lat, kr], -1)[0].bfloat16())
    assert (cache.mean_scale > 0).all()
