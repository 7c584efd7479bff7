"""The paged latent cache and what reads it, as a program that serves many
sequences of a DeepSeek-V3-style model at once calls them.

Four operators over one pool of pages that the sequences share (a sequence's
pages stand in its row of a table; ``lens`` counts its positions, the rows of
the present step included, so row j of M sees ``lens - M + j + 1`` of them):

- ``append``: a step's latent and rotated key rows into the pages, and each
  touched page's summary (the mean row in 8 bits) anew;
- ``attend``: absorbed attention of every sequence's rows over its pages;
- ``select``: the pages a row shall attend to, by a score of the summaries;
- ``sparse``: absorbed attention over the selected pages only.

Pages hold bf16 (queries and outputs in bf16 too), or pairs of f16 that stand
for f32 (``x = hi + lo / 2048``, queries and outputs in f32).  Sizes are
DeepSeek-V3's (128 heads, latent 512 + rope 64; fewer heads where they are
split over devices) and config 1's tiny model.
"""
import functools
import math
import random

import torch

own = False

WIDE, TINY = (512, 64), (64, 16)
SCALE = 1.0 / math.sqrt(192.0)
KEEP_FIRST, KEEP_LAST = 1, 2
LARGEST = 64 * 128 * 4608  # sequences x heads x positions of attend_batch, about


def listed():
    return [
        # a decode step of 48 ragged sequences writes one row each: latency
        dict(name="append_step", kind="append", fmt="bf16", shape="wide", page=64, batch=48, rows=1, ctx=2500),
        # prompts of three sequences, a chunk of 777 rows each, kept to f32's accuracy
        dict(name="append_prompts", kind="append", fmt="f16x2", shape="wide", page=64, batch=3, rows=777, ctx=1900),
        # one sequence's token over a short context: latency
        dict(name="attend_one", kind="attend", fmt="bf16", shape="wide", page=64, batch=1, rows=1, ctx=509, heads=128),
        # a serving batch's decode step, every length up to 8192
        dict(name="attend_batch", kind="attend", fmt="bf16", shape="wide", page=64, batch=64, rows=1, ctx=8192, heads=128),
        # two verify rows of a few long conversations
        dict(name="attend_verify", kind="attend", fmt="bf16", shape="wide", page=64, batch=4, rows=2, ctx=32768, heads=128),
        # an eighth of the heads (split over eight devices), small pages, an odd batch
        dict(name="attend_shard", kind="attend", fmt="bf16", shape="wide", page=16, batch=37, rows=1, ctx=6001, heads=16),
        # three verify rows at f32's accuracy
        dict(name="attend_pairs", kind="attend", fmt="f16x2", shape="wide", page=32, batch=11, rows=3, ctx=4099, heads=128),
        # the pages of one row of a long context: latency
        dict(name="select_one", kind="select", fmt="bf16", shape="wide", page=64, batch=1, rows=1, ctx=32768, heads=128, top_k=32),
        # of a batch's verify rows
        dict(name="select_batch", kind="select", fmt="bf16", shape="wide", page=64, batch=24, rows=2, ctx=40000, heads=128, top_k=48),
        # one row over 32 of its 512 pages
        dict(name="sparse_one", kind="sparse", fmt="bf16", shape="wide", page=64, batch=1, rows=1, ctx=32768, heads=128, top_k=32),
        # a batch's verify rows, each over pages of its own
        dict(name="sparse_batch", kind="sparse", fmt="bf16", shape="wide", page=64, batch=24, rows=2, ctx=16000, heads=128, top_k=48),
        # half the heads at f32's accuracy, small pages
        dict(name="sparse_pairs", kind="sparse", fmt="f16x2", shape="wide", page=32, batch=13, rows=1, ctx=9001, heads=64, top_k=40),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "select", "sparse", "sparse"])
    shape = "tiny" if rng.random() < 0.12 else "wide"
    c = dict(kind=kind, fmt=rng.choice(["bf16", "bf16", "f16x2"]), shape=shape, page=rng.choice([16, 32, 64, 64, 128]))
    if kind == "append":
        c["rows"] = rng.choice([1, 1, 2, 3, 4, _log(rng, 5, 1500)])
        c["batch"] = _log(rng, 1, 96 if c["rows"] < 5 else max(1, 2300 // c["rows"]))
        c["ctx"] = c["rows"] + _log(rng, 1, 4000)
        return c
    c["rows"], c["batch"] = rng.choice([1, 1, 1, 2, 3, 4]), _log(rng, 1, 64)
    c["heads"] = 4 if shape == "tiny" else rng.choice([128, 128, 128, 64, 32, 16])
    most = LARGEST // (c["batch"] * c["rows"] * max(32, c["heads"]))
    if c["fmt"] == "f16x2":
        most //= 4  # its products cost three times a bf16 one's, its rows twice the bytes
    if shape == "tiny":
        most = min(most, 1500)
    c["ctx"] = max(8, _log(rng, 16, min(32768, most)))
    if kind != "attend":
        c["top_k"] = _log(rng, 4, 64)
    if kind == "sparse":
        c["top_k"] = max(4, min(c["top_k"], most // c["page"]))
    if c["batch"] > 2 and kind != "select" and rng.random() < 0.4:
        c["pad"] = rng.randint(1, 2)  # sequences of a batch padded to a fixed size: nothing to see
    return c


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 29)


def _lens(case):
    """Ragged lengths, the longest first; as many empty ones last as the case pads with."""
    n, m, ctx = case["batch"], case["rows"], case["ctx"]
    lens = [ctx] + [max(m, int(ctx * ((k * 0.6180339887) % 1.0))) for k in range(1, n)]
    pad = case.get("pad", 0)
    return lens[:n - pad] + [0] * pad


def _width(case):
    return -(-case["ctx"] // case["page"])


def _shape(case):
    return WIDE if case["shape"] == "wide" else TINY


def _stored(fmt, x):
    """f32 values as a page holds them: bf16, or the two planes of f16."""
    if fmt == "bf16":
        return x.bfloat16()
    hi = x.half()
    return torch.stack([hi, ((x - hi.float()) * 2048.0).half()], -2)


def _values(fmt, rows):
    """The values that stored rows stand for, in f32."""
    if fmt == "bf16":
        return rows.float()
    return rows[..., 0, :].float() + rows[..., 1, :].float() / 2048.0


def _summary(fmt, rows, live):
    """Codes and scales of the mean rows of pages [..., page, row], over the live positions [..., page]."""
    s = (_values(fmt, rows).double() * live[..., None]).sum(-2)
    top = s.abs().amax(-1)
    codes = torch.round(s * 127.0 / torch.where(top > 0, top, 1.0)[..., None])
    return codes.to(torch.int8), (top / (127.0 * live.sum(-1).clamp(min=1))).float()


def _pool(case, seed):
    """The pool, its table and lengths.  Pages stand in the pool in any order, and rows behind a
    sequence's end hold what was there before; a page's rows are alike, as a text's passages are."""
    g, page, (L, P) = _gen(seed), case["page"], _shape(case)
    order = random.Random(seed * 31 + 7)
    lens = _lens(case)
    order.shuffle(lens)
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + 3
    ids = list(range(n_pages))
    order.shuffle(ids)
    table, at = [[-1] * _width(case) for _ in lens], 0
    for row, k in zip(table, need):
        row[:k] = ids[at:at + k]
        at += k
    x = torch.randn((n_pages, page, L + P), device="cuda", generator=g)
    x += 0.6 * torch.randn((n_pages, 1, L + P), device="cuda", generator=g)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return g, _stored(case["fmt"], x), i32(table), i32(lens)


@functools.lru_cache(None)
def _context():
    """The one context of a serving program."""
    import undertow_amd as U
    return U.Context(0)


def prepare(case, seed):
    g, pages, table, lens = _pool(case, seed)
    L, P = _shape(case)
    B, M = case["batch"], case["rows"]
    st = dict(kind=case["kind"], fmt=case["fmt"], page=case["page"], L=L, pages=pages, table=table, lens=lens)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    live = torch.ones(pages.shape[:2], dtype=torch.float64, device="cuda")
    if case["kind"] in ("append", "select"):
        st["mean"], st["mean_scale"] = _summary(case["fmt"], pages, live)
    if case["kind"] == "append":
        st["latent"], st["krot"] = rnd(B, M, L), rnd(B, M, P)
    else:
        st["rows"] = M
        q = torch.bfloat16 if case["fmt"] == "bf16" else torch.float32
        st["qabs"], st["q_rope"] = rnd(B, M, case["heads"], L).to(q), rnd(B, M, case["heads"], P).to(q)
    if "top_k" in case:
        st["top_k"] = case["top_k"]
    if case["kind"] == "sparse":  # a choice in ascending order, the first and the last pages among it
        n = (lens[:, None] - M + torch.arange(1, M + 1, device="cuda")).clamp(min=0)
        score = rnd(B, M, _width(case)).double()
        st["sel"] = _pick(score, -(-n // case["page"]), case["top_k"])
    if own:
        import undertow_amd as U
        st["cache"] = U.PagedCache(_context(), pages, latent=L, rope=P, mean=st.get("mean"), mean_scale=st.get("mean_scale"))
    return st


# ------------------------------------------------------------- plain forms
def _positions(st):
    """Positions that each row sees: [B, M]."""
    m = st["rows"]
    return (st["lens"][:, None] - m + torch.arange(1, m + 1, device=st["lens"].device)).clamp(min=0).long()


def _attention(q, kv, L, seen):
    """q [N, R, D] over kv [N, T, D] where seen [N, R, T] says so; a row that sees nothing gets zeros."""
    s = (torch.bmm(q, kv.transpose(1, 2).contiguous()) * SCALE).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    return torch.bmm(p, kv[..., :L].contiguous()) / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _attend(st):
    B, M, H, L = st["qabs"].shape
    kv = _values(st["fmt"], st["pages"][st["table"].clamp(min=0).long()]).flatten(1, 2)
    q = torch.cat([st["qabs"], st["q_rope"]], -1).float().reshape(B, M * H, -1)
    seen = torch.arange(kv.shape[1], device=kv.device) < _positions(st)[..., None]
    out = _attention(q, kv, L, seen.repeat_interleave(H, 1))
    return out.reshape(B, M, H, L).to(st["qabs"].dtype)


def _sparse(st):
    B, M, H, L = st["qabs"].shape
    page, sel = st["page"], st["sel"].long()
    phys = st["table"].long()[:, None].expand(B, M, -1).gather(2, sel.clamp(min=0))
    kv = _values(st["fmt"], st["pages"][phys.clamp(min=0)]).reshape(B * M, -1, L + st["q_rope"].shape[-1])
    at = sel[..., None] * page + torch.arange(page, device=sel.device)
    seen = ((at < _positions(st)[..., None, None]) & (sel >= 0)[..., None]).reshape(B * M, 1, -1)
    q = torch.cat([st["qabs"], st["q_rope"]], -1).float().reshape(B * M, H, -1)
    return _attention(q, kv, L, seen).reshape(B, M, H, L).to(st["qabs"].dtype)


def _pick(score, n_pages, top_k):
    """The first and last pages and then the best scores, ties to the lowest page; ascending, -1 behind them."""
    W = score.shape[-1]
    at = torch.arange(W, device=score.device)
    forced = (at < KEEP_FIRST) | (at >= n_pages[..., None] - KEEP_LAST)
    score = torch.where(forced, math.inf, score).masked_fill(at >= n_pages[..., None], -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top_k]
    best = torch.where(best < n_pages[..., None], best, W).sort(-1).values
    best = torch.where(best < W, best, -1)
    return torch.nn.functional.pad(best, (0, top_k - best.shape[-1]), value=-1).int()


def _select(st):
    B, M, H, _ = st["qabs"].shape
    q = torch.cat([st["qabs"], st["q_rope"]], -1).double()
    top = q.abs().amax(-1)
    codes = torch.round(q * 127.0 / torch.where(top > 0, top, 1.0)[..., None]).float().reshape(B, M * H, -1)
    at = st["table"].clamp(min=0).long()
    # sums of 576 products of 7 bits are whole numbers under 2^24: exact in f32
    dots = torch.bmm(codes, st["mean"][at].float().transpose(1, 2).contiguous()).reshape(B, M, H, -1)
    score = (dots.clamp(min=0).double() * (top / 127.0)[..., None]).sum(2) * st["mean_scale"][at].double()[:, None]
    return _pick(score, -(-_positions(st) // st["page"]), st["top_k"])


def _append(st):
    M, page, pages, lens = st["latent"].shape[1], st["page"], st["pages"], st["lens"].long()
    table = st["table"].long()
    pos = lens[:, None] - M + torch.arange(M, device=lens.device)
    phys = table.gather(1, pos // page)
    pages[phys, pos % page] = _stored(st["fmt"], torch.cat([st["latent"], st["krot"]], -1))
    # the pages that the rows fall into, the last one again where a sequence touches fewer than another
    first, last = pos[:, :1] // page, pos[:, -1:] // page
    at = torch.minimum(first + torch.arange((M + page - 2) // page + 1, device=lens.device), last)
    touched = table.gather(1, at)
    live = (at[..., None] * page + torch.arange(page, device=lens.device) < lens[:, None, None]).double()
    st["mean"][touched], st["mean_scale"][touched] = _summary(st["fmt"], pages[touched], live)


def run(st):
    kind = st["kind"]
    if own:
        c, where = st["cache"], (st["table"], st["lens"])
        if kind == "attend":
            return c.attend(*where, st["qabs"], st["q_rope"], SCALE)
        if kind == "sparse":
            return c.attend_pages(*where, st["qabs"], st["q_rope"], SCALE, st["sel"])
        if kind == "select":
            return c.select(*where, st["qabs"], st["q_rope"], st["top_k"], keep_first=KEEP_FIRST, keep_last=KEEP_LAST)
        c.append(*where, st["latent"], st["krot"])
    elif kind != "append":
        return {"attend": _attend, "sparse": _sparse, "select": _select}[kind](st)
    else:
        _append(st)
    return dict(pages=st["pages"], mean=st["mean"] * st["mean_scale"][:, None])


# -------------------------------------------------------------- accounting
def work(case):
    L, P = _shape(case)
    D, page, B, M = L + P, case["page"], case["batch"], case["rows"]
    row = D * (2 if case["fmt"] == "bf16" else 4)
    lens = _lens(case)
    if case["kind"] == "append":
        touched = [(n - 1) // page - (n - M) // page + 1 for n in lens]
        older = sum((n - M) % page for n in lens)
        return dict(bytes=B * M * (D * 4 + row) + older * row + sum(touched) * (D + 4), flops=(B * M + older) * D)
    H, q = case["heads"], 2 if case["fmt"] == "bf16" else 4
    seen = [[max(0, n - M + j + 1) for j in range(M)] for n in lens]
    if case["kind"] == "attend":
        return dict(bytes=sum(lens) * row + B * M * H * (D + L) * q, flops=2 * H * (D + L) * sum(map(sum, seen)))
    most = [[-(-n // page) for n in r] for r in seen]
    if case["kind"] == "select":
        return dict(bytes=sum(max(r) for r in most) * (D + 4) + B * M * (H * D * q + 4 * case["top_k"]), flops=2 * H * D * sum(map(sum, most)))
    # a row's chosen pages are full but for the last
    rows = [[min(k, case["top_k"]) * page - (-n) % page for n, k in zip(r, m) if n] for r, m in zip(seen, most)]
    total = sum(map(sum, rows))
    shared = sum(min(sum(r), n) for r, n in zip(rows, lens))
    return dict(bytes=shared * row + B * M * H * (D + L) * q, flops=2 * H * (D + L) * total)


# ------------------------------------------------------- 64-bit references
def _exact_rows(case, pages, table, at):
    """Row values of one sequence at positions `at`, in 64 bits."""
    x = pages[table[at // case["page"]].long(), at % case["page"]]
    return x.double() if case["fmt"] == "bf16" else x[:, 0].double() + x[:, 1].double() * 2.0 ** -11


def _exact_mean(case, pages, phys, live):
    x = pages[phys, :live]
    s = (x.double() if case["fmt"] == "bf16" else x[:, 0].double() + x[:, 1].double() * 2.0 ** -11).sum(0)
    top = s.abs().max()
    return torch.round(s * 127.0 / top) * (top / (127.0 * live)).float().double() if top > 0 else s * 0


def exact(case, seed):
    st = prepare(case, seed)
    pages, table, lens = st["pages"], st["table"], st["lens"].tolist()
    M, page, L = case["rows"], case["page"], st["L"]
    if case["kind"] == "append":
        x = torch.cat([st["latent"], st["krot"]], -1)
        means = st["mean"].double() * st["mean_scale"].double()[:, None]
        whole = pages.double()
        for b, n in enumerate(lens):
            at = torch.arange(n - M, n, device="cuda")
            phys, off = table[b][at // page].long(), at % page
            if case["fmt"] == "bf16":
                pages[phys, off], whole[phys, off] = x[b].bfloat16(), x[b].double()
            else:
                hi = x[b].half()
                rest = (x[b].double() - hi.double()) * 2.0 ** 11
                pages[phys, off] = torch.stack([hi, rest.half()], 1)
                whole[phys, off] = torch.stack([hi.double(), rest], 1)
            for k in range((n - M) // page, (n - 1) // page + 1):
                means[table[b, k].long()] = _exact_mean(case, pages, table[b, k].long(), min(page, n - k * page))
        return dict(pages=whole, mean=means)
    q = torch.cat([st["qabs"], st["q_rope"]], -1).double()
    if case["kind"] == "select":
        out = torch.full((case["batch"], M, case["top_k"]), -1, dtype=torch.int32)
        for b, n in enumerate(lens):
            for j in range(M):
                k = -(-(n - M + j + 1) // page)
                at = table[b, :k].long()
                top = q[b, j].abs().amax(-1)
                dots = torch.round(q[b, j] * 127.0 / top[:, None]) @ st["mean"][at].double().T
                score = (dots.relu() * (top / 127.0)[:, None]).sum(0) * st["mean_scale"][at].double()
                score = score.tolist()
                forced = set(range(min(KEEP_FIRST, k))) | set(range(max(0, k - KEEP_LAST), k))
                rest = sorted((p for p in range(k) if p not in forced), key=lambda p: (-score[p], p))
                got = sorted(sorted(forced) + rest[:max(0, case["top_k"] - len(forced))])
                out[b, j, :len(got)] = torch.tensor(got, dtype=torch.int32)
        return out
    out = torch.zeros(st["qabs"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        for j in range(M):
            sees = n - M + j + 1
            if sees <= 0:
                continue
            at = torch.arange(sees, device="cuda")
            if case["kind"] == "sparse":
                chosen = st["sel"][b, j][st["sel"][b, j] >= 0].long()
                at = (chosen[:, None] * page + torch.arange(page, device="cuda")).flatten()
                at = at[at < sees]
            kv = _exact_rows(case, pages, table[b], at)
            out[b, j] = torch.softmax(q[b, j] @ kv.T * SCALE, -1) @ kv[:, :L]
    return out
