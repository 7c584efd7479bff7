"""The paged latent cache in 8 bits, and attention with a window and a few
first positions, as a program that serves many sequences of a DeepSeek-V3-style
model at once calls them.

A sequence's pages stand in its row of a table; ``lens`` counts its positions,
the rows of the present step included, so row j of M sees ``lens - M + j + 1``
of them.  8-bit pages hold codes, and for each position a scale of its latent
part and one of its rotated key: ``scale = max|x| / 127``, ``code = rint(127 x
/ max|x|)``.  Five operators:

- ``append``: a step's rows quantised into their 8-bit pages, and each touched
  page's summary (the mean row in 8 bits) anew;
- ``read``: rows read back from the pages, in f32 or bf16;
- ``attend``: absorbed attention of every sequence's rows over its 8-bit pages;
- ``sparse``: the same over listed pages only;
- ``window``: absorbed attention of each row over the last ``window`` of the
  positions up to its own and the sequence's first ``sinks``, over pages of any
  format (bf16; pairs of f16, ``x = hi + lo / 2048``; 8 bits).

Queries and outputs are bf16, with pairs f32.  Sizes are DeepSeek-V3's (128
heads, latent 512 + rope 64; fewer heads where they are split over devices)
and config 1's tiny model.
"""
import functools
import math
import random

import torch

own = False

WIDE, TINY = (512, 64), (64, 16)
SCALE = 1.0 / math.sqrt(192.0)
LARGEST = 64 * 128 * 4608  # sequences x heads x positions of attend8_batch, about


def listed():
    return [
        # a decode step of 48 ragged sequences writes one row each: latency
        dict(name="append8_step", kind="append", fmt="i8", shape="wide", page=64, batch=48, rows=1, ctx=300),
        # prompts of three sequences, a chunk of 777 rows each
        dict(name="append8_prompts", kind="append", fmt="i8", shape="wide", page=64, batch=3, rows=777, ctx=1900),
        # a short sequence read back for the reconstructed form of attention: latency
        dict(name="read8_one", kind="read", fmt="i8", shape="wide", page=64, batch=1, rows=257, ctx=257, out="bf16"),
        # a ragged batch's whole contexts read back in f32, as a move to another pool does
        dict(name="read8_batch", kind="read", fmt="i8", shape="wide", page=64, batch=16, rows=8192, ctx=8192, out="f32"),
        # one sequence's token over a short context: latency
        dict(name="attend8_one", kind="attend", fmt="i8", shape="wide", page=64, batch=1, rows=1, ctx=509, heads=128),
        # a serving batch's decode step, every length up to 8192
        dict(name="attend8_batch", kind="attend", fmt="i8", shape="wide", page=64, batch=64, rows=1, ctx=8192, heads=128),
        # an eighth of the heads (split over eight devices), small pages, an odd batch of long contexts
        dict(name="attend8_shard", kind="attend", fmt="i8", shape="wide", page=16, batch=37, rows=1, ctx=12001, heads=16),
        # one row over 32 of its 512 pages: latency
        dict(name="sparse8_one", kind="sparse", fmt="i8", shape="wide", page=64, batch=1, rows=1, ctx=32768, heads=128, top_k=32),
        # a batch's verify rows, each over pages of its own
        dict(name="sparse8_batch", kind="sparse", fmt="i8", shape="wide", page=64, batch=24, rows=2, ctx=16000, heads=128, top_k=48),
        # one long conversation's token, the window and four first positions: latency
        dict(name="window_one", kind="window", fmt="bf16", shape="wide", page=64, batch=1, rows=1, ctx=16384, heads=128, window=1024, sinks=4),
        # a batch's two verify rows, windows longer than some of the sequences, over 8-bit pages
        dict(name="window8_batch", kind="window", fmt="i8", shape="wide", page=64, batch=40, rows=2, ctx=12000, heads=128, window=4096, sinks=64),
        # an odd batch's three verify rows at f32's accuracy, half the heads, an odd window
        dict(name="window_pairs", kind="window", fmt="f16x2", shape="wide", page=32, batch=13, rows=3, ctx=5003, heads=64, window=777, sinks=5),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "read", "attend", "attend", "attend", "sparse", "window", "window", "window"])
    shape = "tiny" if rng.random() < 0.12 else "wide"
    c = dict(kind=kind, fmt="i8", shape=shape, page=rng.choice([16, 32, 64, 64, 128]))
    if kind == "append":
        c["rows"] = rng.choice([1, 1, 2, 3, 4, _log(rng, 5, 1500)])
        c["batch"] = _log(rng, 1, 96 if c["rows"] < 5 else max(1, 2300 // c["rows"]))
        c["ctx"] = c["rows"] + _log(rng, 1, 600)
        return c
    if kind == "read":
        c["fmt"] = rng.choice(["i8", "i8", "bf16", "f16x2"])
        c["out"] = rng.choice(["f32", "bf16"])
        c["batch"] = _log(rng, 1, 48)
        c["ctx"] = _log(rng, 8, min(16384, 65536 // c["batch"]))
        c["rows"] = rng.choice([c["ctx"], max(1, c["ctx"] // 3)])
        return c
    c["rows"], c["batch"] = rng.choice([1, 1, 1, 2, 3, 4]), _log(rng, 1, 64)
    c["heads"] = 4 if shape == "tiny" else rng.choice([128, 128, 128, 64, 32, 16])
    if kind == "window":
        c["fmt"] = rng.choice(["i8", "i8", "bf16", "f16x2"])
    most = LARGEST // (c["batch"] * c["rows"] * max(32, c["heads"]))
    if c["fmt"] == "f16x2":
        most //= 4  # its products cost three times a bf16 one's, its rows twice the bytes
    if shape == "tiny":
        most = min(most, 1500)
    if kind == "window":
        c["window"] = max(8, _log(rng, 16, min(4096, most)))
        c["sinks"] = rng.choice([0, 1, 4, _log(rng, 5, 128)])
        c["ctx"] = max(8, _log(rng, 64, 16384 if c["batch"] < 24 else 8192))
    else:
        c["ctx"] = max(8, _log(rng, 16, min(32768, most)))
    if kind == "sparse":
        c["top_k"] = max(4, min(_log(rng, 4, 64), most // c["page"]))
    if c["batch"] > 2 and rng.random() < 0.4:
        c["pad"] = rng.randint(1, 2)  # sequences of a batch padded to a fixed size: nothing to see
    return c


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 6151 + 17)


def _lens(case):
    """Ragged lengths, the longest first; as many empty ones last as the case pads with."""
    n, m, ctx = case["batch"], case["rows"], case["ctx"]
    least = 1 if case["kind"] == "read" else m
    lens = [ctx] + [max(least, int(ctx * ((k * 0.6180339887) % 1.0))) for k in range(1, n)]
    pad = case.get("pad", 0)
    return lens[:n - pad] + [0] * pad


def _width(case):
    return -(-case["ctx"] // case["page"])


def _shape(case):
    return WIDE if case["shape"] == "wide" else TINY


def _parts(x, L):
    return x[..., :L], x[..., L:]


def _quantised(x, L):
    """Codes and scales of f32 rows, each part of a row by itself."""
    codes, scales = [], []
    for part in _parts(x, L):
        top = part.abs().amax(-1, keepdim=True).double()
        codes.append(torch.round(part.double() * 127.0 / torch.where(top > 0, top, 1.0)).to(torch.int8))
        scales.append((top / 127.0).float())
    return torch.cat(codes, -1), torch.cat(scales, -1)


def _values(pool, rows, scales=None):
    """The values that stored rows stand for, in f32 (in 64 bits where the scales are)."""
    if pool["fmt"] == "bf16":
        return rows.float()
    if pool["fmt"] == "f16x2":
        return rows[..., 0, :].float() + rows[..., 1, :].float() / 2048.0
    lat, rope = _parts(rows, pool["L"])
    return torch.cat([lat * scales[..., :1], rope * scales[..., 1:]], -1)


def _at(pool, *index):
    """The values of the pool's rows at an index."""
    return _values(pool, pool["pages"][index], pool["scales"][index] if "scales" in pool else None)


def _summary(st, pages, live):
    """Codes and scales of the mean rows of pages, over the live positions [..., page]; in 64 bits,
    since a mean next to a border between two codes takes one or the other."""
    s = (_values(st, st["pages"][pages], st["scales"][pages].double()) * live[..., None]).sum(-2)
    top = s.abs().amax(-1)
    codes = torch.round(s * 127.0 / torch.where(top > 0, top, 1.0)[..., None])
    return codes.to(torch.int8), (top / (127.0 * live.sum(-1).clamp(min=1))).float()


def _pool(case, seed):
    """The pool, its table and lengths.  Pages stand in the pool in any order, and rows behind a
    sequence's end hold what was there before; a page's rows are alike, as a text's passages are,
    and a text's first position is several times as large as the others."""
    g, page, (L, P) = _gen(seed), case["page"], _shape(case)
    order = random.Random(seed * 29 + 3)
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
    first = [row[0] for row, k in zip(table, need) if k]
    x[first, 0] *= 3.0
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    st = dict(case, L=L, P=P, table=i32(table), lens=i32(lens))
    if case["fmt"] == "i8":
        codes, scales = zip(*(_quantised(part, L) for part in x.split(1024)))
        st["pages"], st["scales"] = torch.cat(codes), torch.cat(scales)
    elif case["fmt"] == "bf16":
        st["pages"] = x.bfloat16()
    else:
        hi = x.half()
        st["pages"] = torch.stack([hi, ((x - hi.float()) * 2048.0).half()], -2)
    return g, st


@functools.lru_cache(None)
def _context():
    """The one context of a serving program."""
    import undertow_amd as U
    return U.Context(0)


def prepare(case, seed):
    g, st = _pool(case, seed)
    B, M = case["batch"], case["rows"]
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    if case["kind"] == "append":
        st["mean"], st["mean_scale"] = _summary(st, slice(None), torch.ones(st["pages"].shape[:2], dtype=torch.float64, device="cuda"))
        st["latent"], st["krot"] = rnd(B, M, st["L"]), rnd(B, M, st["P"])
    elif case["kind"] == "read":  # the last rows of each sequence, or all of a shorter one
        st["starts"] = (st["lens"] - M).clamp(min=0).int()
    else:
        q = torch.float32 if case["fmt"] == "f16x2" else torch.bfloat16
        st["qabs"], st["q_rope"] = rnd(B, M, case["heads"], st["L"]).to(q), rnd(B, M, case["heads"], st["P"]).to(q)
    if case["kind"] == "sparse":  # a choice in ascending order, the first and the last two pages among it
        st["sel"] = _choice(rnd(B, M, _width(case)), -(-_ends(st) // case["page"]), case["top_k"])
    if own:
        import undertow_amd as U
        st["cache"] = U.PagedCache(_context(), st["pages"], latent=st["L"], rope=st["P"], mean=st.get("mean"),
                                   mean_scale=st.get("mean_scale"), scales=st.get("scales"))
    return st


def _ends(st):
    """One past the last position that each row sees: [B, M]."""
    m = st["rows"]
    return (st["lens"][:, None] - m + torch.arange(1, m + 1, device=st["lens"].device)).clamp(min=0).long()


def _choice(score, n_pages, top_k):
    W = score.shape[-1]
    at = torch.arange(W, device=score.device)
    score = torch.where((at < 1) | (at >= n_pages[..., None] - 2), math.inf, score).masked_fill(at >= n_pages[..., None], -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top_k]
    best = torch.where(best < n_pages[..., None], best, W).sort(-1).values
    best = torch.where(best < W, best, -1)
    return torch.nn.functional.pad(best, (0, top_k - best.shape[-1]), value=-1).int()


# ------------------------------------------------------------- plain forms
def _attention(q, kv, L, seen):
    """q [N, R, D] over kv [N, T, D] where seen [N, R, T] says so; a row that sees nothing gets zeros."""
    s = (torch.bmm(q, kv.transpose(1, 2).contiguous()) * SCALE).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    return torch.bmm(p, kv[..., :L].contiguous()) / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _query(st, n):
    return torch.cat([st["qabs"], st["q_rope"]], -1).float().reshape(n, -1, st["L"] + st["P"])


def _attend(st):
    B, M, H, L = st["qabs"].shape
    kv = _at(st, st["table"].clamp(min=0).long()).flatten(1, 2)
    seen = torch.arange(kv.shape[1], device=kv.device) < _ends(st)[..., None]
    out = _attention(_query(st, B), kv, L, seen.repeat_interleave(H, 1))
    return out.reshape(B, M, H, L).to(st["qabs"].dtype)


def _sparse(st):
    B, M, H, L = st["qabs"].shape
    page, sel = st["page"], st["sel"].long()
    phys = st["table"].long()[:, None].expand(B, M, -1).gather(2, sel.clamp(min=0))
    kv = _at(st, phys.clamp(min=0)).reshape(B * M, -1, L + st["P"])
    at = sel[..., None] * page + torch.arange(page, device=sel.device)
    seen = ((at < _ends(st)[..., None, None]) & (sel >= 0)[..., None]).reshape(B * M, 1, -1)
    return _attention(_query(st, B * M), kv, L, seen).reshape(B, M, H, L).to(st["qabs"].dtype)


def _window(st):
    """Over the first positions and those that a row of the step has in its window."""
    B, M, H, L = st["qabs"].shape
    window, sinks, page, lens = st["window"], st["sinks"], st["page"], st["lens"].long()
    span = torch.arange(window + M - 1, device=lens.device)
    start = (lens - M + 1 - window).clamp(min=0)
    pos = torch.cat([torch.arange(sinks, device=lens.device).expand(B, -1), start[:, None] + span], 1)
    # a first position that the windows reach counts there
    once = torch.cat([torch.arange(sinks, device=lens.device) < start[:, None], (span >= 0).expand(B, -1)], 1)
    held = pos.clamp(max=st["table"].shape[1] * page - 1)
    phys = st["table"].long().gather(1, held // page).clamp(min=0)
    end = _ends(st)[..., None]
    near = (pos[:, None] >= end - window) | (pos[:, None] < sinks)
    seen = once[:, None] & (pos[:, None] < end) & near
    out = _attention(_query(st, B), _at(st, phys, held % page), L, seen.repeat_interleave(H, 1))
    return out.reshape(B, M, H, L).to(st["qabs"].dtype)


def _read(st):
    pos = st["starts"].long()[:, None] + torch.arange(st["rows"], device=st["lens"].device)
    there = pos < st["lens"].long()[:, None]
    held = torch.where(there, pos, 0)
    phys = st["table"].long().gather(1, held // st["page"]).clamp(min=0)
    x = torch.where(there[..., None], _at(st, phys, held % st["page"]), 0.0)
    x = x.bfloat16() if st["out"] == "bf16" else x
    return tuple(part.contiguous() for part in _parts(x, st["L"]))


def _append(st):
    M, page, lens, table = st["latent"].shape[1], st["page"], st["lens"].long(), st["table"].long()
    pos = lens[:, None] - M + torch.arange(M, device=lens.device)
    phys = table.gather(1, pos // page)
    codes, scales = _quantised(torch.cat([st["latent"], st["krot"]], -1), st["L"])
    st["pages"][phys, pos % page], st["scales"][phys, pos % page] = codes, scales
    # the pages that the rows fall into, the last one again where a sequence touches fewer than another
    first, last = pos[:, :1] // page, pos[:, -1:] // page
    at = torch.minimum(first + torch.arange((M + page - 2) // page + 1, device=lens.device), last)
    touched = table.gather(1, at)
    live = (at[..., None] * page + torch.arange(page, device=lens.device) < lens[:, None, None]).double()
    st["mean"][touched], st["mean_scale"][touched] = _summary(st, touched, live)


def run(st):
    kind = st["kind"]
    if own:
        c, where = st["cache"], (st["table"], st["lens"])
        if kind == "read":
            return c.read(*where, st["rows"], starts=st["starts"], dtype=torch.bfloat16 if st["out"] == "bf16" else torch.float32)
        if kind == "attend":
            return c.attend(*where, st["qabs"], st["q_rope"], SCALE)
        if kind == "sparse":
            return c.attend_pages(*where, st["qabs"], st["q_rope"], SCALE, st["sel"])
        if kind == "window":
            return c.attend_window(*where, st["qabs"], st["q_rope"], SCALE, st["window"], sinks=st["sinks"])
        c.append(*where, st["latent"], st["krot"])
    elif kind != "append":
        return {"read": _read, "attend": _attend, "sparse": _sparse, "window": _window}[kind](st)
    else:
        _append(st)
    lat, rope = _parts(st["pages"], st["L"])
    return dict(latent=lat * st["scales"][..., :1], krot=rope * st["scales"][..., 1:], mean=st["mean"] * st["mean_scale"][:, None])


# -------------------------------------------------------------- accounting
def work(case):
    L, P = _shape(case)
    D, page, B, M = L + P, case["page"], case["batch"], case["rows"]
    row = {"i8": D + 8, "bf16": 2 * D, "f16x2": 4 * D}[case["fmt"]]
    lens = _lens(case)
    if case["kind"] == "append":
        touched = [(n - 1) // page - (n - M) // page + 1 for n in lens]
        older = sum((n - M) % page for n in lens)
        return dict(bytes=B * M * (D * 4 + row) + older * row + sum(touched) * (D + 4), flops=(2 * B * M + older) * D)
    if case["kind"] == "read":
        return dict(bytes=sum(min(n, M) for n in lens) * row + B * M * D * (4 if case["out"] == "f32" else 2), flops=sum(min(n, M) for n in lens) * D)
    H, q = case["heads"], 4 if case["fmt"] == "f16x2" else 2
    ends = [[max(0, n - M + j + 1) for j in range(M)] for n in lens]
    heads = B * M * H * (D + L) * q
    if case["kind"] == "attend":
        return dict(bytes=sum(lens) * row + heads, flops=2 * H * (D + L) * sum(map(sum, ends)))
    if case["kind"] == "window":
        window, sinks = case["window"], case["sinks"]
        seen = [[min(n, window) + min(max(0, n - window), sinks) for n in r] for r in ends]
        once = [n - max(0, max(0, n - M + 1 - window) - sinks) for n in lens]
        return dict(bytes=sum(once) * row + heads, flops=2 * H * (D + L) * sum(map(sum, seen)))
    # a row's chosen pages are full but for the last
    rows = [[min(-(-n // page), case["top_k"]) * page - (-n) % page for n in r if n] for r in ends]
    shared = sum(min(sum(r), n) for r, n in zip(rows, lens))
    return dict(bytes=shared * row + heads, flops=2 * H * (D + L) * sum(map(sum, rows)))


# ------------------------------------------------------- 64-bit references
def _exact_rows(st, phys, off):
    """Row values of pages `phys` at offsets `off`, in 64 bits."""
    x, L = st["pages"][phys, off].double(), st["L"]
    if st["fmt"] == "i8":
        s = st["scales"][phys, off].double()
        x[..., :L] *= s[..., :1]
        x[..., L:] *= s[..., 1:]
        return x
    return x if st["fmt"] == "bf16" else x[..., 0, :] + x[..., 1, :] * 2.0 ** -11


def exact(case, seed):
    st = prepare(case, seed)
    table, lens = st["table"], st["lens"].tolist()
    M, page, L = case["rows"], case["page"], st["L"]
    if case["kind"] == "append":
        n_pages = st["pages"].shape[0]
        whole = torch.stack([_exact_rows(st, p, torch.arange(page, device="cuda")) for p in range(n_pages)])
        means = st["mean"].double() * st["mean_scale"].double()[:, None]
        x = torch.cat([st["latent"], st["krot"]], -1).double()
        for b, n in enumerate(lens):
            at = torch.arange(n - M, n, device="cuda")
            for lo, hi in ((0, L), (L, x.shape[-1])):
                top = x[b, :, lo:hi].abs().max(-1, keepdim=True).values
                step = top / 127.0
                whole[table[b][at // page].long(), at % page, lo:hi] = torch.round(x[b, :, lo:hi] * 127.0 / top) * step.float().double()
            for k in range((n - M) // page, (n - 1) // page + 1):
                p, live = int(table[b, k]), min(page, n - k * page)
                s = whole[p, :live].sum(0)
                top = s.abs().max()
                means[p] = torch.round(s * 127.0 / top) * (top / (127.0 * live)) if top > 0 else s * 0
        return dict(latent=whole[..., :L], krot=whole[..., L:], mean=means)
    if case["kind"] == "read":
        out = torch.zeros((case["batch"], M, L + st["P"]), dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            at = torch.arange(int(st["starts"][b]), n, device="cuda")[:M]
            out[b, :len(at)] = _exact_rows(st, table[b][at // page].long(), at % page)
        return out[..., :L], out[..., L:]
    q = torch.cat([st["qabs"], st["q_rope"]], -1).double()
    out = torch.zeros(st["qabs"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        for j in range(M):
            sees = n - M + j + 1
            if sees <= 0:
                continue
            at = torch.arange(sees, device="cuda")
            if case["kind"] == "window":
                at = at[(at < case["sinks"]) | (at >= sees - case["window"])]
            elif case["kind"] == "sparse":
                chosen = st["sel"][b, j][st["sel"][b, j] >= 0].long()
                at = (chosen[:, None] * page + torch.arange(page, device="cuda")).flatten()
                at = at[at < sees]
            kv = _exact_rows(st, table[b][at // page].long(), at % page)
            out[b, j] = torch.softmax(q[b, j] @ kv.T * SCALE, -1) @ kv[:, :L]
    return out
