"""The paged latent cache in plain torch, 64 bits: what its tests compare with."""
import math

import torch

STEP = 2.0 ** -11  # of the second f16 plane


def stored(fmt, x):
    """f32 rows as a page holds them (fmt "bf16" or "f16x2")."""
    if fmt == "bf16":
        return x.bfloat16()
    c = torch.where(x.isfinite(), x.clamp(-65504.0, 65504.0), x)
    hi = c.half()
    return torch.stack([hi, torch.where(c.isfinite(), ((c - hi.float()) / STEP).half(), 0.0)], -2)


def values(fmt, rows):
    return rows.double() if fmt == "bf16" else rows[..., 0, :].double() + rows[..., 1, :].double() * STEP


class Pool:
    """A pool whose every row is NaN until something is put there, and the
    tables of sequences that lie in it in random order; entries behind a
    sequence's last page are ids that exist nowhere."""

    def __init__(self, seed, fmt, lens, page, L, P, width=None, spare=2, fill=True):
        self.g = torch.Generator().manual_seed(seed)
        self.fmt, self.page, self.L, self.P, self.D = fmt, page, L, P, L + P
        self.lens = list(lens)
        need = [-(-n // page) for n in self.lens]
        self.n_pages = sum(need) + spare
        width = max(max(need), 1) if width is None else width
        ids, at = torch.randperm(self.n_pages, generator=self.g).tolist(), 0
        self.table = torch.full((len(lens), width), 2**31 - 1, dtype=torch.int32)
        self.table[:, 1::2] = -1
        for b, k in enumerate(need):
            self.table[b, :k] = torch.tensor(ids[at:at + k], dtype=torch.int32)
            at += k
        shape = (self.n_pages, page, L + P) if fmt == "bf16" else (self.n_pages, page, 2, L + P)
        self.pages = torch.full(shape, math.nan, dtype=torch.bfloat16 if fmt == "bf16" else torch.float16)
        if fill:
            for b, n in enumerate(self.lens):
                self.put(b, 0, self.randn(n, L + P))

    def randn(self, *s):
        return torch.randn(s, generator=self.g)

    def where(self, b, pos):
        return self.table[b, pos // self.page].long(), pos % self.page

    def put(self, b, start, x):
        at = torch.arange(start, start + len(x))
        self.pages[self.where(b, at)] = stored(self.fmt, x)

    def rows(self, b, pos):
        return values(self.fmt, self.pages[self.where(b, pos)])

    def queries(self, M, H):
        t = torch.bfloat16 if self.fmt == "bf16" else torch.float32
        B = len(self.lens)
        return self.randn(B, M, H, self.L).to(t), self.randn(B, M, H, self.P).to(t)

    def cuda(self, **more):
        import undertow_amd as U
        return U.PagedCache(more.pop("ctx"), self.pages.cuda(), self.L, self.P, **more)

    def lens32(self):
        return torch.tensor(self.lens, dtype=torch.int32)


def seen(n, M):
    """Positions that the M rows of a sequence of n positions see."""
    return [max(0, n - M + j + 1) for j in range(M)]


def attend(kv, q, L, scale):
    """One row's heads q [H, D] over kv [T, D] -> (context [H, L], and two
    measures of what an error is relative to: the weighted mean distance of a
    value from the context, and sum_t p_t |v_t|)."""
    if len(kv) == 0:
        z = torch.zeros((q.shape[0], L), dtype=torch.float64, device=q.device)
        return z, z, z
    p = torch.softmax(q @ kv.T * scale, -1)
    v = kv[:, :L]
    out = p @ v
    # sum_t p_t |v_t - out| <= sqrt(sum_t p_t (v_t - out)^2)
    spread = (p @ (v * v) - out * out).clamp(min=0).sqrt()
    return out, spread, p @ v.abs()


def summary(x):
    """(codes, scale) of the mean of rows x [n, D] (64 bits)."""
    s = x.sum(0)
    top = s.abs().max()
    if not top > 0:
        return torch.zeros_like(s).to(torch.int8), torch.zeros((), dtype=torch.float32)
    return torch.round(s * 127.0 / top).to(torch.int8), (top / (127.0 * len(x))).float()


def select(q, codes, scales, np_, keep_first, keep_last, top_k, weights=None):
    """q [H, D] f64, the sequence's page summaries in order -> the list of pages."""
    H = q.shape[0]
    score = [0.0] * np_
    for h in range(H):
        top = q[h].abs().max().item()
        if not (0 < top < math.inf):
            continue
        c = torch.round(q[h] * 127.0 / top)
        w = 1.0 if weights is None else float(weights[h])
        dots = (codes[:np_].double() @ c).tolist()
        for k in range(np_):
            score[k] += w * (top / 127.0) * max(0.0, dots[k])
    score = [score[k] * float(scales[k]) for k in range(np_)]
    forced = [k for k in range(np_) if k < keep_first or k >= np_ - keep_last]
    rest = sorted((k for k in range(np_) if k not in set(forced)), key=lambda k: (-score[k], k))
    got = sorted(forced + rest[:max(0, top_k - len(forced))])[:top_k]
    return got + [-1] * (top_k - len(got))
