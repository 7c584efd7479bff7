"""The paged latent cache in 8 bits, and windows, in plain torch, 64 bits: what
their tests compare with."""
import math

import torch

import paged_ref as R


def quantised(x, L):
    """(codes int8, scales f32 [.., 2]) of f32 rows [.., D]: each part by its
    own largest, half to even; a part that is not finite has codes 0 and the
    scale NaN."""
    codes, scales = [], []
    for part in (x[..., :L].double(), x[..., L:].double()):
        top = part.abs().amax(-1, keepdim=True)
        ok = top.isfinite()
        c = torch.round(torch.where(ok, part, 0.0) * 127.0 / torch.where(ok & (top > 0), top, 1.0))
        codes.append(c.to(torch.int8))
        scales.append(torch.where(ok, top / 127.0, math.nan).float())
    return torch.cat(codes, -1), torch.cat(scales, -1)


def values8(codes, scales, L):
    """What codes stand for, in 64 bits."""
    s = scales.double()
    return torch.cat([codes[..., :L].double() * s[..., :1], codes[..., L:].double() * s[..., 1:]], -1)


class Pool8(R.Pool):
    """Pool in 8 bits: every row's codes are any and its scales NaN until
    something is put there."""

    def __init__(self, seed, lens, page, L, P, width=None, spare=2, fill=True):
        super().__init__(seed, "bf16", lens, page, L, P, width, spare, fill=False)
        shape = self.pages.shape
        self.pages = torch.randint(-128, 128, shape, generator=self.g).to(torch.int8)
        self.scales = torch.full(tuple(shape[:2]) + (2,), math.nan)
        if fill:
            for b, n in enumerate(self.lens):
                self.put(b, 0, self.randn(n, L + P))

    def put(self, b, start, x):
        at = self.where(b, torch.arange(start, start + len(x)))
        self.pages[at], self.scales[at] = quantised(x, self.L)

    def rows(self, b, pos):
        at = self.where(b, pos)
        return values8(self.pages[at], self.scales[at], self.L)

    def cuda(self, **more):
        import undertow_amd as U
        return U.PagedCache(more.pop("ctx"), self.pages.cuda(), self.L, self.P, scales=self.scales.cuda(), **more)


def pool(fmt, seed, lens, page, L, P, width=None):
    return Pool8(seed, lens, page, L, P, width) if fmt == "i8" else R.Pool(seed, fmt, lens, page, L, P, width)


def positions(n, window=None, sinks=0):
    """Positions that a row whose own is n - 1 sees."""
    at = torch.arange(max(n, 0))
    return at if window is None else at[(at < sinks) | (at >= n - window)]


def score_step(kv, q, L, scale):
    """How far a score may be off for the rounding of each part of a head's
    query to 16 bits of its largest (half a step of 2 max / 65024): [H]."""
    off = 0.0
    for lo, hi in ((0, L), (L, kv.shape[-1])):
        k = kv[:, lo:hi].abs().sum(-1).max() if len(kv) else 0.0
        off = off + q[:, lo:hi].abs().amax(-1) / 32512.0 / 2.0 * k
    return off * abs(scale)


def largest(kv, q, L, scale):
    """Positions times the largest share that one has in a context: [H, 1]."""
    p = torch.softmax(q @ kv.T * scale, -1)
    return len(kv) * (p * kv[:, :L].abs().amax(-1)).amax(-1, keepdim=True)


def close(fmt, got, want, spread, mass, step=0.0, top=0.0):
    """As the attention tests of the other formats; 8 bits: an output is
    rounded once (2^-8 of it); a weight times its position's scale to 11 bits
    in the numerator alone (2^-11 sum_t p_t |v_t|; one below 2^-24 of the
    largest by 2^-35 of that: `top`); where a row's positions are cut, each
    part's context to 11 bits (2^-11 of its share, and those add up to no more
    than sum_t p_t |v_t|); a score is off by `step`, which moves the context by
    that times its spread; and what is left is f32 arithmetic."""
    got = got.double().cpu()
    want, spread, mass = want.cpu(), spread.cpu(), mass.cpu()
    assert torch.isfinite(got).all()
    if fmt == "bf16":
        tol = 2.0 ** -8 * (want.abs() + spread) + 6e-5 * spread + 2.0 ** -20 * mass + 1e-30
    elif fmt == "f16x2":
        tol = 5.2e-5 * spread + 2.0 ** -20 * (mass + want.abs()) + 1e-30
    else:
        tol = 2.0 ** -8 * want.abs() + (6e-5 + 1.05 * step) * spread + 2 * 2.0 ** -11 * mass + 2.0 ** -35 * top + 1e-30
    err = (got - want).abs()
    assert (err <= tol).all(), float((err / tol).max())


def check(pool, fmt, got, qabs, qrope, scale, sel=None, window=None, sinks=0, only=None):
    """Every row of `got` (of the sequences `only`) against 64 bits (on the
    device that `got` is on); rows that see nothing are zeros."""
    B, M, H, L = qabs.shape
    for b, n in enumerate(pool.lens):
        if only is not None and b not in only:
            continue
        for j in range(M):
            at = positions(n - M + j + 1, window, sinks)
            if sel is not None:
                listed = [torch.arange(k * pool.page, min(len(at), (k + 1) * pool.page)) for k in sel[b, j].tolist()
                          if 0 <= k and k * pool.page < len(at)]
                at = torch.cat(listed) if listed else at[:0]
            if len(at) == 0:
                assert (got[b, j] == 0).all()
                continue
            kv = pool.rows(b, at).to(got.device)
            q = torch.cat([qabs[b, j], qrope[b, j]], -1).double().to(got.device)
            want, spread, mass = R.attend(kv, q, L, scale)
            step = score_step(kv, q, L, scale)[:, None].cpu() if fmt == "i8" else 0.0
            close(fmt, got[b, j], want, spread, mass, step, largest(kv, q, L, scale).cpu() if fmt == "i8" else 0.0)
