"""Plain 64-bit forms of the serving operators (windowed attention, shared prefix, accumulated weights, eviction) and the
tolerances that follow from the kernels' arithmetic.

Tolerance of an attention output, per element, with eps/2 the largest relative error of one rounding to the storage
type and A = sum_j p_j |v_j|:

    eps/2 |out|            the output's own rounding
  + eps/2 A   (one_p)      P enters the second product rounded to the storage type (tensor-memory kernels)
  + 2e-4 A                 everything held in 32 bits: a score is a sum of D products and is off by at most
                           (D + 2) 2^-23 sum_d |q_d k_d| scale, below 6e-5 for D = 128 and the unit-variance data of
                           these tests (sum |q k| scale < 4 sigma = 4); a weight's relative error is that in the
                           numerator plus that in the normaliser, plus 2^-22 of exp2 and 2^-17 where P is split in two

The base-2 log-sum-exp is off by a score's error times log2(e), 1e-4, and a weight by the relative 2e-4.
"""

import math

import torch

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attend64(q, k, v, see, scale):
    """One kv head: q (rows, D), k / v (tokens, D), see (rows, tokens) bool. Returns out, lse (base 2), weights, A; the rows
    of K and V that no query sees are not looked at."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    see = see.cpu()
    seen = see.any(0)
    k, v = torch.where(seen[:, None], k, 0.0), torch.where(seen[:, None], v, 0.0)
    x = (q @ k.T * scale).masked_fill(~see, -math.inf)
    lse = torch.logsumexp(x, -1) if x.shape[1] else torch.full((q.shape[0],), -math.inf, dtype=torch.float64)
    p = torch.exp(x - torch.where(lse == -math.inf, 0.0, lse)[:, None])
    return p @ v, lse / math.log(2.0), p, p @ v.abs()


def check(got, lse, want, want_lse, spread, dtype, one_p=False):
    got, lse = got.double().cpu(), lse.double().cpu()
    h = half_step(dtype)
    assert not got.isnan().any() and not lse.isnan().any()
    off = (got - want).abs() - (h * want.abs() + ((h if one_p else 0.0) + 2e-4) * spread + 1e-30)
    if dtype == torch.float16:
        off -= 2.0 ** -25  # half a step of the subnormal numbers of fp16
    assert off.max() <= 0, f"out is off by {off.max():.3g} more than its tolerance"
    assert torch.equal(lse == -math.inf, want_lse == -math.inf)
    live = want_lse != -math.inf
    assert ((lse - want_lse)[live].abs() <= 1e-4 + 2.0 ** -22 * want_lse[live].abs()).all()


class Paged:
    """A paged cache with requests of the given lengths; whatever belongs to no token holds NaN."""

    def __init__(self, lens, hq, hkv, d, page, dtype, seed=0, extra=3, q_rows=None):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.hq, self.hkv, self.d, self.page, self.dtype = list(lens), hq, hkv, d, page, dtype
        self.scale = d ** -0.5
        pages = [-(-n // page) for n in lens]
        total = sum(pages) + extra
        perm = torch.randperm(total, generator=g)
        self.ids, self.spare = perm[:sum(pages)], perm[sum(pages):]
        self.ptr = [0]
        for p in pages:
            self.ptr.append(self.ptr[-1] + p)
        rn = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
        self.q = rn(len(lens) if q_rows is None else q_rows, hq, d)
        self.k, self.v = rn(total, page, hkv, d), rn(total, page, hkv, d)
        used = torch.zeros(total, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            for t in range(n):
                used[self.ids[self.ptr[b] + t // page], t % page] = True
        self.k[~used], self.v[~used] = math.nan, math.nan
        self.last = [n - (p - 1) * page if p else 0 for n, p in zip(lens, pages)]

    def rows(self, b):
        """K and V of request b's tokens, (tokens, HKV, D)."""
        idx = self.ids[self.ptr[b]:self.ptr[b + 1]]
        return tuple(c[idx].flatten(0, 1)[:self.lens[b]] for c in (self.k, self.v))

    def poison(self, b, tokens, value):
        for t in tokens:
            at = self.ids[self.ptr[b] + t // self.page]
            self.k[at, t % self.page], self.v[at, t % self.page] = value, value

    def args(self):
        """q, caches, tables and scale on the GPU, in the operators' order."""
        i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).cuda()  # noqa: E731
        return [self.q.cuda(), self.k.cuda(), self.v.cuda(), i32(self.ptr), i32(self.ids),
                None if self.page == 1 else i32(self.last), self.scale]

    def want(self, see_of, before=None):
        """(out, lse, weights per request (HQ, tokens), A): request b sees the tokens see_of(b, n); ``before`` = (k, v) of
        tokens that every request sees in front of its own."""
        grp = self.hq // self.hkv
        out, lse, spread, ws = [], [], [], []
        for b, n in enumerate(self.lens):
            k, v = self.rows(b)
            see = see_of(b, n)
            if before is not None:
                k, v = torch.cat([before[0], k]), torch.cat([before[1], v])
                see = torch.cat([torch.ones(before[0].shape[0], dtype=torch.bool), see])
            per = [attend64(self.q[b, h * grp:(h + 1) * grp], k[:, h], v[:, h], see[None].expand(grp, -1), self.scale)
                   for h in range(self.hkv)]
            out.append(torch.cat([p[0] for p in per]))
            lse.append(torch.cat([p[1] for p in per]))
            ws.append(torch.cat([p[2] for p in per]))
            spread.append(torch.cat([p[3] for p in per]))
        return torch.stack(out), torch.stack(lse), ws, torch.stack(spread)
