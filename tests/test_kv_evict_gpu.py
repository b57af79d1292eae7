"""Eviction from a paged cache by accumulated attention weight. What stays and where it goes is compared exactly."""

import math

import pytest
import torch

from _serving import DT, Paged, check

pytestmark = pytest.mark.gpu


def _ops():
    from cleave_b200 import ops

    return ops


def _chosen(row, n, keep, sinks, recent):
    """The kept indices of one (request, head), ascending: `row` a list of floats, missing entries weigh 0."""
    first = min(sinks, keep)
    tail = min(recent, keep - first)
    w = lambda j: row[j] if j < len(row) else 0.0  # noqa: E731
    rank = lambda j: (0, 0.0, j) if math.isnan(w(j)) else (1, -w(j), j)  # noqa: E731
    middle = sorted(range(first, n - tail), key=rank)[:keep - first - tail]
    return list(range(first)) + sorted(middle) + list(range(n - tail, n))


class Case:
    def __init__(self, lens, hkv, d, page, dtype, budget, sums=None, max_len=None, seed=0, short=0):
        """`short`: destination pages that the last request lacks."""
        self.c = Paged(lens, hkv, hkv, d, page, dtype, seed=seed, extra=3 + sum(-(-min(n, budget) // page) for n in lens))
        self.budget, self.page = budget, page
        g = torch.Generator().manual_seed(seed + 1)
        max_len = max(lens) if max_len is None else max_len
        self.sums = torch.randn(len(lens), hkv, max_len, generator=g).mul(2).sub(5).exp() if sums is None else sums
        room = [-(-min(n, budget) // page) for n in lens]
        room[-1] -= short
        self.dptr = [0]
        for p in room:
            self.dptr.append(self.dptr[-1] + p)
        self.dst = self.c.spare[:self.dptr[-1]]
        self.keep = [min(n, budget, p * page) for n, p in zip(lens, room)]

    def run(self, sinks, recent):
        i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).cuda()  # noqa: E731
        _, k, v, ptr, ids, last, _ = self.c.args()
        kept, sums, new_last = _ops().kv_cache_evict(k, v, self.sums.cuda(), ptr, ids, last, i32(self.dptr), i32(self.dst),
                                                     budget=self.budget, sinks=sinks, recent=recent)
        return k.cpu(), v.cpu(), kept.cpu(), sums.cpu(), new_last.cpu()

    def check(self, sinks, recent):
        c = self.c
        k, v, kept, sums, last = self.run(sinks, recent)
        want_k, want_v = c.k.clone(), c.v.clone()
        want_kept = torch.full(kept.shape, -1, dtype=torch.int32)
        want_sums = torch.zeros_like(self.sums)
        max_len = self.sums.shape[2]
        for b, n in enumerate(c.lens):
            kk, vv = c.rows(b)
            for h in range(c.hkv):
                ids = _chosen(self.sums[b, h].tolist(), n, self.keep[b], sinks, recent)
                want_kept[b, h, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
                for i, j in enumerate(ids):
                    if i < max_len:
                        want_sums[b, h, i] = self.sums[b, h, j] if j < max_len else 0.0
                    at = self.dst[self.dptr[b] + i // self.page]
                    want_k[at, i % self.page, h], want_v[at, i % self.page, h] = kk[j, h], vv[j, h]
        assert torch.equal(kept, want_kept)
        bits = lambda t: t.view(torch.int16 if t.element_size() == 2 else torch.int32)  # noqa: E731
        assert torch.equal(bits(sums), bits(want_sums))
        assert torch.equal(bits(k), bits(want_k)) and torch.equal(bits(v), bits(want_v))
        assert last.tolist() == [(m - 1) % self.page + 1 if m else 0 for m in self.keep]


LENS = [0, 1, 37, 64, 65, 200, 513]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("page", [1, 5, 16, 64])
@pytest.mark.parametrize("hkv,d", [(2, 128), (3, 64), (1, 128)])
@pytest.mark.parametrize("budget,sinks,recent", [(64, 4, 20), (100, 0, 0), (1, 0, 0)])
def test_evict(dt, page, hkv, d, budget, sinks, recent):
    Case(LENS, hkv, d, page, DT[dt], budget, seed=page).check(sinks, recent)


@pytest.mark.parametrize("budget,sinks,recent", [(10, 10, 0), (10, 0, 10), (10, 3, 7), (513, 1, 1), (1000, 4, 100), (512, 0, 511), (1, 1, 0)])
def test_budgets(budget, sinks, recent):
    Case(LENS, 2, 64, 16, torch.bfloat16, budget, seed=7).check(sinks, recent)


@pytest.mark.parametrize("max_len", [9000, 40000, 1000])
def test_long_requests(max_len):
    Case([9000, 4097], 2, 64, 64, torch.bfloat16, 3000, max_len=max_len, seed=8).check(4, 1000)


def test_requests_longer_than_a_block_holds():
    Case([70001, 33000], 1, 64, 64, torch.bfloat16, 20000, seed=16).check(4, 1000)


def test_more_heads_than_rows_of_a_block():
    Case([300, 20], 130, 64, 16, torch.float16, 70, seed=9).check(2, 30)


@pytest.mark.parametrize("kind", ["equal", "few", "zero_signs", "special", "negative", "neighbours"])
def test_ties_and_special_values(kind):
    lens, hkv, n = [300, 150], 2, 300
    g = torch.Generator().manual_seed(3)
    base = torch.rand(2, hkv, n, generator=g)
    if kind == "equal":
        s = torch.full((2, hkv, n), 0.5)
    elif kind == "few":
        s = (base * 4).floor() / 4
    elif kind == "zero_signs":
        s = torch.where(base < 0.5, -0.0, 0.0)
    elif kind == "special":
        s = base.clone()
        s[..., ::7], s[..., 3::11], s[..., 5::13] = math.nan, math.inf, -math.inf
        s[..., 2::17] = -math.nan
    elif kind == "negative":
        s = base - 0.5
    else:  # values that differ in their last bits, subnormal ones among them
        s = (torch.randint(0, 40, (2, hkv, n), generator=g, dtype=torch.int32) + 1).view(torch.float32)
    Case(lens, hkv, 64, 16, torch.bfloat16, 100, sums=s, seed=4).check(3, 10)


@pytest.mark.parametrize("nans", [5, 87, 88, 150])
def test_more_nans_than_stay(nans):
    """The keys then span the whole 32-bit range, and the range of the last histogram ends at its last number."""
    s = torch.rand(2, 2, 300, generator=torch.Generator().manual_seed(17))
    s[..., 0:20], s[..., 20:60] = math.inf, -math.inf
    s[..., 100:100 + nans] = math.nan
    Case([300, 260], 2, 64, 16, torch.bfloat16, 100, sums=s, seed=4).check(3, 10)


@pytest.mark.parametrize("max_len", [1, 50, 129, 600])
def test_tokens_without_a_record_weigh_nothing(max_len):
    Case([513, 130, 4], 2, 64, 16, torch.bfloat16, 100, max_len=max_len, seed=5).check(4, 20)


def test_fewer_destination_pages_keep_fewer_tokens():
    Case([513, 130], 2, 64, 16, torch.bfloat16, 100, seed=6, short=3).check(4, 20)
    Case([513, 130], 2, 64, 16, torch.bfloat16, 100, seed=6, short=7).check(40, 60)


def test_requests_may_share_their_source_pages():
    c = Case([200, 200], 2, 64, 16, torch.bfloat16, 64, seed=10)
    _, k, v, ptr, ids, last, _ = c.c.args()
    half = ids.numel() // 2
    ids = torch.cat([ids[:half], ids[:half]])
    i32 = lambda t: torch.as_tensor(t, dtype=torch.int32).cuda()  # noqa: E731
    kept, sums, _ = _ops().kv_cache_evict(k, v, c.sums.cuda(), ptr, ids, last, i32(c.dptr), i32(c.dst), budget=64, sinks=2, recent=9)
    kk, _ = c.c.rows(0)
    for b in range(2):
        for h in range(2):
            want = _chosen(c.sums[b, h].tolist(), 200, 64, 2, 9)
            assert kept[b, h].tolist() == want
            got = k.cpu()[c.dst[c.dptr[b]:c.dptr[b + 1]]].flatten(0, 1)[:64, h]
            assert torch.equal(got, kk[want, h])


def test_rows_of_pages_that_do_not_exist_are_not_written():
    c = Case([200, 90], 2, 64, 16, torch.bfloat16, 64, seed=11)
    want = c.run(2, 9)
    c.dst = c.dst.clone()
    gone = int(c.dst[1])
    c.dst[1] = 10 ** 9
    k, v, kept, sums, last = c.run(2, 9)
    same = torch.ones(k.shape[0], dtype=torch.bool)
    same[gone] = False
    bits = lambda t: t.view(torch.int16)  # noqa: E731
    assert torch.equal(bits(k)[same], bits(want[0])[same]) and torch.equal(bits(v)[same], bits(want[1])[same])
    assert torch.equal(bits(k)[gone], bits(c.c.k)[gone])
    assert torch.equal(kept, want[2]) and torch.equal(sums, want[3]) and torch.equal(last, want[4])


def test_decode_evict_decode():
    """The operators as a server runs them: steps that accumulate, an eviction, and a step over what is left."""
    ops, dt = _ops(), torch.bfloat16
    lens, budget, page = [300, 70, 513], 128, 16
    c = Paged(lens, 8, 2, 128, page, dt, seed=12, extra=3 + sum(-(-min(n, budget) // page) for n in lens))
    args = c.args()
    sums = torch.zeros(3, 2, 513, device="cuda")
    for _ in range(2):
        ops.gqa_paged_decode_weights(*args, sums)
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    dptr = [0]
    for n in lens:
        dptr.append(dptr[-1] + -(-min(n, budget) // page))
    dst = i32(c.spare[:dptr[-1]])
    kept, new_sums, last = ops.kv_cache_evict(args[1], args[2], sums, *args[3:6], i32(dptr), dst, budget=budget, sinks=4, recent=32)
    out, lse = ops.gqa_paged_decode_weights(args[0], args[1], args[2], i32(dptr), dst, last, c.scale, new_sums)
    # the same step over an uncut cache in which the evicted rows are not seen, head by head
    from _serving import attend64

    for b, n in enumerate(lens):
        k, v = c.rows(b)
        for h in range(2):
            ids = kept[b, h].cpu()
            ids = ids[ids >= 0].long()
            assert len(ids) == min(n, budget)
            rows = slice(4 * h, 4 * h + 4)
            see = torch.ones(4, len(ids), dtype=torch.bool)
            want, want_lse, p, spread = attend64(c.q[b, rows], k[ids, h], v[ids, h], see, c.scale)
            check(out[b, rows], lse[b, rows], want, want_lse, spread, dt)
            grown = p.sum(0) + sums[b, h].cpu().double()[ids]
            assert ((new_sums[b, h, :len(ids)].cpu().double() - grown).abs() <= 3e-4 * grown).all()
            assert (new_sums[b, h, len(ids):] == 0).all()


def test_captured_and_replayed():
    c = Case([300, 513], 2, 64, 16, torch.bfloat16, 100, seed=13)
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    _, k, v, ptr, ids, last, _ = c.c.args()
    sums, dptr, dst = c.sums.cuda(), i32(c.dptr), i32(c.dst)
    call = lambda: _ops().kv_cache_evict(k, v, sums, ptr, ids, last, dptr, dst, budget=100, sinks=4, recent=9)  # noqa: E731
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = call()
    other = torch.rand(sums.shape, generator=torch.Generator().manual_seed(0))
    sums.copy_(other)
    c.sums = other
    g.replay()
    torch.cuda.synchronize()
    want = c.run(4, 9)
    for a, b in zip((k, v, *held), want):
        assert torch.equal(a.cpu().view(torch.int16 if a.element_size() == 2 else torch.int32),
                           b.view(torch.int16 if b.element_size() == 2 else torch.int32))


def test_refusals():
    ops = _ops()
    c = Case([40, 20], 2, 64, 16, torch.bfloat16, 16, seed=14)
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    _, k, v, ptr, ids, last, _ = c.c.args()
    good = [k, v, c.sums.cuda(), ptr, ids, last, i32(c.dptr), i32(c.dst)]

    def refuse(error, at=None, value=None, budget=16, sinks=2, recent=4):
        a = list(good)
        if at is not None:
            a[at] = value
        with pytest.raises(error):
            ops.kv_cache_evict(*a, budget=budget, sinks=sinks, recent=recent)

    for kw in (dict(budget=0), dict(sinks=-1), dict(recent=-1), dict(sinks=10, recent=10)):
        refuse(ValueError, **kw)
    refuse(ValueError, 0, k.cpu())
    refuse(ValueError, 1, v[:, :, :1])
    refuse(TypeError, 0, k.float())
    refuse(TypeError, 2, good[2].double())
    refuse(ValueError, 2, good[2][:, :1].contiguous())
    refuse(ValueError, 2, good[2].transpose(1, 2))
    refuse(TypeError, 3, ptr.long())
    refuse(ValueError, 3, ptr[:-1].contiguous())
    refuse(TypeError, 5, None)
    refuse(ValueError, 6, good[6][:-1].contiguous())
    refuse(ValueError, 7, good[7].cpu())
