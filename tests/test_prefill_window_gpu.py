"""Causal prefill over a sliding window with sinks, ragged and paged, against a 64-bit form."""

import math

import pytest
import torch

from _serving import DT, attend64, check

pytestmark = pytest.mark.gpu


def _ops():
    from cleave_b200 import ops

    return ops


class Case:
    """Requests with (query rows, keys); keys that no query sees hold NaN, and so do rows of K, V that belong to nobody."""

    def __init__(self, lens, hq, hkv, d, dtype, window, sinks, paged, seed=0, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.hkv, self.dtype, self.window, self.sinks, self.paged = lens, hkv, dtype, window, sinks, paged
        self.scale = d ** -0.5
        self.qp, self.kp = [0], [0]
        for a, b in lens:
            self.qp.append(self.qp[-1] + a)
            self.kp.append(self.kp[-1] + b)
        rn = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
        self.q = rn(max(1, self.qp[-1]), hq, d)
        total = self.kp[-1]
        self.k, self.v = rn(total + spare, hkv, d), rn(total + spare, hkv, d)
        self.k[total:], self.v[total:] = math.nan, math.nan
        self.see = []
        for r, (a, b) in enumerate(lens):
            p, j = torch.arange(b - a, b)[:, None], torch.arange(b)[None]
            see = (j <= p) & ((j > p - window) | (j < sinks))
            self.see.append(see)
            unseen = torch.nonzero(~see.any(0)).flatten() + self.kp[r]
            self.k[unseen], self.v[unseen] = math.nan, math.nan
        self.perm = torch.randperm(total + spare, generator=g)

    def want(self):
        grp = self.q.shape[1] // self.hkv
        out, spread = torch.zeros(self.q.shape, dtype=torch.float64), torch.zeros(self.q.shape, dtype=torch.float64)
        lse = torch.full(self.q.shape[:2], -math.inf, dtype=torch.float64)
        for r, (a, b) in enumerate(self.lens):
            qs, ks = slice(self.qp[r], self.qp[r] + a), slice(self.kp[r], self.kp[r] + b)
            for h in range(self.q.shape[1]):
                out[qs, h], lse[qs, h], _, spread[qs, h] = attend64(self.q[qs, h], self.k[ks, h // grp], self.v[ks, h // grp],
                                                                    self.see[r], self.scale)
        return out, lse, spread

    def args(self):
        i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).cuda()  # noqa: E731
        if not self.paged:
            return [self.q.cuda(), self.k.cuda(), self.v.cuda(), i32(self.qp), i32(self.kp), self.scale, self.window, self.sinks]
        k, v = torch.empty_like(self.k), torch.empty_like(self.v)
        k[self.perm], v[self.perm] = self.k, self.v
        return [self.q.cuda(), k[:, None].cuda(), v[:, None].cuda(), i32(self.qp), i32(self.kp), i32(self.perm[:self.kp[-1]]), self.scale,
                self.window, self.sinks]

    def call(self, *a, **kw):
        ops = _ops()
        r = (ops.gqa_paged_prefill_window if self.paged else ops.gqa_ragged_prefill_window)(*a, **kw)
        ops.check_workspace(ops.workspace("attn_prefill", 0, "cuda"))
        return r

    def run(self):
        args = self.args()
        out, lse = torch.full_like(args[0], math.nan), torch.full(args[0].shape[:2], math.nan, device="cuda")
        return self.call(*args, out=out, lse=lse)

    def check(self):
        want, want_lse, spread = self.want()
        check(*self.run(), want, want_lse, spread, self.dtype, one_p=True)


LENS = [(1, 1), (7, 7), (0, 50), (130, 130), (1, 300), (64, 200), (129, 500), (20, 5), (3, 0), (300, 300)]
PAGED = pytest.mark.parametrize("paged", [False, True])


@PAGED
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64), (10, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(100, 4), (33, 0), (1, 1), (128, 130)])
def test_window_prefill(paged, dt, hq, hkv, d, window, sinks):
    Case(LENS, hq, hkv, d, DT[dt], window, sinks, paged, seed=window).check()


@PAGED
@pytest.mark.parametrize("window", [1, 2, 64, 127, 128, 129, 400, 2 ** 31 - 1])
@pytest.mark.parametrize("sinks", [0, 1, 64, 127, 128, 129, 300, 2 ** 31 - 1])
def test_window_and_sink_counts(paged, window, sinks):
    Case([(700, 700), (5, 900), (140, 650)], 2, 1, 64, torch.bfloat16, window, sinks, paged, seed=1).check()


@PAGED
@pytest.mark.parametrize("n", [127, 128, 129, 255, 256, 257, 511])
def test_one_request(paged, n):
    Case([(n, n)], 2, 2, 128, torch.float16, 130, 3, paged, seed=n).check()


@PAGED
def test_one_token_behind_a_long_context(paged):
    Case([(1, 5000)], 8, 2, 128, torch.bfloat16, 1000, 4, paged, seed=2).check()


@PAGED
def test_more_items_than_processors(paged):
    """Persistent form: 40 requests of up to 3 query tiles and 8 heads."""
    g = torch.Generator().manual_seed(3)
    lens = [(int(a), int(a + b)) for a, b in zip(torch.randint(0, 300, (40,), generator=g), torch.randint(0, 300, (40,), generator=g))]
    Case(lens, 8, 2, 64, torch.bfloat16, 140, 2, paged, seed=4).check()


@PAGED
@pytest.mark.parametrize("hq,hkv,d", [(12, 4, 64), (8, 8, 128), (10, 2, 64)])
def test_more_items_than_processors_of_odd_groups(paged, hq, hkv, d):
    """The blocks of an item are then two tiles of query rows, and the second exists in some items of a CTA and not in others."""
    g = torch.Generator().manual_seed(13)
    lens = []
    for i in range(60):  # at most 128 rows, up to 256, and a little over 256
        n = int(torch.randint(1, 129, (1,), generator=g)) + (0, 128, 256)[i % 3]
        lens.append((n, n + int(torch.randint(0, 200, (1,), generator=g))))
    Case(lens, hq, hkv, d, torch.bfloat16, 140, 2, paged, seed=14).check()


@PAGED
@pytest.mark.parametrize("hq,hkv,d", [(12, 4, 128), (8, 8, 64), (10, 2, 128)])
def test_long_prompts_persistent_of_odd_groups(paged, hq, hkv, d):
    Case([(2500, 2600), (100, 900), (1, 1), (3000, 3000)], hq, hkv, d, torch.float16, 700, 4, paged, seed=15).check()


@PAGED
def test_long_prompt_persistent(paged):
    Case([(2500, 2600)], 16, 4, 128, torch.bfloat16, 700, 4, paged, seed=5).check()


@PAGED
def test_growing_scores(paged):
    """Scores that climb with the key's place, and rows whose first visible key comes late: the reference maximum follows."""
    c = Case([(600, 600)], 2, 1, 64, torch.bfloat16, 90, 1, paged, seed=6)
    c.q[...] = 0
    c.q[..., 0] = 1.0
    c.k[:600, :, 0] = (torch.arange(600) // 8).to(c.dtype)[:, None] * 4 - 150
    c.check()


@PAGED
def test_isolation_of_neighbours(paged):
    """A request whose keys and values are all NaN leaves the others' rows alone."""
    lens = [(50, 50), (40, 40), (130, 170)]
    c = Case(lens, 4, 2, 128, torch.bfloat16, 60, 2, paged, seed=7)
    want, want_lse, spread = c.want()
    c.k[50:90], c.v[50:90] = math.nan, math.nan
    out, lse = c.run()
    rows = torch.cat([torch.arange(50), torch.arange(90, 220)])
    check(out[rows.cuda()], lse[rows.cuda()], want[rows], want_lse[rows], spread[rows], c.dtype, one_p=True)


@PAGED
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_rows_in_front_of_the_keys_are_empty_whatever_the_others_see(paged, value):
    """20 rows over 5 keys: the first 15 see none of them."""
    c = Case([(20, 5)], 4, 2, 128, torch.bfloat16, 3, 0, paged, seed=40)
    c.v[:5] = value
    out, lse = c.run()
    assert (out[:15] == 0).all() and (lse[:15] == -math.inf).all() and (lse[15:] > -math.inf).all()


@PAGED
def test_row_offsets_behind_the_rows_are_clipped(paged):
    c = Case([(30, 30), (40, 60)], 4, 2, 64, torch.bfloat16, 20, 2, paged, seed=41)
    args = c.args()
    want, want_lse = c.call(*args)
    args[0] = torch.cat([args[0], args[0][:1]])[:70]
    args[3] = torch.tensor([0, 30, 2000], dtype=torch.int32, device="cuda")
    out, lse = c.call(*args)
    assert torch.equal(out[:30], want[:30]) and torch.equal(lse[:30], want_lse[:30])


def test_pages_of_unseen_keys_may_be_gone():
    c = Case([(70, 900), (5, 300)], 4, 2, 128, torch.bfloat16, 100, 3, True, seed=8)
    args = c.args()
    for r in range(2):
        unseen = torch.nonzero(~c.see[r].any(0)).flatten() + c.kp[r]
        args[5][unseen.cuda()] = 2 ** 31 - 1 if r else -1
    want, want_lse, spread = c.want()
    check(*c.call(*args), want, want_lse, spread, c.dtype, one_p=True)


@PAGED
@pytest.mark.parametrize("head,rest", [(0, 9), (5, 0), (5, 300)])
def test_rows_of_no_request(paged, head, rest):
    c = Case([(40, 60), (150, 150)], 4, 2, 64, torch.float16, 50, 2, paged, seed=9)
    want, want_lse, spread = c.want()
    args = c.args()
    n = args[0].shape[0]
    pad = lambda m: torch.full((m, *args[0].shape[1:]), math.nan, dtype=c.dtype, device="cuda")  # noqa: E731
    args[0] = torch.cat([pad(head), args[0], pad(rest)])
    args[3] = args[3] + head
    out, lse = c.call(*args)
    check(out[head:head + n], lse[head:head + n], want, want_lse, spread, c.dtype, one_p=True)
    for rows in (slice(0, head), slice(head + n, None)):
        assert (out[rows] == 0).all() and (lse[rows] == -math.inf).all()
    mine, mine_lse = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
    c.call(*args, out=mine, lse=mine_lse)
    assert torch.equal(mine[head:head + n], out[head:head + n]) and torch.equal(mine_lse[head:head + n], lse[head:head + n])
    for rows in (slice(0, head), slice(head + n, None)):
        assert (mine[rows] == 7).all() and (mine_lse[rows] == 7).all()
    mine_lse = torch.full_like(lse, 7.0)
    out2, _ = c.call(*args, lse=mine_lse)
    assert (out2[:head] == 0).all() and (mine_lse[:head] == 7).all()


@PAGED
def test_a_window_over_everything_is_the_plain_prefill(paged):
    ops = _ops()
    c = Case([(150, 150), (20, 400)], 8, 2, 128, torch.bfloat16, 400, 0, paged, seed=10)
    c.k.nan_to_num_(0.0), c.v.nan_to_num_(0.0)
    a = c.args()
    plain = (ops.gqa_paged_prefill if paged else ops.gqa_ragged_prefill)(*a[:-2])
    mine = c.call(*a)
    torch.testing.assert_close(plain[0].float(), mine[0].float(), rtol=2 ** -7, atol=2 ** -7)
    torch.testing.assert_close(plain[1], mine[1], rtol=0, atol=1e-4)


def test_prefill_then_decode():
    """A prompt of n tokens in one prefill, and its last token alone as a decode step, agree."""
    ops = _ops()
    c = Case([(333, 333)], 8, 2, 128, torch.bfloat16, 77, 5, True, seed=11)
    want, want_lse, spread = c.want()
    q, k, v, _, kp, idx, scale, window, sinks = c.args()
    out, lse = ops.gqa_paged_decode_window(q[-1:].contiguous(), k, v, kp, idx, None, scale, window, sinks)
    check(out, lse, want[-1:], want_lse[-1:], spread[-1:], c.dtype)
    full, full_lse = c.run()
    check(full[-1:], full_lse[-1:], want[-1:], want_lse[-1:], spread[-1:], c.dtype, one_p=True)


@PAGED
@pytest.mark.parametrize("rows", [200, 2600])
def test_captured_and_replayed(paged, rows):
    cs = [Case([(rows, rows), (5, 70)], 8, 2, 128, torch.bfloat16, 300, 4, paged, seed=20 + i) for i in range(2)]
    args = [c.args() for c in cs]
    ops = _ops()
    fn = ops.gqa_paged_prefill_window if paged else ops.gqa_ragged_prefill_window
    eager = [fn(*a) for a in args]
    torch.cuda.synchronize()
    graphs, held = [], []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(fn(*a))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for o, l in held:
            o.zero_(), l.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (o, l), (eo, el) in zip(held, eager):
            assert torch.equal(o, eo) and torch.equal(l, el)


def test_refusals():
    ops = _ops()
    c = Case([(20, 30)], 4, 2, 64, torch.bfloat16, 10, 1, True, seed=30)
    q, k, v, qp, kp, idx, scale, _, _ = c.args()
    for window, sinks in ((0, 0), (-1, 3), (5, -1)):
        with pytest.raises(ValueError):
            ops.gqa_paged_prefill_window(q, k, v, qp, kp, idx, scale, window, sinks)
        with pytest.raises(ValueError):
            ops.gqa_ragged_prefill_window(q, k[:, 0], v[:, 0], qp, kp, scale, window, sinks)
    bad = lambda error, fn, *a, **kw: pytest.raises(error, fn, *a, **kw)  # noqa: E731
    paged = lambda q=q, k=k, v=v, qp=qp, kp=kp, idx=idx, **kw: ops.gqa_paged_prefill_window(q, k, v, qp, kp, idx, scale, 10, 1, **kw)  # noqa: E731
    ragged = lambda q=q, k=k[:, 0], v=v[:, 0], qp=qp, kp=kp, **kw: ops.gqa_ragged_prefill_window(q, k, v, qp, kp, scale, 10, 1, **kw)  # noqa: E731
    for fn in (paged, ragged):
        bad(ValueError, fn, q=q.cpu())
        bad(ValueError, fn, q=q[:, :3].contiguous())
        bad(ValueError, fn, q=q[:, :, ::2])
        bad(TypeError, fn, q=q.half())
        bad(TypeError, fn, qp=qp.long())
        bad(ValueError, fn, qp=qp[:1].contiguous())
        bad(ValueError, fn, kp=kp.cpu())
        bad(ValueError, fn, out=torch.empty_like(q[:10]))
        bad(ValueError, fn, lse=torch.empty(20, 4, device="cuda", dtype=torch.float64))
    bad(ValueError, paged, idx=idx[:0])
    bad(TypeError, paged, idx=idx.long())
    bad(ValueError, paged, k=k[:, 0], v=v[:, 0])
    from cleave_b200 import Cb200Error

    odd = torch.zeros(20, 4, 96, device="cuda", dtype=torch.bfloat16)
    pool = torch.zeros(30, 2, 96, device="cuda", dtype=torch.bfloat16)
    bad(Cb200Error, ragged, q=odd, k=pool, v=pool)
