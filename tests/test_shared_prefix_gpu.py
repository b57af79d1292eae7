"""Decode of a batch that shares a prefix, against a 64-bit form over prefix ++ own tokens."""

import math

import pytest
import torch

from _serving import DT, Paged, check

pytestmark = pytest.mark.gpu


def _ops():
    from cleave_b200 import ops

    return ops


class Case(Paged):
    """The prefix is one more request of the same pool, the last one, which has no query."""

    def __init__(self, prefix, lens, hq, hkv, d, page, dtype, seed=0):
        super().__init__([*lens, prefix], hq, hkv, d, page, dtype, seed=seed)
        self.prefix = prefix
        self.before = self.rows(len(lens))
        self.lens.pop()
        n = self.ptr.pop()
        self.pre_ids, self.ids = self.ids[self.ptr[-1]:n], self.ids[:self.ptr[-1]]
        self.last.pop()
        self.q = self.q[:-1].contiguous()

    def run(self, extra_pages=0, **kw):
        ops = _ops()
        q, k, v, ptr, ids, last, scale = self.args()
        pre = torch.cat([self.pre_ids, torch.full((extra_pages,), -1)]).to(torch.int32).cuda()
        out, lse = torch.full_like(q, math.nan), torch.full(q.shape[:2], math.nan, device="cuda")
        ops.gqa_paged_decode_shared_prefix(q, k, v, pre, self.prefix, ptr, ids, last, scale, out=out, lse=lse, **kw)
        ops.check_workspace(ops.workspace("attn_decode", 0, "cuda"))
        return out, lse

    def check(self, **kw):
        want, want_lse, _, spread = self.want(lambda b, n: torch.ones(n, dtype=torch.bool), self.before)
        check(*self.run(**kw), want, want_lse, spread, self.dtype, one_p=True)


LENS = [0, 1, 15, 64, 65, 300]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("page", [1, 5, 16, 64, 128])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64), (40, 2, 128), (12, 4, 64)])
@pytest.mark.parametrize("prefix", [333, 64])
def test_shared_prefix(dt, page, hq, hkv, d, prefix):
    Case(prefix, LENS, hq, hkv, d, page, DT[dt], seed=page).check()


@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 65, 127, 128, 129, 191, 192, 193, 256, 1000, 5000])
@pytest.mark.parametrize("page", [16, 64])
def test_prefix_lengths(prefix, page):
    Case(prefix, [0, 1, 100], 8, 2, 128, page, torch.bfloat16, seed=3).check()


@pytest.mark.parametrize("batch,hq,hkv", [(1, 8, 2), (31, 8, 2), (32, 8, 2), (33, 8, 2), (130, 8, 2), (40, 20, 4), (9, 28, 2), (3, 128, 1), (3, 100, 1), (150, 2, 2)])
def test_blocks_of_query_rows(batch, hq, hkv):
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 40, (batch,), generator=g).tolist()
    Case(300, lens, hq, hkv, 64, 16, torch.float16, seed=4).check()


@pytest.mark.parametrize("page", [16, 64])
def test_nothing_behind_the_prefix(page):
    Case(500, [0, 0, 0], 8, 2, 128, page, torch.bfloat16, seed=5).check()
    c = Case(0, [0, 0], 8, 2, 128, page, torch.bfloat16, seed=5)
    out, lse = c.run()
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("big", [1.0, 40.0])
def test_growing_scores(page, big):
    """Keys whose scores climb along the prefix: the reference maximum has to follow them. Scores of +-40 * sqrt(D) * scale
    would leave the tolerance's data range, so the climbing keys are multiples of one direction that q holds exactly."""
    c = Case(900, [5, 0], 4, 2, 64, page, torch.bfloat16, seed=6)
    c.q[...] = 0
    c.q[..., 0] = 1.0
    for t in range(900):
        c.k[c.pre_ids[t // page], t % page, :, 0] = round(t / 899 * 32) * 0.25 * big
    c.before = tuple(x[c.pre_ids].flatten(0, 1)[:900] for x in (c.k, c.v))
    c.check()


def _low_scores(c, n, first):
    """Keys whose scores are exact products, about -280 in log2 units; the first `first` of the prefix score -inf."""
    c.q[...] = 0
    c.q[..., 0] = 4.0
    live = torch.arange(c.k[..., 0].numel()).view(c.k.shape[:-1]) % 8
    c.k[..., 0] = -(384.0 + 2 * live).to(c.dtype)
    for t in range(first):
        c.k[c.pre_ids[t // c.page], t % c.page, :, 0] = -math.inf
    c.before = tuple(x[c.pre_ids].flatten(0, 1)[:n] for x in (c.k, c.v))


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("max_ctas", [0, 1])  # every tile a part of its own; all of them one part
@pytest.mark.parametrize("first", [128, 200, 300])
def test_keys_of_weight_zero_in_front_of_low_scores(first, max_ctas, page):
    """A part of the prefix, or its first tile, whose scores are all -inf holds nothing: no score of 0 that would outweigh the others."""
    c = Case(300, [0, 70, 1], 4, 2, 64, page, torch.bfloat16, seed=11)
    _low_scores(c, 300, first)
    c.check(max_ctas=max_ctas)


def test_more_prefix_pages_than_used():
    Case(130, [3, 70], 8, 2, 128, 64, torch.bfloat16, seed=7).check(extra_pages=4)


def test_small_grid_and_bit_stability():
    c = Case(3000, [700, 5, 64], 32, 8, 128, 64, torch.bfloat16, seed=8)
    c.check(max_ctas=3)
    a, b = c.run(), c.run()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_agrees_with_decode_over_joined_tables():
    ops, c = _ops(), Case(640, [100, 3, 700], 8, 2, 128, 64, torch.float16, seed=9)
    c.k.nan_to_num_(0.0), c.v.nan_to_num_(0.0)
    q, k, v, ptr, ids, last, scale = c.args()
    joined, jptr = [], [0]
    for b in range(3):
        joined += [c.pre_ids, c.ids[c.ptr[b]:c.ptr[b + 1]]]
        jptr.append(jptr[-1] + 10 + c.ptr[b + 1] - c.ptr[b])
    a = ops.gqa_paged_decode(q, k, v, torch.tensor(jptr, dtype=torch.int32).cuda(), torch.cat(joined).to(torch.int32).cuda(), last, scale)
    b = c.run()
    torch.testing.assert_close(a[0].float(), b[0].float(), rtol=2 ** -9, atol=2 ** -9)
    torch.testing.assert_close(a[1], b[1], rtol=0, atol=1e-4)


def test_page_ids_outside_the_pool_are_clipped():
    c = Case(300, [20, 0], 8, 2, 128, 64, torch.bfloat16, seed=10)
    c.k.nan_to_num_(0.0), c.v.nan_to_num_(0.0)
    c.pre_ids = c.pre_ids.clone()
    c.pre_ids[1], c.pre_ids[2] = -7, 10 ** 9
    a = c.run()
    c.pre_ids[1], c.pre_ids[2] = 0, c.k.shape[0] - 1
    b = c.run()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_captured_and_replayed():
    ops = _ops()
    cs = [Case(700, [300, 0, 5], 8, 2, 128, 64, torch.bfloat16, seed=20 + i) for i in range(2)]
    args = [c.args() for c in cs]
    pre = [c.pre_ids.to(torch.int32).cuda() for c in cs]
    call = lambda i: ops.gqa_paged_decode_shared_prefix(*args[i][:3], pre[i], 700, *args[i][3:])  # noqa: E731
    eager = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    graphs, held = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(call(i))
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
        for i in range(2):
            assert torch.equal(held[i][0], eager[i][0]) and torch.equal(held[i][1], eager[i][1])


def test_refusals():
    from cleave_b200 import Cb200Error

    ops, c = _ops(), Case(100, [20, 5], 8, 2, 128, 16, torch.bfloat16, seed=30)
    q, k, v, ptr, ids, last, scale = c.args()
    pre = c.pre_ids.to(torch.int32).cuda()
    call = lambda pre=pre, n=100, q=q, k=k, v=v: ops.gqa_paged_decode_shared_prefix(q, k, v, pre, n, ptr, ids, last, scale)  # noqa: E731
    for n in (-1, pre.numel() * 16 + 1):
        with pytest.raises(ValueError):
            call(n=n)
    with pytest.raises(TypeError):
        call(pre=pre.long())
    with pytest.raises(ValueError):
        call(pre=pre.cpu())
    with pytest.raises(ValueError):
        call(q=q.cpu())
    wide = torch.zeros(2, 130, 64, device="cuda", dtype=torch.bfloat16)
    pool = torch.zeros(20, 16, 1, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(Cb200Error):
        call(q=wide, k=pool, v=pool)
