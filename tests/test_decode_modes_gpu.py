"""Decode over a sliding window with sinks, and decode that accumulates attention weights, against 64-bit forms."""

import math

import pytest
import torch

from _serving import DT, Paged, check

pytestmark = pytest.mark.gpu


def _ops():
    from cleave_b200 import ops

    return ops


def _window_see(window, sinks):
    def see(b, n):
        j = torch.arange(n)
        return (j >= n - window) | (j < sinks)

    return see


def _run_window(c, window, sinks, **kw):
    ops = _ops()
    args = c.args()
    out = torch.full_like(args[0], math.nan)
    lse = torch.full(args[0].shape[:2], math.nan, device="cuda")
    ops.gqa_paged_decode_window(*args, window, sinks, out=out, lse=lse, **kw)
    ops.check_workspace(ops.workspace("attn_decode", 0, "cuda"))
    return out, lse


def _check_window(c, window, sinks, **kw):
    want, want_lse, _, spread = c.want(_window_see(window, sinks))
    out, lse = _run_window(c, window, sinks, **kw)
    check(out, lse, want, want_lse, spread, c.dtype)


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 127, 129, 300, 700]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("page", [1, 5, 16, 64, 128])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64), (40, 2, 128), (12, 4, 64)])
@pytest.mark.parametrize("window,sinks", [(128, 4), (65, 0), (1, 1)])
def test_window_decode(dt, page, hq, hkv, d, window, sinks):
    _check_window(Paged(LENS, hq, hkv, d, page, DT[dt], seed=page), window, sinks)


@pytest.mark.parametrize("window", [1, 16, 63, 64, 65, 100, 640, 2 ** 31 - 1, 2 ** 40])
@pytest.mark.parametrize("sinks", [0, 1, 15, 16, 64, 100, 700, 2 ** 31 - 1])
def test_window_and_sink_counts(window, sinks):
    _check_window(Paged(LENS + [64 * 9], 8, 2, 128, 64, torch.bfloat16, seed=3), window, sinks)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_tokens_outside_the_window_do_not_matter(page, value):
    c = Paged([700, 90, 333], 8, 2, 128, page, torch.bfloat16, seed=5)
    window, sinks = 77, 5
    for b, n in enumerate(c.lens):
        c.poison(b, range(sinks, n - window), value)
    _check_window(c, window, sinks)


def test_pages_behind_the_window_may_be_gone():
    """Table entries of pages without a token that takes part name no page at all."""
    c = Paged([900, 640], 8, 2, 128, 64, torch.bfloat16, seed=6)
    want, want_lse, _, spread = c.want(_window_see(130, 4))
    args = c.args()
    table = args[4].clone()
    table[1:(900 - 130) // 64] = -1
    table[15 + 1:15 + (640 - 130) // 64] = 2 ** 31 - 1
    args[4] = table
    out, lse = _ops().gqa_paged_decode_window(*args, 130, 4)
    check(out, lse, want, want_lse, spread, c.dtype)


@pytest.mark.parametrize("max_ctas", [1, 3, 0])
def test_window_decode_cut_over_ctas(max_ctas):
    _check_window(Paged([5000, 1, 300, 4097], 8, 2, 128, 64, torch.float16, seed=7), 4000, 70, max_ctas=max_ctas)


def test_a_window_over_everything_is_the_plain_decode():
    ops, c = _ops(), Paged([700, 0, 129], 8, 2, 128, 64, torch.bfloat16, seed=8)
    c.k.nan_to_num_(0.0), c.v.nan_to_num_(0.0)
    a, b = ops.gqa_paged_decode(*c.args()), ops.gqa_paged_decode_window(*c.args(), 700)
    torch.testing.assert_close(a[0].float(), b[0].float(), rtol=2 ** -7, atol=2 ** -7)  # P is rounded once more in the first
    torch.testing.assert_close(a[1], b[1], rtol=0, atol=1e-4)


def test_window_decode_is_bit_stable():
    c = Paged([3000, 1, 2222], 32, 8, 128, 64, torch.bfloat16, seed=9)
    a, b = _run_window(c, 1500, 4), _run_window(c, 1500, 4)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def _run_weights(c, sums, **kw):
    ops = _ops()
    out, lse = ops.gqa_paged_decode_weights(*c.args(), sums, **kw)
    ops.check_workspace(ops.workspace("attn_decode", 0, "cuda"))
    return out, lse


def _check_weights(c, max_len, steps=1, **kw):
    want, want_lse, ws, spread = c.want(lambda b, n: torch.ones(n, dtype=torch.bool))
    g = torch.Generator().manual_seed(1)
    start = torch.rand(len(c.lens), c.hkv, max_len, generator=g)
    sums = start.cuda()
    for _ in range(steps):
        out, lse = _run_weights(c, sums, **kw)
    check(out, lse, want, want_lse, spread, c.dtype)
    for b, n in enumerate(c.lens):
        n = min(n, max_len)
        grown = ws[b].view(c.hkv, c.hq // c.hkv, ws[b].shape[-1]).sum(1)[:, :n]
        total = start[b, :, :n].double() + steps * grown
        # each addition rounds to 2^-24 of the sum, each weight is off by the relative 2e-4
        assert ((sums[b, :, :n].double().cpu() - total).abs() <= steps * (2e-4 * grown + 2 ** -24 * total)).all()
        assert torch.equal(sums[b, :, n:].cpu(), start[b, :, n:])


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("page", [1, 5, 16, 64, 128])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64), (40, 2, 128), (12, 4, 64)])
def test_decode_weights(dt, page, hq, hkv, d):
    _check_weights(Paged(LENS, hq, hkv, d, page, DT[dt], seed=20 + page), 700)


@pytest.mark.parametrize("max_len", [1, 7, 64, 301, 2000])
def test_weights_of_tokens_that_fit(max_len):
    _check_weights(Paged([0, 1, 300, 1999], 8, 2, 128, 64, torch.bfloat16, seed=30), max_len, steps=2)


@pytest.mark.parametrize("lens", [[300, 41], [1], [0, 0], [64] * 5])
def test_accumulators_wider_than_the_page_table(lens):
    _check_weights(Paged(lens, 8, 2, 128, 16, torch.bfloat16, seed=34), 5003, steps=2)


def test_wide_accumulators_need_no_scratch_of_their_width():
    """Accumulators for 2^20 tokens over a page table of 320: the call's temporary memory follows the latter."""
    ops, c = _ops(), Paged([300], 8, 2, 128, 64, torch.bfloat16, seed=35)
    args, sums = c.args(), torch.zeros(1, 2, 1 << 20, device="cuda")
    ops.gqa_paged_decode_weights(*args, sums)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.gqa_paged_decode_weights(*args, sums)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20
    assert (sums[..., 300:] == 0).all()


def test_weights_of_requests_that_share_pages():
    """Three requests over one page list: every one has sums of its own."""
    c = Paged([300], 8, 2, 128, 64, torch.float16, seed=31, q_rows=3)
    want = []
    for r in range(3):
        one = Paged([300], 8, 2, 128, 64, torch.float16, seed=31, q_rows=3)
        one.q = c.q[r:r + 1]
        want.append(one.want(lambda b, n: torch.ones(n, dtype=torch.bool)))
    args = c.args()
    args[3] = torch.tensor([0, 5, 10, 15], dtype=torch.int32, device="cuda")
    args[4] = args[4].repeat(3)
    args[5] = args[5].repeat(3)
    sums = torch.zeros(3, 2, 300, device="cuda")
    out, lse = _ops().gqa_paged_decode_weights(*args, sums)
    for r, (o, l, w, spread) in enumerate(want):
        check(out[r:r + 1], lse[r:r + 1], o, l, spread, c.dtype)
        grown = w[0].view(2, 4, 300).sum(1)
        assert ((sums[r].double().cpu() - grown).abs() <= 2.1e-4 * grown).all()


@pytest.mark.parametrize("max_ctas", [1, 3, 0])
def test_weights_cut_over_ctas(max_ctas):
    _check_weights(Paged([5000, 1, 300, 4097], 8, 2, 128, 64, torch.float16, seed=32), 5000, max_ctas=max_ctas)


def test_sums_may_start_anywhere():
    c = Paged([70, 41], 4, 1, 64, 16, torch.bfloat16, seed=32)
    whole = torch.zeros(3, 1, 71, device="cuda")
    want = torch.zeros(2, 1, 71, device="cuda")
    _ops().gqa_paged_decode_weights(*c.args(), whole[1:])
    _ops().gqa_paged_decode_weights(*c.args(), want)
    assert torch.equal(whole[1:], want) and (whole[0] == 0).all()


def test_rows_without_a_finite_score_add_nothing():
    c = Paged([70, 40], 4, 2, 64, 16, torch.bfloat16, seed=31)
    c.q.abs_().add_(0.5)
    for t in range(40):
        c.poison(1, [t], -math.inf)
    sums = torch.full((2, 2, 70), 0.25, device="cuda")
    _ops().gqa_paged_decode_weights(*c.args(), sums)
    assert (sums[1] == 0.25).all() and (sums[0] > 0.25).all()


def test_weights_add_up_to_the_query_heads():
    c = Paged([700, 1, 64], 8, 2, 128, 64, torch.bfloat16, seed=33)
    sums = torch.zeros(3, 2, 704, device="cuda")
    _run_weights(c, sums)
    torch.testing.assert_close(sums.sum(-1), torch.full((3, 2), 4.0, device="cuda"), rtol=2e-4, atol=0)


@pytest.mark.parametrize("kind", ["window", "weights"])
def test_captured_and_replayed(kind):
    """Two graphs captured on one stream, replayed beside each other on two, give what the eager calls give."""
    ops = _ops()
    cs = [Paged([3000, 5, 700], 8, 2, 128, 64, torch.bfloat16, seed=40 + i) for i in range(2)]
    args = [c.args() for c in cs]
    sums = [torch.zeros(3, 2, 3000, device="cuda") for _ in cs]
    call = lambda i: (ops.gqa_paged_decode_window(*args[i], 2000, 4) if kind == "window"  # noqa: E731
                      else ops.gqa_paged_decode_weights(*args[i], sums[i]))
    eager = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    eager_sums = [s.clone() for s in sums]
    graphs, held = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(call(i))
        graphs.append(g)
    for s in sums:
        s.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for s in sums:
            s.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(held[i][0], eager[i][0]) and torch.equal(held[i][1], eager[i][1])
            if kind == "weights":
                assert torch.equal(sums[i], eager_sums[i])


def test_on_another_stream():
    ops, c = _ops(), Paged([3000, 5, 700], 8, 2, 128, 64, torch.bfloat16, seed=44)
    args = c.args()
    want = ops.gqa_paged_decode_window(*args, 2000, 4)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        got = ops.gqa_paged_decode_window(*args, 2000, 4)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals():
    ops, c = _ops(), Paged([30, 2], 8, 2, 128, 16, torch.bfloat16, seed=50)
    a = c.args()
    for window, sinks in ((0, 0), (-5, 0), (4, -1)):
        with pytest.raises(ValueError):
            ops.gqa_paged_decode_window(*a, window, sinks)
    with pytest.raises(ValueError):
        ops.gqa_paged_decode_window(a[0].transpose(0, 1), *a[1:], 8)
    with pytest.raises(TypeError):
        ops.gqa_paged_decode_window(*a[:3], a[3].long(), *a[4:], 8)
    with pytest.raises(ValueError):
        ops.gqa_paged_decode_window(*a[:4], a[4].cpu(), *a[5:], 8)
    with pytest.raises(TypeError):
        ops.gqa_paged_decode_window(*a[:5], None, a[6], 8)
    for bad in (torch.zeros(2, 2, 30, device="cuda", dtype=torch.float64), ):
        with pytest.raises(TypeError):
            ops.gqa_paged_decode_weights(*a, bad)
    for bad in (torch.zeros(2, 30, device="cuda"), torch.zeros(2, 8, 30, device="cuda"), torch.zeros(2, 2, 30),
                torch.zeros(2, 30, 2, device="cuda").transpose(1, 2)):
        with pytest.raises(ValueError):
            ops.gqa_paged_decode_weights(*a, bad)
    from cleave_b200 import Cb200Error

    with pytest.raises(Cb200Error):
        ops.gqa_paged_decode_weights(*a, torch.zeros(2, 2, 0, device="cuda"))
