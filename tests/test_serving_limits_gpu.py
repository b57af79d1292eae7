"""The serving operators at the edges of what they accept: the most requests of a launch, rows of unusual widths, results that start on
a 16-byte boundary only."""

import math

import pytest
import torch

import test_kv_evict_gpu as evict
import test_prefill_window_gpu as prefill
from _serving import Paged, check

pytestmark = pytest.mark.gpu


def _small_batch(batch, d):
    """`batch` requests of 0 .. 4 tokens; the decode variants hold a table of them in shared memory."""
    return Paged([(7 * i) % 5 for i in range(batch)], 2, 1, d, 16, torch.bfloat16, seed=1)


@pytest.mark.parametrize("d,most", [(128, 3997), (64, 16285)])
@pytest.mark.parametrize("op", ["window", "weights", "prefix"])
def test_most_requests_of_a_launch(op, d, most):
    from cleave_b200 import Cb200Error, ops

    c = _small_batch(most, d)
    want, want_lse, ws, spread = c.want(lambda b, n: torch.ones(n, dtype=torch.bool))
    q, k, v, ptr, ids, last, scale = c.args()
    sums = torch.zeros(most, 1, 4, device="cuda")
    if op == "window":
        out, lse = ops.gqa_paged_decode_window(q, k, v, ptr, ids, last, scale, 4)
    elif op == "weights":
        out, lse = ops.gqa_paged_decode_weights(q, k, v, ptr, ids, last, scale, sums)
        for b in range(0, most, 97):
            n = c.lens[b]
            assert ((sums[b, 0, :n].double().cpu() - ws[b].sum(0)).abs() <= 2e-4 * ws[b].sum(0) + 2.0 ** -24).all()
            assert (sums[b, 0, n:] == 0).all()
    else:
        out, lse = ops.gqa_paged_decode_shared_prefix(q, k, v, ids[:1].contiguous(), 0, ptr, ids, last, scale)
    check(out, lse, want, want_lse, spread, c.dtype)
    c = _small_batch(most + 1, d)
    q, k, v, ptr, ids, last, scale = c.args()
    with pytest.raises(Cb200Error):
        if op == "window":
            ops.gqa_paged_decode_window(q, k, v, ptr, ids, last, scale, 4)
        elif op == "weights":
            ops.gqa_paged_decode_weights(q, k, v, ptr, ids, last, scale, torch.zeros(most + 1, 1, 4, device="cuda"))
        else:
            ops.gqa_paged_decode_shared_prefix(q, k, v, ids[:1].contiguous(), 0, ptr, ids, last, scale)


def test_many_requests_behind_a_prefix():
    """2000 requests: 16 blocks of query rows of one kv head."""
    import test_shared_prefix_gpu as prefix

    prefix.Case(200, [(7 * i) % 5 for i in range(2000)], 2, 1, 64, 16, torch.bfloat16, seed=2).check()


@pytest.mark.parametrize("paged", [False, True])
def test_many_prompts(paged):
    prefill.Case([(i % 3, i % 3 + i % 7) for i in range(3000)], 2, 1, 64, torch.float16, 5, 1, paged, seed=3).check()


def test_eviction_of_many_requests():
    evict.Case([(5 * i) % 23 for i in range(3000)], 2, 8, 4, torch.bfloat16, 9, max_len=22, seed=4).check(2, 3)


@pytest.mark.parametrize("d", [8, 24, 80, 192, 576])
def test_eviction_of_rows_of_any_width(d):
    evict.Case([0, 37, 200], 3, d, 16, torch.float16, 50, seed=d).check(2, 9)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("d", [64, 128])
def test_decode_into_results_on_a_16_byte_boundary(page, d):
    from cleave_b200 import ops

    c = Paged([300, 0, 70], 8, 2, d, page, torch.bfloat16, seed=5)
    args = c.args()
    want = ops.gqa_paged_decode_window(*args, 100, 4)
    room = torch.full((args[0].numel() + 16,), math.nan, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((3 * 8 + 1,), math.nan, device="cuda")
    got = ops.gqa_paged_decode_window(*args, 100, 4, out=room[8:-8].view(args[0].shape), lse=lse[1:].view(3, 8))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert room[:8].isnan().all() and room[-8:].isnan().all() and lse[0].isnan()


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_into_results_on_a_16_byte_boundary(paged, d):
    c = prefill.Case([(150, 200), (3, 0), (40, 40)], 4, 2, d, torch.bfloat16, 60, 2, paged, seed=6)
    args = c.args()
    want = c.call(*args)
    room = torch.full((args[0].numel() + 16,), math.nan, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((args[0].shape[0] * 4 + 1,), math.nan, device="cuda")
    got = c.call(*args, out=room[8:-8].view(args[0].shape), lse=lse[1:].view(-1, 4))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert room[:8].isnan().all() and room[-8:].isnan().all() and lse[0].isnan()
