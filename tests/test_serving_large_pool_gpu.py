"""The serving operators on pools whose offsets pass 32 bits: the same pages at the end of a pool of 5 GB give the same bits as
in a small pool."""

import pytest
import torch

pytestmark = pytest.mark.gpu

HQ, HKV, D, DT = 32, 8, 128, torch.bfloat16
ROW = HKV * D * 2  # bytes of a token in K or V


def _pools(page, pages):
    """Small caches of `pages` pages, and large ones that hold the same pages at their end; the first page id there."""
    g = torch.Generator().manual_seed(page)
    small = [torch.randn(pages, page, HKV, D, generator=g).to(DT).cuda() for _ in range(2)]
    total = 5 * 2 ** 30 // (page * ROW) + pages
    large = [torch.empty(total, page, HKV, D, dtype=DT, device="cuda") for _ in range(2)]
    for a, b in zip(small, large):
        b[total - pages:] = a
    assert large[0].numel() > 2 ** 31
    return small, large, total - pages


def _i32(v):
    return torch.as_tensor(v, dtype=torch.int32).cuda()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("op", ["window", "weights", "prefix"])
def test_decode(op, page):
    from cleave_b200 import ops

    lens = [700, 65, 300]
    small, large, base = _pools(page, 90)
    need = [-(-n // page) for n in lens]
    ids = torch.randperm(90, generator=torch.Generator().manual_seed(1))[:sum(need)]
    ptr = _i32([0, need[0], need[0] + need[1], sum(need)])
    last = _i32([n - (p - 1) * page for n, p in zip(lens, need)])
    q = torch.randn(3, HQ, D, generator=torch.Generator().manual_seed(2)).to(DT).cuda()
    got = []
    for (k, v), shift in ((small, 0), (large, base)):
        t = _i32(ids + shift)
        if op == "window":
            got.append(ops.gqa_paged_decode_window(q, k, v, ptr, t, last, 0.09, 200, 5))
        elif op == "weights":
            sums = torch.zeros(3, HKV, 700, device="cuda")
            got.append((*ops.gqa_paged_decode_weights(q, k, v, ptr, t, last, 0.09, sums), sums))
        else:
            got.append(ops.gqa_paged_decode_shared_prefix(q, k, v, t, 130, ptr, t, last, 0.09))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_eviction():
    from cleave_b200 import ops

    small, large, base = _pools(16, 80)
    sums = torch.rand(1, HKV, 700, generator=torch.Generator().manual_seed(3)).cuda()
    got = []
    for (k, v), shift in ((small, 0), (large, base)):
        r = ops.kv_cache_evict(k, v, sums, _i32([0, 44]), _i32(torch.arange(44) + shift), _i32([12]), _i32([0, 20]),
                               _i32(torch.arange(50, 70) + shift), budget=320, sinks=4, recent=50)
        got.append((*r, k[shift:], v[shift:]))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("paged", [False, True])
def test_prefill(paged):
    from cleave_b200 import ops

    small, large, base = _pools(1, 600)
    q = torch.randn(150, HQ, D, generator=torch.Generator().manual_seed(4)).to(DT).cuda()
    qp = _i32([0, 0, 150])
    if paged:
        ids = torch.randperm(600, generator=torch.Generator().manual_seed(5))
        got = [ops.gqa_paged_prefill_window(q, k, v, qp, _i32([0, 0, 600]), _i32(ids + shift), 0.09, 100, 3)
               for (k, v), shift in ((small, 0), (large, base))]
    else:  # a request without query rows in front of the one that is computed
        got = [ops.gqa_ragged_prefill_window(q, k[:, 0], v[:, 0], qp, _i32([0, shift, shift + 600]), 0.09, 100, 3)
               for (k, v), shift in ((small, 0), (large, base))]
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_counts_past_32_bits_are_refused():
    """Tables and accumulators of 2 ** 32 + 4 entries, which a 32-bit count would take for 4. Nothing of them is read."""
    from cleave_b200 import ops

    (k, v), _, _ = _pools(64, 6)
    q = torch.zeros(1, HQ, D, dtype=DT, device="cuda")
    n = 2 ** 32 + 4
    ptr, ids, last = _i32([0, 2]), _i32([0, 1]), _i32([64])
    many = torch.empty(n, dtype=torch.int32, device="cuda")
    sums = torch.zeros(1, HKV, 100, device="cuda")
    bad = lambda fn, *a, **kw: pytest.raises(ValueError, fn, *a, **kw).match("2\\*\\*31")  # noqa: E731
    bad(ops.gqa_paged_decode_window, q, k, v, ptr, many, last, 0.1, 10)
    bad(ops.gqa_paged_decode_weights, q, k, v, ptr, many, last, 0.1, sums)
    bad(ops.gqa_paged_decode_shared_prefix, q, k, v, many, 100, ptr, ids, last, 0.1)
    bad(ops.gqa_paged_decode_shared_prefix, q, k, v, many[:2 ** 26 + 1], 2 ** 32 + 1, ptr, ids, last, 0.1)
    bad(ops.kv_cache_evict, k, v, sums, ptr, many, last, ptr, ids, budget=8)
    bad(ops.kv_cache_evict, k, v, sums, ptr, ids, last, ptr, many, budget=8)
    bad(ops.gqa_paged_prefill_window, q, k.view(-1, 1, HKV, D), v.view(-1, 1, HKV, D), _i32([0, 1]), ptr, many, 0.1, 10)
    del many
    one_head = [torch.zeros(4, 64, 1, D, dtype=DT, device="cuda") for _ in range(2)]
    wide = torch.empty(1, 1, n, device="cuda")
    bad(ops.gqa_paged_decode_weights, q[:, :4].contiguous(), *one_head, ptr, ids, last, 0.1, wide)
    bad(ops.kv_cache_evict, *one_head, wide, ptr, ids, last, ptr, _i32([2, 3]), budget=8)


@pytest.mark.parametrize("last", [2 ** 31 - 1, 17, -1, -2 ** 31])
@pytest.mark.parametrize("op", ["plain", "window", "weights", "prefix", "evict"])
def test_last_page_lengths_are_clipped_to_the_page(op, last):
    """Whatever the table says about a last page, it holds between 0 and all of its 16 tokens; 2 ** 31 - 1 must not wrap to none."""
    from cleave_b200 import ops

    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(12, 16, 2, 64, generator=g).to(DT).cuda() for _ in range(2))
    q, sums = torch.randn(2, 8, 64, generator=g).to(DT).cuda(), torch.rand(2, 2, 80, generator=g).cuda()
    ptr, ids = _i32([0, 5, 7]), _i32([3, 0, 5, 1, 2, 4, 6])
    got = []
    for n in (last, min(max(last, 0), 16)):
        table = (ptr, ids, _i32([n, 9]))
        if op == "evict":
            kk, vv = k.clone(), v.clone()
            got.append((*ops.kv_cache_evict(kk, vv, sums, *table, _i32([0, 2, 4]), _i32([7, 8, 9, 10]), budget=30, sinks=2, recent=5), kk, vv))
        elif op == "weights":
            w = sums.clone()
            got.append((*ops.gqa_paged_decode_weights(q, k, v, *table, 0.1, w), w))
        elif op == "prefix":
            got.append(ops.gqa_paged_decode_shared_prefix(q, k, v, ids, 30, *table, 0.1))
        elif op == "window":
            got.append(ops.gqa_paged_decode_window(q, k, v, *table, 0.1, 50, 2))
        else:
            got.append(ops.gqa_paged_decode(q, k, v, *table, 0.1))
    assert all(torch.equal(a, b) for a, b in zip(*got))
