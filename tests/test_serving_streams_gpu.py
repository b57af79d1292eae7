"""The serving operators on two streams at once: the same bits as one after the other."""

import pytest
import torch

from _serving import Paged

pytestmark = pytest.mark.gpu


def _i32(v):
    return torch.as_tensor(v, dtype=torch.int32).cuda()


def _calls(op, seed):
    """A call of the operator on inputs of its own, whose results are fresh tensors in every call."""
    from cleave_b200 import ops

    lens, budget, page = [900 + 100 * seed, 33, 500], 200, 16
    c = Paged(lens, 8, 2, 128, page, torch.bfloat16, seed=seed, extra=60)
    args = c.args()
    q, k, v, ptr, ids, last, scale = args
    if op == "window":
        return lambda: ops.gqa_paged_decode_window(*args, 300, 4)
    if op == "weights":
        def weights():
            sums = torch.zeros(3, 2, max(lens), device="cuda")
            return (*ops.gqa_paged_decode_weights(*args, sums), sums)
        return weights
    if op == "prefix":
        pre = ids[:40].contiguous()
        return lambda: ops.gqa_paged_decode_shared_prefix(q, k, v, pre, 633, ptr, ids, last, scale)
    if op == "evict":
        sums = torch.rand(3, 2, max(lens), generator=torch.Generator().manual_seed(seed)).cuda()
        room = [-(-min(n, budget) // page) for n in lens]
        dptr, dst = _i32([0, room[0], room[0] + room[1], sum(room)]), _i32(c.spare[:sum(room)])

        def evict():
            kk, vv = k.clone(), v.clone()
            r = ops.kv_cache_evict(kk, vv, sums, ptr, ids, last, dptr, dst, budget=budget, sinks=4, recent=30)
            return (*r, kk.view(torch.int16), vv.view(torch.int16))
        return evict
    g = torch.Generator().manual_seed(seed)
    rows = 700 + 200 * seed
    q, k, v = (torch.randn(rows, h, 128, generator=g).to(torch.bfloat16).cuda() for h in (8, 2, 2))
    qp = _i32([0, 150, rows])
    if op == "ragged":
        return lambda: ops.gqa_ragged_prefill_window(q, k, v, qp, qp, 0.09, 200, 4)
    perm = _i32(torch.randperm(rows, generator=g))
    return lambda: ops.gqa_paged_prefill_window(q, k[:, None], v[:, None], qp, qp, perm, 0.09, 200, 4)


@pytest.mark.parametrize("op", ["window", "weights", "prefix", "evict", "ragged", "paged"])
def test_two_streams_at_once(op):
    calls = [_calls(op, seed) for seed in range(2)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        got = [[], []]
        for _ in range(3):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    got[i].append(calls[i]())
        torch.cuda.synchronize()
        for i in range(2):
            for r in got[i]:
                assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_eager_calls_after_a_capture_on_their_stream(monkeypatch):
    """A graph of the plain decode is captured on a fresh stream and not replayed: what it allocated holds anything."""
    from cleave_b200 import ops

    c = Paged([900, 33, 500], 8, 2, 128, 16, torch.bfloat16, seed=3)
    c.k.nan_to_num_(0.0), c.v.nan_to_num_(0.0)
    args = c.args()
    want, plain = ops.gqa_paged_decode_window(*args, 300, 4), ops.gqa_paged_decode(*args)
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    monkeypatch.setattr(ops, "_workspaces", {})
    with torch.cuda.graph(graph, stream=stream):
        held = ops.gqa_paged_decode(*args)
    with torch.cuda.stream(stream):
        got = ops.gqa_paged_decode_window(*args, 300, 4)
    torch.cuda.synchronize()
    assert len(ops._workspaces) == 2
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, plain))
