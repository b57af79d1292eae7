"""What the kernel just in front of a call writes is what the call reads. The second kernel of the shared prefix reads Q, tables and the
requests' own tokens, and the eviction's copy tables and rows, without waiting for the first kernel of their call, which
starts them only once everything before it is done."""

import pytest
import torch

from _serving import Paged

pytestmark = pytest.mark.gpu


def _i32(v):
    return torch.as_tensor(v, dtype=torch.int32).cuda()


class Steps:
    """Two sets of inputs that are written, in turn, into one set of buffers right before each call."""

    def __init__(self, op):
        self.op, self.page = op, 16
        lens = [[300, 33, 0, 180, 64], [90, 0, 210, 17, 333]]
        cs = [Paged(n, 32, 8, 128, self.page, torch.bfloat16, seed=i, extra=120 - sum(-(-x // 16) for x in n)) for i, n in enumerate(lens)]
        args = [c.args() for c in cs]
        n_ids = max(a[4].numel() for a in args)
        g = torch.Generator().manual_seed(9)
        self.x = [torch.randn(5, 256, generator=g).to(torch.bfloat16).cuda() for _ in cs]
        self.w = (torch.randn(256, 4096, generator=g) / 16).to(torch.bfloat16).cuda()
        pad = lambda t: torch.cat([t, t.new_zeros(n_ids - t.numel())])  # noqa: E731
        self.sets = [dict(k=a[1].nan_to_num_(0.0), v=a[2].nan_to_num_(0.0), ptr=a[3], ids=pad(a[4]), last=a[5], pre=_i32(torch.randperm(120, generator=g)[:50]),
                          sums=torch.rand(5, 8, 333, generator=g).cuda(), dptr=_i32([0, 4, 7, 11, 12, 16]),
                          dst=_i32([t for t in range(120) if t not in set(c.ids.tolist())][:16])) for a, c in zip(args, cs)]
        self.buf = {name: torch.empty_like(t) for name, t in self.sets[0].items()}
        self.q = torch.empty(5, 32, 128, dtype=torch.bfloat16, device="cuda")

    def step(self, i):
        """Writes set i and calls; Q last, by a kernel that lets the next one start early."""
        from cleave_b200 import ops

        b = self.buf
        for name, t in self.sets[i].items():
            b[name].copy_(t)
        if self.op == "evict":
            r = ops.kv_cache_evict(b["k"], b["v"], b["sums"], b["ptr"], b["ids"], b["last"], b["dptr"], b["dst"], budget=64, sinks=4, recent=30)
            return (*r, b["k"].clone(), b["v"].clone())
        ops.matmul(self.x[i], self.w, out=self.q.view(5, 4096))
        if self.op == "prefix":
            return ops.gqa_paged_decode_shared_prefix(self.q, b["k"], b["v"], b["pre"], 790, b["ptr"], b["ids"], b["last"], 0.09)
        return (*ops.gqa_paged_decode_weights(self.q, b["k"], b["v"], b["ptr"], b["ids"], b["last"], 0.09, b["sums"]), b["sums"].clone())


@pytest.mark.parametrize("op", ["prefix", "weights", "evict"])
@pytest.mark.parametrize("captured", [False, True])
def test_inputs_written_right_before_the_call(op, captured):
    s = Steps(op)
    want = []
    for i in range(2):
        want.append([t.clone() for t in s.step(i)])
        torch.cuda.synchronize()
    order = [0, 1, 1, 0, 1, 0, 0, 1] * 3
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = [s.step(i) for i in order]
        for _ in range(3):
            graph.replay()
    else:
        got = [s.step(i) for i in order]
    torch.cuda.synchronize()
    for i, r in zip(order, got):
        assert all(torch.equal(a, b) for a, b in zip(r, want[i]))
