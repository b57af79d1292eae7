"""A key that a row sees and whose score is NaN: the row's softmax is NaN, in the output, the log-sum-exp and the weights. Rows that do not see it are as
they were."""

import math

import pytest
import torch

import test_prefill_window_gpu as prefill
import test_shared_prefix_gpu as prefix
from _serving import DT, Paged

pytestmark = pytest.mark.gpu


def _rows_are_nan(got, clean, bad):
    """Rows `bad` (a mask over the first axis) are NaN, the others the same bits as in `clean`."""
    for x, y in zip(got, clean):
        assert x[bad].isnan().all()
        assert torch.equal(x[~bad], y[~bad])


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("at", [range(3, 4), range(0, 128), range(699, 700)])
@pytest.mark.parametrize("kind", ["window", "weights"])
def test_decode(kind, at, page, dt):
    from cleave_b200 import ops

    c = Paged([700, 300], 8, 2, 128, page, DT[dt], seed=1)
    got = []
    for poison in (False, True):
        for t in at if poison else ():
            c.k[c.ids[t // page], t % page] = math.nan
        if kind == "window":
            got.append(ops.gqa_paged_decode_window(*c.args(), 600, 150))
        else:
            sums = torch.zeros(2, 2, 700, device="cuda")
            got.append((*ops.gqa_paged_decode_weights(*c.args(), sums), sums))
    _rows_are_nan(got[1], got[0], torch.tensor([True, False], device="cuda"))


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("at", [range(3, 4), range(0, 128), range(499, 500)])
def test_shared_prefix(at, page):
    c = prefix.Case(500, [0, 70], 8, 2, 128, page, torch.bfloat16, seed=2)
    for t in at:
        c.k[c.pre_ids[t // page], t % page] = math.nan
    for bound in (0, 1):
        assert all(x.isnan().all() for x in c.run(max_ctas=bound))


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("at", [range(3, 4), range(0, 128), range(130, 258)])
def test_window_prefill(at, paged):
    """Rows 0 .. 399 over 400 keys and a window of 300; a tile of NaN in front of finite ones among them."""
    c = prefill.Case([(400, 400)], 4, 2, 128, torch.bfloat16, 300, 2, paged, seed=3)
    clean = c.run()
    c.k[list(at)] = math.nan
    p = torch.arange(400)
    bad = torch.zeros(400, dtype=torch.bool)
    for t in at:
        bad |= (p >= t) & ((p < t + 300) | (t < 2))
    _rows_are_nan(c.run(), clean, bad.cuda())
