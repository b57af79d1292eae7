"""Rows in which one key holds nearly all of the softmax weight and its value is zero, as attention sinks have it: the output is
then made of weights of 2^-16 .. 2^-24, which in fp16 are subnormal numbers or none."""

import math

import pytest
import torch

import test_prefill_window_gpu as prefill
import test_shared_prefix_gpu as prefix
from _serving import DT, Paged, check

pytestmark = pytest.mark.gpu

# The sink's score is one exact product (every other component of its key is zero), so the tolerances of _serving hold: the other
# scores keep their unit variance. On top of them, where P is a single 16-bit number: it is stored times 2^7, so a
# weight below 2^-21 of the reference is off by at most 2^-32 of the reference, evenly spread and independent of the others'
# errors: their sum over n values of unit variance stays below five of its standard deviations, 5 sqrt(n / 3) 2^-32, less than
# 6 sqrt(n) 2^-33 (the row's sum is at least 1).
NATS = [11.0, 14.0, 15.5]


def _dominate(c, at, nats, q0=4.0):
    """Component 0 of every query is q0 and of every key 0; the keys `at` (an index of c.k) have the score `nats`, and no value."""
    c.q[..., 0] = q0
    c.k[..., 0] = 0.0
    c.k[at], c.v[at] = 0.0, 0.0
    k0 = c.k[..., 0]
    k0[at] = nats / (c.scale * q0)


def _check(got, want, n, dtype, one_p):
    out, lse, spread = want
    extra = 6 * math.sqrt(n) * 2.0 ** -33 if one_p and dtype == torch.float16 else 0.0
    check(*got, out, lse, spread + extra / 2e-4, dtype, one_p=one_p)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("nats", NATS)
@pytest.mark.parametrize("kind", ["window", "weights"])
def test_decode(kind, nats, page, dt):
    from cleave_b200 import ops

    c = Paged([4100, 700], 8, 2, 128, page, DT[dt], seed=1)
    rows = [(c.ids[c.ptr[b] + t // page], t % page) for b in range(2) for t in (0, 17, 34, 51)]  # one in each warp's share of a tile
    _dominate(c, tuple(torch.tensor(x) for x in zip(*rows)), nats)
    see = lambda b, n: torch.ones(n, dtype=torch.bool)  # noqa: E731
    want, want_lse, _, spread = c.want(see)
    if kind == "window":
        got = ops.gqa_paged_decode_window(*c.args(), 4096, 64, max_ctas=1)
    else:
        got = ops.gqa_paged_decode_weights(*c.args(), torch.zeros(2, 2, 4100, device="cuda"), max_ctas=1)
    _check(got, (want, want_lse, spread), 4100, c.dtype, False)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("nats", NATS)
def test_window_prefill(nats, paged, dt):
    c = prefill.Case([(150, 4200)], 4, 2, 128, DT[dt], 4000, 4, paged, seed=2)
    _dominate(c, torch.tensor([0]), nats)
    _check(c.run(), c.want(), 4200, c.dtype, True)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("nats", NATS)
@pytest.mark.parametrize("own", [0, 300])
def test_shared_prefix(own, nats, page, dt):
    """The prefix in one part: whatever its first key dominates is scaled by that key's score."""
    c = prefix.Case(3000, [own, own], 8, 2, 128, page, DT[dt], seed=3)
    _dominate(c, (c.pre_ids[:1], torch.tensor([0])), nats)
    c.before = tuple(x[c.pre_ids].flatten(0, 1)[:3000] for x in (c.k, c.v))
    want, want_lse, _, spread = c.want(lambda b, n: torch.ones(n, dtype=torch.bool), c.before)
    _check(c.run(max_ctas=1), (want, want_lse, spread), 3000 + own, c.dtype, True)
