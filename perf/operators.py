"""The serving operators on paged caches, as cases that can be timed and compared: windowed attention with sinks
(decode and prefill), decode of a batch that shares a prefix, decode that accumulates attention weights, and the
eviction that reads them.

``run`` computes an operator in plain fp32 torch operations, or through ``cleave_b200.ops`` where ``own`` is true.
Lengths follow from a case alone (``lens_seed``), values and page tables from the seed given to ``prepare``.
"""

import math
import random

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
LOG2E = 1.4426950408889634


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a single chat request on a local-attention layer: one short launch, latency counts
        dict(name="window decode b1", op="window_decode", batch=1, hq=32, hkv=8, d=128, page=64, lo=700, hi=700, window=128, sinks=4, dtype="bf16", lens_seed=0),
        # an ordinary serving batch, small pages
        dict(name="window decode b64 p16", op="window_decode", batch=64, hq=32, hkv=8, d=128, page=16, lo=500, hi=8192, window=1000, sinks=4, dtype="f16", lens_seed=1),
        # the largest batch of the decode benchmark, long contexts cut to a window
        dict(name="window decode b128 p64", op="window_decode", batch=128, hq=32, hkv=8, d=128, page=64, lo=512, hi=16384, window=4096, sinks=64, dtype="bf16", lens_seed=2),
        # a few chunks of a chunked prefill, some of them single tokens, one token per page
        dict(name="window prefill chunks", op="window_prefill", paged=True, batch=5, hq=32, hkv=8, d=128, qlo=1, qhi=130, ctx=900, window=256, sinks=4, dtype="f16", lens_seed=3),
        # one long prompt
        dict(name="window prefill 8191", op="window_prefill", paged=False, batch=1, hq=32, hkv=8, d=128, qlo=8191, qhi=8191, ctx=0, window=1024, sinks=4, dtype="bf16", lens_seed=4),
        # a handful of users behind a short system prompt
        dict(name="shared prefix b4", op="shared_prefix", batch=4, hq=32, hkv=8, d=128, page=16, prefix=1000, lo=1, hi=64, dtype="f16", lens_seed=5),
        # a batch of samples of one prompt
        dict(name="shared prefix b64 8192", op="shared_prefix", batch=64, hq=32, hkv=8, d=128, page=64, prefix=8192, lo=1, hi=512, dtype="bf16", lens_seed=6),
        # many users behind one long document
        dict(name="shared prefix b128 32768", op="shared_prefix", batch=128, hq=32, hkv=8, d=128, page=64, prefix=32768, lo=100, hi=2048, dtype="bf16", lens_seed=7),
        # decode steps whose attention weights are accumulated for a later eviction
        dict(name="weights b8", op="weights", batch=8, hq=32, hkv=8, d=128, page=64, lo=100, hi=1500, dtype="bf16", lens_seed=8),
        dict(name="weights b64 p16", op="weights", batch=64, hq=32, hkv=8, d=128, page=16, lo=512, hi=8192, dtype="f16", lens_seed=9),
        # the eviction of one request, and of a batch that has outgrown its budget
        dict(name="evict b1", op="evict", batch=1, hkv=8, d=128, page=64, lo=1500, hi=1500, budget=512, sinks=4, recent=128, dtype="bf16", lens_seed=10),
        dict(name="evict b32", op="evict", batch=32, hkv=8, d=128, page=16, lo=1000, hi=8192, budget=2048, sinks=4, recent=500, dtype="bf16", lens_seed=11),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("window_decode", "window_prefill", "shared_prefix", "weights", "evict"))
    hq, hkv = rng.choice(((32, 8), (32, 8), (32, 4), (8, 8), (16, 2), (12, 4), (32, 1), (40, 8)))
    c = dict(op=op, hq=hq, hkv=hkv, d=rng.choice((64, 128, 128)), dtype=rng.choice(("bf16", "f16")), lens_seed=rng.randrange(1 << 20))
    if op != "window_prefill":
        c["page"] = rng.choice((1, 16, 32, 64, 64, 128))
    if op == "window_decode":
        c["batch"], c["hi"] = _log(rng, 1, 128), _log(rng, 64, 16384)
        c["lo"] = rng.randint(1, c["hi"])
        c["window"], c["sinks"] = _log(rng, 16, 4096), rng.choice((0, 1, 4, 4, 16, 64))
    elif op == "window_prefill":
        c["paged"], c["batch"], c["qhi"] = rng.choice((True, False)), _log(rng, 1, 12), _log(rng, 1, 4096)
        c["qlo"], c["ctx"] = rng.randint(1, c["qhi"]), rng.choice((0, 0, _log(rng, 1, 2048)))
        while c["batch"] > 1 and c["batch"] * c["hq"] * c["qhi"] * (c["qhi"] + c["ctx"]) > 32 * 8191 * 8191 // 2:
            c["batch"] -= 1
        c["window"], c["sinks"] = _log(rng, 16, 2048), rng.choice((0, 1, 4, 4, 16, 64))
    elif op == "shared_prefix":
        c["batch"], c["prefix"], c["hi"] = _log(rng, 1, 96), _log(rng, 16, 32768), _log(rng, 1, 2048)
        c["lo"] = rng.randint(1, c["hi"])
    elif op == "weights":
        c["batch"], c["hi"] = _log(rng, 1, 48), _log(rng, 16, 8192)
        c["lo"] = rng.randint(1, c["hi"])
    else:
        del c["hq"]
        c["batch"], c["hi"] = _log(rng, 1, 32), _log(rng, 200, 8192)
        c["lo"] = rng.randint(100, c["hi"])
        c["budget"] = _log(rng, 64, 2048)
        c["sinks"], c["recent"] = rng.choice((0, 1, 4, 16)), rng.randint(0, c["budget"] // 2)
    return c


def _lens(case, lo="lo", hi="hi"):
    r = random.Random("%d %s" % (case["lens_seed"], lo))
    return [r.randint(case[lo], case[hi]) for _ in range(case["batch"])]


def _prefill_lens(case):
    """(query rows, keys) of each request: whole prompts, or chunks behind a context of up to `ctx` tokens."""
    r = random.Random("%d ctx" % case["lens_seed"])
    q = _lens(case, "qlo", "qhi")
    return q, [n + (r.randint(0, case["ctx"]) if case["ctx"] else 0) for n in q]


def _seen(n_q, n_kv, window, sinks):
    """Visible (query, key) pairs of one request."""
    p = range(n_kv - n_q, n_kv)
    return sum(min(i + 1, window) + min(sinks, max(0, i + 1 - window)) for i in p)


def work(case):
    d, op, hkv = case["d"], case["op"], case["hkv"]
    row = 2 * hkv * d * 2  # bytes of one token's K and V rows
    if op == "evict":
        lens = _lens(case)
        kept = [min(n, case["budget"]) for n in lens]
        sums = 4 * hkv * (sum(lens) + case["batch"] * max(lens))
        return {"bytes": 2 * row * sum(kept) + sums + 4 * hkv * sum(kept), "flops": 0}
    hq = case["hq"]
    if op == "window_prefill":
        nq, nk = _prefill_lens(case)
        pairs = sum(_seen(a, b, case["window"], case["sinks"]) for a, b in zip(nq, nk))
        return {"bytes": sum(nk) * row + sum(nq) * hq * (4 * d + 4), "flops": 4 * d * hq * pairs}
    lens, qo = _lens(case), case["batch"] * hq * (4 * d + 4)
    if op == "window_decode":
        t = sum(min(n, case["window"] + case["sinks"]) for n in lens)
        return {"bytes": t * row + qo, "flops": 4 * d * hq * t}
    if op == "shared_prefix":
        t, p = sum(lens), case["prefix"]
        return {"bytes": (t + p) * row + qo, "flops": 4 * d * hq * (t + p * case["batch"])}
    t = sum(lens)
    return {"bytes": t * row + qo + 8 * hkv * t, "flops": 4 * d * hq * t}


# ------------------------------------------------------------------------------------------------ inputs
def _table(lens, page):
    """(indptr in pages, tokens of each request's last page)."""
    pages = [-(-n // page) for n in lens]
    ptr = [0]
    for p in pages:
        ptr.append(ptr[-1] + p)
    return ptr, [n - (p - 1) * page if p else 0 for n, p in zip(lens, pages)]


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, d, hkv = DT[case["dtype"]], case["d"], case["hkv"]
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.float32).to(dt)  # noqa: E731
    rn16 = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=dt)  # noqa: E731
    perm = lambda n: torch.randperm(n, generator=g, device="cuda").to(torch.int32)  # noqa: E731
    s = dict(case=case, scale=d ** -0.5)
    if case["op"] == "window_prefill":
        nq, nk = _prefill_lens(case)
        tq, tk = sum(nq), sum(nk)
        qp, kp = [0], [0]
        for a, b in zip(nq, nk):
            qp.append(qp[-1] + a)
            kp.append(kp[-1] + b)
        s.update(q=1.5 * rn(tq, case["hq"], d), qo_indptr=_i32(qp), kv_indptr=_i32(kp), lq=max(nq), lk=max(nk))
        if case["paged"]:
            s.update(k=rn16(tk + 7, 1, hkv, d), v=rn16(tk + 7, 1, hkv, d), kv_indices=perm(tk + 7)[:tk].contiguous())
        else:
            s.update(k=rn16(tk, hkv, d), v=rn16(tk, hkv, d))
        return s
    page, lens = case["page"], _lens(case)
    ptr, last = _table(lens, page)
    s.update(page=page, longest=max(lens), kv_indptr=_i32(ptr), last=_i32(last))
    extra = 0
    if case["op"] == "shared_prefix":
        extra = -(-case["prefix"] // page)
    elif case["op"] == "evict":
        dptr, _ = _table([min(n, case["budget"]) for n in lens], page)
        extra = dptr[-1]
        s["dst_indptr"] = _i32(dptr)
    order = perm(ptr[-1] + extra)
    s.update(kv_indices=order[:ptr[-1]].contiguous(), other=order[ptr[-1]:].contiguous(),
             k=rn16(ptr[-1] + extra, page, hkv, d), v=rn16(ptr[-1] + extra, page, hkv, d))
    if case["op"] in ("weights", "evict"):
        # sums of attention weights are heavy-tailed; tokens behind a request's end have none
        w = torch.randn(case["batch"], hkv, max(lens), generator=g, device="cuda").mul_(2.0).sub_(5.0).exp_()
        w.masked_fill_(torch.arange(max(lens), device="cuda") >= _i32(lens)[:, None, None], 0.0)
        s["sums"] = w
    if case["op"] != "evict":
        s["q"] = 1.5 * rn(case["batch"], case["hq"], d)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _rows(s, pos, live):
    """fp32 K and V rows (batch, HKV, tokens, D) of the tokens `pos` of every request."""
    at = s["kv_indptr"][:-1, None].long() + torch.where(live, pos, 0) // s["page"]
    page = s["kv_indices"][at.clamp_(max=s["kv_indices"].numel() - 1)].long()
    slot = torch.where(live, pos, 0) % s["page"]
    return (s["k"][page, slot].float().transpose(1, 2), s["v"][page, slot].float().transpose(1, 2))


def _request_lens(s):
    pages = s["kv_indptr"][1:].long() - s["kv_indptr"][:-1].long()
    return torch.where(pages > 0, (pages - 1) * s["page"] + s["last"].long(), 0)


def _softmax_parts(scores):
    """(row maximum made finite, exponentials, their sums) over the last axis; a row of -inf gives zeros."""
    m = scores.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(scores - m)
    return m, e, e.sum(-1, keepdim=True)


def _answer(o, m, l, dtype):
    out = torch.where(l > 0, o / torch.where(l > 0, l, torch.ones_like(l)), torch.zeros_like(o)).to(dtype)
    return out, ((m + torch.log(l)) * LOG2E).squeeze(-1)


def _plain_decode(s, pos, live):
    """Decode over the tokens `pos` (batch, tokens) that are `live`: (out, lse, weights (batch, HQ, tokens))."""
    q, hkv = s["q"], s["k"].shape[2]
    b, hq, d = q.shape
    k, v = _rows(s, pos, live)
    sc = torch.matmul(q.float().view(b, hkv, hq // hkv, d), k.transpose(-1, -2)) * s["scale"]
    sc = sc.masked_fill(~live[:, None, None, :], -math.inf)
    m, e, l = _softmax_parts(sc)
    out, lse = _answer(torch.matmul(e, v), m, l, q.dtype)
    return out.reshape(b, hq, d), lse.reshape(b, hq), e / torch.where(l > 0, l, torch.ones_like(l))


def _plain_window_decode(s):
    c, n = s["case"], _request_lens(s)[:, None]
    w = min(c["window"], s["longest"])
    sink = torch.arange(c["sinks"], device="cuda")[None, :]
    win = n - w + torch.arange(w, device="cuda")[None, :]
    pos = torch.cat([sink.expand(n.shape[0], -1), win], 1)
    live = torch.cat([sink < n - w, win >= 0], 1)
    return _plain_decode(s, pos, live)[:2]


def _plain_window_prefill(s):
    c, q, hkv = s["case"], s["q"], s["k"].shape[-2]
    qp, kp = s["qo_indptr"].long(), s["kv_indptr"].long()
    nq, nk = (qp[1:] - qp[:-1])[:, None], (kp[1:] - kp[:-1])[:, None]
    i, j = torch.arange(s["lq"], device="cuda")[None, :], torch.arange(s["lk"], device="cuda")[None, :]
    iq = (qp[:-1, None] + i).clamp(max=q.shape[0] - 1)
    ik = torch.where(j < nk, kp[:-1, None] + j, 0)
    if c["paged"]:
        ik = s["kv_indices"][ik].long()
        k, v = s["k"][ik, 0], s["v"][ik, 0]
    else:
        k, v = s["k"][ik], s["v"][ik]
    b, hq, d = nq.shape[0], q.shape[1], q.shape[2]
    grp = hq // hkv
    qq = q[iq].float().view(b, -1, hkv, grp, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    sc = torch.matmul(qq, k.float().permute(0, 2, 3, 1)).mul_(s["scale"]).view(b, hkv, grp, s["lq"], s["lk"])
    p = (i + nk - nq)[:, :, None]
    jj = j[:, None, :]
    see = (jj <= p) & ((jj > p - c["window"]) | (jj < c["sinks"])) & (jj < nk[:, :, None])
    sc.masked_fill_(~see[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = sc.sub_(m).exp_()
    l = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(b, hkv, grp * s["lq"], s["lk"]), v.float().transpose(1, 2)).view(b, hkv, grp, s["lq"], d)
    out, lse = _answer(o, m, l, q.dtype)
    real = i < nq
    return out.permute(0, 3, 1, 2, 4).reshape(b, s["lq"], hq, d)[real], lse.permute(0, 3, 1, 2).reshape(b, s["lq"], hq)[real]


def _plain_shared_prefix(s):
    c, q, hkv = s["case"], s["q"], s["k"].shape[2]
    b, hq, d = q.shape
    grp = hq // hkv
    qq = q.float().view(b, hkv, grp, d)
    t = torch.arange(c["prefix"], device="cuda")
    page, slot = s["other"][t // s["page"]].long(), t % s["page"]
    kp, vp = s["k"][page, slot].float().transpose(0, 1), s["v"][page, slot].float().transpose(0, 1)
    sp = torch.matmul(qq.transpose(0, 1).reshape(hkv, b * grp, d), kp.transpose(1, 2)) * s["scale"]
    mp, ep, lp = _softmax_parts(sp)
    op = torch.matmul(ep, vp)
    back = lambda x: x.view(hkv, b, grp, -1).transpose(0, 1)  # noqa: E731
    mp, lp, op = back(mp), back(lp), back(op)
    n = _request_lens(s)[:, None]
    pos = torch.arange(s["longest"], device="cuda")[None, :].expand(b, -1)
    live = pos < n
    k, v = _rows(s, pos, live)
    ss = torch.matmul(qq, k.transpose(-1, -2)) * s["scale"]
    ss = ss.masked_fill(~live[:, None, None, :], -math.inf)
    ms, es, ls = _softmax_parts(ss)
    os_ = torch.matmul(es, v)
    m = torch.where(ls > 0, torch.maximum(mp, ms), mp)
    fp, fs = torch.exp(mp - m), torch.where(ls > 0, torch.exp(ms - m), torch.zeros_like(m))
    out, lse = _answer(op * fp + os_ * fs, m, lp * fp + ls * fs, q.dtype)
    return out.reshape(b, hq, d), lse.reshape(b, hq)


def _plain_weights(s):
    n = _request_lens(s)[:, None]
    pos = torch.arange(s["longest"], device="cuda")[None, :].expand(n.shape[0], -1)
    out, lse, w = _plain_decode(s, pos, pos < n)
    s["sums"] += w.sum(2)
    return out, lse, s["sums"]


def _plain_evict(s):
    c, w = s["case"], s["sums"]
    b, hkv, longest = w.shape
    n = _request_lens(s)[:, None, None]
    j = torch.arange(longest, device="cuda")
    budget = n.clamp(max=c["budget"])
    room = budget - torch.minimum(torch.full_like(n, c["sinks"]), budget)
    fixed = (j < c["sinks"]) | ((j >= n - torch.minimum(torch.full_like(n, c["recent"]), room)) & (j < n))
    rank = torch.where(j < n, torch.where(fixed, math.inf, w.double()), -math.inf)  # sums are finite here
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    keep = torch.zeros(b, hkv, longest, dtype=torch.bool, device="cuda")
    keep.scatter_(-1, order, torch.arange(longest, device="cuda").expand_as(order) < budget)
    kept = torch.sort(torch.where(keep, j, longest), dim=-1).values[..., :min(c["budget"], longest)]
    if kept.shape[-1] < c["budget"]:
        kept = torch.nn.functional.pad(kept, (0, c["budget"] - kept.shape[-1]), value=longest)
    live = kept < longest
    sums = torch.zeros_like(w)
    head = min(c["budget"], longest)
    sums[..., :head] = torch.where(live, w.gather(-1, torch.where(live, kept, 0)), 0.0)[..., :head]
    bb, hh, ii = torch.nonzero(live, as_tuple=True)
    src, ps = kept[bb, hh, ii], s["page"]
    sp = s["kv_indices"][s["kv_indptr"].long()[bb] + src // ps].long()
    dp = s["other"][s["dst_indptr"].long()[bb] + ii // ps].long()
    s["k"][dp, ii % ps, hh] = s["k"][sp, src % ps, hh]
    s["v"][dp, ii % ps, hh] = s["v"][sp, src % ps, hh]
    new = budget.view(-1)
    last = torch.where(new > 0, (new - 1) % ps + 1, 0)
    return s["k"], s["v"], torch.where(live, kept, -1).int(), sums, last.int()


PLAIN = {"window_decode": _plain_window_decode, "window_prefill": _plain_window_prefill, "shared_prefix": _plain_shared_prefix,
         "weights": _plain_weights, "evict": _plain_evict}


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    from cleave_b200 import ops

    c = s["case"]
    if c["op"] == "window_prefill":
        if c["paged"]:
            return ops.gqa_paged_prefill_window(s["q"], s["k"], s["v"], s["qo_indptr"], s["kv_indptr"], s["kv_indices"], s["scale"],
                                                c["window"], c["sinks"])
        return ops.gqa_ragged_prefill_window(s["q"], s["k"], s["v"], s["qo_indptr"], s["kv_indptr"], s["scale"], c["window"], c["sinks"])
    last = s["last"] if s["page"] != 1 else None
    table = (s["kv_indptr"], s["kv_indices"], last)
    if c["op"] == "window_decode":
        return ops.gqa_paged_decode_window(s["q"], s["k"], s["v"], *table, s["scale"], c["window"], c["sinks"])
    if c["op"] == "shared_prefix":
        return ops.gqa_paged_decode_shared_prefix(s["q"], s["k"], s["v"], s["other"], c["prefix"], *table, s["scale"])
    if c["op"] == "weights":
        out, lse = ops.gqa_paged_decode_weights(s["q"], s["k"], s["v"], *table, s["scale"], s["sums"])
        return out, lse, s["sums"]
    kept, sums, new_last = ops.kv_cache_evict(s["k"], s["v"], s["sums"], *table, s["dst_indptr"], s["other"],
                                              budget=c["budget"], sinks=c["sinks"], recent=c["recent"])
    return s["k"], s["v"], kept, sums, new_last


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ 64 bits
def _attend64(q, k, v, see, scale):
    """One kv head: q (rows, D), k / v (tokens, D), see (rows, tokens) or None. (out, base-2 lse, weights)"""
    x = (q.double() @ k.double().T) * scale
    if see is not None:
        x = x.masked_fill(~see, -math.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[:, None])
    return p @ v.double(), lse / math.log(2.0), p


def exact(case, seed):
    s = prepare(case, seed)
    op, hkv, scale = case["op"], case["hkv"], s["scale"]
    f64 = dict(dtype=torch.float64, device="cuda")
    if op == "window_prefill":
        q, d = s["q"], case["d"]
        grp = case["hq"] // hkv
        out, lse = torch.zeros(q.shape, **f64), torch.full(q.shape[:2], -math.inf, **f64)
        qp, kp = s["qo_indptr"].tolist(), s["kv_indptr"].tolist()
        for r in range(case["batch"]):
            a, b, e, f = qp[r], qp[r + 1], kp[r], kp[r + 1]
            kk, vv = (s[x][s["kv_indices"][e:f].long(), 0] if case["paged"] else s[x][e:f] for x in ("k", "v"))
            at = torch.arange(f - e - (b - a), f - e, device="cuda")[:, None]
            key = torch.arange(f - e, device="cuda")[None]
            see = (key <= at) & ((at - key < case["window"]) | (key < case["sinks"]))
            for h in range(case["hq"]):
                out[a:b, h], lse[a:b, h], _ = _attend64(q[a:b, h], kk[:, h // grp], vv[:, h // grp], see, scale)
        return out, lse
    page, lens = case["page"], _lens(case)
    ptr = s["kv_indptr"].tolist()
    if op == "evict":
        k, v, w = s["k"].double(), s["v"].double(), s["sums"]
        kept = torch.full((case["batch"], hkv, case["budget"]), -1, dtype=torch.int32)
        sums, last = torch.zeros(w.shape, dtype=torch.float64), []
        src, dst, dptr = s["kv_indices"].tolist(), s["other"].tolist(), s["dst_indptr"].tolist()
        frm, to = [], []
        wl = w.cpu().double().numpy()
        for r, n in enumerate(lens):
            m = min(n, case["budget"])
            first = min(case["sinks"], m)
            tail = min(case["recent"], m - first)
            last.append((m - 1) % page + 1 if m else 0)
            for h in range(hkv):
                if m == n:
                    ids = list(range(n))
                else:
                    row = wl[r, h]
                    middle = sorted(range(first, n - tail), key=lambda t: (-row[t], t))[:m - first - tail]
                    ids = list(range(first)) + sorted(middle) + list(range(n - tail, n))
                kept[r, h, :m] = torch.tensor(ids, dtype=torch.int32)
                sums[r, h, :m] = torch.from_numpy(wl[r, h][ids])
                frm += [((src[ptr[r] + t // page]) * page + t % page) * hkv + h for t in ids]
                to += [((dst[dptr[r] + i // page]) * page + i % page) * hkv + h for i in range(m)]
        frm, to = torch.tensor(frm, device="cuda"), torch.tensor(to, device="cuda")
        for t in (k, v):
            flat = t.view(-1, case["d"])
            flat[to] = flat[frm]
        return k, v, kept, sums, torch.tensor(last, dtype=torch.int32)
    q = s["q"]
    grp = case["hq"] // hkv
    out, lse = torch.zeros(q.shape, **f64), torch.full(q.shape[:2], -math.inf, **f64)
    pre = s["other"].long() if op == "shared_prefix" else None
    for r, n in enumerate(lens):
        idx = s["kv_indices"][ptr[r]:ptr[r + 1]].long()
        kk, vv = (s[x][idx].flatten(0, 1)[:n] for x in ("k", "v"))
        see = None
        if op == "shared_prefix":
            kk, vv = (torch.cat([s[x][pre].flatten(0, 1)[:case["prefix"]], t]) for x, t in (("k", kk), ("v", vv)))
        elif op == "window_decode":
            key = torch.arange(n, device="cuda")
            see = ((n - 1 - key < case["window"]) | (key < case["sinks"]))[None]
        for h in range(hkv):
            rows = slice(h * grp, (h + 1) * grp)
            out[r, rows], lse[r, rows], p = _attend64(q[r, rows], kk[:, h], vv[:, h], see, scale)
            if op == "weights":
                if r == 0 and h == 0:
                    total = s["sums"].double()
                total[r, h, :n] += p.sum(0)
    return (out, lse, total) if op == "weights" else (out, lse)
