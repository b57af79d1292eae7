"""Refusals of the serving operators that come before any device call, so that they run without a GPU."""

import ctypes as C

import pytest
import torch

from cleave_b200 import _lib, ops

OK, BAD_ARG, UNSUPPORTED, ALIGNMENT, WORKSPACE, CUDA = 0, 1, 2, 3, 4, 5


def _decode(**kw):
    a = _lib.AttnDecodeArgs()
    a.q = a.k_cache = a.v_cache = a.kv_indptr = a.kv_indices = a.kv_last_page_len = a.out = a.lse = 4096
    a.batch, a.num_qo_heads, a.num_kv_heads, a.head_dim, a.page_size, a.num_pages, a.num_kv_indices = 2, 8, 2, 128, 16, 10, 8
    a.q_rows, a.dtype, a.sm_scale = 1, _lib.BF16, 0.1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _window(window=10, sinks=2, **kw):
    return _lib.lib().cb200_attn_decode_window(C.byref(_decode(**kw)), window, sinks, None)


def _weights(sums=4096, max_len=100, scratch=4096, nbytes=1 << 30, **kw):
    return _lib.lib().cb200_attn_decode_weights(C.byref(_decode(**kw)), sums, max_len, scratch, nbytes, None)


def _prefix(indices=4096, n=4, length=50, scratch=4096, nbytes=1 << 30, **kw):
    return _lib.lib().cb200_attn_decode_shared_prefix(C.byref(_decode(**kw)), indices, n, length, scratch, nbytes, None)


@pytest.mark.parametrize("call", [_window, _weights, _prefix])
def test_decode_variants_refuse_bad_arguments(call):
    assert call(kv_indptr=None) == BAD_ARG  # paged caches only
    assert call(batch=0) == BAD_ARG and call(num_kv_heads=0) == BAD_ARG and call(num_qo_heads=7) == BAD_ARG
    assert call(page_size=0) == BAD_ARG and call(num_pages=0) == BAD_ARG and call(num_kv_indices=-1) == BAD_ARG
    assert call(head_dim=96) == UNSUPPORTED and call(dtype=7) == UNSUPPORTED
    assert call(q_rows=2) == UNSUPPORTED
    assert call(page_size=1 << 16, num_pages=1 << 15) == UNSUPPORTED                     # places in the pool in 32 bits
    assert call(batch=1, num_qo_heads=1, num_kv_heads=1, page_size=64, num_kv_indices=(1 << 24) + 1) == UNSUPPORTED  # and in a request


def test_decode_variants_refuse_their_own_arguments():
    assert _window(window=0) == BAD_ARG and _window(window=-1) == BAD_ARG and _window(sinks=-1) == BAD_ARG
    assert _weights(sums=None) == BAD_ARG and _weights(max_len=0) == BAD_ARG and _weights(lse=None) == BAD_ARG
    assert _prefix(length=-1) == BAD_ARG and _prefix(n=-1) == BAD_ARG
    L = _lib.lib()
    for f in (L.cb200_attn_decode_weights_scratch_bytes, L.cb200_attn_decode_shared_prefix_scratch_bytes):
        assert f(C.byref(_decode()), 0) == 0 and f(C.byref(_decode(batch=0)), 10) == 0
    assert L.cb200_attn_decode_weights_scratch_bytes(C.byref(_decode()), 9) == 2 * 8 * 16 * 4  # rows of whole 32-byte runs
    assert L.cb200_attn_decode_window(None, 1, 0, None) == BAD_ARG
    assert L.cb200_attn_decode_weights(None, 4096, 1, 4096, 4096, None) == BAD_ARG
    assert L.cb200_attn_decode_shared_prefix(None, 4096, 1, 1, 4096, 4096, None) == BAD_ARG


def test_scores_are_kept_for_no_more_tokens_than_the_page_table_holds():
    f = _lib.lib().cb200_attn_decode_weights_scratch_bytes
    bytes_of = lambda max_len, **kw: f(C.byref(_decode(**kw)), max_len)  # noqa: E731
    assert bytes_of(131072) == bytes_of(128) == 2 * 8 * 128 * 4  # 8 pages of 16 tokens
    assert bytes_of(127) == 2 * 8 * 128 * 4 and bytes_of(120) == 2 * 8 * 120 * 4
    assert bytes_of(131072, num_kv_indices=3, page_size=5) == 2 * 8 * 16 * 4
    assert bytes_of(131072, num_kv_indices=0) == 0
    assert bytes_of(2 ** 31 - 1, num_kv_indices=2 ** 31 - 1) == 2 * 8 * 2 ** 31 * 4
    assert bytes_of(100, num_kv_indices=-1) == 0


def test_window_prefill_refuses_bad_arguments():
    def call(window=10, sinks=2, fill=0, **kw):
        a = _lib.AttnPrefillRaggedArgs()
        a.q = a.k = a.v = a.qo_indptr = a.kv_indptr = a.out = a.lse = a.workspace = 4096
        a.workspace_bytes = 1 << 20
        a.batch, a.total_q, a.total_kv, a.num_qo_heads, a.num_kv_heads, a.head_dim, a.dtype, a.causal = 2, 50, 60, 8, 2, 64, _lib.F16, 1
        for k, v in kw.items():
            setattr(a, k, v)
        return _lib.lib().cb200_attn_prefill_ragged_window(C.byref(a), window, sinks, fill, None)

    assert _lib.lib().cb200_attn_prefill_ragged_window(None, 1, 0, 0, None) == BAD_ARG
    for kw in (dict(window=0), dict(window=-5), dict(sinks=-1), dict(fill=4), dict(fill=-1), dict(batch=0), dict(total_q=0), dict(total_kv=0),
               dict(num_kv_heads=3), dict(num_qo_heads=0), dict(q=None), dict(v=None), dict(out=None), dict(qo_indptr=None)):
        assert call(**kw) == BAD_ARG, kw
    assert call(head_dim=96) == UNSUPPORTED and call(dtype=9) == UNSUPPORTED
    assert call(total_q=(1 << 30) + 1, num_qo_heads=2) == UNSUPPORTED
    assert call(kv_indices=4096, num_kv_indices=(1 << 30) + 1) == UNSUPPORTED
    assert call(k=4100) == ALIGNMENT and call(out=4104) == ALIGNMENT
    assert call(workspace=None) == WORKSPACE and call(workspace_bytes=16) == WORKSPACE


def test_eviction_refuses_bad_arguments():
    def call(**kw):
        a = _lib.KvEvictArgs()
        for name, kind in a._fields_:
            if kind is C.c_void_p:
                setattr(a, name, 4096)
        a.batch, a.num_kv_heads, a.head_dim, a.page_size, a.num_pages, a.num_kv_indices, a.num_dst_indices = 2, 2, 64, 16, 20, 8, 4
        a.max_len, a.budget, a.sinks, a.recent = 100, 32, 4, 8
        for k, v in kw.items():
            setattr(a, k, v)
        return _lib.lib().cb200_kv_evict(C.byref(a), None)

    assert _lib.lib().cb200_kv_evict(None, None) == BAD_ARG
    for name in ("batch", "num_kv_heads", "head_dim", "page_size", "num_pages", "max_len", "budget"):
        assert call(**{name: 0}) == BAD_ARG and call(**{name: -1}) == BAD_ARG, name
    for kw in (dict(sinks=-1), dict(recent=-1), dict(sinks=20, recent=13), dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), dict(num_kv_indices=-1),
               dict(num_dst_indices=-1), dict(kv_last_page_len=None), dict(kv_indices=None), dict(dst_indices=None)):
        assert call(**kw) == BAD_ARG, kw
    for name in ("k_cache", "v_cache", "weight_sums", "kv_indptr", "dst_indptr", "kept", "kept_sums", "dst_last_page_len"):
        assert call(**{name: None}) == BAD_ARG, name
    assert call(head_dim=60) == UNSUPPORTED and call(batch=65536) == UNSUPPORTED
    for name in ("budget", "max_len", "num_kv_indices"):
        assert call(**{name: (1 << 30) + 1}) == UNSUPPORTED, name
    assert call(k_cache=4104) == ALIGNMENT


def test_operators_refuse_host_tensors():
    h, i = lambda *s: torch.zeros(*s, dtype=torch.float16), lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    q, c = h(2, 8, 64), h(4, 16, 2, 64)
    tables = i(3), i(4), i(2)
    for fn, args in ((ops.gqa_paged_decode_window, (q, c, c, *tables, 0.1, 8)),
                     (ops.gqa_paged_decode_weights, (q, c, c, *tables, 0.1, torch.zeros(2, 2, 9))),
                     (ops.gqa_paged_decode_shared_prefix, (q, c, c, i(1), 10, *tables, 0.1)),
                     (ops.gqa_ragged_prefill_window, (q, h(2, 2, 64), h(2, 2, 64), i(3), i(3), 0.1, 8)),
                     (ops.gqa_paged_prefill_window, (q, h(2, 1, 2, 64), h(2, 1, 2, 64), i(3), i(3), i(2), 0.1, 8))):
        with pytest.raises(ValueError, match="CUDA"):
            fn(*args)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_cache_evict(c, c, torch.zeros(2, 2, 9), *tables, i(3), i(4), budget=8)


@pytest.mark.parametrize("window,sinks", [(0, 0), (-3, 1), (4, -1)])
def test_windows_that_hold_nothing_are_refused(window, sinks):
    for fn, n in ((ops.gqa_paged_decode_window, 7), (ops.gqa_ragged_prefill_window, 6), (ops.gqa_paged_prefill_window, 7)):
        with pytest.raises(ValueError, match="window"):
            fn(*[None] * n, window, sinks)


@pytest.mark.parametrize("budget", [0, -1, 2 ** 31, 2 ** 32 + 5, 2 ** 40])
def test_budgets_that_hold_nothing_or_pass_32_bits_are_refused(budget):
    """2 ** 32 + 5 would be cut to 5."""
    with pytest.raises(ValueError, match="budget"):
        ops.kv_cache_evict(*[None] * 8, budget=budget)
