"""tk_kv_read without a GPU: which ranges are refused before anything would run (the calls that pass end with "no device")."""
import ctypes as C

import numpy as np
import pytest

from titan_engine_b200 import PagedKVCache
from titan_engine_b200 import _lib as L


def _cache(dtype, **kw):
    args = dict(num_layers=2, num_heads=4, num_kv_heads=2, head_dim=128, num_pages=16, max_seqs=4, max_pages_per_seq=8, max_step_tokens=128,
                dtype=dtype, host_only=True)
    args.update(kw)
    return PagedKVCache(**args)


def _read(c, seq, start, count, layer=0):
    p = lambda x: np.array([x], np.int32).ctypes.data_as(C.POINTER(C.c_int32))  # noqa: E731
    return c._lib.tk_kv_read(c._h, layer, 1, p(seq), p(start), p(count), None, None, c.cfg.io_dtype, None)


def test_fp8_tokens_of_a_page_that_the_step_completes_are_refused_before_the_append():
    """Until the layer's append they are in the 16-bit open page, afterwards in the sealed one; nothing tells which a replayed
    append has left, so the range is refused."""
    c = _cache("fp8")
    s = c.seq_alloc()
    c.step_begin([s], [20])                                 # completes page 0, opens page 1
    assert _read(c, s, 0, 1) == L.TK_UNSUPPORTED
    assert _read(c, s, 10, 8) == L.TK_UNSUPPORTED           # both pages
    assert _read(c, s, 16, 4) == L.TK_CUDA_ERROR            # the open page: the next check answers (no device)
    c.step_begin([s], [16])                                 # completes page 1, opens page 2
    for layer in range(2):
        assert _read(c, s, 0, 16, layer) == L.TK_CUDA_ERROR
        assert _read(c, s, 16, 4, layer) == L.TK_UNSUPPORTED
        assert _read(c, s, 32, 4, layer) == L.TK_CUDA_ERROR
    child = c.fork(s)                                       # shares the page
    assert _read(c, child, 16, 4) == L.TK_UNSUPPORTED
    c.step_begin([s], [1])                                  # completes nothing
    assert _read(c, s, 0, 37) == L.TK_CUDA_ERROR


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_pools_without_an_open_page_do_not_refuse_them(dtype):
    c = _cache(dtype)
    s = c.seq_alloc()
    c.step_begin([s], [20])
    c.step_begin([s], [16])
    assert _read(c, s, 16, 4) == L.TK_CUDA_ERROR


def test_a_loaded_state_has_no_step_to_wait_for():
    c = _cache("fp8")
    s = c.seq_alloc()
    c.step_begin([s], [20])
    c.state_load(c.state_save())
    assert _read(c, s, 0, 16) == L.TK_CUDA_ERROR


def test_a_token_in_a_cold_page_is_refused():
    c = _cache("bf16", hot_window=32, cold_pages=8)
    s = c.seq_alloc()
    c.step_begin([s], [100])
    c.step_begin([s], [1])                                  # the first pages leave for the host's pool
    cold = int((c.page_table(s) < 0).sum())
    assert 0 < cold < 6
    assert _read(c, s, 0, 1) == L.TK_UNSUPPORTED
    assert _read(c, s, 16 * cold - 1, 2) == L.TK_UNSUPPORTED
    assert _read(c, s, 16 * cold, 101 - 16 * cold) == L.TK_CUDA_ERROR       # hot pages: the next check answers (no device)
