"""Output tensors of PagedKVCache's attention calls, on a handle without a device (the library is not reached with a bad one, and answers
"no device" for a good one)."""
import pytest
import torch

from titan_engine_b200 import KvError, PagedKVCache
from titan_engine_b200 import _lib as L

H, HKV, D, SEQS, TOKENS = 8, 2, 64, 3, 3


@pytest.fixture(params=["bf16", "int8"])
def cache(request):
    c = PagedKVCache(1, H, HKV, D, 16, 4, 8, dtype=request.param, io_dtype="bf16", max_step_tokens=64, host_only=True)
    c.device = torch.device("cpu")
    c._stream = lambda: None
    c.step_begin([c.seq_alloc() for _ in range(SEQS)], [1] * SEQS)
    return c


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def _calls(c):
    k, v, q = _t(TOKENS, HKV, D), _t(TOKENS, HKV, D), _t(TOKENS, H, D)
    return {
        "append_decode": lambda out: c.append_decode(0, k, v, q, out),
        "rope_append_decode": lambda out: c.rope_append_decode(0, k, v, q, 10000.0, 1.0, out),
        "decode_multi": lambda out: c.decode_multi(0, q, out),
        "append_decode_multi": lambda out: c.append_decode_multi(0, k, v, q, out),
    }


@pytest.mark.parametrize("name", ["append_decode", "rope_append_decode", "decode_multi", "append_decode_multi"])
def test_an_output_larger_than_the_step_is_taken_and_a_bad_one_is_not(cache, name):
    call = _calls(cache)[name]
    for good in (_t(TOKENS, H, D), _t(TOKENS + 5, H, D), _t(TOKENS, H * D), _t((TOKENS + 1) * H * D)):
        with pytest.raises(KvError) as e:
            call(good)
        assert e.value.status == L.TK_CUDA_ERROR
    for bad in (_t(TOKENS - 1, H, D), _t(TOKENS, H, D, dtype=torch.float32), _t(TOKENS, H, 2 * D)[..., ::2], _t(D, H, TOKENS).permute(2, 1, 0)):
        with pytest.raises(KvError) as e:
            call(bad)
        assert e.value.status == L.TK_INVALID_ARG


@pytest.mark.parametrize("shape", [(TOKENS, H, D), (TOKENS, HKV, H // HKV * D), (TOKENS, 1, H * D), (1, TOKENS, H * D), (TOKENS, H * D),
                                   (TOKENS, HKV, H // HKV, D), (TOKENS * H * D,)])
def test_a_new_output_has_the_shape_that_is_documented(cache, shape):
    """[rows, H, Dv], however the queries are split."""
    cache._check = lambda status: None                      # (the calls end with "no device")
    k, v, q = _t(TOKENS, HKV, D), _t(TOKENS, HKV, D), _t(*shape)
    for out in (cache.decode(0, q), cache.append_decode(0, k, v, q), cache.rope_append_decode(0, k, v, q, 10000.0), cache.decode_multi(0, q),
                cache.append_decode_multi(0, k, v, q)):
        assert out.shape == (TOKENS, H, D) and out.dtype == q.dtype and out.is_contiguous()
