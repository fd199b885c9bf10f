"""One output buffer for every step of a loop: the step's rows are written, the rows behind them are as they were."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_a_larger_output_keeps_its_other_rows(dtype):
    from titan_engine_b200 import PagedKVCache
    H, HKV, D = 8, 2, 128
    c = PagedKVCache(1, H, HKV, D, 64, 4, 32, dtype=dtype, io_dtype="bf16", max_step_tokens=256)
    g = torch.Generator(device=c.device)
    g.manual_seed(1)
    rows = lambda n, h: torch.randn(n, h, D, device=c.device, generator=g).to(torch.bfloat16)  # noqa: E731
    a, b = c.seq_alloc(), c.seq_alloc()
    for new in ([40, 3], [1, 1], [3, 2], [1, 70]):
        n = sum(new)
        k, v, q = rows(n, HKV), rows(n, HKV), rows(n, H)
        c.step_begin([a, b], new)
        buf = torch.full((128, H, D), 3.0, dtype=torch.bfloat16, device=c.device)
        got = c.append_decode_multi(0, k, v, q, buf)
        assert got is buf
        want = c.decode_multi(0, q.view(n, HKV, -1))        # queries split by kv head: the output's shape is its own
        assert want.shape == (n, H, D) and torch.equal(buf[:n], want) and (buf[n:] == 3.0).all()
        buf.fill_(3.0)
        c.decode_multi(0, q, buf)
        assert torch.equal(buf[:n], want) and (buf[n:] == 3.0).all()
        if new == [1, 1]:
            buf.fill_(3.0)
            c.append_decode(0, k, v, q, buf)
            assert torch.equal(buf[:n], c.decode(0, q)) and (buf[n:] == 3.0).all()
            one = c.rope_append_decode(0, k, v, q, 10000.0)
            buf.fill_(3.0)
            c.rope_append_decode(0, k, v, q, 10000.0, 1.0, buf)
            assert torch.equal(buf[:n], one) and (buf[n:] == 3.0).all()
    c.device_status()
