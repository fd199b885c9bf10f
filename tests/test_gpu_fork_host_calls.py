"""A fork while calls of the asynchronous host-buffer path are still held back: the child's copy of the open page has their rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "int8", "fp8"])
def test_fork_sees_the_rows_of_held_back_calls(dtype):
    from titan_engine_b200 import PagedKVCache
    layers = 3                                              # launched in groups of 1, 1, 2: the third call is held back
    c = PagedKVCache(layers, 4, 2, 128, 16, 4, 8, dtype=dtype, io_dtype="bf16", max_step_tokens=64)
    g = torch.Generator()
    g.manual_seed(2)
    row = lambda n, h: torch.randn(n, h, 128, generator=g).to(torch.bfloat16).pin_memory()  # noqa: E731
    s = c.seq_alloc()
    c.step_begin([s], [20])
    for layer in range(layers):
        c.append(layer, row(20, 2).to(c.device), row(20, 2).to(c.device))
    c.step_begin([s], [1])
    io = [(row(1, 2), row(1, 2), row(1, 4), torch.empty(1, 4, 128, dtype=torch.bfloat16).pin_memory()) for _ in range(layers)]
    for layer in range(layers):
        c.append_decode_host_async(layer, *io[layer])
    child = c.fork(s)
    c.host_wait()
    for layer in range(layers):
        rows = c.read(layer, [child], [20], [1])
        for mine, parent, given in zip(rows, c.read(layer, [s], [20], [1]), io[layer]):
            assert torch.equal(mine, parent)
            if dtype != "int8":                             # an open row: the given bits
                assert torch.equal(mine.cpu(), given)
    c.device_status()
