"""Growth of the split-KV workspace of multi-token steps when the device has little room left."""
import re

import pytest
import torch

pytestmark = pytest.mark.gpu

H, HKV, D = 8, 2, 128


class Steps:
    def __init__(self, dtype):
        from titan_engine_b200 import PagedKVCache
        self.c = PagedKVCache(1, H, HKV, D, 600, 4, 300, dtype=dtype, io_dtype="bf16", max_step_tokens=4096)
        self.g = torch.Generator(device=self.c.device)
        self.g.manual_seed(3)
        self.s = self.c.seq_alloc()
        for _ in range(2):
            self.c.step_begin([self.s], [2000])
            self.c.append(0, self.rows(2000, HKV), self.rows(2000, HKV))

    def rows(self, n, h):
        return torch.randn(n, h, D, device=self.c.device, generator=self.g).to(torch.bfloat16)

    def begin(self, n):
        self.c.truncate(self.s, 4000)
        self.c.step_begin([self.s], [n])
        self.k, self.v, self.q = self.rows(n, HKV), self.rows(n, HKV), self.rows(n, H)
        self.c.append(0, self.k, self.v)

    def limit(self, nbytes):
        assert self.c._lib.tk_kv_selftest_workspace_limit(self.c._h, nbytes) == 0

    def need(self):
        """Bytes that the step's workspace takes: what the refusal of an allocation says."""
        from titan_engine_b200 import KvError
        self.limit(1)
        with pytest.raises(KvError, match="workspace") as e:
            self.c.decode_multi(0, self.q)
        self.limit(0)
        return int(re.search(r"workspace of (\d+) bytes", str(e.value)).group(1))


# new tokens of a first, a slightly larger and a large step: drafted tokens on a 16-bit pool, split prompt chunks on an INT8 pool
SIZES = pytest.mark.parametrize("dtype,small,more,large", [("bf16", 20, 22, 30), ("int8", 40, 44, 80)])


@SIZES
def test_growth_where_only_the_new_buffer_fits(dtype, small, more, large):
    """Without a captured graph the outgrown buffer goes first, as much memory as the step needs is enough."""
    t = Steps(dtype)
    t.begin(small)
    first = t.need()
    t.limit(first)
    a = t.c.decode_multi(0, t.q).clone()
    t.begin(large)
    second = t.need()
    assert second > first
    t.limit(second)
    b = t.c.decode_multi(0, t.q).clone()
    t.limit(0)
    assert torch.equal(t.c.decode_multi(0, t.q), b) and torch.isfinite(a).all() and torch.isfinite(b).all()
    t.c.device_status()


@SIZES
def test_growth_next_to_a_captured_buffer_takes_what_fits(dtype, small, more, large):
    """The graph keeps the outgrown buffer; where twice its size does not fit beside it, what the step needs does."""
    t = Steps(dtype)
    t.begin(small)
    first, q, k, v = t.need(), t.q, t.k, t.v
    want = t.c.decode_multi(0, q).clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = t.c.decode_multi(0, q)
    t.begin(more)
    second = t.need()
    assert first < second < 2 * first
    t.limit(first + second)
    out = t.c.decode_multi(0, t.q).clone()
    t.limit(0)
    assert torch.equal(t.c.decode_multi(0, t.q), out) and torch.isfinite(out).all()
    t.c.truncate(t.s, 4000)                                 # the captured step again
    t.c.step_begin([t.s], [small])
    t.c.append(0, k, v)
    for _ in range(2):
        got.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    t.c.device_status()
