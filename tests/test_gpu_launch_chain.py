"""Attention calls that follow each other with nothing between: of one layer again, and fed with each other's output.  Launches overlap
where they may; the results are those of launches that never do."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("ctx", [[20], [40] * 12, [3000, 17, 900, 1]])
def test_outputs_as_queries_and_layers_again(dtype, ctx):
    from titan_engine_b200 import PagedKVCache
    L, H, HKV, D, n = 3, 8, 2, 128, len(ctx)
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    rows = lambda m, h: torch.randn(m, h, D, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
    old = [(rows(sum(ctx), HKV), rows(sum(ctx), HKV)) for _ in range(L)]
    new = [(rows(n, HKV), rows(n, HKV)) for _ in range(L)]
    q = rows(n, H)
    runs = []
    for overlap in (False, True):
        c = PagedKVCache(L, H, HKV, D, 400, 16, 200, dtype=dtype, io_dtype="bf16", max_step_tokens=4096, launch_overlap=overlap)
        seqs = [c.seq_alloc() for _ in ctx]
        c.step_begin(seqs, ctx)
        for layer in range(L):
            c.append(layer, *old[layer])
        for _ in range(8):
            c.step_begin(seqs, [1] * n)
            outs = []
            x = q
            for layer in (0, 1, 2, 0, 1, 2):                # each fed with the output of the one before
                x = c.append_decode(layer, *new[layer], x)
                outs.append(x)
            x = c.decode(0, q)
            y = c.decode(1, q)
            outs += [x, y, c.decode(2, x), c.decode(0, y)]  # ... and of the one before that
            k = x[:, :HKV].contiguous()
            for layer in range(L):                          # new rows taken from an output
                x = c.append_decode(layer, k, new[layer][1], x)
                k = x.view(n * H, D)[:n * HKV].view(n, HKV, D)
                outs.append(x)
            for s, m in zip(seqs, ctx):
                if dtype != "fp8":
                    c.truncate(s, m)
        runs.append([x.clone() for x in outs])
        c.device_status()
        c.close()
    for a, b in zip(*runs):
        assert torch.equal(a, b) and torch.isfinite(a).all()
