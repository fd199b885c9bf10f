"""Reads of an FP8 pool in the middle of a step: tokens of a page that the step completes are in the open page before the layer's
append and in the sealed page after it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_fp8_read_between_step_begin_and_the_appends():
    from titan_engine_b200 import KvError, PagedKVCache
    from titan_engine_b200 import _lib as L
    c = PagedKVCache(2, 4, 2, 128, 16, 4, 8, dtype="fp8", io_dtype="bf16", max_step_tokens=64)
    for layer in range(2):                                  # whatever the pages' last owners left
        pool, scales, _ = c.layer_views(layer)
        pool.fill_(0x7F)
        scales.fill_(float("nan"))
    g = torch.Generator(device=c.device)
    g.manual_seed(5)
    rows = lambda n: [torch.randn(n, 2, 128, device=c.device, generator=g).to(torch.bfloat16) for _ in range(2)]  # noqa: E731
    s = c.seq_alloc()
    k0, v0 = rows(20)
    c.step_begin([s], [20])
    for layer in range(2):
        c.append(layer, k0, v0)
    full = [[x.clone() for x in c.read(layer, [s])] for layer in range(2)]
    assert torch.equal(full[0][0][16:], k0[16:])            # the open page: the rows' own bits
    k1, v1 = rows(16)
    c.step_begin([s], [16])                                 # completes page 1, tokens 16 .. 31
    child = c.fork(s)
    for layer in range(2):
        for seq in (s, child):
            k, v = c.read(layer, [seq], [0], [16])
            assert torch.equal(k, full[layer][0][:16]) and torch.equal(v, full[layer][1][:16])
            with pytest.raises(KvError) as e:
                c.read(layer, [seq], [10], [8])
            assert e.value.status == L.TK_UNSUPPORTED
    c.append(0, k1, v1)
    for got, old, new in zip(c.read(0, [s], out_dtype=torch.float32), (k0, v0), (k1, v1)):
        want = torch.cat([old, new]).float()
        scale = want[16:32].abs().amax(dim=(0, 2)).clamp_min(1e-30) / 448      # a page's, per kv head
        # a code is off by half a step: 2^-4 of the value, or 2^-10 scales among e4m3's subnormals; the scale and the product by 2^-24,
        # the quotient that was rounded too
        off = want[16:32].abs() * (2.0 ** -4 + 2.0 ** -20) + scale[None, :, None] * 2.0 ** -10
        assert ((got[16:32] - want[16:32]).abs() <= off).all()
        assert torch.equal(got[32:], want[32:])             # the open page again
    with pytest.raises(KvError):
        c.read(1, [s], [16], [4])                           # layer 1 has not appended yet
    c.append(1, k1, v1)
    assert all(torch.equal(a, b) for a, b in zip(c.read(1, [s]), c.read(0, [s])))
    c.device_status()
