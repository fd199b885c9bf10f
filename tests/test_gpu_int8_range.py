"""INT8 pools: bf16 queries of very different size in one tile of the chunk kernel."""
import numpy as np
import pytest
import torch

from int8_plain import attention, check, stands_for
from test_gpu_int8 import Pair

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("small", [-24, -10, -1, 0, 2, 6])
@pytest.mark.parametrize("D", [64, 128])
def test_small_queries_beside_large_ones(small, D):
    """One head of four has queries of nearly 2^15, the others of about 2^small, and keys of about 2^-small give those scores of
    about 1: the large ones must not cost the small ones their bits (those of 2^0 and more are exact under the tile's power of two, below it
    every row has one of its own)."""
    p = Pair(8, 2, D, "bf16")
    s = p.alloc()
    n, held = 90, 150
    for m in (held, n):
        p.c.step_begin([s], [m])
        k, v = p.rows(m, 2, 2.0 ** -small), p.rows(m, 2)
        p.k[s] = np.concatenate([p.k[s], stands_for(k.float().cpu().numpy())])
        p.v[s] = np.concatenate([p.v[s], stands_for(v.float().cpu().numpy())])
        if m == held:
            p.c.append(0, k, v)
    q = p.rows(n, 8, 2.0 ** small)
    q[:, 1::4] = (q[:, 1::4].float() * 2.0 ** (12 - small)).clamp(-32640.0, 32640.0).to(q.dtype)
    q[5, 1, 3] = 32640.0                                    # the largest bf16 below 2^15
    got = p.c.append_decode_multi(0, k, v, q).float().cpu().numpy()
    items, _, n_decode = p.c.step_prefill_plan()
    assert len(items) and n_decode == 0                     # the chunk kernel takes them all
    want, bound = attention(q.float().cpu().numpy(), p.k[s], p.v[s], np.arange(held, held + n) + 1, "bf16")
    ordinary = np.arange(8) % 4 != 1
    check(got[:, ordinary], want[:, ordinary], bound[:, ordinary], "small queries")
    assert np.isfinite(got).all()
    large = bound[:, ~ordinary] < np.abs(want[:, ~ordinary])        # (where scores of 2^20 leave the bound a meaning)
    assert (np.abs(got - want)[:, ~ordinary][large] <= bound[:, ~ordinary][large]).all()
