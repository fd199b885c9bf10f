"""INT8 pools: merges of more parts than shared memory holds weights for, the exchange of partial rows, appends on a capped step."""
import ctypes as C

import numpy as np
import pytest
import torch

from test_gpu_int8 import Pair

pytestmark = pytest.mark.gpu


def test_chunk_of_more_parts_than_the_merge_has_room_for():
    """256 rows in more than 110 parts at D = 64: the parts' weights do not fit shared memory."""
    p = Pair(16, 1, 64, "bf16", pages=2600, seqs=2, mpps=2600)
    a = p.alloc()
    p.grow([a], [40000])
    k, v = p.begin([a], [16])
    q = p.rows(16, 16)
    got = p.c.append_decode_multi(0, k, v, q)
    items, ct, n_decode = p.c.step_prefill_plan()
    assert n_decode == 0 and len(items) == -(-40016 // ct[0]) > 110
    p.check_chunk(got, [a], [16], q)
    p.check_chunk(p.c.decode_multi_f32(0, q), [a], [16], q, out="fp32")


@pytest.mark.parametrize("H,Hkv,D", [(8, 1, 64), (8, 1, 128)])
def test_decode_of_more_parts_than_the_merge_has_room_for(H, Hkv, D):
    """8 rows in more than 375 parts of one page."""
    p = Pair(H, Hkv, D, "fp16", pages=500, seqs=2, mpps=500, chunk_tokens=16)
    a = p.alloc()
    p.grow([a], [6100])
    k, v = p.begin([a], [1])
    q = p.rows(1, H)
    got = p.c.append_decode(0, k, v, q)
    assert p.c.step_num_work_items * H > 3000
    p.check_decode(got, [a], q)
    p.check_decode(p.c.decode_f32(0, q), [a], q, out="fp32")


def test_exchange_alone_in_the_world_equals_decode():
    from titan_engine_b200 import dist
    p = Pair(8, 2, 128, "bf16")
    seqs = [p.alloc() for _ in range(3)]
    p.grow(seqs, [300, 17, 1])
    p.c.step_begin(seqs)
    ex = dist.PeerExchange(24, 130, rank=0, world=1)
    for _ in range(3):
        q = p.rows(3, 8)
        got = p.c.decode_exchange(0, q, ex)
        p.check_decode(got, seqs, q)
    ex.status()
    ex.close()


def test_append_decode_on_a_capped_step():
    """The new row goes to the sequence's end, whatever the cap lets the query see."""
    p = Pair(8, 2, 64, "bf16")
    seqs = [p.alloc() for _ in range(3)]
    p.grow(seqs, [50, 333, 16])
    k, v = p.begin(seqs, [1, 1, 1])
    for s, n in zip(seqs, (50, 333, 16)):                   # the same step again, capped
        p.c.truncate(s, n)
    ids, one, cap = np.array(seqs, np.int32), np.ones(3, np.int32), np.array([7, 400, 16], np.int32)
    ptr = lambda x: x.ctypes.data_as(C.POINTER(C.c_int32))  # noqa: E731
    assert p.c._lib.tk_kv_step_begin_capped(p.c._h, 3, ptr(ids), ptr(one), ptr(cap), p.c._stream()) == 0
    p.c._n_seqs = p.c._n_tokens = 3
    q = p.rows(3, 8)
    n0 = p.c.launch_count
    got = p.c.append_decode(0, k, v, q)
    assert p.c.launch_count - n0 == 2                       # an append of its own: the fused one writes the last token that is seen
    p.check_decode(got, seqs, q, caps=[7, 400, 16])
    for s in seqs:
        p.check_rows(s)
