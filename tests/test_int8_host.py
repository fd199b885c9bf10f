"""INT8 pools without a GPU: the rounding of the codes, the configuration, and the calls that are refused."""
import numpy as np
import pytest

from titan_engine_b200 import KvError, PagedKVCache
from titan_engine_b200 import _lib as L

from int8_plain import quantise, stands_for


def _cache(**kw):
    args = dict(num_layers=1, num_heads=8, num_kv_heads=2, head_dim=64, num_pages=8, max_seqs=4, max_pages_per_seq=8, max_step_tokens=64, dtype="int8",
                host_only=True)
    args.update(kw)
    return PagedKVCache(**args)


@pytest.mark.parametrize("off", [-1, 0, 1])
def test_code_rounding_is_exact_for_every_pair_of_significands(off):
    """The kernel's float32 steps (a product with 127 times a reciprocal that may be one unit in the last place off, the snap to
    20 significant bits, one addition of a constant) against integer arithmetic, for every value / amax of 11-bit significands
    and every exponent gap at which a code is not 0."""
    f32 = np.float32
    b = np.arange(1024, 2048, dtype=np.int64)[:, None]                     # amax = b
    inv = ((f32(1.0) / b.astype(f32)).view(np.int32) + off).view(f32)
    to_code = f32(127.0) * inv
    for gap in range(0, 10):
        a = np.arange(1024, 2048, dtype=np.int64)[None, :]                 # x = a / 2^gap <= amax
        y = (a.astype(f32) / f32(2.0 ** gap)) * to_code
        snapped = ((y.view(np.uint32) + np.uint32(8)) & np.uint32(0xFFFFFFF0)).view(f32)
        got = (snapped + f32(12582912.0 + 128.0)).astype(f32).view(np.uint32).astype(np.int64) & 0xFF
        num, den = 2 * 127 * a, 2 * b * 2 ** gap                            # 127 x / amax = num / den
        q, rem = (num + den // 2) // den, (num + den // 2) % den
        want = np.where((rem == 0) & (q % 2 == 1), q - 1, q)                # a tie went up: take the even neighbour
        ok = a <= b * 2 ** gap
        assert (np.broadcast_to(got - 128, ok.shape)[ok] == want[ok]).all(), gap


def test_scale_is_the_rounded_quotient_for_every_significand():
    """amax * fl(1/127) and one residual step, in exact arithmetic rounded as the fused operations round, = fl(amax / 127)."""
    from fractions import Fraction

    def rn(x):                                                              # nearest float32 of a positive fraction
        e = 0
        while x >= 2 ** 24: x /= 2; e += 1
        while x < 2 ** 23: x *= 2; e -= 1
        n = x.numerator // x.denominator
        r = x - n
        n += r > Fraction(1, 2) or (r == Fraction(1, 2) and n % 2 == 1)
        return Fraction(n) * Fraction(2) ** e

    k127 = rn(Fraction(1, 127))
    for a in range(1024, 2049):
        q = rn(a * k127)
        r = a - q * 127                                                     # exact: far fewer than 24 significant bits
        assert rn(r * k127 + q) == rn(Fraction(a, 127))


def test_plain_rounding_of_ties_zeros_and_extremes():
    codes, scale = quantise(np.array([[2.0, 1.0, -1.0, 0.0], [0.0, 0.0, 0.0, 0.0], [np.inf, 1.0, -np.inf, 2.0 ** 64]]))
    assert codes[0].tolist() == [127, 64, -64, 0]                           # 63.5 -> 64 (even)
    assert codes[1].tolist() == [0, 0, 0, 0] and scale[1] > 0
    assert codes[2].tolist() == [127, 0, -127, 127]
    assert np.isfinite(stands_for(np.array([[np.inf, 1.0]]))).all()


@pytest.mark.parametrize("bad", [
    dict(page_size=32), dict(decode_impl="simt"), dict(chunk_tokens=4096), dict(hot_window=64, cold_pages=4),
    dict(head_dim=192, v_head_dim=128), dict(head_dim=96), dict(num_heads=6, num_kv_heads=2),
])
def test_refused_configurations(bad):
    with pytest.raises(KvError) as e:
        _cache(**bad)
    assert e.value.status == L.TK_INVALID_ARG


def test_arena_holds_codes_and_scales():
    c = _cache(num_layers=3, num_pages=5, head_dim=128)
    assert c.memory_bytes == 3 * ((5 * 2 * (2 * 16 * 128 + 2 * 16 * 4) + 1023) // 1024 * 1024)
    assert c.cfg.io_dtype == L.TK_BF16 and _cache(io_dtype="fp16").cfg.io_dtype == L.TK_FP16


def test_any_length_may_be_cut_adopted_and_capped():
    c = _cache()
    s = c.seq_alloc()
    c.step_begin([s], [37])
    c.truncate(s, 21)                                       # inside a full page
    assert c.seq_len(s) == 21
    t = c.seq_alloc()
    c.adopt(t, [6, 7], 19)
    assert c.seq_len(t) == 19
    a, b = np.array([s, t], np.int32), np.array([1, 1], np.int32)
    cap = np.array([5, 0], np.int32)
    import ctypes as C
    p = lambda x: x.ctypes.data_as(C.POINTER(C.c_int32))  # noqa: E731
    assert c._lib.tk_kv_step_begin_capped(c._h, 2, p(a), p(b), p(cap), None) == L.TK_OK


@pytest.mark.parametrize("tokens,heads,chunk", [
    (300, 64, 256), (8192, 64, 512), (16384, 64, 896), (32768, 64, 896), (40000, 64, 1024), (65536, 64, 2048), (131072, 64, 2048),
    (152000, 64, 2048), (170000, 64, 1536), (300000, 64, 2048), (131072, 128, 1536)])
def test_chunk_of_a_decode_step(tokens, heads, chunk):
    """One sequence on 8 kv heads: two items per SM of 148 (where it would be less than 1.7, down to 896 tokens each), and no launch
    of a little more than one wave: of 592 items, or of 444 where the rows of a kv head are two column blocks."""
    c = PagedKVCache(1, heads, 8, 128, 20000, 1, 20000, dtype="int8", io_dtype="bf16", max_step_tokens=tokens, host_only=True)
    s = c.seq_alloc()
    c.step_begin([s], [tokens - 1])
    c.step_begin([s], [1])
    assert c.step_chunk_tokens == chunk


def test_compute_calls_need_a_device():
    c = _cache()
    s = c.seq_alloc()
    c.step_begin([s], [3])
    with pytest.raises(KvError) as e:
        c.read(0, [s])
    assert e.value.status == L.TK_CUDA_ERROR
    assert c._lib.tk_kv_read(c._h, 0, 0, None, None, None, None, None, L.TK_BF16, None) == L.TK_CUDA_ERROR
    assert c._lib.tk_kv_read(c._h, 1, 0, None, None, None, None, None, L.TK_BF16, None) == L.TK_INVALID_ARG
    assert c._lib.tk_kv_read(None, 0, 0, None, None, None, None, None, L.TK_BF16, None) == L.TK_INVALID_ARG
    assert c._lib.tk_kv_decode_multi(c._h, 0, None, None, None) == L.TK_CUDA_ERROR


def test_unaligned_tensors_are_refused_before_anything_runs():
    """The kernels move 16-byte vectors; an address is looked at, never read."""
    c = _cache()
    c.step_begin([c.seq_alloc()], [1])
    lib, h, at, off = c._lib, c._h, 4096, 4096 + 2
    for i in range(2):
        kv = [off if i == j else at for j in range(2)]
        assert lib.tk_kv_append(h, 0, *kv, None, None) == L.TK_INVALID_ARG
        assert lib.tk_kv_decode(h, 0, *kv, None) == L.TK_INVALID_ARG
        assert lib.tk_kv_decode_multi(h, 0, *kv, None) == L.TK_INVALID_ARG
        assert lib.tk_kv_append_decode(h, 0, at, at, *kv, None) == L.TK_INVALID_ARG
        assert lib.tk_kv_append_decode_multi(h, 0, at, at, *kv, None) == L.TK_INVALID_ARG
        assert lib.tk_kv_append_decode_multi(h, 0, *kv, at, at, None) == L.TK_INVALID_ARG
        assert lib.tk_kv_read(h, 0, 0, None, None, None, *kv, L.TK_BF16, None) == L.TK_INVALID_ARG
    assert lib.tk_kv_decode_partial(h, 0, at, at + 4, None) == L.TK_INVALID_ARG
    for i in range(4):
        args = [off if i == j else at for j in range(4)]
        assert lib.tk_kv_rope_append_decode(h, 0, *args, 10000.0, 1.0, None) == L.TK_INVALID_ARG
    assert lib.tk_kv_decode(h, 0, at, at, None) == L.TK_CUDA_ERROR          # aligned: the next check answers


@pytest.mark.parametrize("shape", [(32, 8), (64, 8), (16, 1), (6, 3), (4, 4)])
@pytest.mark.parametrize("lens", [
    ([0, 5000, 33, 0, 40000, 700, 17], [300, 1, 4096, 70, 37, 3, 129]),
    ([1100, 518, 1240], [24, 334, 440]),
    ([65536], [20]), ([0], [8192]), ([3] * 40, [17] * 40),
])
def test_chunk_work_list_covers_every_row_once(shape, lens):
    """The 256-row tiles and their split-KV parts cover every (query token, head) and every position it sees exactly once; rows
    that fit one 16-row tile stay with the decode kernel; the list fits the step's buffers."""
    H, Hkv = shape
    G = H // Hkv
    ctx, new = lens
    c = _cache(num_heads=H, num_kv_heads=Hkv, num_pages=sum((a + b + 15) // 16 for a, b in zip(ctx, new)) + 1, max_seqs=len(ctx),
               max_pages_per_seq=max((a + b + 15) // 16 for a, b in zip(ctx, new)), max_step_tokens=sum(new))
    seqs = [c.seq_alloc() for _ in ctx]
    for s, n in zip(seqs, ctx):
        c.reserve(s, n)
    c.step_begin(seqs, new)
    items, ct, n_decode = c.step_prefill_plan()
    tpt = 256 // G
    small = [i for i, n in enumerate(new) if n * G <= 16]
    assert len(items) == 0 or n_decode == sum(-(-(a + b) // c.step_chunk_tokens) * Hkv for i, (a, b) in enumerate(zip(ctx, new)) if i in small)
    seen = {}
    for b, chunk, kvh, tile in items.tolist():
        assert b not in small and 0 <= kvh < Hkv and ct[b] % 64 == 0 and ct[b] <= 32768
        p_last = ctx[b] + min(new[b], (tile + 1) * tpt) - 1
        t0, t1 = chunk * ct[b], min((chunk + 1) * ct[b], p_last + 1)
        assert tile * tpt < new[b] and t1 > t0
        seen.setdefault((b, kvh, tile), []).append((t0, t1))
    for b, n in enumerate(new):
        for kvh in range(Hkv if b not in small else 0):
            for tile in range(-(-n // tpt)):
                spans = sorted(seen.pop((b, kvh, tile)))
                p_last = ctx[b] + min(n, (tile + 1) * tpt) - 1
                assert spans[0][0] == 0 and spans[-1][1] == p_last + 1 and all(x[1] == y[0] for x, y in zip(spans, spans[1:]))
                assert len(spans) == p_last // ct[b] + 1
    assert not seen
