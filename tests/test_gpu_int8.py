"""INT8 pools on the GPU against int8_plain.py: codes and scales bit for bit, rows read back bit for bit, attention within the
bound derived there."""
import numpy as np
import pytest
import torch

from int8_plain import attention, check, quantise, stands_for

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(autouse=True)
def _need_cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    yield
    torch.cuda.synchronize()


class Pair:
    """An INT8 cache of one layer and, for every sequence, the rows that were appended to it."""

    def __init__(self, H, Hkv, D, io="bf16", pages=256, seqs=8, mpps=256, poison=True, seed=0, **kw):
        from titan_engine_b200 import PagedKVCache
        self.H, self.Hkv, self.D, self.io = H, Hkv, D, io
        kw.setdefault("max_step_tokens", 4096)
        self.c = PagedKVCache(kw.pop("layers", 1), H, Hkv, D, pages, seqs, mpps, dtype="int8", io_dtype=io, **kw)
        self.dev = self.c.device
        if poison:                                          # whatever a page's last owner left: NaN scales, every code bit set
            codes, scales, _ = self.c.layer_views(0)
            codes.fill_(255)
            scales.fill_(float("nan"))
        self.g = torch.Generator(device=self.dev)
        self.g.manual_seed(seed)
        self.k, self.v = {}, {}

    def rows(self, n, heads, scale=1.0):
        return (torch.randn(n, heads, self.D, device=self.dev, generator=self.g) * scale).to(TYPES[self.io])

    def alloc(self):
        s = self.c.seq_alloc()
        self.k[s] = self.v[s] = np.zeros((0, self.Hkv, self.D), np.float32)
        return s

    def begin(self, seqs, n_new, vscale=1.0):
        """Begins a step and makes its rows; the plain copies take them over."""
        self.c.step_begin(seqs, n_new)
        n = sum(n_new)
        k = self.rows(n, self.Hkv)
        v = self.rows(n, self.Hkv) * (vscale * torch.exp(torch.randn(n, self.Hkv, 1, device=self.dev, generator=self.g))).to(TYPES[self.io])
        kf, vf, at = k.float().cpu().numpy(), v.float().cpu().numpy(), 0
        for s, m in zip(seqs, n_new):
            self.k[s] = np.concatenate([self.k[s], stands_for(kf[at:at + m])])
            self.v[s] = np.concatenate([self.v[s], stands_for(vf[at:at + m])])
            at += m
        return k, v

    def grow(self, seqs, n_new, vscale=1.0):
        at = 0
        while at < max(n_new):                              # in steps that the cache takes
            part = [min(max(n - at, 0), 1024) for n in n_new]
            k, v = self.begin(seqs, part, vscale)
            self.c.append(0, k, v)
            at += 1024

    def check_decode(self, got, seqs, q, caps=None, out=None):
        qf = q.float().cpu().numpy()
        for i, s in enumerate(seqs):
            lim = len(self.k[s]) if caps is None else min(caps[i], len(self.k[s]))
            want, bound = attention(qf[i:i + 1], self.k[s], self.v[s], [lim], out or self.io)
            check(got[i:i + 1].float().cpu().numpy(), want, bound, f"sequence {s}, {lim} tokens")

    def check_chunk(self, got, seqs, n_new, q, out=None):
        qf, at = q.float().cpu().numpy(), 0
        for s, m in zip(seqs, n_new):
            n = len(self.k[s])
            want, bound = attention(qf[at:at + m], self.k[s], self.v[s], np.arange(n - m, n) + 1, out or self.io)
            check(got[at:at + m].float().cpu().numpy(), want, bound, f"sequence {s}, {m} new of {n} tokens")
            at += m

    def check_rows(self, s, what=""):
        k, v = self.c.read(0, [s], out_dtype=torch.float32)
        np.testing.assert_array_equal(k.cpu().numpy(), self.k[s], err_msg=what)
        np.testing.assert_array_equal(v.cpu().numpy(), self.v[s], err_msg=what)


# ---- write and read back ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("io", ["bf16", "fp16"])
@pytest.mark.parametrize("Hkv,D", [(1, 64), (3, 64), (2, 128), (8, 128)])
def test_append_codes_and_scales(Hkv, D, io):
    p = Pair(Hkv * 2, Hkv, D, io, seqs=4)
    a, b, c = p.alloc(), p.alloc(), p.alloc()
    before = p.c.layer_views(0)[0].clone()
    p.grow([a, b, c], [37, 1, 160])
    p.grow([a, b, c], [1, 0, 16])
    assert p.c.layer_views(0)[1].shape == (256, Hkv, 2, 16)
    codes, scales, _ = p.c.layer_views(0)
    for s in (a, b, c):
        n = len(p.k[s])
        pages = torch.from_numpy(p.c.page_table(s).astype(np.int64)).to(p.dev)
        for kv, rows in ((0, p.k[s]), (1, p.v[s])):
            got = codes[pages, :, kv].permute(0, 2, 1, 3).reshape(-1, Hkv, D)[:n].cpu().numpy().astype(np.float32) - 128
            sc = scales[pages, :, kv].permute(0, 2, 1).reshape(-1, Hkv)[:n].cpu().numpy()
            np.testing.assert_array_equal(got * sc[..., None], rows)
            assert np.abs(got).max() == 127
            # rows of the last page behind the sequence, and pages of nobody, are as they were
            tail = codes[pages[-1], :, kv, n - 16 * (len(pages) - 1):]
            assert (tail == 255).all()
        p.check_rows(s)
    used = np.concatenate([p.c.page_table(s) for s in (a, b, c)])
    idle = torch.from_numpy(np.setdiff1d(np.arange(256), used)).to(p.dev)
    assert torch.equal(codes[idle], before[idle])


@pytest.mark.parametrize("io", ["bf16", "fp16"])
def test_append_extreme_rows(io):
    p = Pair(4, 2, 64, io, seqs=2)
    s = p.alloc()
    t = TYPES[io]
    big, tiny = torch.finfo(t).max, torch.finfo(t).smallest_normal
    x = torch.randn(12, 2, 64, device=p.dev, generator=p.g).to(t)
    x[0] = 0
    x[1, 0] = 0; x[1, 0, 5] = -3.0
    x[2] = x[2].sign() * 1.5; x[2, :, 1::2] = 0.75          # exact halves of the maximum: ties at 63.5
    x[3] *= tiny * 4
    x[4, 0, 0] = big
    x[5, 0, 0] = float("inf"); x[5, 1, 3] = -float("inf")
    x[6, 0, 9] = float("nan")
    x[7] = torch.finfo(t).tiny
    x[8] = x[8].clamp(-1, 1); x[8, :, 0] = 127.0 / 128
    p.c.step_begin([s], [12])
    p.c.append(0, x, x.flip(0).contiguous())
    k, v = p.c.read(0, [s], out_dtype=torch.float32)
    for got, src in ((k, x), (v, x.flip(0))):
        src = src.float().cpu().numpy()
        nan = np.isnan(src).any(axis=-1)
        assert nan.sum() == 1
        got = got.cpu().numpy()
        assert np.isnan(got[nan]).all()                     # a NaN poisons its row, and no other
        np.testing.assert_array_equal(got[~nan], stands_for(src[~nan]))


def test_append_slots_and_empty_step():
    p = Pair(4, 2, 64)
    a, b = p.alloc(), p.alloc()
    k, v = p.begin([a, b], [18, 3])
    slots = torch.full((21,), -7, dtype=torch.int64, device=p.dev)
    p.c.append(0, k, v, slots)
    assert slots.tolist() == [p.c.slot(a, i) for i in range(18)] + [p.c.slot(b, i) for i in range(3)]
    p.c.step_begin([a, b], [0, 0])
    z = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=p.dev)
    p.c.append(0, z, z)
    p.check_rows(a); p.check_rows(b)


@pytest.mark.parametrize("io", ["bf16", "fp16"])
def test_read_ranges_in_every_output_type(io):
    p = Pair(8, 2, 128, io)
    a, b, e = p.alloc(), p.alloc(), p.alloc()
    p.grow([a, b], [75, 33])
    seqs, start, count = [b, a, a, e, b], [0, 15, 3, 0, 33], [33, 50, 1, 0, 0]
    want_k = np.concatenate([p.k[s][i:i + n] for s, i, n in zip(seqs, start, count)])
    want_v = np.concatenate([p.v[s][i:i + n] for s, i, n in zip(seqs, start, count)])
    k, v = p.c.read(0, seqs, start, count, out_dtype=torch.float32)
    np.testing.assert_array_equal(k.cpu().numpy(), want_k)
    np.testing.assert_array_equal(v.cpu().numpy(), want_v)
    k, v = p.c.read(0, seqs, start, count)
    assert k.dtype == TYPES[io] and torch.equal(k.cpu(), torch.from_numpy(want_k).to(TYPES[io]))
    assert torch.equal(v.cpu(), torch.from_numpy(want_v).to(TYPES[io]))
    k, _ = p.c.read(0, [a, b])
    assert k.shape[0] == 108
    k, _ = p.c.read(0, [])
    assert k.shape[0] == 0


@pytest.mark.parametrize("dtype,D,Dv", [("bf16", 128, 0), ("fp16", 64, 0), ("fp8", 128, 0), ("bf16", 192, 128)])
@pytest.mark.parametrize("ps", [16, 8])
def test_read_of_the_other_pools(dtype, D, Dv, ps):
    """16-bit pools give their bits back; FP8 pools sealed pages (codes * scale) and the rows of the open page."""
    from titan_engine_b200 import PagedKVCache
    Dv = Dv or D
    c = PagedKVCache(1, 4, 2, D, 64, 3, 32, dtype=dtype, v_head_dim=Dv if Dv != D else 0, max_step_tokens=256, page_size=ps)
    s = [c.seq_alloc() for _ in range(3)]
    n = [37, 16, 5]
    c.step_begin(s, n)
    g = torch.Generator(device=c.device); g.manual_seed(5)
    k = torch.randn(58, 2, D, device=c.device, generator=g).to(c.io_torch_dtype)
    v = torch.randn(58, 2, Dv, device=c.device, generator=g).to(c.io_torch_dtype)
    c.append(0, k, v)
    seqs, start, count = [s[1], s[0], s[2], s[0]], [3, 0, 1, 31], [13, 37, 4, 6]
    rows = torch.cat([torch.arange(o + a, o + a + m) for o, a, m in zip([37, 0, 53, 0], start, count)]).to(c.device)
    want = [k[rows], v[rows]]
    if dtype == "fp8":
        pool, scales, _ = c.layer_views(0)
        for kv in (0, 1):
            for b, at in zip(s, (0, 37, 53)):
                for i, page in enumerate(c.page_table(b)[:c.seq_len(b) // ps]):
                    sealed = pool[page, :, kv].view(torch.float8_e4m3fn).float() * scales[page, :, kv, None, None]
                    (k, v)[kv][at + ps * i:at + ps * (i + 1)] = sealed.transpose(0, 1).to(c.io_torch_dtype)
        want = [k[rows], v[rows]]
    for out in (c.io_torch_dtype, torch.float32):
        got = c.read(0, seqs, start, count, out_dtype=out)
        for x, y in zip(got, want):
            if dtype == "fp8" and out == torch.float32:
                assert torch.equal(x.to(c.io_torch_dtype), y)
            else:
                assert torch.equal(x, y.to(out))


def test_read_refusals():
    from titan_engine_b200 import KvError
    from titan_engine_b200 import _lib as L
    p = Pair(4, 2, 64)
    a = p.alloc()
    p.grow([a], [20])
    for seqs, start, count in (([a], [0], [21]), ([a], [-1], [3]), ([a], [3], [-1]), ([a], [21], [0]), ([7], [0], [0]),
                               ([-1], [0], [1]), ([99], [0], [1]), ([a], [2 ** 31 - 1], [2 ** 31 - 1])):
        with pytest.raises(KvError) as e:
            p.c.read(0, seqs, start, count)
        assert e.value.status == L.TK_INVALID_ARG
    with pytest.raises(KvError):
        p.c.read(0, [a], [0, 1], [1])
    with pytest.raises(KvError):
        p.c.read(0, [a], out_dtype=torch.float16)
    with pytest.raises(KvError):
        p.c.read(3, [a])


def test_unaligned_views_are_refused():
    """A contiguous view that starts inside a 16-byte vector, for every tensor of every call."""
    from titan_engine_b200 import KvError
    p = Pair(4, 2, 64)
    a = p.alloc()
    p.grow([a], [20])
    k, v = p.begin([a], [1])
    q = p.rows(1, 4)

    def off(x):
        return torch.cat([x.flatten()[:1], x.flatten()])[1:].view(x.shape)

    calls = {"append": (p.c.append, [k, v]), "decode": (p.c.decode, [q, q.clone()]),
             "append_decode": (p.c.append_decode, [k, v, q, q.clone()]), "decode_multi": (p.c.decode_multi, [q, q.clone()]),
             "append_decode_multi": (p.c.append_decode_multi, [k, v, q, q.clone()])}
    for name, (call, args) in calls.items():
        for i in range(len(args)):
            with pytest.raises(KvError, match="aligned"):
                call(0, *[off(x) if i == j else x for j, x in enumerate(args)])
    with pytest.raises(KvError, match="aligned"):
        p.c.rope_append_decode(0, off(k), v, q, 10000.0)
    p.check_decode(p.c.append_decode(0, k, v, q), [a], q)


def test_read_after_fork_and_truncation_needs_no_step():
    p = Pair(8, 2, 64)
    a = p.alloc()
    p.grow([a], [41])
    child = p.c.fork(a)
    p.k[child], p.v[child] = p.k[a], p.v[a]
    p.check_rows(child)
    p.c.truncate(a, 35)
    p.k[a], p.v[a] = p.k[a][:35], p.v[a][:35]
    p.check_rows(a); p.check_rows(child)
    p.grow([a, child], [9, 1])                              # each writes its own copy of the last page
    p.check_rows(a); p.check_rows(child)


def test_read_many_pages_in_several_launches():
    p = Pair(1, 1, 64, pages=2600, seqs=3, mpps=2500, max_step_tokens=40000)
    a, b = p.alloc(), p.alloc()
    p.grow([a, b], [36005, 77])
    k, v = p.c.read(0, [b, a], [5, 2], [72, 36003], out_dtype=torch.float32)
    np.testing.assert_array_equal(k.cpu().numpy(), np.concatenate([p.k[b][5:77], p.k[a][2:]]))
    np.testing.assert_array_equal(v.cpu().numpy(), np.concatenate([p.v[b][5:77], p.v[a][2:]]))


# ---- one token per sequence -----------------------------------------------------------------------------------
@pytest.mark.parametrize("n", [1, 15, 16, 17, 255, 256, 257, 2049])
@pytest.mark.parametrize("H,Hkv,D,io", [(8, 2, 64, "fp16"), (32, 8, 128, "bf16")])
def test_decode_lengths(H, Hkv, D, io, n):
    p = Pair(H, Hkv, D, io)
    s = p.alloc()
    p.grow([s], [n])
    p.c.step_begin([s])
    q = p.rows(1, H)
    p.check_decode(p.c.decode(0, q), [s], q)


@pytest.mark.parametrize("H,Hkv,D,io", [(4, 4, 64, "bf16"), (6, 3, 128, "fp16"), (8, 2, 64, "fp16"), (16, 2, 128, "bf16"), (16, 1, 128, "fp16"),
                                        (16, 1, 64, "bf16"), (64, 8, 128, "bf16")])
@pytest.mark.parametrize("separate", [False, True])
def test_append_decode_ragged_batch(H, Hkv, D, io, separate):
    p = Pair(H, Hkv, D, io, separate_combine=separate)
    seqs = [p.alloc() for _ in range(6)]
    p.grow(seqs, [0, 16, 1, 700, 31, 130])
    for vscale in (1.0, 1e-4, 300.0):                       # probabilities times tiny and large value scales
        k, v = p.begin(seqs, [1] * 6, vscale)
        q = p.rows(6, H, 2.0)
        p.check_decode(p.c.append_decode(0, k, v, q), seqs, q)
    for s in seqs:
        p.check_rows(s)


def test_decode_large_queries():
    """bf16 queries far outside fp16's range, next to ordinary ones and zeros."""
    p = Pair(8, 2, 128, "bf16")
    seqs = [p.alloc() for _ in range(4)]
    p.grow(seqs, [40, 40, 7, 200])
    p.c.step_begin(seqs)
    q = p.rows(4, 8)
    q[0, 1::2] *= 1e-30
    q[1] = 0
    q[2, 0] *= 2.0 ** 60
    got = p.c.decode(0, q)
    p.check_decode(got[:2], seqs[:2], q[:2])
    p.check_decode(got[3:], seqs[3:], q[3:])
    want, bound = attention(q[2:3].float().cpu().numpy(), p.k[seqs[2]], p.v[seqs[2]], [7], "bf16")
    check(got[2:3, 1:].float().cpu().numpy(), want[:, 1:], bound[:, 1:])
    # with such a query one key takes all: its value row
    s = np.einsum("d,ld->l", q[2, 0].double().cpu().numpy(), p.k[seqs[2]][:, 0].astype(np.float64))
    np.testing.assert_allclose(got[2, 0].float().cpu().numpy(), p.v[seqs[2]][s.argmax(), 0], rtol=2 ** -8)


def test_decode_mixed_value_scales():
    """Rows whose scales are 2^60 apart in one sequence."""
    p = Pair(4, 1, 64, "bf16")
    s = p.alloc()
    for vs in (1.0, 2.0 ** 40, 2.0 ** -20, 1.0):
        p.grow([s], [19], vs)
    p.c.step_begin([s])
    q = p.rows(1, 4)
    p.check_decode(p.c.decode(0, q), [s], q)


def test_decode_empty_sequences_caps_and_f32():
    p = Pair(8, 2, 128, "bf16")
    a, b, c = p.alloc(), p.alloc(), p.alloc()
    p.grow([a, b], [50, 333])
    p.c.step_begin([a, c, b])
    q = p.rows(3, 8)
    got = p.c.decode(0, q)
    assert (got[1] == 0).all()                              # attends to nothing
    p.check_decode(got[[0, 2]], [a, b], q[[0, 2]])
    p.check_decode(p.c.decode_f32(0, q)[[0, 2]], [a, b], q[[0, 2]], out="fp32")
    import ctypes as C
    ids, cap = np.array([a, b], np.int32), np.array([7, 300], np.int32)
    ptr = lambda x: x.ctypes.data_as(C.POINTER(C.c_int32))  # noqa: E731
    assert p.c._lib.tk_kv_step_begin_capped(p.c._h, 2, ptr(ids), None, ptr(cap), p.c._stream()) == 0
    p.c._n_seqs = 2
    p.check_decode(p.c.decode(0, q[:2].contiguous()), [a, b], q[:2], caps=[7, 300])


def test_decode_partials_merge_to_the_whole():
    """Two caches hold a sequence's halves, as two ranks do: their partial rows merge to the attention over all of it."""
    import ctypes as C
    left, right = Pair(8, 2, 128, seed=1), Pair(8, 2, 128, seed=2)
    a, b = left.alloc(), right.alloc()
    left.grow([a], [77]); right.grow([b], [300])
    left.c.step_begin([a]); right.c.step_begin([b])
    q = left.rows(1, 8)
    parts = torch.cat([left.c.decode_partial(0, q), right.c.decode_partial(0, q)])
    out = torch.empty(1, 8, 128, dtype=torch.float32, device=left.dev)
    assert left.c._lib.tk_combine_partials(parts.data_ptr(), 2, 8, 128, out.data_ptr(), 0, left.c._stream()) == 0
    whole = attention(q.float().cpu().numpy(), np.concatenate([left.k[a], right.k[b]]), np.concatenate([left.v[a], right.v[b]]), [377], "fp32")
    check(out.cpu().numpy(), *whole)


# ---- chunks of new tokens ----------------------------------------------------------------------------------------
CHUNKS = [
    (8, 2, 64, "fp16", [0, 0], [1, 2]),
    (8, 2, 64, "fp16", [5, 0, 130], [3, 70, 1]),
    (32, 8, 128, "bf16", [100, 0, 16], [4, 4, 4]),
    (32, 8, 128, "bf16", [0, 500], [129, 17]),
    (4, 4, 128, "fp16", [33], [300]),
    (16, 1, 128, "bf16", [0, 7, 1000], [1, 33, 8]),
    (16, 1, 64, "fp16", [200, 0], [40, 16]),
    (6, 3, 64, "bf16", [0, 63], [65, 64]),
    (16, 2, 128, "fp16", [1500], [257]),
]


@pytest.mark.parametrize("case", range(len(CHUNKS)))
def test_chunk_attention(case):
    H, Hkv, D, io, ctx, new = CHUNKS[case]
    p = Pair(H, Hkv, D, io, seed=case)
    seqs = [p.alloc() for _ in ctx]
    p.grow(seqs, ctx)
    k, v = p.begin(seqs, new)
    q = p.rows(sum(new), H, 1.5)
    p.check_chunk(p.c.append_decode_multi(0, k, v, q), seqs, new, q)
    p.check_chunk(p.c.decode_multi_f32(0, q), seqs, new, q, out="fp32")
    for s in seqs:
        p.check_rows(s)
    p.c.device_status()


@pytest.mark.parametrize("vscale", [1e-4, 300.0])
def test_chunk_value_scales(vscale):
    p = Pair(8, 2, 128, "fp16")
    s = p.alloc()
    p.grow([s], [90], 1.0)
    k, v = p.begin([s], [150], vscale)
    q = p.rows(150, 8, 2.0)
    p.check_chunk(p.c.append_decode_multi(0, k, v, q), [s], [150], q)


def test_chunk_large_queries():
    """bf16 queries far outside fp16's range next to ordinary ones, tiny ones and zeros in one tile."""
    p = Pair(8, 2, 128, "bf16")
    s = p.alloc()
    p.grow([s], [200])
    k, v = p.begin([s], [90])
    q = p.rows(90, 8)
    q[3, 1::2] *= 1e-30
    q[4] = 0
    q[40:44, 0] *= 2.0 ** 60
    got = p.c.append_decode_multi(0, k, v, q).float().cpu().numpy()
    want, bound = attention(q.float().cpu().numpy(), p.k[s], p.v[s], np.arange(200, 290) + 1, "bf16")
    plain = np.ones((90, 8), bool)
    plain[40:44, 0] = False
    check(got[plain], want[plain], bound[plain])
    for t in range(40, 44):                                 # with such a query one key takes all: its value row
        best = np.einsum("d,ld->l", q[t, 0].double().cpu().numpy(), p.k[s][:201 + t, 0].astype(np.float64)).argmax()
        np.testing.assert_allclose(got[t, 0], p.v[s][best, 0], rtol=2 ** -8)


@pytest.mark.parametrize("H,Hkv,D,io", [(8, 2, 128, "bf16"), (8, 1, 64, "fp16"), (16, 1, 128, "fp16")])
def test_chunk_rows_around_the_tile_halves(H, Hkv, D, io):
    """(token, head) rows just below, at and above 128 and 256 of them, over contexts that end inside a page and a block."""
    G = H // Hkv
    new = [n for r in (128, 256) for n in (r // G - 1, r // G, r // G + 1)]
    ctx = [0, 63, 64, 65, 15, 449]
    p = Pair(H, Hkv, D, io, seqs=6, pages=512)
    seqs = [p.alloc() for _ in new]
    p.grow(seqs, ctx)
    k, v = p.begin(seqs, new)
    q = p.rows(sum(new), H, 1.5)
    p.check_chunk(p.c.append_decode_multi(0, k, v, q), seqs, new, q)


def test_chunk_split_over_a_long_context():
    """Few rows and a long context: the chunk's tile is split along the context and the parts merge."""
    p = Pair(8, 2, 128, "bf16", pages=1400, mpps=700)
    a, b = p.alloc(), p.alloc()
    p.grow([a, b], [9001, 5000], 1.0)
    new = [30, 7]
    for vscale in (1.0, 2.0 ** 30):
        k, v = p.begin([a, b], new, vscale)
        q = p.rows(37, 8, 2.0)
        p.check_chunk(p.c.append_decode_multi(0, k, v, q), [a, b], new, q)
        items, ct, _ = p.c.step_prefill_plan()
        assert len(items) and ct[0] < 9000                  # really split


def test_nan_rows_poison_only_the_queries_that_see_them():
    p = Pair(4, 1, 64, "bf16")
    a, b = p.alloc(), p.alloc()
    p.grow([a, b], [30, 30])
    k, v = p.begin([a, b], [100, 3])
    k[60, 0, 5] = float("nan")
    v[80, 0, 1] = float("nan")
    q = p.rows(103, 4)
    got = p.c.append_decode_multi(0, k, v, q)
    assert torch.isnan(got[60:100]).all() and torch.isfinite(got[:60]).all() and torch.isfinite(got[100:]).all()
    p.k[a][90], p.v[a][110] = 0, 0
    n = 60
    want, bound = attention(q[:n].float().cpu().numpy(), p.k[a][:90], p.v[a][:90], np.arange(30, 30 + n) + 1, "bf16")
    check(got[:n].float().cpu().numpy(), want, bound)
    p.c.step_begin([b, a])
    out = p.c.decode(0, q[:2].contiguous())
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1]).all()


def test_chunk_refusals():
    from titan_engine_b200 import KvError
    from titan_engine_b200 import _lib as L
    import ctypes as C
    p = Pair(8, 2, 64)
    a, b = p.alloc(), p.alloc()
    p.grow([a, b], [20, 5])
    p.c.step_begin([a, b], [1, 0])
    with pytest.raises(KvError) as e:
        p.c.decode_multi(0, p.rows(1, 8))
    assert e.value.status == L.TK_INVALID_ARG               # b appends nothing
    ids, one, cap = np.array([a], np.int32), np.array([2], np.int32), np.array([9], np.int32)
    ptr = lambda x: x.ctypes.data_as(C.POINTER(C.c_int32))  # noqa: E731
    assert p.c._lib.tk_kv_step_begin_capped(p.c._h, 1, ptr(ids), ptr(one), ptr(cap), p.c._stream()) == 0
    p.c._n_seqs, p.c._n_tokens = 1, 2
    with pytest.raises(KvError) as e:
        p.c.decode_multi(0, p.rows(2, 8))
    assert e.value.status == L.TK_UNSUPPORTED


# ---- as they are used together -------------------------------------------------------------------------------------
def test_prompt_draft_rollback_decode_and_export():
    """A prompt chunk, drafted tokens of which some are dropped inside a page, decode steps, a fork, and the rows read back."""
    p = Pair(16, 4, 128, "bf16", pages=400)
    a, b = p.alloc(), p.alloc()
    k, v = p.begin([a, b], [200, 45])
    q = p.rows(245, 16)
    p.check_chunk(p.c.append_decode_multi(0, k, v, q), [a, b], [200, 45], q)
    for keep in (1, 3, 4):
        k, v = p.begin([a, b], [4, 4])
        q = p.rows(8, 16)
        p.check_chunk(p.c.append_decode_multi(0, k, v, q), [a, b], [4, 4], q)
        for s in (a, b):
            n = len(p.k[s]) - 4 + keep
            p.c.truncate(s, n)
            p.k[s], p.v[s] = p.k[s][:n], p.v[s][:n]
    c = p.c.fork(a)
    p.k[c], p.v[c] = p.k[a], p.v[a]
    for _ in range(3):
        k, v = p.begin([a, b, c], [1, 1, 1])
        q = p.rows(3, 16)
        p.check_decode(p.c.append_decode(0, k, v, q), [a, b, c], q)
    for s in (a, b, c):
        p.check_rows(s)
    p.c.device_status()


def test_scheduler_drives_an_int8_cache():
    from titan_engine_b200.scheduler import BatchScheduler
    p = Pair(8, 2, 128, "bf16", pages=80, seqs=4, mpps=40, max_step_tokens=128)
    sch = BatchScheduler(p.c, 4, 96)
    for n, m in ((70, 3), (5, 6), (130, 2), (33, 4)):
        sch.submit(n, m)
    lens, checked = {}, 0
    for _ in range(12):
        rows = sch.next()
        if not rows:
            break
        seqs, new = [r.seq for r in rows], [r.n_new for r in rows]
        for s, n in zip(seqs, new):
            if p.c.seq_len(s) == n:                         # admitted (or admitted again) in this step
                p.k[s] = p.v[s] = np.zeros((0, 2, 128), np.float32)
        n = sum(new)
        k, v, q = p.rows(n, 2), p.rows(n, 2), p.rows(n, 8)
        kf, vf, at = k.float().cpu().numpy(), v.float().cpu().numpy(), 0
        for s, m in zip(seqs, new):
            p.k[s] = np.concatenate([p.k[s], stands_for(kf[at:at + m])])
            p.v[s] = np.concatenate([p.v[s], stands_for(vf[at:at + m])])
            at += m
        p.check_chunk(p.c.append_decode_multi(0, k, v, q), seqs, new, q)
        checked += n
        sch.commit([False] * len(rows))
    assert checked >= 238


def test_rope_and_host_buffer_paths():
    """rope_append_decode = the rotated rows through append_decode; append_decode_host = the device path."""
    p, r = Pair(8, 2, 64, "fp16", seed=3), Pair(8, 2, 64, "fp16", seed=3)
    seqs = [p.alloc(), p.alloc()]
    assert [r.alloc(), r.alloc()] == seqs
    p.grow(seqs, [20, 3]); r.grow(seqs, [20, 3])
    k, v = p.begin(seqs, [1, 1])
    r.c.step_begin(seqs, [1, 1])
    q = p.rows(2, 8)
    pos = torch.tensor([20.0, 3.0], device=p.dev)
    freq = (1.0 / torch.pow(torch.tensor(10000.0, device=p.dev), torch.arange(0, 64, 2, device=p.dev).float() / 64))
    ang = pos[:, None, None] * freq

    def rot(x):
        x = x.float()
        x0, x1 = x[..., 0::2], x[..., 1::2]
        return torch.stack([x0 * ang.cos() - x1 * ang.sin(), x0 * ang.sin() + x1 * ang.cos()], -1).flatten(-2).to(torch.float16)

    got = r.c.rope_append_decode(0, k, v, q, 10000.0)
    want = p.c.append_decode(0, rot(k), v, rot(q))
    # the two rotations may round a value to neighbouring fp16 numbers and a code to its neighbour: 1/127 of a key
    assert (got.float() - want.float()).abs().max() < 0.05
    hk, hv, hq = (x.cpu().pin_memory() for x in (rot(k), v, rot(q)))
    out = torch.empty(2, 8, 64, dtype=torch.float16).pin_memory()
    p.c.append_decode_host(0, hk, hv, hq, out)
    assert torch.equal(out, want.cpu())


@pytest.mark.parametrize("io,D", [("bf16", 64), ("bf16", 128), ("fp16", 64), ("fp16", 128)])
def test_rope_append_decode_against_64_bits(io, D):
    """The rows that rope_append_decode leaves in the cache, and its result, against rotations in 64 bits.  An angle (position x
    inverse frequency) carries a few FP32 roundings, far below a step of the 16-bit type: a rotated value is the nearest 16-bit
    number or its neighbour, a distance of at most one step u = eps of the type, relative.  A stored row is then within
    half a code plus u of the rotation; a score of query q and key k within d = u sum |q_i k_i| / sqrt(D), which moves every
    probability by at most a factor e^(2 d)."""
    p = Pair(8, 2, D, io)
    seqs, held = [p.alloc() for _ in range(3)], [0, 20, 300]
    p.grow(seqs, held)
    k, v = p.begin(seqs, [1, 1, 1])
    q = p.rows(3, 8)
    got = p.c.rope_append_decode(0, k, v, q, 10000.0).float().cpu().numpy().astype(np.float64)
    u = torch.finfo(TYPES[io]).eps

    def rot(x, pos):                                        # one token's heads [h, D]
        x = x.double().cpu().numpy()
        ang = pos / 10000.0 ** (np.arange(0, D, 2) / D)
        y = np.empty_like(x)
        y[:, 0::2] = x[:, 0::2] * np.cos(ang) - x[:, 1::2] * np.sin(ang)
        y[:, 1::2] = x[:, 0::2] * np.sin(ang) + x[:, 1::2] * np.cos(ang)
        return y

    for i, (s, n) in enumerate(zip(seqs, held)):
        ks, vs = (x.double().cpu().numpy() for x in p.c.read(0, [s], out_dtype=torch.float32))
        want = rot(k[i], n)
        amax = np.abs(want).max(-1, keepdims=True) * (1 + u)
        assert (np.abs(ks[n] - want) <= amax * (0.51 / 127 + u)).all()
        np.testing.assert_array_equal(vs[n], p.v[s][n])
        np.testing.assert_array_equal(ks[:n], p.k[s][:n])
        qr = torch.from_numpy(rot(q[i], n)).to(TYPES[io]).double().numpy()
        out, bound = attention(qr[None], ks, vs, [n + 1], io)
        kk, vv = np.repeat(ks, 4, 1), np.repeat(np.abs(vs), 4, 1)              # [tokens, H, D]
        d = (u * np.abs(qr[None] * kk).sum(-1) / np.sqrt(D)).max(0)            # per head
        top = (np.exp(2 * d) - 1)[:, None] * vv.max(0)
        assert (np.abs(got[i] - out[0]) <= bound[0] + top).all()


def test_read_in_several_launches_captured_and_on_two_streams():
    """A read of more pages than one launch lists, replayed from a graph, next to an eager one of the same rows on another stream."""
    p = Pair(2, 1, 64, "bf16", pages=2100, seqs=2, mpps=2100, max_step_tokens=40000, poison=False)
    a = p.alloc()
    n = 2050 * 16 - 3
    k, v = p.begin([a], [n])
    p.c.append(0, k, v)
    want = [x.clone() for x in p.c.read(0, [a, a], [0, 5], [n, 40])]
    np.testing.assert_array_equal(want[0][:n].double().cpu().numpy(), torch.from_numpy(p.k[a]).to(torch.bfloat16).double().numpy())
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        got = p.c.read(0, [a, a], [0, 5], [n, 40])
    for x in got:
        x.zero_()
    torch.cuda.synchronize()
    graph.replay()
    with torch.cuda.stream(side):
        there = p.c.read(0, [a, a], [0, 5], [n, 40])
    graph.replay()
    torch.cuda.synchronize()
    for x, y, z in zip(want, got, there):
        assert torch.equal(x, y) and torch.equal(x, z) and torch.equal(x[n:], x[5:45])


def test_captured_step_replays_next_to_eager_calls_on_another_stream():
    p = Pair(8, 2, 128, "bf16", layers=2)
    other = Pair(8, 2, 128, "bf16", seed=9)
    seqs = [p.alloc(), p.alloc()]
    t = other.alloc()
    p.grow(seqs, [100, 37]); other.grow([t], [513])
    k, v = p.begin(seqs, [1, 1])
    q = p.rows(2, 8)
    want = p.c.append_decode(0, k, v, q).clone()
    rows = [x.clone() for x in p.c.read(0, seqs)]
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        got = p.c.append_decode(0, k, v, q)
        again = p.c.read(0, seqs)
    other.c.step_begin([t])
    qo = other.rows(1, 8)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        outs = [other.c.decode(0, qo) for _ in range(3)]
    for _ in range(3):
        got.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all(torch.equal(x, y) for x, y in zip(again, rows))
    for o in outs:
        other.check_decode(o, [t], qo)


def test_captured_chunk_keeps_its_workspace_when_a_larger_step_grows_it():
    """A split chunk whose workspace the handle has to allocate: refused inside a capture, which lives on; captured after one
    eager run; a larger step then takes a larger workspace and the graph still has its own."""
    from titan_engine_b200 import KvError
    p = Pair(8, 2, 128, pages=512, mpps=256)
    a, b, new = p.alloc(), p.alloc(), 60
    p.grow([a, b], [3900, 3300])
    k, v = p.begin([a], [new])
    q = p.rows(new, 8)
    graph, first = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(first):
        p.c.append(0, k, v)
        with pytest.raises(KvError, match="workspace"):
            p.c.decode_multi(0, q)
    first.replay()
    want = p.c.decode_multi(0, q).clone()
    p.check_chunk(want, [a], [new], q)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = p.c.decode_multi(0, q)
    kb, vb = p.begin([b], [2 * new])                        # twice the rows
    qb = p.rows(2 * new, 8)
    p.check_chunk(p.c.append_decode_multi(0, kb, vb, qb), [b], [2 * new], qb)
    p.c.truncate(a, 3900)
    p.c.step_begin([a], [new])                              # the captured step again; the rows that truncate cut are gone
    p.c.append(0, k, v)
    for _ in range(2):
        got.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_pending_timeout_leaves_the_output_alone():
    p = Pair(8, 2, 128)
    s = p.alloc()
    p.grow([s], [300])
    k, v = p.begin([s], [40])
    p.c.append(0, k, v)
    q = p.rows(40, 8)
    from titan_engine_b200 import KvError
    for call, rows in ((p.c.decode, 1), (p.c.decode_multi, 40)):
        out = torch.full((rows, 8, 128), 7.0, dtype=torch.bfloat16, device=p.dev)
        p.c.selftest_set_status(4)
        call(0, q[:rows].contiguous(), out)
        with pytest.raises(KvError):
            p.c.device_status()
        assert (out == 7.0).all()
    p.check_chunk(p.c.decode_multi(0, q), [s], [40], q)


def test_same_bits_every_time():
    p = Pair(32, 8, 128, "bf16", pages=600, mpps=300)
    seqs = [p.alloc() for _ in range(3)]
    p.grow(seqs, [2000, 17, 4000])
    k, v = p.begin(seqs, [70, 1, 3])
    q = p.rows(74, 32)
    first = p.c.append_decode_multi(0, k, v, q).clone()
    for _ in range(3):
        assert torch.equal(p.c.decode_multi(0, q), first)
    one = p.c.decode(0, q[:3].contiguous()).clone()
    for _ in range(3):
        assert torch.equal(p.c.decode(0, q[:3].contiguous()), one)
