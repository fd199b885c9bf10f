// int8_prefill.cu — attention for every token of a chunk over an INT8 pool on the 5th-generation tensor cores.
//
// Mathematics: that of int8_decode.cu.  With codes K, V and the scales ks, vs of their rows,
//   x_j = ks_j (q K_j) log2(e)/sqrt(D) + log2(vs_j),   w_j = 2^(x_j - m),   out = sum_j w_j V_j / sum_j w_j / vs_j
// the codes enter the products as fp16 without rounding, w_j <= 2^8 is the only value rounded to 16 bits, sums are FP32,
// a bf16 query row is scaled by a power of two to fit fp16.
//
// One CTA per SM = one tile of 256 (token, head) rows of a (sequence, kv head) x a range of the context, as two halves of
// 128 rows (the lanes of tensor memory) that take turns on the tensor pipe.  Per block of 64 tokens (4 pages):
//   loader warp      one bulk copy per page: the page's tile - codes and scales - is contiguous; 4 stages
//   4 expander warps codes -> fp16 into the 128-byte-swizzled slabs the MMAs read (2 K and 2 V stages), and the three
//                    numbers per token the softmax needs: ks log2(e)/sqrt(D), log2 vs, 1/vs (4 stages)
//   MMA thread       S = Q K^T (M 128, N 64) and O += W V (M 128, N D, W from tensor memory) for both halves
//   16 softmax warps 16 rows each, as fragments: a speculative pass against the current reference, redone when a score exceeds it
//                    by 2^8 or the block is cut; only then O is rescaled (prefill_tc.cu describes the scheme)
// The expansion is what an 8-bit cache costs over a 16-bit one: 2 D values per token - about 800 warp instructions a block of
// some 6200 - shared here by 256 rows where two CTAs of 128 rows would each do it.  Tensor memory: per half two S buffers of
// 64 columns and O of D: all 512 columns at D = 128.
// Bound: a block of 256 rows x 64 tokens at D = 128 is 1024 clocks of the tensor pipe and 1024 of the special-function unit.  It
// takes about 2480: the shared-memory pipe is used by loads and stores for half of them (1337 wavefronts, 768 of which are the
// softmax warps reading the three numbers of each token) and feeds the operands of the MMAs for 41 %; issue slots 63 %, ALU
// 46 %, special-function unit 42 %.  A CTA's start and end take as long as 5 blocks: reading its item, 64 KB of queries (by bulk
// copies, 64 of them, it took longer), the first expansion and the first block's look at the scores, the output's way out.
// Measured: 0.37-0.40 ms for 8 chunks of 1024 tokens on contexts up to 2843 (32 heads, 8 kv heads), 1.13-1.28 ms = 860-970 TFLOP/s
// for a prompt of 8192 (64 heads).
// Every wait is bounded; on expiry the status word is set, nothing is written, and the CTA waits for its copies and frees its
// tensor memory before it returns.  No cluster, no multicast, this GPU's memory only.
#include "int8_cache.cuh"
#include "tk_merge.cuh"
#include "tk_mma.cuh"
#include "tk_tcgen05.cuh"

#include <type_traits>

namespace tk {

namespace {

constexpr int kPfRows = kPrefillRowsInt8;       // 256: two halves of kTcRows
constexpr int kPfBlock = 64;                    // context tokens per block (4 pages)
constexpr int kPfRaw = 4;                       // stages of raw tiles: K is expanded two blocks ahead of V
constexpr int kPfGroups = 1;                    // 16-row groups per softmax warp: 1 (16 warps) 0.403 / 1.165 ms, 2 (8 warps) 0.417 / 1.282
constexpr int kPfSoftWarps = kPfRows / (16 * kPfGroups), kPfExpWarps = 4;
constexpr int kPfMmaWarp = kPfSoftWarps + kPfExpWarps, kPfLoadWarp = kPfMmaWarp + 2;    // an MMA warp for each half
constexpr int kPfThreads = (kPfSoftWarps + 8) * 32;     // 6 warpgroups: 4 of softmax, expanders, (two MMA warps, loader, an idle warp)
constexpr int kPfSoftThreads = kPfSoftWarps * 32;
constexpr int kPfRegsSoft = 96, kPfRegsOther = 48;
constexpr int kPfExpThreads = kPfExpWarps * 32;
constexpr uint32_t kPfTmemCols = 512, kPfHalfCols = 256, kPfColO = 128;   // half h: S at 256h and 256h + 64, O at 256h + 128

template <int D>
struct PfCfg {
    static constexpr int HALVES = D / 64;                   // 64-dim halves of a row: 128 bytes of fp16 each
    static constexpr int TILE = i8_tile_bytes(D);
    static constexpr int Q_BYTES = HALVES * kPfRows * 128;  // [tile half][dim half][128 rows][128 B]
    static constexpr int SLAB = HALVES * kPfBlock * 128;    // K or V of a block: [dim half][64 tokens][128 B]
    static constexpr int HALF = kPfBlock * 128;
    static constexpr int RAW = 4 * TILE;
    static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + 2 * SLAB, OFF_RAW = OFF_V + 2 * SLAB, OFF_SC = OFF_RAW + kPfRaw * RAW,
                         OFF_E = OFF_SC + 4 * 3 * kPfBlock * 4, OFF_PAGES = OFF_E + kPfRows * 4, OFF_BARS = OFF_PAGES + kPrefillMaxPages * 4,
                         SMEM = OFF_BARS + 512 + 1024;
};

// two FP32 values in one 64-bit register
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack_x2(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ f32x2 pack_x2(uint32_t lo, uint32_t hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ float2 unpack_x2(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 fma_x2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 mul_x2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 add_x2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float pf_lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pf_pow2i(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// contiguous copy, global -> this CTA's shared memory; the other tiles of the sequence read the same pages: keep them in L2
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(policy));
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(policy) : "memory");
}

// What an expander thread does to every block: the same 16 columns of every 16th (D = 64: 32nd) row, all addresses constants away
// from `from` and `to`.
template <int D>
struct PfExpander {
    static constexpr int CPR = D / 16, ROWS = kPfExpThreads / CPR;      // 16-code chunks per row, rows per pass
    int et;
    bool swap;
    uint32_t from, to_lo, to_hi;
    __device__ __forceinline__ PfExpander() {
        uint32_t tid;
        asm volatile("mov.u32 %0, %%tid.x;" : "=r"(tid));
        et = (int)tid - kPfSoftWarps * 32;
        const int er = et / CPR, ec = et % CPR;
        from = (uint32_t)((er / kI8Page) * i8_tile_bytes(D) + (er % kI8Page) * D + ec * 16);
        // 16 codes = two 16-byte chunks of the fp16 row.  At D = 128 a quarter warp stores one row: lanes of the second dim half
        // store their chunks in the other order, or both halves would meet in the same banks.
        swap = D == 128 && ec >= 4;
        to_lo = (uint32_t)((ec >> 2) * PfCfg<D>::HALF + er * 128) + (((2 * (ec & 3) + (swap ? 1 : 0)) ^ (er & 7)) << 4);
        to_hi = to_lo ^ 16u;
    }
    __device__ __forceinline__ void operator()(uint32_t raw, int kv, uint32_t slab) const {
#pragma unroll
        for (int i = 0; i < kPfBlock / ROWS; i++) {
            const uint4 w = lds128(raw + from + i * (ROWS / kI8Page) * i8_tile_bytes(D) + i8_row_off(D, kv, 0));
            const uint32_t a0 = swap ? w.z : w.x, a1 = swap ? w.w : w.y, b0 = swap ? w.x : w.z, b1 = swap ? w.y : w.w;
            sts128(slab + to_lo + i * ROWS * 128, make_uint4(i8_expand<0x4140>(a0), i8_expand<0x4342>(a0), i8_expand<0x4140>(a1), i8_expand<0x4342>(a1)));
            sts128(slab + to_hi + i * ROWS * 128, make_uint4(i8_expand<0x4140>(b0), i8_expand<0x4342>(b0), i8_expand<0x4140>(b1), i8_expand<0x4342>(b1)));
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
};

// An item of the work list and where its rows are.  Read at the start of a CTA and again behind its loop over the context: kept,
// these would be a dozen registers that the loop does not have.
struct PfItem {
    int b, chunk, kvh, tile, seq, len, nq, ct, q_base, poff, cbase;
    int tok_first, tok_cnt, p_last;
    bool split;                                             // the tile's context is more than one chunk
    __device__ __forceinline__ PfItem(const PrefillDev& pf, int sh) {
        ld(pf.items + blockIdx.x, b, chunk, kvh, tile);
        ld(pf.info + 2 * blockIdx.x, seq, len, nq, ct);
        int unused;
        ld(pf.info + 2 * blockIdx.x + 1, q_base, poff, cbase, unused);
        tok_first = tile * (kPfRows >> sh);
        tok_cnt = min(nq - tok_first, kPfRows >> sh);
        p_last = len - nq + tok_first + tok_cnt - 1;
        split = p_last >= ct;
    }
    static __device__ __forceinline__ void ld(const int4* p, int& x, int& y, int& z, int& w) {
        asm volatile("ld.global.nc.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(x), "=r"(y), "=r"(z), "=r"(w) : "l"(p));
    }
};

template <int D, bool IO_BF16>
__global__ void __launch_bounds__(kPfThreads, 1)
prefill_int8_kernel(Geometry g, const uint8_t* __restrict__ pool, PrefillDev pf, const int32_t* __restrict__ page_table,
                    const uint16_t* __restrict__ q, void* __restrict__ out, int out_dtype, float* __restrict__ partials,
                    int* __restrict__ counters, int* __restrict__ status, int sh /* log2 of the heads per kv head */) {
    using C = PfCfg<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *s_q = smem, *s_k = smem + C::OFF_K, *s_v = smem + C::OFF_V, *s_raw = smem + C::OFF_RAW;
    float* s_sc = (float*)(smem + C::OFF_SC);               // [4][3][64]: ks log2(e)/sqrt(D), log2 vs, 1/vs
    float* s_e = (float*)(smem + C::OFF_E);                 // [256] power of two of the row's query
    int32_t* s_pages = (int32_t*)(smem + C::OFF_PAGES);
    uint64_t* bars = (uint64_t*)(smem + C::OFF_BARS);
    uint64_t *rawfull = bars, *rawempty = bars + 4, *kfull = bars + 8, *kempty = bars + 10, *vfull = bars + 12, *vempty = bars + 14,
             *bar_s = bars + 16 /* [half][2] */, *p_ready = bars + 20 /* [half][2] */, *bar_o = bars + 24 /* [half] */;
    uint32_t* s_tmem = (uint32_t*)(bars + 26);
    int* s_flag = (int*)(s_tmem + 1);
    uint32_t* s_wmax = (uint32_t*)(bars + 28);              // [16 softmax warps] prologue: largest and smallest query magnitudes

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = 1 << sh;
    const PfItem it(pf, sh);
    const int len = it.len, tok_first = it.tok_first, tok_cnt = it.tok_cnt, kvh = it.kvh, q_base = it.q_base;
    const int halves = tok_cnt * G > kTcRows ? 2 : 1;
    const int base_pos = len - it.nq;
    const int t0 = it.chunk * it.ct, t1 = min(t0 + it.ct, it.p_last + 1);
    const int n_pages = (t1 - t0 + kI8Page - 1) / kI8Page;
    const int n_blocks = (n_pages + 3) / 4;
    const int32_t* pt_row = page_table + (size_t)it.seq * g.max_pages_per_seq + t0 / kI8Page;

    // ---- prologue ----
    constexpr int LPR = D / 8, QV = kPfRows * LPR / kPfSoftThreads;      // 16-byte vectors per query row, per softmax thread
    uint4 qv[QV];
    if (tid < kPfSoftThreads) {
#pragma unroll
        for (int i = 0; i < QV; i++) {
            const int r = (i * kPfSoftThreads + tid) / LPR, c = tid % LPR;
            const size_t row = (size_t)(q_base + tok_first + (r >> sh)) * g.H + (size_t)kvh * G + (r & (G - 1));
            qv[i] = (r >> sh) < tok_cnt ? __ldg(reinterpret_cast<const uint4*>(q + row * D) + c) : make_uint4(0, 0, 0, 0);
        }
    }
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(smem_u32(&kfull[i]), kPfExpWarps); mbar_init(smem_u32(&vfull[i]), kPfExpWarps);
            mbar_init(smem_u32(&kempty[i]), halves); mbar_init(smem_u32(&vempty[i]), halves);
            mbar_init(smem_u32(&bar_o[i]), 1);
        }
        for (int i = 0; i < 4; i++) {
            mbar_init(smem_u32(&bar_s[i]), 2);              // the commit of S and a plain arrival of its MMA warp
            mbar_init(smem_u32(&p_ready[i]), kPfSoftWarps / 2);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kPfMmaWarp) {
        tmem_alloc(smem_u32(s_tmem), kPfTmemCols);
        tmem_relinquish();
    }
    // one copy per page of the block; `pages_of` = the page table itself for the first blocks, its copy in shared memory later
    auto load_block = [&](int blk, const int32_t* pages_of) {
        const int s = blk % kPfRaw, pages = min(4, n_pages - 4 * blk);
        const uint32_t bar = smem_u32(&rawfull[s]);
        if (lane == 0) mbar_expect_tx(bar, pages * C::TILE);
        __syncwarp();
        if (lane < pages)
            bulk_load(smem_u32(s_raw + s * C::RAW + lane * C::TILE), pool + ((size_t)pages_of[4 * blk + lane] * g.Hkv + kvh) * C::TILE, C::TILE, bar);
    };
    if (warp == kPfLoadWarp) {
        if (lane == 0) {
            for (int i = 0; i < kPfRaw; i++) { mbar_init(smem_u32(&rawfull[i]), 1); mbar_init(smem_u32(&rawempty[i]), kPfExpWarps); }
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        asm volatile("bar.arrive 3, %0;" ::"n"(kPfExpThreads + 32) : "memory");      // the expander warps may wait on them
        for (int blk = 0; blk < kPfRaw && blk < n_blocks; blk++) load_block(blk, pt_row);
    }
    for (int i = tid; i < n_pages; i += kPfThreads) s_pages[i] = pt_row[i];

    const uint32_t raw_u = smem_u32(s_raw), k_u = smem_u32(s_k), v_u = smem_u32(s_v);
    // bf16 queries as fp16: the largest element of the tile becomes 2^14 .. 2^15, one power of two 2^e0 for all rows.  Elements
    // below fp16's normal range (2^-14) are off by at most 2^-25, so that every eight of them (a 16-byte vector) whose largest comes
    // to 2^0 or more are as good as FP32.  Where some do not, or where a query reaches 2^15 (`wide`), every row has a power of its
    // own and its scores are multiplied by it: off by at most 2^-39 of the row's largest element then, far below the rounding of
    // the row's sums.
    int e0 = 0;
    bool wide = false;
    auto tile_power = [&]() {                               // from what the softmax warps left
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < kPfSoftWarps; i++) w = __vmaxu2(w, s_wmax[i]);
        const uint32_t m_all = w >> 16, least = 0x8000u - (w & 0xFFFFu);      // bf16 patterns; `least` of the vectors that are not zero
        e0 = m_all ? max((int)(m_all >> 7) - 127 - 14, -100) : 0;
        wide = e0 > 0 || (m_all >> 7) > (least >> 7) + 14;
    };
    bool staged = true;                                     // expander: no wait of the prologue ran out
    if (warp < kPfSoftWarps) {
        if (IO_BF16) {
            uint32_t m = 0, n = 0x7FFFu;                    // largest of all vectors; smallest of those that are not zero, minus 1
#pragma unroll
            for (int i = 0; i < QV; i++) {
                const uint32_t v = i8_absmax8(qv[i]);
                m = max(m, v);
                n = min(n, v - 1u);
            }
            m = __reduce_max_sync(0xFFFFFFFFu, m);
            n = __reduce_min_sync(0xFFFFFFFFu, n);
            if (lane == 0) s_wmax[warp] = m << 16 | (0x7FFFu - n);
            asm volatile("bar.sync 2, %0;" ::"n"(kPfSoftThreads) : "memory");
            tile_power();
        }
#pragma unroll
        for (int i = 0; i < QV; i++) {
            const int r = (i * kPfSoftThreads + tid) / LPR, c = tid % LPR;
            uint4 x = qv[i];
            if (IO_BF16) {
                int e = e0;
                if (wide) {                                 // uniform
                    uint32_t rm = i8_absmax8(x);
#pragma unroll
                    for (int off = LPR / 2; off > 0; off >>= 1) rm = max(rm, __shfl_xor_sync(0xFFFFFFFFu, rm, off));
                    e = rm ? max((int)(rm >> 7) - 127 - 14, -100) : 0;
                    if (c == 0) s_e[r] = pf_pow2i(e);
                }
                const float down = pf_pow2i(-e);
                uint32_t* w = &x.x;
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const float2 f = i8_unpack2<true>(w[u]);
                    w[u] = pack2<false>(f.x * down, f.y * down);
                }
            }
            // 128-byte-swizzled K-major rows: 16-byte chunk c of a row sits at chunk c ^ (row & 7)
            *reinterpret_cast<uint4*>(s_q + ((r / kTcRows) * C::HALVES + (c >> 3)) * (kTcRows * 128) + (r % kTcRows) * 128 +
                                      (((c & 7) ^ (r & 7)) << 4)) = x;
        }
    } else if (warp < kPfMmaWarp) {
        asm volatile("bar.sync 3, %0;" ::"n"(kPfExpThreads + 32) : "memory");
        // meanwhile: the slabs of K(0), K(1) and V(0); the numbers of the tokens follow when the queries' power of two is known
        // (the CTA's first S 1200 clocks earlier)
        const PfExpander<D> expand;
        auto raw_here = [&](int blk) { return mbar_wait_bounded_tight(smem_u32(&rawfull[blk]), 0u, status); };
        staged = __all_sync(0xFFFFFFFFu, raw_here(0));
        if (staged) expand(raw_u, 0, k_u);
        if (staged && n_blocks > 1) {
            staged = __all_sync(0xFFFFFFFFu, raw_here(1));
            if (staged) expand(raw_u + C::RAW, 0, k_u + C::SLAB);
        }
        if (staged) expand(raw_u, 1, v_u);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // generic writes above -> visible to the MMAs
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (IO_BF16) tile_power();
    const uint32_t tmem = *s_tmem;

    bool alive = true;
    constexpr float kLazy = 8.0f;

    // Registers: 768 threads x 80 at launch; 96 for the four softmax warpgroups, 48 for the other two (512 x 96 + 256 x 48 = 61440,
    // what the block was launched with).
    // One arrival per warp, after all its lanes' writes.
    auto warp_arrive = [&](uint64_t* bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(bar));
    };
    // A role other than softmax ends at the barrier that all threads of the CTA meet on, whatever became of it.
    auto leave = [&]() {
        tc_fence_before();
        asm volatile("bar.sync 1, %0;" ::"n"(kPfThreads) : "memory");
    };
    if (warp >= kPfMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPfRegsOther));
    if (warp - kPfMmaWarp < halves) {
        // ===== MMA warps, one per half of the tile: an elected lane feeds the tensor pipe =====
        // (one warp for both halves made each wait for the other's barriers)
        const int half = warp - kPfMmaWarp;
        constexpr uint32_t kIdescS = instr_desc(false, false, kPfBlock), kIdescO = instr_desc(false, true, D);
        const uint64_t dq = smem_desc(smem_u32(s_q + half * C::HALVES * kTcRows * 128), 16), desc_k = smem_desc(smem_u32(s_k), 16),
                       desc_v = smem_desc(smem_u32(s_v), C::HALF);
        const uint32_t at = tmem + half * kPfHalfCols;
        auto await = [&](uint64_t* bar, uint32_t parity) {
            const bool done = __all_sync(0xFFFFFFFFu, mbar_wait_bounded_tight(smem_u32(bar), parity, status));
            tc_fence_after();
            return done;
        };
        auto issue_s = [&](int blk) {                        // S = Q K^T
            const uint64_t dk = desc_k + (uint64_t)(((blk & 1) * C::SLAB) >> 4);
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ks++)
                    tc_mma_ss(at + 64u * (blk & 1), dq + (uint64_t)(((ks >> 2) * (kTcRows * 128) + (ks & 3) * 32) >> 4),
                              dk + (uint64_t)(((ks >> 2) * C::HALF + (ks & 3) * 32) >> 4), kIdescS, ks > 0);
                tc_commit(smem_u32(&bar_s[2 * half + (blk & 1)]));
                mbar_arrive(smem_u32(&bar_s[2 * half + (blk & 1)]));     // passes on what kfull said: the numbers of the block's tokens are there
                tc_commit(smem_u32(&kempty[blk & 1]));
            }
            __syncwarp();
        };
        auto issue_o = [&](int blk) {                        // O += W V, 16 tokens per MMA: 8 columns of W, 16 rows of the V slab
            const uint64_t dv = desc_v + (uint64_t)(((blk & 1) * C::SLAB) >> 4);
            const uint32_t acc = blk > 0 ? 1u : 0u;
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < 4; ks++)
                    tc_mma_ts(at + kPfColO, at + 64u * (blk & 1) + 8 * ks, dv + (uint64_t)((ks * 2048) >> 4), kIdescO, ks > 0 ? 1u : acc);
                tc_commit(smem_u32(&bar_o[half]));
                tc_commit(smem_u32(&vempty[blk & 1]));
            }
            __syncwarp();
        };
        bool ok = true;
        for (int blk = 0; blk < 2 && blk < n_blocks && ok; blk++) {
            ok = await(&kfull[blk], 0u);
            if (ok) issue_s(blk);
        }
        for (int blk = 0; blk < n_blocks && ok; blk++) {
            const int s = blk & 1;
            const uint32_t ph = (uint32_t)((blk >> 1) & 1);
            // W of this block is in tensor memory (and O rescaled): O += W V, then S of the block after next.  The warp's MMAs run in
            // order: S(blk+2) overwrites the columns after W V has read them
            ok = await(&vfull[s], ph) && await(&p_ready[2 * half + s], ph);
            if (!ok) break;
            issue_o(blk);
            if (blk + 2 < n_blocks) {
                ok = await(&kfull[s], ph ^ 1u);
                if (ok) issue_s(blk + 2);
            }
        }
    } else if (warp == kPfLoadWarp) {
        // ===== loader warp (the first kPfRaw blocks left in the prologue) =====
        int issued = min(kPfRaw, n_blocks);
        for (int blk = kPfRaw; blk < n_blocks; blk++) {
            if (!__all_sync(0xFFFFFFFFu, mbar_wait_bounded_tight(smem_u32(&rawempty[blk % kPfRaw]), (uint32_t)((blk / kPfRaw - 1) & 1), status))) break;
            load_block(blk, s_pages);
            issued = blk + 1;
        }
        // no copy of this CTA may be in flight when it returns, whatever became of the other roles
        for (int blk = max(0, issued - kPfRaw); blk < issued; blk++)
            (void)__all_sync(0xFFFFFFFFu, mbar_wait_bounded_tight(smem_u32(&rawfull[blk % kPfRaw]), (uint32_t)((blk / kPfRaw) & 1), status));
    }
    leave();
    if (warp == kPfMmaWarp) tmem_dealloc(tmem, kPfTmemCols); // tensor memory goes back on every path
    return;
    }
    if (warp >= kPfSoftWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPfRegsOther));
        // ===== expander warps: codes -> fp16 slabs =====
        const float sc2E = kLog2e / sqrtf((float)D) * (IO_BF16 && !wide ? pf_pow2i(e0) : 1.0f);
        const PfExpander<D> expand;                          // (again: its registers were not kept over the barrier)
        const int et = expand.et;
        const uint32_t sc_u = smem_u32(s_sc);
        auto numbers = [&](int blk) {
            if (et < kPfBlock) {
                // (the numbers of block blk - 4 are out of use: S of block blk - 2, whose slab was just handed back, was
                // issued after every row's W of block blk - 4)
                const uint32_t t = raw_u + (blk % kPfRaw) * C::RAW + (et / kI8Page) * C::TILE;
                const bool in = t0 + blk * kPfBlock + et < t1;      // behind the range: whatever the page's last owner left
                const float ks = lds32(t + i8_scale_off(D, 0, et % kI8Page)), vs = lds32(t + i8_scale_off(D, 1, et % kI8Page));
                const uint32_t o = sc_u + (((blk & 3) * 3 * kPfBlock + et) << 2);
                sts32(o, in ? ks * sc2E : 0.0f);
                sts32(o + 4 * kPfBlock, in ? pf_lg2(vs) : 0.0f);
                sts32(o + 8 * kPfBlock, in ? __fdividef(1.0f, vs) : 0.0f);
            }
        };
        auto expand_k = [&](int blk) {
            const int s = blk & 1, rs = blk % kPfRaw;
            if (!mbar_wait_bounded_tight(smem_u32(&rawfull[rs]), (uint32_t)((blk / kPfRaw) & 1), status)) return false;
            if (!mbar_wait_bounded_tight(smem_u32(&kempty[s]), (uint32_t)(((blk >> 1) - 1) & 1), status)) return false;
            numbers(blk);
            expand(raw_u + rs * C::RAW, 0, k_u + s * C::SLAB);
            warp_arrive(&kfull[s]);
            return true;
        };
        auto give_v = [&](int blk) {
            warp_arrive(&vfull[blk & 1]);
            if (lane == 0) mbar_arrive(smem_u32(&rawempty[blk % kPfRaw]));
        };
        auto expand_v = [&](int blk) {
            const int s = blk & 1, rs = blk % kPfRaw;
            if (blk >= 2 && !mbar_wait_bounded_tight(smem_u32(&vempty[s]), (uint32_t)(((blk >> 1) - 1) & 1), status)) return false;
            expand(raw_u + rs * C::RAW, 1, v_u + s * C::SLAB);
            give_v(blk);
            return true;
        };
        bool ok = staged;
        if (ok) {                                            // what the prologue has expanded
            for (int blk = 0; blk < 2 && blk < n_blocks; blk++) { numbers(blk); warp_arrive(&kfull[blk]); }
            give_v(0);
        }
        // W V of block i - 2 and S of block i end together: they hand back the slabs of V(i) and K(i + 2), needed in this order
        for (int blk = 0; blk < n_blocks && ok; blk++) ok = (blk == 0 || expand_v(blk)) && (blk + 2 >= n_blocks || expand_k(blk + 2));
        leave();
        return;
    }
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPfRegsSoft));
    if (warp < halves * (kPfSoftWarps / 2)) {
        // ===== softmax warps =====
        // A warp owns 16 rows (tensor-memory lanes; the two that share a 32-lane window, and a scheduler, take a half of it each),
        // as fragments: thread t holds, of rows t/4 and t/4 + 8, the columns 2 (t%4), +1 of every eight.  The numbers of a
        // token are then read once for 16 rows (with a row per thread each would be a broadcast of its own: 192 shared-memory
        // wavefronts per 32 rows and block instead of 48).  Four warps per scheduler, because the pass is a chain of TMEM load,
        // multiply-add, exponential, conversion: with two, of 32 rows each, it took 2200 clocks a block of which the
        // special-function unit worked 1024.
        constexpr int NR = 2 * kPfGroups, WPH = kPfSoftWarps / 2;    // rows per thread, warps per half
        const int half = warp / WPH, quad = lane & 3;
        const int lane0 = (warp & 3) * 32 + (warp % WPH >> 2) * 16;  // first tensor-memory lane of the warp
        const int row0 = half * kTcRows + lane0 + (lane >> 2);       // + 8 rr
        const uint32_t base = tmem + half * kPfHalfCols + ((uint32_t)lane0 << 16);
        float m2[NR];                                        // per row: reference (base 2)
        f32x2 l2[NR];                                        // ... sums over this thread's even and odd columns
        int lim[NR];                                         // positions the row sees
#pragma unroll
        for (int rr = 0; rr < NR; rr++) {
            const int row = row0 + 8 * rr;
            m2[rr] = -1e30f;
            l2[rr] = 0ull;
            // (rows without a token: zero queries, nothing of theirs is written; unmasked, so that they cost no careful pass)
            lim[rr] = (row >> sh) < tok_cnt ? base_pos + tok_first + (row >> sh) + 1 : len;
        }
        const uint32_t e_u = smem_u32(s_e) + 4 * row0;       // the rows' powers of two, 8 rows apart
        auto power = [&](int rr) { const float e = IO_BF16 && wide ? lds32(e_u + 32 * rr) : 1.0f; return pack_x2(e, e); };
        const bool idle = ((row0 - (lane >> 2)) >> sh) >= tok_cnt;   // no row of this warp has a token: whatever W holds, nobody reads its O
        int lim_min = lim[0];
#pragma unroll
        for (int rr = 1; rr < NR; rr++) lim_min = min(lim_min, lim[rr]);
        // blocks that every row of the warp sees whole (none where the rows have powers of two of their own)
        const int n_whole = IO_BF16 && wide ? 0 : (min(__reduce_min_sync(0xFFFFFFFFu, lim_min), t1) - t0) / kPfBlock;
        bool started = false;
        for (int blk = 0; blk < n_blocks; blk++) {
            const int buf = blk & 1;
            const uint32_t col_s = base + 64u * buf;         // S of this block; its first 32 columns become W
            const int tok_base = t0 + blk * kPfBlock;
            const uint32_t sc = smem_u32(s_sc) + (((blk & 3) * 3 * kPfBlock + 2 * quad) << 2);
            const bool ok = mbar_wait_bounded_tight(smem_u32(&bar_s[2 * half + buf]), (uint32_t)((blk >> 1) & 1), status);
            if (!__all_sync(0xFFFFFFFFu, ok)) { alive = false; break; }
            tc_fence_after();
            bool rescale = false;
            float alpha[NR];
            if (!idle) {
                // The weights of the block against the current references, 16 columns of S at a time, the next 16 on their way; S
                // stays in tensor memory until W goes over it.  -> false, with nothing changed, where `check` is set and a score exceeds
                // its row's reference by more than 2^kLazy.
                auto weigh = [&](auto masked, bool check) -> bool {
                    constexpr bool M = decltype(masked)::value;
                    uint32_t pr[kPfGroups][16];              // W of the rows as 16x128b fragments
                    f32x2 nm[NR], tl[NR];                    // tl: the block's share of the sums
                    float top = -1e30f;
#pragma unroll
                    for (int rr = 0; rr < NR; rr++) { tl[rr] = 0ull; nm[rr] = pack_x2(-m2[rr], -m2[rr]); }
                    f32x2 E[NR];
                    int nv[NR];                              // of a row: tokens of the block it sees, from this thread's first column on
#pragma unroll
                    for (int rr = 0; rr < NR; rr++)
                        if (M) { E[rr] = power(rr); nv[rr] = min(lim[rr], t1) - tok_base - 2 * quad; }
                    f32x2 sr[2][kPfGroups][4];
#pragma unroll
                    for (int gi = 0; gi < kPfGroups; gi++) tmem_ld_frag16(col_s + ((uint32_t)(16 * gi) << 16), sr[0][gi]);
#pragma unroll
                    for (int qt = 0; qt < 4; qt++) {
#pragma unroll
                        for (int gi = 0; gi < kPfGroups; gi++) tc_wait_ld_frag16(sr[qt & 1][gi]);
                        if (qt < 3) {
#pragma unroll
                            for (int gi = 0; gi < kPfGroups; gi++) tmem_ld_frag16(col_s + 16 * (qt + 1) + ((uint32_t)(16 * gi) << 16), sr[(qt + 1) & 1][gi]);
                        }
#pragma unroll
                        for (int k = 0; k < 2; k++) {        // tokens 16 qt + 8 k + 2 quad, +1
                            const int t = 16 * qt + 8 * k;
                            const f32x2 ks = lds64(sc + 4 * t), lv = lds64(sc + 4 * (kPfBlock + t)), iv = lds64(sc + 4 * (2 * kPfBlock + t));
#pragma unroll
                            for (int rr = 0; rr < NR; rr++) {
                                const f32x2 a = sr[qt & 1][rr >> 1][2 * k + (rr & 1)];
                                const f32x2 u = add_x2(lv, nm[rr]);
                                float2 x = unpack_x2(M ? fma_x2(mul_x2(a, ks), E[rr], u) : fma_x2(a, ks, u));
                                if (M) {                     // (also where the scale of a token the row does not see is a NaN)
                                    x.x = t < nv[rr] ? x.x : -INFINITY;
                                    x.y = t + 1 < nv[rr] ? x.y : -INFINITY;
                                }
                                top = fmaxf(top, fmaxf(x.x, x.y));
                                const float w0 = ex2(x.x), w1 = ex2(x.y);
                                if (M) {
                                    const float2 ivf = unpack_x2(iv);
                                    tl[rr] = add_x2(tl[rr], pack_x2(t < nv[rr] ? w0 * ivf.x : 0.0f, t + 1 < nv[rr] ? w1 * ivf.y : 0.0f));
                                } else {
                                    tl[rr] = fma_x2(pack_x2(w0, w1), iv, tl[rr]);
                                }
                                pr[rr >> 1][4 * qt + 2 * k + (rr & 1)] = pack2<false>(w0, w1);
                            }
                        }
                    }
                    if (__any_sync(0xFFFFFFFFu, top > kLazy) && check) return false;
#pragma unroll
                    for (int rr = 0; rr < NR; rr++) l2[rr] = add_x2(l2[rr], tl[rr]);
#pragma unroll
                    for (int gi = 0; gi < kPfGroups; gi++) tmem_st_half32(col_s + ((uint32_t)(16 * gi) << 16), pr[gi]);     // W over the columns S was read from
                    return true;
                };
                // speculating that the references stay; a row without one (its first block, or none of it seen so far) has to look first
                bool look = !started;
                if (!look) look = !(blk < n_whole ? weigh(std::false_type{}, true) : weigh(std::true_type{}, true));
                if (look) {                                  // new references for the rows that need one, then the weights
                    float mx[NR];
                    f32x2 E[NR];
                    int nv[NR];
#pragma unroll
                    for (int rr = 0; rr < NR; rr++) { mx[rr] = -INFINITY; E[rr] = power(rr); alpha[rr] = 1.0f; nv[rr] = min(lim[rr], t1) - tok_base - 2 * quad; }
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int gi = 0; gi < kPfGroups; gi++) {
                            uint32_t sf[16];
                            tmem_ld_frag32(col_s + 32 * h + ((uint32_t)(16 * gi) << 16), sf);
                            tc_wait_ld16(sf);
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const int t = 32 * h + 8 * k;
                                const f32x2 ks = lds64(sc + 4 * t), lv = lds64(sc + 4 * (kPfBlock + t));
#pragma unroll
                                for (int hh = 0; hh < 2; hh++) {
                                    const int rr = 2 * gi + hh;
                                    const float2 x = unpack_x2(fma_x2(mul_x2(pack_x2(sf[4 * k + 2 * hh], sf[4 * k + 2 * hh + 1]), ks), E[rr], lv));
                                    mx[rr] = fmaxf(mx[rr], t < nv[rr] ? x.x : -INFINITY);
                                    mx[rr] = fmaxf(mx[rr], t + 1 < nv[rr] ? x.y : -INFINITY);
                                }
                            }
                        }
                    started = true;
#pragma unroll
                    for (int rr = 0; rr < NR; rr++) {         // the four threads of a row agree
                        mx[rr] = fmaxf(mx[rr], __shfl_xor_sync(0xFFFFFFFFu, mx[rr], 1));
                        mx[rr] = fmaxf(mx[rr], __shfl_xor_sync(0xFFFFFFFFu, mx[rr], 2));
                        if (mx[rr] > m2[rr] + kLazy) {
                            alpha[rr] = ex2(m2[rr] - mx[rr]);    // a row's first block: 0
                            m2[rr] = mx[rr];
                            rescale = true;
                        }
                        started = started && m2[rr] > -1e29f;
                        l2[rr] = mul_x2(l2[rr], pack_x2(alpha[rr], alpha[rr]));
                    }
                    started = __all_sync(0xFFFFFFFFu, started);
                    rescale = __any_sync(0xFFFFFFFFu, rescale);
                    (void)weigh(std::true_type{}, false);
                }
            }
            // O += W V of the previous block must be done before O is rescaled.  S of this block was committed behind W V of
            // block blk-2, so the barrier's phase is blk-1 or later; the last block waits in any case, so that the wait after
            // the loop cannot meet a barrier that is two phases away
            if (blk > 0 && (rescale || blk == n_blocks - 1)) {
                if (!__all_sync(0xFFFFFFFFu, mbar_wait_bounded_tight(smem_u32(&bar_o[half]), (uint32_t)((blk - 1) & 1), status))) { alive = false; break; }
                tc_fence_after();
                if (rescale) {
#pragma unroll
                    for (int part = 0; part < D / 32; part++)
#pragma unroll
                        for (int gi = 0; gi < kPfGroups; gi++) {
                            uint32_t of[16];
                            const uint32_t at = base + kPfColO + 32 * part + ((uint32_t)(16 * gi) << 16);
                            tmem_ld_frag32(at, of);
                            tc_wait_ld16(of);
#pragma unroll
                            for (int c = 0; c < 16; c++) of[c] = __float_as_uint(__uint_as_float(of[c]) * alpha[2 * gi + ((c >> 1) & 1)]);
                            tmem_st_frag32(at, of);
                        }
                }
            }
            tc_wait_st();
            tc_fence_before();
            warp_arrive(&p_ready[2 * half + buf]);           // these rows' W (and O) are ready for the tensor pipe
        }
        if (alive && !__all_sync(0xFFFFFFFFu, mbar_wait_bounded_tight(smem_u32(&bar_o[half]), (uint32_t)((n_blocks - 1) & 1), status))) alive = false;
        tc_fence_after();

        const bool poisoned = __any_sync(0xFFFFFFFFu, !alive || __ldcg(status) != 0);   // fail closed, whole warps at a time
        if (!poisoned && !idle) {
            const PfItem it(pf, sh);
            float f[NR];
            float* prow[NR];
            size_t qo[NR];
            bool valid[NR];
#pragma unroll
            for (int rr = 0; rr < NR; rr++) {
                const float2 lf = unpack_x2(l2[rr]);
                float l = lf.x + lf.y;
                l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
                l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
                const int row = row0 + 8 * rr, tok = it.tok_first + (row >> sh), head = it.kvh * G + (row & (G - 1));
                valid[rr] = (row >> sh) < it.tok_cnt;
                qo[rr] = ((size_t)(it.q_base + tok) * g.H + head) * D;
                prow[rr] = nullptr;
                f[rr] = l == 0.0f ? 0.0f : 1.0f / l;         // l counts weights over value scales: at least one term of any size
                if (it.split) {                                 // (o, m, l) of this chunk, brought to l in [1, 2)
                    prow[rr] = partials + (size_t)it.poff * g.H * (D + 2) + partial_off(it.chunk, tok * g.H + head, it.nq * g.H, D);
                    const uint32_t ex = (__float_as_uint(l) >> 23) & 0xFFu;
                    const int k = ex == 0 || ex >= 254 ? 0 : (int)ex - 127;
                    f[rr] = pf_pow2i(-k);
                    if (valid[rr] && quad == 0)
                        *reinterpret_cast<float2*>(prow[rr] + D) = make_float2(l == 0.0f ? -1e30f : (m2[rr] + (float)k) * 0.6931471805599453f, l * f[rr]);
                }
            }
            // 16-bit rows go through shared memory, where this warp's query rows were (every product of its half is done), and leave
            // as 16 bytes per lane; written from the fragments, four bytes per lane, they took 4000 clocks per tile
            const bool staged_out = !it.split && out_dtype != DT_FP32;
            const uint32_t s_o = smem_u32(s_q + half * C::HALVES * kTcRows * 128);
#pragma unroll
            for (int part = 0; part < D / 32; part++)
#pragma unroll
                for (int gi = 0; gi < kPfGroups; gi++) {
                    uint32_t of[16];
                    tmem_ld_frag32(base + kPfColO + 32 * part + ((uint32_t)(16 * gi) << 16), of);
                    tc_wait_ld16(of);
#pragma unroll
                    for (int hh = 0; hh < 2; hh++) {
                        const int rr = 2 * gi + hh, row = lane0 + (lane >> 2) + 8 * rr;
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const float o0 = __uint_as_float(of[4 * k + 2 * hh]) * f[rr], o1 = __uint_as_float(of[4 * k + 2 * hh + 1]) * f[rr];
                            const int c = 32 * part + 8 * k + 2 * quad;
                            if (staged_out)      sts32(s_o + (c >> 6) * (kTcRows * 128) + row * 128 + ((((c >> 3) & 7) ^ (row & 7)) << 4) + 4 * quad,
                                                       __uint_as_float(pack2<IO_BF16>(o0, o1)));
                            else if (!valid[rr]) continue;
                            else if (it.split)      *reinterpret_cast<float2*>(prow[rr] + c) = make_float2(o0, o1);
                            else                 *reinterpret_cast<float2*>((float*)out + qo[rr] + c) = make_float2(o0, o1);
                        }
                    }
                }
            if (staged_out) {
                __syncwarp();
                constexpr int LPO = D / 8;                   // lanes per row
#pragma unroll
                for (int i = 0; i < 16 * kPfGroups * LPO / 32; i++) {
                    const int r = lane0 + (i * 32 + lane) / LPO, c = lane % LPO, row = half * kTcRows + r;
                    if ((row >> sh) >= it.tok_cnt) continue;
                    const uint4 x = lds128(s_o + (c >> 3) * (kTcRows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
                    *reinterpret_cast<uint4*>((uint16_t*)out + ((size_t)(it.q_base + it.tok_first + (row >> sh)) * g.H + it.kvh * G + (row & (G - 1))) * D + c * 8) = x;
                }
            }
        }
    }

    leave();
    const PfItem fin(pf, sh);
    if (!fin.split) return;
    const int n_chunks = fin.p_last / fin.ct + 1;
    // the CTA that arrives last for the tile merges its chunks (nothing is written while the status word is set)
    if (tid == 0) {
        __threadfence();
        const int tiles = (fin.nq + (kPfRows >> sh) - 1) / (kPfRows >> sh);
        int* c = counters + fin.cbase + fin.kvh * tiles + fin.tile;
        const int last = atomicAdd(c, 1) == n_chunks - 1;
        if (last) *c = 0;
        *s_flag = last;
    }
    asm volatile("bar.sync 2, %0;" ::"n"(kPfSoftThreads) : "memory");
    if (!*s_flag) return;
    __threadfence();                                        // see the other CTAs' rows
    if (__ldcg(status) != 0) return;
    const int rows = G * fin.tok_cnt;
    const size_t chunk_stride = (size_t)fin.nq * g.H * (D + 2);
    const float* region = partials + (size_t)fin.poff * g.H * (D + 2);
    auto column = [&](int row) { return (size_t)(fin.tok_first + (row >> sh)) * g.H + fin.kvh * G + (row & (G - 1)); };
    if (rows * n_chunks * 4 > C::OFF_BARS) {                // (more weights than shared memory)
        const MergeOut mo{nullptr, out, nullptr, out_dtype, nullptr, status};
        merge_rows(g, mo, fin.b, fin.kvh, G, 0, n_chunks, region, MergeMap{rows, fin.nq * g.H, fin.q_base + fin.tok_first, fin.tok_first, 0}, kPfSoftWarps);
        return;
    }
    // The merge of tk_merge.cuh for all rows at once (row after row its chain of L2 loads took 22 us for 256 rows): a thread per row
    // for the weights, then every thread its columns of eight rows with the loads of four chunks in flight.
    float* s_w = reinterpret_cast<float*>(smem);            // [rows][n_chunks] weight times the row's normaliser
    if (tid < rows) {
        const float* ml = region + column(tid) * (D + 2) + D;
        float M = -1e30f, L = 0.0f;
        for (int r = 0; r < n_chunks; r++) {
            const float2 c = __ldcg(reinterpret_cast<const float2*>(ml + r * chunk_stride));
            const float mn = fmaxf(M, c.x);
            L = L * expf(M - mn) + c.y * expf(c.x - mn);
            M = mn;
            s_w[tid * n_chunks + r] = c.x;
        }
        const float inv = 1.0f / (L + 1e-8f);
        for (int r = 0; r < n_chunks; r++) s_w[tid * n_chunks + r] = expf(s_w[tid * n_chunks + r] - M) * inv;
    }
    asm volatile("bar.sync 2, %0;" ::"n"(kPfSoftThreads) : "memory");
    constexpr int U = 8, R = 4, PER = kPfSoftThreads / (D / 2);     // rows a pass of all threads covers
    const int d = 2 * (tid % (D / 2));
    for (int row_a = tid / (D / 2); row_a < rows; row_a += U * PER) {
        float2 acc[U];
#pragma unroll
        for (int u = 0; u < U; u++) acc[u] = make_float2(0.0f, 0.0f);
        for (int rb = 0; rb < n_chunks; rb += R) {
            float2 x[R][U];
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int u = 0; u < U; u++)
                    x[r][u] = rb + r < n_chunks && row_a + u * PER < rows
                                  ? __ldcg(reinterpret_cast<const float2*>(region + column(row_a + u * PER) * (D + 2) + d + (rb + r) * chunk_stride))
                                  : make_float2(0.0f, 0.0f);
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (rb + r < n_chunks && row_a + u * PER < rows) {
                        const float w = s_w[(row_a + u * PER) * n_chunks + rb + r];
                        acc[u].x += x[r][u].x * w;
                        acc[u].y += x[r][u].y * w;
                    }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int row = row_a + u * PER;
            if (row >= rows) break;
            const size_t at = ((size_t)(fin.q_base + fin.tok_first + (row >> sh)) * g.H + fin.kvh * G + (row & (G - 1))) * D + d;
            if (out_dtype == DT_FP32) *reinterpret_cast<float2*>((float*)out + at) = acc[u];
            else                      *reinterpret_cast<uint32_t*>((uint16_t*)out + at) = pack2<IO_BF16>(acc[u].x, acc[u].y);
        }
    }
}

template <int D, bool IO_BF16>
cudaError_t launch_d(const Geometry& g, const LayerPtrs& lp, const PrefillDev& pf, const int32_t* page_table, const void* q, void* out,
                     int out_dtype, float* partials, int* counters, int* status, cudaStream_t s) {
    auto kern = prefill_int8_kernel<D, IO_BF16>;
    int sh = 0;                                             // the planner lays out these items for powers of two only
    while (g.Hkv << sh < g.H) sh++;
    if (g.Hkv << sh != g.H || sh > 7) return cudaErrorInvalidValue;
    static bool attr_done[64] = {};                         // per instantiation and device
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, PfCfg<D>::SMEM);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    kern<<<pf.n_items, kPfThreads, PfCfg<D>::SMEM, s>>>(g, (const uint8_t*)lp.pool, pf, page_table, (const uint16_t*)q, out, out_dtype, partials,
                                                        counters, status, sh);
    return cudaGetLastError();
}

}  // namespace

// Work list, counters and split regions as for launch_prefill_mma, laid out for tiles of kPrefillRowsInt8 rows.
cudaError_t launch_prefill_int8(const Geometry& g, const LayerPtrs& lp, const PrefillDev& pf, const int32_t* page_table, const void* q,
                                void* out, int out_dtype, float* partials, int* counters, int* status, cudaStream_t s) {
    if (pf.n_items <= 0) return cudaSuccess;
    if (out_dtype != DT_FP32 && out_dtype != g.io_dtype) return cudaErrorInvalidValue;
    if (g.io_dtype == DT_BF16) return g.D == 128 ? launch_d<128, true>(g, lp, pf, page_table, q, out, out_dtype, partials, counters, status, s)
                                                 : launch_d<64, true>(g, lp, pf, page_table, q, out, out_dtype, partials, counters, status, s);
    return g.D == 128 ? launch_d<128, false>(g, lp, pf, page_table, q, out, out_dtype, partials, counters, status, s)
                      : launch_d<64, false>(g, lp, pf, page_table, q, out, out_dtype, partials, counters, status, s);
}

}  // namespace tk
