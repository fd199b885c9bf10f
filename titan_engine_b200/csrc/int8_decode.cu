// int8_decode.cu — attention over an INT8 pool for one token per sequence, or for a few tokens of a sequence together:
// TMA-staged tiles, tensor-core products on the codes, online softmax, split-KV partials.
//
// Mathematics.  With k_j = ks_j K_j and v_j = vs_j V_j (codes K, V, one scale per token),
//   x_j = ks_j (q K_j) log2(e)/sqrt(D) + log2(vs_j),   w_j = 2^(x_j - m),   out = sum_j w_j V_j / sum_j w_j / vs_j
// The products run on the codes themselves, expanded to fp16 without rounding; the scale of a key multiplies its score in
// FP32 and the scale of a value enters the EXPONENT, so that the only quantity that is rounded to 16 bits, w_j, is at
// most 2^4 for every magnitude of the values (a probability times a small scale would fall among fp16's
// subnormals).  m is the running reference, moved when some x_j exceeds it by 4.  Sums are FP32.  A row's (o, m, l) is
// brought to l in [1, 2) before it leaves the CTA, so that the rows merge like those of any other pool (tk_merge.cuh).
// bf16 queries are scaled by a power of two per (token, head) to fit fp16: exact down to 2^-28 of the largest element.
//
// Schedule.  As decode_mma.cu's FP8 form: one CTA per (sequence, kv head, chunk of pages), each of 4 warps owning every
// 4th page and a ring of TMA stages of its own; both products transposed (S^T = K Q^T, O^T = V^T W^T) so that tokens and
// dims fill the 16 rows of m16n8k16 and 8 (token, head) pairs its columns; NB column blocks share one expansion of
// the codes.  A tile brings its scales along (int8_cache.cuh): one TMA box per page.  On decode steps the warp that holds
// the last page quantises the new token into shared memory and into the pool: no append launch.
// Bound: HBM (D + 4 bytes per token and kv head for K and for V).  Measured at D = 128: 32 sequences of 32768 tokens, 64 heads
// on 8: 337-390 us = 5.7-6.6 TB/s (issue slots 60 %, tensor pipe 18 %); 64 sequences of 1024-8192, 32 heads: 101-108 us, of which
// about 10 are the launch's start and drain; one sequence of 65536 tokens: 39 us, where starting and merging are a third.
#include "int8_cache.cuh"
#include "tk_merge.cuh"
#include "tk_mma.cuh"

namespace tk {

namespace {

// One column block (128 registers) leaves room for 4 CTAs per SM, two (168) for 3; the stages share out the shared memory.  Measured
// at D = 128, one block: 2 stages x 4 CTAs 364 us, 3 x 3 377, 4 x 2 438 (32 sequences of 32768 tokens, 64 heads); two blocks:
// 3 x 3 168 us, 2 x 4 (spilling) 175 (64 sequences, 4 tokens each; with the queries' fragments in shared memory 2 x 4 is 1 % faster than 3 x 3,
// less than it adds).
template <int D, int NB>
struct I8Cfg {
    static constexpr int CTAS = NB == 1 ? 4 : 3;
    static constexpr int STAGES = D == 64 ? 4 : NB == 1 ? 2 : 3;
    static constexpr int TILE = i8_tile_bytes(D);
    static constexpr int LINES = TILE / 128;                // the tile as lines of 128 bytes: one TMA box
    static constexpr int STAGE = (TILE + 1023) / 1024 * 1024;   // the 128-byte swizzle repeats every 1024 bytes
    static constexpr int SMEM = kWarps * STAGES * STAGE + 1024 + 256;
    static constexpr int SCALES = 2 * kI8Page * D;          // byte offset of the scale line; its line number is a multiple of 8: not swizzled
};

constexpr int kMergeCells = 3000;           // (row, chunk) pairs whose (m, l) fit the shared memory of the smallest configuration

// byte offset inside a stage of 16-byte chunk c of code row r (K rows 0-15, V rows 16-31), under the swizzle
template <int D>
__device__ __forceinline__ uint32_t i8_swz(int r, int c) {
    if (D == 128) return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
    return (uint32_t)((r >> 1) * 128 + (((((r & 1) << 2) + c) ^ ((r >> 1) & 7)) << 4));
}

__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

template <int D, bool IO_BF16, int NB>
__global__ void __launch_bounds__(kWarps * 32, I8Cfg<D, NB>::CTAS)
decode_int8_kernel(const __grid_constant__ CUtensorMap tmap, Geometry g, uint8_t* __restrict__ pool, StepDev st,
                   const int32_t* __restrict__ page_table, const uint16_t* __restrict__ q, float* __restrict__ partials,
                   int* __restrict__ status, MergeOut mo, FuseAppend fa, int multi) {
    using C = I8Cfg<D, NB>;
    constexpr int KS = D / 16, kI8Stages = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = (uint64_t*)(smem + kWarps * kI8Stages * C::STAGE);
    int* s_flag = (int*)(bars + kWarps * kI8Stages);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int gr = lane >> 2, j = lane & 3;
    const int G = g.H / g.Hkv;

    // the next layer's launch may start beside this one's last wave (decode_mma.cu says what it may touch before pdl_wait)
    pdl_launch_dependents();
    const int4 it = st.items[blockIdx.x];
    const int b = it.x, chunk = it.y, kvh = it.z;
    const int seq = st.seq[b], len = st.len[b];
    const int nq = multi ? st.nq[b] : 1;                    // query tokens: token t sees positions < len - nq + t + 1
    const int rows = G * nq;                                // columns of the products that carry data (<= 8 NB)
    const int q_row0 = multi ? st.q_base[b] : b;
    const int t0 = chunk * st.chunk_tokens, t1 = min(len, t0 + st.chunk_tokens);
    const int n_pages = t1 > t0 ? (t1 - t0 + kPage - 1) / kPage : 0;
    const int lp0 = t0 / kPage;
    const int n_w = n_pages > warp ? (n_pages - warp + kWarps - 1) / kWarps : 0;     // pages of this warp (<= 32)
    const int new_tok = fa.k != nullptr ? st.new_tok[b] : -1;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kWarps * kI8Stages; i++) mbar_init(smem_u32(&bars[i]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    int my_page = 0;                                        // lane i keeps the warp's i-th page
    if (lane < n_w) my_page = page_table[(size_t)seq * g.max_pages_per_seq + lp0 + warp + kWarps * lane];
    uint8_t* wstage = smem + (size_t)warp * kI8Stages * C::STAGE;
    auto issue = [&](int i) {
        const int page = __shfl_sync(0xFFFFFFFFu, my_page, i);
        if (lane == 0) {
            const uint32_t bar = smem_u32(&bars[warp * kI8Stages + i % kI8Stages]);
            mbar_expect_tx(bar, C::TILE);
            tma_load_2d(smem_u32(wstage + (size_t)(i % kI8Stages) * C::STAGE), &tmap, 0, (page * g.Hkv + kvh) * C::LINES, bar);
        }
    };
    for (int i = 0; i < kI8Stages && i < n_w; i++) issue(i);

    // Q^T as the B operand: column 8 nb + gr = (token, head) pair; k index (2j, 2j+1) <-> dims 16kk + 4j, +1 and
    // (2j+8, 2j+9) <-> dims 16kk + 4j + 2, +3, the order in which a lane's four code bytes arrive
    uint32_t qb[NB][KS][2];
    float f0[NB], f1[NB];                                   // log2(e)/sqrt(D) x 2^e for this lane's accumulator columns 2j, 2j+1
    int lim0[NB], lim1[NB];                                 // positions they see
    const float sc2 = kLog2e / sqrtf((float)D);
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        const int col = 8 * nb + gr;
        const bool on = col < rows;
        const uint16_t* qrow = q + ((size_t)(q_row0 + (on ? col / G : 0)) * g.H + (size_t)kvh * G + (on ? col % G : 0)) * D;
        int e = 0;
#pragma unroll
        for (int kk = 0; kk < KS; kk++) {
            const uint2 x = on ? *reinterpret_cast<const uint2*>(qrow + 16 * kk + 4 * j) : make_uint2(0, 0);
            qb[nb][kk][0] = x.x; qb[nb][kk][1] = x.y;
            if (!IO_BF16 && fa.rope_tab) {
                const float2* tab = fa.rope_tab + (size_t)b * (D / 2);
                qb[nb][kk][0] = rope_pair<false>(x.x, tab, 16 * kk + 4 * j);
                qb[nb][kk][1] = rope_pair<false>(x.y, tab, 16 * kk + 4 * j + 2);
            }
            if (IO_BF16 && fa.rope_tab) {
                const float2* tab = fa.rope_tab + (size_t)b * (D / 2);
                qb[nb][kk][0] = rope_pair<true>(x.x, tab, 16 * kk + 4 * j);
                qb[nb][kk][1] = rope_pair<true>(x.y, tab, 16 * kk + 4 * j + 2);
            }
        }
        if (IO_BF16) {
            uint32_t m = 0;                                 // largest magnitude of the row: its bf16 pattern
#pragma unroll
            for (int kk = 0; kk < KS; kk++) m = __vmaxu2(m, __vmaxu2(qb[nb][kk][0] & 0x7FFF7FFFu, qb[nb][kk][1] & 0x7FFF7FFFu));
            m = max(m & 0xFFFFu, m >> 16);
            m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
            m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
            e = m ? max((int)(m >> 7) - 127 - 14, -100) : 0;    // the largest element becomes 2^14 .. 2^15
            const float down = pow2i(-e);
#pragma unroll
            for (int kk = 0; kk < KS; kk++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float2 v = i8_unpack2<true>(qb[nb][kk][i]);
                    qb[nb][kk][i] = pack2<false>(v.x * down, v.y * down);
                }
        }
        const float up = sc2 * pow2i(e);
        f0[nb] = __shfl_sync(0xFFFFFFFFu, up, 8 * j);       // column 2j is held by lanes 8j .. 8j+3
        f1[nb] = __shfl_sync(0xFFFFFFFFu, up, 8 * j + 4);
        const int c0 = 8 * nb + 2 * j, c1 = c0 + 1;
        lim0[nb] = c0 < rows ? len - nq + c0 / G + 1 : 0;
        lim1[nb] = c1 < rows ? len - nq + c1 / G + 1 : 0;
    }

    // o[nb][2c] / [2c+1]: even / odd dims of 32-dim chunk c; element [0],[1] = (dim 32c + 2gr (+1), columns 2j, 2j+1),
    // [2],[3] = (dim 32c + 16 + 2gr (+1), the same columns).  m in base-2 units, l over this lane's tokens only.
    constexpr int NT = D / 16;
    float o[NB][NT][4], m0[NB], m1[NB], l0[NB], l1[NB];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        m0[nb] = m1[nb] = -1e30f;
        l0[nb] = l1[nb] = 0.0f;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) o[nb][nt][0] = o[nb][nt][1] = o[nb][nt][2] = o[nb][nt][3] = 0.0f;
    }
    const int sure = multi ? len - nq + 1 : len;            // positions that every column sees

    for (int i = 0; i < n_w; i++) {
        const int s = i % kI8Stages;
        // warp-uniform verdict; a wait that gave up has set the status word and no output is written
        if (!__all_sync(0xFFFFFFFFu, mbar_wait_bounded(smem_u32(&bars[warp * kI8Stages + s]), (uint32_t)((i / kI8Stages) & 1), status))) {
            // (no copy of this warp may land after the CTA is gone: wait, with the same limit, for those behind the one that is late)
            for (int f = i; f < min(i + kI8Stages, n_w); f++)
                (void)mbar_wait_bounded(smem_u32(&bars[warp * kI8Stages + f % kI8Stages]), (uint32_t)((f / kI8Stages) & 1), status);
            break;
        }
        uint8_t* stg = wstage + (size_t)s * C::STAGE;
        const uint32_t stg_u = smem_u32(stg);
        const int tok_base = (lp0 + warp + kWarps * i) * kPage;

        if (new_tok >= 0 && tok_base == ((len - 1) & ~(kPage - 1))) {
            // this page takes the token the step appends: D/8 lanes hold its K row, the next D/8 its V row
            constexpr int L8 = D / 8;
            const int r = (len - 1) & (kPage - 1), kv = (lane / L8) & 1, c = lane % L8;
            const int page = __shfl_sync(0xFFFFFFFFu, my_page, i);
            uint4 x = *reinterpret_cast<const uint4*>((const uint16_t*)(kv ? fa.v : fa.k) + ((size_t)new_tok * g.Hkv + kvh) * D + c * 8);
            if (fa.rope_tab && kv == 0) {
                const float2* tab = fa.rope_tab + (size_t)b * (D / 2);
                x.x = rope_pair<IO_BF16>(x.x, tab, c * 8 + 0);
                x.y = rope_pair<IO_BF16>(x.y, tab, c * 8 + 2);
                x.z = rope_pair<IO_BF16>(x.z, tab, c * 8 + 4);
                x.w = rope_pair<IO_BF16>(x.w, tab, c * 8 + 6);
            }
            uint32_t m = i8_absmax8(x);
#pragma unroll
            for (int off = L8 / 2; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, off));
            const I8Row row = i8_row(i8_amax_value<IO_BF16>(m));
            const uint2 codes = i8_codes8<IO_BF16, true>(x, row.to_code);
            if (lane < 2 * L8) {
                uint8_t* tile = pool + ((size_t)page * g.Hkv + kvh) * C::TILE;
                *reinterpret_cast<uint2*>(stg + i8_swz<D>(kv * kPage + r, c >> 1) + 8 * (c & 1)) = codes;
                *reinterpret_cast<uint2*>(tile + i8_row_off(D, kv, r) + c * 8) = codes;
                if (c == 0) {
                    *reinterpret_cast<float*>(stg + i8_scale_off(D, kv, r)) = row.scale;
                    *reinterpret_cast<float*>(tile + i8_scale_off(D, kv, r)) = row.scale;
                }
            }
            __syncwarp();
        }

        // scales of this lane's tokens gr and gr + 8
        const float* sc = reinterpret_cast<const float*>(stg + C::SCALES);
        float ks0 = sc[gr], ks1 = sc[gr + 8], vs0 = sc[16 + gr], vs1 = sc[24 + gr];

        // ---- S^T = K Q^T ----
        float sT[NB][4], uT[NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; nb++) sT[nb][0] = sT[nb][1] = sT[nb][2] = sT[nb][3] = uT[nb][0] = uT[nb][1] = uT[nb][2] = uT[nb][3] = 0.0f;
        const int mi = lane >> 3;                           // matrix this lane addresses: token half mi & 1, 16-dim chunk mi >> 1
        {
            const int row = ((mi & 1) << 3) + (lane & 7);
#pragma unroll
            for (int cp = 0; cp < D / 32; cp++) {
                uint32_t r0, r1, r2, r3;
                ldsm_x4(stg_u + i8_swz<D>(row, 2 * cp + (mi >> 1)), r0, r1, r2, r3);
                const uint32_t a0[4] = {i8_expand<0x4140>(r0), i8_expand<0x4140>(r1), i8_expand<0x4342>(r0), i8_expand<0x4342>(r1)};
                const uint32_t a1[4] = {i8_expand<0x4140>(r2), i8_expand<0x4140>(r3), i8_expand<0x4342>(r2), i8_expand<0x4342>(r3)};
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    mma16816<false>(sT[nb], a0, qb[nb][2 * cp][0], qb[nb][2 * cp][1]);
                    mma16816<false>(uT[nb], a1, qb[nb][2 * cp + 1][0], qb[nb][2 * cp + 1][1]);
                }
            }
        }
        // ---- weights: this lane has tokens gr ([0],[1]) and gr + 8 ([2],[3]) of columns 2j ([0],[2]) and 2j+1 ([1],[3]) ----
        const bool cut = tok_base + kPage > min(t1, sure);
        if (cut) {                                          // scales behind the sequence are whatever the page's last owner left
            if (tok_base + gr >= t1) { ks0 = 0.0f; vs0 = 1.0f; }
            if (tok_base + gr + 8 >= t1) { ks1 = 0.0f; vs1 = 1.0f; }
        }
        const float lv0 = lg2(vs0), lv1 = lg2(vs1), iv0 = __fdividef(1.0f, vs0), iv1 = __fdividef(1.0f, vs1);
        uint32_t bfr[NB][2];
        float x[NB][4], xa[NB], xb[NB];
        bool over = false;
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            x[nb][0] = fmaf(sT[nb][0] + uT[nb][0], ks0 * f0[nb], lv0); x[nb][1] = fmaf(sT[nb][1] + uT[nb][1], ks0 * f1[nb], lv0);
            x[nb][2] = fmaf(sT[nb][2] + uT[nb][2], ks1 * f0[nb], lv1); x[nb][3] = fmaf(sT[nb][3] + uT[nb][3], ks1 * f1[nb], lv1);
            if (cut) {
                const int p0 = tok_base + gr, p1 = p0 + 8;
                if (p0 >= min(lim0[nb], t1)) x[nb][0] = -INFINITY;
                if (p0 >= min(lim1[nb], t1)) x[nb][1] = -INFINITY;
                if (p1 >= min(lim0[nb], t1)) x[nb][2] = -INFINITY;
                if (p1 >= min(lim1[nb], t1)) x[nb][3] = -INFINITY;
            }
            xa[nb] = fmaxf(x[nb][0], x[nb][2]); xb[nb] = fmaxf(x[nb][1], x[nb][3]);
            over = over || xa[nb] > m0[nb] + 4.0f || xb[nb] > m1[nb] + 4.0f;
        }
        if (__any_sync(0xFFFFFFFFu, over)) {                // new references, in all column blocks at once
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    xa[nb] = fmaxf(xa[nb], __shfl_xor_sync(0xFFFFFFFFu, xa[nb], off));
                    xb[nb] = fmaxf(xb[nb], __shfl_xor_sync(0xFFFFFFFFu, xb[nb], off));
                }
                const float na = fmaxf(m0[nb], xa[nb]), nc = fmaxf(m1[nb], xb[nb]);
                const float al0 = ex2(m0[nb] - na), al1 = ex2(m1[nb] - nc);
                l0[nb] *= al0; l1[nb] *= al1;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) { o[nb][nt][0] *= al0; o[nb][nt][2] *= al0; o[nb][nt][1] *= al1; o[nb][nt][3] *= al1; }
                m0[nb] = na; m1[nb] = nc;
            }
        }
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            const float w0 = ex2(x[nb][0] - m0[nb]), w1 = ex2(x[nb][1] - m1[nb]), w2 = ex2(x[nb][2] - m0[nb]), w3 = ex2(x[nb][3] - m1[nb]);
            if (cut) {                                      // a masked weight counts nothing also where its token's scale is a NaN
                l0[nb] += (w0 == 0.0f ? 0.0f : w0 * iv0) + (w2 == 0.0f ? 0.0f : w2 * iv1);
                l1[nb] += (w1 == 0.0f ? 0.0f : w1 * iv0) + (w3 == 0.0f ? 0.0f : w3 * iv1);
            } else {
                l0[nb] = fmaf(w0, iv0, fmaf(w2, iv1, l0[nb]));
                l1[nb] = fmaf(w1, iv0, fmaf(w3, iv1, l1[nb]));
            }
            const uint32_t c0 = pack2<false>(w0, w1), c1 = pack2<false>(w2, w3);     // W^T as the B operand: transposed below
            asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(bfr[nb][0]) : "r"(c0));
            asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(bfr[nb][1]) : "r"(c1));
        }
        // ---- O^T += V^T W^T ----
        {
            const int row = 16 + ((mi & 1) << 3) + (lane & 7);
#pragma unroll
            for (int cp = 0; cp < D / 32; cp++) {
                uint32_t r0, r1, r2, r3;                    // bytes: (even dim, odd dim) of token 2j, the same of token 2j+1
                ldsm_x4_t(stg_u + i8_swz<D>(row, 2 * cp + (mi >> 1)), r0, r1, r2, r3);
                const uint32_t ae[4] = {i8_expand<0x4240>(r0), i8_expand<0x4240>(r2), i8_expand<0x4240>(r1), i8_expand<0x4240>(r3)};
                const uint32_t ao[4] = {i8_expand<0x4341>(r0), i8_expand<0x4341>(r2), i8_expand<0x4341>(r1), i8_expand<0x4341>(r3)};
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    mma16816<false>(o[nb][2 * cp], ae, bfr[nb][0], bfr[nb][1]);
                    mma16816<false>(o[nb][2 * cp + 1], ao, bfr[nb][0], bfr[nb][1]);
                }
            }
        }
        __syncwarp();
        if (i + kI8Stages < n_w) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            issue(i + kI8Stages);
        }
    }

    // ---- merge the 4 warps through shared memory (the stages are idle now) ----
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
            l0[nb] += __shfl_xor_sync(0xFFFFFFFFu, l0[nb], off);
            l1[nb] += __shfl_xor_sync(0xFFFFFFFFu, l1[nb], off);
        }
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem);            // [kWarps][rows][D+2]
    auto red_at = [&](int w, int row, int d) -> float& { return red[((size_t)w * rows + row) * (D + 2) + d]; };
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int hh = 0; hh < 2; hh++) {
            const int row = 8 * nb + 2 * j + hh;
            if (row < rows) {
#pragma unroll
                for (int c = 0; c < D / 32; c++) {
                    *reinterpret_cast<float2*>(&red_at(warp, row, 32 * c + 2 * gr)) = make_float2(o[nb][2 * c][hh], o[nb][2 * c + 1][hh]);
                    *reinterpret_cast<float2*>(&red_at(warp, row, 32 * c + 16 + 2 * gr)) = make_float2(o[nb][2 * c][2 + hh], o[nb][2 * c + 1][2 + hh]);
                }
                if (gr == 0) {
                    red_at(warp, row, D) = hh ? m1[nb] : m0[nb];
                    red_at(warp, row, D + 1) = hh ? l1[nb] : l0[nb];
                }
            }
        }
    __syncthreads();
    // per row: the largest reference M, the factor 2^(m_w - M - k) of each warp's sums, and (m, l) of the row; l counts weights over
    // value scales, which may be of any size: 2^-k brings it to [1, 2)
    float* fac = red + kWarps * rows * (D + 2);             // [rows][kWarps + 2]
    if (threadIdx.x < rows) {
        const int row = threadIdx.x;
        float M = -1e30f, l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) M = fmaxf(M, red_at(w, row, D));
#pragma unroll
        for (int w = 0; w < kWarps; w++) l += red_at(w, row, D + 1) * ex2(red_at(w, row, D) - M);
        const uint32_t ex = (__float_as_uint(l) >> 23) & 0xFFu;
        const int k = ex == 0 || ex >= 254 ? 0 : (int)ex - 127;
#pragma unroll
        for (int w = 0; w < kWarps; w++) fac[row * (kWarps + 2) + w] = ex2(red_at(w, row, D) - M) * pow2i(-k);
        fac[row * (kWarps + 2) + kWarps] = l == 0.0f ? -1e30f : (M + (float)k) * 0.6931471805599453f;    // natural-log units, as split-KV rows carry it
        fac[row * (kWarps + 2) + kWarps + 1] = l * pow2i(-k);
    }
    __syncthreads();
    pdl_wait();
    const int prow = st.chunk_base[b] + chunk;
    const int heads_per_row = multi ? g.H * st.nq_max : g.H;
    // the only chunk of its sequence: the result goes straight out (nothing is written while the status word is set)
    const bool direct = mo.counters && mo.out && !mo.partial_out && !mo.peer && st.chunk_base[b + 1] - st.chunk_base[b] == 1;
    if (direct && __ldcg(status) != 0) return;
    for (int idx = threadIdx.x; idx < rows * (D / 2); idx += blockDim.x) {
        const int row = idx / (D / 2), d = 2 * (idx % (D / 2));
        const float* f = fac + row * (kWarps + 2);
        float v0 = 0.0f, v1 = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float2 x = *reinterpret_cast<const float2*>(&red_at(w, row, d));
            v0 += x.x * f[w];
            v1 += x.y * f[w];
        }
        const int tok = multi ? row / G : 0, head = kvh * G + (multi ? row % G : row);
        if (direct) {
            const float inv = 1.0f / (f[kWarps + 1] + 1e-8f);
            const size_t at = ((size_t)(q_row0 + tok) * g.H + head) * D + d;
            if (mo.out_dtype == DT_FP32) *reinterpret_cast<float2*>((float*)mo.out + at) = make_float2(v0 * inv, v1 * inv);
            else                         *reinterpret_cast<uint32_t*>((uint16_t*)mo.out + at) = pack2<IO_BF16>(v0 * inv, v1 * inv);
        } else {
            float* o_row = partials + partial_off(prow, tok * g.H + head, heads_per_row, D);
            *reinterpret_cast<float2*>(o_row + d) = make_float2(v0, v1);
            if (d == 0) *reinterpret_cast<float2*>(o_row + D) = make_float2(f[kWarps], f[kWarps + 1]);
        }
    }
    if (direct || !mo.counters) return;

    // The CTA that arrives last for (b, kvh) merges the sequence's chunks.
    const int r0 = st.chunk_base[b], n = st.chunk_base[b + 1] - r0;
    if (mo.partial_out || mo.peer || rows * n > kMergeCells) {
        merge_if_last(g, st, mo, b, kvh, G, partials, s_flag, MergeMap{rows, heads_per_row, q_row0, 0, 0});
        return;
    }
    // The same merge (tk_merge.cuh) for all rows of the group at once, the first chunks' rows on their way while the weights are
    // computed: a row after the other, 16 rows were four rounds of a chain of L2 loads per warp - 11 us at the end of the
    // launch, where nothing else runs.
    __syncthreads();                                        // the CTA's partial rows are complete ...
    if (threadIdx.x == 0) {
        __threadfence();                                    // ... and ordered before the ticket, device-wide
        int* c = mo.counters + (size_t)b * g.Hkv + kvh;
        const int last = atomicAdd(c, 1) == n - 1;
        if (last) *c = 0;
        *s_flag = last;
    }
    __syncthreads();
    if (!*s_flag) return;
    __threadfence();
    if (__ldcg(status) != 0) return;
    constexpr int U = 8 * NB * (D / 2) / (kWarps * 32), R = 32 / U;     // pairs of columns per thread, chunks in flight together
    const float* col[U];                                    // this thread's columns in the first chunk's row
    const size_t chunk_stride = (size_t)heads_per_row * (D + 2);
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int idx = u * kWarps * 32 + threadIdx.x, row = min(idx / (D / 2), rows - 1);
        col[u] = partials + partial_off(r0, (multi ? (row / G) * g.H + row % G : row) + kvh * G, heads_per_row, D) + 2 * (idx % (D / 2));
    }
    float2 x[R][U];
    auto fetch = [&](int rb) {
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int u = 0; u < U; u++)
                x[r][u] = rb + r < n ? __ldcg(reinterpret_cast<const float2*>(col[u] + (rb + r) * chunk_stride)) : make_float2(0.0f, 0.0f);
    };
    fetch(0);
    float2* ml = reinterpret_cast<float2*>(smem);           // [rows][n] (m, l), then (weight, l)
    float* s_inv = reinterpret_cast<float*>(ml + rows * n);
    {
        const int row = threadIdx.x >> 3, t = threadIdx.x & 7;      // eight threads per row
        const bool on = row < rows;
        const float* at = partials + partial_off(r0, (multi ? (min(row, rows - 1) / G) * g.H + min(row, rows - 1) % G : min(row, rows - 1)) + kvh * G, heads_per_row, D) + D;
        float M = -1e30f, L = 0.0f;
        for (int r = t; on && r < n; r += 8) {
            const float2 c = __ldcg(reinterpret_cast<const float2*>(at + r * chunk_stride));
            ml[row * n + r] = c;
            M = fmaxf(M, c.x);
        }
#pragma unroll
        for (int off = 4; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, off));
        for (int r = t; on && r < n; r += 8) {              // (this thread's own entries)
            float2& c = ml[row * n + r];
            c.x = expf(c.x - M);
            L += c.y * c.x;
        }
#pragma unroll
        for (int off = 4; off > 0; off >>= 1) L += __shfl_xor_sync(0xFFFFFFFFu, L, off);
        if (on && t == 0) s_inv[row] = 1.0f / (L + 1e-8f);
    }
    __syncthreads();
    float2 acc[U];
#pragma unroll
    for (int u = 0; u < U; u++) acc[u] = make_float2(0.0f, 0.0f);
    for (int rb = 0; rb < n; rb += R) {
        if (rb > 0) fetch(rb);
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (rb + r >= n) break;
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int row = min((u * kWarps * 32 + (int)threadIdx.x) / (D / 2), rows - 1);
                const float w = ml[row * n + rb + r].x;
                acc[u].x += x[r][u].x * w;
                acc[u].y += x[r][u].y * w;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int idx = u * kWarps * 32 + threadIdx.x, row = idx / (D / 2), d = 2 * (idx % (D / 2));
        if (row >= rows) break;
        const float inv = s_inv[row];
        const size_t at = ((size_t)(q_row0 + (multi ? row / G : 0)) * g.H + kvh * G + (multi ? row % G : row)) * D + d;
        if (mo.out_dtype == DT_FP32) *reinterpret_cast<float2*>((float*)mo.out + at) = make_float2(acc[u].x * inv, acc[u].y * inv);
        else                         *reinterpret_cast<uint32_t*>((uint16_t*)mo.out + at) = pack2<IO_BF16>(acc[u].x * inv, acc[u].y * inv);
    }
}

template <int D, bool IO_BF16, int NB>
cudaError_t launch_one(const CUtensorMap* map, const Geometry& g, const LayerPtrs& lp, const StepDev& st, const int32_t* page_table,
                       const void* q, float* partials, int* status, const MergeOut& mo, const FuseAppend& fa, bool multi,
                       bool overlap_prev, cudaStream_t s) {
    auto kern = decode_int8_kernel<D, IO_BF16, NB>;
    static bool attr_done[64] = {};                         // per instantiation and device
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (I8Cfg<D, NB>::SMEM));
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(st.n_items); cfg.blockDim = dim3(kWarps * 32); cfg.dynamicSmemBytes = (I8Cfg<D, NB>::SMEM); cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = overlap_prev ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, *map, g, (uint8_t*)lp.pool, st, page_table, (const uint16_t*)q, partials, status, mo, fa,
                              multi ? 1 : 0);
}

template <int D, bool IO_BF16>
cudaError_t launch_nb(bool wide, const CUtensorMap* map, const Geometry& g, const LayerPtrs& lp, const StepDev& st,
                      const int32_t* page_table, const void* q, float* partials, int* status, const MergeOut& mo,
                      const FuseAppend& fa, bool multi, bool overlap_prev, cudaStream_t s) {
    return wide ? launch_one<D, IO_BF16, 2>(map, g, lp, st, page_table, q, partials, status, mo, fa, multi, overlap_prev, s)
                : launch_one<D, IO_BF16, 1>(map, g, lp, st, page_table, q, partials, status, mo, fa, multi, overlap_prev, s);
}

}  // namespace

// The layer's pool as lines of 128 bytes, one box = one tile, 128-byte swizzle.
cudaError_t make_int8_tensor_map(const Geometry& g, void* layer_pool, CUtensorMap* out) {
    static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
    if (!encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult qres;
        cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres);
        if (e != cudaSuccess) return e;
        if (qres != cudaDriverEntryPointSuccess || !fn) return cudaErrorNotSupported;
        encode = (PFN_cuTensorMapEncodeTiled_v12000)fn;
    }
    const int lines = i8_tile_bytes(g.D) / 128;
    cuuint64_t dims[2] = {128, (cuuint64_t)g.num_pages * g.Hkv * lines};
    cuuint64_t strides[1] = {128};
    cuuint32_t box[2] = {128, (cuuint32_t)lines};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, layer_pool, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// multi: the step's nq[b] new tokens of each sequence (rows already in the pool), (heads per kv head) x nq <= 16; q and out are
// [n_tokens][H][D], partial rows hold H * nq_max columns.  Otherwise one token per sequence at position len - 1.
cudaError_t launch_decode_int8(const Geometry& g, const LayerPtrs& lp, const CUtensorMap* map, const StepDev& st,
                               const int32_t* page_table, const void* q, float* partials, int* status, cudaStream_t s,
                               const MergeOut& mo, const FuseAppend& fa, bool multi, bool overlap_prev) {
    if (st.n_items <= 0) return cudaSuccess;
    const int rows = g.H / g.Hkv * (multi ? st.nq_max : 1);
    if (rows > 16 || st.chunk_tokens > kPage * kWarps * 32) return cudaErrorNotSupported;
    const bool wide = rows > 8;
    if (g.io_dtype == DT_BF16)
        return g.D == 128 ? launch_nb<128, true>(wide, map, g, lp, st, page_table, q, partials, status, mo, fa, multi, overlap_prev, s)
                          : launch_nb<64, true>(wide, map, g, lp, st, page_table, q, partials, status, mo, fa, multi, overlap_prev, s);
    return g.D == 128 ? launch_nb<128, false>(wide, map, g, lp, st, page_table, q, partials, status, mo, fa, multi, overlap_prev, s)
                      : launch_nb<64, false>(wide, map, g, lp, st, page_table, q, partials, status, mo, fa, multi, overlap_prev, s);
}

}  // namespace tk
