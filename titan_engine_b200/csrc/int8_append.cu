// int8_append.cu — a step's K/V rows quantised into an INT8 pool as they are appended: one scale per (token, kv head) row
// of K and of V, no open page, so that a sequence may be cut or continued at any token.
//
// The FP8 pool seals whole pages when they are complete (append.cu); the reference has neither (its KVCache::update copies
// FP32 rows, src/inference/kv_cache.cpp:121-151; its one absmax quantiser is FP4, src/compute/cuda/fp4.cu:102-113).
// HBM-bound byte movement for a prompt (2 D bytes read and D + 4 written per row), launch latency for a decode step.
#include "int8_cache.cuh"

namespace tk {

namespace {

constexpr int kI8AppendThreads = 256;
constexpr int kI8Vec = 4;              // 16-byte vectors of a row per lane

// u / d for u < 2^31 as a product (Granlund and Montgomery's division by invariant integers): (mul_hi(u, m) + u) >> s.
struct Divisor {
    uint32_t d, m;
    int s;
    __device__ __forceinline__ uint32_t of(uint32_t u) const { return (__umulhi(u, m) + u) >> s; }
};
Divisor divisor(uint32_t d) {
    int s = 0;
    while ((1ull << s) < d) s++;
    return Divisor{d, (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
}

// D / 32 lanes hold a row, a lane eight values of each quarter of it; a row's K and V are separate rows here: unit u = (token,
// K|V, kv head).  The kernel is bound by issue slots as much as by HBM: what is done once per row and lane (addresses, the
// reduction, the reciprocal) costs as many instructions as ten values, hence several vectors per lane.  Measured, 64 prompts of
// 512 tokens, 8 kv heads, D = 128 (201 MB read and written): one vector per lane 53 us, two 43, four 39 = 5.2 TB/s; two rows in
// flight per thread with four vectors each 41.
template <bool BF16, int D>
__global__ void __launch_bounds__(kI8AppendThreads)
append_int8_kernel(Geometry g, uint8_t* __restrict__ pool, StepDev st, Divisor per_tok, const int32_t* __restrict__ page_table,
                   const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, int64_t* __restrict__ slots_out) {
    constexpr int LANES = D / (8 * kI8Vec);
    const int c = threadIdx.x % LANES;
    const uint32_t u = (blockIdx.x * kI8AppendThreads + threadIdx.x) / LANES;
    const bool live = u < (uint32_t)st.n_tokens * per_tok.d;         // (rows of a step fit the GPU's memory: below 2^31)
    const uint32_t t = per_tok.of(u), rem = u - t * per_tok.d, kv = rem >= (uint32_t)g.Hkv, h = kv ? rem - g.Hkv : rem;
    uint4 x[kI8Vec];
    int slot = 0;
    if (live) {
        const uint16_t* src = (kv ? v : k) + ((size_t)t * g.Hkv + h) * D + c * 8;
#pragma unroll
        for (int e = 0; e < kI8Vec; e++) x[e] = *reinterpret_cast<const uint4*>(src + e * (D / kI8Vec));
        slot = st.tok_dst[t];
    } else {
#pragma unroll
        for (int e = 0; e < kI8Vec; e++) x[e] = make_uint4(0, 0, 0, 0);
    }
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < kI8Vec; e++) m = max(m, i8_absmax8(x[e]));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    const bool huge = __any_sync(0xFFFFFFFFu, !(i8_amax_value<BF16>(m) <= kI8AmaxMax));    // values that saturate, or a NaN
    if (!live) return;
    const I8Row row = i8_row(i8_amax_value<BF16>(m));
    uint8_t* tile = pool + ((size_t)(slot / kI8Page) * g.Hkv + h) * i8_tile_bytes(D);
    const int r = slot % kI8Page;
    uint2* to = reinterpret_cast<uint2*>(tile + i8_row_off(D, kv, r) + c * 8);
#pragma unroll
    for (int e = 0; e < kI8Vec; e++)
        to[e * LANES] = huge ? i8_codes8<BF16, true>(x[e], row.to_code) : i8_codes8<BF16, false>(x[e], row.to_code);
    if (c == 0) {
        *reinterpret_cast<float*>(tile + i8_scale_off(D, kv, r)) = row.scale;
        if (slots_out && rem == 0) {
            const int pos = st.tok_pos[t];
            slots_out[t] = (int64_t)page_table[(size_t)st.seq[st.tok_b[t]] * g.max_pages_per_seq + pos / kI8Page] * kI8Page + pos % kI8Page;
        }
    }
}

template <bool BF16, int D>
cudaError_t launch_d(const Geometry& g, const LayerPtrs& lp, const StepDev& st, const int32_t* page_table, const void* k,
                     const void* v, int64_t* slots_out, cudaStream_t s) {
    constexpr int ROWS = kI8AppendThreads / (D / (8 * kI8Vec));
    const long long units = (long long)st.n_tokens * 2 * g.Hkv;
    append_int8_kernel<BF16, D><<<(unsigned)((units + ROWS - 1) / ROWS), kI8AppendThreads, 0, s>>>(
        g, (uint8_t*)lp.pool, st, divisor(2 * (uint32_t)g.Hkv), page_table, (const uint16_t*)k, (const uint16_t*)v, slots_out);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_append_int8(const Geometry& g, const LayerPtrs& lp, const StepDev& st, const int32_t* page_table,
                               const void* k, const void* v, int64_t* slots_out, cudaStream_t s) {
    if (st.n_tokens <= 0) return cudaSuccess;
    if (g.io_dtype == DT_BF16) return g.D == 128 ? launch_d<true, 128>(g, lp, st, page_table, k, v, slots_out, s)
                                                 : launch_d<true, 64>(g, lp, st, page_table, k, v, slots_out, s);
    return g.D == 128 ? launch_d<false, 128>(g, lp, st, page_table, k, v, slots_out, s)
                      : launch_d<false, 64>(g, lp, st, page_table, k, v, slots_out, s);
}

}  // namespace tk
