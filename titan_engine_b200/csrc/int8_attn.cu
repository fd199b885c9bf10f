// int8_attn.cu — attention over an INT8 pool, one CTA per (query token, head): chunks of new tokens.
//
// out = sum_j p_j v_j with p = softmax(q k_j / sqrt(D)) over the positions up to the query's own, k_j and v_j the rows the
// codes stand for; running maximum from -1e30, FP32 sums, normaliser 1 / (sum + 1e-8): the arithmetic of
// attention_decode_kernel (reference: src/compute/cuda/attention.cu:58-157) as an online softmax.
#include "int8_cache.cuh"
#include "tk_merge.cuh"

namespace tk {

namespace {

constexpr int kI8Warps = 4;

template <bool BF16, int D>
__global__ void __launch_bounds__(kI8Warps * 32)
attn_int8_kernel(Geometry g, const uint8_t* __restrict__ pool, StepDev st, const int32_t* __restrict__ page_table,
                 const uint16_t* __restrict__ q, void* __restrict__ out, int out_dtype, const int* __restrict__ status) {
    constexpr int E = D / 32;
    __shared__ float red[kI8Warps][D + 2];
    if (__ldcg(status) != 0) return;                        // fail closed: a wait timed out on this handle
    const int row = blockIdx.x, h = blockIdx.y, kvh = h / (g.H / g.Hkv);
    const int b = st.tok_b[row], lim = st.tok_pos[row] + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float qf[E], o[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        const uint16_t w = q[((size_t)row * g.H + h) * D + lane * E + e];
        qf[e] = BF16 ? __uint_as_float((uint32_t)w << 16) : __half2float(__ushort_as_half(w));
        o[e] = 0.0f;
    }
    const float scale = 1.0f / sqrtf((float)D);
    float m = -1e30f, l = 0.0f;
    for (int t = warp; t < lim; t += kI8Warps) {
        const int page = page_table[(size_t)st.seq[b] * g.max_pages_per_seq + t / kI8Page], r = t % kI8Page;
        const uint8_t* tile = pool + ((size_t)page * g.Hkv + kvh) * i8_tile_bytes(D);
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) dot += qf[e] * ((float)tile[i8_row_off(D, 0, r) + lane * E + e] - 128.0f);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, off);
        const float s = dot * *reinterpret_cast<const float*>(tile + i8_scale_off(D, 0, r)) * scale;
        const float mn = fmaxf(m, s), alpha = expf(m - mn), p = expf(s - mn);
        const float pv = p * *reinterpret_cast<const float*>(tile + i8_scale_off(D, 1, r));
        l = l * alpha + p;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = o[e] * alpha + pv * ((float)tile[i8_row_off(D, 1, r) + lane * E + e] - 128.0f);
        m = mn;
    }
#pragma unroll
    for (int e = 0; e < E; e++) red[warp][lane * E + e] = o[e];
    if (lane == 0) { red[warp][D] = m; red[warp][D + 1] = l; }
    __syncthreads();
    float M = -1e30f, L = 0.0f;
    for (int w = 0; w < kI8Warps; w++) M = fmaxf(M, red[w][D]);
    for (int w = 0; w < kI8Warps; w++) L += red[w][D + 1] * expf(red[w][D] - M);
    const float inv = 1.0f / (L + 1e-8f);
    for (int d = threadIdx.x; d < D; d += kI8Warps * 32) {
        float acc = 0.0f;
        for (int w = 0; w < kI8Warps; w++) acc += red[w][d] * expf(red[w][D] - M);
        store_out(out, ((size_t)row * g.H + h) * D + d, acc * inv, out_dtype);
    }
}

}  // namespace

cudaError_t launch_attn_int8(const Geometry& g, const LayerPtrs& lp, const StepDev& st, const int32_t* page_table, const void* q,
                             void* out, int out_dtype, const int* status, cudaStream_t s) {
    const dim3 grid(st.n_tokens, g.H);
    if (grid.x == 0) return cudaSuccess;
    auto kern = g.io_dtype == DT_BF16 ? (g.D == 128 ? attn_int8_kernel<true, 128> : attn_int8_kernel<true, 64>)
                                      : (g.D == 128 ? attn_int8_kernel<false, 128> : attn_int8_kernel<false, 64>);
    kern<<<grid, kI8Warps * 32, 0, s>>>(g, (const uint8_t*)lp.pool, st, page_table, (const uint16_t*)q, out, out_dtype, status);
    return cudaGetLastError();
}

}  // namespace tk
