// read_back.cu — rows of token ranges of the cache, dequantised into contiguous K and V tensors: every storage type.
//
// The reference hands out the slab itself (KVCache::k_cache / v_cache, src/inference/kv_cache.h:42-48); a paged or quantised
// pool has no such rows to point at.  HBM-bound: a row's bytes are read once and written once in the output type.
// The list of pages is a kernel ARGUMENT (up to 32 KB): nothing is uploaded and no device buffer is involved, so calls on
// several streams, and calls captured into graphs, share nothing, and pages that a call since the last step has moved
// (a fork, a truncation) are read where they are now.
// Measured, INT8, D = 128, 8 kv heads: 98,519 tokens of 32 sequences as bf16 (612 MB) 102 us = 0.92 of the copy rate; a few pages
// 6 us, the launch.
#include "int8_cache.cuh"
#include "tk_mma.cuh"

#include <cuda_fp8.h>

namespace tk {

namespace {

constexpr int kReadThreads = 128;

template <int N>
struct ReadList { ReadItem item[N]; };

__device__ __forceinline__ void put8(void* out, size_t i, const float (&f)[8], int dt) {
    if (dt == DT_FP32) {
        *reinterpret_cast<float4*>((float*)out + i) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4*>((float*)out + i + 4) = make_float4(f[4], f[5], f[6], f[7]);
        return;
    }
    uint4 w;
    uint32_t* p = &w.x;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (dt == DT_BF16) { const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]); p[j] = *reinterpret_cast<const uint32_t*>(&h); }
        else               { const __half2 h = __floats2half2_rn(f[2 * j], f[2 * j + 1]); p[j] = *reinterpret_cast<const uint32_t*>(&h); }
    }
    *reinterpret_cast<uint4*>((uint16_t*)out + i) = w;
}

// INT8: one CTA per (listed page, kv head), its 32 rows of D codes in one round of eight codes per thread, all loads first.
template <int N, int D>
__global__ void __launch_bounds__(kReadThreads)
read_int8_kernel(Geometry g, const uint8_t* __restrict__ pool, const __grid_constant__ ReadList<N> list, void* __restrict__ k_out,
                 void* __restrict__ v_out, int out_dtype) {
    constexpr int LANES = D / 8, U = 2 * kI8Page * LANES / kReadThreads, ROWS = kReadThreads / LANES;
    pdl_launch_dependents();
    const ReadItem it = list.item[blockIdx.x / g.Hkv];
    const int h = blockIdx.x % g.Hkv, c = threadIdx.x % LANES;
    const uint8_t* tile = pool + ((size_t)it.page * g.Hkv + h) * i8_tile_bytes(D);
    uint2 w[U];
    float scale[U];
#pragma unroll
    for (int i = 0; i < U; i++) {                           // rows it.row0 .. of K, then of V
        const int r = i * ROWS + threadIdx.x / LANES, kv = r >= it.n_rows, row = it.row0 + (kv ? r - it.n_rows : r);
        if (r < 2 * it.n_rows) {
            w[i] = __ldcs(reinterpret_cast<const uint2*>(tile + i8_row_off(D, kv, row) + c * 8));
            scale[i] = *reinterpret_cast<const float*>(tile + i8_scale_off(D, kv, row));
        }
    }
#pragma unroll
    for (int i = 0; i < U; i++) {
        const int r = i * ROWS + threadIdx.x / LANES, kv = r >= it.n_rows;
        if (r >= 2 * it.n_rows) break;
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; j++)                          // the byte under 2^23: 2^23 + code + 128, exact
            f[j] = __fmul_rn(__uint_as_float(__byte_perm(j < 4 ? w[i].x : w[i].y, 0x4B000000u, 0x7440 | (j & 3))) - 8388736.0f, scale[i]);
        put8(kv ? v_out : k_out, ((size_t)(it.out_row + (kv ? r - it.n_rows : r)) * g.Hkv + h) * D + c * 8, f, out_dtype);
    }
    pdl_wait();                                             // this launch does not end before the one it overlapped
}

// The other pools: one CTA per (listed page, kv head).  A thread moves eight values of a row at a time.  32 sequences of 2048-6144
// tokens, 8 kv heads, D = 128, to bf16: a bf16 pool 178 us = 6.1 TB/s (HBM), an FP8 pool 173 us = 4.7 TB/s (three quarters of
// the bytes in the same time; not profiled).
template <int N>
__global__ void __launch_bounds__(kReadThreads)
read_rows_kernel(Geometry g, LayerPtrs lp, const __grid_constant__ ReadList<N> list, void* __restrict__ k_out, void* __restrict__ v_out,
                 int out_dtype) {
    pdl_launch_dependents();
    const ReadItem it = list.item[blockIdx.x / g.Hkv];
    const int h = blockIdx.x % g.Hkv;
    const bool open = it.page < 0;                          // FP8: the 16-bit open page of sequence -1 - page
    const int vk = g.D / 8, vv = g.Dv / 8, n_k = it.n_rows * vk, n_vec = n_k + it.n_rows * vv;
    const int stored = open ? g.io_dtype : g.dtype;
    const size_t tile16 = open ? tile_offset(g, -1 - it.page, h, 0) : tile_offset(g, it.page, h, 0);
    for (int i = threadIdx.x; i < n_vec; i += kReadThreads) {
        const int kv = i >= n_k, ii = kv ? i - n_k : i, per = kv ? vv : vk, dim = per * 8;
        const int row = ii / per, c = ii % per, r = it.row0 + row;
        const size_t o = ((size_t)(it.out_row + row) * g.Hkv + h) * dim + c * 8;
        float f[8];
        if (stored == DT_FP8) {
            const uint2 w = *reinterpret_cast<const uint2*>((const uint8_t*)lp.pool + tile16 + (size_t)(kv ? g.ps * g.D : 0) + (size_t)r * dim + c * 8);
            const float scale = lp.scales[((size_t)it.page * g.Hkv + h) * 2 + kv];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const __half_raw hr = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)((j < 4 ? w.x >> (8 * j) : w.y >> (8 * j - 32)) & 0xFFu), __NV_E4M3);
                f[j] = __fmul_rn(__half2float(*reinterpret_cast<const __half*>(&hr)), scale);
            }
        } else {
            const uint4 w = *reinterpret_cast<const uint4*>((const uint16_t*)(open ? lp.open_pages : lp.pool) + tile16 +
                                                            (size_t)(kv ? g.ps * g.D : 0) + (size_t)r * dim + c * 8);
            if (out_dtype != DT_FP32) {                     // the stored type is the output's: bits, not values
                *reinterpret_cast<uint4*>((uint16_t*)(kv ? v_out : k_out) + o) = w;
                continue;
            }
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 t = stored == DT_BF16 ? i8_unpack2<true>(ws[j]) : i8_unpack2<false>(ws[j]);
                f[2 * j] = t.x; f[2 * j + 1] = t.y;
            }
        }
        put8(kv ? v_out : k_out, o, f, out_dtype);
    }
    pdl_wait();                                             // this launch does not end before the one it overlapped
}

template <int N>
cudaError_t launch_n(const Geometry& g, const LayerPtrs& lp, const ReadItem* items, int n, void* k_out, void* v_out, int out_dtype,
                     bool overlap_prev, cudaStream_t s) {
    static_assert(sizeof(ReadList<N>) <= 32000, "kernel arguments hold at most 32764 bytes");
    ReadList<N> list;
    for (int i = 0; i < n; i++) list.item[i] = items[i];
    for (int i = n; i < N; i++) list.item[i] = ReadItem{0, 0, 0, 0};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n * (unsigned)g.Hkv); cfg.blockDim = dim3(kReadThreads); cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = overlap_prev ? 1 : 0;
    if (g.dtype != DT_INT8) return cudaLaunchKernelEx(&cfg, read_rows_kernel<N>, g, lp, list, k_out, v_out, out_dtype);
    if (g.D == 128) return cudaLaunchKernelEx(&cfg, read_int8_kernel<N, 128>, g, (const uint8_t*)lp.pool, list, k_out, v_out, out_dtype);
    return cudaLaunchKernelEx(&cfg, read_int8_kernel<N, 64>, g, (const uint8_t*)lp.pool, list, k_out, v_out, out_dtype);
}

}  // namespace

// Reads the listed pages' rows; *n_launches kernels were launched.
cudaError_t launch_read_rows(const Geometry& g, const LayerPtrs& lp, const ReadItem* items, int n_items, void* k_out, void* v_out,
                             int out_dtype, cudaStream_t s, int* n_launches) {
    *n_launches = 0;
    for (int at = 0; at < n_items;) {
        const int n = n_items - at < kReadItemsBig ? n_items - at : kReadItemsBig;
        // the launches of one call read the same pool and write disjoint rows: a later one may start while the one before drains
        cudaError_t e = n <= kReadItemsSmall ? launch_n<kReadItemsSmall>(g, lp, items + at, n, k_out, v_out, out_dtype, at > 0, s)
                                             : launch_n<kReadItemsBig>(g, lp, items + at, n, k_out, v_out, out_dtype, at > 0, s);
        if (e != cudaSuccess) return e;
        (*n_launches)++;
        at += n;
    }
    return cudaSuccess;
}

}  // namespace tk
