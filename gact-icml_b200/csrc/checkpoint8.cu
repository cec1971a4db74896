// 8-bit activation checkpoints: rows -> codes + scales, and back (format: blocks8.cuh).
#include "blocks8.cuh"

namespace gact {

constexpr int kCThreads = 256;

struct Ckpt8Args {
    const void* x; int64_t ld; int64_t rows; int cols;
    int8_t* codes; uint8_t* scales;
    int chunks;               // chunks of 8 elements per padded row
    PhiloxKeys rk;
};

// A thread takes 8 consecutive elements, 4 neighbouring lanes a block.  U chunks per thread are loaded before the first
// is worked on.  Chunks are numbered through all padded rows, so a warp's accesses are contiguous whatever the row length.
template <int DT, bool VEC, bool STOCH, int U>
__global__ void __launch_bounds__(kCThreads) checkpoint8_kernel(const __grid_constant__ Ckpt8Args a) {
    using T = typename Elem<DT>::T;
    const int64_t total = a.rows * a.chunks;
    const int64_t first = (int64_t)blockIdx.x * (kCThreads * U) + threadIdx.x;
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t i = first + u * kCThreads;
        const int64_t r = i / a.chunks;
        if (i < total) load_row8<DT, VEC>((const T*)a.x + r * a.ld, (int)(i - r * a.chunks) * 8, a.cols, v[u]);
        else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[u][j] = 0.0f;
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t i = first + u * kCThreads;
        uint32_t byte;
        const uint2 w = codes8<DT, STOCH>(v[u], a.rk, (uint64_t)i, byte);
        if (i < total) {
            st_stream_u2(a.codes + i * 8, w);
            if ((threadIdx.x & 3) == 0) a.scales[i >> 2] = (uint8_t)byte;
        }
    }
}

struct Restore8Args {
    const int8_t* codes; const uint8_t* scales;
    int64_t rows; int cols; int chunks;
    void* out; int64_t ld;
};

template <int DT, bool VEC, int U>
__global__ void __launch_bounds__(kCThreads) restore8_kernel(const __grid_constant__ Restore8Args a) {
    using T = typename Elem<DT>::T;
    const int64_t total = a.rows * a.chunks;
    const int64_t first = (int64_t)blockIdx.x * (kCThreads * U) + threadIdx.x;
    uint2 w[U];
    uint32_t b[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t i = first + u * kCThreads;
        w[u] = make_uint2(0u, 0u);
        b[u] = 1;
        if (i < total) {
            w[u] = ld_stream_u2(a.codes + i * 8);
            b[u] = a.scales[i >> 2];
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t i = first + u * kCThreads;
        if (i >= total) continue;
        const int64_t r = i / a.chunks;
        float v[8];
        restore8(w[u], scale_down8(b[u]), v);
        store_row8<DT, VEC>((T*)a.out + r * a.ld, (int)(i - r * a.chunks) * 8, a.cols, v);
    }
}

// Rows of 16-bit elements into rows of another pitch (operands whose rows do not start on 16-byte boundaries get a copy
// that a tensor map can describe).
__global__ void __launch_bounds__(kCThreads) repitch16_kernel(const uint16_t* __restrict__ src, int64_t ld, int64_t rows, int cols,
                                                              uint16_t* __restrict__ dst, int64_t ldd) {
    const int64_t stride = (int64_t)gridDim.x * kCThreads;
    for (int64_t i = (int64_t)blockIdx.x * kCThreads + threadIdx.x; i < rows * cols; i += stride) {
        const int64_t r = i / cols;
        const int c = (int)(i - r * cols);
        dst[r * ldd + c] = src[r * ld + c];
    }
}

// Four chunks a thread once that still fills the GPU, else one (a small tensor is bound by latency).
template <int DT, bool VEC, bool STOCH> static int launch_ckpt(const Ckpt8Args& a, cudaStream_t s) {
    const int64_t total = a.rows * a.chunks;
    if (total >= (int64_t)sm_count() * 2048 * 4) {
        const int64_t blocks = (total + kCThreads * 4 - 1) / (kCThreads * 4);
        checkpoint8_kernel<DT, VEC, STOCH, 4><<<(unsigned)blocks, kCThreads, 0, s>>>(a);
    } else {
        const int64_t blocks = (total + kCThreads - 1) / kCThreads;
        checkpoint8_kernel<DT, VEC, STOCH, 1><<<(unsigned)blocks, kCThreads, 0, s>>>(a);
    }
    return cudaGetLastError() == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
}
template <int DT> static int dispatch_ckpt(const Ckpt8Args& a, bool stoch, cudaStream_t s) {
    const bool vec = rows_aligned(a.x, a.ld, a.cols, Elem<DT>::kBytes);
    if (vec) return stoch ? launch_ckpt<DT, true, true>(a, s) : launch_ckpt<DT, true, false>(a, s);
    return stoch ? launch_ckpt<DT, false, true>(a, s) : launch_ckpt<DT, false, false>(a, s);
}

template <int DT, bool VEC> static int launch_restore(const Restore8Args& a, cudaStream_t s) {
    const int64_t total = a.rows * a.chunks;
    if (total >= (int64_t)sm_count() * 2048 * 4) {
        const int64_t blocks = (total + kCThreads * 4 - 1) / (kCThreads * 4);
        restore8_kernel<DT, VEC, 4><<<(unsigned)blocks, kCThreads, 0, s>>>(a);
    } else {
        const int64_t blocks = (total + kCThreads - 1) / kCThreads;
        restore8_kernel<DT, VEC, 1><<<(unsigned)blocks, kCThreads, 0, s>>>(a);
    }
    return cudaGetLastError() == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
}
template <int DT> static int dispatch_restore(const Restore8Args& a, cudaStream_t s) {
    return rows_aligned(a.out, a.ld, a.cols, Elem<DT>::kBytes) ? launch_restore<DT, true>(a, s) : launch_restore<DT, false>(a, s);
}

}  // namespace gact

using namespace gact;

extern "C" int64_t gact_checkpoint8_pitch(int64_t cols) { return cols < 0 ? -1 : pitch8(cols); }

extern "C" int gact_checkpoint8(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, int stochastic, uint64_t seed,
                                void* codes, void* scales, void* stream) {
    if (dtype < GACT_F32 || dtype > GACT_BF16) return GACT_ERR_DTYPE;
    if (rows < 0 || cols < 0 || cols > GACT_MAX_COLS || ld < cols || (cols && rows > GACT_MAX_ELEMENTS / pitch8(cols))) return GACT_ERR_SIZE;
    if (rows == 0 || cols == 0) return GACT_OK;
    if (!x || !codes || !scales) return GACT_ERR_NULL;
    if (((uintptr_t)x & (uintptr_t)(elem_bytes_of(dtype) - 1)) || ((uintptr_t)codes & 31)) return GACT_ERR_ALIGN;
    Ckpt8Args a;
    a.x = x; a.ld = ld; a.rows = rows; a.cols = (int)cols;
    a.codes = (int8_t*)codes; a.scales = (uint8_t*)scales; a.chunks = (int)(pitch8(cols) / 8);
    a.rk = philox_round_keys(seed);
    cudaStream_t s = (cudaStream_t)stream;
    switch (dtype) {
    case GACT_F32: return dispatch_ckpt<GACT_F32>(a, stochastic != 0, s);
    case GACT_F16: return dispatch_ckpt<GACT_F16>(a, stochastic != 0, s);
    default: return dispatch_ckpt<GACT_BF16>(a, stochastic != 0, s);
    }
}

extern "C" int gact_restore8(const void* codes, const void* scales, int64_t rows, int64_t cols, int dtype, void* out, int64_t ld,
                             void* stream) {
    if (dtype < GACT_F32 || dtype > GACT_BF16) return GACT_ERR_DTYPE;
    if (rows < 0 || cols < 0 || cols > GACT_MAX_COLS || ld < cols || (cols && rows > GACT_MAX_ELEMENTS / pitch8(cols))) return GACT_ERR_SIZE;
    if (rows == 0 || cols == 0) return GACT_OK;
    if (!codes || !scales || !out) return GACT_ERR_NULL;
    if (((uintptr_t)out & (uintptr_t)(elem_bytes_of(dtype) - 1)) || ((uintptr_t)codes & 31)) return GACT_ERR_ALIGN;
    Restore8Args a;
    a.codes = (const int8_t*)codes; a.scales = (const uint8_t*)scales; a.rows = rows; a.cols = (int)cols;
    a.chunks = (int)(pitch8(cols) / 8); a.out = out; a.ld = ld;
    cudaStream_t s = (cudaStream_t)stream;
    switch (dtype) {
    case GACT_F32: return dispatch_restore<GACT_F32>(a, s);
    case GACT_F16: return dispatch_restore<GACT_F16>(a, s);
    default: return dispatch_restore<GACT_BF16>(a, s);
    }
}

extern "C" int gact_repitch16(const void* src, int64_t ld, int64_t rows, int64_t cols, void* dst, int64_t ld_dst, void* stream) {
    if (rows < 0 || cols < 0 || cols > GACT_MAX_COLS || ld < cols || ld_dst < cols) return GACT_ERR_SIZE;
    if (rows == 0 || cols == 0) return GACT_OK;
    if (!src || !dst) return GACT_ERR_NULL;
    if (((uintptr_t)src & 1) || ((uintptr_t)dst & 1)) return GACT_ERR_ALIGN;
    const int64_t want = (rows * cols + kCThreads - 1) / kCThreads, cap = (int64_t)sm_count() * 16;
    repitch16_kernel<<<(unsigned)(want < cap ? want : cap), kCThreads, 0, (cudaStream_t)stream>>>((const uint16_t*)src, ld, rows, (int)cols,
                                                                                                  (uint16_t*)dst, ld_dst);
    return cudaGetLastError() == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
}
