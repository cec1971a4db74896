// 8-bit activation checkpoints: rows -> codes + scales, and back (format: blocks8.cuh).  Bound by HBM: bf16 65536 x 4096 takes
// 126 us (0.99 of the copy bandwidth), back 121; with stochastic rounding 200 (the generator: 20.4 instructions an element instead of
// 12.7, issue slots 74 % busy).
#include "blocks8.cuh"

namespace gact {

constexpr int kCThreads = 256;

struct Ckpt8Args {
    const void* x; int64_t ld; int64_t rows; int cols;
    int8_t* codes; uint8_t* scales;
    int chunks;               // chunks of 8 elements per padded row
    int tiles;                // tiles of 256 columns per row
    Divisor by;               // chunks or tiles of a row, by the way the kernel walks
    Noise8 noise;
};
struct Restore8Args {
    const int8_t* codes; const uint8_t* scales;
    int64_t rows; int cols; int chunks; int tiles; Divisor by;
    void* out; int64_t ld;
};

// A thread takes 8 consecutive elements, 4 neighbouring lanes a block of 32.
//   FLAT: chunks are numbered through all padded rows, so a warp's accesses are contiguous whatever the row length.
//   else: a warp takes 256 columns of a row (rows that do not start on 16-byte boundaries: one division per warp, and the
//         element-wise accesses of Row8 run along the row).
// U chunks per thread are loaded before the first is worked on.
template <bool FLAT, int U> struct Walk {
    int64_t chunk[U], row[U];
    int col[U];
    __device__ __forceinline__ Walk(int64_t rows, int chunks, int tiles, const Divisor& by) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (FLAT) {
                const int64_t i = (int64_t)blockIdx.x * (kCThreads * U) + u * kCThreads + threadIdx.x;
                row[u] = by.div(i);
                col[u] = (int)(i - row[u] * chunks) * 8;
                chunk[u] = row[u] < rows ? i : -1;
            } else {
                const int64_t w = (int64_t)blockIdx.x * (kCThreads / 32 * U) + u * (kCThreads / 32) + (threadIdx.x >> 5);
                row[u] = by.div(w);
                const int c = (int)(w - row[u] * tiles) * 32 + (threadIdx.x & 31);
                col[u] = c * 8;
                chunk[u] = (row[u] < rows && c < chunks) ? row[u] * chunks + c : -1;
            }
        }
    }
};

template <int DT, bool VEC, bool FLAT, bool STOCH, int U>
__global__ void __launch_bounds__(kCThreads) checkpoint8_kernel(const __grid_constant__ Ckpt8Args a) {
    using T = typename Elem<DT>::T;
    __shared__ __align__(16) uint8_t stage[VEC || FLAT ? 16 : kCThreads * 8 * Elem<DT>::kBytes];
    void* mine = stage + (VEC || FLAT ? 0 : (threadIdx.x >> 5) * Stage8<DT, false>::kBytes);
    const Walk<FLAT, U> w(a.rows, a.chunks, a.tiles, a.by);
    const uint2 high = STOCH ? a.noise.high() : make_uint2(0u, 0u);
    Row8<DT, VEC, 32> x[U];
    uint32_t raw[U][RawRegs<DT>::N];
#pragma unroll
    for (int u = 0; u < U; u++) {
        if constexpr (VEC || !FLAT) {
            x[u].load((const T*)a.x, a.ld, w.row[u], a.rows, w.col[u], a.cols);
        } else {
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; j++)
                f[j] = (w.chunk[u] >= 0 && w.col[u] + j < a.cols) ? Elem<DT>::to_float(((const T*)a.x)[w.row[u] * a.ld + w.col[u] + j]) : 0.0f;
            const float2 p[4] = {make_float2(f[0], f[1]), make_float2(f[2], f[3]), make_float2(f[4], f[5]), make_float2(f[6], f[7])};
            pairs_to_raw<DT>(p, raw[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        if constexpr (VEC || !FLAT) x[u].get(mine, raw[u]);
        float2 v[4];
        raw_to_pairs<DT>(raw[u], v);
        uint32_t byte;
        const uint2 c = codes8<STOCH>(v, absmax8<DT>(raw[u]), a.noise, high, (uint64_t)w.chunk[u], byte, top_byte8<DT>());
        if (w.chunk[u] >= 0) {
            st_stream_u2(a.codes + w.chunk[u] * 8, c);
            if ((threadIdx.x & 3) == 0) a.scales[w.chunk[u] >> 2] = (uint8_t)byte;
        }
    }
}

template <int DT, bool VEC, bool FLAT, int U>
__global__ void __launch_bounds__(kCThreads) restore8_kernel(const __grid_constant__ Restore8Args a) {
    using T = typename Elem<DT>::T;
    __shared__ __align__(16) uint8_t stage[VEC || FLAT ? 16 : kCThreads * 8 * Elem<DT>::kBytes];
    void* mine = stage + (VEC || FLAT ? 0 : (threadIdx.x >> 5) * Stage8<DT, false>::kBytes);
    const Walk<FLAT, U> w(a.rows, a.chunks, a.tiles, a.by);
    uint2 c[U];
    uint32_t b[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        c[u] = make_uint2(0u, 0u);
        b[u] = 1;
        if (w.chunk[u] >= 0) {
            c[u] = ld_stream_u2(a.codes + w.chunk[u] * 8);
            b[u] = a.scales[w.chunk[u] >> 2];
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        float2 v[4];
        restore_pairs(c[u], scale_down8(b[u]), v);
        if constexpr (VEC || !FLAT) {
            Row8<DT, VEC, 32>::store((T*)a.out, a.ld, w.row[u], a.rows, w.col[u], a.cols, mine, v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (w.chunk[u] >= 0 && w.col[u] + j < a.cols)
                    ((T*)a.out)[w.row[u] * a.ld + w.col[u] + j] = Elem<DT>::from_float(j & 1 ? v[j / 2].y : v[j / 2].x);
        }
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

// Four chunks a thread once that still fills the GPU, else one (a small tensor is bound by latency).  Measured, four / one in us,
// bf16 rows of 1024: 1024 rows 2.6 / 2.0, 4096 3.8 / 3.5, 9472 (where the rule changes) 6.5 / 7.2, 65536 33.8 / 39.7; back 2.2 / 1.9,
// 3.5 / 3.3, 6.3 / 7.0, 32.1 / 36.9.
// Rows that do not start on 16-byte boundaries are walked along the row where the warps' 256 columns are full enough: the element-wise
// accesses then run side by side, but lanes past the end of a row idle.  Measured on 8 M elements, along the row / flat in us,
// bf16 (fp32): 127 columns 12.9 / 7.2 (13.9 / 10.1), 161 10.9 / 8.1 (12.1 / 10.2), 255 7.8 / 7.4 (9.0 / 11.1), 257 12.8 / 7.9
// (13.6 / 10.5); on 16 M: 513 17.4 / 16.6 (18.7 / 20.1), 771 16.1 / 16.2 (17.5 / 20.3), 1003 14.1 / 16.5 (16.0 / 21.0).  Restoring, where
// the stores are the element-wise side, pays sooner: 65 columns 21.8 / 23.1 (26.5 / 21.1), 73 19.8 / 24.7 (24.4 / 26.2), 97
// 15.7 / 24.7 (20.2 / 26.2), 257 12.0 / 23.8 (13.9 / 30.5).
static bool along_row_ckpt(int cols, int tiles) { return 4 * (int64_t)cols >= 3 * 256 * (int64_t)tiles; }
static bool along_row_restore(int cols) { return cols >= 72; }
template <bool FLAT> static int64_t walk_blocks(int64_t rows, int chunks, int tiles, int u) {
    const int64_t per = (int64_t)(FLAT ? kCThreads : kCThreads / 32) * u;
    return (rows * (FLAT ? chunks : tiles) + per - 1) / per;
}
static bool walk_big(int64_t rows, int chunks) { return rows * chunks >= (int64_t)sm_count() * 2048 * 4; }

template <int DT, bool VEC, bool FLAT, bool STOCH> static void launch_ckpt(Ckpt8Args a, cudaStream_t s) {
    a.by = Divisor::of(FLAT ? a.chunks : a.tiles);
    if (walk_big(a.rows, a.chunks))
        checkpoint8_kernel<DT, VEC, FLAT, STOCH, 4><<<(unsigned)walk_blocks<FLAT>(a.rows, a.chunks, a.tiles, 4), kCThreads, 0, s>>>(a);
    else
        checkpoint8_kernel<DT, VEC, FLAT, STOCH, 1><<<(unsigned)walk_blocks<FLAT>(a.rows, a.chunks, a.tiles, 1), kCThreads, 0, s>>>(a);
}
template <int DT, bool STOCH> static int dispatch_ckpt(const Ckpt8Args& a, cudaStream_t s) {
    if (rows_aligned(a.x, a.ld, a.cols, Elem<DT>::kBytes)) launch_ckpt<DT, true, true, STOCH>(a, s);
    else if (along_row_ckpt(a.cols, a.tiles)) launch_ckpt<DT, false, false, STOCH>(a, s);
    else launch_ckpt<DT, false, true, STOCH>(a, s);
    return cudaGetLastError() == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
}

template <int DT, bool VEC, bool FLAT> static void launch_restore(Restore8Args a, cudaStream_t s) {
    a.by = Divisor::of(FLAT ? a.chunks : a.tiles);
    if (walk_big(a.rows, a.chunks))
        restore8_kernel<DT, VEC, FLAT, 4><<<(unsigned)walk_blocks<FLAT>(a.rows, a.chunks, a.tiles, 4), kCThreads, 0, s>>>(a);
    else
        restore8_kernel<DT, VEC, FLAT, 1><<<(unsigned)walk_blocks<FLAT>(a.rows, a.chunks, a.tiles, 1), kCThreads, 0, s>>>(a);
}
template <int DT> static int dispatch_restore(const Restore8Args& a, cudaStream_t s) {
    if (rows_aligned(a.out, a.ld, a.cols, Elem<DT>::kBytes)) launch_restore<DT, true, true>(a, s);
    else if (along_row_restore(a.cols)) launch_restore<DT, false, false>(a, s);
    else launch_restore<DT, false, true>(a, s);
    return cudaGetLastError() == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
}

}  // namespace gact

using namespace gact;

extern "C" int64_t gact_checkpoint8_pitch(int64_t cols) { return cols < 0 ? -1 : pitch8(cols); }

extern "C" int gact_checkpoint8(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, int rounding, uint64_t seed,
                                void* codes, void* scales, void* stream) {
    if (dtype < GACT_F32 || dtype > GACT_BF16) return GACT_ERR_DTYPE;
    if (rows < 0 || cols < 0 || cols > GACT_MAX_COLS || ld < cols || (cols && rows > GACT_MAX_ELEMENTS / pitch8(cols))) return GACT_ERR_SIZE;
    if (rows == 0 || cols == 0) return GACT_OK;
    if (const int st = rounding_status(rounding, seed, GACT_CODES_STOCHASTIC | GACT_CODES_DEVICE_SEED)) return st;
    if (!x || !codes || !scales) return GACT_ERR_NULL;
    if (((uintptr_t)x & (uintptr_t)(elem_bytes_of(dtype) - 1)) || ((uintptr_t)codes & 31)) return GACT_ERR_ALIGN;
    Ckpt8Args a;
    a.x = x; a.ld = ld; a.rows = rows; a.cols = (int)cols;
    a.codes = (int8_t*)codes; a.scales = (uint8_t*)scales; a.chunks = (int)(pitch8(cols) / 8);
    a.tiles = (int)((cols + 255) / 256);
    const bool stochastic = rounding & GACT_CODES_STOCHASTIC;
    a.noise = Noise8::of(seed, rounding & GACT_CODES_DEVICE_SEED, 0);
    cudaStream_t s = (cudaStream_t)stream;
    switch (dtype) {
    case GACT_F32: return stochastic ? dispatch_ckpt<GACT_F32, true>(a, s) : dispatch_ckpt<GACT_F32, false>(a, s);
    case GACT_F16: return stochastic ? dispatch_ckpt<GACT_F16, true>(a, s) : dispatch_ckpt<GACT_F16, false>(a, s);
    default: return stochastic ? dispatch_ckpt<GACT_BF16, true>(a, s) : dispatch_ckpt<GACT_BF16, false>(a, s);
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
    a.chunks = (int)(pitch8(cols) / 8); a.tiles = (int)((cols + 255) / 256); a.out = out; a.ld = ld;
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
