// Layer norm over the last dimension: forward (with the 8-bit checkpoint of its input) and backward from that checkpoint.
//
//   mean = sum(x) / H,  r = 1 / sqrt(sum((x - mean)^2) / H + eps),  y = (x - mean) r w + b
//   x^ = (x' - mean) r with x' the kept input (restored codes, or x itself),  g = dy w
//   dx = r (g - sum(g)/H - x^ sum(g x^)/H),  dw = sum over rows of dy x^,  db = sum over rows of dy
//
// Both passes are bound by HBM: forward reads x and writes y and 33/32 bytes of codes per element, backward reads dy and
// the codes and writes dx.  Statistics, sums and the weight gradients are fp32; the variance is taken around the mean
// (x stays in registers, so the second look at it is free).
#include "blocks8.cuh"

namespace gact {

struct LnArgs {
    const void* x; int64_t ldx;
    const void* w; const void* b; int wf32;          // weight / bias in fp32 (else in the type of x); null: 1 and 0
    int64_t rows; int cols; float inv_cols; float eps;
    void* y;
    float* mean; float* rstd;
    int8_t* codes; uint8_t* scales; int chunks; int stochastic; PhiloxKeys rk;
};

// 8 weights starting at column `col` (fp32 or the type of x), `fill` past the end or without a weight
template <int DT, bool VEC>
__device__ __forceinline__ void load_param8(const void* p, int f32, int col, int cols, float fill, float (&v)[8]) {
    if (p == nullptr) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = fill;
    } else if (f32 || DT == GACT_F32) {
        if (VEC && col < cols) {
            const float4 a = __ldg((const float4*)((const float*)p + col)), b = __ldg((const float4*)((const float*)p + col) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = (col + j < cols) ? __ldg((const float*)p + col + j) : 0.0f;
        }
    } else {
        using T = typename Elem<DT>::T;
        if (VEC && col < cols) {
            const uint4 a = __ldg((const uint4*)((const T*)p + col));
            const uint32_t raw[4] = {a.x, a.y, a.z, a.w};
            if constexpr (DT != GACT_F32) raw_to_float<DT>(raw, v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = (col + j < cols) ? Elem<DT>::to_float(((const T*)p)[col + j]) : 0.0f;
        }
    }
}

// Sum over the TPR threads of a row.  Up to 32 threads: shuffles inside an aligned part of a warp.  More: the block is one
// row; `buf` holds one value per warp and is used by alternating halves, so one barrier per sum is enough.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* buf) {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o >= 1; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        const int lane = threadIdx.x & 31;
        if (lane == 0) buf[threadIdx.x >> 5] = v;
        __syncthreads();
        v = lane < W ? buf[lane] : 0.0f;
#pragma unroll
        for (int o = W / 2; o >= 1; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
        v = __shfl_sync(kFull, v, 0);
    }
    return v;
}

// A row is held by TPR threads, CH chunks of 8 elements each (chunk c of thread t: columns (t + c TPR) 8 ..).
template <int DT, int TPR, int CH, bool VEC>
__global__ void __launch_bounds__(TPR > 128 ? TPR : 128) layer_norm_kernel(const __grid_constant__ LnArgs a) {
    using T = typename Elem<DT>::T;
    __shared__ float buf[2][32];
    const int t = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x / TPR) + threadIdx.x / TPR;
    const bool live = row < a.rows;
    const T* xr = (const T*)a.x + row * a.ldx;
    float v[CH][8];
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; c++) load_row8<DT, VEC>(xr, (t + c * TPR) * 8, live ? a.cols : 0, v[c]);
#pragma unroll
    for (int c = 0; c < CH; c++)
#pragma unroll
        for (int j = 0; j < 8; j++) sum += v[c][j];
    const float mean = row_sum<TPR>(sum, buf[0]) * a.inv_cols;
    float sq = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; c++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float d = v[c][j] - mean;
            if (VEC ? (t + c * TPR) * 8 < a.cols : (t + c * TPR) * 8 + j < a.cols) sq = fmaf(d, d, sq);
        }
    const float rstd = 1.0f / sqrtf(row_sum<TPR>(sq, buf[1]) * a.inv_cols + a.eps);
    if (live && t == 0 && a.mean) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const int col = (t + c * TPR) * 8;
        if (a.codes) {
            uint32_t byte;
            const uint64_t chunk = (uint64_t)row * a.chunks + (t + c * TPR);
            const uint2 w = a.stochastic ? codes8<DT, true>(v[c], a.rk, chunk, byte) : codes8<DT, false>(v[c], a.rk, chunk, byte);
            if (live && t + c * TPR < a.chunks) {
                st_stream_u2(a.codes + chunk * 8, w);
                if ((t & 3) == 0) a.scales[chunk >> 2] = (uint8_t)byte;
            }
        }
        float w[8], b[8], o[8];
        load_param8<DT, VEC>(a.w, a.wf32, col, a.cols, 1.0f, w);
        load_param8<DT, VEC>(a.b, a.wf32, col, a.cols, 0.0f, b);
#pragma unroll
        for (int j = 0; j < 8; j++) o[j] = fmaf((v[c][j] - mean) * rstd, w[j], b[j]);
        store_row8<DT, VEC>((T*)a.y + row * a.cols, col, live ? a.cols : 0, o);
    }
}

template <int DT, int TPR, int CH> static int launch_ln(const LnArgs& a, bool vec, cudaStream_t s) {
    // several rows per block while a row is at most a warp, fewer when there are few rows
    int block = TPR > 128 ? TPR : 128;
    if (TPR <= 32)
        while (block > 32 && a.rows * TPR < (int64_t)sm_count() * block) block /= 2;
    else block = TPR;
    const int64_t per = block / TPR;
    const int64_t blocks = (a.rows + per - 1) / per;
    if (vec) layer_norm_kernel<DT, TPR, CH, true><<<(unsigned)blocks, block, 0, s>>>(a);
    else layer_norm_kernel<DT, TPR, CH, false><<<(unsigned)blocks, block, 0, s>>>(a);
    return cudaGetLastError() == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
}
template <int DT> static int dispatch_ln(const LnArgs& a, bool vec, cudaStream_t s) {
    const int h = a.cols;
    if (h <= 32) return launch_ln<DT, 4, 1>(a, vec, s);
    if (h <= 64) return launch_ln<DT, 8, 1>(a, vec, s);
    if (h <= 128) return launch_ln<DT, 16, 1>(a, vec, s);
    if (h <= 256) return launch_ln<DT, 32, 1>(a, vec, s);
    if (h <= 512) return launch_ln<DT, 32, 2>(a, vec, s);
    if (h <= 1024) return launch_ln<DT, 32, 4>(a, vec, s);
    if (h <= 2048) return launch_ln<DT, 128, 2>(a, vec, s);
    if (h <= 4096) return launch_ln<DT, 256, 2>(a, vec, s);
    if (h <= 8192) return launch_ln<DT, 512, 2>(a, vec, s);
    return launch_ln<DT, 1024, 2>(a, vec, s);
}

// ---- backward -------------------------------------------------------------------------------------------------------
struct LnBwdArgs {
    const void* dy; int64_t ldy;
    const void* x; int64_t ldx;                       // the input itself, or null:
    const int8_t* codes; const uint8_t* scales; int chunks;
    const float* mean; const float* rstd;
    const void* w; int wf32;
    int64_t rows; int cols; float inv_cols;
    void* dx;                                          // null: weight gradients only
    float* partial;                                    // [gridDim][2 * width]: dw, db; null: no weight gradients
    int width;
};

// A thread owns CH fixed chunks of 8 columns, so the weight gradients of a block's rows stay in its registers; a block
// walks rows blockIdx, blockIdx + grid, ..., R of them (per row group) side by side so that R rows' loads are in flight
// and one barrier serves 2 R sums.  Block sums go to `partial`, added up in a fixed order afterwards: no atomics.
template <int DT, int TPR, int CH, int R, bool VEC, bool COMP>
__global__ void __launch_bounds__(TPR > 128 ? TPR : 128) layer_norm_backward_kernel(const __grid_constant__ LnBwdArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int BLOCK = TPR > 128 ? TPR : (TPR > 32 ? TPR : 128);
    constexpr int GROUPS = BLOCK / TPR;
    __shared__ float2 buf[2][R][32];
    __shared__ float fold[GROUPS > 1 ? BLOCK * 16 : 1];
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    float w[CH][8], dw[CH][8], db[CH][8];
#pragma unroll
    for (int c = 0; c < CH; c++) {
        load_param8<DT, VEC>(a.w, a.wf32, (t + c * TPR) * 8, a.cols, 1.0f, w[c]);
#pragma unroll
        for (int j = 0; j < 8; j++) dw[c][j] = db[c][j] = 0.0f;
    }
    int phase = 0;
    const int64_t step = (int64_t)gridDim.x * GROUPS * R;
    for (int64_t r0 = ((int64_t)blockIdx.x * GROUPS) * R; r0 < a.rows; r0 += step, phase ^= 1) {
        float g[R][CH][8], xh[R][CH][8];
        float2 s[R];
        float rs[R];
#pragma unroll
        for (int k = 0; k < R; k++) {
            const int64_t row = r0 + k * GROUPS + grp;
            const bool live = row < a.rows;
            const float mean = live ? a.mean[row] : 0.0f;
            rs[k] = live ? a.rstd[row] : 0.0f;
#pragma unroll
            for (int c = 0; c < CH; c++) {
                const int col = (t + c * TPR) * 8;
                load_row8<DT, VEC>((const T*)a.dy + row * a.ldy, col, live ? a.cols : 0, g[k][c]);
                if constexpr (COMP) {
                    uint2 q = make_uint2(0u, 0u);
                    uint32_t byte = 1;
                    if (live && t + c * TPR < a.chunks) {
                        const int64_t chunk = row * a.chunks + (t + c * TPR);
                        q = ld_stream_u2(a.codes + chunk * 8);
                        byte = a.scales[chunk >> 2];
                    }
                    restore8(q, scale_down8(byte), xh[k][c]);
                } else {
                    load_row8<DT, VEC>((const T*)a.x + row * a.ldx, col, live ? a.cols : 0, xh[k][c]);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) xh[k][c][j] = (xh[k][c][j] - mean) * rs[k];
            }
        }
#pragma unroll
        for (int k = 0; k < R; k++) {
            s[k] = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int c = 0; c < CH; c++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    // a column past the end has g = 0 (its dy reads as 0) but a NaN scale or an infinite mean must not leak
                    // out of it: only real columns take part
                    if (VEC ? (t + c * TPR) * 8 < a.cols : (t + c * TPR) * 8 + j < a.cols) {
                        dw[c][j] = fmaf(g[k][c][j], xh[k][c][j], dw[c][j]);
                        db[c][j] += g[k][c][j];
                        g[k][c][j] *= w[c][j];
                        s[k].x += g[k][c][j];
                        s[k].y = fmaf(g[k][c][j], xh[k][c][j], s[k].y);
                    }
                }
        }
#pragma unroll
        for (int k = 0; k < R; k++) {
#pragma unroll
            for (int o = (TPR < 32 ? TPR : 32) / 2; o >= 1; o >>= 1) {
                s[k].x += __shfl_xor_sync(kFull, s[k].x, o);
                s[k].y += __shfl_xor_sync(kFull, s[k].y, o);
            }
        }
        if constexpr (TPR > 32) {
            constexpr int W = TPR / 32;
            const int lane = threadIdx.x & 31;
            if (lane == 0) {
#pragma unroll
                for (int k = 0; k < R; k++) buf[phase][k][threadIdx.x >> 5] = s[k];
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < R; k++) {
                s[k] = lane < W ? buf[phase][k][lane] : make_float2(0.0f, 0.0f);
#pragma unroll
                for (int o = W / 2; o >= 1; o >>= 1) {
                    s[k].x += __shfl_xor_sync(kFull, s[k].x, o);
                    s[k].y += __shfl_xor_sync(kFull, s[k].y, o);
                }
                s[k].x = __shfl_sync(kFull, s[k].x, 0);
                s[k].y = __shfl_sync(kFull, s[k].y, 0);
            }
        }
        if (a.dx) {
#pragma unroll
            for (int k = 0; k < R; k++) {
                const int64_t row = r0 + k * GROUPS + grp;
                const float c1 = s[k].x * a.inv_cols, c2 = s[k].y * a.inv_cols;
#pragma unroll
                for (int c = 0; c < CH; c++) {
                    float o[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) o[j] = rs[k] * (g[k][c][j] - c1 - xh[k][c][j] * c2);
                    store_row8<DT, VEC>((T*)a.dx + row * a.cols, (t + c * TPR) * 8, row < a.rows ? a.cols : 0, o);
                }
            }
        }
    }
    if (!a.partial) return;
    if constexpr (GROUPS > 1) {
        // fold the row groups of the block: fold[j][thread]
#pragma unroll
        for (int j = 0; j < 8; j++) {
            fold[j * BLOCK + threadIdx.x] = dw[0][j];
            fold[(8 + j) * BLOCK + threadIdx.x] = db[0][j];
        }
        __syncthreads();
        if (grp == 0) {
            for (int k = 1; k < GROUPS; k++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    dw[0][j] += fold[j * BLOCK + k * TPR + t];
                    db[0][j] += fold[(8 + j) * BLOCK + k * TPR + t];
                }
        }
    }
    if (grp == 0) {
        float* p = a.partial + (int64_t)blockIdx.x * 2 * a.width;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int col = (t + c * TPR) * 8;
            if (col >= a.width) continue;
            *(float4*)(p + col) = make_float4(dw[c][0], dw[c][1], dw[c][2], dw[c][3]);
            *(float4*)(p + col + 4) = make_float4(dw[c][4], dw[c][5], dw[c][6], dw[c][7]);
            *(float4*)(p + a.width + col) = make_float4(db[c][0], db[c][1], db[c][2], db[c][3]);
            *(float4*)(p + a.width + col + 4) = make_float4(db[c][4], db[c][5], db[c][6], db[c][7]);
        }
    }
}

// Blocks of the backward pass: about 2 x 512 threads per SM keep enough rows in flight, more only lengthens the sum of
// the partials (each block writes 2 x cols floats).
static int64_t ln_bwd_blocks(int64_t rows, int64_t cols) {
    const int tpr = cols <= 32 ? 4 : cols <= 64 ? 8 : cols <= 128 ? 16 : cols <= 256 ? 32 : cols <= 512 ? 64 : cols <= 1024 ? 128 : cols <= 2048 ? 256
                  : 512;
    const int block = tpr > 32 ? tpr : 128;
    const int64_t groups = block / tpr;
    const int64_t most = (int64_t)sm_count() * (1024 / block);
    const int64_t want = (rows + groups - 1) / groups;
    return want < most ? want : most;
}

template <int DT, int TPR, int CH, int R> static int launch_ln_bwd(const LnBwdArgs& a, bool vec, int64_t blocks, cudaStream_t s) {
    const int block = TPR > 32 ? TPR : 128;
    if (a.codes) {
        if (vec) layer_norm_backward_kernel<DT, TPR, CH, R, true, true><<<(unsigned)blocks, block, 0, s>>>(a);
        else layer_norm_backward_kernel<DT, TPR, CH, R, false, true><<<(unsigned)blocks, block, 0, s>>>(a);
    } else {
        if (vec) layer_norm_backward_kernel<DT, TPR, CH, R, true, false><<<(unsigned)blocks, block, 0, s>>>(a);
        else layer_norm_backward_kernel<DT, TPR, CH, R, false, false><<<(unsigned)blocks, block, 0, s>>>(a);
    }
    return cudaGetLastError() == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
}
template <int DT> static int dispatch_ln_bwd(const LnBwdArgs& a, bool vec, int64_t blocks, cudaStream_t s) {
    const int h = a.cols;
    if (h <= 32) return launch_ln_bwd<DT, 4, 1, 2>(a, vec, blocks, s);
    if (h <= 64) return launch_ln_bwd<DT, 8, 1, 2>(a, vec, blocks, s);
    if (h <= 128) return launch_ln_bwd<DT, 16, 1, 2>(a, vec, blocks, s);
    if (h <= 256) return launch_ln_bwd<DT, 32, 1, 2>(a, vec, blocks, s);
    if (h <= 512) return launch_ln_bwd<DT, 64, 1, 2>(a, vec, blocks, s);
    if (h <= 1024) return launch_ln_bwd<DT, 128, 1, 2>(a, vec, blocks, s);
    if (h <= 2048) return launch_ln_bwd<DT, 256, 1, 2>(a, vec, blocks, s);
    if (h <= 4096) return launch_ln_bwd<DT, 512, 1, 2>(a, vec, blocks, s);
    if (h <= 8192) return launch_ln_bwd<DT, 512, 2, 1>(a, vec, blocks, s);
    return launch_ln_bwd<DT, 512, 4, 1>(a, vec, blocks, s);
}

// ---- sums of partials over the blocks that wrote them ---------------------------------------------------------------
constexpr int kRCols = 32, kRRows = 16;
struct ReduceArgs { const float* partial; int parts; int64_t width; void* out0; int64_t n0; void* out1; int64_t n1; };

template <int DT>
__global__ void __launch_bounds__(kRCols * kRRows) reduce_columns_kernel(const ReduceArgs a) {
    __shared__ float buf[kRRows][kRCols + 1];
    const int tx = threadIdx.x % kRCols, ty = threadIdx.x / kRCols;
    const int64_t c = (int64_t)blockIdx.x * kRCols + tx;
    float sum = 0.0f;
    if (c < a.width)
        for (int p = ty; p < a.parts; p += kRRows) sum += a.partial[(int64_t)p * a.width + c];
    buf[ty][tx] = sum;
    __syncthreads();
    if (ty == 0 && c < a.width) {
#pragma unroll
        for (int k = 1; k < kRRows; k++) sum += buf[k][tx];
        using T = typename Elem<DT>::T;
        const int64_t half = a.width / 2;
        if (a.out1) {                                   // two rows of width / 2
            if (c < half) { if (c < a.n0 && a.out0) ((T*)a.out0)[c] = Elem<DT>::from_float(sum); }
            else if (c - half < a.n1) ((T*)a.out1)[c - half] = Elem<DT>::from_float(sum);
        } else if (c < a.n0) {
            ((T*)a.out0)[c] = Elem<DT>::from_float(sum);
        }
    }
}

int reduce_columns(const float* partial, int parts, int64_t width, void* out0, int64_t n0, void* out1, int64_t n1, int dtype, cudaStream_t s) {
    const ReduceArgs a{partial, parts, width, out0, n0, out1, n1};
    const unsigned blocks = (unsigned)((width + kRCols - 1) / kRCols);
    switch (dtype) {
    case GACT_F32: reduce_columns_kernel<GACT_F32><<<blocks, kRCols * kRRows, 0, s>>>(a); break;
    case GACT_F16: reduce_columns_kernel<GACT_F16><<<blocks, kRCols * kRRows, 0, s>>>(a); break;
    default: reduce_columns_kernel<GACT_BF16><<<blocks, kRCols * kRRows, 0, s>>>(a); break;
    }
    return cudaGetLastError() == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
}

static bool ln_sizes_ok(int64_t rows, int64_t cols) {
    return rows >= 0 && cols >= 1 && cols <= GACT_LAYER_NORM_MAX_COLS && rows <= GACT_MAX_ELEMENTS / pitch8(cols) && rows <= (1LL << 30);
}
static bool param_ok(const void* p, int dtype) { return !p || ((uintptr_t)p & (uintptr_t)(elem_bytes_of(dtype) - 1)) == 0; }

}  // namespace gact

using namespace gact;

extern "C" int gact_layer_norm(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, const void* weight, const void* bias,
                               int param_dtype, double eps, void* y, float* mean, float* rstd, void* codes, void* scales, int stochastic,
                               uint64_t seed, void* stream) {
    if (dtype < GACT_F32 || dtype > GACT_BF16 || (param_dtype != dtype && param_dtype != GACT_F32)) return GACT_ERR_DTYPE;
    if (!ln_sizes_ok(rows, cols) || ld < cols) return GACT_ERR_SIZE;
    if (rows == 0) return GACT_OK;
    if (!x || !y || (codes && !scales) || (!mean != !rstd)) return GACT_ERR_NULL;
    const uintptr_t em = (uintptr_t)(elem_bytes_of(dtype) - 1);
    if (((uintptr_t)x & em) || ((uintptr_t)y & em) || ((uintptr_t)codes & 31) || !param_ok(weight, param_dtype) || !param_ok(bias, param_dtype))
        return GACT_ERR_ALIGN;
    LnArgs a;
    a.x = x; a.ldx = ld; a.w = weight; a.b = bias; a.wf32 = param_dtype == GACT_F32;
    a.rows = rows; a.cols = (int)cols; a.inv_cols = 1.0f / (float)cols; a.eps = (float)eps;
    a.y = y; a.mean = mean; a.rstd = rstd; a.codes = (int8_t*)codes; a.scales = (uint8_t*)scales;
    a.chunks = (int)(pitch8(cols) / 8); a.stochastic = stochastic; a.rk = philox_round_keys(seed);
    const bool vec = rows_aligned(x, ld, cols, elem_bytes_of(dtype)) && rows_aligned(y, cols, cols, elem_bytes_of(dtype)) &&
                     (((uintptr_t)weight | (uintptr_t)bias) & 15) == 0;
    cudaStream_t s = (cudaStream_t)stream;
    switch (dtype) {
    case GACT_F32: return dispatch_ln<GACT_F32>(a, vec, s);
    case GACT_F16: return dispatch_ln<GACT_F16>(a, vec, s);
    default: return dispatch_ln<GACT_BF16>(a, vec, s);
    }
}

extern "C" int64_t gact_layer_norm_backward_scratch_bytes(int64_t rows, int64_t cols) {
    if (!ln_sizes_ok(rows, cols)) return -1;
    return ln_bwd_blocks(rows, cols) * 2 * ((cols + 7) / 8 * 8) * (int64_t)sizeof(float);
}

extern "C" int gact_layer_norm_backward(const void* dy, int dtype, int64_t rows, int64_t cols, int64_t ld_dy, const void* x, int64_t ld_x,
                                        const void* codes, const void* scales, const float* mean, const float* rstd, const void* weight,
                                        int param_dtype, void* dx, void* dweight, void* dbias, void* scratch, void* stream) {
    if (dtype < GACT_F32 || dtype > GACT_BF16 || (param_dtype != dtype && param_dtype != GACT_F32)) return GACT_ERR_DTYPE;
    if (!ln_sizes_ok(rows, cols) || ld_dy < cols || (x && ld_x < cols)) return GACT_ERR_SIZE;
    cudaStream_t s = (cudaStream_t)stream;
    const bool params = dweight || dbias;
    if (rows == 0) {
        // no rows: the sums over the rows are zero
        const size_t bytes = (size_t)cols * elem_bytes_of(param_dtype);
        if (dweight && cudaMemsetAsync(dweight, 0, bytes, s) != cudaSuccess) return GACT_ERR_LAUNCH;
        if (dbias && cudaMemsetAsync(dbias, 0, bytes, s) != cudaSuccess) return GACT_ERR_LAUNCH;
        return GACT_OK;
    }
    if (!dy || !mean || !rstd || (!x && (!codes || !scales)) || (params && !scratch)) return GACT_ERR_NULL;
    if (!dx && !params) return GACT_OK;
    const uintptr_t em = (uintptr_t)(elem_bytes_of(dtype) - 1);
    if (((uintptr_t)dy & em) || ((uintptr_t)x & em) || ((uintptr_t)dx & em) || ((uintptr_t)codes & 31) || ((uintptr_t)scratch & 15) ||
        !param_ok(weight, param_dtype) || !param_ok(dweight, param_dtype) || !param_ok(dbias, param_dtype))
        return GACT_ERR_ALIGN;
    LnBwdArgs a;
    a.dy = dy; a.ldy = ld_dy; a.x = x; a.ldx = ld_x; a.codes = x ? nullptr : (const int8_t*)codes; a.scales = (const uint8_t*)scales;
    a.chunks = (int)(pitch8(cols) / 8); a.mean = mean; a.rstd = rstd; a.w = weight; a.wf32 = param_dtype == GACT_F32;
    a.rows = rows; a.cols = (int)cols; a.inv_cols = 1.0f / (float)cols; a.dx = dx;
    a.partial = params ? (float*)scratch : nullptr; a.width = (int)((cols + 7) / 8 * 8);
    const int eb = elem_bytes_of(dtype);
    const bool vec = rows_aligned(dy, ld_dy, cols, eb) && (!x || rows_aligned(x, ld_x, cols, eb)) && (!dx || rows_aligned(dx, cols, cols, eb)) &&
                     ((uintptr_t)weight & 15) == 0;
    const int64_t blocks = ln_bwd_blocks(rows, cols);
    int st;
    switch (dtype) {
    case GACT_F32: st = dispatch_ln_bwd<GACT_F32>(a, vec, blocks, s); break;
    case GACT_F16: st = dispatch_ln_bwd<GACT_F16>(a, vec, blocks, s); break;
    default: st = dispatch_ln_bwd<GACT_BF16>(a, vec, blocks, s); break;
    }
    if (st != GACT_OK || !params) return st;
    // both halves are summed; a gradient nobody asked for is not stored
    return reduce_columns((const float*)scratch, (int)blocks, 2 * (int64_t)a.width, dweight ? dweight : nullptr, dweight ? cols : 0,
                          dbias ? dbias : dweight, dbias ? cols : 0, param_dtype, s);
}
