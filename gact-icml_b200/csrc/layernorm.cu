// Layer norm over the last dimension: forward (with the 8-bit checkpoint of its input) and backward from that checkpoint.
//
//   mean = sum(x) / H,  r = 1 / sqrt(sum((x - mean)^2) / H + eps),  y = (x - mean) r w + b
//   x^ = (x' - mean) r with x' the kept input (restored codes, or x itself),  g = dy w
//   centred codes keep x - mean instead:  x^ = x' r.  Half a code's step is then at most 1/127 of the largest deviation from the
//   mean; that of x grows with the mean, and seen through r it has no bound (fp32 rows of 100 +- 1: dw 30 % off, centred 0.9 %)
//   dx = r (g - sum(g)/H - x^ sum(g x^)/H),  dw = sum over rows of dy x^,  db = sum over rows of dy
//
// Both passes are bound by HBM: forward reads x and writes y and 33/32 bytes of codes per element, backward reads dy and
// the codes and writes dx.  Statistics, sums and the weight gradients are fp32; the variance is taken around the mean
// (x stays in registers, so the second look at it is free); 1 / H is a factor, r comes from rsqrtf, and (x' - mean) r is one
// multiply-add x' r - mean r in the backward pass: fp32 outputs are off by 1.7e-7, half again as much as with a division, a square
// root and a subtraction.  Measured in bf16: 65536 x 4096 forward 262 us (centred 271), backward 252 (0.79 and 0.82 of the copy
// bandwidth); 65536 x 1024 66 to 70 and 74; 8192 x 1024 11.9 and 15.6 (of which 4 the sum of the partials), fp32 16.2 and 19.9;
// 128 x 1024 2.7 and 5.0 (launches).
#include "blocks8.cuh"
#include "tcgen05.cuh"

namespace gact {

struct LnArgs {
    const void* x; int64_t ldx;
    const void* w; const void* b; int wf32;          // weight / bias in fp32 (else in the type of x); null: 1 and 0
    int64_t rows; int cols; float inv_cols; float eps;
    void* y;
    float* stats;                                    // (mean, or 0 with `center`; 1 / deviation) per row, or null
    int8_t* codes; uint8_t* scales; int chunks; int stochastic, center; Noise8 noise;
};

// 8 weights starting at column `col` (fp32 or the type of x); `none` without a weight, 0 past the end
template <int DT>
__device__ __forceinline__ void load_param8(const void* p, int f32, int col, int cols, float none, float (&f)[8]) {
    using T = typename Elem<DT>::T;
#pragma unroll
    for (int j = 0; j < 8; j++)
        f[j] = !p ? none : col + j >= cols ? 0.0f : f32 ? __ldg((const float*)p + col + j) : Elem<DT>::to_float(((const T*)p)[col + j]);
}
// all W of them into shared memory as fp32, by the whole block
template <int DT, int W>
__device__ __forceinline__ void stage_params(const void* p, int f32, int cols, float none, float* to) {
    const bool wide = p && ((uintptr_t)p & 15) == 0;
    for (int col = threadIdx.x * 8; col < W; col += blockDim.x * 8) {
        float f[8];
        if (wide && col + 8 <= cols && (f32 || DT == GACT_F32)) {
            const float4 a = __ldg((const float4*)((const float*)p + col)), b = __ldg((const float4*)((const float*)p + col) + 1);
            f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
        } else if (wide && col + 8 <= cols) {
            if constexpr (DT != GACT_F32) {
                const uint4 a = __ldg((const uint4*)((const typename Elem<DT>::T*)p + col));
                const uint32_t raw[4] = {a.x, a.y, a.z, a.w};
                raw_to_float<DT>(raw, f);
            }
        } else {
            load_param8<DT>(p, f32, col, cols, none, f);
        }
        *(float4*)(to + col) = make_float4(f[0], f[1], f[2], f[3]);
        *(float4*)(to + col + 4) = make_float4(f[4], f[5], f[6], f[7]);
    }
}

// A row is held by TPR threads, CH chunks of 8 elements each (chunk c of thread t: columns (t + c TPR) 8 ..).  Resident blocks walk the rows; the next row's loads are
// issued before the current row is worked on, and weight and bias wait in shared memory as fp32.
template <int DT, int TPR, int CH, bool VEC>
__global__ void __launch_bounds__(TPR > 128 ? TPR : 128) layer_norm_kernel(const __grid_constant__ LnArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int SUB = TPR < 32 ? TPR : 32, W = TPR * CH * 8, WARPS = TPR > 32 ? TPR / 32 : 1;
    using Row = Row8<DT, VEC, SUB>;
    extern __shared__ __align__(128) uint8_t dyn[];
    float* pw = (float*)dyn;
    float* pb = pw + W;
    void* stage = dyn + 2 * W * sizeof(float) + (threadIdx.x >> 5) * Stage8<DT, VEC>::kBytes;
    __shared__ float buf[2][2][WARPS];
    const int t = threadIdx.x % TPR, groups = blockDim.x / TPR, grp = threadIdx.x / TPR, lane = threadIdx.x & 31;
    const int64_t step = (int64_t)gridDim.x * groups;
    int64_t row = (int64_t)blockIdx.x * groups + grp;
    Row x[CH];
#pragma unroll
    for (int c = 0; c < CH; c++) x[c].load((const T*)a.x, a.ldx, row, a.rows, (t + c * TPR) * 8, a.cols);
    stage_params<DT, W>(a.w, a.wf32, a.cols, 1.0f, pw);
    stage_params<DT, W>(a.b, a.wf32, a.cols, 0.0f, pb);
    __syncthreads();
    // a sum over the threads of the row; the buffers alternate from sum to sum and from row to row: one barrier each
    auto row_sum = [&](float v, float* b) {
#pragma unroll
        for (int o = SUB / 2; o >= 1; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
        if constexpr (TPR > 32) {
            if (lane == 0) b[threadIdx.x >> 5] = v;
            __syncthreads();
            v = b[0];
#pragma unroll
            for (int i = 1; i < WARPS; i++) v += b[i];
        }
        return v;
    };
    // (groups of a block run the same number of steps: `row - grp` decides)
    for (int phase = 0; row - grp < a.rows; row += step, phase ^= 1) {
        float2 v[CH][4];
        uint32_t top[CH];
#pragma unroll
        for (int c = 0; c < CH; c++) {
            uint32_t raw[RawRegs<DT>::N];
            x[c].get(stage, raw);
            raw_to_pairs<DT>(raw, v[c]);
            top[c] = absmax8<DT>(raw);
        }
#pragma unroll
        for (int c = 0; c < CH; c++) x[c].load((const T*)a.x, a.ldx, row + step, a.rows, (t + c * TPR) * 8, a.cols);
        float2 s2 = splat2(0.0f);
#pragma unroll
        for (int c = 0; c < CH; c++) s2 = add2(s2, add2(add2(v[c][0], v[c][1]), add2(v[c][2], v[c][3])));
        float mean = row_sum(s2.x + s2.y, buf[phase][0]) * a.inv_cols;
        float2 q2 = splat2(0.0f);
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int col = (t + c * TPR) * 8;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float2 d = add2(v[c][i], splat2(-mean));
                if (VEC) { if (col >= a.cols) d = splat2(0.0f); }
                else {
                    if (col + 2 * i >= a.cols) d.x = 0.0f;
                    if (col + 2 * i + 1 >= a.cols) d.y = 0.0f;
                }
                q2 = fma2(d, d, q2);
            }
        }
        // rsqrtf: at most 2 steps off
        const float rstd = rsqrtf(row_sum(q2.x + q2.y, buf[phase][1]) * a.inv_cols + a.eps);
        const bool live = row < a.rows;
        uint32_t last = top_byte8<DT>();
        // what the backward pass has to take off the kept values, and 1 / deviation: centred codes have lost the mean already
        if (live && t == 0 && a.stats) ((float2*)a.stats)[row] = make_float2(a.center ? 0.0f : mean, rstd);
        if (a.center) {
            // (in place: what follows is written for the deviations and a mean of 0; they are fp32 and restored as such, so the
            // range of x's type does not bound them)
            last = top_byte8<GACT_F32>();
#pragma unroll
            for (int c = 0; c < CH; c++) {
                const int col = (t + c * TPR) * 8;
                float m = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    v[c][i] = add2(v[c][i], splat2(-mean));
                    if (VEC) { if (col >= a.cols) v[c][i] = splat2(0.0f); }
                    else {
                        if (col + 2 * i >= a.cols) v[c][i].x = 0.0f;
                        if (col + 2 * i + 1 >= a.cols) v[c][i].y = 0.0f;
                    }
                    m = absmax3(m, v[c][i]);
                }
                top[c] = __float_as_uint(m) & 0x7fffffffu;
            }
            mean = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int col = (t + c * TPR) * 8;
            float2 o[4];
            if (a.codes) {
                uint32_t byte;
                const uint64_t chunk = (uint64_t)row * a.chunks + (t + c * TPR);
                const uint2 q = a.stochastic ? codes8<true>(v[c], top[c], a.noise, a.noise.high(), chunk, byte, last)
                                             : codes8<false>(v[c], top[c], a.noise, make_uint2(0u, 0u), chunk, byte, last);
                if (live && t + c * TPR < a.chunks) {
                    st_stream_u2(a.codes + chunk * 8, q);
                    if ((t & 3) == 0) a.scales[chunk >> 2] = (uint8_t)byte;
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const float4 w = *(const float4*)(pw + col + 2 * i), b = *(const float4*)(pb + col + 2 * i);
                o[i] = fma2(mul2(add2(v[c][i], splat2(-mean)), splat2(rstd)), make_float2(w.x, w.y), make_float2(b.x, b.y));
                o[i + 1] = fma2(mul2(add2(v[c][i + 1], splat2(-mean)), splat2(rstd)), make_float2(w.z, w.w), make_float2(b.z, b.w));
            }
            Row::store((T*)a.y, a.cols, row, a.rows, col, a.cols, stage, o);
        }
    }
}

template <int DT, int TPR, int CH, bool VEC> static int launch_ln_vec(const LnArgs& a, cudaStream_t s) {
    auto* k = layer_norm_kernel<DT, TPR, CH, VEC>;
    constexpr int kBlock = TPR > 32 ? TPR : 128;
    constexpr int kSmem = 2 * TPR * CH * 8 * (int)sizeof(float) + kBlock / 32 * Stage8<DT, VEC>::kBytes;
    static std::atomic<bool> allowed[kMaxDevices];
    if (kSmem > 40 * 1024 && !allow_smem(k, kSmem, allowed)) return GACT_ERR_LAUNCH;
    static std::atomic<int> cache[kMaxDevices];
    const int64_t per = kBlock / TPR, want = (a.rows + per - 1) / per;
    const int64_t most = (int64_t)sm_count() * resident_blocks(k, kBlock, kSmem, cache);
    k<<<(unsigned)(want < most ? want : most), kBlock, kSmem, s>>>(a);
    return cudaGetLastError() == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
}
template <int DT, int TPR, int CH> static int launch_ln(const LnArgs& a, bool vec, cudaStream_t s) {
    return vec ? launch_ln_vec<DT, TPR, CH, true>(a, s) : launch_ln_vec<DT, TPR, CH, false>(a, s);
}
// Many rows: 32 elements per thread, so that the reductions, the row's scalars and the addresses (about 100 instructions per
// thread and row) do not bound the kernel.  Few rows: latency counts, and every row is spread over as many threads as it has
// chunks.  Measured, 32 elements a thread / spread in us, bf16: 600 rows of 1024 3.5 / 3.1, of 4096 7.2 / 6.8; 1200 rows of 512
// 3.5 / 3.1, of 1024 4.0 / 4.1, of 4096 9.9 / 10.4; 4800 rows of 512 5.5 / 5.6, of 1024 8.4 / 8.6, of 4096 23.9 / 30.2.
template <int DT> static int dispatch_ln(const LnArgs& a, bool vec, cudaStream_t s) {
    const int h = a.cols;
    if (vec && a.rows > (int64_t)sm_count() * 8 && h > 64 && h <= 8192) {
        if (h <= 128) return launch_ln_vec<DT, 8, 2, true>(a, s);
        if (h <= 256) return launch_ln_vec<DT, 8, 4, true>(a, s);
        if (h <= 512) return launch_ln_vec<DT, 16, 4, true>(a, s);
        if (h <= 1024) return launch_ln_vec<DT, 32, 4, true>(a, s);
        if (h <= 2048) return launch_ln_vec<DT, 64, 4, true>(a, s);
        if (h <= 4096) return launch_ln_vec<DT, 128, 4, true>(a, s);
        return launch_ln_vec<DT, 256, 4, true>(a, s);
    }
    if (h <= 32) return launch_ln<DT, 4, 1>(a, vec, s);
    if (h <= 64) return launch_ln<DT, 8, 1>(a, vec, s);
    if (h <= 128) return launch_ln<DT, 16, 1>(a, vec, s);
    if (h <= 256) return launch_ln<DT, 32, 1>(a, vec, s);
    if (h <= 512) return launch_ln<DT, 64, 1>(a, vec, s);
    if (h <= 1024) return launch_ln<DT, 128, 1>(a, vec, s);
    if (h <= 2048) return launch_ln<DT, 256, 1>(a, vec, s);
    if (h <= 4096) return launch_ln<DT, 512, 1>(a, vec, s);
    if (h <= 8192) return launch_ln<DT, 512, 2>(a, vec, s);
    return launch_ln<DT, 512, 4>(a, vec, s);
}

constexpr int kLnBwdRows = 2;                       // rows a block (or row group) of the plain kernel works on side by side

// ---- backward -------------------------------------------------------------------------------------------------------
struct LnBwdArgs {
    const void* dy; int64_t ldy;
    const void* x; int64_t ldx;                       // the input itself, or null:
    const int8_t* codes; const uint8_t* scales; int chunks;
    const float* stats;
    const void* w; int wf32;
    int64_t rows; int cols; float inv_cols;
    void* dx;                                          // null: weight gradients only
    float* partial;                                    // [gridDim][2 * width]: dw, db; null: no weight gradients
    int width;
    uint32_t wait_limit; int withhold; int* report;    // rings: bounded waits; diagnostics; the host's word
};

// Wherever the rings below were not measured to be faster.  A thread owns CH fixed chunks of 8 columns, so the weight gradients of a block's rows stay in its registers; a block
// walks the rows, R of them (per row group) side by side: one barrier serves 2 R sums, and the next R rows' loads are issued
// before the current ones are worked on.  Block sums go to `partial`, added up in a fixed order afterwards: no atomics.
template <int DT, int TPR, int CH, int R, bool VEC, bool COMP>
__global__ void __launch_bounds__(TPR > 128 ? TPR : 128, 512 / (TPR > 128 ? TPR : 128)) layer_norm_backward_kernel(const __grid_constant__ LnBwdArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int BLOCK = TPR > 32 ? TPR : 128, GROUPS = BLOCK / TPR, SUB = TPR < 32 ? TPR : 32;
    using Row = Row8<DT, VEC, SUB>;
    __shared__ float2 buf[2][R][TPR > 32 ? TPR / 32 : 1];
    __shared__ __align__(16) uint8_t staging[VEC ? 16 : BLOCK / 32 * Stage8<DT, VEC>::kBytes];
    __shared__ float fold[GROUPS > 1 ? BLOCK * 16 : 1];
    void* stage = staging + (threadIdx.x >> 5) * Stage8<DT, VEC>::kBytes;
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR, lane = threadIdx.x & 31;
    float2 w[CH][4], dw[CH][4], db[CH][4];
#pragma unroll
    for (int c = 0; c < CH; c++) {
        float f[8];
        load_param8<DT>(a.w, a.wf32, (t + c * TPR) * 8, a.cols, 1.0f, f);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            w[c][i] = make_float2(f[2 * i], f[2 * i + 1]);
            dw[c][i] = db[c][i] = splat2(0.0f);
        }
    }
    Row py[R][CH], px[COMP ? 1 : R][COMP ? 1 : CH];
    uint2 pq[R][CH];
    uint32_t pe[R][CH];
    float2 ps[R];
    auto fetch = [&](int64_t base) {
#pragma unroll
        for (int k = 0; k < R; k++) {
            const int64_t row = base + k * GROUPS + grp;
            const bool live = row < a.rows;
            ps[k] = live ? ld_ahead_float2((const float2*)a.stats + row) : make_float2(0.0f, 0.0f);
#pragma unroll
            for (int c = 0; c < CH; c++) {
                py[k][c].load((const T*)a.dy, a.ldy, row, a.rows, (t + c * TPR) * 8, a.cols);
                if constexpr (COMP) {
                    pq[k][c] = make_uint2(0u, 0u);
                    pe[k][c] = 1;
                    if (live && t + c * TPR < a.chunks) {
                        const int64_t chunk = row * a.chunks + (t + c * TPR);
                        pq[k][c] = ld_stream_u2(a.codes + chunk * 8);
                        pe[k][c] = ld_ahead_byte(a.scales + (chunk >> 2));
                    }
                } else {
                    px[k][c].load((const T*)a.x, a.ldx, row, a.rows, (t + c * TPR) * 8, a.cols);
                }
            }
        }
    };
    const int64_t step = (int64_t)gridDim.x * GROUPS * R;
    int64_t r0 = (int64_t)blockIdx.x * GROUPS * R;
    fetch(r0);
    for (int phase = 0; r0 < a.rows; r0 += step, phase ^= 1) {
        float2 g[R][CH][4], xh[R][CH][4];
        float2 s[R];
        float rs[R];
#pragma unroll
        for (int k = 0; k < R; k++) {
            rs[k] = ps[k].y;
            const float2 off = splat2(-ps[k].x * ps[k].y);
#pragma unroll
            for (int c = 0; c < CH; c++) {
                uint32_t raw[RawRegs<DT>::N];
                py[k][c].get(stage, raw);
                raw_to_pairs<DT>(raw, g[k][c]);
                // x^ = x' r - mean r; a code is a small integer and its scale a power of two, so x' r is one product
                float2 up;
                if constexpr (COMP) {
                    code_pairs(pq[k][c], xh[k][c]);
                    up = splat2(scale_down8(pe[k][c]) * rs[k]);
                } else {
                    px[k][c].get(stage, raw);
                    raw_to_pairs<DT>(raw, xh[k][c]);
                    up = splat2(rs[k]);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) xh[k][c][i] = fma2(xh[k][c][i], up, off);
            }
        }
        fetch(r0 + step);
#pragma unroll
        for (int k = 0; k < R; k++) {
            float2 s1 = splat2(0.0f), s2 = splat2(0.0f);
#pragma unroll
            for (int c = 0; c < CH; c++) {
                const int col = (t + c * TPR) * 8;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    // a column past the end has dy = 0, but a NaN scale of the row's last block must not leak out of it
                    if (VEC) { if (col >= a.cols) xh[k][c][i] = splat2(0.0f); }
                    else {
                        if (col + 2 * i >= a.cols) xh[k][c][i].x = 0.0f;
                        if (col + 2 * i + 1 >= a.cols) xh[k][c][i].y = 0.0f;
                    }
                    dw[c][i] = fma2(g[k][c][i], xh[k][c][i], dw[c][i]);
                    db[c][i] = add2(db[c][i], g[k][c][i]);
                    g[k][c][i] = mul2(g[k][c][i], w[c][i]);
                    s1 = add2(s1, g[k][c][i]);
                    s2 = fma2(g[k][c][i], xh[k][c][i], s2);
                }
            }
            s[k] = make_float2(s1.x + s1.y, s2.x + s2.y);
#pragma unroll
            for (int o = SUB / 2; o >= 1; o >>= 1) {
                s[k].x += __shfl_xor_sync(kFull, s[k].x, o);
                s[k].y += __shfl_xor_sync(kFull, s[k].y, o);
            }
        }
        if constexpr (TPR > 32) {
            constexpr int W = TPR / 32;
            if (lane == 0) {
#pragma unroll
                for (int k = 0; k < R; k++) buf[phase][k][threadIdx.x >> 5] = s[k];
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < R; k++) {
                // every lane adds the warps' sums itself (a broadcast read each), in warp order
                s[k] = buf[phase][k][0];
#pragma unroll
                for (int i = 1; i < W; i++) s[k] = add2(s[k], buf[phase][k][i]);
            }
        }
        if (a.dx) {
#pragma unroll
            for (int k = 0; k < R; k++) {
                const int64_t row = r0 + k * GROUPS + grp;
                // r (g - c1 - x^ c2)
                const float2 c1 = splat2(-s[k].x * a.inv_cols), c2 = splat2(-s[k].y * a.inv_cols);
#pragma unroll
                for (int c = 0; c < CH; c++) {
                    float2 o[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) o[i] = mul2(fma2(xh[k][c][i], c2, add2(g[k][c][i], c1)), splat2(rs[k]));
                    Row::store((T*)a.dx, a.cols, row, a.rows, (t + c * TPR) * 8, a.cols, stage, o);
                }
            }
        }
    }
    if (!a.partial) return;
    if constexpr (GROUPS > 1) {
        // fold the row groups of the block: fold[j][thread]
#pragma unroll
        for (int i = 0; i < 4; i++) {
            fold[(4 * i) * BLOCK + threadIdx.x] = dw[0][i].x;
            fold[(4 * i + 1) * BLOCK + threadIdx.x] = dw[0][i].y;
            fold[(4 * i + 2) * BLOCK + threadIdx.x] = db[0][i].x;
            fold[(4 * i + 3) * BLOCK + threadIdx.x] = db[0][i].y;
        }
        __syncthreads();
        if (grp == 0) {
            for (int k = 1; k < GROUPS; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float* f = fold + k * TPR + t;
                    dw[0][i] = add2(dw[0][i], make_float2(f[(4 * i) * BLOCK], f[(4 * i + 1) * BLOCK]));
                    db[0][i] = add2(db[0][i], make_float2(f[(4 * i + 2) * BLOCK], f[(4 * i + 3) * BLOCK]));
                }
        }
    }
    if (grp == 0) {
        float* p = a.partial + (int64_t)blockIdx.x * 2 * a.width;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int col = (t + c * TPR) * 8;
            if (col >= a.width) continue;
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                *(float4*)(p + col + 2 * i) = make_float4(dw[c][i].x, dw[c][i].y, dw[c][i + 1].x, dw[c][i + 1].y);
                *(float4*)(p + a.width + col + 2 * i) = make_float4(db[c][i].x, db[c][i].y, db[c][i + 1].x, db[c][i + 1].y);
            }
        }
    }
}

// ---- long rows: rings of bulk copies ----------------------------------------------------------------------------------
// Rows that start on 16-byte boundaries are brought into shared memory by bulk copies (one elected thread, one instruction
// per row and tensor), kRingStages rows deep, and worked on there: a row is read from shared memory as often as it is needed,
// so it costs no registers while it waits and the loads in flight do not depend on the number of warps.  The block works on
// one row.  Waits are bounded (see mbar_wait); one that runs out is recorded and the block goes on to its end without waiting.
constexpr int kRingStages = 3;
__device__ int g_norm_error = 0;

struct RowRing {
    uint32_t bar, limit; volatile int* dead; uint32_t issued, taken;      // rows issued and taken so far
    __device__ __forceinline__ uint32_t stage(uint32_t n) const { return n % kRingStages; }
    // the next row to work on has landed; returns its stage
    __device__ __forceinline__ uint32_t take() {
        const uint32_t s = stage(taken);
        mbar_wait(bar + 8 * s, (taken / kRingStages) & 1, limit, dead);
        taken++;
        return s;
    }
    // elected thread: announces a row of `bytes`; the copies follow
    __device__ __forceinline__ uint32_t announce(uint32_t bytes) {
        const uint32_t s = stage(issued);
        mbar_expect_tx(bar + 8 * s, bytes);
        issued++;
        return s;
    }
    // elected thread, at the end: a ring that gave up waits (again bounded) for the copies that may still be in flight
    __device__ __forceinline__ void close(int* host_word) {
        if (!*dead) return;
        report_wait(&g_norm_error, host_word);
        for (uint32_t j = issued > (uint32_t)kRingStages ? issued - kRingStages : 0; j < issued; j++)
            mbar_drain(bar + 8 * (j % kRingStages), (j / kRingStages) & 1, limit);
    }
};
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
template <int DT> __device__ __forceinline__ void take_raw(const uint8_t* row, int chunk, uint32_t (&raw)[RawRegs<DT>::N]) {
    const uint4* p = (const uint4*)(row + chunk * 8 * Elem<DT>::kBytes);
    const uint4 a = p[0];
    raw[0] = a.x; raw[1] = a.y; raw[2] = a.z; raw[3] = a.w;
    if constexpr (DT == GACT_F32) {
        const uint4 b = p[1];
        raw[4] = b.x; raw[5] = b.y; raw[6] = b.z; raw[7] = b.w;
    }
}

// dy and the codes of a row are read twice, before and after the sums; the weight gradients of a thread's columns stay in its
// registers.
template <int DT, int TPR, int CH>
__global__ void __launch_bounds__(TPR) layer_norm_backward_ring_kernel(const __grid_constant__ LnBwdArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int W = TPR * CH * 8, WARPS = TPR / 32, N = RawRegs<DT>::N;
    constexpr int YROW = W * Elem<DT>::kBytes, ROW = YROW + W;
    extern __shared__ __align__(128) uint8_t dyn[];               // weights (fp32), rings
    float* pw = (float*)dyn;
    __shared__ __align__(8) uint64_t bars[kRingStages];
    __shared__ float2 buf[2][WARPS];
    __shared__ volatile int dead;
    const int t = threadIdx.x, lane = threadIdx.x & 31;
    uint8_t* ring = dyn + W * sizeof(float);
    if (t == 0) {
        dead = 0;
        for (int i = 0; i < kRingStages; i++) mbar_init(smem_addr(bars + i), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    RowRing r{smem_addr(bars), a.wait_limit, &dead, 0, 0};
    const int64_t step = gridDim.x;
    int64_t row = blockIdx.x;
    const uint32_t ybytes = (uint32_t)a.cols * Elem<DT>::kBytes, xbytes = (uint32_t)a.chunks * 8;
    auto issue = [&](int64_t w) {
        // (a ring that gave up issues nothing more: announcing bytes on a phase that never completed would be a second arrival
        // on it, which faults)
        if (w < a.rows && !dead) {
            const uint32_t s = r.announce(ybytes + xbytes), to = smem_addr(ring + s * ROW), bar = r.bar + 8 * s;
            if (!(a.withhold && w == 0)) bulk_copy(to, (const T*)a.dy + w * a.ldy, ybytes, bar);      // (withhold: diagnostics)
            bulk_copy(to + YROW, a.codes + w * a.chunks * 8, xbytes, bar);
        }
    };
    if (t == 0)
        for (int i = 0; i < kRingStages - 1; i++) issue(row + i * step);
    // statistics and scales are a few bytes per row: plain loads, one row ahead
    float2 ps = splat2(0.0f);
    uint32_t pe[CH];
    auto fetch = [&](int64_t w) {
        if (w < a.rows) {
            ps = ld_ahead_float2((const float2*)a.stats + w);
            const uint8_t* p = a.scales + ((w * a.chunks + t) >> 2);
#pragma unroll
            for (int c = 0; c < CH; c++)
                if (t + c * TPR < a.chunks) pe[c] = ld_ahead_byte(p + c * (TPR / 4));
        }
    };
#pragma unroll
    for (int c = 0; c < CH; c++) pe[c] = 1;
    fetch(row);
    stage_params<DT, W>(a.w, a.wf32, a.cols, 1.0f, pw);
    __syncthreads();
    float2 dw[CH][4], db[CH][4];
#pragma unroll
    for (int c = 0; c < CH; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) dw[c][i] = db[c][i] = splat2(0.0f);
    T* dx = (T*)a.dx + row * a.cols + t * 8;
    for (int phase = 0; row < a.rows; row += step, phase ^= 1) {
        const float rs = ps.y, off = -ps.x * ps.y;
        float up[CH];
#pragma unroll
        for (int c = 0; c < CH; c++) up[c] = scale_down8(pe[c]) * rs;
        fetch(row + step);
        const uint8_t* in = ring + r.take() * ROW;
        // dy and x^ of chunk c: x^ = x' r - mean r; a code is a small integer and its scale a power of two, so x' r is one product
        auto expand = [&](int c, float2 (&g)[4], float2 (&xh)[4]) {
            uint32_t raw[N];
            take_raw<DT>(in, t + c * TPR, raw);
            raw_to_pairs<DT>(raw, g);
            code_pairs(*(const uint2*)(in + YROW + (t + c * TPR) * 8), xh);
#pragma unroll
            for (int i = 0; i < 4; i++) xh[i] = fma2(xh[i], splat2(up[c]), splat2(off));
        };
        float2 s1 = splat2(0.0f), s2 = splat2(0.0f);
#pragma unroll
        for (int c = 0; c < CH; c++) {
            if ((t + c * TPR) * 8 < a.cols) {                    // (past the row: whatever the ring holds)
                float2 g[4], xh[4];
                expand(c, g, xh);
                const float* pc = pw + (t + c * TPR) * 8;
                const float4 wa = *(const float4*)pc, wb = *(const float4*)(pc + 4);
                const float2 w[4] = {make_float2(wa.x, wa.y), make_float2(wa.z, wa.w), make_float2(wb.x, wb.y), make_float2(wb.z, wb.w)};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    dw[c][i] = fma2(g[i], xh[i], dw[c][i]);
                    db[c][i] = add2(db[c][i], g[i]);
                    g[i] = mul2(g[i], w[i]);
                    s1 = add2(s1, g[i]);
                    s2 = fma2(g[i], xh[i], s2);
                }
            }
        }
        float2 s = make_float2(s1.x + s1.y, s2.x + s2.y);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) s = add2(s, make_float2(__shfl_xor_sync(kFull, s.x, o), __shfl_xor_sync(kFull, s.y, o)));
        // (two buffers in turn: one barrier per row is enough)
        if (lane == 0) buf[phase][threadIdx.x >> 5] = s;
        __syncthreads();
        s = buf[phase][0];
#pragma unroll
        for (int i = 1; i < WARPS; i++) s = add2(s, buf[phase][i]);
        // every thread is past the row before this one: its stage takes the row kRingStages - 1 steps on
        if (t == 0) issue(row + (kRingStages - 1) * step);
        if (a.dx) {
            // r (g - c1 - x^ c2)
            const float2 e1 = splat2(-s.x * a.inv_cols * rs), e2 = splat2(-s.y * a.inv_cols * rs);
#pragma unroll
            for (int c = 0; c < CH; c++) {
                if ((t + c * TPR) * 8 < a.cols) {
                    float2 g[4], xh[4];
                    expand(c, g, xh);
                    const float* pc = pw + (t + c * TPR) * 8;
                    const float4 wa = *(const float4*)pc, wb = *(const float4*)(pc + 4);
                    const float2 w[4] = {make_float2(wa.x, wa.y), make_float2(wa.z, wa.w), make_float2(wb.x, wb.y), make_float2(wb.z, wb.w)};
#pragma unroll
                    for (int i = 0; i < 4; i++) g[i] = fma2(xh[i], e2, fma2(mul2(g[i], w[i]), splat2(rs), e1));
                    uint32_t raw[N];
                    pairs_to_raw<DT>(g, raw);
                    st_stream_u4(dx + c * TPR * 8, make_uint4(raw[0], raw[1], raw[2], raw[3]));
                    if constexpr (DT == GACT_F32) st_stream_u4(dx + c * TPR * 8 + 4, make_uint4(raw[4], raw[5], raw[6], raw[7]));
                }
            }
        }
        dx += step * a.cols;
    }
    if (t == 0) r.close(a.report);
    if (!a.partial) return;
    float* p = a.partial + (int64_t)blockIdx.x * 2 * a.width;
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const int col = (t + c * TPR) * 8;
        if (col < a.width) {
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                *(float4*)(p + col + 2 * i) = make_float4(dw[c][i].x, dw[c][i].y, dw[c][i + 1].x, dw[c][i + 1].y);
                *(float4*)(p + a.width + col + 2 * i) = make_float4(db[c][i].x, db[c][i].y, db[c][i + 1].x, db[c][i + 1].y);
            }
        }
    }
}

// Rings take the place of the plain kernel's shape of 512 threads a row, where many rows let a block run ahead.  Measured, ring / plain
// in us, from codes: bf16 4800 x 2056 21.7 / 27.6, 4800 x 4096 31.9 / 30.7, 8192 x 3200 38.3 / 44.2, 65536 x 4096 266 / 316; fp32 (twice
// the bytes per row) 8192 x 4096 67 / 63, 16384 x 4096 115 / 116, 65536 x 4096 408 / 467.  At 2400 rows they lose (4096 columns
// 25.5 / 21), with other shapes of the plain kernel too (65536 x 2048 175 / 140, x 1024 127 / 72, x 8192 693 / 522), and from x
// itself (65536 x 4096 329 / 290).  The diagnostics hook, which is there to see a copy lost, takes them wherever they fit.
constexpr int kRingCols = 4096;
static bool ln_ring(bool vec, bool codes, int dtype, int64_t rows, int64_t cols, bool forced) {
    if (!vec || !codes || cols > kRingCols) return false;
    return forced || (cols > 2048 && rows > (int64_t)sm_count() * (dtype == GACT_F32 ? 96 : 32));
}

// Shapes and blocks of the backward pass.  The number of blocks decides how many partial sums there are (2 x cols floats per
// block), so it must not depend on anything but the sizes: 512 threads per SM for the plain kernel, and for the rings as many
// blocks as their registers and shared memory let an SM hold.
struct LnBwdShape { int block, rows_per_step, per_sm; };
static LnBwdShape ln_bwd_shape(bool ring, int64_t cols) {
    if (ring) return {128, 1, 4};
    const int tpr = cols <= 32 ? 4 : cols <= 64 ? 8 : cols <= 128 ? 16 : cols <= 256 ? 32 : cols <= 512 ? 64 : cols <= 1024 ? 128 : cols <= 2048 ? 256 : 512;
    const int block = tpr > 32 ? tpr : 128;
    return {block, block / tpr * (cols <= 4096 ? kLnBwdRows : 1), 512 / block};
}
static int64_t ln_bwd_blocks(bool ring, int64_t rows, int64_t cols) {
    const LnBwdShape p = ln_bwd_shape(ring, cols);
    const int64_t want = (rows + p.rows_per_step - 1) / p.rows_per_step, most = (int64_t)sm_count() * p.per_sm;
    return want < most ? want : most;
}

template <int DT> static int launch_ln_bwd_ring(const LnBwdArgs& a, int64_t blocks, cudaStream_t s) {
    constexpr int TPR = 128, kSmem = kRingCols * ((int)sizeof(float) + kRingStages * (Elem<DT>::kBytes + 1));
    auto* k = layer_norm_backward_ring_kernel<DT, TPR, kRingCols / (TPR * 8)>;
    static std::atomic<bool> allowed[kMaxDevices];
    if (!allow_smem(k, kSmem, allowed)) return GACT_ERR_LAUNCH;
    k<<<(unsigned)blocks, TPR, kSmem, s>>>(a);
    return cudaGetLastError() == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
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
template <int DT> static int dispatch_ln_bwd(const LnBwdArgs& a, bool vec, bool ring, int64_t blocks, cudaStream_t s) {
    const int h = a.cols;
    if (ring) return launch_ln_bwd_ring<DT>(a, blocks, s);
    if (h <= 32) return launch_ln_bwd<DT, 4, 1, kLnBwdRows>(a, vec, blocks, s);
    if (h <= 64) return launch_ln_bwd<DT, 8, 1, kLnBwdRows>(a, vec, blocks, s);
    if (h <= 128) return launch_ln_bwd<DT, 16, 1, kLnBwdRows>(a, vec, blocks, s);
    if (h <= 256) return launch_ln_bwd<DT, 32, 1, kLnBwdRows>(a, vec, blocks, s);
    if (h <= 512) return launch_ln_bwd<DT, 64, 1, kLnBwdRows>(a, vec, blocks, s);
    if (h <= 1024) return launch_ln_bwd<DT, 128, 1, kLnBwdRows>(a, vec, blocks, s);
    if (h <= 2048) return launch_ln_bwd<DT, 256, 1, kLnBwdRows>(a, vec, blocks, s);
    if (h <= 4096) return launch_ln_bwd<DT, 512, 1, kLnBwdRows>(a, vec, blocks, s);
    if (h <= 8192) return launch_ln_bwd<DT, 512, 2, 1>(a, vec, blocks, s);
    return launch_ln_bwd<DT, 512, 4, 1>(a, vec, blocks, s);
}

// ---- sums of partials over the blocks that wrote them ---------------------------------------------------------------
constexpr int kRCols = 32;
struct ReduceArgs { const float* partial; int parts; int64_t width; void* out0; int64_t n0; void* out1; int64_t n1; };

template <int DT, int kRRows>
__global__ void __launch_bounds__(kRCols * kRRows) reduce_columns_kernel(const ReduceArgs a) {
    __shared__ float buf[kRRows][kRCols + 1];
    const int tx = threadIdx.x % kRCols, ty = threadIdx.x / kRCols;
    const int64_t c = (int64_t)blockIdx.x * kRCols + tx;
    float sum = 0.0f;
    if (c < a.width) {
        const float* q = a.partial + (int64_t)ty * a.width + c;
        const int64_t step = (int64_t)kRRows * a.width;
        int p = ty;
        // eight loads in flight per thread: the partials are few and the kernel is all latency
        for (; p + 7 * kRRows < a.parts; p += 8 * kRRows, q += 8 * step) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = q[i * step];
#pragma unroll
            for (int i = 0; i < 8; i++) sum += v[i];
        }
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = p + i * kRRows < a.parts ? q[i * step] : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) sum += v[i];
    }
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

template <int DT> static void launch_reduce(const ReduceArgs& a, int chains, cudaStream_t s) {
    const unsigned blocks = (unsigned)((a.width + kRCols - 1) / kRCols);
    if (chains == kSumChains) reduce_columns_kernel<DT, kSumChains><<<blocks, kRCols * kSumChains, 0, s>>>(a);
    else reduce_columns_kernel<DT, 32><<<blocks, kRCols * 32, 0, s>>>(a);
}
int reduce_columns(const float* partial, int parts, int64_t width, void* out0, int64_t n0, void* out1, int64_t n1, int dtype, int chains, cudaStream_t s) {
    const ReduceArgs a{partial, parts, width, out0, n0, out1, n1};
    switch (dtype) {
    case GACT_F32: launch_reduce<GACT_F32>(a, chains, s); break;
    case GACT_F16: launch_reduce<GACT_F16>(a, chains, s); break;
    default: launch_reduce<GACT_BF16>(a, chains, s); break;
    }
    return cudaGetLastError() == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
}

int norm_error_word() {
    int v = 0;
    return cudaMemcpyFromSymbol(&v, g_norm_error, sizeof(int)) == cudaSuccess ? v : -1;
}
int norm_error_clear() {
    const int zero = 0;
    return cudaMemcpyToSymbol(g_norm_error, &zero, sizeof(int)) == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
}

static bool ln_sizes_ok(int64_t rows, int64_t cols) {
    return rows >= 0 && cols >= 1 && cols <= GACT_LAYER_NORM_MAX_COLS && rows <= GACT_MAX_ELEMENTS / pitch8(cols) && rows <= (1LL << 30);
}
static bool param_ok(const void* p, int dtype) { return !p || ((uintptr_t)p & (uintptr_t)(elem_bytes_of(dtype) - 1)) == 0; }

}  // namespace gact

using namespace gact;

extern "C" int gact_layer_norm(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, const void* weight, const void* bias,
                               int param_dtype, double eps, void* y, float* stats, void* codes, void* scales, int rounding,
                               uint64_t seed, void* stream) {
    if (dtype < GACT_F32 || dtype > GACT_BF16 || (param_dtype != dtype && param_dtype != GACT_F32)) return GACT_ERR_DTYPE;
    if (!ln_sizes_ok(rows, cols) || ld < cols) return GACT_ERR_SIZE;
    if (rows == 0) return GACT_OK;
    if (const int st = rounding_status(rounding, seed, GACT_CODES_STOCHASTIC | GACT_CODES_DEVICE_SEED | GACT_CODES_CENTERED)) return st;
    if (!x || !y || (codes && !scales)) return GACT_ERR_NULL;
    const uintptr_t em = (uintptr_t)(elem_bytes_of(dtype) - 1);
    if (((uintptr_t)x & em) || ((uintptr_t)y & em) || ((uintptr_t)codes & 31) || ((uintptr_t)stats & 7) || !param_ok(weight, param_dtype) ||
        !param_ok(bias, param_dtype))
        return GACT_ERR_ALIGN;
    LnArgs a;
    a.x = x; a.ldx = ld; a.w = weight; a.b = bias; a.wf32 = param_dtype == GACT_F32;
    a.rows = rows; a.cols = (int)cols; a.inv_cols = 1.0f / (float)cols; a.eps = (float)eps;
    a.y = y; a.stats = stats; a.codes = (int8_t*)codes; a.scales = (uint8_t*)scales;
    a.chunks = (int)(pitch8(cols) / 8); a.noise = Noise8::of(seed, rounding & GACT_CODES_DEVICE_SEED, 0);
    a.stochastic = (rounding & GACT_CODES_STOCHASTIC) != 0; a.center = codes && (rounding & GACT_CODES_CENTERED);
    const bool vec = rows_aligned(x, ld, cols, elem_bytes_of(dtype)) && rows_aligned(y, cols, cols, elem_bytes_of(dtype));
    cudaStream_t s = (cudaStream_t)stream;
    switch (dtype) {
    case GACT_F32: return dispatch_ln<GACT_F32>(a, vec, s);
    case GACT_F16: return dispatch_ln<GACT_F16>(a, vec, s);
    default: return dispatch_ln<GACT_BF16>(a, vec, s);
    }
}

extern "C" int64_t gact_layer_norm_backward_scratch_bytes(int64_t rows, int64_t cols) {
    if (!ln_sizes_ok(rows, cols)) return -1;
    // (whichever kernel the operands' type and alignment pick)
    const int64_t a = cols <= kRingCols ? ln_bwd_blocks(true, rows, cols) : 0, b = ln_bwd_blocks(false, rows, cols);
    return (a > b ? a : b) * 2 * ((cols + 7) / 8 * 8) * (int64_t)sizeof(float);
}

extern "C" int gact_layer_norm_backward(const void* dy, int dtype, int64_t rows, int64_t cols, int64_t ld_dy, const void* x, int64_t ld_x,
                                        const void* codes, const void* scales, const float* stats, const void* weight,
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
    if (!dy || !stats || (!x && (!codes || !scales)) || (params && !scratch)) return GACT_ERR_NULL;
    if (!dx && !params) return GACT_OK;
    const uintptr_t em = (uintptr_t)(elem_bytes_of(dtype) - 1);
    if (((uintptr_t)dy & em) || ((uintptr_t)x & em) || ((uintptr_t)dx & em) || ((uintptr_t)codes & 31) || ((uintptr_t)scratch & 15) || ((uintptr_t)stats & 7) ||
        !param_ok(weight, param_dtype) || !param_ok(dweight, param_dtype) || !param_ok(dbias, param_dtype))
        return GACT_ERR_ALIGN;
    LnBwdArgs a;
    a.dy = dy; a.ldy = ld_dy; a.x = x; a.ldx = ld_x; a.codes = x ? nullptr : (const int8_t*)codes; a.scales = (const uint8_t*)scales;
    a.chunks = (int)(pitch8(cols) / 8); a.stats = stats; a.w = weight; a.wf32 = param_dtype == GACT_F32;
    a.rows = rows; a.cols = (int)cols; a.inv_cols = 1.0f / (float)cols; a.dx = dx;
    a.partial = params ? (float*)scratch : nullptr; a.width = (int)((cols + 7) / 8 * 8);
    const PipelineHook hook = pipeline_hook(kWaitLimit);
    a.wait_limit = hook.limit; a.withhold = hook.withhold; a.report = pipeline_report_word();
    const int eb = elem_bytes_of(dtype);
    const bool vec = rows_aligned(dy, ld_dy, cols, eb) && (!x || rows_aligned(x, ld_x, cols, eb)) && (!dx || rows_aligned(dx, cols, cols, eb));
    const bool ring = ln_ring(vec, a.codes != nullptr, dtype, rows, cols, hook.withhold != 0);
    const int64_t blocks = ln_bwd_blocks(ring, rows, cols);
    int st;
    switch (dtype) {
    case GACT_F32: st = dispatch_ln_bwd<GACT_F32>(a, vec, ring, blocks, s); break;
    case GACT_F16: st = dispatch_ln_bwd<GACT_F16>(a, vec, ring, blocks, s); break;
    default: st = dispatch_ln_bwd<GACT_BF16>(a, vec, ring, blocks, s); break;
    }
    if (st != GACT_OK || !params) return st;
    // both halves are summed; a gradient nobody asked for is not stored
    return reduce_columns((const float*)scratch, (int)blocks, 2 * (int64_t)a.width, dweight ? dweight : nullptr, dweight ? cols : 0,
                          dbias ? dbias : dweight, dbias ? cols : 0, param_dtype, 32, s);
}
