// Linear layers on the 5th-generation tensor cores:
//
//   forward        z = x W^T + b,  y = act(z) + residual;  z is kept as an 8-bit checkpoint made in the epilogue
//   act backward   dz = dy act'(z'),  db = sum over rows of dz   (z' restored from the checkpoint)
//   data gradient  dx = dz W
//   weight grad.   dW = dz^T x'
//
// One matrix-product kernel serves all three products (the operands are read in the layout they have in memory: K-major or
// MN-major tiles), persistent, one block per SM: warp 0 feeds a ring of operand tiles with tensor-map copies, one thread of
// warp 1 issues tcgen05.mma into one of two TMEM accumulators, eight warps work on the other one (epilogue), and the two warps
// that are left do side jobs.  Bounds, measured on 8192 rows, 1024 -> 4096 features, bf16 (68.7 GFLOP a product, 41.5 us at the
// measured 1655 TFLOP/s): forward 54 us, with GELU and the pre-activation's checkpoint 68 (the epilogue's instructions and
// TMEM reads; at a reduction of 4096, 32768 rows, 75 to 160 of 860 to 945), data gradient 53, weight gradient 54; the tensor pipe is busy 83 % of
// the cycles in which the SMs work, and 64 or 512 tiles over 74 pairs of SMs leave 7 to 14 % of them idle at the end.
// Widening the codes inside the weight gradient instead of restoring x beside the data gradient was built and measured: 80 us
// instead of 52 + 2.
#include "blocks8.cuh"
#include "tcgen05.cuh"

namespace gact {

__device__ int g_linear_error = 0;

constexpr int kBM = 128, kBK = 64;            // tile rows, reduction per stage (64 16-bit elements = one 128-byte swizzle row)
constexpr int kGThreads = 384;                // warps: 0 copies, 1 products, 2 TMEM, 2 and 3 side jobs, 4..11 epilogue
constexpr int kEpiWarps = 8;

enum { kEpiStore = 0, kEpiLinear = 1, kEpiPartial = 2 };

// Work that the two idle warps of a product's blocks do beside it, in its shadow and without launches of their own:
// the checkpoint of x beside the forward product (kind 1), x restored from its checkpoint beside the data gradient, for the
// weight gradient that follows (kind 2), and the bias gradient's partial sums added up beside either gradient.
struct SideJob {
    int kind;
    const void* x; int64_t ld; int stochastic; Noise8 noise;       // 1: rows of cols elements on 16-byte boundaries
    int8_t* codes; uint8_t* scales;
    void* out;                                                     // 2: rows of the codes' pitch
    int64_t rows; int cols, chunks; Divisor by;
    const float* partial; int parts; int64_t width; void* sums; int64_t n;     // column sums, or partial null
};

struct GemmArgs {
    int64_t M, N; int ktiles;                 // output rows, columns, reduction in stages
    int tiles_m, tiles_n, splits, per_split;  // stages per split
    // epilogue
    void* out; int64_t ldo; int ovec;         // bytes per store: 32, 16 or 2
    const void* bias;
    const void* res; int64_t ldr; int rvec;
    int act;
    void* z; int zvec;                        // pre-activation in the operand type (row pitch N), or
    int8_t* zcodes; uint8_t* zscales; int64_t zpitch;   // as 8-bit checkpoint
    int stochastic; Noise8 noise;
    float* partial;                           // [splits][M][pitchN] fp32
    int64_t ldp;
    SideJob side;
    uint32_t wait_limit; int withhold; int* report;      // bounded waits; diagnostics; the host's word
};

__device__ __forceinline__ void st_v8(void* p, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.u32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

// ---- activations, two values at a time -------------------------------------------------------------------------------
__device__ __forceinline__ float fast_rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float fast_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float2 rcp2(float2 x) { return make_float2(fast_rcp(x.x), fast_rcp(x.y)); }
__device__ __forceinline__ float2 exp2_2(float2 x) { return make_float2(fast_exp2(x.x), fast_exp2(x.y)); }
constexpr float kLog2e = 1.4426950408889634f;

// Phi(z) = (1 + erf(z / sqrt 2)) / 2 through Abramowitz & Stegun 7.1.26 (|error| of erf <= 1.5e-7): with
// t = 1 / (1 + 0.3275911 |z| / sqrt 2), erfc(|z| / sqrt 2) = t (a1 + t (a2 + ...)) exp(-z^2 / 2).  One exponential serves
// Phi and the density.  For negative z nothing cancels against 1, so the tail is as good as the polynomial: relative to Phi it is
// off by 3e-6 down to z = -2, 5e-4 to -4, 1.6e-3 to -5, 1e-2 to -8, 4e-2 at -13 (its bound is absolute; 1 + erf in fp32 has no
// digit left at -6).  A value of bf16, off by up to 2e-3 itself, notices from about -5 on, where |GELU| is below 1.5e-6.  The
// coefficients are halved here, so that the polynomial gives the tail of Phi directly.
__device__ __forceinline__ float2 normal_cdf2(float2 z, float2& gauss) {
    const float2 az = make_float2(fabsf(z.x), fabsf(z.y));
    gauss = exp2_2(mul2(mul2(z, splat2(-0.5f * kLog2e)), z));
    const float2 t = rcp2(fma2(az, splat2(0.3275911f * 0.70710678118654752f), splat2(1.0f)));
    float2 p = fma2(t, splat2(0.5f * 1.061405429f), splat2(0.5f * -1.453152027f));
    p = fma2(t, p, splat2(0.5f * 1.421413741f));
    p = fma2(t, p, splat2(0.5f * -0.284496736f));
    p = fma2(t, p, splat2(0.5f * 0.254829592f));
    const float2 tail = mul2(mul2(p, t), gauss), rest = fma2(tail, splat2(-1.0f), splat2(1.0f));
    return make_float2(z.x < 0.0f ? tail.x : rest.x, z.y < 0.0f ? tail.y : rest.y);
}
// 1 / (1 + exp(-u)); an exponential that overflows gives 0
__device__ __forceinline__ float2 sigmoid2(float2 u) { return rcp2(add2(exp2_2(mul2(u, splat2(-kLog2e))), splat2(1.0f))); }
constexpr float kTanhA = 1.5957691216057308f;       // 2 sqrt(2 / pi): (1 + tanh u) / 2 = sigmoid(2 u)

template <int ACT> __device__ __forceinline__ float2 act_value2(float2 z) {
    if constexpr (ACT == GACT_ACT_RELU) {
        return make_float2(z.x > 0.0f ? z.x : (z.x != z.x ? z.x : 0.0f), z.y > 0.0f ? z.y : (z.y != z.y ? z.y : 0.0f));
    } else if constexpr (ACT == GACT_ACT_GELU) {
        float2 g;
        return mul2(z, normal_cdf2(z, g));
    } else if constexpr (ACT == GACT_ACT_GELU_TANH) {
        return mul2(z, sigmoid2(mul2(mul2(z, splat2(kTanhA)), fma2(mul2(z, z), splat2(0.044715f), splat2(1.0f)))));
    } else if constexpr (ACT == GACT_ACT_SILU) {
        return mul2(z, sigmoid2(z));
    }
    return z;
}
template <int ACT> __device__ __forceinline__ float2 act_slope2(float2 z) {
    if constexpr (ACT == GACT_ACT_RELU) {
        return make_float2(z.x > 0.0f ? 1.0f : (z.x != z.x ? z.x : 0.0f), z.y > 0.0f ? 1.0f : (z.y != z.y ? z.y : 0.0f));
    } else if constexpr (ACT == GACT_ACT_GELU) {
        float2 g;
        const float2 c = normal_cdf2(z, g);
        return fma2(mul2(z, splat2(0.39894228040143268f)), g, c);
    } else if constexpr (ACT == GACT_ACT_GELU_TANH) {
        // (z^2 is capped: where it would overflow, p (1 - p) is 0 and the product has to stay 0)
        float2 q = mul2(z, z);
        q = make_float2(q.x > 1e9f ? 1e9f : q.x, q.y > 1e9f ? 1e9f : q.y);
        const float2 p = sigmoid2(mul2(mul2(z, splat2(kTanhA)), fma2(q, splat2(0.044715f), splat2(1.0f))));
        const float2 r = mul2(mul2(z, p), fma2(p, splat2(-1.0f), splat2(1.0f)));
        return fma2(r, fma2(q, splat2(3.0f * 0.044715f * kTanhA), splat2(kTanhA)), p);
    } else if constexpr (ACT == GACT_ACT_SILU) {
        const float2 p = sigmoid2(z);
        return fma2(mul2(z, p), fma2(p, splat2(-1.0f), splat2(1.0f)), p);
    }
    return splat2(1.0f);
}

// ---- epilogue of 32 rows x 32 columns: a lane holds one row --------------------------------------------------------------
// Rows on 16-byte boundaries are written and read by their own lane, 32 or 16 bytes at a time.  Other rows (and the ragged
// last columns) go through shared memory, where the tile is turned around: lane l takes column l of one row after the other,
// so that an access covers 64 contiguous bytes instead of 2 bytes of 32 rows (`stage`: 32 x 17 words of the warp).
constexpr int kStageWords = 32 * 17;

template <int DT>
__device__ __forceinline__ void store32(void* base, int64_t ld, int vec, int64_t row, int64_t M, int64_t n, int64_t N, const float2 (&v)[16], uint32_t* stage) {
    using T = typename Elem<DT>::T;
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; i++) w[i] = pack2<DT>(v[i].x, v[i].y);
    if (n + 32 <= N && vec >= 16) {
        if (row >= M) return;
        T* p = (T*)base + row * ld + n;
        if (vec == 32) {
            const uint32_t a[8] = {w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]}, b[8] = {w[8], w[9], w[10], w[11], w[12], w[13], w[14], w[15]};
            st_v8(p, a);
            st_v8(p + 16, b);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) *(uint4*)(p + 8 * i) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
    } else {
        const int lane = threadIdx.x & 31;
        const int64_t row0 = row - lane;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 16; i++) stage[lane * 17 + i] = w[i];
        __syncwarp();
        uint16_t* p = (uint16_t*)base + row0 * ld + n + lane;
        const int rows = (int)(M - row0 < 32 ? M - row0 : 32);
        if (n + lane < N)
            for (int r = 0; r < rows; r++, p += ld) *p = ((const uint16_t*)(stage + r * 17))[lane];
    }
}
template <int DT>
__device__ __forceinline__ void add32(const void* base, int64_t ld, int vec, int64_t row, int64_t M, int64_t n, int64_t N, float2 (&v)[16], uint32_t* stage) {
    using T = typename Elem<DT>::T;
    uint32_t w[16];
    if (n + 32 <= N && vec >= 16) {
        if (row >= M) return;
        const T* p = (const T*)base + row * ld + n;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint4 u = __ldg((const uint4*)(p + 8 * i));
            w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
        }
    } else {
        const int lane = threadIdx.x & 31;
        const int64_t row0 = row - lane;
        const uint16_t* p = (const uint16_t*)base + row0 * ld + n + lane;
        const int rows = (int)(M - row0 < 32 ? M - row0 : 32);
        __syncwarp();
#pragma unroll 8
        for (int r = 0; r < 32; r++, p += ld) ((uint16_t*)(stage + r * 17))[lane] = (n + lane < N && r < rows) ? __ldg(p) : (uint16_t)0;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 16; i++) w[i] = stage[lane * 17 + i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t raw[4] = {w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
        float2 f[4];
        raw_to_pairs<DT>(raw, f);
#pragma unroll
        for (int j = 0; j < 4; j++) v[4 * i + j] = add2(v[4 * i + j], f[j]);
    }
}
template <int ACT> __device__ __forceinline__ void activate32(float2 (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = act_value2<ACT>(v[i]);
}

// z = v + bias -> checkpoint of z, y = act(z) + residual -> out.  Called by whole warps (rows past M store nothing);
// `bias`: the 32 biases as fp32 in shared memory (zeros past N or without one).
template <int DT>
__device__ __forceinline__ void linear_epilogue32(const GemmArgs& a, int64_t row, int64_t n, const float* bias, float2 (&v)[16], uint32_t* stage) {
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        const float4 b = *(const float4*)(bias + 2 * i);
        v[i] = add2(v[i], make_float2(b.x, b.y));
        v[i + 1] = add2(v[i + 1], make_float2(b.z, b.w));
    }
    if (a.zcodes) {
        // columns past N are zero: their weights and biases are
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) m = absmax3(m, v[i]);
        const uint32_t byte = scale_byte8(__float_as_uint(m) & 0x7fffffffu);
        const float up = scale_up8(byte);
        const uint64_t at = (uint64_t)row * a.zpitch + n;
        uint32_t w[8];
        if (!a.stochastic && a.act != GACT_ACT_RELU) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float2 p = fma2(v[2 * i], splat2(up), splat2(12582912.0f)), q = fma2(v[2 * i + 1], splat2(up), splat2(12582912.0f));
                w[i] = pack4(__float_as_uint(p.x), __float_as_uint(p.y), __float_as_uint(q.x), __float_as_uint(q.y));
            }
        } else {
            const uint2 high = a.noise.high();
#pragma unroll
            for (int i = 0; i < 8; i++) {
                uint32_t c[4];
                uint4 r = make_uint4(0u, 0u, 0u, 0u);
                if (a.stochastic) r = noise8(a.noise, high, at / 8 + i / 2);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float z = (j & 1) ? v[2 * i + j / 2].y : v[2 * i + j / 2].x;
                    c[j] = a.stochastic ? code8_noise(z, up, noise8_at(r, (i & 1) * 4 + j)) : code8(z, up);
                    // ReLU's slope is decided by the sign of z: a positive z keeps a positive code
                    if (a.act == GACT_ACT_RELU && z > 0.0f && (c[j] & 0xffu) == 0u) c[j] = 1u;
                }
                w[i] = pack4(c[0], c[1], c[2], c[3]);
            }
        }
        if (byte >= top_byte8<GACT_F32>()) {
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = byte == 255u ? 0u : clamp_codes63(w[i]);
        }
        if (row < a.M) {
            st_v8(a.zcodes + at, w);
            a.zscales[at >> 5] = (uint8_t)byte;
        }
    }
    if (a.z) store32<DT>(a.z, a.N, a.zvec, row, a.M, n, a.N, v, stage);
    switch (a.act) {
    case GACT_ACT_RELU: activate32<GACT_ACT_RELU>(v); break;
    case GACT_ACT_GELU: activate32<GACT_ACT_GELU>(v); break;
    case GACT_ACT_GELU_TANH: activate32<GACT_ACT_GELU_TANH>(v); break;
    case GACT_ACT_SILU: activate32<GACT_ACT_SILU>(v); break;
    default: break;
    }
    if (a.res) add32<DT>(a.res, a.ldr, a.rvec, row, a.M, n, a.N, v, stage);
    store32<DT>(a.out, a.ldo, a.ovec, row, a.M, n, a.N, v, stage);
}
template <int DT> __device__ __forceinline__ float bias_at(const GemmArgs& a, int64_t n) {
    return a.bias && n < a.N ? Elem<DT>::to_float(((const typename Elem<DT>::T*)a.bias)[n]) : 0.0f;
}

// ---- side jobs ---------------------------------------------------------------------------------------------------------
// Worker `w` of `n` warps.  Eight chunks per lane are loaded before the first is worked on: with two warps per SM the loads in
// flight decide (measured beside a product: about 1.2 TB/s over the GPU).
template <int DT>
__device__ __forceinline__ void side_job(const SideJob& j, int w, int n) {
    using T = typename Elem<DT>::T;
    const int lane = threadIdx.x & 31;
    constexpr int U = 8;
    if (j.partial) {
        // 32 columns per warp; eight sums (part p goes to sum p mod 8), then those in order, as reduce_columns adds them
        for (int64_t c = (int64_t)w * 32 + lane; c - lane < j.n; c += (int64_t)n * 32) {
            if (c < j.n) {
                float v[kSumChains], sum;
#pragma unroll
                for (int i = 0; i < kSumChains; i++) v[i] = 0.0f;
                const float* q = j.partial + c;
                for (int p = 0; p < j.parts; p += kSumChains, q += kSumChains * j.width) {
                    float u[kSumChains];
#pragma unroll
                    for (int i = 0; i < kSumChains; i++) u[i] = p + i < j.parts ? q[i * j.width] : 0.0f;
#pragma unroll
                    for (int i = 0; i < kSumChains; i++) v[i] += u[i];
                }
                sum = v[0];
#pragma unroll
                for (int i = 1; i < kSumChains; i++) sum += v[i];
                ((T*)j.sums)[c] = Elem<DT>::from_float(sum);
            }
        }
    }
    const int64_t total = j.rows * j.chunks;
    if (j.kind == 1) {
        const uint2 high = j.noise.high();
        for (int64_t i0 = (int64_t)w * 32 * U; i0 < total; i0 += (int64_t)n * 32 * U) {
            uint32_t raw[U][4];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int64_t i = i0 + u * 32 + lane, row = j.by.div(i);
                const int col = (int)(i - row * j.chunks) * 8;
                const T* p = (const T*)j.x + row * j.ld + col;
                raw[u][0] = raw[u][1] = raw[u][2] = raw[u][3] = 0u;
                if (i < total && col + 8 <= j.cols) {
                    const uint4 a = ld_stream_u4(p);
                    raw[u][0] = a.x; raw[u][1] = a.y; raw[u][2] = a.z; raw[u][3] = a.w;
                } else if (i < total) {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (col + e < j.cols) raw[u][e >> 1] |= (uint32_t)((const uint16_t*)p)[e] << (16 * (e & 1));
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int64_t i = i0 + u * 32 + lane;
                float2 v[4];
                raw_to_pairs<DT>(raw[u], v);
                uint32_t byte;
                const uint32_t m = absmax8<DT>(raw[u]);
                const uint2 q = j.stochastic ? codes8<true>(v, m, j.noise, high, (uint64_t)i, byte, top_byte8<DT>()) : codes8<false>(v, m, j.noise, high, (uint64_t)i, byte, top_byte8<DT>());
                if (i < total) {
                    st_stream_u2(j.codes + i * 8, q);
                    if ((lane & 3) == 0) j.scales[i >> 2] = (uint8_t)byte;
                }
            }
        }
    } else if (j.kind == 2) {
        for (int64_t i0 = (int64_t)w * 32 * U; i0 < total; i0 += (int64_t)n * 32 * U) {
            uint2 q[U];
            uint32_t b[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int64_t i = i0 + u * 32 + lane;
                q[u] = make_uint2(0u, 0u);
                b[u] = 1;
                if (i < total) {
                    q[u] = ld_stream_u2(j.codes + i * 8);
                    b[u] = ld_ahead_byte(j.scales + (i >> 2));
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int64_t i = i0 + u * 32 + lane;
                if (i < total) {
                    float2 v[4];
                    restore_pairs(q[u], scale_down8(b[u]), v);
                    *(uint4*)((T*)j.out + i * 8) = make_uint4(pack2<DT>(v[0].x, v[0].y), pack2<DT>(v[1].x, v[1].y), pack2<DT>(v[2].x, v[2].y), pack2<DT>(v[3].x, v[3].y));
                }
            }
        }
    }
}

// ---- the matrix product ----------------------------------------------------------------------------------------------
// CG blocks (a cluster) work on one tile of CG * 128 rows and BN columns: each holds its own 128 rows of A, BN / CG columns
// of B and the accumulators of its rows.  A pair reads every B tile once for 256 rows, which halves the shared-memory
// traffic that bounds a single block's products.
template <int CG, int BN> struct Ring {
    static constexpr int kCols = BN / CG;                     // columns of B per block
    static constexpr int kA = kBM * kBK * 2, kB = kCols * kBK * 2, kStage = kA + kB;
    static constexpr int kStages = 196608 / kStage < 8 ? 196608 / kStage : 8;
    static constexpr int kBytes = kStages * kStage + 1024 /* alignment */ + 256 /* barriers */;
};

struct Unit { int64_t m0, n0; int k0, k1, split; };

// Units (tile x split of the reduction) in an order that keeps concurrently running tiles close together: bands of tile
// rows, inside a band row by row of columns.
template <int CG, int BN> __device__ __forceinline__ Unit unit_at(const GemmArgs& a, int64_t u) {
    constexpr int kBand = 16 / CG;
    const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n;
    Unit x;
    x.split = (int)(u / tiles);
    const int64_t t = u - x.split * tiles;
    const int64_t band = t / ((int64_t)kBand * a.tiles_n);
    const int rows = (int)min((int64_t)kBand, (int64_t)a.tiles_m - band * kBand);
    const int64_t in = t - band * kBand * a.tiles_n;
    x.m0 = (band * kBand + in % rows) * (kBM * CG);
    x.n0 = (in / rows) * BN;
    x.k0 = x.split * a.per_split;
    x.k1 = min(a.ktiles, x.k0 + a.per_split);
    return x;
}

template <int DT, bool A_MN, bool B_MN, int CG, int BN, int EPI>
__global__ void __cluster_dims__(CG, 1, 1) __launch_bounds__(kGThreads, 1)
gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ GemmArgs a) {
    using R = Ring<CG, BN>;
    constexpr int S = R::kStages;
    constexpr uint32_t kTmem = 2 * BN;
    extern __shared__ uint8_t raw[];
    uint8_t* base = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    const uint32_t ring = smem_addr(base);
    uint64_t* bars = (uint64_t*)(base + S * R::kStage);
    const uint32_t full = smem_addr(bars), empty = full + 8 * S, acc_full = empty + 8 * S, acc_empty = acc_full + 16, drain = acc_empty + 16;
    __shared__ uint32_t tmem_slot;
    __shared__ __align__(16) float bias[2][EPI == kEpiLinear ? BN : 4];
    __shared__ uint32_t stage[EPI == kEpiPartial ? 1 : kEpiWarps][EPI == kEpiPartial ? 1 : kStageWords];
    __shared__ volatile int dead;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 1 ? 0u : cluster_rank();

    if (threadIdx.x == 0) {
        dead = 0;
        // full, acc_empty: those of block 0 are used; empty, acc_full: each block has its own
        for (int i = 0; i < S; i++) { mbar_init(full + 8 * i, 1); mbar_init(empty + 8 * i, 1); }
        for (int i = 0; i < 2; i++) { mbar_init(acc_full + 8 * i, 1); mbar_init(acc_empty + 8 * i, CG * kEpiWarps); }
        mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_map(&map_a);
        prefetch_map(&map_b);
    }
    __syncwarp();
    if (warp == 2) tmem_alloc<CG>(smem_addr(&tmem_slot), kTmem);
    tc_fence_before();
    if constexpr (CG == 1) __syncthreads();
    else cluster_sync();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const int64_t units = (int64_t)a.tiles_m * a.tiles_n * a.splits;
    const int64_t first = blockIdx.x / CG, stride = gridDim.x / CG;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t it = 0;
            const uint32_t full0 = CG == 1 ? full : peer_addr(full, 0);
            for (int64_t u = first; u < units && !dead; u += stride) {
                const Unit x = unit_at<CG, BN>(a, u);
                const int m0 = (int)(x.m0 + rank * kBM), n0 = (int)(x.n0 + rank * R::kCols);
                for (int k = x.k0; k < x.k1; k++, it++) {
                    const uint32_t s = it % S, ph = (it / S) & 1;
                    if (!mbar_wait(empty + 8 * s, ph ^ 1, a.wait_limit, &dead)) break;
                    const uint32_t bar = full0 + 8 * s, da = ring + s * R::kStage, db = da + R::kA;
                    // block 0 announces the bytes of both (the other's may land first: the phase still waits for this arrival)
                    if (rank == 0) mbar_expect_tx(full + 8 * s, CG * R::kStage);
                    if (A_MN) {
#pragma unroll
                        for (int i = 0; i < kBM / 64; i++) tma_load_2d<CG>(da + i * 8192, &map_a, m0 + 64 * i, k * kBK, bar);
                    } else {
                        tma_load_2d<CG>(da, &map_a, k * kBK, m0, bar);
                    }
                    if (a.withhold && it == 0 && blockIdx.x == 0) {
                        // (diagnostics: this stage never fills)
                    } else if (B_MN) {
#pragma unroll
                        for (int i = 0; i < R::kCols / 64; i++) tma_load_2d<CG>(db + i * 8192, &map_b, n0 + 64 * i, k * kBK, bar);
                    } else {
                        tma_load_2d<CG>(db, &map_b, k * kBK, n0, bar);
                    }
                }
            }
            // the last stages have been read by the products, or the block gives up: then the copies that were issued (at most
            // one per stage; block 0's barriers count both blocks') land before the blocks end
            const uint32_t tail = it > (uint32_t)S ? it - S : 0;
            for (uint32_t j = tail; j < it; j++) mbar_wait(empty + 8 * (j % S), (j / S) & 1, a.wait_limit, &dead);
            if (dead) {
                report_wait(&g_linear_error, a.report);
                if (rank == 0)
                    for (uint32_t j = tail; j < it; j++) mbar_drain(full + 8 * (j % S), (j / S) & 1, a.wait_limit);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = mma_idesc(CG * kBM, BN, DT == GACT_BF16, A_MN, B_MN);
            uint32_t it = 0, n = 0;
            for (int64_t u = first; u < units && !dead; u += stride, n++) {
                const Unit x = unit_at<CG, BN>(a, u);
                const uint32_t acc = n & 1;
                if (!mbar_wait(acc_empty + 8 * acc, ((n >> 1) & 1) ^ 1, a.wait_limit, &dead)) break;
                tc_fence_after();
                const uint32_t d = tmem + acc * BN;
                for (int k = x.k0; k < x.k1; k++, it++) {
                    const uint32_t s = it % S, ph = (it / S) & 1;
                    if (!mbar_wait(full + 8 * s, ph, a.wait_limit, &dead)) break;
                    tc_fence_after();
                    const uint32_t sa = ring + s * R::kStage, sb = sa + R::kA;
#pragma unroll
                    for (int j = 0; j < kBK / 16; j++) {
                        const uint64_t da = smem_desc(sa + j * (A_MN ? 2048 : 32), A_MN ? 8192 : 16);
                        const uint64_t db = smem_desc(sb + j * (B_MN ? 2048 : 32), B_MN ? 8192 : 16);
                        mma_f16<CG>(d, da, db, idesc, (k > x.k0 || j > 0) ? 1u : 0u);
                    }
                    mma_commit<CG>(empty + 8 * s);
                }
                mma_commit<CG>(acc_full + 8 * acc);
            }
            // every product has finished before TMEM is given back
            mma_commit<CG>(drain);
            mbar_drain(drain, 0, a.wait_limit);
        }
        __syncwarp();
    } else if (warp < 4) {
        side_job<DT>(a.side, (int)blockIdx.x * 2 + warp - 2, (int)gridDim.x * 2);
    } else {
        const int q = warp & 3, half = (warp - 4) >> 2;
        const uint32_t acc_empty0 = CG == 1 ? acc_empty : peer_addr(acc_empty, 0);
        uint32_t n = 0;
        for (int64_t u = first; u < units; u += stride, n++) {
            const Unit x = unit_at<CG, BN>(a, u);
            const uint32_t acc = n & 1;
            constexpr int kSpan = BN / 2;             // columns per warp
            if constexpr (EPI == kEpiLinear) {
                // this tile's biases as fp32; the buffers alternate, so one barrier of the epilogue warps per tile is enough
                const int e = threadIdx.x - 128;
                if (e < BN) bias[acc][e] = bias_at<DT>(a, x.n0 + e);
                asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory");
            }
            // (a warp that gave up goes on through the tiles without storing: every warp meets every barrier)
            const bool ok = mbar_wait(acc_full + 8 * acc, (n >> 1) & 1, a.wait_limit, &dead);
            if (!__all_sync(kFull, ok)) continue;
            tc_fence_after();
            const int64_t row = x.m0 + rank * kBM + q * 32 + lane;
#pragma unroll 1
            for (int c = 0; c < kSpan; c += 32) {
                const int64_t col = x.n0 + half * kSpan + c;
                if (col >= a.N) break;
                uint32_t r[32];
                tmem_load32(tmem + ((uint32_t)(q * 32) << 16) + acc * BN + half * kSpan + c, r);
                if constexpr (EPI == kEpiPartial) {
                    if (row < a.M) {
                        float* p = a.partial + ((int64_t)x.split * a.M + row) * a.ldp + col;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint32_t w[8] = {r[8 * i], r[8 * i + 1], r[8 * i + 2], r[8 * i + 3], r[8 * i + 4], r[8 * i + 5], r[8 * i + 6], r[8 * i + 7]};
                            st_v8(p + 8 * i, w);
                        }
                    }
                    __syncwarp();
                } else {
                    float2 v[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) v[i] = make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
                    if constexpr (EPI == kEpiLinear) linear_epilogue32<DT>(a, row, col, bias[acc] + half * kSpan + c, v, stage[warp - 4]);
                    else store32<DT>(a.out, a.ldo, a.ovec, row, a.M, col, a.N, v, stage[warp - 4]);
                    __syncwarp();
                }
            }
            tc_fence_before();
            if (lane == 0) {
                if constexpr (CG == 1) mbar_arrive(acc_empty + 8 * acc);
                else mbar_arrive_cluster(acc_empty0 + 8 * acc);
            }
        }
        // the last commit arrives in both blocks: block 1 too must have seen it before its shared memory may end (every other
        // arrival from block 0 has been waited for above).  One thread that is through its tiles waits, so the bound counts from there.
        if constexpr (CG == 2)
            if (rank == 1 && warp == 4 && lane == 0) mbar_drain(drain, 0, a.wait_limit);
    }
    __syncwarp();
    tc_fence_before();
    if constexpr (CG == 1) __syncthreads();
    else cluster_sync();
    tc_fence_after();
    if (warp == 2) tmem_free<CG>(tmem, kTmem);
}

// Adds the partial sums of the splits in order and runs the epilogue: one thread per 32 columns of a row, 128 rows and the
// same 32 columns per block.
template <int DT>
__global__ void __launch_bounds__(128) gemm_join_linear_kernel(const __grid_constant__ GemmArgs a) {
    __shared__ __align__(16) float bias[32];
    __shared__ uint32_t stage[4][kStageWords];
    const int64_t n = (int64_t)blockIdx.y * 32;
    if (threadIdx.x < 32) bias[threadIdx.x] = bias_at<DT>(a, n + threadIdx.x);
    __syncthreads();
    const int64_t row = (int64_t)blockIdx.x * 128 + threadIdx.x;
    float2 v[16];
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = splat2(0.0f);
    for (int s = 0; s < a.splits && row < a.M; s++) {
        const float4* p = (const float4*)(a.partial + ((int64_t)s * a.M + row) * a.ldp + n);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float4 f = p[j];
            v[2 * j] = add2(v[2 * j], make_float2(f.x, f.y));
            v[2 * j + 1] = add2(v[2 * j + 1], make_float2(f.z, f.w));
        }
    }
    linear_epilogue32<DT>(a, row, n, bias, v, stage[threadIdx.x >> 5]);
}

// The same without an epilogue: one thread per 8 columns, neighbours side by side.
template <int DT>
__global__ void __launch_bounds__(256) gemm_join_kernel(const __grid_constant__ GemmArgs a) {
    using T = typename Elem<DT>::T;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.M * (a.ldp / 8)) return;
    const int64_t row = i / (a.ldp / 8), n = (i - row * (a.ldp / 8)) * 8;
    if (n >= a.N) return;
    float2 v[4] = {splat2(0.0f), splat2(0.0f), splat2(0.0f), splat2(0.0f)};
    const float* p = a.partial + row * a.ldp + n;
#pragma unroll 4
    for (int s = 0; s < a.splits; s++, p += a.M * a.ldp) {
        const float4 x = *(const float4*)p, y = *(const float4*)(p + 4);
        v[0] = add2(v[0], make_float2(x.x, x.y));
        v[1] = add2(v[1], make_float2(x.z, x.w));
        v[2] = add2(v[2], make_float2(y.x, y.y));
        v[3] = add2(v[3], make_float2(y.z, y.w));
    }
    T* out = (T*)a.out + row * a.ldo + n;
    if (a.ovec >= 16 && n + 8 <= a.N) {
        *(uint4*)out = make_uint4(pack2<DT>(v[0].x, v[0].y), pack2<DT>(v[1].x, v[1].y), pack2<DT>(v[2].x, v[2].y), pack2<DT>(v[3].x, v[3].y));
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (n + j < a.N) out[j] = Elem<DT>::from_float(j & 1 ? v[j / 2].y : v[j / 2].x);
    }
}

// ---- host side --------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled encode_tiled() {
    static std::atomic<void*> cached{nullptr};
    void* f = cached.load(std::memory_order_acquire);
    if (!f) {
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return nullptr;
        cached.store(f, std::memory_order_release);
    }
    return (EncodeTiled)f;
}

// rows x cols elements, row pitch ld; tile of 64 elements x `box` rows, 128-byte swizzle, zeros outside
static bool make_map(CUtensorMap* m, int dtype, const void* p, int64_t rows, int64_t cols, int64_t ld, int box) {
    EncodeTiled f = encode_tiled();
    if (!f) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t boxes[2] = {64, (cuuint32_t)box};
    const cuuint32_t ones[2] = {1, 1};
    return f(m, dtype == GACT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, (void*)p, dims, strides, boxes, ones,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Plan { int cg, bn, splits, per_split; int64_t tiles_m, tiles_n; double ns; };

// Tile shape (two blocks on 256 x 256, one on 128 x 128 or 128 x 64) and splits of the reduction: the combination with the
// least estimated time.  Measured on products of 16 to 8192 rows (nanoseconds): a launch with one stage takes `fixed`, every
// further stage of a block `stage` (a stage moves 24 to 32 KB into an SM, which at these sizes is what takes the time), so the
// busiest block's stages count; joining splits costs a second launch (with the linear epilogue a longer one) and the partial
// sums' way through L2.
static Plan plan_gemm(int64_t M, int64_t N, int64_t K, bool linear) {
    struct Shape { int cg, bn; double fixed, stage; };
    static const Shape shapes[3] = {{2, 256, 5600.0, 390.0}, {1, 128, 4400.0, 370.0}, {1, 64, 4100.0, 335.0}};
    const int sms = sm_count();
    const int64_t kt = (K + kBK - 1) / kBK;
    Plan best = {};
    double best_t = 1e300;
    for (const Shape& h : shapes) {
        Plan p;
        p.cg = h.cg; p.bn = h.bn;
        p.tiles_m = (M + kBM * h.cg - 1) / (kBM * h.cg);
        p.tiles_n = (N + h.bn - 1) / h.bn;
        const int64_t tiles = p.tiles_m * p.tiles_n, slots = sms / h.cg;
        for (int64_t splits = 1; splits <= 16 && (splits == 1 || tiles * splits <= 4 * slots); splits++) {
            p.per_split = (int)((kt + splits - 1) / splits);
            p.splits = (int)((kt + p.per_split - 1) / p.per_split);
            if (p.splits != splits || (splits > 1 && p.per_split < 2)) continue;
            const int64_t rounds = (tiles * splits + slots - 1) / slots;
            double t = h.fixed + (double)(rounds * p.per_split - 1) * h.stage;
            if (splits > 1) t += (linear ? 6000.0 : 2800.0) + (double)(splits * 2 + 1) * (double)M * (double)N * 4.0 / 8000.0;
            if (t < best_t) { best_t = t; best = p; best.ns = t; }
        }
    }
    return best;
}

static int64_t gemm_scratch(int64_t M, int64_t N, int64_t K, bool linear) {
    const Plan p = plan_gemm(M, N, K, linear);
    return p.splits > 1 ? (int64_t)p.splits * M * pitch8(N) * 4 : 0;
}

static int vec_bytes(const void* p, int64_t ld) {
    const uintptr_t v = (uintptr_t)p | (uintptr_t)(ld * 2);
    return (v & 31) == 0 ? 32 : (v & 15) == 0 ? 16 : 2;
}

template <int DT, bool A_MN, bool B_MN, int CG, int BN, int EPI>
static int launch_gemm_kernel(const CUtensorMap& ma, const CUtensorMap& mb, const GemmArgs& a, cudaStream_t s) {
    auto* k = gemm_kernel<DT, A_MN, B_MN, CG, BN, EPI>;
    static std::atomic<bool> allowed[kMaxDevices];
    if (!allow_smem(k, Ring<CG, BN>::kBytes, allowed)) return GACT_ERR_LAUNCH;
    const int64_t units = (int64_t)a.tiles_m * a.tiles_n * a.splits, slots = sm_count() / CG;
    const int64_t grid = (units < slots ? units : slots) * CG;
    k<<<(unsigned)grid, kGThreads, Ring<CG, BN>::kBytes, s>>>(ma, mb, a);
    return cudaGetLastError() == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
}
template <int DT, bool A_MN, bool B_MN, int EPI>
static int launch_gemm_shape(const Plan& p, const CUtensorMap& ma, const CUtensorMap& mb, const GemmArgs& a, cudaStream_t s) {
    if (p.cg == 2) return launch_gemm_kernel<DT, A_MN, B_MN, 2, 256, EPI>(ma, mb, a, s);
    if (p.bn == 128) return launch_gemm_kernel<DT, A_MN, B_MN, 1, 128, EPI>(ma, mb, a, s);
    return launch_gemm_kernel<DT, A_MN, B_MN, 1, 64, EPI>(ma, mb, a, s);
}

// C (M x N) = A B with the reduction over K.  A: K-major (M rows of K) or MN-major (K rows of M); B likewise with N.
template <int DT, bool A_MN, bool B_MN, bool LINEAR>
static int run_gemm(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t K, GemmArgs a, void* scratch, cudaStream_t s) {
    const Plan p = plan_gemm(a.M, a.N, K, LINEAR);
    CUtensorMap ma, mb;
    const bool ok = make_map(&ma, DT, A, A_MN ? K : a.M, A_MN ? a.M : K, lda, A_MN ? 64 : kBM) &&
                    make_map(&mb, DT, B, B_MN ? K : a.N, B_MN ? a.N : K, ldb, B_MN ? 64 : p.bn / p.cg);
    if (!ok) return GACT_ERR_LAUNCH;
    const PipelineHook hook = pipeline_hook(kWaitLimit);
    a.wait_limit = hook.limit; a.withhold = hook.withhold; a.report = pipeline_report_word();
    a.ktiles = (int)((K + kBK - 1) / kBK);
    a.tiles_m = (int)p.tiles_m; a.tiles_n = (int)p.tiles_n; a.splits = p.splits; a.per_split = p.per_split;
    constexpr int kEpi = LINEAR ? kEpiLinear : kEpiStore;
    if (p.splits == 1) return launch_gemm_shape<DT, A_MN, B_MN, kEpi>(p, ma, mb, a, s);
    a.partial = (float*)scratch;
    a.ldp = pitch8(a.N);
    const int st = launch_gemm_shape<DT, A_MN, B_MN, kEpiPartial>(p, ma, mb, a, s);
    if (st != GACT_OK) return st;
    if constexpr (LINEAR) {
        gemm_join_linear_kernel<DT><<<dim3((unsigned)((a.M + 127) / 128), (unsigned)(a.ldp / 32)), 128, 0, s>>>(a);
    } else {
        const int64_t threads = a.M * (a.ldp / 8);
        gemm_join_kernel<DT><<<(unsigned)((threads + 255) / 256), 256, 0, s>>>(a);
    }
    return cudaGetLastError() == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
}

// ---- dz = dy act'(z'), db = sum dz --------------------------------------------------------------------------------------
struct ActBwdArgs {
    const void* dy; int64_t ldy;
    const void* z; int64_t ldz; const int8_t* codes; const uint8_t* scales; int chunks;
    int act; int64_t rows; int cols;
    void* dz; int64_t ldo;
    float* partial; int width;
};
constexpr int kAWarps = 8;

// A warp owns 256 columns (8 per lane) and walks rows, kARows of them side by side.  A block takes eight such sets at a time.
// 64 registers and four blocks per SM: loading the next rows ahead instead took 84 registers and was a quarter slower.
// dz is rounded to the operands' 16 bits, for the tensor cores read it: against 64 bits the products' error is then 0.0023 instead of
// 0.0017 in bf16 (0.0003 instead of 0.0002 in fp16).  The bias gradient sums the products before they are rounded.
constexpr int kARows = 2;
//
// TABLE: a pre-activation from a checkpoint is an 8-bit code times a power of two, so there are 256 slopes per exponent.  Those
// of the exponents -14 .. 4 are computed once per block; a slope is then one shared-memory read instead of about 20
// instructions (the kernel was bound by issuing them: GELU on 8192 x 4096 took 59 us, with the table 32 to 34; floor 26).  Larger exponents
// equal the last row (a code's step is past the bend); below, |z| < 0.004 and the slope is its tangent at 0 (the next term,
// z^3 / 4, is below 2^-25); a NaN block's tangent is NaN.
constexpr int kLowExp = -14, kHighExp = 4, kTableRows = kHighExp - kLowExp + 1;

template <int DT, bool VEC, bool COMP, int ACT, bool TABLE>
__global__ void __launch_bounds__(kAWarps * 32, 4) act_backward_kernel(const __grid_constant__ ActBwdArgs a) {
    using T = typename Elem<DT>::T;
    using Row = Row8<DT, VEC, 32>;
    constexpr bool kAct = ACT != GACT_ACT_NONE;
    constexpr int U = kARows;
    constexpr float kSlope0 = ACT == GACT_ACT_SILU ? 0.5f : 0.79788456080286536f;       // second derivative at 0
    static_assert(!TABLE || (COMP && kAct), "the table is indexed by codes");
    __shared__ float fold[kAWarps][8][33];
    __shared__ __align__(16) uint8_t staging[VEC ? 16 : kAWarps * Stage8<DT, VEC>::kBytes];
    __shared__ __align__(1024) float table[TABLE ? kTableRows : 1][TABLE ? 256 : 1];
    if constexpr (TABLE) {
        for (int i = threadIdx.x; i < kTableRows * 128; i += kAWarps * 32) {
            // entries 2 i and 2 i + 1: row by exponent, column by the code's byte
            const int e = i / 128 + kLowExp, c = (i % 128) * 2;
            const float step = __uint_as_float((uint32_t)(127 + e) << 23);
            const float2 v = act_slope2<ACT>(make_float2((float)(int8_t)c * step, (float)(int8_t)(c + 1) * step));
            *(float2*)(&table[0][0] + 2 * i) = v;
        }
        __syncthreads();
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    void* stage = staging + warp * Stage8<DT, VEC>::kBytes;
    const int col = (blockIdx.x * 32 + lane) * 8;
    float2 db[4];
#pragma unroll
    for (int i = 0; i < 4; i++) db[i] = splat2(0.0f);
    const int64_t step = (int64_t)gridDim.y * kAWarps;
    Row py[U], pz[kAct && !COMP ? U : 1];
    uint2 pq[U];
    uint32_t pe[U];
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t row = r + u * step;
            py[u].load((const T*)a.dy, a.ldy, row, a.rows, col, a.cols);
            if constexpr (kAct && COMP) {
                pq[u] = make_uint2(0u, 0u);
                pe[u] = 1;
                if (row < a.rows && col < a.cols) {
                    const int64_t chunk = row * a.chunks + (col >> 3);
                    pq[u] = ld_stream_u2(a.codes + chunk * 8);
                    pe[u] = ld_ahead_byte(a.scales + (chunk >> 2));
                }
            } else if constexpr (kAct) {
                pz[u].load((const T*)a.z, a.ldz, row, a.rows, col, a.cols);
            }
        }
    };
    int64_t r = (int64_t)blockIdx.y * kAWarps + warp;
    for (; r < a.rows; r += U * step) {
        fetch(r);
        uint32_t rawy[U][RawRegs<DT>::N], rawz[U][RawRegs<DT>::N];
        uint2 q[U];
        float down[U];
        int row_of[U];                                   // the table's row, or -1
#pragma unroll
        for (int u = 0; u < U; u++) {
            py[u].get(stage, rawy[u]);
            if constexpr (kAct && COMP) {
                q[u] = pq[u];
                down[u] = scale_down8(pe[u]);
                const int e = (int)pe[u] - 127 - kLowExp;
                row_of[u] = pe[u] == 255u ? -1 : e < kTableRows ? e : kTableRows - 1;       // (e < 0: the tangent)
            } else if constexpr (kAct) {
                pz[u].get(stage, rawz[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            float2 g[4], z[4];
            raw_to_pairs<DT>(rawy[u], g);
            if constexpr (kAct) {
                if (TABLE && row_of[u] >= 0) {
                    const uint32_t t = smem_addr(table) + (uint32_t)row_of[u] * 1024u;       // (rows start on 1024 bytes)
                    auto slope = [&](uint32_t off) {
                        float v;
                        asm("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"((off & 0x3fcu) | t));
                        return v;
                    };
                    g[0] = mul2(g[0], make_float2(slope(q[u].x << 2), slope(q[u].x >> 6)));
                    g[1] = mul2(g[1], make_float2(slope(q[u].x >> 14), slope(q[u].x >> 22)));
                    g[2] = mul2(g[2], make_float2(slope(q[u].y << 2), slope(q[u].y >> 6)));
                    g[3] = mul2(g[3], make_float2(slope(q[u].y >> 14), slope(q[u].y >> 22)));
                } else {
                    if constexpr (COMP) restore_pairs(q[u], down[u], z);
                    else raw_to_pairs<DT>(rawz[u], z);
#pragma unroll
                    for (int i = 0; i < 4; i++) g[i] = mul2(g[i], TABLE ? fma2(z[i], splat2(kSlope0), splat2(0.5f)) : act_slope2<ACT>(z[i]));
                }
                Row::store((T*)a.dz, a.ldo, r + u * step, a.rows, col, a.cols, stage, g);
            } else if (a.dz) {
                Row::store((T*)a.dz, a.ldo, r + u * step, a.rows, col, a.cols, stage, g);
            }
            // (the sum takes the products before they are rounded; rows past the end have dy = 0 and a finite slope)
#pragma unroll
            for (int i = 0; i < 4; i++) db[i] = add2(db[i], g[i]);
        }
    }
    if (!a.partial) return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        fold[warp][2 * i][lane] = db[i].x;
        fold[warp][2 * i + 1][lane] = db[i].y;
    }
    __syncthreads();
    // thread (l, j): column blockIdx.x * 256 + l * 8 + j
    const int j = threadIdx.x & 7, l = threadIdx.x >> 3;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kAWarps; w++) sum += fold[w][j][l];
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c < a.width) a.partial[(int64_t)blockIdx.y * a.width + c] = sum;
}

// Filling the table takes about a microsecond: worth it from 5 rows per warp on (with the grid below).  Measured, table / computed in us,
// 4096 columns, GELU (SiLU): 1184 rows 8.0 / 7.6 (7.4 / 6.7), 1400 9.0 / 9.4 (8.7 / 8.5), 2048 11.4 / 12.4 (11.1 / 11.7), 8192
// 32 / 39 (31 / 37).
static bool act_bwd_table(int64_t rows, int64_t cols) { return rows * ((cols + 255) / 256) >= (int64_t)sm_count() * 4 * kAWarps * 5; }
// Parts of the rows (blocks per strip of 256 columns): four blocks per SM.  The count must not depend on anything but the sizes.
static int64_t act_bwd_parts(int64_t rows, int64_t cols) {
    const int64_t strips = (cols + 255) / 256;
    int64_t parts = ((int64_t)sm_count() * 4 + strips - 1) / strips;
    const int64_t most = (rows + kAWarps - 1) / kAWarps;
    if (parts > most) parts = most;
    return parts < 1 ? 1 : parts > 65535 ? 65535 : parts;
}

template <int DT, int ACT> static void launch_act_bwd(const ActBwdArgs& a, bool vec, dim3 grid, cudaStream_t s) {
    const int block = kAWarps * 32;
    if constexpr (ACT == GACT_ACT_NONE) {
        if (vec) act_backward_kernel<DT, true, false, ACT, false><<<grid, block, 0, s>>>(a);
        else act_backward_kernel<DT, false, false, ACT, false><<<grid, block, 0, s>>>(a);
    } else if (a.codes) {
        // (ReLU's slope is a comparison: no table)
        constexpr bool kHasTable = ACT != GACT_ACT_RELU;
        if (vec && kHasTable && act_bwd_table(a.rows, a.cols)) act_backward_kernel<DT, true, true, ACT, kHasTable><<<grid, block, 0, s>>>(a);
        else if (vec) act_backward_kernel<DT, true, true, ACT, false><<<grid, block, 0, s>>>(a);
        else act_backward_kernel<DT, false, true, ACT, false><<<grid, block, 0, s>>>(a);
    } else {
        if (vec) act_backward_kernel<DT, true, false, ACT, false><<<grid, block, 0, s>>>(a);
        else act_backward_kernel<DT, false, false, ACT, false><<<grid, block, 0, s>>>(a);
    }
}
template <int DT> static void dispatch_act_bwd(const ActBwdArgs& a, bool vec, dim3 grid, cudaStream_t s) {
    switch (a.act) {
    case GACT_ACT_RELU: return launch_act_bwd<DT, GACT_ACT_RELU>(a, vec, grid, s);
    case GACT_ACT_GELU: return launch_act_bwd<DT, GACT_ACT_GELU>(a, vec, grid, s);
    case GACT_ACT_GELU_TANH: return launch_act_bwd<DT, GACT_ACT_GELU_TANH>(a, vec, grid, s);
    case GACT_ACT_SILU: return launch_act_bwd<DT, GACT_ACT_SILU>(a, vec, grid, s);
    default: return launch_act_bwd<DT, GACT_ACT_NONE>(a, vec, grid, s);
    }
}

static bool dims_ok(int64_t rows, int64_t cin, int64_t cout) {
    return rows >= 0 && cin >= 1 && cout >= 1 && cin <= GACT_MAX_COLS && cout <= GACT_MAX_COLS && rows <= (1LL << 30) &&
           rows <= GACT_MAX_ELEMENTS / pitch8(cin) && rows <= GACT_MAX_ELEMENTS / pitch8(cout);
}
// operands of the products are read by tensor maps: 16-byte aligned base and row pitch
static bool map_ok(const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0; }

int linear_error_word() {
    int v = 0;
    return cudaMemcpyFromSymbol(&v, g_linear_error, sizeof(int)) == cudaSuccess ? v : -1;
}
int linear_error_clear() {
    const int zero = 0;
    return cudaMemcpyToSymbol(g_linear_error, &zero, sizeof(int)) == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
}

}  // namespace gact

using namespace gact;

extern "C" int64_t gact_linear_scratch_bytes(int64_t rows, int64_t cin, int64_t cout, int direction) {
    if (!dims_ok(rows, cin, cout) || direction < 0 || direction > 2) return -1;
    if (rows == 0) return 0;
    return direction == 0 ? gemm_scratch(rows, cout, cin, true) : direction == 1 ? gemm_scratch(rows, cin, cout, false) : gemm_scratch(cout, cin, rows, false);
}

static SideJob sums_job(const void* partial, int64_t rows, int64_t cols, void* sums) {
    SideJob j = {};
    j.partial = (const float*)partial; j.parts = (int)act_bwd_parts(rows, cols); j.width = (cols + 7) / 8 * 8; j.sums = sums; j.n = cols;
    return j;
}
// Whether a side job beside a product is worth it.  Measured: a block's pair of idle warps makes 2 elements of a checkpoint or
// restores 4 a nanosecond (64 x 1024 beside a single block: 32 us); beside full epilogues and copies all of them together make
// 204, or restore 345.
// A checkpoint beside the product slows its epilogue by more than the kernel of its own takes, except where it saves little
// more than the launch; a restored x is free while it ends well before the product (8192 x 1024 beside 4096 -> 1024: 2 us
// instead of 6.5; 8192 x 4096 beside 1024 -> 4096: 44 us instead of 18).
static bool beside(int kind, int64_t M, int64_t N, int64_t K, int64_t elements) {
    const Plan p = plan_gemm(M, N, K, kind == 1);
    const double blocks = (double)(p.tiles_m * p.tiles_n * p.splits * p.cg), sms = sm_count();
    const double pairs = blocks < sms ? blocks : sms, each = kind == 1 ? 2.0 : 4.0, all = kind == 1 ? 204.0 : 345.0;
    const double alone = (double)elements / (each * pairs), shared = (double)elements / all;
    return (alone <= 4000.0 && shared <= 2000.0) || (kind == 2 && (alone > shared ? alone : shared) <= 0.75 * p.ns);
}

extern "C" int gact_linear(const void* x, int64_t ld_x, const void* weight, int64_t ld_w, const void* bias, const void* residual, int64_t ld_res,
                           int dtype, int64_t rows, int64_t cin, int64_t cout, int act, void* y, void* xcodes, void* xscales, void* z, void* zcodes,
                           void* zscales, int rounding, uint64_t seed, void* scratch, void* stream) {
    if (dtype != GACT_F16 && dtype != GACT_BF16) return GACT_ERR_DTYPE;
    if (act < GACT_ACT_NONE || act > GACT_ACT_SILU) return GACT_ERR_MODE;
    if (!dims_ok(rows, cin, cout) || ld_x < cin || ld_w < cin || (residual && ld_res < cout)) return GACT_ERR_SIZE;
    if (rows == 0) return GACT_OK;
    if (const int st = rounding_status(rounding, seed, GACT_CODES_STOCHASTIC | GACT_CODES_DEVICE_SEED)) return st;
    if (!x || !weight || !y || (xcodes && !xscales) || (zcodes && !zscales)) return GACT_ERR_NULL;
    if (!map_ok(x, ld_x) || !map_ok(weight, ld_w) || (((uintptr_t)y | (uintptr_t)z | (uintptr_t)bias | (uintptr_t)residual) & 1) ||
        ((uintptr_t)zcodes & 31) || ((uintptr_t)xcodes & 31) || ((uintptr_t)scratch & 31))
        return GACT_ERR_ALIGN;
    if (gemm_scratch(rows, cout, cin, true) && !scratch) return GACT_ERR_NULL;
    GemmArgs a = {};
    a.M = rows; a.N = cout; a.out = y; a.ldo = cout; a.ovec = vec_bytes(y, cout);
    a.bias = bias;
    a.res = residual; a.ldr = ld_res; a.rvec = vec_bytes(residual, ld_res);
    a.act = act; a.z = z; a.zvec = vec_bytes(z, cout);
    a.zcodes = (int8_t*)zcodes; a.zscales = (uint8_t*)zscales; a.zpitch = pitch8(cout);
    // the codes of the pre-activation draw their noise from another key than those of the input
    const bool stochastic = rounding & GACT_CODES_STOCHASTIC, on_device = rounding & GACT_CODES_DEVICE_SEED;
    a.stochastic = stochastic; a.noise = Noise8::of(seed, on_device, 0x9E3779B97F4A7C15ull);
    if (xcodes) {
        if (beside(1, rows, cout, cin, rows * cin)) {
            SideJob& j = a.side;
            j.kind = 1; j.x = x; j.ld = ld_x; j.stochastic = stochastic; j.noise = Noise8::of(seed, on_device, 0);
            j.codes = (int8_t*)xcodes; j.scales = (uint8_t*)xscales; j.rows = rows; j.cols = (int)cin; j.chunks = (int)(pitch8(cin) / 8);
            j.by = Divisor::of(j.chunks);
        } else {
            const int st = gact_checkpoint8(x, dtype, rows, cin, ld_x, rounding, seed, xcodes, xscales, stream);
            if (st != GACT_OK) return st;
        }
    }
    cudaStream_t s = (cudaStream_t)stream;
    return dtype == GACT_F16 ? run_gemm<GACT_F16, false, false, true>(x, ld_x, weight, ld_w, cin, a, scratch, s)
                             : run_gemm<GACT_BF16, false, false, true>(x, ld_x, weight, ld_w, cin, a, scratch, s);
}

extern "C" int gact_linear_dgrad(const void* dz, int64_t ld_dz, const void* weight, int64_t ld_w, int dtype, int64_t rows, int64_t cin, int64_t cout,
                                 void* dx, const void* dbias_partial, void* dbias, const void* xcodes, const void* xscales, void* x_restored,
                                 void* scratch, void* stream) {
    if (dtype != GACT_F16 && dtype != GACT_BF16) return GACT_ERR_DTYPE;
    if (!dims_ok(rows, cin, cout) || ld_dz < cout || ld_w < cin) return GACT_ERR_SIZE;
    if (rows == 0) return GACT_OK;
    if (!dz || !weight || !dx || (gemm_scratch(rows, cin, cout, false) && !scratch) || (!dbias_partial != !dbias) || (x_restored && (!xcodes || !xscales)))
        return GACT_ERR_NULL;
    if (!map_ok(dz, ld_dz) || !map_ok(weight, ld_w) || ((uintptr_t)dx & 1) || ((uintptr_t)dbias & 1) || ((uintptr_t)dbias_partial & 3) ||
        ((uintptr_t)xcodes & 31) || ((uintptr_t)x_restored & 15) || ((uintptr_t)scratch & 31))
        return GACT_ERR_ALIGN;
    GemmArgs a = {};
    a.M = rows; a.N = cin; a.out = dx; a.ldo = cin; a.ovec = vec_bytes(dx, cin);
    if (dbias) a.side = sums_job(dbias_partial, rows, cout, dbias);
    if (x_restored) {
        const int64_t pitch = pitch8(cin);
        if (beside(2, rows, cin, cout, rows * cin)) {
            SideJob& j = a.side;
            j.kind = 2; j.codes = (int8_t*)xcodes; j.scales = (uint8_t*)xscales; j.out = x_restored;
            j.rows = rows; j.cols = (int)cin; j.chunks = (int)(pitch / 8);
        } else {
            const int st = gact_restore8(xcodes, xscales, rows, cin, dtype, x_restored, pitch, stream);
            if (st != GACT_OK) return st;
        }
    }
    cudaStream_t s = (cudaStream_t)stream;
    return dtype == GACT_F16 ? run_gemm<GACT_F16, false, true, false>(dz, ld_dz, weight, ld_w, cout, a, scratch, s)
                             : run_gemm<GACT_BF16, false, true, false>(dz, ld_dz, weight, ld_w, cout, a, scratch, s);
}

extern "C" int gact_linear_wgrad(const void* dz, int64_t ld_dz, const void* x, int64_t ld_x, int dtype, int64_t rows, int64_t cin, int64_t cout,
                                 void* dweight, const void* dbias_partial, void* dbias, void* scratch, void* stream) {
    if (dtype != GACT_F16 && dtype != GACT_BF16) return GACT_ERR_DTYPE;
    if (!dims_ok(rows, cin, cout) || ld_dz < cout || ld_x < cin) return GACT_ERR_SIZE;
    cudaStream_t s = (cudaStream_t)stream;
    if (!dweight) return GACT_ERR_NULL;
    if (rows == 0) {
        if (dbias && cudaMemsetAsync(dbias, 0, (size_t)cout * 2, s) != cudaSuccess) return GACT_ERR_LAUNCH;
        return cudaMemsetAsync(dweight, 0, (size_t)(cin * cout * 2), s) == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
    }
    if (!dz || !x || (gemm_scratch(cout, cin, rows, false) && !scratch) || (!dbias_partial != !dbias)) return GACT_ERR_NULL;
    if (!map_ok(dz, ld_dz) || !map_ok(x, ld_x) || ((uintptr_t)dweight & 1) || ((uintptr_t)dbias & 1) || ((uintptr_t)dbias_partial & 3) ||
        ((uintptr_t)scratch & 31))
        return GACT_ERR_ALIGN;
    GemmArgs a = {};
    a.M = cout; a.N = cin; a.out = dweight; a.ldo = cin; a.ovec = vec_bytes(dweight, cin);
    if (dbias) a.side = sums_job(dbias_partial, rows, cout, dbias);
    return dtype == GACT_F16 ? run_gemm<GACT_F16, true, true, false>(dz, ld_dz, x, ld_x, rows, a, scratch, s)
                             : run_gemm<GACT_BF16, true, true, false>(dz, ld_dz, x, ld_x, rows, a, scratch, s);
}

extern "C" int64_t gact_act_backward_scratch_bytes(int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 1 || cols > GACT_MAX_COLS) return -1;
    return act_bwd_parts(rows, cols) * ((cols + 7) / 8 * 8) * (int64_t)sizeof(float);
}

extern "C" int gact_act_backward(const void* dy, int dtype, int64_t rows, int64_t cols, int64_t ld_dy, int act, const void* z, int64_t ld_z,
                                 const void* zcodes, const void* zscales, void* dz, int64_t ld_dz, void* dbias, void* scratch, void* stream) {
    if (dtype != GACT_F16 && dtype != GACT_BF16) return GACT_ERR_DTYPE;
    if (act < GACT_ACT_NONE || act > GACT_ACT_SILU) return GACT_ERR_MODE;
    if (rows < 0 || cols < 1 || cols > GACT_MAX_COLS || rows > GACT_MAX_ELEMENTS / pitch8(cols) || ld_dy < cols || (z && ld_z < cols) ||
        (dz && ld_dz < cols))
        return GACT_ERR_SIZE;
    cudaStream_t s = (cudaStream_t)stream;
    if (rows == 0) return !dbias || cudaMemsetAsync(dbias, 0, (size_t)cols * 2, s) == cudaSuccess ? GACT_OK : GACT_ERR_LAUNCH;
    if (!dy || (act != GACT_ACT_NONE && (!dz || (!z && (!zcodes || !zscales)))) || (dbias && !scratch)) return GACT_ERR_NULL;
    if (act == GACT_ACT_NONE && !scratch && !dz) return GACT_OK;
    if ((((uintptr_t)dy | (uintptr_t)z | (uintptr_t)dz | (uintptr_t)dbias) & 1) || ((uintptr_t)zcodes & 31) || ((uintptr_t)scratch & 15)) return GACT_ERR_ALIGN;
    ActBwdArgs a;
    a.dy = dy; a.ldy = ld_dy; a.z = z; a.ldz = ld_z; a.codes = z ? nullptr : (const int8_t*)zcodes; a.scales = (const uint8_t*)zscales;
    a.chunks = (int)(pitch8(cols) / 8); a.act = act; a.rows = rows; a.cols = (int)cols; a.dz = dz; a.ldo = ld_dz;
    a.partial = (float*)scratch; a.width = (int)((cols + 7) / 8 * 8);
    const bool vec = rows_aligned(dy, ld_dy, cols, 2) && (!dz || rows_aligned(dz, ld_dz, cols, 2)) &&
                     (act == GACT_ACT_NONE || !z || rows_aligned(z, ld_z, cols, 2));
    const int64_t parts = act_bwd_parts(rows, cols);
    const dim3 grid((unsigned)((cols + 255) / 256), (unsigned)parts);
    if (dtype == GACT_F16) dispatch_act_bwd<GACT_F16>(a, vec, grid, s);
    else dispatch_act_bwd<GACT_BF16>(a, vec, grid, s);
    if (cudaGetLastError() != cudaSuccess) return GACT_ERR_LAUNCH;
    return dbias ? reduce_columns((const float*)scratch, (int)parts, a.width, dbias, cols, nullptr, 0, dtype, kSumChains, s) : GACT_OK;
}
