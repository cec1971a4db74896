// The 8-bit activation checkpoint, and eight-element row accesses shared by the operators that keep one.
//
// A row of `cols` elements is cut into blocks of 32 (the last one may be short).  A block stores one scale byte b, the
// biased exponent of a power of two, and a signed byte per element:
//     b    = max(1, ((bits(max|x|) + 0x20000) >> 23) - 6)      255 when the block holds a NaN or an infinity
//     code = rint(x * 2^(127-b))   (or floor(x * 2^(127-b) + u), u in (0,1) from Philox)
//     x'   = code * 2^(b-127)      (NaN where b = 255)
// Adding 0x20000 to the bits carries into the exponent exactly when the largest magnitude would reach 127 steps, so it
// always lands in [63.5, 127) steps and no code needs a clamp.  Scales are powers of two, so the scaling is exact: a code
// does not depend on which kernel computed it, and a restored value (a 7-bit integer times a power of two) is exact in
// bf16, fp16 (above its subnormals) and fp32: backward passes read codes without a second rounding.
// The one exception is the highest binade of the type, where a code of 64 would restore to the next power of two, out
// of range: there magnitudes stop at 63 steps.
#pragma once

#include <type_traits>

#include "gact_common.cuh"

namespace gact {

constexpr int kBlock8 = GACT_BLOCK8;      // elements per scale

static __host__ __device__ __forceinline__ int64_t pitch8(int64_t cols) { return (cols + kBlock8 - 1) / kBlock8 * kBlock8; }

// highest scale byte a finite value of the type can give: 64 steps of it are out of range
template <int DT> __device__ __forceinline__ constexpr uint32_t top_byte8() { return DT == GACT_F16 ? 137u : 249u; }

// scale byte from the largest |x| of a block, given as its fp32 bit pattern (ordered like the magnitudes, NaN on top)
__device__ __forceinline__ uint32_t scale_byte8(uint32_t absmax) {
    const int b = (int)((absmax + 0x20000u) >> 23) - 6;
    return absmax >= 0x7f800000u ? 255u : (uint32_t)max(b, 1);
}
// 2^(127-b); 0 for b = 255, which sends every finite element to code 0 (NaN and inf are caught by the caller)
__device__ __forceinline__ float scale_up8(uint32_t b) { return b == 255u ? 0.0f : __uint_as_float((254u - b) << 23); }
// 2^(b-127); NaN for b = 255
__device__ __forceinline__ float scale_down8(uint32_t b) { return b == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(b << 23); }

// Noise of stochastic rounding: Philox4x32-7, one call per 8 consecutive elements of the padded row layout (low half of the
// counter = element index / 8), 16 bits each: u = (r + 0.5) / 65536.  A seed is the key; one that lies on the device (a captured
// launch cannot be given another key) is the high half of the counter instead.
struct Noise8 {
    PhiloxKeys rk; const uint2* word;
    static Noise8 of(uint64_t seed, bool on_device, uint64_t other) {
        return {philox_round_keys((on_device ? 0 : seed) + other), on_device ? (const uint2*)(uintptr_t)seed : nullptr};
    }
    __device__ __forceinline__ uint2 high() const { return word ? __ldg(word) : make_uint2(0u, 0u); }
};
__device__ __forceinline__ uint4 noise8(const Noise8& n, uint2 high, uint64_t chunk) {
    return philox4x32<7>((uint32_t)chunk, (uint32_t)(chunk >> 32), high.x, high.y, n.rk);
}
// the `rounding` argument of the entry points: a known combination, and a seed on the device that can be read
static inline int rounding_status(int rounding, uint64_t seed, int known) {
    if ((rounding & ~known) || ((rounding & GACT_CODES_DEVICE_SEED) && !(rounding & GACT_CODES_STOCHASTIC))) return GACT_ERR_MODE;
    if (rounding & GACT_CODES_DEVICE_SEED) return !seed ? GACT_ERR_NULL : (seed & 7) ? GACT_ERR_ALIGN : GACT_OK;
    return GACT_OK;
}
__device__ __forceinline__ float noise8_at(const uint4& r, int j) {
    const uint32_t w = word_of(r, j >> 1);
    const uint32_t h = (j & 1) ? (w >> 16) : (w & 0xffffu);
    return __fmaf_rn((float)h, 1.0f / 65536.0f, 0.5f / 65536.0f);
}

// One code in the low byte.  |x * up| < 127, so adding 1.5 * 2^23 leaves the rounded integer in the low mantissa bits;
// rounding that sum down instead of to nearest gives floor(x * up + u) (the product is exact, x * up + u keeps 2^-17).
__device__ __forceinline__ uint32_t code8(float x, float up) { return __float_as_uint(__fmaf_rn(x, up, 12582912.0f)); }
__device__ __forceinline__ uint32_t code8_noise(float x, float up, float u) {
    return __float_as_uint(__fadd_rd(__fmaf_rn(x, up, u), 12582912.0f));
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// codes of the highest binade: keep |code| <= 63
static __device__ __noinline__ uint32_t clamp_codes63(uint32_t w) {
    uint32_t out = 0;
    for (int i = 0; i < 4; i++) {
        int c = (int)(int8_t)(w >> (8 * i));
        c = min(63, max(-63, c));
        out |= (uint32_t)(c & 0xff) << (8 * i);
    }
    return out;
}

// Loads that are issued a step ahead of their use.  As volatile statements they stay where they are written; plain loads were
// moved down to their first use, where every step waited for them.
__device__ __forceinline__ uint32_t ld_ahead_byte(const uint8_t* p) {
    uint32_t v;
    asm volatile("ld.global.nc.u8 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ float2 ld_ahead_float2(const float2* p) {
    float2 v;
    asm volatile("ld.global.nc.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ld_ahead_u16(const uint16_t* p) {
    uint16_t v;
    asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ld_ahead_u32(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}

// ---- eight consecutive elements of a row, as four pairs (two fp32 operations per instruction) -----------------------
template <int DT> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (DT == GACT_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *(const uint32_t*)&h;
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *(const uint32_t*)&h;
    }
}
template <int DT> __device__ __forceinline__ void raw_to_pairs(const uint32_t (&raw)[RawRegs<DT>::N], float2 (&v)[4]) {
    float f[8];
    raw_to_float<DT>(raw, f);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = make_float2(f[2 * i], f[2 * i + 1]);
}
template <int DT> __device__ __forceinline__ void pairs_to_raw(const float2 (&v)[4], uint32_t (&raw)[RawRegs<DT>::N]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (DT == GACT_F32) { raw[2 * i] = __float_as_uint(v[i].x); raw[2 * i + 1] = __float_as_uint(v[i].y); }
        else raw[i] = pack2<DT>(v[i].x, v[i].y);
    }
}
// the larger of m and two magnitudes; NaN if there is one
__device__ __forceinline__ float absmax3(float m, float2 v) {
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(m), "f"(v.x), "f"(v.y));
    return m;
}
// the largest magnitude of the eight, as an fp32 bit pattern
template <int DT> __device__ __forceinline__ uint32_t absmax8(const uint32_t (&raw)[RawRegs<DT>::N]) {
    uint32_t m;
    if constexpr (DT == GACT_F32) {
        m = raw[0] & 0x7fffffffu;
#pragma unroll
        for (int i = 1; i < 8; i++) m = max(m, raw[i] & 0x7fffffffu);
    } else if constexpr (DT == GACT_BF16) {
        // |.| of two at a time, NaN kept; the sign of the result is the xor of both and is dropped at the end
        asm("{ .reg .b32 a, b; max.NaN.xorsign.abs.bf16x2 a, %1, %2; max.NaN.xorsign.abs.bf16x2 b, %3, %4; max.NaN.xorsign.abs.bf16x2 %0, a, b; }"
            : "=r"(m) : "r"(raw[0]), "r"(raw[1]), "r"(raw[2]), "r"(raw[3]));
        m = max((m << 16) & 0x7fffffffu, m & 0x7fff0000u);
    } else {
        asm("{ .reg .b32 a, b; max.NaN.xorsign.abs.f16x2 a, %1, %2; max.NaN.xorsign.abs.f16x2 b, %3, %4; max.NaN.xorsign.abs.f16x2 %0, a, b; }"
            : "=r"(m) : "r"(raw[0]), "r"(raw[1]), "r"(raw[2]), "r"(raw[3]));
        const float2 f = __half22float2(*(const __half2*)&m);
        m = max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu);
    }
    return m;
}

// The codes of 8 consecutive elements (chunk number `chunk` of the padded rows); a block of 32 lies in 4 neighbouring
// lanes and every lane of the warp must call.  `m`: the lane's largest magnitude; `last`: top_byte8 of the type that the codes
// are restored to.  Returns the scale byte too.
template <bool STOCH>
__device__ __forceinline__ uint2 codes8(const float2 (&v)[4], uint32_t m, const Noise8& noise, uint2 high, uint64_t chunk, uint32_t& byte, uint32_t last) {
    m = max(m, __shfl_xor_sync(kFull, m, 1));
    m = max(m, __shfl_xor_sync(kFull, m, 2));
    byte = scale_byte8(m);
    const float up = scale_up8(byte);
    uint32_t c[8];
    if constexpr (STOCH) {
        const uint4 r = noise8(noise, high, chunk);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            c[2 * i] = code8_noise(v[i].x, up, noise8_at(r, 2 * i));
            c[2 * i + 1] = code8_noise(v[i].y, up, noise8_at(r, 2 * i + 1));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 t = fma2(v[i], splat2(up), splat2(12582912.0f));
            c[2 * i] = __float_as_uint(t.x);
            c[2 * i + 1] = __float_as_uint(t.y);
        }
    }
    uint2 w = make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
    if (byte >= last) {
        if (byte == 255u) w = make_uint2(0u, 0u);
        else w = make_uint2(clamp_codes63(w.x), clamp_codes63(w.y));
    }
    return w;
}
// eight codes as integers in fp32 (exact): the byte with its sign bit flipped goes into the mantissa of 2^23 (offset
// binary), one subtraction takes the offset off again
__device__ __forceinline__ void code_pairs(uint2 w, float2 (&v)[4]) {
    const uint32_t a = w.x ^ 0x80808080u, b = w.y ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t q = i < 2 ? a : b;
        v[i] = add2(make_float2(__uint_as_float(__byte_perm(q, 0x4b000000u, 0x7540 | (2 * (i & 1)))),
                                __uint_as_float(__byte_perm(q, 0x4b000000u, 0x7540 | (2 * (i & 1) + 1)))),
                    splat2(-8388736.0f));
    }
}
__device__ __forceinline__ void restore_pairs(uint2 w, float down, float2 (&v)[4]) {
    code_pairs(w, v);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = mul2(v[i], splat2(down));
}

// A lane's 8 elements of a row, from memory.  VEC: rows start on 16-byte boundaries and hold a multiple of 8 elements,
// one or two 16-byte accesses.  Otherwise a warp reads its 32 x 8 elements one lane-contiguous 32 at a time and turns
// them around in shared memory (8 elements per lane straight from memory would touch every sector eight times).
// SUB lanes of the warp share a row (32: the whole warp); rows of the lane groups follow one another.
template <int DT, bool VEC, int SUB> struct Row8 {
    using T = typename Elem<DT>::T;
    using U = typename std::conditional<DT == GACT_F32, uint32_t, uint16_t>::type;
    static constexpr int N = VEC ? RawRegs<DT>::N : 8;
    uint32_t r[N];

    // base + row * ld: the row of this lane's group; col: the lane's first column; nothing is read at or past `cols`
    __device__ __forceinline__ void load(const T* base, int64_t ld, int64_t row, int64_t rows, int col, int cols) {
        if constexpr (VEC) {
            if (row < rows && col < cols) {
                const T* p = base + row * ld + col;
                const uint4 a = ld_stream_u4(p);
                r[0] = a.x; r[1] = a.y; r[2] = a.z; r[3] = a.w;
                if constexpr (DT == GACT_F32) {
                    const uint4 b = ld_stream_u4(p + 4);
                    r[4] = b.x; r[5] = b.y; r[6] = b.z; r[7] = b.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; i++) r[i] = 0;
            }
        } else {
            const int lane = threadIdx.x & 31;
            const int64_t row0 = row - lane / SUB;
            const int col0 = col - (lane % SUB) * 8;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int e = i * 32 + lane, g = e / (SUB * 8), c = col0 + e % (SUB * 8);
                r[i] = 0u;
                if (row0 + g < rows && c < cols) {
                    if constexpr (DT == GACT_F32) r[i] = ld_ahead_u32((const uint32_t*)base + (row0 + g) * ld + c);
                    else r[i] = ld_ahead_u16((const uint16_t*)base + (row0 + g) * ld + c);
                }
            }
        }
    }
    // the elements in storage format; `stage`: 256 elements of the warp (not used with VEC)
    __device__ __forceinline__ void get(void* stage, uint32_t (&raw)[RawRegs<DT>::N]) const {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < N; i++) raw[i] = r[i];
        } else {
            const int lane = threadIdx.x & 31;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; i++) ((U*)stage)[i * 32 + lane] = (U)r[i];
            __syncwarp();
            const uint4 a = ((const uint4*)stage)[DT == GACT_F32 ? 2 * lane : lane];
            raw[0] = a.x; raw[1] = a.y; raw[2] = a.z; raw[3] = a.w;
            if constexpr (DT == GACT_F32) {
                const uint4 b = ((const uint4*)stage)[2 * lane + 1];
                raw[4] = b.x; raw[5] = b.y; raw[6] = b.z; raw[7] = b.w;
            }
        }
    }
    static __device__ __forceinline__ void store(T* base, int64_t ld, int64_t row, int64_t rows, int col, int cols, void* stage, const float2 (&v)[4]) {
        uint32_t raw[RawRegs<DT>::N];
        pairs_to_raw<DT>(v, raw);
        if constexpr (VEC) {
            if (row < rows && col < cols) {
                T* p = base + row * ld + col;
                st_stream_u4(p, make_uint4(raw[0], raw[1], raw[2], raw[3]));
                if constexpr (DT == GACT_F32) st_stream_u4(p + 4, make_uint4(raw[4], raw[5], raw[6], raw[7]));
            }
        } else {
            const int lane = threadIdx.x & 31;
            const int64_t row0 = row - lane / SUB;
            const int col0 = col - (lane % SUB) * 8;
            __syncwarp();
            ((uint4*)stage)[DT == GACT_F32 ? 2 * lane : lane] = make_uint4(raw[0], raw[1], raw[2], raw[3]);
            if constexpr (DT == GACT_F32) ((uint4*)stage)[2 * lane + 1] = make_uint4(raw[4], raw[5], raw[6], raw[7]);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int e = i * 32 + lane, g = e / (SUB * 8), c = col0 + e % (SUB * 8);
                if (row0 + g < rows && c < cols) ((U*)base)[(row0 + g) * ld + c] = ((const U*)stage)[e];
            }
        }
    }
};
// bytes of shared memory per warp that Row8 needs
template <int DT, bool VEC> struct Stage8 { static constexpr int kBytes = VEC ? 0 : 256 * Elem<DT>::kBytes; };

// Division by a number known at launch: for i < 2^31 one multiplication, i / d = i * mul >> (31 + s) with s = ceil(log2 d)
// and mul = floor(2^(31+s) / d) + 1 < 2^32 (the excess mul * d - 2^(31+s) is at most d <= 2^s, so the error stays below 1 / d).
// Larger indices take the 64-bit division (a hundred instructions, which would bound the kernel).
struct Divisor {
    uint32_t mul, shift; int64_t d;
    static Divisor of(int64_t d) {
        Divisor v;
        int s = 0;
        while ((1LL << s) < d) s++;
        v.mul = (uint32_t)((1ULL << (31 + s)) / (uint64_t)d + 1);
        v.shift = 31 + s;
        v.d = d;
        return v;
    }
    __device__ __forceinline__ int64_t div(int64_t i) const {
        return i < (1LL << 31) ? (int64_t)(((uint64_t)(uint32_t)i * mul) >> shift) : i / d;
    }
};

// Lets a kernel use `bytes` of dynamic shared memory, once per device.
template <class K> static inline bool allow_smem(K kernel, int bytes, std::atomic<bool> (&done)[kMaxDevices]) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return false;
    if (!done[dev].load(std::memory_order_relaxed)) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
        done[dev].store(true, std::memory_order_relaxed);
    }
    return true;
}

// Blocks of a kernel that one SM holds, asked of the runtime once per device.
template <class K> static inline int resident_blocks(K kernel, int threads, size_t smem, std::atomic<int> (&cache)[kMaxDevices]) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 1;
    int n = cache[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess || n < 1) n = 1;
        cache[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

static inline bool rows_aligned(const void* p, int64_t ld, int64_t cols, int elem_bytes) {
    return ((uintptr_t)p & 15) == 0 && (ld * elem_bytes) % 16 == 0 && cols % 8 == 0;
}
static inline int elem_bytes_of(int dtype) { return dtype == GACT_F32 ? 4 : 2; }

// out[c] = T(sum over p of partial[p * width + c]) in a fixed order (`chains` sums, part p in sum p mod chains, then those in
// order; 8 or 32); defined in layernorm.cu, shared by the operators that reduce a bias or weight gradient over the rows.
// Columns [0, n0) go to out0; with out1, columns [0, width / 2) to out0 and the second half to out1 (null: skipped).
constexpr int kSumChains = 8;                 // the chains of the linear layers' bias gradient, wherever it is finished
int reduce_columns(const float* partial, int parts, int64_t width, void* out0, int64_t n0, void* out1, int64_t n1, int dtype, int chains, cudaStream_t s);

}  // namespace gact
