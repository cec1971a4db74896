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

// Noise of stochastic rounding: Philox4x32-7 keyed by the seed, one call per 8 consecutive elements of the padded row
// layout (counter = element index / 8), 16 bits each: u = (r + 0.5) / 65536.
__device__ __forceinline__ uint4 noise8(const PhiloxKeys& rk, uint64_t chunk) {
    return philox4x32<7>((uint32_t)chunk, (uint32_t)(chunk >> 32), 0u, 0u, rk);
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

// Four codes -> four floats: the byte with its sign bit flipped goes into the mantissa of 2^23 (offset binary), one
// subtraction takes the offset off again, one multiplication applies the power of two; all exact.
__device__ __forceinline__ void restore4(uint32_t w, float down, float (&v)[4]) {
    w ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; i++)
        v[i] = __fmul_rn(__fsub_rn(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540 | i)), 8388736.0f), down);
}
__device__ __forceinline__ void restore8(uint2 w, float down, float (&v)[8]) {
    float a[4], b[4];
    restore4(w.x, down, a);
    restore4(w.y, down, b);
#pragma unroll
    for (int i = 0; i < 4; i++) { v[i] = a[i]; v[4 + i] = b[i]; }
}

// The codes of 8 consecutive elements (chunk `c` of a row), computed by 4 neighbouring lanes per block; every lane of
// the warp must call.  Returns the scale byte too.  Chunks past the row's end hold zeros.
template <int DT, bool STOCH>
__device__ __forceinline__ uint2 codes8(const float (&v)[8], const PhiloxKeys& rk, uint64_t chunk, uint32_t& byte) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    m = max(m, __shfl_xor_sync(kFull, m, 1));
    m = max(m, __shfl_xor_sync(kFull, m, 2));
    byte = scale_byte8(m);
    const float up = scale_up8(byte);
    uint32_t c[8];
    if constexpr (STOCH) {
        const uint4 r = noise8(rk, chunk);
#pragma unroll
        for (int j = 0; j < 8; j++) c[j] = code8_noise(v[j], up, noise8_at(r, j));
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) c[j] = code8(v[j], up);
    }
    uint2 w = make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
    if (byte >= top_byte8<DT>()) {
        if (byte == 255u) w = make_uint2(0u, 0u);
        else w = make_uint2(clamp_codes63(w.x), clamp_codes63(w.y));
    }
    return w;
}

// ---- eight consecutive elements of a row --------------------------------------------------------------------------
// VEC: rows start on 16-byte boundaries and hold a multiple of 8 elements; otherwise element by element.
template <int DT, bool VEC>
__device__ __forceinline__ void load_row8(const typename Elem<DT>::T* row, int col, int cols, float (&v)[8]) {
    if constexpr (VEC) {
        uint32_t raw[RawRegs<DT>::N];
        if (col < cols) {
            const uint4 a = ld_stream_u4(row + col);
            raw[0] = a.x; raw[1] = a.y; raw[2] = a.z; raw[3] = a.w;
            if constexpr (DT == GACT_F32) {
                const uint4 b = ld_stream_u4(row + col + 4);
                raw[4] = b.x; raw[5] = b.y; raw[6] = b.z; raw[7] = b.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < RawRegs<DT>::N; i++) raw[i] = 0;
        }
        raw_to_float<DT>(raw, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = (col + j < cols) ? Elem<DT>::to_float(row[col + j]) : 0.0f;
    }
}

template <int DT> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (DT == GACT_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *(const uint32_t*)&h;
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *(const uint32_t*)&h;
    }
}

template <int DT, bool VEC>
__device__ __forceinline__ void store_row8(typename Elem<DT>::T* row, int col, int cols, const float (&v)[8]) {
    if constexpr (VEC) {
        if (col < cols) {
            if constexpr (DT == GACT_F32) {
                st_stream_u4(row + col, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])));
                st_stream_u4(row + col + 4, make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])));
            } else {
                st_stream_u4(row + col, make_uint4(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7])));
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (col + j < cols) row[col + j] = Elem<DT>::from_float(v[j]);
    }
}

static inline bool rows_aligned(const void* p, int64_t ld, int64_t cols, int elem_bytes) {
    return ((uintptr_t)p & 15) == 0 && (ld * elem_bytes) % 16 == 0 && cols % 8 == 0;
}
static inline int elem_bytes_of(int dtype) { return dtype == GACT_F32 ? 4 : 2; }

// out[c] = T(sum over p of partial[p * width + c]) in a fixed order; defined in layernorm.cu, shared by the operators
// that reduce a bias or weight gradient over the rows.  Columns [0, n0) go to out0, [n0, n0 + n1) to out1 (null: skipped).
int reduce_columns(const float* partial, int parts, int64_t width, void* out0, int64_t n0, void* out1, int64_t n1, int dtype, cudaStream_t s);

}  // namespace gact
