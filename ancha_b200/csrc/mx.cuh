// Microscaled arrays: rows of 8-bit or 4-bit floating-point elements with one scale for each block
// of consecutive elements of a row, and the device arithmetic that makes and expands them.
//
//   format       element        block  block scale                  array scale
//   ANCHA_MXF8   E4M3 (8 bit)   32     E8M0, 2^(code - 127)         -
//   ANCHA_MXF4   E2M1 (4 bit)   32     E8M0                         -
//   ANCHA_NVF4   E2M1 (4 bit)   16     E4M3                         one f32 (device) or 1
//
// Elements lie row-major, `ld` bytes apart, the even column of a 4-bit pair in the low half of its
// byte. Scales lie in the order in which the tensor cores take them: 512-byte tiles of 128 rows by
// four blocks, tiles of one row range side by side,
//   byte(row, block) = ((row / 128) * kt + block / 4) * 512 + (row % 32) * 16 + (row % 128) / 32 * 4 + block % 4
// with kt = ceil(blocks / 4). What a tile holds behind the last row or block is written as 0.
#pragma once

#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include "tc.cuh"

namespace ancha {

enum : int { MXF8 = ANCHA_MXF8, MXF4 = ANCHA_MXF4, NVF4 = ANCHA_NVF4 };

// Limits of an array: its coordinates are the tensor maps' 32-bit ones, and no byte count leaves 64 bits.
constexpr int64_t kMaxMxRows = (int64_t(1) << 31) - 512, kMaxMxCols = (int64_t(1) << 31) - 512;
constexpr int64_t kMaxMxLd = int64_t(1) << 32;  // rows apart: bytes of an array, elements of a matrix
constexpr int kMaxNormCols = 32768;

// A validated ancha_mx_array.
struct MxArray {
    int format;
    int64_t rows;
    int cols;
    uint8_t* data;
    int64_t ld;
    uint8_t* scales;
    const float* global_scale;  // device, NVF4 only; null = 1
};

__host__ __device__ constexpr int mx_block(int format) { return format == NVF4 ? 16 : 32; }
// Bytes of `cols` elements.
__host__ __device__ constexpr int64_t mx_bytes(int format, int64_t cols) {
    return format == MXF8 ? cols : (cols + 1) / 2;
}
// Bytes of a row that are written: the elements and zeros up to a multiple of 16.
__host__ __device__ constexpr int64_t mx_row_bytes(int format, int64_t cols) {
    return (mx_bytes(format, cols) + 15) / 16 * 16;
}
// Scale tiles along a row.
__host__ __device__ constexpr int64_t mx_ktiles(int format, int64_t cols) {
    return (cols + 4 * mx_block(format) - 1) / (4 * mx_block(format));
}

struct MxLinear {
    MxArray x, w;           // [m, k], [n, k], one format
    const float* bias;      // [n] or null
    const void* residual;   // [m, n] of res_type or null
    int res_type;
    int64_t ldr;
    int act;                // ANCHA_ACT_NONE / GELU / TANH
    void* out;              // [m, n] of out_type, or null with out_mx
    int out_type;
    int64_t ldo;
    const MxArray* out_mx;  // [m, n] or null
};

int mx_quantize(const void* x, int dtype, int64_t ldx, const MxArray& out, cudaStream_t s);
int mx_dequantize(const MxArray& x, void* out, int dtype, int64_t ldo, cudaStream_t s);
int mx_add_rms_norm(const void* x, int dtype, int64_t ldx, const void* residual, int res_type, int64_t ldr,
                    void* residual_out, int64_t ldro, const float* gain, double eps, const MxArray& out,
                    cudaStream_t s);
int mx_linear(const MxLinear& q, cudaStream_t s);

#ifdef __CUDACC__

// Offset of the 32-bit word that holds the scales of a row's blocks 4 kw .. 4 kw + 3.
__device__ __forceinline__ int64_t mx_scale_word(int64_t row, int kw, int64_t kt) {
    return ((row >> 7) * kt + kw) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4;
}

__device__ __forceinline__ float e4m3_value(uint32_t code) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3);
    return __half2float(__half(h));
}

// 2^(code - 127); 255 is NaN and 0 the f32 subnormal 2^-127.
__device__ __forceinline__ float e8m0_value(uint32_t code) {
    return __uint_as_float(code == 255 ? 0x7FC00000u : code == 0 ? 0x00400000u : code << 23);
}

// The value a block's scale code stands for, without the array scale.
template <int FMT>
__device__ __forceinline__ float mx_scale_value(uint32_t code) {
    return FMT == NVF4 ? e4m3_value(code) : e8m0_value(code);
}

// How a block is quantised: the code of its scale, and each element as v * factor (MX: a power of two, exact) or
// v / factor (NVF4). A block with an infinity or a NaN has the scale NaN and elements 0; `live` is false for it, and
// where the divisor is 0.
struct MxBlock {
    uint32_t code;
    float factor;
    bool live;
};

// `amax_bits`: the largest of the block's |v| as f32 bits (as integers NaN > infinity > every number).
// MX: the least power of two at which |v| max still rounds into the element's range, which for E4M3 is
// up to 464 (a tie with the unrepresentable 480, to the even 448) and for E2M1 below 7. Rounding the
// largest element down where that is its nearest value costs less than halving the resolution of the
// rest: on normal data the rms error is 11.2 % for E2M1, against 11.5 % with the next power of two
// from 6 on and 11.5 % with one power of two for all of [4, 8); 2.65 % for E4M3 (2.94 % for the latter).
template <int FMT>
__device__ __forceinline__ MxBlock mx_block_scale(uint32_t amax_bits, float global) {
    MxBlock b;
    const bool bad = amax_bits >= 0x7F800000u;
    if (FMT == NVF4) {
        const float s = bad ? 0.f : fminf(__uint_as_float(amax_bits) / (6.f * global), 448.f);
        b.code = __nv_cvt_float_to_fp8(s, __NV_SATFINITE, __NV_E4M3);
        b.factor = e4m3_value(b.code) * global;
        b.live = !bad && b.factor > 0.f;
        if (bad) b.code = 0x7F;
    } else {
        const int field = (int)(amax_bits >> 23);
        const uint32_t mantissa = amax_bits & 0x7FFFFFu;
        const int top = FMT == MXF8 ? mantissa > 0x680000u : mantissa >= 0x600000u;
        const int code = max(field - (FMT == MXF8 ? 8 : 2) + top, 0);
        b.code = bad ? 255u : (uint32_t)code;
        b.factor = __uint_as_float((uint32_t)(254 - code) << 23);
        b.live = !bad;
    }
    return b;
}

// max(m, |a|, |b|); NaN where one is.
__device__ __forceinline__ float absmax(float m, float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
    return d;
}

__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}
__device__ __forceinline__ uint32_t pack_e2m1(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\tmov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// Codes of N elements of one block (or a part of one), 4 or 8 to a word.
// NVF4: dividing every element costs eight instructions or more. The product with the rounded reciprocal is off
// by less than 2^-22 of the quotient, so where rounding it down and up by 2^-21 gives one code that is the
// quotient's too; otherwise (next to a border) the elements are divided.
template <int FMT, int N>
__device__ __forceinline__ void mx_encode(const float (&v)[N], const MxBlock& b, uint32_t (&w)[N / (FMT == MXF8 ? 4 : 8)]) {
    constexpr int PER = FMT == MXF8 ? 4 : 8, W = N / PER;
    const uint32_t mask = b.live ? 0xffffffffu : 0u;
    if constexpr (FMT == NVF4) {
        const float r = __frcp_rn(b.factor), lo = r * (1.f - 0x1p-21f), hi = r * (1.f + 0x1p-21f);
        bool same = b.factor > 1e-30f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            float t[8], u[8];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const uint64_t x = f2(v[8 * i + j], v[8 * i + j + 1]);
                f2_split(fmul2(x, f2(lo, lo)), t[j], t[j + 1]);
                f2_split(fmul2(x, f2(hi, hi)), u[j], u[j + 1]);
            }
            w[i] = pack_e2m1(t) & mask;
            same = same && w[i] == (pack_e2m1(u) & mask);
        }
        if (!same && b.live) {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                float t[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = __fdiv_rn(v[8 * i + j], b.factor);
                w[i] = pack_e2m1(t);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            float t[PER];
#pragma unroll
            for (int j = 0; j < PER; j += 2)
                f2_split(fmul2(f2(v[PER * i + j], v[PER * i + j + 1]), f2(b.factor, b.factor)), t[j], t[j + 1]);
            if constexpr (FMT == MXF8) w[i] = pack_e4m3(t[0], t[1], t[2], t[3]) & mask;
            else w[i] = pack_e2m1(t) & mask;
        }
    }
}

template <int FMT>
__device__ __forceinline__ float2 mx_pair_values(uint32_t code) {
    const __half2_raw h = FMT == MXF8 ? __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)code, __NV_E4M3)
                                      : __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)code, __NV_E2M1);
    return __half22float2(__half2(h));
}

#endif  // __CUDACC__

}  // namespace ancha
