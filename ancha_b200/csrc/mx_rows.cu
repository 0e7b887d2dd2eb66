// Row kernels of the microscaled formats: quantisation, expansion, and the residual addition with
// RMS norm whose output is quantised. All are bounded by HBM: each element is read once and written
// once. A thread owns eight consecutive elements of a row (one 16-byte load of 16-bit elements, two of
// f32), so a block's maximum is a shuffle over four lanes (two for NVF4) and the four scales of a
// 32-bit scale word meet in 16 (8) neighbouring lanes.
#include "mx.cuh"

#include <algorithm>

namespace ancha {
namespace {

// Eight elements of a row from column c, zeros from column `cols` on. `vec`: the row starts on a
// 16-byte boundary (c is a multiple of 8).
__device__ __forceinline__ void load8(const void* row, int dtype, bool vec, int c, int cols, float (&v)[8]) {
    if (vec && c + 8 <= cols) {
        if (dtype == ELT_F32) {
            const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(row) + c);
            const float4 a = p[0], b = p[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + c);
            const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = dtype == ELT_BF16
                                     ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[j]))
                                     : __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
                v[2 * j] = f.x;
                v[2 * j + 1] = f.y;
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        v[j] = 0.f;
        if (c + j < cols)
            v[j] = dtype == ELT_F32    ? static_cast<const float*>(row)[c + j]
                   : dtype == ELT_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(row)[c + j])
                                       : __half2float(static_cast<const __half*>(row)[c + j]);
    }
}

__device__ __forceinline__ void store8(void* row, int dtype, bool vec, int c, int cols, const float (&v)[8]) {
    if (vec && c + 8 <= cols) {
        if (dtype == ELT_F32) {
            float4* p = reinterpret_cast<float4*>(static_cast<float*>(row) + c);
            p[0] = make_float4(v[0], v[1], v[2], v[3]);
            p[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (dtype == ELT_BF16) {
                    const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                    u[j] = *reinterpret_cast<const uint32_t*>(&t);
                } else {
                    const __half2 t = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
                    u[j] = *reinterpret_cast<const uint32_t*>(&t);
                }
            }
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(row) + c) = make_uint4(u[0], u[1], u[2], u[3]);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (c + j < cols) store_elt(row, c + j, v[j], dtype);
}

template <int FMT>
constexpr int block_lanes() { return mx_block(FMT) / 8; }  // lanes of a block, and of a scale word
template <int FMT>
constexpr int word_lanes() { return 4 * block_lanes<FMT>(); }

// Quantise the lane's eight elements (zeros behind the row's end) and write their codes and, from the
// first lane of each scale word, its four scales. All lanes of the warp take part; `store` false for
// lanes that have nothing to write.
template <int FMT>
__device__ __forceinline__ void quantize8(const float (&v)[8], int c, int64_t row, int cols, int64_t kt, uint8_t* data,
                                          int64_t ld, uint8_t* scales, float global, bool store) {
    constexpr int LB = block_lanes<FMT>();
    uint32_t a = __float_as_uint(absmax(absmax(absmax(absmax(0.f, v[0], v[1]), v[2], v[3]), v[4], v[5]), v[6], v[7]));
#pragma unroll
    for (int o = 1; o < LB; o *= 2) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
    const MxBlock b = mx_block_scale<FMT>(a, global);
    const int lane = threadIdx.x % 32;
    uint32_t word = b.code << (8 * (lane / LB % 4));
    word |= __shfl_xor_sync(0xffffffffu, word, LB);
    word |= __shfl_xor_sync(0xffffffffu, word, 2 * LB);
    if (!store) return;
    uint32_t w[FMT == MXF8 ? 2 : 1];
    mx_encode<FMT, 8>(v, b, w);
    const int64_t at = mx_bytes(FMT, c);
    if (at < mx_row_bytes(FMT, cols)) {
        uint8_t* d = data + row * ld + at;
        if constexpr (FMT == MXF8)
            *reinterpret_cast<uint2*>(d) = make_uint2(w[0], w[1]);
        else
            *reinterpret_cast<uint32_t*>(d) = w[0];
    }
    if (lane % word_lanes<FMT>() == 0)
        *reinterpret_cast<uint32_t*>(scales + mx_scale_word(row, c / (4 * mx_block(FMT)), kt)) = word;
}

// One scale word (128 elements, 64 for NVF4) per 16 (8) lanes; the rows up to the end of the last scale
// tile are walked too, for their zero scales.
template <int FMT>
__global__ void __launch_bounds__(256) quantize_kernel(const void* __restrict__ x, int dtype, int vec, int64_t ldx,
                                                       MxArray o, int kt, int64_t words) {
    constexpr int LW = word_lanes<FMT>();
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LW;
    const bool some = i < words;
    const int64_t row = some ? (words <= 0xffffffffll ? (int64_t)((uint32_t)i / (uint32_t)kt) : i / kt) : 0;
    const int kw = some ? (int)(i - row * kt) : 0;
    const int c = (kw * LW + threadIdx.x % LW) * 8;
    float v[8] = {};
    const bool live = some && row < o.rows;
    if (live) load8(static_cast<const uint8_t*>(x) + row * ldx * (dtype == ELT_F32 ? 4 : 2), dtype, vec, c, o.cols, v);
    const float g = FMT == NVF4 && o.global_scale ? *o.global_scale : 1.f;
    quantize8<FMT>(v, c, row, o.cols, kt, o.data, o.ld, o.scales, g, live);
    if (some && !live && threadIdx.x % LW == 0)
        *reinterpret_cast<uint32_t*>(o.scales + mx_scale_word(row, kw, kt)) = 0;
}

template <int FMT>
__global__ void __launch_bounds__(256) dequantize_kernel(MxArray x, int kt, int chunks, int64_t total, void* out,
                                                         int dtype, int vec, int64_t ldo) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t row = total <= 0xffffffffll ? (int64_t)((uint32_t)i / (uint32_t)chunks) : i / chunks;
    const int c = (int)(i - row * chunks) * 8;
    const float g = FMT == NVF4 && x.global_scale ? *x.global_scale : 1.f;
    const int b = c / mx_block(FMT);
    const float s = mx_scale_value<FMT>(x.scales[mx_scale_word(row, b / 4, kt) + b % 4]) * g;
    const uint8_t* d = x.data + row * x.ld + mx_bytes(FMT, c);
    uint32_t u[2];
    if (FMT == MXF8) {
        const uint2 q = *reinterpret_cast<const uint2*>(d);
        u[0] = q.x; u[1] = q.y;
    } else {
        u[0] = *reinterpret_cast<const uint32_t*>(d);
    }
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t code = FMT == MXF8 ? u[j / 2] >> (16 * (j % 2)) & 0xffffu : u[0] >> (8 * j) & 0xffu;
        const float2 f = mx_pair_values<FMT>(code);
        v[2 * j] = f.x * s;
        v[2 * j + 1] = f.y * s;
    }
    store8(static_cast<uint8_t*>(out) + row * ldo * (dtype == ELT_F32 ? 4 : 2), dtype, vec, c, x.cols, v);
}

struct NormArgs {
    const void* x;
    const void* residual;  // null: the stream is x
    void* residual_out;    // null: not written
    const float* gain;     // null: 1
    int dtype, res_type, vec, vec_r, vec_ro, vec_g;
    int64_t ldx, ldr, ldro;
    double eps;
    MxArray o;
    int kt;
    int64_t rows_padded;
};

// Adds v * v to sum + err, where err gathers the rounding errors: the square's by an FMA, the
// addition's by Knuth's two-sum. The _rn forms keep the compiler from contracting them.
__device__ __forceinline__ void add_square(float& sum, float& err, float v) {
    const float p = __fmul_rn(v, v), e = __fmaf_rn(v, v, -p);
    const float s = __fadd_rn(sum, p), t = __fsub_rn(s, sum);
    err = __fadd_rn(err, __fadd_rn(e, __fadd_rn(__fsub_rn(sum, __fsub_rn(s, t)), __fsub_rn(p, t))));
    sum = s;
}

// W warps per row, up to CH chunks of eight elements per thread, held in registers: each element is
// read once. The sum of squares keeps its rounding errors and ends in f64, so 1/rms is the rounded exact one but for rare ties and does not depend on
// how a row is spread over threads: next to the quantiser's borders its last bit decides.
template <int FMT, int W, int CH>
__global__ void __launch_bounds__(W > 8 ? 32 * W : 256) add_rms_norm_kernel(const __grid_constant__ NormArgs a) {
    constexpr int THREADS = W > 8 ? 32 * W : 256, ROWS = THREADS / (32 * W);
    __shared__ double part[THREADS / 32];
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / (32 * W);
    const int t = threadIdx.x % (32 * W), warp = threadIdx.x / 32;
    const bool live = row < a.o.rows;
    const int cols = a.o.cols;
    float v[CH][8];
    float sum = 0.f, err = 0.f;
    if (live) {
        const uint8_t* x = static_cast<const uint8_t*>(a.x) + row * a.ldx * (a.dtype == ELT_F32 ? 4 : 2);
        const uint8_t* r = static_cast<const uint8_t*>(a.residual) + row * a.ldr * (a.res_type == ELT_F32 ? 4 : 2);
        uint8_t* ro = static_cast<uint8_t*>(a.residual_out) + row * a.ldro * (a.res_type == ELT_F32 ? 4 : 2);
#pragma unroll
        for (int i = 0; i < CH; ++i) load8(x, a.dtype, a.vec, (t + i * 32 * W) * 8, cols, v[i]);
        if (a.residual) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const int c = (t + i * 32 * W) * 8;
                float u[8];
                load8(r, a.res_type, a.vec_r, c, cols, u);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[i][j] += u[j];
                    // The norm is that of the stream as it is held.
                    if (a.res_type == ELT_BF16) v[i][j] = __bfloat162float(__float2bfloat16_rn(v[i][j]));
                    if (a.res_type == ELT_F16) v[i][j] = __half2float(__float2half_rn(v[i][j]));
                }
            }
        }
        if (a.residual_out) {
#pragma unroll
            for (int i = 0; i < CH; ++i) store8(ro, a.res_type, a.vec_ro, (t + i * 32 * W) * 8, cols, v[i]);
        }
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) add_square(sum, err, v[i][j]);
    }
    double d = (double)sum + (double)err;
    if (live && !(sum > 1e-30f && sum < 1e37f)) {  // squares near f32's ends (and NaN): in f64
        d = 0.0;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) d = fma((double)v[i][j], (double)v[i][j], d);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (W > 1) {
        if (threadIdx.x % 32 == 0) part[warp] = d;
        __syncthreads();
        d = 0.0;
#pragma unroll
        for (int i = 0; i < W; ++i) d += part[warp / W * W + i];
    }
    const float inv = (float)(1.0 / sqrt(d / cols + a.eps));
    const float g = FMT == NVF4 && a.o.global_scale ? *a.o.global_scale : 1.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = (t + i * 32 * W) * 8;
        if (i > 0 && (c - 8 * (t % 32)) >= cols) break;  // the warp's chunk lies behind the row
        float u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = 1.f;
        if (a.gain) load8(a.gain, ELT_F32, a.vec_g, c, cols, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = live && c + j < cols ? v[i][j] * inv * u[j] : 0.f;
        const bool word = c / (4 * mx_block(FMT)) < a.kt;
        quantize8<FMT>(u, c, row, cols, a.kt, a.o.data, a.o.ld, a.o.scales, g, live && word);
        if (!live && word && row < a.rows_padded && t % word_lanes<FMT>() == 0)
            *reinterpret_cast<uint32_t*>(a.o.scales + mx_scale_word(row, c / (4 * mx_block(FMT)), a.kt)) = 0;
    }
}

bool rows_aligned(const void* p, int64_t ld, int dtype) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (int64_t)elt_size(dtype) % 16 == 0;
}

template <int FMT, int W, int CH>
int launch_norm(const NormArgs& a, cudaStream_t s) {
    constexpr int THREADS = W > 8 ? 32 * W : 256, ROWS = THREADS / (32 * W);
    const int64_t blocks = ceil_div(a.rows_padded, ROWS);
    if (blocks > 0x7fffffff) return fail(ANCHA_E_UNSUPPORTED, "add_rms_norm: too many rows");
    add_rms_norm_kernel<FMT, W, CH><<<(unsigned)blocks, THREADS, 0, s>>>(a);
    return check_launch("add_rms_norm");
}

template <int FMT>
int norm_by_width(const NormArgs& a, cudaStream_t s) {
    const int chunks = (int)ceil_div(a.o.cols, 8);
    if (chunks <= 64) return launch_norm<FMT, 1, 2>(a, s);
    if (chunks <= 128) return launch_norm<FMT, 1, 4>(a, s);
    if (chunks <= 512) return launch_norm<FMT, 4, 4>(a, s);
    if (chunks <= 1024) return launch_norm<FMT, 8, 4>(a, s);
    if (chunks <= 4096) return launch_norm<FMT, 32, 4>(a, s);
    return fail(ANCHA_E_UNSUPPORTED, "add_rms_norm: rows wider than 32768");
}

}  // namespace

int mx_quantize(const void* x, int dtype, int64_t ldx, const MxArray& o, cudaStream_t s) {
    const int kt = (int)mx_ktiles(o.format, o.cols), lw = o.format == NVF4 ? 8 : 16;
    const int64_t words = ceil_div(o.rows, 128) * 128 * kt, blocks = ceil_div(words * lw, 256);
    if (blocks > 0x7fffffff) return fail(ANCHA_E_UNSUPPORTED, "mx_quantize: too many elements for one launch");
    if (!blocks) return ANCHA_OK;
    const int vec = rows_aligned(x, ldx, dtype);
    const unsigned n = (unsigned)blocks;
    if (o.format == MXF8) quantize_kernel<MXF8><<<n, 256, 0, s>>>(x, dtype, vec, ldx, o, kt, words);
    else if (o.format == MXF4) quantize_kernel<MXF4><<<n, 256, 0, s>>>(x, dtype, vec, ldx, o, kt, words);
    else quantize_kernel<NVF4><<<n, 256, 0, s>>>(x, dtype, vec, ldx, o, kt, words);
    return check_launch("mx_quantize");
}

int mx_dequantize(const MxArray& x, void* out, int dtype, int64_t ldo, cudaStream_t s) {
    const int kt = (int)mx_ktiles(x.format, x.cols), chunks = (int)ceil_div(x.cols, 8);
    const int64_t total = x.rows * chunks, blocks = ceil_div(total, 256);
    if (blocks > 0x7fffffff) return fail(ANCHA_E_UNSUPPORTED, "mx_dequantize: too many elements for one launch");
    if (!blocks) return ANCHA_OK;
    const int vec = rows_aligned(out, ldo, dtype);
    const unsigned n = (unsigned)blocks;
    if (x.format == MXF8) dequantize_kernel<MXF8><<<n, 256, 0, s>>>(x, kt, chunks, total, out, dtype, vec, ldo);
    else if (x.format == MXF4) dequantize_kernel<MXF4><<<n, 256, 0, s>>>(x, kt, chunks, total, out, dtype, vec, ldo);
    else dequantize_kernel<NVF4><<<n, 256, 0, s>>>(x, kt, chunks, total, out, dtype, vec, ldo);
    return check_launch("mx_dequantize");
}

int mx_add_rms_norm(const void* x, int dtype, int64_t ldx, const void* residual, int res_type, int64_t ldr,
                    void* residual_out, int64_t ldro, const float* gain, double eps, const MxArray& o,
                    cudaStream_t s) {
    if (!o.rows) return ANCHA_OK;
    NormArgs a{};
    a.x = x; a.residual = residual; a.residual_out = residual_out; a.gain = gain;
    a.dtype = dtype; a.res_type = res_type;
    a.ldx = ldx; a.ldr = ldr; a.ldro = ldro;
    a.vec = rows_aligned(x, ldx, dtype);
    a.vec_r = residual && rows_aligned(residual, ldr, res_type);
    a.vec_ro = residual_out && rows_aligned(residual_out, ldro, res_type);
    a.vec_g = gain && reinterpret_cast<uintptr_t>(gain) % 16 == 0;
    a.eps = eps;
    a.o = o;
    a.kt = (int)mx_ktiles(o.format, o.cols);
    a.rows_padded = ceil_div(o.rows, 128) * 128;
    return o.format == MXF8 ? norm_by_width<MXF8>(a, s) : o.format == MXF4 ? norm_by_width<MXF4>(a, s)
                                                                           : norm_by_width<NVF4>(a, s);
}

}  // namespace ancha
