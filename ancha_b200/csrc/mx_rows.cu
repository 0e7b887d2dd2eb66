// Row kernels of the microscaled formats: quantisation, expansion, and the residual addition with
// RMS norm whose output is quantised. All are bound by HBM: each element is read once and written
// once. What costs next to it is instruction issue, so a thread owns sixteen consecutive elements of a row: a
// block of NVF4, half a block of the others (one shuffle for its maximum), whole 16-byte stores of 8-bit
// codes, and index arithmetic and scale shared by sixteen (against eight elements: 48060 x 1536 f16 -> mxf8 61 -> 41 us).
// Measured against HBM's 6549 GB/s: that 84 %, 16384 x 4096 mxf8 -> f32 96 %, norm of 48060 x 384 f32 46 us = 80 %,
// norm of 16384 x 4096 bf16 -> nvf4 95 us = 71 % (issue: its square sums, and two conversions an element).
#include "mx.cuh"

#include <algorithm>
#include <cfloat>

namespace ancha {
namespace {

constexpr int PER = 16;  // elements of a row per thread

struct Words8 {
    uint32_t w[8];
};

// Sixteen 16-bit elements and their values (the branch on the type is taken once for all).
__device__ __forceinline__ void unpack16(const Words8& q, int type, float (&v)[PER]) {
    if (type == ELT_BF16) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[2 * j] = __uint_as_float(q.w[j] << 16);
            v[2 * j + 1] = __uint_as_float(q.w[j] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&q.w[j]));
            v[2 * j] = f.x;
            v[2 * j + 1] = f.y;
        }
    }
}
__device__ __forceinline__ Words8 pack16(const float (&v)[PER], int type) {
    Words8 q;
    if (type == ELT_BF16) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            q.w[j] = *reinterpret_cast<const uint32_t*>(&t);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const __half2 t = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
            q.w[j] = *reinterpret_cast<const uint32_t*>(&t);
        }
    }
    return q;
}

__device__ __forceinline__ float element(const void* row, int dtype, int c) {
    return dtype == ELT_F32    ? static_cast<const float*>(row)[c]
           : dtype == ELT_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(row)[c])
                               : __half2float(static_cast<const __half*>(row)[c]);
}

// How a row's address allows it to be reached: an element at a time, in 16-byte or in 32-byte pieces.
enum : int { BY_ELEMENT = 0, BY_16 = 1, BY_32 = 2 };

__device__ __forceinline__ Words8 ld32(const void* p, int access) {
    Words8 q;
    if (access == BY_32) {
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(q.w[0]), "=r"(q.w[1]), "=r"(q.w[2]), "=r"(q.w[3]), "=r"(q.w[4]), "=r"(q.w[5]), "=r"(q.w[6]),
                       "=r"(q.w[7])
                     : "l"(p)
                     : "memory");
    } else {
        const uint4 a = static_cast<const uint4*>(p)[0], b = static_cast<const uint4*>(p)[1];
        q = {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
    }
    return q;
}
__device__ __forceinline__ void st32(void* p, int access, const Words8& q) {
    if (access == BY_32) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(q.w[0]), "r"(q.w[1]), "r"(q.w[2]),
                     "r"(q.w[3]), "r"(q.w[4]), "r"(q.w[5]), "r"(q.w[6]), "r"(q.w[7])
                     : "memory");
    } else {
        static_cast<uint4*>(p)[0] = make_uint4(q.w[0], q.w[1], q.w[2], q.w[3]);
        static_cast<uint4*>(p)[1] = make_uint4(q.w[4], q.w[5], q.w[6], q.w[7]);
    }
}

// Slot of element e (0 .. 511) of a warp's exchange buffer: lanes reading sixteen consecutive ones and lanes reading
// neighbours both meet 32 banks.
constexpr int EXCHANGE = 512 + 32;
__device__ __forceinline__ int slot(int e) { return e + (e >> 4); }

// Sixteen elements of a row from column c (a multiple of 16) for every lane, zeros from column `cols` on (cols 0: a lane
// without a row). GROUP neighbouring lanes hold neighbouring chunks of one row; where its address allows no vector loads
// they read neighbouring elements together (fetch16) and then exchange them through `buf`, a warp's (settle16, which all
// its lanes call): several chunks can be on their way before the first exchange waits for its own.
template <int GROUP>
__device__ __forceinline__ void fetch16(const void* row, int dtype, int access, int c, int cols, float (&v)[PER]) {
    if (access != BY_ELEMENT) {
        if (c + PER <= cols) {
            if (dtype == ELT_F32) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const Words8 q = ld32(static_cast<const float*>(row) + c + 8 * h, access);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[8 * h + j] = __uint_as_float(q.w[j]);
                }
            } else {
                unpack16(ld32(static_cast<const uint16_t*>(row) + c, access), dtype, v);
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = 0.f;
        if (c < cols) {  // the row's last, shorter chunk
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (c + j < cols) v[j] = element(row, dtype, c + j);
        }
        return;
    }
    const int sub = threadIdx.x % GROUP, first = c - sub * PER + sub;
#pragma unroll
    for (int k = 0; k < PER; ++k) v[k] = first + k * GROUP < cols ? element(row, dtype, first + k * GROUP) : 0.f;
}
template <int GROUP>
__device__ __forceinline__ void settle16(int access, float* buf, float (&v)[PER]) {
    if (access != BY_ELEMENT) return;
    const int lane = threadIdx.x % 32, sub = lane % GROUP, base = (lane - sub) * PER + sub;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < PER; ++k) buf[slot(base + k * GROUP)] = v[k];
    __syncwarp();
#pragma unroll
    for (int j = 0; j < PER; ++j) v[j] = buf[slot(lane * PER + j)];
}

// The way back; columns from `cols` on are not written.
template <int GROUP>
__device__ __forceinline__ void store16(void* row, int dtype, int access, int c, int cols, float* buf, const float (&v)[PER]) {
    if (access != BY_ELEMENT) {
        if (c + PER <= cols) {
            Words8 q;
            if (dtype == ELT_F32) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) q.w[j] = __float_as_uint(v[8 * h + j]);
                    st32(static_cast<float*>(row) + c + 8 * h, access, q);
                }
            } else {
                st32(static_cast<uint16_t*>(row) + c, access, pack16(v, dtype));
            }
            return;
        }
        if (c < cols) {
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (c + j < cols) store_elt(row, c + j, v[j], dtype);
        }
        return;
    }
    const int lane = threadIdx.x % 32, sub = lane % GROUP, base = (lane - sub) * PER;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < PER; ++j) buf[slot(lane * PER + j)] = v[j];
    __syncwarp();
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int col = c - sub * PER + k * GROUP + sub;
        if (col < cols) store_elt(row, col, buf[slot(base + k * GROUP + sub)], dtype);
    }
}

// n / d for n < 2^31 by a multiplication (d >= 1; Granlund and Montgomery's round-up method).
struct FastDiv {
    uint32_t d, mul, shift;
};
FastDiv fast_div(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    return {d, (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
}
__device__ __forceinline__ uint32_t divide(uint32_t n, const FastDiv& f) {
    return (__umulhi(n, f.mul) + n) >> f.shift;
}

template <int FMT>
constexpr int block_lanes() { return mx_block(FMT) / PER; }  // lanes of a block, and of a scale word
template <int FMT>
constexpr int word_lanes() { return 4 * block_lanes<FMT>(); }

// Quantise the lane's sixteen elements (zeros behind the row's end) and write their codes and, from the
// first lane of each scale word, its four scales. All lanes of the warp take part; `store` false for
// lanes that have nothing to write.
template <int FMT>
__device__ __forceinline__ void quantize16(const float (&v)[PER], int c, int64_t row, int cols, int64_t kt, uint8_t* data,
                                           int64_t ld, uint8_t* scales, float global, bool store) {
    constexpr int LB = block_lanes<FMT>();
    float a = 0.f;
#pragma unroll
    for (int j = 0; j < PER; j += 2) a = absmax(a, v[j], v[j + 1]);
    uint32_t bits = __float_as_uint(a);
    if (LB == 2) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
    const MxBlock b = mx_block_scale<FMT>(bits, global);
    const int lane = threadIdx.x % 32;
    uint32_t word = b.code << (8 * (lane / LB % 4));
    word |= __shfl_xor_sync(0xffffffffu, word, LB);
    word |= __shfl_xor_sync(0xffffffffu, word, 2 * LB);
    if (!store) return;
    uint32_t w[FMT == MXF8 ? 4 : 2];
    mx_encode<FMT, PER>(v, b, w);
    const int64_t at = mx_bytes(FMT, c);
    if (at < mx_row_bytes(FMT, cols)) {
        uint8_t* d = data + row * ld + at;
        if constexpr (FMT == MXF8)
            *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
        else
            *reinterpret_cast<uint2*>(d) = make_uint2(w[0], w[1]);
    }
    if (lane % word_lanes<FMT>() == 0)
        *reinterpret_cast<uint32_t*>(scales + mx_scale_word(row, c / (4 * mx_block(FMT)), kt)) = word;
}

// One scale word (128 elements, 64 for NVF4) per eight (four) lanes; the rows up to the end of the last scale
// tile are walked too, for their zero scales. row0: the launch's first row.
template <int FMT>
__global__ void __launch_bounds__(256) quantize_kernel(const void* __restrict__ x, int dtype, int access, int64_t ldx,
                                                       const __grid_constant__ MxArray o, FastDiv kt, uint32_t words, int64_t row0) {
    constexpr int LW = word_lanes<FMT>();
    const uint32_t i = (uint32_t)(((uint64_t)blockIdx.x * 256 + threadIdx.x) / LW);
    const bool some = i < words;
    const uint32_t r = divide(i, kt);
    const int kw = (int)(i - r * kt.d), c = (kw * LW + threadIdx.x % LW) * PER;
    const int64_t row = row0 + r;
    __shared__ float exchange[8][EXCHANGE];
    float v[PER];
    const bool live = some && row < o.rows;
    fetch16<LW>(static_cast<const uint8_t*>(x) + row * ldx * (dtype == ELT_F32 ? 4 : 2), dtype, access, c, live ? o.cols : 0, v);
    settle16<LW>(access, exchange[threadIdx.x / 32], v);
    const float g = FMT == NVF4 && o.global_scale ? *o.global_scale : 1.f;
    quantize16<FMT>(v, c, row, o.cols, kt.d, o.data, o.ld, o.scales, g, live);
    if (some && !live && threadIdx.x % LW == 0)
        *reinterpret_cast<uint32_t*>(o.scales + mx_scale_word(row, kw, kt.d)) = 0;
}

// Sixteen elements per thread, eight neighbouring threads in one row (`groups`: eights of chunks of a row).
constexpr int DEQ_GROUP = 8;
template <int FMT>
__global__ void __launch_bounds__(256) dequantize_kernel(const __grid_constant__ MxArray x, int kt, FastDiv groups, uint32_t total,
                                                         void* out, int dtype, int access, int64_t ldo, int64_t row0) {
    __shared__ float exchange[8][EXCHANGE];
    const uint32_t i = (uint32_t)(((uint64_t)blockIdx.x * 256 + threadIdx.x) / DEQ_GROUP);
    const uint32_t r = divide(i, groups);
    const int64_t row = row0 + r;
    const int c = ((int)(i - r * groups.d) * DEQ_GROUP + threadIdx.x % DEQ_GROUP) * PER;
    const bool live = i < total && c < x.cols;
    float v[PER] = {};
    if (live) {
        const float g = FMT == NVF4 && x.global_scale ? *x.global_scale : 1.f;
        const int b = c / mx_block(FMT);
        const uint32_t code = x.scales[mx_scale_word(row, b / 4, kt) + b % 4];
        const uint8_t* d = x.data + row * x.ld + mx_bytes(FMT, c);
        uint32_t u[FMT == MXF8 ? 4 : 2];
        if constexpr (FMT == MXF8) {
            const uint4 q = *reinterpret_cast<const uint4*>(d);
            u[0] = q.x; u[1] = q.y; u[2] = q.z; u[3] = q.w;
        } else {
            const uint2 q = *reinterpret_cast<const uint2*>(d);
            u[0] = q.x; u[1] = q.y;
        }
        const float s = mx_scale_value<FMT>(code) * g;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t pair = FMT == MXF8 ? u[j / 2] >> (16 * (j % 2)) & 0xffffu : u[j / 4] >> (8 * (j % 4)) & 0xffu;
            const float2 f = mx_pair_values<FMT>(pair);
            v[2 * j] = f.x * s;
            v[2 * j + 1] = f.y * s;
        }
    }
    store16<DEQ_GROUP>(static_cast<uint8_t*>(out) + row * ldo * (dtype == ELT_F32 ? 4 : 2), dtype, access, c, i < total ? x.cols : 0,
                       exchange[threadIdx.x / 32], v);
}

struct NormArgs {
    const void* x;
    const void* residual;  // null: the stream is x
    void* residual_out;    // null: not written
    const float* gain;     // null: 1
    int dtype, res_type, access, access_r, access_ro, access_g;
    int64_t ldx, ldr, ldro;
    double eps, inv_cols;  // inv_cols: 1 / cols
    MxArray o;
    int kt;
    int64_t rows_padded;
};

// Adds the squares of a pair (two sums, one per half) with the rounding errors gathered in err: the squares' by
// an FMA, the additions' by Knuth's two-sum, on packed pairs (their _rn forms are not contracted).
__device__ __forceinline__ void add_squares(uint64_t& sum, uint64_t& err, uint64_t v) {
    const uint64_t zero = 0, p = fmul2(v, v), minus_p = fsub2(zero, p), e = ffma2(v, v, minus_p);
    const uint64_t s = fadd2(sum, p), t = fsub2(s, sum);
    err = fadd2(err, fadd2(e, fadd2(fsub2(sum, fsub2(s, t)), fsub2(p, t))));
    sum = s;
}

// 1 / sqrt(x) in f64, rounded to f32: the f32 estimate (2 ulp) and one Newton step in f64, which squares its error.
// The result leaves f32's normal numbers for rows of subnormal numbers (up to 1e47) or of the largest ones (down to
// 3e-39), and for rows of zeros, where it is 1 / sqrt(eps), whatever that is. Towards these ends a power of two of it,
// `pre`, is left to the row's elements, which take it exactly, and what is still too large (zeros) is f32's largest number.
__device__ __forceinline__ float inverse_root(double x, float& pre) {
    pre = 1.f;
    if (!(x > 1e-30 && x < 1e30)) {
        pre = x < 1.0 ? 0x1p64f : 0x1p-24f;
        const double r = 1.0 / (sqrt(x) * pre);
        return r > FLT_MAX ? FLT_MAX : (float)r;  // NaN stays
    }
    const double r = rsqrtf((float)x);
    return (float)fma(0.5 * r, fma(-x * r, r, 1.0), r);
}

// W warps per row, up to CH chunks of sixteen elements per thread, held in registers: each element is
// read once. The sum of squares keeps its rounding errors and ends in f64, so 1/rms is the rounded exact one but
// for rare ties and does not depend on how a row is spread over threads: next to the quantiser's borders its last
// bit decides.
// The bounds on registers are the measured best: 64 for one warp to a row (48 spills: 47 us for 48060 x 384, 60 us
// with no bound, 46 us so), 40 for eight (16384 x 4096 95 us, 101 us with 48).
template <int FMT, int W, int CH>
__global__ void __launch_bounds__(W > 8 ? 32 * W : 256, W > 8 ? 1 : W == 8 ? 6 : W == 1 ? 4 : 5)
add_rms_norm_kernel(const __grid_constant__ NormArgs a) {
    constexpr int THREADS = W > 8 ? 32 * W : 256, ROWS = THREADS / (32 * W);
    __shared__ double part[THREADS / 32];
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / (32 * W);
    const int t = threadIdx.x % (32 * W), warp = threadIdx.x / 32;
    const bool live = row < a.o.rows;
    const int cols = a.o.cols;
    __shared__ float exchange[THREADS / 32][EXCHANGE];
    float* buf = exchange[warp];
    float v[CH][PER];
    float sum = 0.f, err = 0.f;
    {
        const int n = live ? cols : 0;
        const uint8_t* x = static_cast<const uint8_t*>(a.x) + row * a.ldx * (a.dtype == ELT_F32 ? 4 : 2);
        const uint8_t* r = static_cast<const uint8_t*>(a.residual) + row * a.ldr * (a.res_type == ELT_F32 ? 4 : 2);
        uint8_t* ro = static_cast<uint8_t*>(a.residual_out) + row * a.ldro * (a.res_type == ELT_F32 ? 4 : 2);
#pragma unroll
        for (int i = 0; i < CH; ++i) fetch16<32>(x, a.dtype, a.access, (t + i * 32 * W) * PER, n, v[i]);
        if (a.residual) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                float u[PER];
                fetch16<32>(r, a.res_type, a.access_r, (t + i * 32 * W) * PER, n, u);
                settle16<32>(a.access, buf, v[i]);
                settle16<32>(a.access_r, buf, u);
#pragma unroll
                for (int j = 0; j < PER; j += 2)
                    f2_split(fadd2(f2(v[i][j], v[i][j + 1]), f2(u[j], u[j + 1])), v[i][j], v[i][j + 1]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < CH; ++i) settle16<32>(a.access, buf, v[i]);
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int c = (t + i * 32 * W) * PER;
            if (a.res_type != ELT_F32 && a.residual) {
                // The norm is that of the stream as it is held.
                const Words8 q = pack16(v[i], a.res_type);
                unpack16(q, a.res_type, v[i]);
                if (a.access_ro != BY_ELEMENT && c + PER <= n) {
                    st32(reinterpret_cast<uint16_t*>(ro) + c, a.access_ro, q);
                    continue;
                }
            }
            if (a.residual_out) store16<32>(ro, a.res_type, a.access_ro, c, n, buf, v[i]);
        }
        uint64_t s2 = 0, e2 = 0;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < PER; j += 2) add_squares(s2, e2, f2(v[i][j], v[i][j + 1]));
        float s1, e1;
        f2_split(s2, sum, s1);
        f2_split(e2, err, e1);
        const float s = __fadd_rn(sum, s1), q = __fsub_rn(s, sum);
        err = __fadd_rn(__fadd_rn(err, e1), __fadd_rn(__fsub_rn(sum, __fsub_rn(s, q)), __fsub_rn(s1, q)));
        sum = s;
    }
    double d = (double)sum + (double)err;
    if (live && t * PER < cols && !(sum > 1e-30f && sum < 1e37f)) {  // squares near f32's ends (and NaN): in f64
        d = 0.0;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < PER; ++j) d = fma((double)v[i][j], (double)v[i][j], d);
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
    float pre;
    const float inv = inverse_root(d * a.inv_cols + a.eps, pre);
    if (pre != 1.f) {  // the same for all of a row's threads
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < PER; ++j) v[i][j] *= pre;
    }
    const float g = FMT == NVF4 && a.o.global_scale ? *a.o.global_scale : 1.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = (t + i * 32 * W) * PER;
        if (c - PER * (t % 32) >= cols) break;  // the warp's chunk lies behind the row
        float u[PER];
        if (a.gain) {
            fetch16<32>(a.gain, ELT_F32, a.access_g, c, cols, u);
            settle16<32>(a.access_g, buf, u);
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j) u[j] = 1.f;
        }
#pragma unroll
        for (int j = 0; j < PER; j += 2)
            f2_split(fmul2(fmul2(f2(v[i][j], v[i][j + 1]), f2(inv, inv)), f2(u[j], u[j + 1])), u[j], u[j + 1]);
        if (!live || c + PER > cols) {
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (!live || c + j >= cols) u[j] = 0.f;
        }
        const bool word = c / (4 * mx_block(FMT)) < a.kt;
        quantize16<FMT>(u, c, row, cols, a.kt, a.o.data, a.o.ld, a.o.scales, g, live && word);
        if (!live && word && row < a.rows_padded && t % word_lanes<FMT>() == 0)
            *reinterpret_cast<uint32_t*>(a.o.scales + mx_scale_word(row, c / (4 * mx_block(FMT)), a.kt)) = 0;
    }
}

int row_access(const void* p, int64_t ld, int dtype) {
    const uint64_t bits = reinterpret_cast<uintptr_t>(p) | (uint64_t)(ld * (int64_t)elt_size(dtype));
    return bits % 32 == 0 ? BY_32 : bits % 16 == 0 ? BY_16 : BY_ELEMENT;
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
    const int chunks = (int)ceil_div(a.o.cols, PER);
    if (chunks <= 32) return launch_norm<FMT, 1, 1>(a, s);
    if (chunks <= 64) return launch_norm<FMT, 2, 1>(a, s);
    if (chunks <= 128) return launch_norm<FMT, 4, 1>(a, s);
    if (chunks <= 256) return launch_norm<FMT, 8, 1>(a, s);
    if (chunks <= 512) return launch_norm<FMT, 16, 1>(a, s);
    if (chunks <= 2048) return launch_norm<FMT, 16, 4>(a, s);
    return fail(ANCHA_E_UNSUPPORTED, "add_rms_norm: rows wider than 32768");
}

}  // namespace

// Launches cover at most 2^30 scale words or chunks, so that their indices stay in 31 bits: arrays above that take several.
constexpr int64_t kLaunchItems = int64_t(1) << 30;

int mx_quantize(const void* x, int dtype, int64_t ldx, const MxArray& o, cudaStream_t s) {
    const int64_t kt = mx_ktiles(o.format, o.cols), rows = ceil_div(o.rows, 128) * 128;
    const int lw = o.format == NVF4 ? word_lanes<NVF4>() : word_lanes<MXF8>(), access = row_access(x, ldx, dtype);
    const FastDiv div = fast_div((uint32_t)kt);
    const int64_t step = std::max<int64_t>(1, kLaunchItems / kt);
    for (int64_t r = 0; r < rows; r += step) {
        const uint32_t words = (uint32_t)(std::min(step, rows - r) * kt);
        const unsigned n = (unsigned)ceil_div((int64_t)words * lw, 256);
        if (o.format == MXF8) quantize_kernel<MXF8><<<n, 256, 0, s>>>(x, dtype, access, ldx, o, div, words, r);
        else if (o.format == MXF4) quantize_kernel<MXF4><<<n, 256, 0, s>>>(x, dtype, access, ldx, o, div, words, r);
        else quantize_kernel<NVF4><<<n, 256, 0, s>>>(x, dtype, access, ldx, o, div, words, r);
        ANCHA_TRY(check_launch("mx_quantize"));
    }
    return ANCHA_OK;
}

int mx_dequantize(const MxArray& x, void* out, int dtype, int64_t ldo, cudaStream_t s) {
    const int kt = (int)mx_ktiles(x.format, x.cols), access = row_access(out, ldo, dtype);
    const int64_t groups = ceil_div(x.cols, PER * DEQ_GROUP);
    const FastDiv div = fast_div((uint32_t)groups);
    const int64_t step = std::max<int64_t>(1, kLaunchItems / groups);
    for (int64_t r = 0; r < x.rows; r += step) {
        const uint32_t total = (uint32_t)(std::min(step, x.rows - r) * groups);
        const unsigned n = (unsigned)ceil_div((int64_t)total * DEQ_GROUP, 256);
        if (x.format == MXF8) dequantize_kernel<MXF8><<<n, 256, 0, s>>>(x, kt, div, total, out, dtype, access, ldo, r);
        else if (x.format == MXF4) dequantize_kernel<MXF4><<<n, 256, 0, s>>>(x, kt, div, total, out, dtype, access, ldo, r);
        else dequantize_kernel<NVF4><<<n, 256, 0, s>>>(x, kt, div, total, out, dtype, access, ldo, r);
        ANCHA_TRY(check_launch("mx_dequantize"));
    }
    return ANCHA_OK;
}

int mx_add_rms_norm(const void* x, int dtype, int64_t ldx, const void* residual, int res_type, int64_t ldr,
                    void* residual_out, int64_t ldro, const float* gain, double eps, const MxArray& o,
                    cudaStream_t s) {
    if (!o.rows) return ANCHA_OK;
    NormArgs a{};
    a.x = x; a.residual = residual; a.residual_out = residual_out; a.gain = gain;
    a.dtype = dtype; a.res_type = res_type;
    a.ldx = ldx; a.ldr = ldr; a.ldro = ldro;
    a.access = row_access(x, ldx, dtype);
    if (residual) a.access_r = row_access(residual, ldr, res_type);
    if (residual_out) a.access_ro = row_access(residual_out, ldro, res_type);
    a.access_g = row_access(gain, 0, ELT_F32);
    a.inv_cols = 1.0 / o.cols;
    a.eps = eps;
    a.o = o;
    a.kt = (int)mx_ktiles(o.format, o.cols);
    a.rows_padded = ceil_div(o.rows, 128) * 128;
    return o.format == MXF8 ? norm_by_width<MXF8>(a, s) : o.format == MXF4 ? norm_by_width<MXF4>(a, s)
                                                                           : norm_by_width<NVF4>(a, s);
}

}  // namespace ancha
