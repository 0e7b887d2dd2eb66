// Product of two microscaled arrays on the block-scaled tensor cores: y = act(x · wᵀ · g + bias) +
// residual, x [m, k], w [n, k], f32 accumulation, y in 32 or 16 bits or quantised again.
//
// The scales need no arithmetic here: tcgen05.mma (kind mxf8f6f4 / mxf4 / mxf4nvf4, block_scale) takes a
// 32-byte K step of both operands from shared memory and their block scales from TMEM, where tcgen05.cp
// puts them 512 bytes (128 rows by 4 blocks) at a time; the stored order of the scales is the order that
// copy wants. One K slab is 128 bytes of a row in every format (128 elements of 8 bits, 256 of 4), four
// instructions; it needs 1 (mxf8), 2 (mxf4) or 4 (nvf4) scale tiles per 128 rows.
//
// Persistent and warp-specialised, as the 16-bit GEMM: warp 0 loads slabs of both operands and their scales by TMA
// through a ring of stages, warp 1 issues the copies and products, the other warps drain the accumulator (32 rows by 64
// columns each). A CTA pair shares a tile of 256 rows by 192 or 256 columns (each CTA holds 128 rows of x, half of w's rows,
// and all of w's scales). Few rows, or few tiles with long K, take the split kernel at the end.
//
// Measured (one B200): 8192^3 nvf4 229 us = 4.8 PFLOP/s, mxf4 199 us = 5.5, mxf8 432 us = 2.5 under the power cap. A K slab of a
// pair takes 0.45 to 0.52 us in every format and at both widths, so neither its products (384 or 512 cycles) nor its 3, 6 or
// 12 scale copies set that alone. 48060 x 1536 x 384 mxf8 with GELU into mxf8 74 us (43 us without GELU): the epilogue warps wait for
// their own latencies, with half of the issue slots and 40 % of the FMA pipe in use; 1 x 4096 x 4096 mxf4 7 us, latency.
#include "mx.cuh"
#include "tc.cuh"

#include <algorithm>
#include <cfloat>

namespace ancha {
namespace {

constexpr int BM = 128, SLAB = 128;          // rows of a CTA's tile, bytes of a K slab
constexpr int OPERAND_BYTES = BM * SLAB;     // 128 rows of a slab
constexpr int SF_TILE = 512;                 // a scale tile
constexpr int STAGING = 4096;                // per epilogue warp: 32 rows x 128 bytes
constexpr int BIAS_BYTES = 256;              // and the bias of its 64 columns
// TMEM: one accumulator or two, then the scales of the slab in work.
constexpr uint32_t SFA_COL = 448, SFB_COL = 464, TMEM_COLS = 512;

constexpr int sf_tiles(int fmt) { return fmt == MXF8 ? 1 : fmt == MXF4 ? 2 : 4; }

template <int FMT, int BN, bool PAIR>
struct Shape {
    static constexpr int SF = sf_tiles(FMT);
    static constexpr int B_ROWS = PAIR ? BN / 2 : BN;   // w's rows in this CTA
    static constexpr int B_BYTES = B_ROWS * SLAB;
    static constexpr int RANGES = (BN + 127) / 128;     // 128-row ranges of w's scales
    static constexpr int SFA_BYTES = SF * SF_TILE, SFB_BYTES = SF * SF_TILE * RANGES;
    static constexpr int STAGE = OPERAND_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES;
    static constexpr int EPI = BN / 16;                 // epilogue warps: 32 rows by 64 columns of the tile each
    static constexpr int THREADS = 64 + 32 * EPI;
    // Stages and bytes of shared memory; with a residual each epilogue warp has a second buffer.
    static constexpr int FIXED = 1024 + 512 + EPI * (STAGING + BIAS_BYTES);
    static constexpr int stages(bool residual) {
        const int fit = (227 * 1024 - FIXED - (residual ? EPI * STAGING : 0)) / STAGE;
        return fit < 6 ? fit : 6;
    }
    static constexpr int bytes(bool residual) {
        return FIXED + (residual ? EPI * STAGING : 0) + stages(residual) * STAGE;
    }
    static_assert(stages(true) >= 2, "shared memory");
    // Accumulators, used in turn. Two of 256 columns and the scales do not fit TMEM's 512: with one, a tile's products
    // start when every epilogue warp has read the tile before into registers.
    static constexpr int ACCS = BN == 256 ? 1 : 2;
};

struct Params {
    int m, n, kbytes;          // kbytes: bytes of a row of x or w that hold elements
    int m_tiles, n_tiles, tiles;
    const float* gx;           // array scales (NVF4) or null
    const float* gw;
    const float* bias;
    const void* residual;
    int64_t ldr;
    int res_type, res_mode, act;  // res_mode: RES_*
    void* out;
    int64_t ldo;
    int out_type, out_mode;    // OUT_*
    MxArray om;
    int okt;                   // scale tiles along a row of om
    int oblock_log2;           // its block
    int rows_padded;           // m rounded to whole scale tiles
    int stages;
    int* err;
};
enum : int { RES_NONE = 0, RES_ELEMENT = 1, RES_TMA = 2 };  // RES_TMA: 16-byte aligned rows
enum : int { OUT_TMA = 0, OUT_PLAIN = 1, OUT_MX = 2 };

// ---- block-scaled tcgen05 -------------------------------------------------------------------

// Scale-tile descriptor: 32 rows of 16 bytes, no swizzle, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t sf_desc(uint32_t smem_addr) {
    return (uint64_t)((smem_addr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}

// A scale tile into four TMEM columns, the same 32 lanes for each of the four lane quarters.
template <bool PAIR>
__device__ __forceinline__ void sf_copy(uint32_t tmem, uint64_t desc) {
    if (PAIR)
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

#define ANCHA_MX_MMA(GROUP, KIND)                                                                       \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                      \
                 "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" \
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)              \
                 : "memory")

template <int FMT, bool PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                    uint32_t accumulate) {
    if (PAIR) {
        if (FMT == MXF8) ANCHA_MX_MMA("2", "mxf8f6f4.block_scale.scale_vec::1X");
        else if (FMT == MXF4) ANCHA_MX_MMA("2", "mxf4.block_scale.scale_vec::2X");
        else ANCHA_MX_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
    } else {
        if (FMT == MXF8) ANCHA_MX_MMA("1", "mxf8f6f4.block_scale.scale_vec::1X");
        else if (FMT == MXF4) ANCHA_MX_MMA("1", "mxf4.block_scale.scale_vec::2X");
        else ANCHA_MX_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
    }
}
#undef ANCHA_MX_MMA

// Instruction descriptor without the scale byte selectors: element types (E4M3 is 0 of mxf8f6f4, E2M1 is 1 of
// mxf4 / mxf4nvf4), N / 8 at bit 17, scale type E8M0 at bit 23, M / 128 at bit 27, both operands K-major.
template <int FMT>
__host__ __device__ constexpr uint32_t idesc_of(int m, int n) {
    return (FMT == MXF8 ? 0u : 1u << 7 | 1u << 10) | (uint32_t)(n >> 3) << 17 | (FMT == NVF4 ? 0u : 1u << 23) |
           (uint32_t)(m >> 7) << 27;
}

// The products of one slab: `steps` (1 to 4) K steps of 32 bytes. Step i takes scale tile i / (4 / SF) and in
// it the byte (1X), byte pair (2X) or all four bytes (4X) of its blocks. sfa, sfb: TMEM columns of the scales
// (4 SF, and 4 SF for each 128 columns of the tile or part of them); sfb_skip: columns of the latter before the
// tile's first.
template <int FMT, bool PAIR, int BN>
__device__ __forceinline__ void slab_products(uint32_t acc, uint32_t sfa, uint32_t sfb, uint32_t a, uint32_t b, uint32_t sa,
                                              uint32_t sb, uint32_t idesc, int steps, bool first, uint32_t sfb_skip = 0) {
    constexpr int SF = sf_tiles(FMT), PER = 4 / SF;  // K steps per scale tile
    constexpr int RANGES = (BN + 127) / 128;  // 128-row ranges of w's scales
#pragma unroll
    for (int t = 0; t < SF; ++t) {
        if (t * PER >= steps) break;
        sf_copy<PAIR>(sfa + 4 * t, sf_desc(sa + t * SF_TILE));
#pragma unroll
        for (int q = 0; q < RANGES; ++q)
            sf_copy<PAIR>(sfb + 4 * (t * RANGES + q), sf_desc(sb + (q * SF + t) * SF_TILE));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i >= steps) break;
        const int t = i / PER;
        const uint32_t id = FMT == MXF8 ? i : FMT == MXF4 ? i % 2 * 2 : 0;
        mma<FMT, PAIR>(acc, umma_desc_sw128(a + i * 32), umma_desc_sw128(b + i * 32), idesc | id << 4 | id << 29,
                       sfa + 4 * t, sfb + 4 * t * RANGES + sfb_skip, !(first && i == 0));
    }
}

// ---- epilogue -------------------------------------------------------------------------------

// GELU(x) = max(x, 0) - u Phi(-u) with u = min(|x|, 13), Phi(-u) = 2^R(u), R a polynomial of degree 9 fitted here to
// log2 Phi(-u) with the weight that its error has in the result, u Phi(-u), but 1.3e-5 at least (linear programming): the
// fit is off by 8e-8 at most and, so that a block of very negative sums keeps its scale and codes, by 8e-4 of what is left of
// them down to -5.5 and 6e-3 beyond. From -13 on that is below f32's normal numbers and the exponential 0. Evaluated in f32:
// rms 6.5e-8 on [-4, 4], 1.1e-7 beyond f32's own rounding at most. (A clamp at 5.5 and degree 7: rms 5.3e-8, but -1.04e-7
// for every x below -5.5; 48060 x 1536 x 384 mxf8 -> mxf8 73 us with it, 74 us so. Degree 10: 77 us.) NaN stays NaN.
// The coefficients lie in constant memory as pairs: as immediates each would cost the packed FMA two moves.
__constant__ float2 kGelu[10] = {{-0.9999902248382568f, -0.9999902248382568f}, {-1.1512339115142822f, -1.1512339115142822f},
                                 {-0.45865750312805176f, -0.45865750312805176f}, {-0.05358625948429108f, -0.05358625948429108f},
                                 {0.008208729326725006f, 0.008208729326725006f}, {-0.0008120433194562793f, -0.0008120433194562793f},
                                 {3.687796197482385e-05f, 3.687796197482385e-05f}, {9.592198466634727e-07f, 9.592198466634727e-07f},
                                 {-1.7287898401718849e-07f, -1.7287898401718849e-07f}, {5.107358092004688e-09f, 5.107358092004688e-09f}};
__device__ __forceinline__ void gelu2(float& x0, float& x1) {
    const uint64_t* c = reinterpret_cast<const uint64_t*>(kGelu);
    float u0, u1;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(u0) : "f"(fabsf(x0)), "f"(13.0f));
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(u1) : "f"(fabsf(x1)), "f"(13.0f));
    const uint64_t u = f2(u0, u1);
    uint64_t r = c[9];
#pragma unroll
    for (int i = 8; i >= 0; --i) r = ffma2(r, u, c[i]);
    float r0, r1;
    f2_split(r, r0, r1);
    x0 = fmaf(-u0, ex2_approx(r0), fmaxf(x0, 0.f));
    x1 = fmaf(-u1, ex2_approx(r1), fmaxf(x1, 0.f));
}

// tanh(x) with a relative error below 1e-6 everywhere, since an output with block scales keeps small numbers' relative
// precision: 1 - 2 / (e^2x + 1) from |x| = 0.5 on (its error of up to 4e-7 is absolute: at 1e-6 it would be a sixth of the
// result), below it x + x^3 P(x^2), P of degree 3 fitted here to the least relative error (linear programming; 8e-8 in
// f32's steps). 48060 x 1536 x 384 mxf8 -> bf16: 72 us, 63 us without the polynomial.
__constant__ float2 kTanh[4] = {{-0.333331435918808f, -0.333331435918808f}, {0.13325878977775574f, 0.13325878977775574f},
                                {-0.05304549261927605f, -0.05304549261927605f}, {0.01724149100482464f, 0.01724149100482464f}};
__device__ __forceinline__ void tanh2(float& x0, float& x1) {
    const uint64_t* c = reinterpret_cast<const uint64_t*>(kTanh);
    const uint64_t x = f2(x0, x1), z = fmul2(x, x);
    uint64_t r = c[3];
#pragma unroll
    for (int i = 2; i >= 0; --i) r = ffma2(r, z, c[i]);
    float s0, s1, t0 = x0, t1 = x1;
    f2_split(ffma2(fmul2(x, z), r, x), s0, s1);
    tanh_fast2(t0, t1);
    x0 = fabsf(x0) < 0.5f ? s0 : t0;
    x1 = fabsf(x1) < 0.5f ? s1 : t1;
}

__device__ void add_plain(const Params& p, float* buf, int64_t row0, int c0, int nv, int lane, float (&v)[32]);

// v[j ..] += four f32, or eight elements of 16 bits.
__device__ __forceinline__ void add4(const float4& q, float (&v)[32], int j) {
    f2_split(fadd2(f2(v[j], v[j + 1]), f2(q.x, q.y)), v[j], v[j + 1]);
    f2_split(fadd2(f2(v[j + 2], v[j + 3]), f2(q.z, q.w)), v[j + 2], v[j + 3]);
}
__device__ __forceinline__ void add8(const uint4& q, int type, float (&v)[32], int j) {
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = type == ELT_BF16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[i]))
                                          : __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        v[j + 2 * i] += f.x;
        v[j + 2 * i + 1] += f.y;
    }
}

// The product of the arrays' scales, which the sums are multiplied by. It may leave f32's normal numbers where the sums times it
// do not: then a power of two of it, `pre`, goes to the sums first. (Sums are 0 or between 2^-20 and 2^54, so neither step
// loses what the result holds; above 2^192 the factor is f32's largest number, which leaves 0 at 0 and overflows all else.)
__device__ __forceinline__ float array_scale(const Params& p, float& pre) {
    const float gx = p.gx ? *p.gx : 1.f, gw = p.gw ? *p.gw : 1.f, g = gx * gw;
    pre = 1.f;
    if (g >= FLT_MIN && g <= FLT_MAX) return g;
    pre = g < 1.f ? 0x1p-64f : 0x1p64f;
    const double r = (double)gx * gw / pre;
    return r > FLT_MAX ? FLT_MAX : (float)r;  // NaN stays
}

// act(acc * alpha + bias) + residual for columns c0 .. c0 + nv of a row (zeros behind them). `bias`: theirs, in shared
// memory; with RES, `res` is the warp's residual buffer: its rows there (32 columns of f32, or 64 of 16 bits of which half
// `half`), or with RES_ELEMENT room to exchange them. The arithmetic runs on packed pairs, one instruction for two
// values: the epilogue's time goes by its instructions (three warps a scheduler, one instruction every seven cycles each).
template <bool SCALED, bool RES>
__device__ __forceinline__ void finish32(const Params& p, const float* bias, uint8_t* res, int half, int lane,
                                         int64_t row0, int c0, int nv, float alpha, const uint32_t (&r)[32], float (&v)[32]) {
    const uint64_t al = f2(alpha, alpha);
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
        const float4 q = *reinterpret_cast<const float4*>(bias + j);
        const uint64_t a = f2(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
        const uint64_t b = f2(__uint_as_float(r[j + 2]), __uint_as_float(r[j + 3]));
        f2_split(SCALED ? ffma2(a, al, f2(q.x, q.y)) : fadd2(a, f2(q.x, q.y)), v[j], v[j + 1]);
        f2_split(SCALED ? ffma2(b, al, f2(q.z, q.w)) : fadd2(b, f2(q.z, q.w)), v[j + 2], v[j + 3]);
    }
    if (p.act == ANCHA_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < 32; j += 2) gelu2(v[j], v[j + 1]);
    } else if (p.act == ANCHA_ACT_TANH) {
#pragma unroll
        for (int j = 0; j < 32; j += 2) tanh2(v[j], v[j + 1]);
    }
    if (RES && p.res_mode == RES_ELEMENT) {
        add_plain(p, reinterpret_cast<float*>(res), row0, c0, nv, lane, v);
    } else if (RES) {
        if (p.res_type == ELT_F32) {
#pragma unroll
            for (int q = 0; q < 8; ++q)
                add4(*reinterpret_cast<const float4*>(res + lane * 128 + ((q ^ (lane & 7)) * 16)), v, 4 * q);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                add8(*reinterpret_cast<const uint4*>(res + lane * 128 + (((q + 4 * half) ^ (lane & 7)) * 16)), p.res_type, v, 8 * q);
        }
    }
    if (nv < 32) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (j >= nv) v[j] = 0.f;
    }
}

__device__ __forceinline__ uint32_t pack16(float a, float b, int type) {
    if (type == ELT_BF16) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&t);
    }
    const __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}

// Elements at .. at + nv (at most 4) of a matrix; `vec`: rows and base are 16-byte aligned.
__device__ __forceinline__ void load4(const void* base, int type, bool vec, int64_t at, int nv, float (&v)[4]) {
    if (vec && nv == 4) {
        if (type == ELT_F32) {
            const float4 q = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
            v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
            return;
        }
        const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + at);
        const uint32_t u[2] = {q.x, q.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 f = type == ELT_BF16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[i]))
                                              : __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < nv)
            v[j] = type == ELT_F32    ? static_cast<const float*>(base)[at + j]
                   : type == ELT_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(base)[at + j])
                                      : __half2float(static_cast<const __half*>(base)[at + j]);
}

__device__ __forceinline__ void store4(void* base, int type, bool vec, int64_t at, int nv, const float (&v)[4]) {
    if (vec && nv == 4) {
        if (type == ELT_F32)
            *reinterpret_cast<float4*>(static_cast<float*>(base) + at) = make_float4(v[0], v[1], v[2], v[3]);
        else
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + at) =
                make_uint2(pack16(v[0], v[1], type), pack16(v[2], v[3], type));
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < nv) store_elt(base, at + j, v[j], type);
}

// A lane's row of 32 values in a staging buffer of 128-byte rows with the 128-byte swizzle: 32 columns of f32, or
// half `h` of 64 columns of 16 bits.
__device__ __forceinline__ void stage_row(uint8_t* buf, int lane, int type, int h, const float (&v)[32]) {
    buf += lane * 128;
    if (type == ELT_F32) {
#pragma unroll
        for (int q = 0; q < 8; ++q)
            *reinterpret_cast<float4*>(buf + ((q ^ (lane & 7)) * 16)) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4*>(buf + (((q + 4 * h) ^ (lane & 7)) * 16)) =
                make_uint4(pack16(v[8 * q], v[8 * q + 1], type), pack16(v[8 * q + 2], v[8 * q + 3], type),
                           pack16(v[8 * q + 4], v[8 * q + 5], type), pack16(v[8 * q + 6], v[8 * q + 7], type));
    }
}

// Outputs and residuals at odd addresses or strides, an element at a time: exchanged through the buffer (a lane's row
// there, columns rotated by the row against bank conflicts) so that a warp touches 32 neighbouring columns of a row,
// eight rows in flight.
template <typename T>
__device__ __forceinline__ void store_rows(T* out, int64_t ld, int rows, int nv, int lane, const float* buf) {
    if (lane >= nv) return;
#pragma unroll 1
    for (int r = 0; r < rows; r += 8) {
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = buf[(r + k) * 32 + (lane ^ (r + k))];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (r + k < rows) store_f(out + (r + k) * ld + lane, x[k]);
    }
}
__device__ __forceinline__ void store_plain(const Params& p, float* buf, int64_t row0, int c0, int nv, int lane,
                                            const float (&v)[32]) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 32; ++j) buf[lane * 32 + (j ^ lane)] = v[j];
    __syncwarp();
    const int rows = (int)min((int64_t)32, p.m - row0);
    const int64_t at = row0 * p.ldo + c0;
    if (p.out_type == ELT_F32) store_rows(static_cast<float*>(p.out) + at, p.ldo, rows, nv, lane, buf);
    else if (p.out_type == ELT_BF16) store_rows(static_cast<__nv_bfloat16*>(p.out) + at, p.ldo, rows, nv, lane, buf);
    else store_rows(static_cast<__half*>(p.out) + at, p.ldo, rows, nv, lane, buf);
}
template <typename T>
__device__ __forceinline__ void load_rows(const T* in, int64_t ld, int rows, int nv, int lane, float* buf) {
#pragma unroll 1
    for (int r = 0; r < 32; r += 8) {
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = r + k < rows && lane < nv ? load_f(in + (r + k) * ld + lane) : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) buf[(r + k) * 32 + (lane ^ (r + k))] = x[k];
    }
}
__device__ __forceinline__ void add_plain(const Params& p, float* buf, int64_t row0, int c0, int nv, int lane, float (&v)[32]) {
    const int rows = (int)min((int64_t)32, p.m - row0);
    const int64_t at = row0 * p.ldr + c0;
    __syncwarp();
    if (p.res_type == ELT_F32) load_rows(static_cast<const float*>(p.residual) + at, p.ldr, rows, nv, lane, buf);
    else if (p.res_type == ELT_BF16) load_rows(static_cast<const __nv_bfloat16*>(p.residual) + at, p.ldr, rows, nv, lane, buf);
    else load_rows(static_cast<const __half*>(p.residual) + at, p.ldr, rows, nv, lane, buf);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] += buf[lane * 32 + (j ^ lane)];
    __syncwarp();
}

// A lane's 32 columns quantised, one block of 32 or two of 16, in its registers; the codes go to its row of the staging
// buffer (half `half` of 64 columns). Returns the scale code, or the two.
template <int FMT>
__device__ __forceinline__ uint32_t stage_mx(const MxArray& o, uint8_t* buf, int half, int lane, const float (&v)[32]) {
    constexpr int B = mx_block(FMT), W = FMT == MXF8 ? 8 : 4;
    const float g = FMT == NVF4 && o.global_scale ? *o.global_scale : 1.f;
    uint32_t codes = 0, w[W];
#pragma unroll
    for (int h = 0; h < 32 / B; ++h) {
        float x[B], a = 0.f;
#pragma unroll
        for (int j = 0; j < B; ++j) x[j] = v[h * B + j];
#pragma unroll
        for (int j = 0; j < B; j += 2) a = absmax(a, x[j], x[j + 1]);
        const MxBlock b = mx_block_scale<FMT>(__float_as_uint(a), g);
        codes |= b.code << (8 * h);
        uint32_t e[W * B / 32];
        mx_encode<FMT, B>(x, b, e);
#pragma unroll
        for (int j = 0; j < W * B / 32; ++j) w[h * (W * B / 32) + j] = e[j];
    }
    // Rows of 64 bytes with the 64-byte swizzle (mxf8), of 32 with the 32-byte swizzle.
    if (FMT == MXF8) {
        buf += lane * 64;
        *reinterpret_cast<uint4*>(buf + ((2 * half) ^ ((lane >> 1) & 3)) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4*>(buf + ((2 * half + 1) ^ ((lane >> 1) & 3)) * 16) = make_uint4(w[4 % W], w[5 % W], w[6 % W], w[7 % W]);
    } else {
        *reinterpret_cast<uint4*>(buf + lane * 32 + (half ^ ((lane >> 2) & 1)) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return codes;
}

// Behind a wait that gave up, with every warp past its last issue: what the CTA has in flight ends before its shared memory and
// TMEM are given back (each bounded again). load_drain: the copies of the last `stages` of `issued` slabs, by one thread;
// product_drain: the products, by a converged warp whose commit on `bar`, unused so far, follows them.
__device__ void load_drain(uint64_t* full, uint32_t stages, uint32_t issued) {
    const long long c0 = clock64();
    for (uint32_t j = issued > stages ? issued - stages : 0; j < issued; ++j)
        while (!mbar_try_wait(&full[j % stages], (j / stages) & 1) && clock64() - c0 < kWaitCycles) {
        }
}
template <bool PAIR>
__device__ __forceinline__ void product_drain(uint64_t* bar) {
    if (elect_one()) {
        if (PAIR) umma_commit_pair(bar, 0x1);
        else umma_commit(bar);
    }
    __syncwarp();
    const long long c0 = clock64();
    while (!mbar_try_wait(bar, 0) && clock64() - c0 < kWaitCycles) {
    }
    __syncwarp();
}

// A converged warp's wait; false where one lane's ran out.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* err) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;  // no clock read where there is no wait
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, err));
}

// The tiles of a CTA (or pair), tile0, tile0 + step, ..., as row and column of the tile grid: divided once.
struct TileWalk {
    int mi, ni, dm, dn, n_tiles;
    __device__ __forceinline__ TileWalk(int tile0, int step, int n) : n_tiles(n) {
        mi = tile0 / n; ni = tile0 - mi * n;
        dm = step / n; dn = step - dm * n;
    }
    __device__ __forceinline__ void next() {
        mi += dm;
        ni += dn;
        if (ni >= n_tiles) {
            ni -= n_tiles;
            ++mi;
        }
    }
};

template <int FMT, int BN, bool PAIR, bool RES>
__global__ void __launch_bounds__(Shape<FMT, BN, PAIR>::THREADS, 1)
linear_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
              const __grid_constant__ CUtensorMap tsa, const __grid_constant__ CUtensorMap tsb,
              const __grid_constant__ CUtensorMap tout, const __grid_constant__ CUtensorMap tres,
              const __grid_constant__ Params p) {
    using S = Shape<FMT, BN, PAIR>;
    constexpr int BMT = PAIR ? 2 * BM : BM, EPI = S::EPI;
    const int stages = p.stages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* a_tiles = smem;
    uint8_t* b_tiles = a_tiles + stages * OPERAND_BYTES;
    uint8_t* staging = b_tiles + stages * S::B_BYTES;  // 1024-byte aligned, as the operands
    uint8_t* residual = staging + EPI * STAGING;  // with RES
    uint8_t* biases = residual + (RES ? EPI * STAGING : 0);
    uint8_t* sa_tiles = biases + EPI * BIAS_BYTES;
    uint8_t* sb_tiles = sa_tiles + stages * S::SFA_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(sb_tiles + stages * S::SFB_BYTES);
    uint64_t* empty = full + stages;
    uint64_t* tfull = empty + stages;   // [2] accumulator ready
    uint64_t* tempty = tfull + 2;       // [2] accumulator drained
    uint64_t* rfull = tempty + 2;       // [EPI] residual arrived
    uint64_t* drain = rfull + EPI;      // used behind an abort alone
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile uint32_t* issued = tmem_slot + 2;  // slabs loaded

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = PAIR ? cluster_ctarank() : 0;
    const int tile0 = PAIR ? (int)blockIdx.x / 2 : (int)blockIdx.x;
    const int tstep = PAIR ? (int)gridDim.x / 2 : (int)gridDim.x;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], PAIR ? 2 * EPI : EPI);
        }
        for (int w = 0; w < EPI; ++w) mbar_init(&rfull[w], 1);
        mbar_init(drain, 1);
        *abort = 0;
        fence_barrier_init();
        fence_proxy_async();
        prefetch_tma(&ta);
        prefetch_tma(&tb);
        prefetch_tma(&tsa);
        prefetch_tma(&tsb);
    }
    if (warp == 1) {
        if (PAIR) {
            tmem_alloc_pair(tmem_slot, TMEM_COLS);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(tmem_slot, TMEM_COLS);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();  // the peer's barriers exist before anything arrives on them
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int slabs = (p.kbytes + SLAB - 1) / SLAB;
    TileWalk walk(tile0, tstep, p.n_tiles);

    if (warp == 0) {
        int s = 0;
        uint32_t it = 0, phase = 1;
        for (int t = tile0; t < p.tiles && !*abort; t += tstep, walk.next()) {
            const int m0 = walk.mi * BMT, n0 = walk.ni * BN;
            for (int kb = 0; kb < slabs; ++kb, ++it) {
                if (!warp_wait(&empty[s], phase, abort, p.err)) break;
                if (elect_one()) {
                    uint8_t* a = a_tiles + s * OPERAND_BYTES;
                    uint8_t* b = b_tiles + s * S::B_BYTES;
                    uint8_t* sa = sa_tiles + s * S::SFA_BYTES;
                    uint8_t* sb = sb_tiles + s * S::SFB_BYTES;
                    if (PAIR) {
                        // Both CTAs' copies complete on the even CTA's barrier, which expects both.
                        const uint32_t fb = mapa_shared(smem_u32(&full[s]), 0);
                        if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * S::STAGE);
                        tma_load_3d_pair(a, &ta, fb, kb * SLAB, m0 + (int)rank * BM, 0);
                        tma_load_3d_pair(b, &tb, fb, kb * SLAB, n0 + (int)rank * S::B_ROWS, 0);
                        tma_load_3d_pair(sa, &tsa, fb, 0, kb * S::SF * 2, m0 / 128 + (int)rank);
                        tma_load_3d_pair(sb, &tsb, fb, 0, kb * S::SF * 2, n0 / 128);
                    } else {
                        mbar_arrive_expect_tx(&full[s], S::STAGE);
                        tma_load_3d(a, &ta, &full[s], kb * SLAB, m0, 0);
                        tma_load_3d(b, &tb, &full[s], kb * SLAB, n0, 0);
                        tma_load_3d(sa, &tsa, &full[s], 0, kb * S::SF * 2, m0 / 128);
                        tma_load_3d(sb, &tsb, &full[s], 0, kb * S::SF * 2, n0 / 128);
                    }
                }
                __syncwarp();
                if (++s == stages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
        if (lane == 0) *issued = it;
    } else if (warp == 1) {
        if (rank == 0) {
            constexpr uint32_t idesc = idesc_of<FMT>(BMT, BN);
            int s = 0;
            uint32_t phase = 0, local = 0;
            for (int t = tile0; t < p.tiles && !*abort; t += tstep, ++local, walk.next()) {
                const uint32_t b = local % S::ACCS;
                if (!warp_wait(&tempty[b], (local / S::ACCS & 1) ^ 1, abort, p.err)) break;
                tc_fence_after();
                const uint32_t acc = tmem + b * BN;
                for (int kb = 0; kb < slabs; ++kb) {
                    if (!warp_wait(&full[s], phase, abort, p.err)) break;
                    tc_fence_after();
                    const int steps = min(4, (p.kbytes - kb * SLAB + 31) / 32);
                    if (elect_one()) {
                        slab_products<FMT, PAIR, BN>(acc, tmem + SFA_COL, tmem + SFB_COL, smem_u32(a_tiles + s * OPERAND_BYTES),
                                                     smem_u32(b_tiles + s * S::B_BYTES), smem_u32(sa_tiles + s * S::SFA_BYTES),
                                                     smem_u32(sb_tiles + s * S::SFB_BYTES), idesc, steps, kb == 0,
                                                     BN == 192 ? (uint32_t)(walk.ni & 1) * 2 : 0);
                        if (PAIR) umma_commit_pair(&empty[s], 0x3);
                        else umma_commit(&empty[s]);
                        if (kb == slabs - 1) {
                            if (PAIR) umma_commit_pair(&tfull[b], 0x3);
                            else umma_commit(&tfull[b]);
                        }
                    }
                    __syncwarp();
                    if (++s == stages) {
                        s = 0;
                        phase ^= 1;
                    }
                }
            }
        }
    } else {
        const int quarter = warp % 4, col0 = (warp - 2) / 4 * 64;
        uint8_t* stage = staging + (warp - 2) * STAGING;
        uint8_t* res = residual + (warp - 2) * STAGING;
        uint64_t* rbar = &rfull[warp - 2];
        float* bias = reinterpret_cast<float*>(biases) + (warp - 2) * 64;
        float alpha = 1.f;
        float pre = 1.f;
        if (FMT == NVF4) alpha = array_scale(p, pre);
        const bool wide = p.out_mode == OUT_TMA && p.out_type == ELT_F32;
        float b0 = 0.f, b1 = 0.f;
        const auto load_bias = [&](int ni) {
            const int c = ni * BN + col0 + lane;
            b0 = c < p.n ? p.bias[c] : 0.f;
            b1 = c + 32 < p.n ? p.bias[c + 32] : 0.f;
        };
        if (p.bias && tile0 < p.tiles) load_bias(walk.ni);
        // The residual's 32 x 32 f32, or 32 x 64 elements of 16 bits, in the layout of the staging buffer.
        const bool res_tma = p.res_mode == RES_TMA, res_wide = p.res_type == ELT_F32;
        uint32_t res_phase = 0;
        bool res_pending = false;
        const auto load_res = [&](int c, int64_t row0) {
            __syncwarp();  // every lane has read the buffer
            if (elect_one()) {
                mbar_arrive_expect_tx(rbar, STAGING);
                tma_load_3d(res, &tres, rbar, c, (int)row0, 0);
            }
            res_pending = true;
        };
        uint32_t local = 0;
        for (int t = tile0; t < p.tiles; t += tstep, ++local) {
            const int c_first = walk.ni * BN + col0, b = local % S::ACCS;
            const int64_t row0 = (int64_t)walk.mi * BMT + (int)rank * BM + quarter * 32, row = row0 + lane;
            const bool some = row0 < p.m && c_first < p.n;
            walk.next();
            // The tile's bias, on its way since the tile before: read when it is needed it would cost the latency of L2.
            __syncwarp();
            bias[lane] = b0;
            bias[32 + lane] = b1;
            if (p.bias && t + tstep < p.tiles) load_bias(walk.ni);
            if (RES && res_tma && some) load_res(c_first, row0);
            if (!warp_wait(&tfull[b], local / S::ACCS & 1, abort, p.err)) break;
            tc_fence_after();
            const uint32_t base = tmem + b * BN + col0 + ((uint32_t)(quarter * 32) << 16);
            bool res_ok = true;
            uint32_t codes = 0, r[2][32];
            tmem_ld32(base, r[0]);
            tmem_ld32(base + 32, r[1]);
            tmem_wait_ld();
            // This warp is done with the accumulator (and with every earlier one).
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                uint64_t* bar = &tempty[b];
                if (PAIR) mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(bar), 0));
                else mbar_arrive(bar);
            }
            if (FMT == NVF4 && pre != 1.f) {
#pragma unroll
                for (int j = 0; j < 64; ++j) r[j / 32][j % 32] = __float_as_uint(__uint_as_float(r[j / 32][j % 32]) * pre);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c0 = c_first + 32 * h, nv = min(32, p.n - c0);
                if (nv <= 0 || !some) continue;
                float v[32];
                if (p.out_mode != OUT_PLAIN && (wide || h == 0)) {
                    if (elect_one()) bulk_wait_read<0>();  // the store that last read the buffer is done with it
                    __syncwarp();
                }
                if (RES && res_pending) {
                    res_ok = warp_wait(rbar, res_phase, abort, p.err);
                    if (!res_ok) break;
                    res_phase ^= 1;
                    res_pending = false;
                }
                finish32<FMT == NVF4, RES>(p, bias + 32 * h, res, h, lane, row0, c0, nv, alpha, r[h], v);
                if (RES && res_tma && res_wide && h == 0 && c0 + 32 < p.n) load_res(c0 + 32, row0);
                if (p.out_mode == OUT_TMA) {
                    stage_row(stage, lane, p.out_type, h, v);
                    if (wide) {
                        fence_proxy_async();
                        __syncwarp();
                        if (elect_one()) {
                            tma_store_3d(&tout, stage, c0, (int)row0, 0);
                            bulk_commit();
                        }
                    }
                } else if (p.out_mode == OUT_PLAIN) {
                    store_plain(p, reinterpret_cast<float*>(stage), row0, c0, nv, lane, v);
                } else {
                    if (p.om.format == MXF8) codes |= stage_mx<MXF8>(p.om, stage, h, lane, v) << (8 * h);
                    else if (p.om.format == MXF4) codes |= stage_mx<MXF4>(p.om, stage, h, lane, v) << (8 * h);
                    else codes |= stage_mx<NVF4>(p.om, stage, h, lane, v) << (16 * h);
                }
            }
            if (RES && !res_ok) break;
            if (p.out_mode != OUT_PLAIN && !wide && some) {
                fence_proxy_async();
                __syncwarp();
                if (elect_one()) {
                    tma_store_3d(&tout, stage, p.out_mode == OUT_MX && p.om.format != MXF8 ? c_first / 2 : c_first, (int)row0, 0);
                    bulk_commit();
                }
            }
            if (p.out_mode == OUT_MX) {
                // The scales of 64 columns; 0 behind the last row and column, as far as the scale tiles reach.
                const int blk = c_first >> p.oblock_log2;
                if (row < p.rows_padded && blk / 4 < p.okt) {
                    uint8_t* sc = p.om.scales + mx_scale_word(row, blk / 4, p.okt) + blk % 4;
                    if (row >= p.m) codes = 0;
                    if (p.oblock_log2 == 5) {
                        *reinterpret_cast<uint16_t*>(sc) = (uint16_t)codes;
                        // The last tile may end in the middle of a scale tile's 128 columns: its last warps write the rest.
                        if (c_first + 64 == p.n_tiles * BN && blk % 4 == 0) *reinterpret_cast<uint16_t*>(sc + 2) = 0;
                    } else {
                        *reinterpret_cast<uint32_t*>(sc) = codes;
                    }
                }
            }
        }
        if (RES && res_pending && lane == 0) {  // after an abort: the copy in flight lands before the CTA exits (bounded)
            const long long c0 = clock64();
            while (!mbar_try_wait(rbar, res_phase) && clock64() - c0 < kWaitCycles) {
            }
        }
        __syncwarp();
        if (elect_one()) bulk_wait<0>();
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (*abort && rank == 0) {  // the even CTA's barriers count the odd one's copies too
        if (threadIdx.x == 0) load_drain(full, stages, *issued);
        if (warp == 1) product_drain<PAIR>(drain);
        __syncthreads();
    }
    // With a pair, neither CTA releases TMEM or exits while the other may still use its shared memory.
    if (PAIR) cluster_sync();
    if (warp == 1) {
        __syncwarp();
        if (PAIR) tmem_dealloc_pair(tmem, TMEM_COLS);
        else tmem_dealloc(tmem, TMEM_COLS);
    }
}

// ---- few tiles ------------------------------------------------------------------------------

// Few rows of x, or few tiles: a cluster of `splits` CTAs shares one tile, each multiplying a part of K, so that
// the weight streams through many SMs. The operands change places: 128 rows of w are the instruction's M and TN rows
// of x its N, so a single token costs 16 columns instead of 128 rows. Each CTA leaves its partial sums in its
// shared memory (over the operands, which are done with); then rank r of the cluster finishes the rows r, r + splits,
// ... of x, adding the ranks' sums in rank order through distributed shared memory. A warp takes a row of x and the
// tile's 128 columns, four to a lane.
template <int FMT, int TN>
struct SplitShape {
    static constexpr int SF = sf_tiles(FMT);
    static constexpr int STAGE = OPERAND_BYTES + TN * SLAB + 2 * SF * SF_TILE;
    static constexpr int FIT = (113 * 1024 - 1280) / STAGE, STAGES = FIT < 5 ? FIT : 5;  // two CTAs per SM
    static constexpr int BYTES = 1024 + STAGES * STAGE + 256;
    static constexpr uint32_t COLS = TN == 128 ? 256 : TN == 64 ? 128 : 64;
    static_assert(TN + 8 * SF <= (int)COLS, "accumulator and scales do not fit");
    static_assert(TN * BM * 4 <= STAGES * STAGE && BYTES <= 113 * 1024, "shared memory");
};
constexpr int SPLIT_WARPS = 6, SPLIT_THREADS = 32 * SPLIT_WARPS;

// Four neighbouring columns per lane, a warp's 128 from c0 on (zeros behind the row's end), quantised.
template <int FMT>
__device__ __forceinline__ void store_mx_lanes(const MxArray& o, int okt, int64_t row, int c0, int lane, const float (&v)[4]) {
    constexpr int B = mx_block(FMT), LB = B / 4;  // lanes of a block
    const float g = FMT == NVF4 && o.global_scale ? *o.global_scale : 1.f;
    uint32_t a = __float_as_uint(absmax(absmax(0.f, v[0], v[1]), v[2], v[3]));
#pragma unroll
    for (int d = 1; d < LB; d *= 2) a = max(a, __shfl_xor_sync(0xffffffffu, a, d));
    const MxBlock b = mx_block_scale<FMT>(a, g);
    float x[8] = {v[0], v[1], v[2], v[3]};
    uint32_t w[FMT == MXF8 ? 2 : 1];
    mx_encode<FMT, 8>(x, b, w);
    const int c = c0 + 4 * lane;
    if (mx_bytes(FMT, c) < mx_row_bytes(FMT, o.cols)) {
        uint8_t* d = o.data + row * o.ld + mx_bytes(FMT, c);
        if (FMT == MXF8) *reinterpret_cast<uint32_t*>(d) = w[0];
        else *reinterpret_cast<uint16_t*>(d) = (uint16_t)w[0];
    }
    if (lane % LB == 0 && c / B < 4 * okt) o.scales[mx_scale_word(row, c / B / 4, okt) + c / B % 4] = (uint8_t)b.code;
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

template <int FMT, int TN>
__global__ void __launch_bounds__(SPLIT_THREADS)
split_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx,
             const __grid_constant__ CUtensorMap tsw, const __grid_constant__ CUtensorMap tsx,
             const __grid_constant__ Params p, int splits) {
    using S = SplitShape<FMT, TN>;
    constexpr int STAGES = S::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* w_tiles = smem;
    uint8_t* x_tiles = w_tiles + STAGES * OPERAND_BYTES;
    uint8_t* sw_tiles = x_tiles + STAGES * TN * SLAB;
    uint8_t* sx_tiles = sw_tiles + STAGES * S::SF * SF_TILE;
    float* partial = reinterpret_cast<float*>(smem);  // [TN][128], once the products are done
    uint64_t* full = reinterpret_cast<uint64_t*>(sx_tiles + STAGES * S::SF * SF_TILE);
    uint64_t* empty = full + STAGES;
    uint64_t* done = empty + STAGES;
    uint64_t* drain = done + 1;  // used behind an abort alone
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile uint32_t* issued = tmem_slot + 2;  // slabs loaded

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = (int)blockIdx.x % splits, n0 = (int)blockIdx.x / splits * BM, m0 = (int)blockIdx.y * TN;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(done, 1);
        mbar_init(drain, 1);
        *abort = 0;
        fence_barrier_init();
        fence_proxy_async();
        prefetch_tma(&tw);
        prefetch_tma(&tx);
        prefetch_tma(&tsw);
        prefetch_tma(&tsx);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, S::COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int slabs = (p.kbytes + SLAB - 1) / SLAB;
    const int kb0 = (int)((int64_t)slabs * rank / splits), kb1 = (int)((int64_t)slabs * (rank + 1) / splits);

    if (warp == 0) {
        uint32_t it = 0;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const int s = it % STAGES;
            if (!warp_wait(&empty[s], ((it / STAGES) & 1) ^ 1, abort, p.err)) break;
            if (elect_one()) {
                mbar_arrive_expect_tx(&full[s], S::STAGE);
                tma_load_3d(w_tiles + s * OPERAND_BYTES, &tw, &full[s], kb * SLAB, n0, 0);
                tma_load_3d(sw_tiles + s * S::SF * SF_TILE, &tsw, &full[s], 0, kb * S::SF * 2, n0 / 128);
                tma_load_3d(x_tiles + s * TN * SLAB, &tx, &full[s], kb * SLAB, m0, 0);
                tma_load_3d(sx_tiles + s * S::SF * SF_TILE, &tsx, &full[s], 0, kb * S::SF * 2, m0 / 128);
            }
            __syncwarp();
        }
        if (lane == 0) *issued = it;
    } else if (warp == 1) {
        constexpr uint32_t idesc = idesc_of<FMT>(BM, TN);
        uint32_t it = 0;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const int s = it % STAGES;
            if (!warp_wait(&full[s], (it / STAGES) & 1, abort, p.err)) break;
            tc_fence_after();
            const int steps = min(4, (p.kbytes - kb * SLAB + 31) / 32);
            if (elect_one()) {
                slab_products<FMT, false, TN>(tmem, tmem + TN, tmem + TN + 4 * S::SF, smem_u32(w_tiles + s * OPERAND_BYTES),
                                              smem_u32(x_tiles + s * TN * SLAB), smem_u32(sw_tiles + s * S::SF * SF_TILE),
                                              smem_u32(sx_tiles + s * S::SF * SF_TILE), idesc, steps, kb == kb0);
                umma_commit(&empty[s]);
                if (kb == kb1 - 1) umma_commit(done);
            }
            __syncwarp();
        }
    }
    const int live = min(TN, p.m - m0);  // rows of x in the tile
    if (warp >= 2) {
        const int quarter = warp % 4;
        if (__all_sync(0xffffffffu, mbar_wait(done, 0, abort, p.err))) {
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < live; c += 16) {
                uint32_t r[16];
                tmem_ld16(tmem + c + ((uint32_t)(quarter * 32) << 16), r);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) partial[(c + j) * BM + quarter * 32 + lane] = __uint_as_float(r[j]);
            }
        } else {  // the sums are missing, which the peers' results show
            for (int c = 0; c < live; ++c) partial[c * BM + quarter * 32 + lane] = __int_as_float(0x7FC00000);
        }
        tc_fence_before();
    }
    __syncwarp();
    cluster_sync();
    if (warp == 1) {
        if (*abort) product_drain<false>(drain);
        tc_fence_after();
        tmem_dealloc(tmem, S::COLS);
    }
    float alpha = 1.f;
    float pre = 1.f;
    if (FMT == NVF4) alpha = array_scale(p, pre);
    const int col = n0 + 4 * lane, nv = min(4, p.n - col);  // this lane's columns
    float bias[4] = {};
    if (p.bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < nv) bias[j] = p.bias[col + j];
    }
    for (int c = rank + warp * splits; c < live; c += SPLIT_WARPS * splits) {
        const int64_t row = m0 + c;
        float res[4] = {};
        if (p.residual) load4(p.residual, p.res_type, p.res_mode == RES_TMA, row * p.ldr + col, nv, res);
        float v[4] = {};
        const uint32_t at = smem_u32(partial + c * BM + 4 * lane);
        for (int k = 0; k < splits; ++k) {
            const float4 q = ld_cluster4(mapa_shared(at, k));
            v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = fmaf(FMT == NVF4 ? v[j] * pre : v[j], alpha, bias[j]);
        if (p.act == ANCHA_ACT_GELU) {
            gelu2(v[0], v[1]);
            gelu2(v[2], v[3]);
        } else if (p.act == ANCHA_ACT_TANH) {
            tanh2(v[0], v[1]);
            tanh2(v[2], v[3]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = j < nv ? v[j] + res[j] : 0.f;
        if (p.out_mode != OUT_MX) store4(p.out, p.out_type, p.out_mode == OUT_TMA, row * p.ldo + col, nv, v);
        else if (p.om.format == MXF8) store_mx_lanes<MXF8>(p.om, p.okt, row, n0, lane, v);
        else if (p.om.format == MXF4) store_mx_lanes<MXF4>(p.om, p.okt, row, n0, lane, v);
        else store_mx_lanes<NVF4>(p.om, p.okt, row, n0, lane, v);
    }
    // Quantised output: the scales of the rows behind the last, in its tile, are 0 (the last row tile's CTAs share them).
    if (p.out_mode == OUT_MX && blockIdx.y == gridDim.y - 1) {
        const int b = mx_block(p.om.format);
        const int64_t end = ((int64_t)p.m + 127) / 128 * 128;
        const int words = max(0, min(p.okt - n0 / (4 * b), BM / (4 * b)));
        for (int64_t i = rank * SPLIT_THREADS + threadIdx.x; i < (end - p.m) * words; i += splits * SPLIT_THREADS)
            *reinterpret_cast<uint32_t*>(p.om.scales + mx_scale_word(p.m + i / words, n0 / (4 * b) + (int)(i % words), p.okt)) = 0;
    }
    __syncwarp();
    if (*abort && threadIdx.x == 0) load_drain(full, STAGES, *issued);
    __syncwarp();
    cluster_sync();  // a CTA's shared memory stays while its peers read it
}

template <int FMT, int TN>
int launch_split(const MxLinear& q, const Params& p, int splits, cudaStream_t s) {
    using S = SplitShape<FMT, TN>;
    auto kernel = split_kernel<FMT, TN>;
    static bool configured[64] = {};
    int dev = 0;
    ANCHA_CUDA(cudaGetDevice(&dev));
    if (!configured[dev & 63]) {
        ANCHA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES));
        configured[dev & 63] = true;
    }
    CUtensorMap tw, tx, tsw, tsx;
    const int64_t kt = mx_ktiles(FMT, q.x.cols);
    ANCHA_TRY(make_tma_bytes(&tw, q.w.data, p.kbytes, p.n, q.w.ld, SLAB, BM, 128));
    ANCHA_TRY(make_tma_bytes(&tx, q.x.data, p.kbytes, p.m, q.x.ld, SLAB, TN, 128));
    ANCHA_TRY(make_tma_scales(&tsw, q.w.scales, kt, ceil_div(p.n, 128), S::SF, 1));
    ANCHA_TRY(make_tma_scales(&tsx, q.x.scales, kt, ceil_div(p.m, 128), S::SF, 1));
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(ceil_div(p.n, BM) * splits), (unsigned)ceil_div(p.m, TN), 1);
    cfg.blockDim = dim3(SPLIT_THREADS, 1, 1);
    cfg.dynamicSmemBytes = S::BYTES;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    ANCHA_CUDA(cudaLaunchKernelEx(&cfg, kernel, tw, tx, tsw, tsx, p, splits));
    return check_launch("mx_linear (split)");
}

// RES: with a residual (the kernel without one keeps its registers and shared memory).
template <int FMT, int BN, bool PAIR, bool RES>
int launch(const MxLinear& q, Params p, cudaStream_t s) {
    using S = Shape<FMT, BN, PAIR>;
    auto kernel = linear_kernel<FMT, BN, PAIR, RES>;
    static int slots[64] = {};  // co-resident CTAs (one per SM) or CTA pairs
    int dev = 0;
    ANCHA_CUDA(cudaGetDevice(&dev));
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(S::THREADS, 1, 1);
    p.stages = S::stages(RES);
    cfg.dynamicSmemBytes = S::bytes(RES);
    cfg.attrs = attr;
    cfg.numAttrs = PAIR ? 1 : 0;
    if (!slots[dev & 63]) {
        ANCHA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::bytes(RES)));
        int n = 0;
        if (PAIR) {
            cfg.gridDim = dim3(2, 1, 1);
            ANCHA_CUDA(cudaOccupancyMaxActiveClusters(&n, (void*)kernel, &cfg));
            if (n < 1) return fail(ANCHA_E_UNSUPPORTED, "mx_linear: no CTA pair fits an SM pair");
        } else {
            ANCHA_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
        }
        slots[dev & 63] = n;
    }
    CUtensorMap ta, tb, tsa, tsb, to;
    const int64_t akt = mx_ktiles(FMT, q.x.cols);
    ANCHA_TRY(make_tma_bytes(&ta, q.x.data, p.kbytes, p.m, q.x.ld, SLAB, BM, 128));
    ANCHA_TRY(make_tma_bytes(&tb, q.w.data, p.kbytes, p.n, q.w.ld, SLAB, S::B_ROWS, 128));
    ANCHA_TRY(make_tma_scales(&tsa, q.x.scales, akt, ceil_div(p.m, 128), S::SF, 1));
    ANCHA_TRY(make_tma_scales(&tsb, q.w.scales, akt, ceil_div(p.n, 128), S::SF, S::RANGES));
    to = ta;
    if (p.out_mode == OUT_MX)
        ANCHA_TRY(make_tma_bytes(&to, p.om.data, mx_row_bytes(p.om.format, p.om.cols), p.m, p.om.ld,
                                 p.om.format == MXF8 ? 64 : 32, 32, p.om.format == MXF8 ? 64 : 32));
    else if (p.out_mode == OUT_TMA)
        ANCHA_TRY(make_tma_store_3d(&to, p.out, p.out_type, p.n, p.m, 1, p.ldo, (int64_t)p.m * p.ldo, p.out_type == ELT_F32 ? 32 : 64, 32));
    CUtensorMap tr = ta;
    if (p.res_mode == RES_TMA)
        ANCHA_TRY(make_tma_store_3d(&tr, p.residual, p.res_type, p.n, p.m, 1, p.ldr, (int64_t)p.m * p.ldr,
                                    p.res_type == ELT_F32 ? 32 : 64, 32));
    p.m_tiles = (int)ceil_div(p.m, PAIR ? 2 * BM : BM);
    p.n_tiles = (int)ceil_div(p.n, BN);
    const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
    if (tiles > 0x7fffffff) return fail(ANCHA_E_UNSUPPORTED, "mx_linear: too many tiles");
    p.tiles = (int)tiles;
    const int units = std::min(p.tiles, slots[dev & 63]);
    cfg.gridDim = dim3(PAIR ? 2 * units : units, 1, 1);
    cfg.stream = s;
    ANCHA_CUDA(cudaLaunchKernelEx(&cfg, kernel, ta, tb, tsa, tsb, to, tr, p));
    return check_launch("mx_linear");
}

template <int FMT, int BN, bool PAIR>
int launch(const MxLinear& q, const Params& p, cudaStream_t s) {
    return p.res_mode != RES_NONE ? launch<FMT, BN, PAIR, true>(q, p, s) : launch<FMT, BN, PAIR, false>(q, p, s);
}

template <int FMT>
int by_shape(const MxLinear& q, const Params& p, cudaStream_t s) {
    // Split where the rows fill no tile, or the tiles are few and K is long (measured, split / whole tiles: 2000x64x8192
    // nvf4 12 / 17 us, 133x1544x1000 mxf8 9.4 / 10.5 us; 65x1536x384 7.2 / 5.4 us, 128x4096x4096 mxf4 12.3 / 10.6 us). Of
    // 1, 2, 4 or 8 parts the most that leave each a slab and need no more than two CTAs per SM.
    const int slabs = (int)ceil_div(p.kbytes, SLAB);
    const int64_t row_tiles = p.m <= 64 ? 1 : ceil_div(p.m, 128), tiles = row_tiles * ceil_div(p.n, 128);
    if (p.m <= 64 || (tiles <= 30 && slabs >= 8)) {
        int splits = 1;
        while (splits < 8 && 2 * splits <= slabs && tiles * 2 * splits <= 296) splits *= 2;
        if (p.m <= 16) return launch_split<FMT, 16>(q, p, splits, s);
        if (p.m <= 64) return launch_split<FMT, 64>(q, p, splits, s);
        return launch_split<FMT, 128>(q, p, splits, s);
    }
    if (p.m > 128 && p.n > 128) {
        // 192 columns a tile, with two whole accumulators in TMEM, where the epilogue is the limit (up to 16 slabs of K) or
        // where they pad n less; else 256, whose operands make fewer bytes (measured, 192 / 256: 48060x1536x384 mxf8
        // gelu 70 / 83 us, 16384x2048x2048 mxf8 80 / 98 us, 8192^3 mxf8 480 / 447 us and nvf4 267 / 236 us).
        if (slabs <= 16 || ceil_div(p.n, 192) * 192 < ceil_div(p.n, 256) * 256)
            return launch<FMT, 192, true>(q, p, s);
        return launch<FMT, 256, true>(q, p, s);
    }
    return launch<FMT, 128, false>(q, p, s);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

int mx_linear(const MxLinear& q, cudaStream_t s) {
    if (!q.x.rows || !q.w.rows) return ANCHA_OK;
    Params p{};
    p.m = (int)q.x.rows; p.n = (int)q.w.rows; p.kbytes = (int)mx_bytes(q.x.format, q.x.cols);
    p.gx = q.x.global_scale; p.gw = q.w.global_scale;
    p.bias = q.bias;
    p.residual = q.residual; p.ldr = q.ldr; p.res_type = q.res_type;
    p.res_mode = !q.residual ? RES_NONE
                 : aligned16(q.residual) && q.ldr * (int64_t)elt_size(q.res_type) % 16 == 0 ? RES_TMA : RES_ELEMENT;
    p.rows_padded = (int)(ceil_div(p.m, 128) * 128);
    p.act = q.act;
    p.out = q.out; p.ldo = q.ldo; p.out_type = q.out_type;
    if (q.out_mx) {
        p.out_mode = OUT_MX;
        p.om = *q.out_mx;
        p.okt = (int)mx_ktiles(p.om.format, p.om.cols);
        p.oblock_log2 = p.om.format == NVF4 ? 4 : 5;
    } else {
        p.out_mode = aligned16(q.out) && q.ldo * (int64_t)elt_size(q.out_type) % 16 == 0 ? OUT_TMA : OUT_PLAIN;
    }
    p.err = device_error_word();
    return q.x.format == MXF8 ? by_shape<MXF8>(q, p, s) : q.x.format == MXF4 ? by_shape<MXF4>(q, p, s)
                                                                             : by_shape<NVF4>(q, p, s);
}

}  // namespace ancha
