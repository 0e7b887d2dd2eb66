// Product of two microscaled arrays with bias, activation and residual.
#include "mx.cuh"
#include "tc.cuh"

namespace ancha {
namespace {

constexpr int T = 64, TK = 32;  // output tile and K step

template <int FMT>
__device__ __forceinline__ float element(const MxArray& a, int64_t row, int col, int64_t kt, float g) {
    if (row >= a.rows || col >= a.cols) return 0.f;
    const uint8_t byte = a.data[row * a.ld + (FMT == MXF8 ? col : col / 2)];
    const float e = FMT == MXF8 ? e4m3_value(byte)
                                : (col % 2 ? mx_pair_values<FMT>(byte).y : mx_pair_values<FMT>(byte).x);
    const int b = col / mx_block(FMT);
    return e * mx_scale_value<FMT>(a.scales[mx_scale_word(row, b / 4, kt) + b % 4]) * g;
}

template <int FMT>
__device__ __forceinline__ void quantize_row(const MxArray& o, const float* v, int64_t row, int c, int64_t kt) {
    constexpr int B = mx_block(FMT);
    const float g = FMT == NVF4 && o.global_scale ? *o.global_scale : 1.f;
    uint32_t a = 0;
    for (int j = 0; j < B; ++j) a = max(a, abs_bits(v[j]));
    const MxBlock b = mx_block_scale<FMT>(a, g);
    for (int j = 0; j < B; j += 2) {
        const uint32_t p = mx_pair<FMT>(mx_scaled<FMT>(v[j], b), mx_scaled<FMT>(v[j + 1], b));
        const int64_t at = mx_bytes(FMT, c + j);
        if (at >= mx_row_bytes(FMT, o.cols)) continue;
        o.data[row * o.ld + at] = (uint8_t)p;
        if (FMT == MXF8) o.data[row * o.ld + at + 1] = (uint8_t)(p >> 8);
    }
    o.scales[mx_scale_word(row, c / B / 4, kt) + c / B % 4] = (uint8_t)b.code;
}

template <int FMT>
__global__ void __launch_bounds__(256) linear_kernel(MxLinear q, MxArray om, bool mx_out) {
    __shared__ float a[TK][T + 1], b[TK][T + 1], o[T][T + 1];
    const int64_t m0 = (int64_t)blockIdx.y * T;
    const int n0 = blockIdx.x * T, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int k = q.x.cols;
    const int64_t kt = mx_ktiles(FMT, k);
    const float gx = FMT == NVF4 && q.x.global_scale ? *q.x.global_scale : 1.f;
    const float gw = FMT == NVF4 && q.w.global_scale ? *q.w.global_scale : 1.f;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < k; k0 += TK) {
        for (int i = threadIdx.x; i < T * TK; i += 256) {
            const int r = i / TK, c = i % TK;
            a[c][r] = element<FMT>(q.x, m0 + r, k0 + c, kt, gx);
            b[c][r] = element<FMT>(q.w, n0 + r, k0 + c, kt, gw);
        }
        __syncthreads();
        for (int c = 0; c < TK; ++c)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[c][ty * 4 + i], b[c][tx * 4 + j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t row = m0 + ty * 4 + i;
            const int col = n0 + tx * 4 + j;
            float v = acc[i][j];
            if (row < q.x.rows && col < q.w.rows) {
                if (q.bias) v += q.bias[col];
                if (q.act == ANCHA_ACT_GELU) v = gelu_fast(v);
                if (q.act == ANCHA_ACT_TANH) v = tanh_fast(v);
                if (q.residual) {
                    const int64_t at = row * q.ldr + col;
                    v += q.res_type == ELT_F32    ? static_cast<const float*>(q.residual)[at]
                         : q.res_type == ELT_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(q.residual)[at])
                                                  : __half2float(static_cast<const __half*>(q.residual)[at]);
                }
                if (!mx_out) store_elt(q.out, row * q.ldo + col, v, q.out_type);
            } else {
                v = 0.f;
            }
            o[ty * 4 + i][tx * 4 + j] = v;
        }
    if (!mx_out) return;
    __syncthreads();
    // One block of the output's format per thread; scales behind the ends are 0.
    const int blk = mx_block(om.format), per_row = T / blk;
    const int64_t okt = mx_ktiles(om.format, om.cols);
    for (int i = threadIdx.x; i < T * per_row; i += 256) {
        const int64_t row = m0 + i / per_row;
        const int c = n0 + i % per_row * blk;
        if (c / blk >= 4 * okt) continue;
        const float* v = &o[i / per_row][i % per_row * blk];
        if (row >= om.rows) om.scales[mx_scale_word(row, c / blk / 4, okt) + c / blk % 4] = 0;
        else if (om.format == MXF8) quantize_row<MXF8>(om, v, row, c, okt);
        else if (om.format == MXF4) quantize_row<MXF4>(om, v, row, c, okt);
        else quantize_row<NVF4>(om, v, row, c, okt);
    }
}

}  // namespace

int mx_linear(const MxLinear& q, cudaStream_t s) {
    if (!q.x.rows || !q.w.rows) return ANCHA_OK;
    // Quantised outputs: whole scale tiles are walked, for the zero scales behind the ends.
    const MxArray om = q.out_mx ? *q.out_mx : MxArray{};
    const int64_t m = q.out_mx ? ceil_div(q.x.rows, 128) * 128 : q.x.rows;
    const int64_t n = q.out_mx ? mx_ktiles(om.format, om.cols) * 4 * mx_block(om.format) : q.w.rows;
    if (ceil_div(m, T) > 65535) return fail(ANCHA_E_UNSUPPORTED, "mx_linear: too many rows");
    const dim3 grid((unsigned)ceil_div(n, T), (unsigned)ceil_div(m, T));
    if (q.x.format == MXF8) linear_kernel<MXF8><<<grid, 256, 0, s>>>(q, om, q.out_mx != nullptr);
    else if (q.x.format == MXF4) linear_kernel<MXF4><<<grid, 256, 0, s>>>(q, om, q.out_mx != nullptr);
    else linear_kernel<NVF4><<<grid, 256, 0, s>>>(q, om, q.out_mx != nullptr);
    return check_launch("mx_linear");
}

}  // namespace ancha
