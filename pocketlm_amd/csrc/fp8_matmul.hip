// Product of FP8 e4m3 activation rows (a scale for each 128 columns of a row)
// and an FP8 e4m3 block-scaled weight (a scale for each 128 x 128 block):
//
//   out[m][n] = sum_b sx[m][b] * sw[n / 128][b] * sum_{k in block b} x[m][k] * w[n][k]
//
// v_mfma_f32_16x16x128_f8f6f4 takes one block of 128 columns: its result is
// the block's inner sum, and the scaled sum over the blocks is kept in fp32 by
// vector fma.  NaN bytes, in the rows or in the weight, are NaN.
#include <algorithm>

#include "common.h"
#include "fp8_mfma.h"

namespace {

using namespace plm_fp8;

enum OutType { kOutF16 = 0, kOutBF16 = 1, kOutF32 = 2 };

typedef int plm_i32x8 __attribute__((ext_vector_type(8)));

struct MatmulArgs {
    const uint8_t* x;
    const float* xs;
    const uint8_t* w;
    const float* ws;
    void* out;
    int64_t m;
    int64_t n;
    int64_t k;
    int64_t scale_cols;  // of ws
    int blocks;          // of 128 columns; the row length of xs
    int out_type;
};

__device__ __forceinline__ void store_out(const MatmulArgs& a, int64_t at, float v) {
    if (a.out_type == kOutBF16)
        static_cast<__bf16*>(a.out)[at] = static_cast<__bf16>(v);
    else if (a.out_type == kOutF16)
        static_cast<_Float16*>(a.out)[at] = static_cast<_Float16>(v);
    else
        static_cast<float*>(a.out)[at] = v;
}

// One result a thread, for rows that are not whole 16-byte pieces.
__global__ __launch_bounds__(256) void fp8_matmul_scalar_kernel(const MatmulArgs a) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (at >= a.m * a.n) return;
    const int64_t m = at / a.n, n = at - m * a.n;
    const uint8_t* x = a.x + m * a.k;
    const uint8_t* w = a.w + n * a.k;
    float sum = 0.0f;
    for (int b = 0; b < a.blocks; ++b) {
        const int64_t end = min(a.k, static_cast<int64_t>(b + 1) * 128);
        float s = 0.0f;
        for (int64_t k = static_cast<int64_t>(b) * 128; k < end; ++k)
            s = fmaf(__builtin_amdgcn_cvt_f32_fp8(static_cast<int>(x[k]), 0),
                     __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w[k]), 0), s);
        sum = fmaf(s, a.xs[m * a.blocks + b] * a.ws[(n >> 7) * a.scale_cols + b], sum);
    }
    store_out(a, at, sum);
}

__device__ __forceinline__ plm_f32x4 mfma_fp8(const plm_u32x4 a0, const plm_u32x4 a1, const plm_u32x4 b0,
                                              const plm_u32x4 b1, const plm_f32x4 c) {
    const plm_i32x8 a = {static_cast<int>(a0.x), static_cast<int>(a0.y), static_cast<int>(a0.z), static_cast<int>(a0.w),
                         static_cast<int>(a1.x), static_cast<int>(a1.y), static_cast<int>(a1.z), static_cast<int>(a1.w)};
    const plm_i32x8 b = {static_cast<int>(b0.x), static_cast<int>(b0.y), static_cast<int>(b0.z), static_cast<int>(b0.w),
                         static_cast<int>(b1.x), static_cast<int>(b1.y), static_cast<int>(b1.z), static_cast<int>(b1.w)};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}

// Few rows: a workgroup owns 16 TA weight rows and 16 TB activation rows; its
// waves take the K blocks w, w + nw, ... and their sums meet in LDS, added in
// wave order.  Lane l holds, of weight row (activation row) l & 15, the bytes
// 16 (l >> 4) .. + 15 of each half of a block: the same columns on both
// sides, which is all that the inner sum needs.
template <int TA, int TB, int P, int MAXW>
__global__ __launch_bounds__(64 * MAXW) void fp8_matmul_rows_kernel(const MatmulArgs a) {
    extern __shared__ plm_f32x4 red[];  // [wave][tile][lane]
    const int nw = blockDim.x >> 6;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int li = lane & 15, qd = lane >> 4;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16 * TA;
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * 16 * TB;
    const uint8_t* wrow[TA];
    const uint8_t* xrow[TB];
    const float* sx[TB];
    const float* sw[TA];
#pragma unroll
    for (int t = 0; t < TA; ++t) {
        // rows past the end repeat the last one; their results are dropped
        const int64_t n = min(n0 + 16 * t + li, a.n - 1);
        wrow[t] = a.w + n * a.k;
        sw[t] = a.ws + (min(n0 + 16 * t, a.n - 1) >> 7) * a.scale_cols;
    }
#pragma unroll
    for (int t = 0; t < TB; ++t) {
        const int64_t m = min(m0 + 16 * t + li, a.m - 1);
        xrow[t] = a.x + m * a.k;
        sx[t] = a.xs + m * a.blocks;
    }
    const bool ragged = (a.k & 127) != 0;
    const int nk = wave < a.blocks ? (a.blocks - 1 - wave) / nw + 1 : 0;
    plm_f32x4 acc[TA][TB];
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j) acc[i][j] = plm_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    plm_u32x4 q[P][TA][2], x[P][TB][2];
    float s[P][TA], t[P][TB];
    auto issue = [&](int slot, int k) {
        const int64_t b = wave + static_cast<int64_t>(k) * nw;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            // past the end of a row: its last 16 bytes, cleared when used
            const int64_t off = min(b * 128 + 64 * h + 16 * qd, a.k - 16);
#pragma unroll
            for (int i = 0; i < TA; ++i) q[slot][i][h] = wload16(wrow[i] + off);
#pragma unroll
            for (int j = 0; j < TB; ++j) x[slot][j][h] = xload16(xrow[j] + off);
        }
#pragma unroll
        for (int i = 0; i < TA; ++i) s[slot][i] = sw[i][b];
#pragma unroll
        for (int j = 0; j < TB; ++j) t[slot][j] = sx[j][b];
    };
    auto compute = [&](int slot, int k) {
        const int64_t b = wave + static_cast<int64_t>(k) * nw;
        if (ragged) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool in = b * 128 + 64 * h + 16 * qd < a.k;
#pragma unroll
                for (int i = 0; i < TA; ++i) q[slot][i][h] = in ? q[slot][i][h] : plm_u32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < TB; ++j) x[slot][j][h] = in ? x[slot][j][h] : plm_u32x4{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int i = 0; i < TA; ++i)
#pragma unroll
            for (int j = 0; j < TB; ++j) {
                const plm_f32x4 d = mfma_fp8(q[slot][i][0], q[slot][i][1], x[slot][j][0], x[slot][j][1],
                                             plm_f32x4{0.0f, 0.0f, 0.0f, 0.0f});
                const float scale = s[slot][i] * t[slot][j];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[e], scale, acc[i][j][e]);
            }
    };
    run_pipelined<P>(nk, issue, compute);
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j) red[((wave * TA + i) * TB + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    // element e: weight row fastest (16 rows are adjacent in an output row)
    const float* rf = reinterpret_cast<const float*>(red);
    for (int e = threadIdx.x; e < TA * TB * 256; e += blockDim.x) {
        const int r = e & 15, c = (e >> 4) & 15, tile = e >> 8;
        const int i = tile % TA, j = tile / TA;
        const int64_t n = n0 + 16 * i + r, m = m0 + 16 * j + c;
        if (n >= a.n || m >= a.m) continue;
        const int at = ((i * TB + j) * 64 + (r >> 2) * 16 + c) * 4 + (r & 3);
        float v = 0.0f;
        for (int w = 0; w < nw; ++w) v += rf[w * TA * TB * 256 + at];
        store_out(a, m * a.n + n, v);
    }
}

template <int TA, int TB, int P, int MAXW>
int launch_rows(const MatmulArgs& a, int waves, hipStream_t st) {
    const int64_t gx = plm::ceil_div(a.n, 16 * TA), gy = plm::ceil_div(a.m, 16 * TB);
    if (gx > 0x7FFFFFFF || gy > 65535) return plm::fail(-2, "too many rows");
    const int bytes = waves * TA * TB * 1024;
    const void* fn = reinterpret_cast<const void*>(&fp8_matmul_rows_kernel<TA, TB, P, MAXW>);
    if (bytes > 64 * 1024) {
        const int code = plm::allow_large_lds(fn, MAXW * TA * TB * 1024);
        if (code != 0) return code;
    }
    hipLaunchKernelGGL((fp8_matmul_rows_kernel<TA, TB, P, MAXW>), dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy)),
                       dim3(static_cast<unsigned>(64 * waves)), static_cast<unsigned>(bytes), st, a);
    return plm::check_launch("fp8_e4m3_block_matmul");
}

}  // namespace

PLM_EXPORT int64_t fp8_e4m3_block_matmul_scratch_bytes(int64_t rows, int64_t out_rows, int64_t in_cols) {
    if (rows <= 0 || out_rows <= 0 || in_cols <= 0) return plm::fail(-2, "bad dimensions");
    return 0;
}

PLM_EXPORT int fp8_e4m3_block_matmul(const uint8_t* x, const float* x_scales, const uint8_t* fp8_weight,
                                     const float* scale_inv, void* out, void* scratch, int64_t scratch_bytes,
                                     int64_t rows, int64_t out_rows, int64_t in_cols, int64_t scale_cols,
                                     int dtype_code) {
    if (x == nullptr || x_scales == nullptr || fp8_weight == nullptr || scale_inv == nullptr || out == nullptr)
        return plm::fail(-1, "null pointer");
    const int64_t most = static_cast<int64_t>(1) << 31;
    if (rows <= 0 || out_rows <= 0 || in_cols <= 0 || rows >= most || out_rows >= most || in_cols >= most ||
        scale_cols < plm::ceil_div(in_cols, 128) || dtype_code < 0 || dtype_code > 2)
        return plm::fail(-2, "bad dimensions");
    const MatmulArgs a = {x,    x_scales, fp8_weight, scale_inv,  out,
                          rows, out_rows, in_cols,    scale_cols, static_cast<int>(plm::ceil_div(in_cols, 128)),
                          dtype_code};
    (void)scratch, (void)scratch_bytes;
    const hipStream_t st = plm::current_stream();
    if (in_cols % 16 != 0 || !plm::aligned16(x) || !plm::aligned16(fp8_weight)) {
        const int64_t groups = plm::ceil_div(rows * out_rows, 256);
        if (groups > 0x7FFFFFFF) return plm::fail(-2, "too many results");
        hipLaunchKernelGGL(fp8_matmul_scalar_kernel, dim3(static_cast<unsigned>(groups)), dim3(256), 0, st, a);
        return plm::check_launch("fp8_e4m3_block_matmul");
    }
    const int waves = std::min(8, a.blocks);
    if (rows <= 16) return launch_rows<1, 1, 4, 8>(a, waves, st);
    if (rows <= 32) return launch_rows<2, 2, 2, 8>(a, waves, st);
    return launch_rows<2, 4, 2, 8>(a, waves, st);
}
