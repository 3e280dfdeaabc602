// Activation rows in FP8 e4m3 with one fp32 scale for each 128 columns, the
// left operand of fp8_e4m3_block_matmul: from rows as they are
// (fp8_e4m3_quantize_rows), or from the RMS norm of rows, a residual added
// first (fp8_e4m3_rms_norm_rows).
//
//   sum = T(x + residual)                       T: the rows' type, to nearest even
//   y   = sum * rsqrt(mean(sum^2) + eps) * w    fp32, as the dense layer's norms; sums of squares
//                                               that leave fp32's range in 64 bits
//   s_b = max(max |y| over block b / 448, 2^-126)
//   q   = e4m3(y / s_b)                         to nearest even
//
// The scale's lower bound keeps 1 / s_b finite (a block of zeros gets 2^-126
// and zero bytes).  A block that holds an infinity or a NaN gets the scale NaN
// and the bytes 0x7F, so the product's row is NaN.
#include "common.h"

namespace {

enum Dtype { kF16 = 0, kBF16 = 1, kF32 = 2 };

constexpr int kPiece = 8;              // columns a thread takes at a time
constexpr int kMaxThreads = 1024;
constexpr int kMaxSteps = 8;           // pieces a thread keeps in registers
constexpr int64_t kMaxCols = static_cast<int64_t>(kMaxThreads) * kMaxSteps * kPiece;
constexpr float kE4m3Max = 448.0f;
constexpr float kSmallestScale = 1.17549435e-38f;  // 2^-126

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <int DT>
struct Row;
template <>
struct Row<kF16> {
    using T = _Float16;
    using V = f16x8;
};
template <>
struct Row<kBF16> {
    using T = __bf16;
    using V = bf16x8;
};
template <>
struct Row<kF32> {
    using T = float;
    using V = f32x8;
};

struct RowsArgs {
    const void* x;
    const void* residual;
    const void* weight;
    uint8_t* out;
    float* scales;
    void* sum;
    int64_t rows;
    int64_t cols;
    int64_t x_stride;
    int64_t residual_stride;
    int blocks;          // scales per row
    int waves;           // per row
    int rows_per;        // rows of a workgroup
    int vec;             // whole pieces, 16-byte aligned rows
    float eps;
};

// Piece c of a row; columns past the row's end are zero.
template <int DT>
__device__ __forceinline__ f32x8 load_piece(const void* row, int64_t c, int64_t cols, bool vec) {
    using T = typename Row<DT>::T;
    const T* p = static_cast<const T*>(row) + c * kPiece;
    f32x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
    if (vec) {
        if constexpr (DT == kF32) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
        } else {
            v = __builtin_convertvector(*reinterpret_cast<const typename Row<DT>::V*>(p), f32x8);
        }
        return v;
    }
#pragma unroll
    for (int i = 0; i < kPiece; ++i)
        if (c * kPiece + i < cols) v[i] = static_cast<float>(p[i]);
    return v;
}

template <int DT>
__device__ __forceinline__ void store_piece(void* row, int64_t c, int64_t cols, bool vec, const f32x8 v) {
    using T = typename Row<DT>::T;
    T* p = static_cast<T*>(row) + c * kPiece;
    if (vec) {
        if constexpr (DT == kF32) {
            *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
        } else {
            *reinterpret_cast<typename Row<DT>::V*>(p) = __builtin_convertvector(v, typename Row<DT>::V);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kPiece; ++i)
        if (c * kPiece + i < cols) p[i] = static_cast<T>(v[i]);
}

// The value rounded to the rows' type.
template <int DT>
__device__ __forceinline__ f32x8 rounded(f32x8 v) {
    if constexpr (DT == kF32)
        return v;
    else
        return __builtin_convertvector(__builtin_convertvector(v, typename Row<DT>::V), f32x8);
}

__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    // over the 16 lanes that hold a 128-column block
#define PLM_ROW_MAX(ctrl) \
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), ctrl, 0xF, 0xF, false)))
    PLM_ROW_MAX(0xB1);
    PLM_ROW_MAX(0x4E);
    PLM_ROW_MAX(0x141);
    PLM_ROW_MAX(0x140);
#undef PLM_ROW_MAX
    return v;
}

// plm_wave_sum in 64 bits; every lane has it.
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off);
    return v;
}

// Whether a row's sum of squares has left fp32: the squares of finite values
// pass its largest number from 2^64 on, and below 2^-63 they lose bits, which
// counts where rms_eps is tiny too.  Such rows are summed again in 64 bits
// (one with an infinity or a NaN comes out as it went in); the others keep the
// fp32 sum's bits and time (one row of 7168 bf16 3.98 us, 509 rows of 3584 4.75;
// with all sums in 64 bits 4.16 and 4.87).
__device__ __forceinline__ bool beyond(float total, const RowsArgs& a) {
    return !(total < 0x1p127f) || total + a.eps * static_cast<float>(a.cols) < 0x1p-80f;
}

__device__ __forceinline__ int pack4(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

// y / scale: the reciprocal's product and one correction by its remainder, so
// that the value that is rounded to e4m3 has been rounded once (values on a
// border between two e4m3 values are common where both operands are 16-bit).
__device__ __forceinline__ float quotient(float y, float scale, float inv) {
    const float q = y * inv;
    return fmaf(fmaf(-q, scale, y), inv, q);
}

// Quantizes the piece of block c / 16 that the 16 lanes of a DPP row hold.
__device__ __forceinline__ void quantize_piece(const RowsArgs& a, int64_t row, int64_t c, const f32x8 y) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kPiece; ++i) m = max(m, __float_as_uint(y[i]) & 0x7FFFFFFFu);
    m = dpp_max(m);
    const bool finite = m < 0x7F800000u;
    const float scale = finite ? fmaxf(__uint_as_float(m) / kE4m3Max, kSmallestScale) : __uint_as_float(0x7FC00000u);
    const float inv = 1.0f / scale;
    if (c * kPiece >= a.cols) return;
    if ((c & 15) == 0) a.scales[row * a.blocks + (c >> 4)] = scale;
    int lo = 0x7F7F7F7F, hi = 0x7F7F7F7F;
    if (finite) {
        float q[kPiece];
#pragma unroll
        for (int i = 0; i < kPiece; ++i) q[i] = quotient(y[i], scale, inv);
        lo = pack4(q[0], q[1], q[2], q[3]);
        hi = pack4(q[4], q[5], q[6], q[7]);
    }
    uint8_t* p = a.out + row * a.cols + c * kPiece;
    if (a.vec) {
        *reinterpret_cast<int2*>(p) = make_int2(lo, hi);
        return;
    }
#pragma unroll
    for (int i = 0; i < kPiece; ++i)
        if (c * kPiece + i < a.cols) p[i] = static_cast<uint8_t>((i < 4 ? lo : hi) >> (8 * (i & 3)));
}

// `waves` waves per row, several rows a workgroup where a row is short; a
// thread keeps its NS pieces of the sum in registers between the two passes,
// so every value is read once (8 pieces, rows above 32768 columns, spill).
// Bound by memory: 8192 x 7168 bf16 with a residual 80 us, 5.2 TB/s.  One row
// of 7168, 3.6 us, and 509 rows of 3584, 5.3 us, are the launch, a trip to
// memory and the workgroup's sum.
template <int DT, int NS, bool NORM>
__global__ __launch_bounds__(kMaxThreads) void fp8_rows_kernel(const RowsArgs a) {
    using T = typename Row<DT>::T;
    __shared__ float red[kMaxThreads / 64];
    __shared__ double red64[kMaxThreads / 64];
    const int wave = threadIdx.x >> 6;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * a.rows_per + wave / a.waves;
    const int t = threadIdx.x - wave / a.waves * a.waves * 64;
    const int step = a.waves * 64;
    const bool live = row < a.rows;
    const bool vec = a.vec != 0;
    f32x8 h[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int64_t c = t + static_cast<int64_t>(i) * step;
        h[i] = f32x8{0, 0, 0, 0, 0, 0, 0, 0};
        if (live && c * kPiece < a.cols)
            h[i] = load_piece<DT>(static_cast<const T*>(a.x) + row * a.x_stride, c, a.cols, vec);
    }
    if constexpr (NORM) {
        if (a.residual != nullptr) {
            f32x8 r[NS];
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const int64_t c = t + static_cast<int64_t>(i) * step;
                r[i] = f32x8{0, 0, 0, 0, 0, 0, 0, 0};
                if (live && c * kPiece < a.cols)
                    r[i] = load_piece<DT>(static_cast<const T*>(a.residual) + row * a.residual_stride, c, a.cols, vec);
            }
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const int64_t c = t + static_cast<int64_t>(i) * step;
                h[i] = rounded<DT>(h[i] + r[i]);
                if (live && c * kPiece < a.cols) store_piece<DT>(static_cast<T*>(a.sum) + row * a.cols, c, a.cols, vec, h[i]);
            }
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int j = 0; j < kPiece; ++j) s = fmaf(h[i][j], h[i][j], s);
        s = plm_wave_sum(s);
        float total = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, s), kSumLane));
        const int own = wave / a.waves;  // of the workgroup's rows
        bool far = false;                // one of them, where they share barriers
        if (a.waves > 1) {
            if ((threadIdx.x & 63) == 0) red[wave] = total;
            __syncthreads();
            for (int r = 0; r < a.rows_per; ++r) {
                float all = 0.0f;
                for (int w = 0; w < a.waves; ++w) all += red[r * a.waves + w];
                far |= beyond(all, a);
                if (r == own) total = all;
            }
        } else {
            far = beyond(total, a);
        }
        float scale = 1.0f / sqrtf(total / static_cast<float>(a.cols) + a.eps);
        if (__builtin_expect(far, 0)) {
            double wide = 0.0;
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int j = 0; j < kPiece; ++j) {
                    const double v = h[i][j];
                    wide = fma(v, v, wide);
                }
            wide = wave_sum64(wide);
            if (a.waves > 1) {
                if ((threadIdx.x & 63) == 0) red64[wave] = wide;
                __syncthreads();
                wide = 0.0;
                for (int w = 0; w < a.waves; ++w) wide += red64[own * a.waves + w];
            }
            if (beyond(total, a)) {
                // the root's power of two goes to the values, which it leaves exact, so that both stay in range
                const double mean = wide / static_cast<double>(a.cols) + static_cast<double>(a.eps);
                const int half = -(__builtin_amdgcn_frexp_exp(mean) >> 1);
                scale = 1.0f / sqrtf(static_cast<float>(__builtin_ldexp(mean, 2 * half)));
#pragma unroll
                for (int i = 0; i < NS; ++i)
#pragma unroll
                    for (int j = 0; j < kPiece; ++j) h[i][j] = ldexpf(h[i][j], half);
            }
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int64_t c = t + static_cast<int64_t>(i) * step;
            if (c * kPiece < a.cols) h[i] = h[i] * scale * load_piece<DT>(a.weight, c, a.cols, vec);
        }
    }
    if (!live) return;  // a whole wave
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int64_t c = t + static_cast<int64_t>(i) * step;
        if (static_cast<int64_t>(i) * step * kPiece < a.cols) quantize_piece(a, row, c, h[i]);
    }
}

template <int DT, int NS>
void launch(const RowsArgs& a, bool norm, dim3 grid, dim3 block, hipStream_t st) {
    if (norm)
        hipLaunchKernelGGL((fp8_rows_kernel<DT, NS, true>), grid, block, 0, st, a);
    else
        hipLaunchKernelGGL((fp8_rows_kernel<DT, NS, false>), grid, block, 0, st, a);
}

template <int DT>
void launch_steps(const RowsArgs& a, int steps, bool norm, dim3 grid, dim3 block, hipStream_t st) {
    if (steps <= 1)
        launch<DT, 1>(a, norm, grid, block, st);
    else if (steps <= 2)
        launch<DT, 2>(a, norm, grid, block, st);
    else if (steps <= 4)
        launch<DT, 4>(a, norm, grid, block, st);
    else
        launch<DT, kMaxSteps>(a, norm, grid, block, st);
}

int run_rows(RowsArgs& a, int dtype_code, bool norm) {
    const int64_t pieces = plm::ceil_div(a.cols, kPiece);
    a.blocks = static_cast<int>(plm::ceil_div(a.cols, 128));
    const int size = dtype_code == kF32 ? 4 : 2;
    auto whole = [&](const void* p, int64_t stride) {
        return p == nullptr || (plm::aligned16(p) && stride * size % 16 == 0);
    };
    a.vec = a.cols % kPiece == 0 && whole(a.x, a.x_stride) && whole(a.residual, a.residual_stride) &&
            whole(a.weight, 0) && whole(a.sum, a.cols) && (reinterpret_cast<uintptr_t>(a.out) & 7u) == 0;
    const bool few = a.rows <= 2 * plm::cu_count();
    int steps = few ? 1 : 2;  // 8192 x 7168 bf16: 1 93 us, 2 79 (5.2 TB/s), 4 102
    while (plm::ceil_div(pieces, steps) > kMaxThreads) steps *= 2;
    while (steps > 1 && pieces <= static_cast<int64_t>(64) * (steps / 2)) steps /= 2;
    a.waves = static_cast<int>(plm::ceil_div(plm::ceil_div(pieces, steps), 64));
    a.rows_per = few ? 1 : (a.waves >= 4 ? 1 : 4 / a.waves);
    const int64_t groups = plm::ceil_div(a.rows, a.rows_per);
    if (groups > 0x7FFFFFFF) return plm::fail(-2, "too many rows");
    const dim3 grid(static_cast<unsigned>(groups)), block(static_cast<unsigned>(64 * a.waves * a.rows_per));
    const hipStream_t st = plm::current_stream();
    if (dtype_code == kF16)
        launch_steps<kF16>(a, steps, norm, grid, block, st);
    else if (dtype_code == kBF16)
        launch_steps<kBF16>(a, steps, norm, grid, block, st);
    else
        launch_steps<kF32>(a, steps, norm, grid, block, st);
    return plm::check_launch(norm ? "fp8_e4m3_rms_norm_rows" : "fp8_e4m3_quantize_rows");
}

bool bad_sizes(int64_t rows, int64_t cols, int64_t stride, int dtype_code) {
    return rows <= 0 || cols <= 0 || cols > kMaxCols || stride < 0 || dtype_code < 0 || dtype_code > 2;
}

}  // namespace

PLM_EXPORT int fp8_e4m3_quantize_rows(const void* x, uint8_t* out_fp8, float* out_scales, int64_t rows, int64_t cols,
                                      int64_t x_stride, int dtype_code) {
    if (x == nullptr || out_fp8 == nullptr || out_scales == nullptr) return plm::fail(-1, "null pointer");
    if (bad_sizes(rows, cols, x_stride, dtype_code)) return plm::fail(-2, "bad dimensions");
    RowsArgs a = {};
    a.x = x;
    a.out = out_fp8;
    a.scales = out_scales;
    a.rows = rows;
    a.cols = cols;
    a.x_stride = x_stride;
    return run_rows(a, dtype_code, false);
}

PLM_EXPORT int fp8_e4m3_rms_norm_rows(const void* x, const void* residual, const void* weight, void* out_sum,
                                      uint8_t* out_fp8, float* out_scales, int64_t rows, int64_t cols,
                                      int64_t x_stride, int64_t residual_stride, int dtype_code, float rms_eps) {
    if (x == nullptr || weight == nullptr || out_fp8 == nullptr || out_scales == nullptr ||
        (residual != nullptr && out_sum == nullptr))
        return plm::fail(-1, "null pointer");
    if (bad_sizes(rows, cols, x_stride, dtype_code) || (residual != nullptr && residual_stride < 0))
        return plm::fail(-2, "bad dimensions");
    RowsArgs a = {};
    a.x = x;
    a.residual = residual;
    a.weight = weight;
    a.sum = residual != nullptr ? out_sum : nullptr;
    a.out = out_fp8;
    a.scales = out_scales;
    a.rows = rows;
    a.cols = cols;
    a.x_stride = x_stride;
    a.residual_stride = residual_stride;
    a.eps = rms_eps;
    return run_rows(a, dtype_code, true);
}
