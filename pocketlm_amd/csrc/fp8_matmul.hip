// Product of FP8 e4m3 activation rows (a scale for each 128 columns of a row)
// and an FP8 e4m3 block-scaled weight (a scale for each 128 x 128 block):
//
//   out[m][n] = sum_b sx[m][b] * sw[n / 128][b] * sum_{k in block b} x[m][k] * w[n][k]
//
// v_mfma_f32_16x16x128_f8f6f4 takes one block of 128 columns: its result is
// the block's inner sum, and the scaled sum over the blocks is kept in fp32 by
// vector fma.  NaN bytes, in the rows or in the weight, are NaN.
#include <algorithm>
#include <type_traits>

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

// Many rows: a workgroup owns 16 TN GN weight rows and 16 TM GM activation
// rows, wave (i, j) of GN x GM of them 16 TN by 16 TM.  Both operands' block
// of 128 columns goes to LDS by loads that write it there (no registers), the
// next block's while this one is multiplied; one barrier a block.
//
// A row's eight 16-byte pieces lie in LDS at piece ^ f(row), so that the
// eight lanes which read together (the same piece of eight rows) touch eight
// different groups of banks; the loads write LDS in lane order, so it is
// their addresses that are permuted.  Weight tile i of a wave holds the rows
// 16 (r / 4) + 4 i + r % 4: a lane then has 4 TN adjacent results of an
// output row.
template <int TN, int TM, int GN, int GM>
struct Tile {
    static constexpr int kWaves = GN * GM;
    static constexpr int kN = 16 * TN * GN, kM = 16 * TM * GM;
    static constexpr int kStage = (kN + kM) * 128;      // bytes of a block's operands
    static constexpr int kLds = 2 * kStage + 4 * kM * 4;  // and four blocks' row scales
};

// Eight results in the output's 16-bit type.
template <bool BF16>
__device__ __forceinline__ plm_u32x4 pack8(const plm_f32x4 a, const plm_f32x4 b) {
    typedef float f32x8 __attribute__((ext_vector_type(8)));
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    const f32x8 v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    if constexpr (BF16)
        return __builtin_bit_cast(plm_u32x4, __builtin_convertvector(v, plm_bf16x8));
    else
        return __builtin_bit_cast(plm_u32x4, __builtin_convertvector(v, f16x8));
}

template <int TN>
__device__ __forceinline__ int swizzle_w(int row) {
    return (row & 3) | ((row / (4 * TN)) & 1) << 2;
}
__device__ __forceinline__ int swizzle_x(int row) { return row & 7; }

// 16 bytes a lane from base + offset to LDS, the wave's KB in lane order at
// `to`.  Not the compiler's builtin: it waits for every load to LDS before any
// read of LDS, also of the other stage.  The wait is load_to_lds_wait's.
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :
                 : "v"(offset), "s"(base), "s"(to)
                 : "memory");
}
__device__ __forceinline__ void load4_to_lds(const void* base, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
                 :
                 : "v"(offset), "s"(base), "s"(to)
                 : "memory");
}
// Until all but the last LEFT of the wave's loads to LDS are there, then until
// the workgroup's waves are here.  One statement: no read of LDS moves in
// between.
template <int LEFT>
__device__ __forceinline__ void load_to_lds_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

template <int TN, int TM, int GN, int GM>
__global__ __launch_bounds__(64 * GN * GM) void fp8_matmul_tile_kernel(const MatmulArgs a) {
    using T = Tile<TN, TM, GN, GM>;
    extern __shared__ char lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, qd = lane >> 4;
    const int wn = wave % GN, wm = wave / GN;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * T::kN, m0 = static_cast<int64_t>(blockIdx.y) * T::kM;

    constexpr int kLag = 2;
    constexpr int kAtOnce = 2;
    constexpr int kScalesAt = TM - 1;
    // a wave's loads: 8 rows each, rows past the end repeat the last one
    constexpr int kLoads = (T::kN + T::kM) / 8 / T::kWaves;
    static_assert((T::kN + T::kM) % (8 * T::kWaves) == 0 && T::kN % (8 * T::kWaves) == 0, "whole loads");
    const uint8_t* wbase = a.w + n0 * a.k;
    const uint8_t* xbase = a.x + m0 * a.k;
    uint32_t src[kLoads];  // from the operand's first row of the workgroup
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int r = (i * T::kWaves + wave) * 8 + (lane >> 3);  // of both operands' rows
        const bool is_w = i < T::kN / 8 / T::kWaves;
        const int rr = is_w ? r : r - T::kN;
        const int f = is_w ? swizzle_w<TN>(rr) : swizzle_x(rr);
        const int last = static_cast<int>(min(is_w ? a.n - 1 - n0 : a.m - 1 - m0, static_cast<int64_t>(T::kN + T::kM)));
        src[i] = static_cast<uint32_t>(min(rr, last)) * static_cast<uint32_t>(a.k) + 16 * ((lane & 7) ^ f);
    }
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
    auto load_part = [&](int b, int i) {
        load_to_lds((i < T::kN / 8 / T::kWaves ? wbase : xbase) + static_cast<int64_t>(b) * 128, src[i],
                    lds_at + (b & 1) * T::kStage + (i * T::kWaves + wave) * 1024);
    };
    const float* scales = reinterpret_cast<const float*>(lds + 2 * T::kStage);
    const int sfirst = wave * 64 % T::kM;
    const float* xs = a.xs + m0 * a.blocks;
    const uint32_t ssrc = static_cast<uint32_t>(min(static_cast<int64_t>((sfirst + lane) % T::kM), a.m - 1 - m0)) * a.blocks * 4;
    const auto ws = (const __attribute__((address_space(4))) float*)(
        a.ws + (min(n0 + 16 * TN * wn, a.n - 1) >> 7) * a.scale_cols);

    plm_f32x4 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = plm_f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    const int wrow = 16 * TN * wn + 4 * TN * (li >> 2) + (li & 3);  // + 4 i
    const int xrow = 16 * TM * wm + li;                              // + 16 j
    const int fw = swizzle_w<TN>(wrow), fx = swizzle_x(xrow);
    const int w0 = wrow * 128 + 16 * (qd ^ fw), w1 = wrow * 128 + 16 * ((qd + 4) ^ fw);
    const int x0 = (T::kN + xrow) * 128 + 16 * (qd ^ fx), x1 = (T::kN + xrow) * 128 + 16 * ((qd + 4) ^ fx);

    auto load_scales = [&](int b) {
        load4_to_lds(xs + min(b, a.blocks - 1), ssrc, lds_at + 2 * T::kStage + ((b & 3) * T::kM + sfirst) * 4);
    };
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_part(0, i);
    load_scales(0);
    load_scales(1);
    float sw = ws[0];
    auto block = [&](int b, auto more, auto masked) {
        constexpr bool MORE = decltype(more)::value, MASKED = decltype(masked)::value;
        load_to_lds_barrier<MORE ? 1 : 0>();
        const float next_w = ws[min(b + 1, a.blocks - 1)];
        const char* stage = lds + (b & 1) * T::kStage;
        const float* sx = scales + (b & 3) * T::kM + xrow;
        auto piece = [&](int at, int h) {
            plm_u32x4 v = *reinterpret_cast<const plm_u32x4*>(stage + at);
            if constexpr (MASKED) {  // columns past the end
                if (static_cast<int64_t>(b) * 128 + 64 * h + 16 * qd >= a.k) v = plm_u32x4{0, 0, 0, 0};
            }
            return v;
        };
        plm_u32x4 w[TN][2];
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            w[i][0] = piece(w0 + i * 512, 0);
            w[i][1] = piece(w1 + i * 512, 1);
        }
        plm_u32x4 v[2][2];
        plm_f32x4 d[kLag + 1];
        float scale[2];
        v[0][0] = piece(x0, 0);
        v[0][1] = piece(x1, 1);
        scale[0] = sx[0] * sw;
        // the adds of a result follow the matrix instruction kLag later
#pragma unroll
        for (int at = 0; at < TN * TM + kLag; ++at) {
            const int i = at % TN, j = at / TN;
            // the next block's loads go out one at a time: all at once they wait for each other before the
            // first product
            if (MORE && i == 0) {
#pragma unroll
                for (int x = kAtOnce * j; x < min(kLoads, kAtOnce * (j + 1)); ++x) load_part(b + 1, x);
                if (j == kScalesAt) load_scales(b + 2);
            }
            if (i == 0 && j + 1 < TM) {
                v[(j + 1) & 1][0] = piece(x0 + (j + 1) * 2048, 0);
                v[(j + 1) & 1][1] = piece(x1 + (j + 1) * 2048, 1);
            }
            if (j < TM)
                d[at % (kLag + 1)] =
                    mfma_fp8(w[i][0], w[i][1], v[j & 1][0], v[j & 1][1], plm_f32x4{0.0f, 0.0f, 0.0f, 0.0f});
            if (at >= kLag) {
                const int was = at - kLag, wi = was % TN, wj = was / TN;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[wi][wj][e] = fmaf(d[was % (kLag + 1)][e], scale[wj & 1], acc[wi][wj][e]);
                if (wi == TN - 1 && wj + 1 < TM) scale[(wj + 1) & 1] = sx[16 * (wj + 1)] * sw;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        // the adds stay in their block: moved past a branch, all results would wait for them in registers
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) asm volatile("" : "+v"(acc[i][j]));
        sw = next_w;
    };
    for (int b = 0; b + 1 < a.blocks; ++b) block(b, std::true_type{}, std::false_type{});
    block(a.blocks - 1, std::false_type{}, std::true_type{});

    // A lane has 4 TN adjacent results of TM rows.  Whole ones of aligned rows
    // are stored by 16 bytes, others by single values through LDS.
    const int64_t n = n0 + 16 * TN * wn + 4 * TN * qd;
    const int per = a.out_type == kOutF32 ? 4 : 8;
    const bool wide = a.n % per == 0 && n0 + T::kN <= a.n && (reinterpret_cast<uintptr_t>(a.out) & 15u) == 0;
    if (wide) {
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            const int64_t m = m0 + 16 * TM * wm + 16 * j + li;
            if (m >= a.m) continue;
            const int64_t at = m * a.n + n;
            if (a.out_type == kOutF32) {
#pragma unroll
                for (int i = 0; i < TN; ++i) *reinterpret_cast<plm_f32x4*>(static_cast<float*>(a.out) + at + 4 * i) = acc[i][j];
            } else if (a.out_type == kOutBF16) {
#pragma unroll
                for (int i = 0; i < TN; i += 2)
                    *reinterpret_cast<plm_u32x4*>(static_cast<uint16_t*>(a.out) + at + 4 * i) =
                        pack8<true>(acc[i][j], acc[i + 1][j]);
            } else {
#pragma unroll
                for (int i = 0; i < TN; i += 2)
                    *reinterpret_cast<plm_u32x4*>(static_cast<uint16_t*>(a.out) + at + 4 * i) =
                        pack8<false>(acc[i][j], acc[i + 1][j]);
            }
        }
        return;
    }
    __syncthreads();
    constexpr int kRow = 16 * TN;
    plm_f32x4* mine = reinterpret_cast<plm_f32x4*>(lds) + wave * 16 * (kRow / 4);
#pragma unroll
    for (int j = 0; j < TM; ++j) {
#pragma unroll
        for (int i = 0; i < TN; ++i) mine[li * (kRow / 4) + TN * qd + i] = acc[i][j];
        // the wave's own: its LDS operations are done in order
        __builtin_amdgcn_wave_barrier();
        for (int e = lane; e < 16 * kRow; e += 64) {
            const int64_t m = m0 + 16 * TM * wm + 16 * j + e / kRow, c = n0 + 16 * TN * wn + e % kRow;
            if (m < a.m && c < a.n) store_out(a, m * a.n + c, reinterpret_cast<const float*>(mine)[e]);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <int TN, int TM, int GN, int GM>
int launch_tile(const MatmulArgs& a, hipStream_t st) {
    using T = Tile<TN, TM, GN, GM>;
    const int64_t gx = plm::ceil_div(a.n, T::kN), gy = plm::ceil_div(a.m, T::kM);
    if (gx > 0x7FFFFFFF || gy > 65535) return plm::fail(-2, "too many rows");
    const void* fn = reinterpret_cast<const void*>(&fp8_matmul_tile_kernel<TN, TM, GN, GM>);
    const int code = plm::allow_large_lds(fn, T::kLds);
    if (code != 0) return code;
    hipLaunchKernelGGL((fp8_matmul_tile_kernel<TN, TM, GN, GM>), dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy)),
                       dim3(64 * T::kWaves), T::kLds, st, a);
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
    if (rows <= 64) return launch_rows<2, 4, 2, 8>(a, waves, st);
    return launch_tile<4, 8, 4, 2>(a, st);
}
