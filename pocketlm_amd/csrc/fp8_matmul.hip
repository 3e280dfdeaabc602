// Product of FP8 e4m3 activation rows (a scale for each 128 columns of a row)
// and an FP8 e4m3 block-scaled weight (a scale for each 128 x 128 block):
//
//   out[m][n] = sum_b sx[m][b] * sw[n / 128][b] * sum_{k in block b} x[m][k] * w[n][k]
//
// v_mfma_f32_16x16x128_f8f6f4 takes one block of 128 columns: its result is
// the block's inner sum, and the scaled sum over the blocks is kept in fp32 by
// vector fma.  NaN bytes, in the rows or in the weight, are NaN.
//
// That instruction adds eight products of adjacent columns at a time and cuts
// each off (towards zero) below 2^-13 of the largest one's power of two; the
// sums of the eights are fp32 (probed; the other e4m3 instructions do the
// same).  A result is off by 1.4e-5 of the results' size on normal values, by
// at most 7 2^-13 of each eight's largest product: taken where the output is
// rounded to 16 bits (2^-8 or 2^-11 of it).  fp32 results come from bf16
// products of the same values (EXACT): every e4m3 value is a bf16 value, and
// v_mfma_f32_16x16x32_bf16 leaves 7e-9 of the results' size.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "fp8_mfma.h"

namespace {

using namespace plm_fp8;

enum OutType { kOutF16 = 0, kOutBF16 = 1, kOutF32 = 2 };

typedef int plm_i32x8 __attribute__((ext_vector_type(8)));
// stored at the alignment of one value
typedef plm_f32x4 any_f32x4 __attribute__((aligned(4)));
typedef plm_u32x4 any_u32x4 __attribute__((aligned(2)));
typedef uint32_t any_u32x2 __attribute__((ext_vector_type(2), aligned(2)));

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
    float* part;
};

__device__ __forceinline__ void store_out(const MatmulArgs& a, int64_t at, float v) {
    if (a.out_type == kOutBF16)
        static_cast<__bf16*>(a.out)[at] = static_cast<__bf16>(v);
    else if (a.out_type == kOutF16)
        static_cast<_Float16*>(a.out)[at] = static_cast<_Float16>(v);
    else
        static_cast<float*>(a.out)[at] = v;
}

// Rows of k bytes to rows of k16, k up to a multiple of 16, zeros behind: the
// other kernels read whole 16-byte pieces.  A thread: one piece.
__global__ __launch_bounds__(256) void fp8_pad_rows_kernel(const uint8_t* __restrict__ from, uint8_t* __restrict__ to,
                                                           int64_t rows, int64_t k, int64_t k16) {
    const int64_t per = k16 / 16;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (at >= rows * per) return;
    const int64_t row = at / per, c = (at - row * per) * 16;
    const uint8_t* src = from + row * k + c;
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (c + i < k) v[i >> 2] |= static_cast<uint32_t>(src[i]) << (8 * (i & 3));
    *reinterpret_cast<uint4*>(to + row * k16 + c) = make_uint4(v[0], v[1], v[2], v[3]);
}

int pad_rows(const uint8_t* from, uint8_t* to, int64_t rows, int64_t k, int64_t k16, hipStream_t st) {
    const int64_t groups = plm::ceil_div(rows * (k16 / 16), 256);
    if (groups > 0x7FFFFFFF) return plm::fail(-2, "too many rows");
    hipLaunchKernelGGL(fp8_pad_rows_kernel, dim3(static_cast<unsigned>(groups)), dim3(256), 0, st, from, to, rows, k, k16);
    return plm::check_launch("fp8_e4m3_block_matmul, pad");
}

// A lane's 32 bytes of a block of an operand's row, as the matrix cores take
// them.
template <bool EXACT>
struct Operand {
    plm_i32x8 v;
    Operand() = default;
    __device__ __forceinline__ Operand(const plm_u32x4 a, const plm_u32x4 b)
        : v{static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w),
            static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w)} {}
};
template <>
struct Operand<true> {
    plm_bf16x8 v[4];
    Operand() = default;
    __device__ __forceinline__ Operand(const plm_u32x4 a, const plm_u32x4 b) {
        weights_to_bf16(a, v[0], v[1]);
        weights_to_bf16(b, v[2], v[3]);
    }
};

__device__ __forceinline__ plm_f32x4 block_sums(const Operand<false>& a, const Operand<false>& b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, plm_f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ plm_f32x4 block_sums(const Operand<true>& a, const Operand<true>& b) {
    plm_f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) d = mfma_bf16(a.v[i], b.v[i], d);
    return d;
}

// Few rows: a workgroup owns 16 TA weight rows and 16 TB activation rows; its
// waves take the K blocks w, w + nw, ... and their sums meet in LDS, added in
// wave order.  Lane l holds, of weight row (activation row) l & 15, the bytes
// 16 (l >> 4) .. + 15 of each half of a block: the same columns on both
// sides, which is all that the inner sum needs.  Operands go straight to
// registers, P blocks ahead once a wave's blocks beyond a multiple of P have
// gone one at a time; bound by the latency of the few loads a wave has (1 x 576
// x 7168 6.6 us, of whose 7 blocks a wave 3 go alone; 1 x 4096 x 4096 5.9).
template <int TA, int TB, int P, int MAXW, bool EXACT>
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
        Operand<EXACT> wo[TA];
#pragma unroll
        for (int i = 0; i < TA; ++i) wo[i] = Operand<EXACT>(q[slot][i][0], q[slot][i][1]);
#pragma unroll
        for (int j = 0; j < TB; ++j) {
            const Operand<EXACT> xo(x[slot][j][0], x[slot][j][1]);
#pragma unroll
            for (int i = 0; i < TA; ++i) {
                const plm_f32x4 d = block_sums(wo[i], xo);
                const float scale = s[slot][i] * t[slot][j];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[e], scale, acc[i][j][e]);
            }
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

template <int TA, int TB, int P, int MAXW, bool EXACT>
int launch_rows(const MatmulArgs& a, int waves, hipStream_t st) {
    const int64_t gx = plm::ceil_div(a.n, 16 * TA), gy = plm::ceil_div(a.m, 16 * TB);
    if (gx > 0x7FFFFFFF || gy > 65535) return plm::fail(-2, "too many rows");
    static_assert(MAXW * TA * TB * 1024 <= 64 * 1024, "LDS that needs no leave");
    const int bytes = waves * TA * TB * 1024;
    const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy)), block(static_cast<unsigned>(64 * waves));
    hipLaunchKernelGGL((fp8_matmul_rows_kernel<TA, TB, P, MAXW, EXACT>), grid, block, static_cast<unsigned>(bytes), st, a);
    return plm::check_launch("fp8_e4m3_block_matmul");
}

// Many rows: a workgroup owns 16 TN GN weight rows and 16 TM GM activation
// rows, wave (i, j) of GN x GM of them 16 TN by 16 TM.  Both operands' blocks
// of 128 columns go to LDS by loads that write it there (no registers), S - 1
// blocks ahead; one barrier a block.  blockIdx.z takes a share of the blocks;
// where there are several, their sums go to `part` in fp32 and
// fp8_matmul_join_kernel adds them.
//
// A row's eight 16-byte pieces lie in LDS at piece ^ f(row), so that the
// eight lanes which read together (the same piece of eight rows) touch eight
// different groups of banks; the loads write LDS in lane order, so it is
// their addresses that are permuted.  Weight tile i of a wave holds the rows
// 4 TN (r / 4) + 4 i + r % 4: a lane then has 4 TN adjacent results of an
// output row.
//
// Bound by the weight's bytes up to 64 rows (64 x 7168 x 16384 31.8 us with
// the join, 3.8 TB/s: every workgroup also reads its 64 rows, half as many
// bytes again, through the same cache) and by the matrix cores from 256 x 256
// tiles on: 4096 x 7168 x 16384 420 us, 2290 TFLOP/s, of which 448 tiles on 256
// compute units leave an eighth unused.
template <int TN, int TM, int GN, int GM, int S>
struct Tile {
    static constexpr int kWaves = GN * GM;
    static constexpr int kN = 16 * TN * GN, kM = 16 * TM * GM;
    static constexpr int kStage = (kN + kM) * 128;  // bytes of a block's operands
    static constexpr int kScales = kM / kWaves;        // of a block's row scales, a wave's
    static constexpr int kScaleSlots = S < 4 ? 4 : 8;  // of kM row scales: more than S blocks ahead
    static constexpr int kLds = S * kStage + kScaleSlots * kM * 4;
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

// These loads take the LDS address from M0, which the compiler has to know as
// written (it warns of any reserved register that is named so).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 16 bytes a lane from base + offset to LDS, the wave's KB in lane order at
// `to`; ONCE: past the caches.  Not the compiler's builtin: it waits for every
// load to LDS before any read of LDS, also of the other stage.  The wait is
// load_to_lds_barrier's.
template <bool ONCE>
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t offset, uint32_t to) {
    if constexpr (ONCE)
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt"
                     :
                     : "v"(offset), "s"(base), "s"(to)
                     : "m0", "memory");
    else
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                     :
                     : "v"(offset), "s"(base), "s"(to)
                     : "m0", "memory");
}
// Four bytes each of the first LANES lanes.  All lanes are active before and after.
template <int LANES>
__device__ __forceinline__ void load4_to_lds(const void* base, uint32_t offset, uint32_t to) {
    static_assert(LANES < 64, "a mask of 64 bits");
    asm volatile("s_mov_b32 m0, %2\n\ts_mov_b64 exec, %3\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1\n\t"
                 "s_mov_b64 exec, -1"
                 :
                 : "v"(offset), "s"(base), "s"(to), "s"((1ull << LANES) - 1)
                 : "m0", "memory");
}
#pragma clang diagnostic pop
// Until all but the last LEFT of the wave's loads to LDS are there, then until
// the workgroup's waves are here.  One statement: no read of LDS moves in
// between.
template <int LEFT>
__device__ __forceinline__ void load_to_lds_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

template <int TN, int TM, int GN, int GM, int S, bool EXACT, bool ONCE>
__global__ __launch_bounds__(64 * GN * GM) void fp8_matmul_tile_kernel(const MatmulArgs a) {
    using T = Tile<TN, TM, GN, GM, S>;
    extern __shared__ char lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, qd = lane >> 4;
    const int wn = wave % GN, wm = wave / GN;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * T::kN, m0 = static_cast<int64_t>(blockIdx.y) * T::kM;

    // this workgroup's blocks
    const int first = static_cast<int>(static_cast<int64_t>(a.blocks) * blockIdx.z / gridDim.z);
    const int blocks = static_cast<int>(static_cast<int64_t>(a.blocks) * (blockIdx.z + 1) / gridDim.z) - first;
    // Rows a multiple of 4096 bytes apart meet in the same memory channels: there each workgroup starts
    // at another of its blocks (16 x 7168 x 16384 33.5 -> 27.1 us, 64 rows 39.8 -> 36.4 when this was
    // tried; with more rows the activations are shared at one block, and 256 rows were 5 % slower).
    const int turn = T::kM <= 64 && gridDim.y == 1 && (a.k & 4095) == 0 ? static_cast<int>(blockIdx.x % blocks) : 0;
    auto turned = [&](int b) { return b + turn >= blocks ? b + turn - blocks : b + turn; };

    constexpr int kLag = 2;  // matrix instructions between a result and its adds
    // A wave's loads of a block: 8 rows each, LW of the weight's and LX of the activations' (of few
    // rows several waves load the same ones).  Rows past the end repeat the last one.
    constexpr int LW = T::kN / 8 / T::kWaves, LX = T::kM / 8 >= T::kWaves ? T::kM / 8 / T::kWaves : 1, L = LW + LX;
    static_assert(T::kN % (8 * T::kWaves) == 0 && (T::kM % (8 * T::kWaves) == 0 || T::kWaves * 8 % T::kM == 0),
                  "whole loads");
    static_assert(T::kWaves % TN == 0, "rows of an operand's loads share their piece");
    const uint8_t* wbase = a.w + n0 * a.k + static_cast<int64_t>(first) * 128;
    const uint8_t* xbase = a.x + m0 * a.k + static_cast<int64_t>(first) * 128;
    uint32_t src[L];  // from the operand's first row of the workgroup
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const bool is_w = i < LW;
        const int r = ((is_w ? i : i - LW) * T::kWaves + wave) * 8 % (is_w ? T::kN : T::kM) + (lane >> 3);
        const int f = is_w ? swizzle_w<TN>(r) : swizzle_x(r);
        const int64_t left = is_w ? a.n - 1 - n0 : a.m - 1 - m0;
        const int last = static_cast<int>(min(left, static_cast<int64_t>(T::kN + T::kM)));
        src[i] = static_cast<uint32_t>(min(r, last)) * static_cast<uint32_t>(a.k) + 16 * ((lane & 7) ^ f);
    }
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
    // in a last block of fewer columns the pieces past a row's end read its last one instead (the
    // columns are cleared when they are used); a lane's piece is the same in all loads of an operand
    const int64_t inside = a.k - 16 - static_cast<int64_t>(a.blocks - 1) * 128;
    auto past = [&](int f) {
        return static_cast<uint32_t>(max(static_cast<int64_t>(16 * ((lane & 7) ^ f)) - inside, static_cast<int64_t>(0)));
    };
    const uint32_t wpast = past(swizzle_w<TN>(wave * 8 + (lane >> 3))), xpast = past(swizzle_x(lane >> 3));
    auto load_part = [&](int b, int i) {
        const bool is_w = i < LW;
        const int from = turned(b);
        const uint32_t back = first + from + 1 < a.blocks ? 0u : is_w ? wpast : xpast;
        const int row = is_w ? (i * T::kWaves + wave) * 8 : T::kN + ((i - LW) * T::kWaves + wave) * 8 % T::kM;
        const uint32_t to = lds_at + b % S * T::kStage + row * 128;
        if (is_w)
            load_to_lds<ONCE>(wbase + static_cast<int64_t>(from) * 128, src[i] - back, to);
        else
            load_to_lds<false>(xbase + static_cast<int64_t>(from) * 128, src[i] - back, to);
    };
    const float* scales = reinterpret_cast<const float*>(lds + S * T::kStage);
    // Each wave its part of the rows' scales: they lie a row's blocks apart, so each is a cache line of its
    // own, and the lines are what the loads take (all of them by every wave: 64 x 7168 x 16384 36.9 us, now
    // 33.0; 1024 x 7168 x 7168 76, now 67).
    const int sfirst = wave * T::kScales;
    const float* xs = a.xs + m0 * a.blocks + first;
    const int64_t srow = min(static_cast<int64_t>(sfirst + lane % T::kScales), a.m - 1 - m0);
    const uint32_t ssrc = static_cast<uint32_t>(srow) * a.blocks * 4;
    auto load_scales = [&](int b) {
        load4_to_lds<T::kScales>(xs + turned(min(b, blocks - 1)), ssrc,
                                 lds_at + S * T::kStage + (b % T::kScaleSlots * T::kM + sfirst) * 4);
    };
    const auto ws = (const __attribute__((address_space(4))) float*)(
        a.ws + (min(n0 + 16 * TN * wn, a.n - 1) >> 7) * a.scale_cols + first);

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

    // In the order of their use: scales 0, block 0, scales 1, block 1, ..., scales S - 1.  Block b sends
    // block b + S - 1 and scales b + S, so behind its own operands S - 1 scales and S - 2 blocks are on
    // their way.
    load_scales(0);
    for (int b = 0; b < S - 1; ++b) {
        if (b < blocks) {
#pragma unroll
            for (int i = 0; i < L; ++i) load_part(b, i);
        }
        load_scales(b + 1);
    }
    float sw = ws[turned(0)];
    auto block = [&](int b, auto more, auto masked) {
        constexpr bool MORE = decltype(more)::value, MASKED = decltype(masked)::value;
        load_to_lds_barrier<MORE ? S - 1 + (S - 2) * L : 0>();
        float next_w = 0.0f;
        const char* stage = lds + b % S * T::kStage;
        const float* sx = scales + b % T::kScaleSlots * T::kM + xrow;
        auto piece = [&](int at, int h) {
            plm_u32x4 v = *reinterpret_cast<const plm_u32x4*>(stage + at);
            if constexpr (MASKED) {  // columns past the end
                if (static_cast<int64_t>(first + b) * 128 + 64 * h + 16 * qd >= a.k) v = plm_u32x4{0, 0, 0, 0};
            }
            return v;
        };
        Operand<EXACT> w[TN], v[2];
        plm_f32x4 d[kLag + 1];
        float raw[TM], scale = 0.0f;
        // What the first product takes is read first.  In the large tile a row tile's operands and scale are
        // read behind the first product of the one before it, and the weight's next scale, which no read of LDS
        // may wait beside, at the block's end (4096 x 7168 x 16384 440 us without this order, 419 with).
        w[0] = Operand<EXACT>(piece(w0, 0), piece(w1, 1));
        v[0] = Operand<EXACT>(piece(x0, 0), piece(x1, 1));
        raw[0] = sx[0];
        if constexpr (TN > 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 1; i < TN; ++i) w[i] = Operand<EXACT>(piece(w0 + i * 512, 0), piece(w1 + i * 512, 1));
        // the adds of a result follow the matrix instruction kLag later
#pragma unroll
        for (int at = 0; at < TN * TM + kLag; ++at) {
            const int i = at % TN, j = at / TN;
            // A later block's loads go out two at a time: all at once they hold up the first products
            // (4096 x 7168 x 16384 all at once 526 us, two 414, one 477 when this was tried).
            if (MORE && i == 0) {
                constexpr int kAtOnce = 2 * TM >= L ? 2 : L;
#pragma unroll
                for (int x = kAtOnce * j; x < min(L, kAtOnce * (j + 1)); ++x) load_part(b + S - 1, x);
                if (j == TM - 1) load_scales(b + S);
            }
            if (i == (TN > 2 ? 1 : 0) && j + 1 < TM) {
                v[(j + 1) & 1] = Operand<EXACT>(piece(x0 + (j + 1) * 2048, 0), piece(x1 + (j + 1) * 2048, 1));
                raw[j + 1] = sx[16 * (j + 1)];
            }
            if (at == TN * TM - 1) next_w = ws[turned(min(b + 1, blocks - 1))];
            if (j < TM) d[at % (kLag + 1)] = block_sums(w[i], v[j & 1]);
            if (at >= kLag) {
                const int was = at - kLag, wi = was % TN, wj = was / TN;
                if (wi == 0) scale = raw[wj] * sw;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[wi][wj][e] = fmaf(d[was % (kLag + 1)][e], scale, acc[wi][wj][e]);
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
    int b = 0;
    for (; b + S - 1 < blocks; ++b) block(b, std::true_type{}, std::false_type{});
    for (; b < blocks; ++b) block(b, std::false_type{}, std::true_type{});

    // A lane has 4 TN adjacent results of TM rows, stored by 16 bytes (rows need no alignment: such
    // stores may start at any value) up to the last columns.
    const int64_t n = n0 + 16 * TN * wn + 4 * TN * qd;
    if (gridDim.z > 1) {  // a.part [share][m][n4], n4 the columns up to a multiple of 4
        const int64_t n4 = (a.n + 3) & ~static_cast<int64_t>(3);
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            const int64_t m = m0 + 16 * TM * wm + 16 * j + li;
#pragma unroll
            for (int i = 0; i < TN; ++i)
                if (m < a.m && n + 4 * i < a.n)
                    *reinterpret_cast<plm_f32x4*>(a.part + (blockIdx.z * a.m + m) * n4 + n + 4 * i) = acc[i][j];
        }
        return;
    }
    if (a.out_type == kOutF32) {
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            const int64_t m = m0 + 16 * TM * wm + 16 * j + li;
            float* to = static_cast<float*>(a.out) + m * a.n + n;
            if (m >= a.m) continue;
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                if (n + 4 * i + 4 <= a.n) {
                    *reinterpret_cast<any_f32x4*>(to + 4 * i) = acc[i][j];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (n + 4 * i + e < a.n) to[4 * i + e] = acc[i][j][e];
                }
            }
        }
        return;
    }
    constexpr int kSide = TN == 1 ? 1 : 2;  // tiles stored together
#pragma unroll
    for (int j = 0; j < TM; ++j) {
        const int64_t m = m0 + 16 * TM * wm + 16 * j + li;
        uint16_t* to = static_cast<uint16_t*>(a.out) + m * a.n + n;
        if (m >= a.m) continue;
#pragma unroll
        for (int i = 0; i < TN; i += kSide) {
            const plm_u32x4 v = a.out_type == kOutBF16 ? pack8<true>(acc[i][j], acc[i + kSide - 1][j])
                                                       : pack8<false>(acc[i][j], acc[i + kSide - 1][j]);
            if (n + 4 * i + 4 * kSide <= a.n) {
                if constexpr (kSide == 2)
                    *reinterpret_cast<any_u32x4*>(to + 4 * i) = v;
                else
                    *reinterpret_cast<any_u32x2*>(to + 4 * i) = any_u32x2{v.x, v.y};
            } else {
#pragma unroll
                for (int e = 0; e < 4 * kSide; ++e)
                    if (n + 4 * i + e < a.n) to[4 * i + e] = static_cast<uint16_t>(v[e >> 1] >> (16 * (e & 1)));
            }
        }
    }
}

// The shares' sums in their order, rounded once.  A thread: four columns.
// Bound by its launch: 4 shares of 64 x 7168 5 us.
__global__ __launch_bounds__(256) void fp8_matmul_join_kernel(const MatmulArgs a, int shares) {
    const int64_t n4 = (a.n + 3) / 4;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (at >= a.m * n4) return;
    const plm_f32x4* part = reinterpret_cast<const plm_f32x4*>(a.part) + at;
    plm_f32x4 v = part[0];
    for (int s = 1; s < shares; ++s) v = v + part[s * a.m * n4];
    const int64_t m = at / n4, n = (at - m * n4) * 4;
    for (int e = 0; e < 4; ++e)
        if (n + e < a.n) store_out(a, m * a.n + n + e, v[e]);
}

// A weight of this size is not in the caches when the next call reads it (other weights come between), and
// where one group of rows reads it, it is read once: its loads leave the caches to the activations.  64, 24 and
// 16 rows with 7168 x 16384: 33.0, 27.9, 27.3 us without, 31.7, 25.7, 24.4 with; 64 x 7168 x 7168 18.9 without,
// 19.7 with.  Several groups find in the caches what the first of them read: 18 rows (two of 16) with
// 12967 x 5936 42.8 us with, 32.2 without, 91 (two of 64) with 14964 x 6800 62.8 and 44.3.
constexpr int64_t kStreamedBytes = static_cast<int64_t>(64) << 20;

template <int TN, int TM, int GN, int GM, int S, bool EXACT = false, bool ONCE = false>
int launch_tile(const MatmulArgs& a, int shares, hipStream_t st) {
    if constexpr (!ONCE && 16 * TM * GM <= 64)
        if (a.m <= 16 * TM * GM && a.n * a.k >= kStreamedBytes)
            return launch_tile<TN, TM, GN, GM, S, EXACT, true>(a, shares, st);
    using T = Tile<TN, TM, GN, GM, S>;
    constexpr int64_t kMostTiles = 65535;  // of a grid's second dimension
    if (plm::ceil_div(a.m, T::kM) > kMostTiles) {  // passes, one after another on the stream
        for (int64_t m = 0; m < a.m; m += kMostTiles * T::kM) {
            MatmulArgs part = a;
            part.m = std::min(a.m - m, kMostTiles * T::kM);
            part.x = a.x + m * a.k;
            part.xs = a.xs + m * a.blocks;
            part.out = static_cast<char*>(a.out) + m * a.n * (a.out_type == kOutF32 ? 4 : 2);
            const int code = launch_tile<TN, TM, GN, GM, S, EXACT, ONCE>(part, shares, st);
            if (code != 0) return code;
        }
        return 0;
    }
    const int64_t gx = plm::ceil_div(a.n, T::kN), gy = plm::ceil_div(a.m, T::kM);
    if (gx > 0x7FFFFFFF) return plm::fail(-2, "too many weight rows");
    const void* fn = reinterpret_cast<const void*>(&fp8_matmul_tile_kernel<TN, TM, GN, GM, S, EXACT, ONCE>);
    int code = T::kLds > 64 * 1024 ? plm::allow_large_lds(fn, T::kLds) : 0;
    if (code != 0) return code;
    hipLaunchKernelGGL((fp8_matmul_tile_kernel<TN, TM, GN, GM, S, EXACT, ONCE>),
                       dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy), static_cast<unsigned>(shares)),
                       dim3(64 * T::kWaves), T::kLds, st, a);
    code = plm::check_launch("fp8_e4m3_block_matmul");
    if (code != 0 || shares == 1) return code;
    hipLaunchKernelGGL(fp8_matmul_join_kernel, dim3(static_cast<unsigned>(plm::ceil_div(a.m * plm::ceil_div(a.n, 4), 256))),
                       dim3(256), 0, st, a, shares);
    return plm::check_launch("fp8_e4m3_block_matmul, join");
}

// How a product runs, from its sizes alone: the least of the times (us, an
// MI355X) that these straight lines give, fitted to 860 timings of 139 shapes
// of 1 to 4096 rows, 134 to 24576 weight rows and 544 to 16384 columns (the
// choice is 2 % slower than the fastest of all that were timed, 13 % at worst;
// on 800 other shapes 2.3 %).
//   tile   a workgroup's time per K block, alone on its compute unit or two on
//          one, for the rounds that the grid takes; 8 us for launch, first loads
//          and stores; at least the weight at 5.85 TB/s
//          (read again by each group of rows where the weight's tiles alone fill
//          the compute units: the groups come one after another then)
//   shares of the blocks (for grids that leave compute units idle): 3.85 us for
//          the join, its sums written and read at 3.6 TB/s
//   rows   its waves' blocks, or the weight at 3.6 TB/s (3.0 above 8 rows)
// Above 24576 weight rows the lines are carried on, checked at 51 sizes up to
// 200000 weight rows and 391 rows: tiles of 32 and 64 rows run in rounds there
// (64 x 36864 x 7168 74 us, with tiles of 16 rows 145; 64 x 129280 x 7168 181 and
// 618; 32 x 37888 x 3584 34 and 45), and groups that read such a weight one after
// another are fewer (391 x 33801 x 11568 with tiles of 256 rows 363, of 128 455).
// EXACT products are chosen by the same lines, without the tile of 256 rows: an
// EXACT block takes four instructions and its operands' conversion, which the
// lines do not know (64 x 7168 x 16384 38.8 us, 2048 x 7168 x 7168 244, 4096 x 7168
// x 16384 1047: 0.92 PFLOP/s of bf16 products).
struct Choice {
    int tile;    // activation rows of a workgroup; 0: the rows kernel
    int shares;  // of the blocks
};

struct TileCost {
    int tile, weight_rows;
    double alone, paired;  // paired 0: one workgroup per compute unit at a time
};
constexpr TileCost kTileCosts[] = {
    {256, 256, 1.42, 0.0}, {128, 128, 0.64, 1.33}, {64, 128, 0.49, 0.0}, {32, 128, 0.48, 0.0}, {16, 128, 0.33, 0.72}};
constexpr int kMostShares = 9;
constexpr int kMostRows = 32;  // of the rows kernel

// EXACT: the tiles up to 128 rows have the registers for its operands.
Choice choice_of(int64_t m, int64_t n, int64_t k, bool exact) {
    const int64_t blocks = plm::ceil_div(k, 128);
    const double bytes = static_cast<double>(n) * static_cast<double>(k);
    const int64_t cus = plm::cu_count();
    if (k >= (1 << 23)) return {0, 1};  // a workgroup's rows pass 32-bit offsets
    Choice best = {0, 1};
    double least = 1e30;
    if (m <= kMostRows)
        least = std::max(3.2 + (m <= 8 ? 0.75 : m <= 16 ? 1.0 : 2.2) * static_cast<double>(plm::ceil_div(blocks, 8)),
                         3.5 + bytes / (m <= 8 ? 3.6e6 : 3.0e6));
    for (const TileCost& c : kTileCosts) {
        if ((c.tile >= 2 * m && c.tile > 16) || (exact && c.tile == 256)) continue;
        const int64_t along = plm::ceil_div(n, c.weight_rows), groups_of_rows = plm::ceil_div(m, c.tile);
        const int64_t tiles = along * groups_of_rows;
        const double reads = along > cus ? static_cast<double>(groups_of_rows) : 1.0;
        for (int64_t s = 1; s <= kMostShares && s <= blocks; ++s) {
            const int64_t groups = tiles * s, per = plm::ceil_div(blocks, s);
            double t = static_cast<double>(per) * c.alone;
            if (c.tile == 256 || (c.paired == 0.0 && s == 1 && groups_of_rows == 1))
                t *= static_cast<double>(plm::ceil_div(groups, cus));
            else if (groups > cus && c.paired > 0.0)
                t = static_cast<double>(per) * c.paired *
                    std::max(1.0, static_cast<double>(groups) / static_cast<double>(2 * cus));
            else if (groups > cus)
                break;
            t = std::max(t + 8.0, reads * bytes / 5.85e6);
            if (s > 1) t += 3.85 + static_cast<double>(s * m) * static_cast<double>(n) * 8.0 / 3.6e6;
            if (t < least) {
                least = t;
                best = {c.tile, static_cast<int>(s)};
            }
        }
    }
    return best;
}

// The call's scratch: the shares' sums, then both operands in rows of whole
// pieces where theirs are not.
struct Scratch {
    int64_t sums;  // bytes
    int64_t k16;   // columns of a row
    int64_t all;   // bytes
};

Scratch scratch_of(const Choice& c, int64_t m, int64_t n, int64_t k) {
    Scratch s;
    s.sums = c.shares > 1 ? c.shares * m * plm::ceil_div(n, 4) * 16 : 0;
    s.k16 = plm::ceil_div(k, 16) * 16;
    s.all = s.sums + (s.k16 != k ? (m + n) * s.k16 : 0);
    return s;
}

bool bad_sizes(int64_t m, int64_t n, int64_t k) {
    const int64_t most = static_cast<int64_t>(1) << 31;
    return m <= 0 || n <= 0 || k <= 0 || m >= most || n >= most || k >= most;
}

}  // namespace

PLM_EXPORT int64_t fp8_e4m3_block_matmul_scratch_bytes(int64_t rows, int64_t out_rows, int64_t in_cols, int dtype_code) {
    if (bad_sizes(rows, out_rows, in_cols) || dtype_code < 0 || dtype_code > 2) return plm::fail(-2, "bad dimensions");
    return scratch_of(choice_of(rows, out_rows, in_cols, dtype_code == kOutF32), rows, out_rows, in_cols).all;
}

PLM_EXPORT int fp8_e4m3_block_matmul(const uint8_t* x, const float* x_scales, const uint8_t* fp8_weight,
                                     const float* scale_inv, void* out, void* scratch, int64_t scratch_bytes,
                                     int64_t rows, int64_t out_rows, int64_t in_cols, int64_t scale_cols,
                                     int dtype_code) {
    if (x == nullptr || x_scales == nullptr || fp8_weight == nullptr || scale_inv == nullptr || out == nullptr)
        return plm::fail(-1, "null pointer");
    if (bad_sizes(rows, out_rows, in_cols) || scale_cols < plm::ceil_div(in_cols, 128) || dtype_code < 0 || dtype_code > 2)
        return plm::fail(-2, "bad dimensions");
    if (!plm::aligned16(x) || !plm::aligned16(fp8_weight)) return plm::fail(-2, "rows and weight must be 16-byte aligned");
    MatmulArgs a = {x,    x_scales, fp8_weight, scale_inv,  out,
                    rows, out_rows, in_cols,    scale_cols, static_cast<int>(plm::ceil_div(in_cols, 128)),
                    dtype_code, nullptr};
    const bool exact = dtype_code == kOutF32;
    const Choice c = choice_of(rows, out_rows, in_cols, exact);
    const Scratch need = scratch_of(c, rows, out_rows, in_cols);
    const hipStream_t st = plm::current_stream();
    if (need.all > 0) {
        char* at = static_cast<char*>(scratch);
        if (at == nullptr) {
            at = static_cast<char*>(plm::workspace(static_cast<size_t>(need.all)));
            if (at == nullptr) return -3;
        } else if (scratch_bytes < need.all || !plm::aligned16(at)) {
            return plm::fail(-3, "scratch must hold fp8_e4m3_block_matmul_scratch_bytes, 16-byte aligned");
        }
        a.part = reinterpret_cast<float*>(at);
        if (need.k16 != in_cols) {
            uint8_t* to = reinterpret_cast<uint8_t*>(at) + need.sums;
            int code = pad_rows(x, to, rows, in_cols, need.k16, st);
            if (code == 0) code = pad_rows(fp8_weight, to + rows * need.k16, out_rows, in_cols, need.k16, st);
            if (code != 0) return code;
            a.x = to;
            a.w = to + rows * need.k16;
            a.k = need.k16;
        }
    }
    const int waves = std::min(8, a.blocks);
    // Tiles of 128 rows: two workgroups fit a compute unit with two stages each; where there is one for each,
    // it takes three (300 x 3000 x 16000 44 -> 36 us, 256 x 7168 x 16384 68 -> 63).
    const bool alone = plm::ceil_div(out_rows, 128) * plm::ceil_div(rows, 128) * c.shares <= plm::cu_count();
    if (exact) {
        switch (c.tile) {
            case 16: return launch_tile<1, 1, 8, 1, 4, true>(a, c.shares, st);
            case 32: return launch_tile<1, 2, 8, 1, 3, true>(a, c.shares, st);
            case 64: return launch_tile<2, 2, 4, 2, 3, true>(a, c.shares, st);
            case 128:
                return alone ? launch_tile<2, 4, 4, 2, 3, true>(a, c.shares, st)
                             : launch_tile<2, 4, 4, 2, 2, true>(a, c.shares, st);
            default: break;
        }
        return rows <= 16 ? launch_rows<1, 1, 4, 8, true>(a, waves, st) : launch_rows<2, 2, 2, 8, true>(a, waves, st);
    }
    switch (c.tile) {
        case 16: return launch_tile<1, 1, 8, 1, 4>(a, c.shares, st);
        case 32: return launch_tile<1, 2, 8, 1, 3>(a, c.shares, st);
        case 64: return launch_tile<2, 2, 4, 2, 3>(a, c.shares, st);
        case 128:
            return alone ? launch_tile<2, 4, 4, 2, 3>(a, c.shares, st) : launch_tile<2, 4, 4, 2, 2>(a, c.shares, st);
        case 256: return launch_tile<4, 8, 4, 2, 2>(a, c.shares, st);
        default: break;
    }
    return rows <= 16 ? launch_rows<1, 1, 4, 8, false>(a, waves, st) : launch_rows<2, 2, 2, 8, false>(a, waves, st);
}
