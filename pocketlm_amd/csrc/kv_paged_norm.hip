// Appends to a paged cache that norm queries and keys head by head before
// their rotation, and appends to a cache of e4m3 values:
//
//   y = x * rsqrt(mean(x^2) + eps) * w      over a head's values, fp32 (sums of squares that leave fp32's
//                                           range in 64 bits); y = x without weights, and for values v
//   z = y rotated to the row's position     fp32
//   16-bit caches and queries: z rounded once
//   e4m3 caches: scale = max(max |z| / 448, 2^-126) of the position and head, z / scale rounded once
//
// The scale's lower bound keeps 1 / scale finite; a head that holds an infinity
// or a NaN gets the scale NaN and bytes 0x7F, as in fp8_rows.hip.
#include <algorithm>

#include "kv_paged.h"

namespace {

using namespace plm_paged;

constexpr float kE4m3Max = 448.0f;
constexpr float kSmallestScale = 1.17549435e-38f;  // 2^-126
constexpr int kThreads = 512;
constexpr int kMostRows = 8;  // of a workgroup

// Workgroups of a compute unit before they take more rows than one: three or
// four are resident (102 registers), and more rows than one pay once all have work
// (5 x 1700 rows of 28 and 4 heads of 128: 30 us with 8 rows a workgroup, 34
// with 4, 55 with 2, 58 with 1; 1 x 512 rows 6.0 us with 1).
constexpr int kBlocks = 4;

struct NormArgs {
    Pages p;
    Scales s;               // of e4m3 caches
    const uint16_t* q;      // null: keys and values alone
    const uint16_t* k;
    const uint16_t* v;
    const uint16_t* q_weight;  // [head_dim] each; null: not normed
    const uint16_t* k_weight;
    uint16_t* q_out;        // [rows][heads][head_dim]
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides, values
    const int* row_starts;  // null: every sequence has rows_per_sequence rows
    const double* freq;     // [pairs]
    int* rejected;
    int rows;
    int block_rows;         // rows of a workgroup
    int rows_per_sequence;
    int heads;              // 0 without q
    int kv_heads;
    int head_dim;
    int pairs;              // rotated pairs of a head
    int pieces;             // threads that hold a head
    int lanes_log2;         // lanes of a head: the next power of two
    float eps;
};

enum Mode { kHalves = 0, kAdjacent = 1, kAny = 2, kAnyAdjacent = 3 };

// Over the 2^log2 adjacent lanes of a head, every one of which gets it.
template <typename F>
__device__ __forceinline__ float over_head(float v, int log2, F op) {
#define PLM_STEP(ctrl) \
    v = op(v, __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(__float_as_uint(v)), ctrl, 0xF, 0xF, false))))
    if (log2 > 0) PLM_STEP(0xB1);   // quad_perm [1,0,3,2]
    if (log2 > 1) PLM_STEP(0x4E);   // quad_perm [2,3,0,1]
    if (log2 > 2) PLM_STEP(0x141);  // row_half_mirror
    if (log2 > 3) PLM_STEP(0x140);  // row_mirror
#undef PLM_STEP
    if (log2 > 4) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    return v;
}

// Whether a head's sum of squares has left fp32 (see fp8_rows.hip).
__device__ __forceinline__ bool beyond(float total, float eps, int n) {
    return !(total < 0x1p127f) || total + eps * static_cast<float>(n) < 0x1p-80f;
}

// y / scale rounded once: the reciprocal's product and a correction by its remainder.
__device__ __forceinline__ float quotient(float y, float scale, float inv) {
    const float q = y * inv;
    return fmaf(fmaf(-q, scale, y), inv, q);
}

__device__ __forceinline__ u32x2 pack8_e4m3(const f32x8 y, float scale, float inv) {
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = quotient(y[i], scale, inv);
    u32x2 o;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int half = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
        o[i] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], half, true));
    }
    return o;
}

// Workgroup (rows, part of a row's heads); a head has 2^lanes_log2 lanes of a
// wave, `pieces` of which hold 16 values each (c and c + half a head, or
// adjacent ones), or 8 in the modes for any size, so that a head's sum and
// maximum are a few register permutes and every value is read once (kAny*: the
// partner of a rotated pair is read again, from the first cache).  The places
// and the angles of all of a workgroup's rows are found at once and the next
// row's values are read while one is at work: a row by itself waits for row
// starts, lengths and page table one after the other.
//
// Bound by memory where rows are many: 125 MB of 5 x 1700 rows (28 and 4 heads
// of 128, fp16) in 30 us, 4.2 TB/s, 119 MB into e4m3 pages in 29 us; one row takes
// 3.6 us, which is its chain of loads.
//
// Five waves a SIMD for e4m3 pages (5 x 1700 rows 29 us, 36 with the four that 102
// registers allow), where more arithmetic stands between loads and stores; four
// for 16-bit ones (39 with five, 31).
template <bool BF16, int MODE, bool E8>
__global__ __launch_bounds__(kThreads, E8 ? 5 : 1) void norm_append_kernel(const NormArgs a) {
    constexpr bool ANY = MODE == kAny || MODE == kAnyAdjacent;
    constexpr int N = ANY ? 1 : 2;  // pieces of 8 values
    constexpr int kPairs = 128;
    __shared__ __attribute__((aligned(16))) float cs[kMostRows][kPairs], sn[kMostRows][kPairs];
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.block_rows;
    const int count = min(static_cast<int64_t>(a.block_rows), a.rows - row0);
    const int lane = threadIdx.x & 63;
    const int all = a.heads + 2 * a.kv_heads;
    const int head = (blockIdx.y * blockDim.x + threadIdx.x) >> a.lanes_log2;
    const int c = threadIdx.x & ((1 << a.lanes_log2) - 1);
    const bool live = head < all && c < a.pieces;
    const bool is_q = head < a.heads, is_k = !is_q && head < a.heads + a.kv_heads;
    const int kvh = is_q ? 0 : is_k ? head - a.heads : head - a.heads - a.kv_heads;
    const int64_t src_row = is_q ? a.q_row : is_k ? a.k_row : a.v_row;
    const uint16_t* src = (is_q   ? a.q + head * a.q_head
                           : is_k ? a.k + kvh * a.k_head
                                  : a.v + kvh * a.v_head) + row0 * src_row;
    const uint16_t* weight = is_q ? a.q_weight : is_k ? a.k_weight : nullptr;
    const bool turned = is_q || is_k;
    int at[2];
    at[0] = ANY || (MODE == kHalves && turned) ? 8 * c : 16 * c;
    at[1] = MODE == kHalves && turned ? a.head_dim / 2 + 8 * c : at[0] + 8;
    u32x4 x[N], ahead[N], w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        ahead[i] = w[i] = u32x4{0, 0, 0, 0};
        if (live) {
            ahead[i] = *reinterpret_cast<const u32x4*>(src + at[i]);
            if (weight != nullptr) w[i] = *reinterpret_cast<const u32x4*>(weight + at[i]);
        }
    }
    const Place places = places_of(a.p, a.row_starts, a.rows_per_sequence, row0, count, lane);
    if (a.rejected != nullptr && threadIdx.x < 64 && blockIdx.y == 0) {
        const int lost = __popcll(__ballot(lane < count && places.pos >= 0 && !places.stored));
        if (lost > 0 && lane == 0) atomicAdd(a.rejected, lost);
    }
    const int low = static_cast<int>(places.pos), high = static_cast<int>(places.pos >> 32);
    for (int base = 0; base < count * a.pairs; base += blockDim.x) {
        // (every lane takes part in the shuffles)
        const int i = base + threadIdx.x;
        const int r = min(static_cast<int>(static_cast<unsigned>(i) / static_cast<unsigned>(a.pairs)), count - 1);
        const int pair = i - r * a.pairs;
        const int64_t pos = static_cast<int64_t>(__shfl(high, r)) << 32 | static_cast<uint32_t>(__shfl(low, r));
        if (pair < a.pairs) {
            constexpr double kTurn = 6.283185307179586476925286766559;
            const double angle = static_cast<double>(max(pos, static_cast<int64_t>(0))) * a.freq[pair];
            const float turn = static_cast<float>(angle - kTurn * rint(angle / kTurn));
            cs[r][pair] = cosf(turn);
            sn[r][pair] = sinf(turn);
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int r = 0; r < count; ++r) {
        const int64_t row = row0 + r;
        const bool placed = __builtin_amdgcn_readlane(high, r) >= 0;
        const bool stored = __builtin_amdgcn_readlane(places.stored ? 1 : 0, r) != 0;
        const uint32_t page = __builtin_amdgcn_readlane(places.page, r);
        const uint32_t slot = __builtin_amdgcn_readlane(places.slot, r);
        f32x8 y[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] = ahead[i];
            y[i] = widen8<BF16>(x[i]);
        }
        const uint16_t* const here = src;
        src += src_row;
        if (live && r + 1 < count)
#pragma unroll
            for (int i = 0; i < N; ++i) ahead[i] = *reinterpret_cast<const u32x4*>(src + at[i]);

        // the norm; every lane of the head takes part
        float scale = 1.0f;
        int shift = 0;
        if (a.q_weight != nullptr || a.k_weight != nullptr) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) sum = fmaf(y[i][j], y[i][j], sum);
            auto add = [](float u, float v) { return u + v; };
            sum = over_head(sum, a.lanes_log2, add);
            scale = 1.0f / sqrtf(sum / static_cast<float>(a.head_dim) + a.eps);
            if (__builtin_expect(__any(weight != nullptr && beyond(sum, a.eps, a.head_dim)), 0)) {
                double wide = 0.0;
#pragma unroll
                for (int i = 0; i < N; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const double v = y[i][j];
                        wide = fma(v, v, wide);
                    }
                for (int off = 1; off < 1 << a.lanes_log2; off <<= 1) wide += __shfl_xor(wide, off);
                if (weight != nullptr && beyond(sum, a.eps, a.head_dim)) {
                    // the root's power of two goes to the values, which it leaves exact, so that both stay in range
                    const double mean = wide / static_cast<double>(a.head_dim) + static_cast<double>(a.eps);
                    shift = -(__builtin_amdgcn_frexp_exp(mean) >> 1);
                    scale = 1.0f / sqrtf(static_cast<float>(__builtin_ldexp(mean, 2 * shift)));
                }
#pragma unroll
                for (int i = 0; i < N; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[i][j] = ldexpf(y[i][j], shift);
            }
            if (weight != nullptr) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const f32x8 wf = widen8<BF16>(w[i]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[i][j] = y[i][j] * scale * wf[j];
                }
            }
        }
        if (live && turned && a.pairs > 0) {  // (lanes without values stay 0: there are no angles for them)
            if constexpr (MODE == kHalves) {
                // (a head has twice as many values as pairs)
                const float* const cc = &cs[r][min(8 * c, kPairs - 8)];
                const float* const ss = &sn[r][min(8 * c, kPairs - 8)];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float u = y[0][j], v = y[1][j];
                    y[0][j] = u * cc[j] - v * ss[j];
                    y[1][j] = v * cc[j] + u * ss[j];
                }
            } else if constexpr (MODE == kAdjacent) {
                const float* const cc = &cs[r][min(8 * c, kPairs - 8)];
                const float* const ss = &sn[r][min(8 * c, kPairs - 8)];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const int pair = 4 * i + j / 2;
                        const float u = y[i][j], v = y[i][j + 1];
                        y[i][j] = u * cc[pair] - v * ss[pair];
                        y[i][j + 1] = v * cc[pair] + u * ss[pair];
                    }
            } else {
                const f32x8 mine = y[0];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int d = 8 * c + j;
                    if (live && d < 2 * a.pairs) {
                        const bool first = MODE == kAnyAdjacent ? (d & 1) == 0 : d < a.pairs;
                        const int pair = MODE == kAnyAdjacent ? d >> 1 : first ? d : d - a.pairs;
                        float o;
                        if constexpr (MODE == kAnyAdjacent) {
                            o = mine[j ^ 1];
                        } else {
                            const int other = first ? d + a.pairs : d - a.pairs;
                            o = widen1<BF16>(here[other]);
                            if (weight != nullptr) o = ldexpf(o, shift) * scale * widen1<BF16>(weight[other]);
                        }
                        y[0][j] = first ? mine[j] * cs[r][pair] - o * sn[r][pair] : mine[j] * cs[r][pair] + o * sn[r][pair];
                    }
                }
            }
        }
        float largest = 0.0f;
        bool finite = true;
        if constexpr (E8) {
            // as integers: a NaN is the largest
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(y[i][j]) & 0x7FFFFFFFu);
            auto most = [](float u, float v) { return __uint_as_float(max(__float_as_uint(u), __float_as_uint(v))); };
            largest = over_head(__uint_as_float(m), a.lanes_log2, most);
            finite = __float_as_uint(largest) < 0x7F800000u;
        }
        if (!live || (!is_q && !stored)) continue;
        if (is_q) {
            uint16_t* out = a.q_out + (row * a.heads + head) * a.head_dim;
#pragma unroll
            for (int i = 0; i < N; ++i)
                *reinterpret_cast<u32x4*>(out + at[i]) = placed ? narrow8<BF16>(y[i]) : u32x4{0, 0, 0, 0};
            continue;
        }
        // (32 bits hold a place's piece of 16 bytes: see Pages)
        const int64_t piece = page * a.p.page_stride + slot * a.p.slot_stride;
        if constexpr (E8) {
            uint8_t* out = reinterpret_cast<uint8_t*>(is_k ? a.p.k : a.p.v) + piece * 16 + kvh * a.p.head_stride;
            const float s = finite ? fmaxf(largest / kE4m3Max, kSmallestScale) : __uint_as_float(0x7FC00000u);
            const float inv = 1.0f / s;
#pragma unroll
            for (int i = 0; i < N; ++i)
                *reinterpret_cast<u32x2*>(out + at[i]) =
                    finite ? pack8_e4m3(y[i], s, inv) : u32x2{0x7F7F7F7Fu, 0x7F7F7F7Fu};
            if (c == 0) (is_k ? a.s.k : a.s.v)[a.s.at(static_cast<int>(page), kvh, slot)] = s;
        } else {
            uint16_t* out = (is_k ? a.p.k : a.p.v) + piece * 8 + kvh * a.p.head_stride;
#pragma unroll
            for (int i = 0; i < N; ++i)  // values v as they are
                *reinterpret_cast<u32x4*>(out + at[i]) = is_k ? narrow8<BF16>(y[i]) : x[i];
        }
    }
}

template <bool BF16, bool E8>
void launch(const NormArgs& a, int mode, dim3 grid, dim3 block, hipStream_t st) {
    switch (mode) {
        case kHalves: hipLaunchKernelGGL((norm_append_kernel<BF16, kHalves, E8>), grid, block, 0, st, a); break;
        case kAdjacent: hipLaunchKernelGGL((norm_append_kernel<BF16, kAdjacent, E8>), grid, block, 0, st, a); break;
        case kAny: hipLaunchKernelGGL((norm_append_kernel<BF16, kAny, E8>), grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL((norm_append_kernel<BF16, kAnyAdjacent, E8>), grid, block, 0, st, a); break;
    }
}

// What both entry points check and launch once the caches are known.
template <bool E8>
int run(NormArgs& a, int64_t rows, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t head_dim,
        int64_t rope_pairs, int interleaved, int dtype_code, const char* name) {
    if (rows <= 0 || rows > kMostInt || heads < 0 || heads > 65535 || rope_pairs < 0 || 2 * rope_pairs > head_dim ||
        (a.row_starts == nullptr && rows % sequences != 0) || !(a.eps >= 0.0f))
        return plm::fail(-2, "bad dimensions");
    auto whole = [](const void* at, int64_t row, int64_t head) {
        return plm::aligned16(at) && row >= 0 && head >= 0 && row % 8 == 0 && head % 8 == 0;
    };
    if ((heads > 0 && (!whole(a.q, a.q_row, a.q_head) || !plm::aligned16(a.q_out))) ||
        !whole(a.k, a.k_row, a.k_head) || !whole(a.v, a.v_row, a.v_head))
        return plm::fail(-2, "row strides and addresses must be multiples of 16 bytes");
    if (!plm::aligned16(a.q_weight) || !plm::aligned16(a.k_weight))
        return plm::fail(-2, "norm weights must be 16-byte aligned");
    a.rows_per_sequence = static_cast<int>(a.row_starts == nullptr ? rows / sequences : 1);
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    a.head_dim = static_cast<int>(head_dim);
    a.pairs = static_cast<int>(rope_pairs);
    // whole pairs of pieces: 16 values a thread, each read once
    const bool whole_head = head_dim % 16 == 0 && (rope_pairs == 0 || 2 * rope_pairs == head_dim);
    const int mode = whole_head ? (rope_pairs > 0 && interleaved ? kAdjacent : kHalves)
                                : (interleaved ? kAnyAdjacent : kAny);
    a.pieces = static_cast<int>(head_dim / (whole_head ? 16 : 8));
    a.lanes_log2 = 0;
    while ((1 << a.lanes_log2) < a.pieces) ++a.lanes_log2;
    const int64_t threads = (heads + 2 * kv_heads) << a.lanes_log2;
    const int64_t parts = plm::ceil_div(threads, kThreads);
    if (parts > 65535) return plm::fail(-2, "too many heads");
    a.rows = static_cast<int>(rows);
    a.block_rows = static_cast<int>(
        std::clamp<int64_t>(rows * parts / (kBlocks * plm::cu_count()), 1, kMostRows));
    const dim3 grid(static_cast<unsigned>(plm::ceil_div(rows, a.block_rows)), static_cast<unsigned>(parts));
    const dim3 block(static_cast<unsigned>(plm::ceil_div(plm::ceil_div(threads, parts), 64) * 64));
    if (dtype_code == 1)
        launch<true, E8>(a, mode, grid, block, plm::current_stream());
    else
        launch<false, E8>(a, mode, grid, block, plm::current_stream());
    return plm::check_launch(name);
}

}  // namespace

PLM_EXPORT int kv_paged_norm_append_u16(const uint16_t* q, const uint16_t* k, const uint16_t* v,
                                        const uint16_t* q_norm_weight, const uint16_t* k_norm_weight, uint16_t* q_out,
                                        uint16_t* k_cache, uint16_t* v_cache, const int* page_table, const int* lengths,
                                        const int* row_starts, const double* rope_frequencies, int* rejected,
                                        int64_t rows, int64_t sequences, int64_t heads, int64_t kv_heads,
                                        int64_t head_dim, int64_t rope_pairs, int interleaved, int64_t q_row_stride,
                                        int64_t q_head_stride, int64_t k_row_stride, int64_t k_head_stride,
                                        int64_t v_row_stride, int64_t v_head_stride, int64_t table_cols,
                                        int64_t num_pages, int64_t page_size, int64_t page_stride, int64_t slot_stride,
                                        int64_t head_stride, float rms_eps, int dtype_code) {
    if (k == nullptr || v == nullptr || k_norm_weight == nullptr ||
        (heads > 0 && (q == nullptr || q_out == nullptr || q_norm_weight == nullptr)) ||
        (rope_pairs > 0 && rope_frequencies == nullptr))
        return plm::fail(-1, "null pointer");
    NormArgs a = {};
    const int code = pages_of(a.p, k_cache, v_cache, page_table, lengths, sequences, table_cols, num_pages, page_size,
                              kv_heads, head_dim, page_stride, slot_stride, head_stride, dtype_code);
    if (code != 0) return code;
    a.q = q, a.k = k, a.v = v;
    a.q_weight = heads > 0 ? q_norm_weight : nullptr;
    a.k_weight = k_norm_weight;
    a.q_out = q_out;
    a.q_row = q_row_stride, a.q_head = q_head_stride;
    a.k_row = k_row_stride, a.k_head = k_head_stride;
    a.v_row = v_row_stride, a.v_head = v_head_stride;
    a.row_starts = row_starts;
    a.freq = rope_frequencies;
    a.rejected = rejected;
    a.eps = rms_eps;
    return run<false>(a, rows, sequences, heads, kv_heads, head_dim, rope_pairs, interleaved, dtype_code,
                      "kv_paged_norm_append_u16");
}

PLM_EXPORT int kv_paged_append_e4m3(const uint16_t* q, const uint16_t* k, const uint16_t* v,
                                    const uint16_t* q_norm_weight, const uint16_t* k_norm_weight, uint16_t* q_out,
                                    uint8_t* k_cache, uint8_t* v_cache, float* k_scales, float* v_scales,
                                    const int* page_table, const int* lengths, const int* row_starts,
                                    const double* rope_frequencies, int* rejected, int64_t rows, int64_t sequences,
                                    int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rope_pairs,
                                    int interleaved, int64_t q_row_stride, int64_t q_head_stride, int64_t k_row_stride,
                                    int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride,
                                    int64_t table_cols, int64_t num_pages, int64_t page_size, int64_t page_stride,
                                    int64_t slot_stride, int64_t head_stride, int64_t scale_page_stride,
                                    int64_t scale_head_stride, float rms_eps, int dtype_code) {
    if (k == nullptr || v == nullptr || (heads > 0 && (q == nullptr || q_out == nullptr)) ||
        (rope_pairs > 0 && rope_frequencies == nullptr))
        return plm::fail(-1, "null pointer");
    NormArgs a = {};
    int code = pages_of<16>(a.p, k_cache, v_cache, page_table, lengths, sequences, table_cols, num_pages, page_size,
                            kv_heads, head_dim, page_stride, slot_stride, head_stride, dtype_code);
    if (code != 0) return code;
    code = scales_of(a.s, a.p, kv_heads, k_scales, v_scales, scale_page_stride, scale_head_stride);
    if (code != 0) return code;
    a.q = q, a.k = k, a.v = v;
    a.q_weight = heads > 0 ? q_norm_weight : nullptr;
    a.k_weight = k_norm_weight;
    a.q_out = q_out;
    a.q_row = q_row_stride, a.q_head = q_head_stride;
    a.k_row = k_row_stride, a.k_head = k_head_stride;
    a.v_row = v_row_stride, a.v_head = v_head_stride;
    a.row_starts = row_starts;
    a.freq = rope_frequencies;
    a.rejected = rejected;
    a.eps = rms_eps;
    return run<true>(a, rows, sequences, heads, kv_heads, head_dim, rope_pairs, interleaved, dtype_code,
                     "kv_paged_append_e4m3");
}
