// A key-value cache in pages: rows appended with their rotation, and the
// attention of one to eight new rows of each sequence over its pages.
//
// The caches are [page][slot][kv head][head_dim] with strides of their own
// (head_dim adjacent), fp16 or bf16.  Position p of sequence b is slot
// p % page_size of page table[b][p / page_size].  lengths[b] is what b holds
// before the call's rows, negative for an idle sequence.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "common.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2 v = {a, b};
    if constexpr (BF16)
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
    else
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

template <bool BF16>
__device__ __forceinline__ f32x8 widen8(u32x4 v) {
    if constexpr (BF16)
        return __builtin_convertvector(__builtin_bit_cast(bf16x8, v), f32x8);
    else
        return __builtin_convertvector(__builtin_bit_cast(f16x8, v), f32x8);
}

template <bool BF16>
__device__ __forceinline__ u32x4 narrow8(const f32x8 v) {
    if constexpr (BF16)
        return __builtin_bit_cast(u32x4, __builtin_convertvector(v, bf16x8));
    else
        return __builtin_bit_cast(u32x4, __builtin_convertvector(v, f16x8));
}

template <bool BF16>
__device__ __forceinline__ float widen1(uint16_t v) {
    if constexpr (BF16)
        return __uint_as_float(static_cast<uint32_t>(v) << 16);
    else
        return static_cast<float>(__builtin_bit_cast(_Float16, v));
}

template <bool BF16>
__device__ __forceinline__ uint16_t narrow1(float v) {
    if constexpr (BF16)
        return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
    else
        return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}

// Where the pages are.  Strides in pieces of 8 values (16 bytes): 32 bits
// reach 64 GiB; the head's offset is added in 64 bits.
struct Pages {
    uint16_t* k;
    uint16_t* v;
    const int* table;    // [sequences][table_cols]
    const int* lengths;  // [sequences]
    int64_t head_stride;  // values
    uint32_t page_stride;
    uint32_t slot_stride;
    uint32_t page_size;
    uint32_t num_pages;
    int table_cols;
    int sequences;
};

// ---------------------------------------------------------------- append

struct AppendArgs {
    Pages p;
    const uint16_t* q;  // null: keys and values alone
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* q_out;    // [rows][heads][head_dim]
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides, values
    const int* row_starts;  // null: every sequence has rows_per_sequence rows
    const double* freq;     // [pairs]
    int* rejected;
    int64_t rows;
    int rows_per_sequence;
    int heads;              // 0 without q
    int kv_heads;
    int head_dim;
    int pairs;              // rotated pairs of a head
    int units;              // per row
};

enum AppendMode { kCopy = 0, kHalves = 1, kAdjacent = 2, kAny = 3, kAnyAdjacent = 4 };

constexpr int kAppendThreads = 256;

// Workgroup (row, part of the row's heads): the angles of the row's position
// once per workgroup (their reduction to one turn in 64 bits: a position of
// 10^6 has its angle to 10^-10), then one unit a thread: 8 pairs of a head
// (16 values), or 8 values of it in the modes for any size.  The row's values
// are on their way while its sequence, page and angles are found.  Bound by
// that chain for a step (64 rows of 28 and 2 x 4 heads of 128 3.6 us), by
// memory for prompts (6800 such rows, 125 MB moved, 25 us, 4.9 TB/s).
template <bool BF16, int MODE>
__global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(const AppendArgs a) {
    __shared__ float cs[128], sn[128];
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 63;
    const int unit = blockIdx.y * blockDim.x + threadIdx.x;
    constexpr bool ANY = MODE == kAny || MODE == kAnyAdjacent;
    const int per = a.head_dim / (ANY ? 8 : 16);
    const bool live = unit < a.units;
    const int head = live ? unit / per : 0, c = live ? unit - head * per : 0;
    const bool is_q = head < a.heads, is_k = !is_q && head < a.heads + a.kv_heads;
    const int kvh = is_q ? 0 : is_k ? head - a.heads : head - a.heads - a.kv_heads;
    const uint16_t* src = is_q   ? a.q + row * a.q_row + head * a.q_head
                          : is_k ? a.k + row * a.k_row + kvh * a.k_head
                                 : a.v + row * a.v_row + kvh * a.v_head;
    const bool turned = is_q || is_k;
    // the two pieces of 8 values: c and c + half a head, or adjacent ones
    const int at0 = ANY ? 8 * c : (MODE == kHalves && turned) ? 8 * c : 16 * c;
    const int at1 = (MODE == kHalves && turned) ? a.head_dim / 2 + 8 * c : at0 + 8;
    u32x4 x0 = {0, 0, 0, 0}, x1 = {0, 0, 0, 0};
    if (live) {
        x0 = *reinterpret_cast<const u32x4*>(src + at0);
        if constexpr (!ANY) x1 = *reinterpret_cast<const u32x4*>(src + at1);
    }

    // the row's sequence and position
    int seq;
    int64_t in_seq;
    if (a.row_starts != nullptr) {
        int count = 0;  // starts at or before the row
        for (int base = 0; base <= a.p.sequences; base += 64) {
            const int i = base + lane;
            const bool before = i <= a.p.sequences && a.row_starts[min(i, a.p.sequences)] <= row;
            count += __popcll(__ballot(before));
        }
        seq = count - 1;
        in_seq = seq >= 0 ? row - a.row_starts[min(seq, a.p.sequences)] : 0;
    } else {
        seq = static_cast<int>(row / a.rows_per_sequence);
        in_seq = row - static_cast<int64_t>(seq) * a.rows_per_sequence;
    }
    const bool in_batch = seq >= 0 && seq < a.p.sequences;
    const int length = in_batch ? a.p.lengths[seq] : -1;
    const int64_t pos = length >= 0 ? length + in_seq : -1;
    const bool placed = pos >= 0;
    bool stored = false;
    uint32_t off = 0;
    if (placed) {
        const int64_t index = pos / a.p.page_size;
        if (index < a.p.table_cols) {
            const int page = a.p.table[static_cast<int64_t>(seq) * a.p.table_cols + index];
            stored = page >= 0 && static_cast<uint32_t>(page) < a.p.num_pages;
            off = static_cast<uint32_t>(page) * a.p.page_stride +
                  static_cast<uint32_t>(pos - index * a.p.page_size) * a.p.slot_stride;
        }
        if (!stored && a.rejected != nullptr && threadIdx.x == 0 && blockIdx.y == 0) atomicAdd(a.rejected, 1);
    }
    if constexpr (MODE != kCopy) {
        for (int i = threadIdx.x; i < a.pairs; i += blockDim.x) {
            constexpr double kTurn = 6.283185307179586476925286766559;
            const double angle = static_cast<double>(placed ? pos : 0) * a.freq[i];
            const float r = static_cast<float>(angle - kTurn * rint(angle / kTurn));
            cs[i] = cosf(r);
            sn[i] = sinf(r);
        }
        __syncthreads();
    }
    if (!live || (!is_q && !stored)) return;
    uint16_t* dst = is_q ? a.q_out + (row * a.heads + head) * a.head_dim
                         : (is_k ? a.p.k : a.p.v) + static_cast<int64_t>(off) * 8 + kvh * a.p.head_stride;
    if (is_q && !placed) {
        *reinterpret_cast<u32x4*>(dst + at0) = u32x4{0, 0, 0, 0};
        if constexpr (!ANY) *reinterpret_cast<u32x4*>(dst + at1) = u32x4{0, 0, 0, 0};
        return;
    }
    if constexpr (MODE == kHalves) {
        if (turned) {
            const f32x8 u = widen8<BF16>(x0), w = widen8<BF16>(x1);
            f32x8 y0, y1;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float cc = cs[8 * c + i], ss = sn[8 * c + i];
                y0[i] = u[i] * cc - w[i] * ss;
                y1[i] = w[i] * cc + u[i] * ss;
            }
            x0 = narrow8<BF16>(y0);
            x1 = narrow8<BF16>(y1);
        }
    } else if constexpr (MODE == kAdjacent) {
        if (turned) {
            f32x8 u = widen8<BF16>(x0), w = widen8<BF16>(x1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float c0 = cs[8 * c + i], s0 = sn[8 * c + i], c1 = cs[8 * c + 4 + i], s1 = sn[8 * c + 4 + i];
                const float u0 = u[2 * i], u1 = u[2 * i + 1], w0 = w[2 * i], w1 = w[2 * i + 1];
                u[2 * i] = u0 * c0 - u1 * s0;
                u[2 * i + 1] = u1 * c0 + u0 * s0;
                w[2 * i] = w0 * c1 - w1 * s1;
                w[2 * i + 1] = w1 * c1 + w0 * s1;
            }
            x0 = narrow8<BF16>(u);
            x1 = narrow8<BF16>(w);
        }
    } else if constexpr (ANY) {
        if (turned) {
            const f32x8 u = widen8<BF16>(x0);
            u32x4 packed;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = 8 * c + i;
                float y = u[i];
                if (d < 2 * a.pairs) {
                    const bool first = MODE == kAnyAdjacent ? (d & 1) == 0 : d < a.pairs;
                    const int pair = MODE == kAnyAdjacent ? d >> 1 : first ? d : d - a.pairs;
                    const int other = MODE == kAnyAdjacent ? d ^ 1 : first ? d + a.pairs : d - a.pairs;
                    const float o = widen1<BF16>(src[other]);
                    y = first ? y * cs[pair] - o * sn[pair] : y * cs[pair] + o * sn[pair];
                }
                const uint32_t bits = narrow1<BF16>(y);
                packed[i >> 1] = (i & 1) ? packed[i >> 1] | bits << 16 : bits;
            }
            x0 = packed;
        }
    }
    *reinterpret_cast<u32x4*>(dst + at0) = x0;
    if constexpr (!ANY) *reinterpret_cast<u32x4*>(dst + at1) = x1;
}

// ---------------------------------------------------------------- attention
//
// A unit is 128 positions of a sequence (an idle or empty one has one unit,
// whose result is the zeros).  The units are dealt to the workgroups of a
// key-value head on the device, from the lengths: no launch, copy or host value
// depends on them.  Where no sequence is much longer than the others' share,
// or all are short, each has a workgroup of its own (Plan::single; 300 of up to
// 250 positions, 4 heads of 128: 29 us, 59 in runs).  Otherwise the units of
// all sequences, one after another, make equal runs, so that ragged batches stay
// balanced (48 sequences of 8000 to 16000 positions: 253 -> 228 us against runs
// that end with their sequence).  A run that holds a sequence's every unit
// writes its result; of the others a run leaves two partials at most: that of
// the sequence it goes on with (slot 2 run) and that of the one it begins and
// does not end (slot 2 run + 1), whatever the number of sequences.

constexpr int kUnit = 128;
constexpr int kAttnWaves = 4;
constexpr int kMaxQueryRows = 8;
constexpr uint32_t kShortRuns = 4;  // units for each run, below which sequences are short
constexpr uint32_t kFewUnits = 4;   // of a sequence that a workgroup takes alone whatever the others are
// Where such workgroups fill the device, a sequence may have 1.5 times the equal share of a run and 12 units, 8
// where they fill half of it: runs that cross sequences and their joins cost more than that much unevenness
// (4 heads of 128; alone / in runs, us: 32 of up to 1000 positions 18 / 21, 64 24 / 35, 64 of 4000 79 / 82, of
// 16000 291 / 271; 300 of 250 29 / 50, of 3000 236 / 254; 63 of 100 and one of 4096 47 / 15).
constexpr uint32_t kUnevenHalves = 3, kUnevenUnits = 12, kUnevenUnitsHalf = 8;

struct AttnArgs {
    Pages p;
    const uint16_t* q;
    uint16_t* out;     // [sequences][rows][heads][head_dim]
    float* part;       // [slot][head and column block][column][head_dim], then the maxima and sums
    float* part_ml;
    uint4* plan;       // {total, runs, align, single}, then {before, units} of each sequence (uint2); null: no join
    int64_t q_seq, q_row, q_head;  // strides, values
    int64_t capacity;  // positions of a table row
    int rows;
    int heads;
    int kv_heads;
    int group;         // query heads per kv head
    int head_dim;
    int columns;       // rows * group: column r * group + h is row r, head h of the group
    int column_blocks;
    uint32_t budget;      // runs of long sequences
    uint32_t short_runs;  // runs of short ones, about
    int single;           // no table row holds more than a few units: each sequence has a workgroup
    uint32_t uneven;      // units of a sequence more than its share that a workgroup may take; 0: never
    uint32_t streamed;    // units from which on the values are read past the caches
    float scale;       // softmax scale * log2(e)
};

// Positions that the last row of sequence b sees.
__device__ __forceinline__ int64_t seen_of(int length, int rows, int64_t capacity) {
    return length < 0 ? 0 : min(static_cast<int64_t>(length) + rows, capacity);
}

__device__ __forceinline__ uint32_t units_of(int length, int rows, int64_t capacity) {
    return max(1u, static_cast<uint32_t>((seen_of(length, rows, capacity) + kUnit - 1) / kUnit));
}

// Inclusive prefix sum over the lanes of a wave (DPP, no LDS).
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v) {
#define PLM_PREFIX(ctrl, rows) \
    v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), ctrl, rows, 0xF, false))
    PLM_PREFIX(0x111, 0xF);  // row_shr:1, 2, 4, 8
    PLM_PREFIX(0x112, 0xF);
    PLM_PREFIX(0x114, 0xF);
    PLM_PREFIX(0x118, 0xF);
    PLM_PREFIX(0x142, 0xA);  // row_bcast:15 into rows 1 and 3
    PLM_PREFIX(0x143, 0xC);  // row_bcast:31 into rows 2 and 3
#undef PLM_PREFIX
    return v;
}

struct Plan {
    uint32_t total;   // units of all sequences, each rounded up to whole multiples of `align`
    uint32_t runs;
    uint32_t align;
    bool single;      // run r is sequence r
    int seq;
    uint32_t before;  // units of the sequences before seq, rounded
    uint32_t units;   // of seq

    __device__ __forceinline__ uint32_t rounded(uint32_t n) const {
        return align == 1 ? n : (n + align - 1) / align * align;
    }
    // run * total / runs
    __device__ __forceinline__ uint32_t start(uint32_t run) const {
        if (total == runs * align) return run * align;
        const uint32_t each = total / runs;
        return run * each + run * (total - each * runs) / runs;
    }
    // The run that holds a unit: the last that starts at or before it.
    __device__ __forceinline__ uint32_t run_of(uint32_t unit) const {
        if (total == runs * align) return unit / align;
        return static_cast<uint32_t>(((static_cast<uint64_t>(unit) + 1) * runs + total - 1) / total - 1);
    }
};

// Of the lanes of a wave (lane 63 has it).
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#define PLM_MAX(ctrl, rows) \
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), ctrl, rows, 0xF, false)))
    PLM_MAX(0x111, 0xF);
    PLM_MAX(0x112, 0xF);
    PLM_MAX(0x114, 0xF);
    PLM_MAX(0x118, 0xF);
    PLM_MAX(0x142, 0xA);
    PLM_MAX(0x143, 0xC);
#undef PLM_MAX
    return __builtin_amdgcn_readlane(v, 63);
}

// The plan, at the sequence that holds the first unit of run `run`.  Every
// thread of a workgroup calls it; false for a run past the last.  (Kept short:
// a small call waits for its instructions as for its data.)
constexpr int kHeld = 2048;  // sequences whose units are read once
__device__ __forceinline__ bool find_plan(const AttnArgs& a, int lane, uint32_t run, uint32_t* held, Plan& plan) {
    const uint32_t n0 = lane < a.p.sequences ? units_of(a.p.lengths[lane], a.rows, a.capacity) : 0;
    if (a.p.sequences > 64) {
        for (int i = threadIdx.x; i < min(a.p.sequences, kHeld); i += 64 * kAttnWaves)
            held[i] = units_of(a.p.lengths[i], a.rows, a.capacity);
        __syncthreads();
    }
    auto units_at = [&](int base) {
        if (base == 0) return n0;
        const int i = base + lane;
        return i >= a.p.sequences ? 0 : base < kHeld ? held[i] : units_of(a.p.lengths[i], a.rows, a.capacity);
    };
    uint32_t longest = 0;
    auto sum = [&] {
        uint32_t mine = 0;
#pragma unroll 1
        for (int base = 0; base < a.p.sequences; base += 64) {
            const uint32_t n = units_at(base);
            mine += plan.rounded(n);
            longest = max(longest, n);
        }
        return static_cast<uint32_t>(__builtin_amdgcn_readlane(wave_prefix(mine), 63));
    };
    // A workgroup for each sequence; or, of long sequences, `budget` equal runs, as many as there is room
    // for; or, of short ones, runs of `align` units that end with their sequence (starting on another costs
    // more than a unit or two), as many as there are compute units (their partials cost as well).
    plan.align = 1;
    plan.total = sum();
    longest = wave_max(longest);
    const uint64_t most = 2 * a.uneven * a.budget + kUnevenHalves * static_cast<uint64_t>(plan.total);
    plan.single = longest <= kFewUnits || (a.uneven > 0 && 2 * static_cast<uint64_t>(longest) * a.budget <= most);
    plan.runs = plan.single ? a.p.sequences : a.budget;
    if (!plan.single && plan.total < kShortRuns * a.budget) {
        plan.align = max(1u, (plan.total + a.short_runs - 1) / a.short_runs);
        if (plan.align > 1) plan.total = sum();
        plan.runs = plan.total / plan.align;
    }
    if (run >= plan.runs) return false;
    if (plan.single) {
        plan.seq = static_cast<int>(run);
        plan.before = 0;
        plan.units = units_of(a.p.lengths[run], a.rows, a.capacity);
        return true;
    }
    const uint32_t unit = plan.start(run);
    uint32_t before = 0;
#pragma unroll 1
    for (int base = 0; base < a.p.sequences; base += 64) {
        const uint32_t n = units_at(base);
        const uint32_t upto = wave_prefix(plan.rounded(n));
        const unsigned long long past = __ballot(before + upto > unit);
        if (past != 0) {
            const int at = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
            plan.seq = base + at;
            plan.units = __builtin_amdgcn_readlane(n, at);
            plan.before = before + __builtin_amdgcn_readlane(upto, at) - plan.rounded(plan.units);
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

__device__ __forceinline__ float swap_max(float v) {
    // over the four lanes l, l ^ 16, l ^ 32, l ^ 48
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float swap_sum(float v) {
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(h[0]) + __uint_as_float(h[1]);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <bool BF16>
__device__ __forceinline__ f32x4 mfma16(const u32x4 a, const u32x4 b, const f32x4 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
}

// exp2(x - m) for a running maximum that may be -inf (nothing seen yet).
__device__ __forceinline__ float exp2_from(float x, float m) { return exp2f(x - (m == -INFINITY ? 0.0f : m)); }

// Two weights as sums of two values of the cache's type each: cut off, so that
// the rest is not negative, and the rest, rounded; together they keep 15 bits
// (fp16 21) of each weight.  The rest of a weight above 0 is not 0: times an
// infinity 0 is NaN, as is the sum of infinities of both signs.
struct Halves {
    uint32_t high, low;
};
template <bool BF16>
__device__ __forceinline__ Halves halves(float a, float b) {
    if constexpr (BF16) {
        const uint32_t ia = __float_as_uint(a), ib = __float_as_uint(b);
        const float ra = a - __uint_as_float(ia & 0xFFFF0000u), rb = b - __uint_as_float(ib & 0xFFFF0000u);
        return {__builtin_amdgcn_perm(ib, ia, 0x07060302u),
                pack2<true>(__builtin_amdgcn_fmed3f(ra, a, 0x1p-126f), __builtin_amdgcn_fmed3f(rb, b, 0x1p-126f))};
    } else {
        const f16x2 high = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(a, b));
        const float ra = a - static_cast<float>(high[0]), rb = b - static_cast<float>(high[1]);
        return {__builtin_bit_cast(uint32_t, high),
                pack2<false>(__builtin_amdgcn_fmed3f(ra, a, 0x1p-24f), __builtin_amdgcn_fmed3f(rb, b, 0x1p-24f))};
    }
}

constexpr uint32_t kNoRow = 0xFFFFFFFFu;

// Workgroup (run, kv head, column block): for each sequence of the run, 4
// waves take every fourth tile of 32 positions, each with a running maximum and
// sum of its own; they meet in LDS at the end.
//
//   scores  S^T = K Q^T: A holds 16 positions x 32 head values as they lie in
//           the cache, B the 16 columns' queries; a lane gets, of column
//           l & 15, four positions of each half tile
//   values  O^T = V^T P^T: B is those eight weights as they are, so A's eight
//           positions are the same: a lane loads eight whole pieces of 8 head
//           values (adjacent lanes adjacent pieces: a position's row at once)
//           and transposes 8 x 8 values by register permutes.  Matrix
//           instruction i has head values 8 r + i in its row r.
//
// Weights go to the second product as two values of the cache's type each
// (halves below), so that the result is as close to 64 bits as with fp32
// weights: rounded once, the error is 2.1e-3 of the results' size in bf16 and
// 2.6e-4 in fp16, so 1.66e-3 and 2.07e-4, which are the output's rounding.  The
// second instruction waits for memory with the first (48 sequences of 8000 to
// 16000 positions 211.5 us with one, 211.7 with two; 6 of 5000 with 4 rows each
// 23.0, 23.7).  In fp16 weights are kept times 2^15, so that a weight is only
// lost below 2^-40 of the row's largest.
//
// Bound by the cache's bytes in large batches: 48 sequences of 8000 to 16000
// positions, 4 key-value heads of 128, 1.2 GB 212 us with the join, 5.7 TB/s.
// Small calls are a chain of trips to memory, lengths, table, keys and values,
// then the join: 700 positions 7.6 + 4.7 us, 6 sequences of up to 5000 positions
// with 4 rows each, 49 MB, 18.6 + 5.0 us.
//
// DP: head_dim rounded up to 64, 128 or 256; EXACT: no rounding.  CT: blocks
// of 16 columns, 1 or 2.  More have workgroups of their own which read the same
// through an L2 that they share: with 4 in a workgroup, one wave a SIMD, 8 rows
// of 7 heads took 29 us for 700 positions and 137 for 50 sequences of 4000, now
// 17 and 108.
template <bool BF16, int DP, bool EXACT, int CT>
__global__ __launch_bounds__(64 * kAttnWaves, DP > 128 ? 1 : 2) void paged_attention_kernel(
    const AttnArgs a) {
    constexpr int KS = DP / 32;               // score steps of 32 head values
    constexpr int NV = DP / 16;               // value instructions
    constexpr int PV = DP == 64 ? 4 : 8;      // adjacent head values of a lane
    constexpr int SETS = NV / PV;             // pieces of a lane per position
    constexpr float kBias = BF16 ? 0.0f : 15.0f;
    __shared__ float meet[2][CT * (NV * 4 + 2)][64];  // at most 35 KB
    __shared__ uint32_t held[kHeld];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hc_count = a.kv_heads * a.column_blocks;
    // The column blocks of a run and head are eight workgroups apart: those are dispatched to one XCD.
    int block = 0, pair = blockIdx.x;  // of run and head
    if (a.column_blocks > 1) {
        const uint32_t pairs = gridDim.x / a.column_blocks;
        const uint32_t group = blockIdx.x / (8 * a.column_blocks), rest = blockIdx.x - group * 8 * a.column_blocks;
        const uint32_t together = min(8u, pairs - 8 * group);
        block = rest / together;
        pair = 8 * group + (rest - block * together);
    }
    const int run = pair / a.kv_heads, kvh = pair - run * a.kv_heads;
    const int hc = kvh * a.column_blocks + block, col0 = block * 16 * CT;
    Plan plan;
    uint32_t unit = 0, run_end;
    if (a.single != 0) {
        plan.align = 1;
        plan.seq = run;
        plan.before = 0;
        plan.units = units_of(a.p.lengths[run], a.rows, a.capacity);
        plan.total = plan.units * static_cast<uint32_t>(a.p.sequences);  // about
        run_end = plan.units;
    } else {
        if (!find_plan(a, lane, static_cast<uint32_t>(run), &held[0], plan)) return;
        unit = plan.single ? 0 : plan.start(run);
        run_end = plan.single ? plan.units : plan.start(run + 1);
        if (blockIdx.x == 0 && threadIdx.x == 0) *a.plan = make_uint4(plan.total, plan.runs, plan.align, plan.single);
    }
    const bool streamed = EXACT && DP >= 128 && plan.total >= a.streamed;
    const bool noted = a.single == 0 && !plan.single && hc == 0 && threadIdx.x == 0;
    int seq = plan.seq;
    uint32_t before = plan.before;
    uint32_t units = plan.units;
    while (unit < run_end) {  // a sequence of the run's
        const int length = a.p.lengths[seq];
        const int seen = static_cast<int>(seen_of(length, a.rows, a.capacity));
        if (noted && unit == before) reinterpret_cast<uint2*>(a.plan + 1)[seq] = make_uint2(before, units);
        const bool whole = unit == before && run_end >= before + units;
        const int begin = static_cast<int>(unit - before) * kUnit;
        const int end = min(seen, static_cast<int>(min(run_end - before, units)) * kUnit);

        // The lane's place anew for each sequence: what follows from it is not kept in registers over the
        // others.
        int again = lane;
        asm volatile("" : "+v"(again));
        const int li = again & 15, g = again >> 4;
        // this lane's columns: queries, and the positions that each sees
        u32x4 q[CT][KS];
        int limit[CT];
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const int col = col0 + 16 * t + li;
            const int r = min(col, a.columns - 1) / a.group, h = min(col, a.columns - 1) - r * a.group;
            const uint16_t* src = a.q + seq * a.q_seq + r * a.q_row + (kvh * a.group + h) * a.q_head;
            limit[t] = col < a.columns ? static_cast<int>(seen_of(length, r + 1, a.capacity)) : 0;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = 32 * s + 8 * g;
                q[t][s] = *reinterpret_cast<const u32x4*>(src + (EXACT || d < a.head_dim ? d : 0));
                if (col >= a.columns || (!EXACT && d >= a.head_dim)) q[t][s] = u32x4{0, 0, 0, 0};
            }
        }
        const int least = static_cast<int>(seen_of(length, 1, a.capacity));  // what every row sees
        const uint16_t* kbase = a.p.k + kvh * a.p.head_stride;
        const uint16_t* vbase = a.p.v + kvh * a.p.head_stride;
        const int* table = a.p.table + static_cast<int64_t>(seq) * a.p.table_cols;

        float m[CT], l[CT];
        f32x4 acc[CT][NV];
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            m[t] = -INFINITY;
            l[t] = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i) acc[t][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        // lane l looks up position t0 + (l & 31) of a tile
        auto page_of = [&](int t0) {
            const int pos = min(t0 + (lane & 31), seen - 1);
            return table[static_cast<uint32_t>(pos) / a.p.page_size];
        };
        auto row_of = [&](int page, int t0) {
            const int pos = t0 + (lane & 31);
            const uint32_t slot = static_cast<uint32_t>(pos) % a.p.page_size;
            const bool there = pos < end && page >= 0 && static_cast<uint32_t>(page) < a.p.num_pages;
            return there ? static_cast<uint32_t>(page) * a.p.page_stride + slot * a.p.slot_stride : kNoRow;
        };
        u32x4 k[2][KS];
        u32x4 v[8][SETS];
        auto load_k = [&](uint32_t row) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t o = __shfl(row, 16 * i + li);
                // a position that is not there reads the cache's first row; its score is replaced
                const uint16_t* src = kbase + static_cast<int64_t>(o == kNoRow ? 0u : o) * 8;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const int d = 32 * s + 8 * g;
                    k[i][s] = *reinterpret_cast<const u32x4*>(src + (EXACT || d < a.head_dim ? d : 0));
                    if (!EXACT && d >= a.head_dim) k[i][s] = u32x4{0, 0, 0, 0};
                }
            }
        };
        uint32_t vrow[8];
        auto load_v = [&](uint32_t row, auto nontemporal) {
            constexpr bool past = decltype(nontemporal)::value;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                vrow[j] = __shfl(row, (j < 4 ? 0 : 12) + 4 * g + j);
                const uint16_t* src = vbase + static_cast<int64_t>(vrow[j] == kNoRow ? 0u : vrow[j]) * 8;
#pragma unroll
                for (int s = 0; s < SETS; ++s) {
                    const int d = PV * li + 128 * s;
                    const uint16_t* at = src + (EXACT || d < a.head_dim ? d : 0);
                    if constexpr (PV == 8) {
                        v[j][s] = past ? __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at))
                                       : *reinterpret_cast<const u32x4*>(at);
                    } else {
                        const u32x2 two = *reinterpret_cast<const u32x2*>(at);
                        v[j][s] = u32x4{two.x, two.y, 0, 0};
                    }
                    if (!EXACT && d >= a.head_dim) v[j][s] = u32x4{0, 0, 0, 0};
                }
            }
        };
        // eight positions of head value PV s + i of the lane's pieces
        auto across = [&](int s, int i) {
            const uint32_t pick = (i & 1) ? 0x07060302u : 0x05040100u;
            u32x4 t;
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = __builtin_amdgcn_perm(v[2 * j + 1][s][i >> 1], v[2 * j][s][i >> 1], pick);
            return t;
        };

        int t0 = begin + 32 * wave;
        if (t0 < end) {
            uint32_t row = row_of(page_of(t0), t0);
            load_k(row);
            load_v(row, std::false_type{});
            int page = page_of(t0 + kUnit);
            for (; t0 < end; t0 += kUnit) {
                // past the range: no position is there, every lane reads the cache's first row
                const uint32_t next = row_of(page, t0 + kUnit);
                page = page_of(t0 + 2 * kUnit);
                f32x4 s[CT][2];
#pragma unroll
                for (int t = 0; t < CT; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        s[t][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int x = 0; x < KS; ++x) s[t][i] = mfma16<BF16>(k[i][x], q[t][x], s[t][i]);
                    }
#pragma unroll
                for (int t = 0; t < CT; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) s[t][i] = s[t][i] * a.scale;
                __builtin_amdgcn_sched_barrier(0);
                load_k(next);
                const bool full = t0 + 32 <= least && __all(row != kNoRow);
                // A row that sees a position has a maximum of at least the lowest number, one that sees
                // none keeps -inf: its result is 0, while scores that are all -inf give 0 / 0.
                float floor[CT];
#pragma unroll
                for (int t = 0; t < CT; ++t) floor[t] = full ? -FLT_MAX : -INFINITY;
                if (!full) {
#pragma unroll
                    for (int t = 0; t < CT; ++t)
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int pos = t0 + (j < 4 ? 0 : 12) + 4 * g + j;
                            if (pos >= limit[t] || vrow[j] == kNoRow)
                                s[t][j >> 2][j & 3] = -INFINITY;
                            else
                                floor[t] = -FLT_MAX;
                        }
                }
                u32x4 w[CT], w_low[CT];
#pragma unroll
                for (int t = 0; t < CT; ++t) {
                    float top = fmaxf(fmaxf(fmaxf(s[t][0][0], s[t][0][1]), fmaxf(s[t][0][2], s[t][0][3])),
                                      fmaxf(fmaxf(s[t][1][0], s[t][1][1]), fmaxf(s[t][1][2], s[t][1][3])));
                    top = fmaxf(m[t], swap_max(fmaxf(top, floor[t])));
                    const float fade = exp2_from(m[t], top);
                    m[t] = top;
                    const float from = top == -INFINITY ? 0.0f : top;
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            // the bias last: a score of 2^24 or more has no room for it
                            s[t][i][j] = exp2f((s[t][i][j] - from) + kBias);
                            sum += s[t][i][j];
                        }
                    l[t] = fmaf(l[t], fade, sum);
#pragma unroll
                    for (int i = 0; i < NV; ++i) acc[t][i] = acc[t][i] * fade;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const Halves x = halves<BF16>(s[t][i >> 1][2 * (i & 1)], s[t][i >> 1][2 * (i & 1) + 1]);
                        w[t][i] = x.high;
                        w_low[t][i] = x.low;
                    }
                }
                if (!full) {
                    // What a row does not see has weight 0, but 0 times a NaN or an infinity left there is
                    // NaN: only what every row sees goes to the matrix cores.
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int pos = t0 + (j < 4 ? 0 : 12) + 4 * g + j;
                        const uint32_t keep = pos < least && vrow[j] != kNoRow ? 0xFFFFFFFFu : 0u;
#pragma unroll
                        for (int x = 0; x < SETS; ++x) v[j][x] = v[j][x] & keep;
                    }
                }
#pragma unroll
                for (int x = 0; x < SETS; ++x)
#pragma unroll
                    for (int i = 0; i < PV; ++i) {
                        const u32x4 values = across(x, i);
#pragma unroll
                        for (int t = 0; t < CT; ++t)
                            acc[t][PV * x + i] =
                                mfma16<BF16>(values, w_low[t], mfma16<BF16>(values, w[t], acc[t][PV * x + i]));
                    }
                // the positions that some of the rows see, at most rows - 1 of them, one at a time
                for (int pos = max(least, t0); pos < min(t0 + 32, seen); ++pos) {
                    const uint32_t there = __builtin_amdgcn_readlane(row, pos - t0);
                    if (there == kNoRow) continue;
                    const int at = pos - t0, from = (at & 12) * 4 + li;  // the lane that has this column's weight of it
                    u32x4 value[SETS][4];
                    const uint16_t* src = vbase + static_cast<int64_t>(there) * 8;
#pragma unroll
                    for (int x = 0; x < SETS; ++x)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int d = PV * (4 * g + j) + 128 * x;
                            const uint16_t* piece = src + (EXACT || d < a.head_dim ? d : 0);
                            if constexpr (PV == 8) {
                                value[x][j] = *reinterpret_cast<const u32x4*>(piece);
                            } else {
                                const u32x2 two = *reinterpret_cast<const u32x2*>(piece);
                                value[x][j] = u32x4{two.x, two.y, 0, 0};
                            }
                        }
#pragma unroll
                    for (int t = 0; t < CT; ++t) {
                        float p = s[t][0][0];
#pragma unroll
                        for (int j = 1; j < 8; ++j) p = (at >> 4) * 4 + (at & 3) == j ? s[t][j >> 2][j & 3] : p;
                        p = __shfl(p, from);
                        const bool sees = pos < limit[t];
#pragma unroll
                        for (int x = 0; x < SETS; ++x)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const f32x8 f = widen8<BF16>(value[x][j]);
#pragma unroll
                                for (int i = 0; i < PV; ++i) {
                                    const float was = acc[t][PV * x + i][j];
                                    acc[t][PV * x + i][j] = sees ? fmaf(p, f[i], was) : was;
                                }
                            }
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                if (streamed) {
                    asm volatile("");  // two sets of loads: merged into one they would all be ordinary ones
                    load_v(next, std::true_type{});
                    asm volatile("");
                } else {
                    load_v(next, std::false_type{});
                }
                row = next;
            }
        }
#pragma unroll
        for (int t = 0; t < CT; ++t) l[t] = swap_sum(l[t]);

        asm volatile("" : "+v"(again));
        {
        const int lane = again, li = again & 15, g = again >> 4;
        // the waves' parts: 2 and 3 into 0 and 1, then 1 into 0
#pragma unroll
        for (int step = 2; step > 0; step >>= 1) {
            if (wave >= step && wave < 2 * step) {
                float(*to)[64] = meet[wave - step];
#pragma unroll
                for (int t = 0; t < CT; ++t) {
                    to[t * (NV * 4 + 2)][lane] = m[t];
                    to[t * (NV * 4 + 2) + 1][lane] = l[t];
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) to[t * (NV * 4 + 2) + 2 + 4 * i + j][lane] = acc[t][i][j];
                }
            }
            __syncthreads();
            if (wave < step) {
                const float(*from)[64] = meet[wave];
#pragma unroll
                for (int t = 0; t < CT; ++t) {
                    const float om = from[t * (NV * 4 + 2)][lane], ol = from[t * (NV * 4 + 2) + 1][lane];
                    const float top = fmaxf(m[t], om);
                    const float f0 = exp2_from(m[t], top), f1 = exp2_from(om, top);
                    m[t] = top;
                    l[t] = l[t] * f0 + ol * f1;
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            acc[t][i][j] = acc[t][i][j] * f0 + from[t * (NV * 4 + 2) + 2 + 4 * i + j][lane] * f1;
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const int col = col0 + 16 * t + li;
            if (wave != 0 || col >= a.columns) continue;
            if (!whole) {
                const int64_t slot = 2 * static_cast<int64_t>(run) + (unit == before ? 1 : 0);
                const int64_t at = (slot * hc_count * CT + hc * CT + t) * 16 + li;
                if (g == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * at) = f32x2{m[t], l[t]};
                float* to = a.part + at * a.head_dim;
#pragma unroll
                for (int s = 0; s < SETS; ++s)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int d = PV * (4 * g + j) + 128 * s;
                        if (!EXACT && d >= a.head_dim) continue;
#pragma unroll
                        for (int i = 0; i < PV; i += 4)
                            *reinterpret_cast<f32x4*>(to + d + i) =
                                f32x4{acc[t][PV * s + i][j], acc[t][PV * s + i + 1][j], acc[t][PV * s + i + 2][j],
                                      acc[t][PV * s + i + 3][j]};
                    }
                continue;
            }
            // a row that sees nothing is zero
            const int r = col / a.group, h = col - r * a.group;
            const bool empty = m[t] == -INFINITY;
            const float inv = 1.0f / l[t];
            uint16_t* to = a.out + ((static_cast<int64_t>(seq) * a.rows + r) * a.heads + kvh * a.group + h) * a.head_dim;
#pragma unroll
            for (int s = 0; s < SETS; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int d = PV * (4 * g + j) + 128 * s;
                    if (!EXACT && d >= a.head_dim) continue;
#pragma unroll
                    for (int i = 0; i < PV; i += 4) {
                        u32x2 o;
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const float y0 = empty ? 0.0f : acc[t][PV * s + i + 2 * x][j] * inv;
                            const float y1 = empty ? 0.0f : acc[t][PV * s + i + 2 * x + 1][j] * inv;
                            o[x] = pack2<BF16>(y0, y1);
                        }
                        *reinterpret_cast<u32x2*>(to + d + i) = o;
                    }
                }
        }
        }
        unit = before += plan.rounded(units);
        if (unit < run_end) units = units_of(a.p.lengths[++seq], a.rows, a.capacity);
    }
}

// Joins the splits of a sequence, a workgroup per query row and head.  Its
// threads first take the splits' maxima and sums (the weights of the splits go
// to LDS), then each a quad of head values of every sets-th split, and the
// sets meet in LDS.  Sequences of one split were written already.  Bound by its
// launch and three trips to memory: 28 to 672 workgroups about 5 us, 48 x 28
// with 4 partials on average 7.4.
constexpr int kJoinThreads = 256;
constexpr int kJoinSplits = 1024;  // at a time

__device__ __forceinline__ float join_reduce(float v, bool is_max, float* red) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const float o = __shfl_xor(v, off);
        v = is_max ? fmaxf(v, o) : v + o;
    }
    if (lane == 0) red[wave] = v;
    __syncthreads();
    v = is_max ? fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])) : (red[0] + red[1]) + (red[2] + red[3]);
    __syncthreads();
    return v;
}

template <bool BF16>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(const AttnArgs a, int ct) {
    __shared__ float weights[kJoinSplits];
    __shared__ f32x4 sums[kJoinThreads];
    __shared__ float red[4];
    const int all = a.rows * a.heads;
    const int seq = blockIdx.x / all;
    const int at = blockIdx.x - seq * all;
    // as the first kernel left it; of no sequence where each had a workgroup
    const uint4 noted = *a.plan;
    const uint2 own = reinterpret_cast<const uint2*>(a.plan + 1)[seq];
    if (noted.w != 0) return;
    Plan plan;
    plan.total = noted.x;
    plan.runs = noted.y;
    plan.align = noted.z;
    // (within the runs also where the lengths were changed under the first kernel)
    const uint32_t run = min(plan.run_of(own.x), plan.runs - 1);
    const int splits = static_cast<int>(min(plan.run_of(own.x + own.y - 1), plan.runs - 1)) - static_cast<int>(run) + 1;
    if (splits <= 1) return;
    const int r = at / a.heads, head = at - r * a.heads;
    const int kvh = head / a.group, col = r * a.group + head - kvh * a.group;
    const int hc_count = a.kv_heads * a.column_blocks;
    const int wide = 16 * ct;
    const int hc = kvh * a.column_blocks + col / wide;
    // partial of split s: first + slot(s) * stride; the first split's is its run's second
    const int64_t stride = static_cast<int64_t>(hc_count) * wide;
    const int64_t first = (2 * static_cast<int64_t>(run) * hc_count + hc) * wide + col % wide;
    auto slot = [](int s) { return max(2 * s, 1); };
    const f32x2* ml = reinterpret_cast<const f32x2*>(a.part_ml) + first;
    float m = -INFINITY;
    for (int s = threadIdx.x; s < splits; s += kJoinThreads) m = fmaxf(m, ml[slot(s) * stride][0]);
    m = join_reduce(m, true, red);
    const int quads = a.head_dim / 4;  // threads of a set
    const int sets = kJoinThreads / quads;
    const int set = threadIdx.x / quads, d = 4 * (threadIdx.x - set * quads);
    const float* part = a.part + first * a.head_dim + d;
    float sum = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int base = 0; base < splits; base += kJoinSplits) {
        const int n = min(kJoinSplits, splits - base);
        if (base > 0) __syncthreads();
        for (int s = threadIdx.x; s < n; s += kJoinThreads) {
            const f32x2 v = ml[slot(base + s) * stride];
            const float w = exp2_from(v[0], m);
            weights[s] = w;
            sum = fmaf(v[1], w, sum);
        }
        __syncthreads();
        if (set < sets) {
#pragma unroll 4
            for (int s = set; s < n; s += sets) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(part + slot(base + s) * stride * a.head_dim);
                const float w = weights[s];
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] = fmaf(x[i], w, acc[i]);
            }
        }
    }
    sums[threadIdx.x] = acc;
    sum = join_reduce(sum, false, red);
    if (threadIdx.x >= quads) return;
    for (int s = 1; s < sets; ++s) acc = acc + sums[s * quads + threadIdx.x];
    const bool empty = m == -INFINITY;
    const float inv = 1.0f / sum;
    u32x2 o;
#pragma unroll
    for (int x = 0; x < 2; ++x)
        o[x] = empty ? 0u : pack2<BF16>(acc[2 * x] * inv, acc[2 * x + 1] * inv);
    *reinterpret_cast<u32x2*>(a.out + ((static_cast<int64_t>(seq) * a.rows + r) * a.heads + head) * a.head_dim + d) = o;
}

// ---------------------------------------------------------------- host side

constexpr int64_t kMostInt = 0x7FFFFFFF;
// Positions are ints, and the attention looks two units ahead of its last one.
constexpr int64_t kMostPositions = kMostInt - 1023;

// The checks and layout that both calls share; 0, or the code of the failure.
int pages_of(Pages& p, void* k_cache, void* v_cache, const int* page_table, const int* lengths, int64_t sequences,
             int64_t table_cols, int64_t num_pages, int64_t page_size, int64_t kv_heads, int64_t head_dim,
             int64_t page_stride, int64_t slot_stride, int64_t head_stride, int dtype_code) {
    if (k_cache == nullptr || v_cache == nullptr || page_table == nullptr || lengths == nullptr)
        return plm::fail(-1, "null pointer");
    if (sequences <= 0 || table_cols <= 0 || num_pages <= 0 || page_size <= 0 || kv_heads <= 0 || head_dim <= 0 ||
        sequences > 65535 || kv_heads > 65535 || num_pages > kMostInt || page_size > kMostInt ||
        table_cols > kMostPositions / page_size || (dtype_code != 0 && dtype_code != 1))
        return plm::fail(-2, "bad dimensions");
    if (head_dim % 8 != 0 || head_dim > 256) return plm::fail(-2, "head_dim must be a multiple of 8 up to 256");
    if (page_stride < 0 || slot_stride < 0 || head_stride < 0 || page_stride % 8 != 0 || slot_stride % 8 != 0 ||
        head_stride % 8 != 0 || !plm::aligned16(k_cache) || !plm::aligned16(v_cache))
        return plm::fail(-2, "cache strides and addresses must be multiples of 16 bytes");
    const double last = static_cast<double>(num_pages - 1) * static_cast<double>(page_stride / 8) +
                        static_cast<double>(page_size - 1) * static_cast<double>(slot_stride / 8);
    if (last >= 4294967295.0 || head_stride > (static_cast<int64_t>(1) << 40))
        return plm::fail(-2, "a cache spans at most 64 GiB");
    p = Pages{static_cast<uint16_t*>(k_cache),
              static_cast<uint16_t*>(v_cache),
              page_table,
              lengths,
              head_stride,
              static_cast<uint32_t>(page_stride / 8),
              static_cast<uint32_t>(slot_stride / 8),
              static_cast<uint32_t>(page_size),
              static_cast<uint32_t>(num_pages),
              static_cast<int>(table_cols),
              static_cast<int>(sequences)};
    return 0;
}

template <bool BF16>
void launch_append(const AppendArgs& a, int mode, dim3 grid, dim3 block, hipStream_t st) {
    switch (mode) {
        case kCopy: hipLaunchKernelGGL((paged_append_kernel<BF16, kCopy>), grid, block, 0, st, a); break;
        case kHalves: hipLaunchKernelGGL((paged_append_kernel<BF16, kHalves>), grid, block, 0, st, a); break;
        case kAdjacent: hipLaunchKernelGGL((paged_append_kernel<BF16, kAdjacent>), grid, block, 0, st, a); break;
        case kAny: hipLaunchKernelGGL((paged_append_kernel<BF16, kAny>), grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL((paged_append_kernel<BF16, kAnyAdjacent>), grid, block, 0, st, a); break;
    }
}

// A call that reads more than this reads its values past the caches, where they
// would displace what is read again (the same batch 226 -> 210 us, 5.8 TB/s;
// calls of 30 to 70 MB, which the last-level cache holds, are 3 % faster without).
constexpr int64_t kStreamedBytes = static_cast<int64_t>(128) << 20;
constexpr double kLittleBytes = 64.0 * (1 << 20);

struct AttnShape {
    int ct;             // blocks of 16 columns in a workgroup
    int column_blocks;
    int64_t budget;     // runs of long sequences
    int64_t short_runs; // of short ones, about
    int64_t runs;       // at most
    bool single;        // a run for each sequence
    uint32_t uneven;    // see AttnArgs
    bool joined;        // a sequence can be in more than one run
    int64_t slots;      // of partials
    size_t bytes;
};

AttnShape shape_of(int64_t sequences, int64_t rows, int64_t heads, int64_t kv_heads, int64_t head_dim,
                   int64_t capacity) {
    AttnShape s;
    const int64_t columns = rows * (heads / kv_heads);
    // Two blocks of columns share what a workgroup reads of the cache, unless all that the tables reach is
    // little for their columns (4 rows of 7 heads of 128, 4 kv heads, us with 1 / 2: 16000 positions 17.7 / 19.7,
    // 16 times 8192 78 / 63).
    const int64_t blocks = plm::ceil_div(columns, 16);
    const double reach = static_cast<double>(sequences * blocks) * static_cast<double>(capacity * kv_heads * head_dim * 4);
    s.ct = head_dim > 128 || blocks == 1 || reach <= kLittleBytes ? 1 : 2;
    s.column_blocks = static_cast<int>(plm::ceil_div(columns, 16 * s.ct));
    const int64_t hc = kv_heads * s.column_blocks;
    const int64_t units = std::max<int64_t>(1, plm::ceil_div(capacity, kUnit));
    // as many workgroups as the compute units hold at once, and as there are compute units
    const int resident = head_dim > 128 ? 1 : 2;
    s.budget = std::max<int64_t>(1, resident * plm::cu_count() / hc);
    s.short_runs = std::max<int64_t>(1, plm::cu_count() / hc);
    s.single = units <= kFewUnits;
    const int64_t groups = sequences * hc;
    s.uneven = groups >= plm::cu_count() ? kUnevenUnits : 2 * groups >= plm::cu_count() ? kUnevenUnitsHalf : 0;
    const int64_t shared = std::min(sequences * units, s.budget + std::min(sequences, kShortRuns * s.budget));
    s.runs = s.single ? sequences : std::max(sequences, shared);
    s.joined = !s.single;
    s.slots = s.joined ? 2 * shared : 0;
    s.bytes = static_cast<size_t>(s.slots) * hc * s.ct * 16 * (head_dim + 2) * sizeof(float);
    if (s.joined) s.bytes += sizeof(uint4) + sizeof(uint2) * sequences;
    return s;
}

template <bool BF16>
void launch_attention(const AttnArgs& a, const AttnShape& s, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(s.runs * a.kv_heads * a.column_blocks)), block(64 * kAttnWaves);
    const int d = a.head_dim;
#define PLM_ATTN(DP, EXACT, CT) hipLaunchKernelGGL((paged_attention_kernel<BF16, DP, EXACT, CT>), grid, block, 0, st, a)
    if (s.ct == 2) {
        if (d == 64)
            PLM_ATTN(64, true, 2);
        else if (d < 64)
            PLM_ATTN(64, false, 2);
        else if (d == 128)
            PLM_ATTN(128, true, 2);
        else
            PLM_ATTN(128, false, 2);
    } else {
        if (d == 64)
            PLM_ATTN(64, true, 1);
        else if (d < 64)
            PLM_ATTN(64, false, 1);
        else if (d == 128)
            PLM_ATTN(128, true, 1);
        else if (d < 128)
            PLM_ATTN(128, false, 1);
        else if (d == 256)
            PLM_ATTN(256, true, 1);
        else
            PLM_ATTN(256, false, 1);
    }
#undef PLM_ATTN
    if (s.joined)
        hipLaunchKernelGGL((paged_join_kernel<BF16>),
                           dim3(static_cast<unsigned>(a.p.sequences * a.rows * a.heads)), dim3(kJoinThreads), 0,
                           st, a, s.ct);
}

bool bad_heads(int64_t rows, int64_t heads, int64_t kv_heads) {
    return rows <= 0 || rows > kMaxQueryRows || heads <= 0 || heads > 65535 || kv_heads <= 0 || heads % kv_heads != 0;
}

}  // namespace

PLM_EXPORT int kv_paged_append_u16(const uint16_t* q, const uint16_t* k, const uint16_t* v, uint16_t* q_out,
                                   uint16_t* k_cache, uint16_t* v_cache, const int* page_table, const int* lengths,
                                   const int* row_starts, const double* rope_frequencies, int* rejected, int64_t rows,
                                   int64_t sequences, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                   int64_t rope_pairs, int interleaved, int64_t q_row_stride, int64_t q_head_stride,
                                   int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride,
                                   int64_t v_head_stride, int64_t table_cols, int64_t num_pages, int64_t page_size,
                                   int64_t page_stride, int64_t slot_stride, int64_t head_stride, int dtype_code) {
    if (k == nullptr || v == nullptr || (heads > 0 && (q == nullptr || q_out == nullptr)) ||
        (rope_pairs > 0 && rope_frequencies == nullptr))
        return plm::fail(-1, "null pointer");
    AppendArgs a = {};
    int code = pages_of(a.p, k_cache, v_cache, page_table, lengths, sequences, table_cols, num_pages, page_size,
                        kv_heads, head_dim, page_stride, slot_stride, head_stride, dtype_code);
    if (code != 0) return code;
    if (rows <= 0 || rows > kMostInt || heads < 0 || heads > 65535 || rope_pairs < 0 || 2 * rope_pairs > head_dim ||
        (row_starts == nullptr && rows % sequences != 0))
        return plm::fail(-2, "bad dimensions");
    auto whole = [](const void* at, int64_t row, int64_t head) {
        return plm::aligned16(at) && row >= 0 && head >= 0 && row % 8 == 0 && head % 8 == 0;
    };
    if ((heads > 0 && (!whole(q, q_row_stride, q_head_stride) || !plm::aligned16(q_out))) ||
        !whole(k, k_row_stride, k_head_stride) || !whole(v, v_row_stride, v_head_stride))
        return plm::fail(-2, "row strides and addresses must be multiples of 16 bytes");
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.q_row = q_row_stride;
    a.q_head = q_head_stride;
    a.k_row = k_row_stride;
    a.k_head = k_head_stride;
    a.v_row = v_row_stride;
    a.v_head = v_head_stride;
    a.row_starts = row_starts;
    a.freq = rope_frequencies;
    a.rejected = rejected;
    a.rows = rows;
    a.rows_per_sequence = static_cast<int>(row_starts == nullptr ? rows / sequences : 1);
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    a.head_dim = static_cast<int>(head_dim);
    a.pairs = static_cast<int>(rope_pairs);
    // whole pairs of pieces: 16 values a thread, each read once
    const bool whole_head = head_dim % 16 == 0 && (rope_pairs == 0 || 2 * rope_pairs == head_dim);
    const int mode = whole_head ? (rope_pairs == 0 ? kCopy : interleaved ? kAdjacent : kHalves)
                                : (interleaved ? kAnyAdjacent : kAny);
    const int64_t units = (heads + 2 * kv_heads) * (head_dim / (whole_head ? 16 : 8));
    a.units = static_cast<int>(units);
    const int64_t parts = plm::ceil_div(units, kAppendThreads);
    if (parts > 65535) return plm::fail(-2, "too many heads");
    const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>(parts));
    const dim3 block(static_cast<unsigned>(plm::ceil_div(plm::ceil_div(units, parts), 64) * 64));
    if (dtype_code == 1)
        launch_append<true>(a, mode, grid, block, plm::current_stream());
    else
        launch_append<false>(a, mode, grid, block, plm::current_stream());
    return plm::check_launch("kv_paged_append_u16");
}

PLM_EXPORT int64_t kv_paged_attention_scratch_bytes(int64_t sequences, int64_t rows, int64_t heads, int64_t kv_heads,
                                                    int64_t head_dim, int64_t capacity) {
    if (sequences <= 0 || sequences > 65535 || bad_heads(rows, heads, kv_heads) || head_dim <= 0 || head_dim > 256 ||
        capacity <= 0 || capacity > kMostPositions)
        return plm::fail(-2, "bad dimensions");
    return static_cast<int64_t>(shape_of(sequences, rows, heads, kv_heads, head_dim, capacity).bytes);
}

PLM_EXPORT int kv_paged_attention_decode_u16(const uint16_t* q, const uint16_t* k_cache, const uint16_t* v_cache,
                                             const int* page_table, const int* lengths, uint16_t* out, void* scratch,
                                             int64_t scratch_bytes, int64_t sequences, int64_t rows, int64_t heads,
                                             int64_t kv_heads, int64_t head_dim, int64_t q_seq_stride,
                                             int64_t q_row_stride, int64_t q_head_stride, int64_t table_cols,
                                             int64_t num_pages, int64_t page_size, int64_t page_stride,
                                             int64_t slot_stride, int64_t head_stride, float softmax_scale,
                                             int dtype_code) {
    if (q == nullptr || out == nullptr) return plm::fail(-1, "null pointer");
    AttnArgs a = {};
    const int code = pages_of(a.p, const_cast<uint16_t*>(k_cache), const_cast<uint16_t*>(v_cache), page_table, lengths,
                              sequences, table_cols, num_pages, page_size, kv_heads, head_dim, page_stride, slot_stride,
                              head_stride, dtype_code);
    if (code != 0) return code;
    if (bad_heads(rows, heads, kv_heads)) return plm::fail(-2, "bad dimensions");
    if (!plm::aligned16(q) || !plm::aligned16(out) || q_seq_stride < 0 || q_row_stride < 0 || q_head_stride < 0 ||
        q_seq_stride % 8 != 0 || q_row_stride % 8 != 0 || q_head_stride % 8 != 0)
        return plm::fail(-2, "query strides and addresses must be multiples of 16 bytes");
    a.capacity = table_cols * page_size;
    const AttnShape s = shape_of(sequences, rows, heads, kv_heads, head_dim, a.capacity);
    if (sequences * plm::ceil_div(a.capacity, kUnit) > kMostInt / 4 ||
        s.runs * kv_heads * s.column_blocks > kMostInt || sequences * rows * heads > kMostInt)
        return plm::fail(-2, "too many sequences, heads or pages");
    void* part = scratch;
    if (s.bytes > 0) {
        if (scratch == nullptr) {
            part = plm::workspace(s.bytes);
            if (part == nullptr) return -3;
        } else if (scratch_bytes < static_cast<int64_t>(s.bytes) || !plm::aligned16(scratch)) {
            return plm::fail(-3, "scratch must hold kv_paged_attention_scratch_bytes, 16-byte aligned");
        }
    }
    a.q = q;
    a.out = out;
    a.q_seq = q_seq_stride;
    a.q_row = q_row_stride;
    a.q_head = q_head_stride;
    a.rows = static_cast<int>(rows);
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    a.group = static_cast<int>(heads / kv_heads);
    a.head_dim = static_cast<int>(head_dim);
    a.columns = a.rows * a.group;
    a.column_blocks = s.column_blocks;
    a.budget = static_cast<uint32_t>(s.budget);
    a.short_runs = static_cast<uint32_t>(s.short_runs);
    a.single = s.single ? 1 : 0;
    a.uneven = s.uneven;
    a.streamed = static_cast<uint32_t>(kStreamedBytes / (kUnit * 4 * kv_heads * head_dim));
    a.scale = softmax_scale * 1.44269504088896340736f;
    a.part = static_cast<float*>(part);
    a.part_ml = a.part + s.slots * kv_heads * s.column_blocks * s.ct * 16 * head_dim;
    // whole vectors of 16 bytes before it: 16 columns or more of head_dim + 2 values
    a.plan = s.joined ? reinterpret_cast<uint4*>(a.part_ml + s.slots * kv_heads * s.column_blocks * s.ct * 32) : nullptr;
    const hipStream_t st = plm::current_stream();
    if (dtype_code == 1)
        launch_attention<true>(a, s, st);
    else
        launch_attention<false>(a, s, st);
    return plm::check_launch("kv_paged_attention_decode_u16");
}
