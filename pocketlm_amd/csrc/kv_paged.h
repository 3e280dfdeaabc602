// What the paged cache's kernels share (kv_paged.hip, kv_paged_norm.hip,
// kv_paged_chunk.hip): types and conversions, where the pages are, the place of
// an appended row, and the host's checks.
#pragma once

#include "common.h"

namespace plm_paged {

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

// The two e4m3 values of a dword's half, and eight of a piece's, as bf16 or fp16 (exact).
template <bool BF16>
__device__ __forceinline__ uint32_t pair_of(uint32_t four, bool upper) {
    if constexpr (BF16)
        return upper ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, 1.0f, true))
                     : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, 1.0f, false));
    else
        return upper ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(four, 1.0f, true))
                     : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(four, 1.0f, false));
}
template <bool BF16>
__device__ __forceinline__ u32x4 eight_of(const u32x4 piece, int half) {
    return u32x4{pair_of<BF16>(piece[2 * half], false), pair_of<BF16>(piece[2 * half], true),
                 pair_of<BF16>(piece[2 * half + 1], false), pair_of<BF16>(piece[2 * half + 1], true)};
}

// Where the pages are.  Strides in pieces of 16 bytes (8 values, 16 of e4m3):
// 32 bits reach 64 GiB; the head's offset is added in 64 bits.
struct Pages {
    uint16_t* k;  // of e4m3 caches: their bytes
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

// The scales of e4m3 caches: a position's and head's at page * page_stride +
// head * head_stride + slot, which 32 bits reach.
struct Scales {
    float* k;
    float* v;
    uint32_t page_stride;
    uint32_t head_stride;

    __device__ __forceinline__ uint32_t at(int page, int head, uint32_t slot) const {
        return static_cast<uint32_t>(page) * page_stride + static_cast<uint32_t>(head) * head_stride + slot;
    }
};

// Where row `row` of a call goes.  Every lane of a wave calls it.
struct Place {
    int64_t pos;   // of the sequence, -1: of none or an idle one
    uint32_t page;
    uint32_t slot;
    bool stored;   // there is a page for it
};
// (row `in_seq` of the call's rows of sequence `seq`)
__device__ __forceinline__ Place place_in(const Pages& p, int seq, int64_t in_seq) {
    const bool in_batch = seq >= 0 && seq < p.sequences;
    const int length = in_batch ? p.lengths[seq] : -1;
    Place at;
    at.pos = length >= 0 ? length + in_seq : -1;
    at.stored = false;
    at.page = at.slot = 0;
    if (at.pos >= 0) {
        const int64_t index = at.pos / p.page_size;
        if (index < p.table_cols) {
            const int page = p.table[static_cast<int64_t>(seq) * p.table_cols + index];
            at.stored = page >= 0 && static_cast<uint32_t>(page) < p.num_pages;
            at.page = static_cast<uint32_t>(page);
            at.slot = static_cast<uint32_t>(at.pos - index * p.page_size);
        }
    }
    return at;
}
__device__ __forceinline__ Place place_of(const Pages& p, const int* row_starts, int rows_per_sequence, int64_t row,
                                          int lane) {
    int seq;
    int64_t in_seq;
    if (row_starts != nullptr) {
        int count = 0;  // starts at or before the row
        for (int base = 0; base <= p.sequences; base += 64) {
            const int i = base + lane;
            const bool before = i <= p.sequences && row_starts[min(i, p.sequences)] <= row;
            count += __popcll(__ballot(before));
        }
        seq = count - 1;
        in_seq = seq >= 0 ? row - row_starts[min(seq, p.sequences)] : 0;
    } else {
        seq = static_cast<int>(row / rows_per_sequence);
        in_seq = row - static_cast<int64_t>(seq) * rows_per_sequence;
    }
    return place_in(p, seq, in_seq);
}

// The same of `count` rows from `row` on, lane r having row r's (the lanes behind them the last one's).
__device__ __forceinline__ Place places_of(const Pages& p, const int* row_starts, int rows_per_sequence, int64_t row,
                                           int count, int lane) {
    int seq;
    int64_t in_seq;
    const int mine = min(lane, count - 1);
    if (row_starts != nullptr) {
        int starts = 0;
        for (int base = 0; base <= p.sequences; base += 64) {
            const int i = base + lane;
            const int start = row_starts[min(i, p.sequences)];
            for (int r = 0; r < count; ++r) {
                const int before = __popcll(__ballot(i <= p.sequences && start <= row + r));
                starts += mine == r ? before : 0;
            }
        }
        seq = starts - 1;
        in_seq = seq >= 0 ? row + mine - row_starts[min(seq, p.sequences)] : 0;
    } else {
        seq = static_cast<int>((row + mine) / rows_per_sequence);
        in_seq = row + mine - static_cast<int64_t>(seq) * rows_per_sequence;
    }
    return place_in(p, seq, in_seq);
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

// The maximum over the lanes of a wave.
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

constexpr int64_t kMostInt = 0x7FFFFFFF;
// Positions are ints, and the attention looks two units ahead of its last one.
constexpr int64_t kMostPositions = kMostInt - 1023;

// The checks and layout that the calls share; 0, or the code of the failure.
// VALUES: a piece's, 8 of 16 bits or 16 of e4m3.
template <int VALUES = 8>
inline int pages_of(Pages& p, void* k_cache, void* v_cache, const int* page_table, const int* lengths,
                    int64_t sequences, int64_t table_cols, int64_t num_pages, int64_t page_size, int64_t kv_heads,
                    int64_t head_dim, int64_t page_stride, int64_t slot_stride, int64_t head_stride, int dtype_code) {
    if (k_cache == nullptr || v_cache == nullptr || page_table == nullptr || lengths == nullptr)
        return plm::fail(-1, "null pointer");
    if (sequences <= 0 || table_cols <= 0 || num_pages <= 0 || page_size <= 0 || kv_heads <= 0 || head_dim <= 0 ||
        sequences > 65535 || kv_heads > 65535 || num_pages > kMostInt || page_size > kMostInt ||
        table_cols > kMostPositions / page_size || (dtype_code != 0 && dtype_code != 1))
        return plm::fail(-2, "bad dimensions");
    if (head_dim % VALUES != 0 || head_dim > 256)
        return plm::fail(-2, "head_dim must be a multiple of %d up to 256", VALUES);
    if (page_stride < 0 || slot_stride < 0 || head_stride < 0 || page_stride % VALUES != 0 ||
        slot_stride % VALUES != 0 || head_stride % VALUES != 0 || !plm::aligned16(k_cache) || !plm::aligned16(v_cache))
        return plm::fail(-2, "cache strides and addresses must be multiples of 16 bytes");
    const double last = static_cast<double>(num_pages - 1) * static_cast<double>(page_stride / VALUES) +
                        static_cast<double>(page_size - 1) * static_cast<double>(slot_stride / VALUES);
    if (last >= 4294967295.0 || head_stride > (static_cast<int64_t>(1) << 40))
        return plm::fail(-2, "a cache spans at most 64 GiB");
    p = Pages{static_cast<uint16_t*>(k_cache),
              static_cast<uint16_t*>(v_cache),
              page_table,
              lengths,
              head_stride,
              static_cast<uint32_t>(page_stride / VALUES),
              static_cast<uint32_t>(slot_stride / VALUES),
              static_cast<uint32_t>(page_size),
              static_cast<uint32_t>(num_pages),
              static_cast<int>(table_cols),
              static_cast<int>(sequences)};
    return 0;
}

// The scales of e4m3 caches whose pages are known; 0, or the code of the failure.
inline int scales_of(Scales& s, const Pages& p, int64_t kv_heads, float* k_scales, float* v_scales, int64_t page_stride,
                     int64_t head_stride) {
    if (k_scales == nullptr || v_scales == nullptr) return plm::fail(-1, "null pointer");
    if (page_stride < 0 || head_stride < 0) return plm::fail(-2, "bad strides of the scales");
    const double last = static_cast<double>(p.num_pages - 1) * static_cast<double>(page_stride) +
                        static_cast<double>(kv_heads - 1) * static_cast<double>(head_stride) + p.page_size;
    if (last >= 4294967296.0) return plm::fail(-2, "scales span at most 16 GiB");
    s = Scales{k_scales, v_scales, static_cast<uint32_t>(page_stride), static_cast<uint32_t>(head_stride)};
    return 0;
}

}  // namespace plm_paged
