// Attention of any number of new rows of each sequence over its pages: whole
// prompts, chunks of them, single tokens among them, packed one sequence after
// another.  Row i of sequence b sees positions 0 .. lengths[b] + i:
//
//   out = sum_p exp(s_p - max s) v_p / sum_p exp(s_p - max s),  s_p = scale q . k_p
//
// in one pass over the positions with the running maximum and sum of the
// softmax.  A column is one row of one query head; column r * group + h of a
// sequence and key-value head is row r, head h of the group, so that a tile of
// keys and values is read once for the whole group.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "kv_paged.h"

namespace {

using namespace plm_paged;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kTile = 64;  // positions, one for each lane that looks up their pages
// A running maximum is only moved once a score is more than 2^kLate above it: weights grow to 2^kLate, the
// accumulators are multiplied in a few tiles instead of all.
constexpr float kLate = 8.0f;
// fp16 weights are kept times 2^7, so that with kLate they end at 2^15 and begin at 2^-31.
__host__ __device__ constexpr float bias_of(bool bf16) { return bf16 ? 0.0f : 7.0f; }

struct ChunkArgs {
    Pages p;
    Scales s;              // of e4m3 caches
    const uint16_t* q;     // [rows][heads][head_dim]
    uint16_t* out;         // the same, contiguous
    const int* row_starts; // [sequences + 1]
    float* part;           // [slot][kv head][column of a tile][head_dim], then the maxima and sums
    float* part_ml;
    uint2* plan;           // {slot of the first piece, splits} of each place; null: no tile is split
    int64_t q_row, q_head; // strides, values
    int64_t capacity;      // positions of a table row
    int rows;
    int heads;
    int kv_heads;
    int group;
    int head_dim;
    int pieces;            // of a head, at most
    int slots;             // of partials, at most
    uint32_t budget;       // pieces that the device takes at once
    uint32_t least_span;   // tiles of a piece, at least
    uint32_t divide;       // position / page_size: position * divide >> 31 + shift
    uint32_t shift;
    uint32_t flip;         // sign bits of the queries, where the softmax scale is negative
    float scale;           // |softmax scale| * log2(e)
};

// The places of a batch: rows before the first sequence (place 0), sequence
// i - 1 (place i), rows behind the last; the first and the last are as idle
// sequences.  Row starts are taken as they come, within 0 .. rows.
__device__ __forceinline__ int start_of(const ChunkArgs& a, int place) {
    if (place == 0) return 0;
    return place > a.p.sequences + 1 ? a.rows : min(max(a.row_starts[place - 1], 0), a.rows);
}
__device__ __forceinline__ int length_of(const ChunkArgs& a, int place) {
    return place == 0 || place > a.p.sequences ? -1 : a.p.lengths[place - 1];
}

// Tiles of `count` positions or columns.
__device__ __forceinline__ uint32_t tiles_of(int64_t count, int tile) {
    return static_cast<uint32_t>((count + tile - 1) / tile);
}
// Positions that row `row` of a sequence sees.
__device__ __forceinline__ int seen_by(const ChunkArgs& a, int length, int row) {
    return length < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(length) + row + 1, a.capacity));
}

struct Piece {
    int place;
    int first;    // row
    int rows;
    int length;
    int tile;     // of the place's columns
    int split;
    int splits;
    int slot;     // of this place's partials, the first
};

// The place of a tile where no tile is split: place i's tiles begin at
// floor(start * group / COLS) + i, which leaves room for each place's last,
// partly filled one.  A search 64 wide.
template <int COLS>
__device__ __forceinline__ int place_of_tile(const ChunkArgs& a, int at, int lane, int& begin) {
    int lo = 0, hi = a.p.sequences + 2;
    auto begin_of = [&](int i) { return static_cast<int>(static_cast<int64_t>(start_of(a, i)) * a.group / COLS) + i; };
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64;
        const int i = lo + lane * step;
        const int count = __popcll(__ballot(i < hi && begin_of(min(i, hi - 1)) <= at));
        lo += (max(count, 1) - 1) * step;
        hi = min(hi, lo + step);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    begin = begin_of(lo);
    return lo;
}

// Piece `at` of a head; false: there is none.  Every lane calls it.
//
// Where tiles are few for the device their positions are split: the places'
// tiles times their middle number of position tiles are the work, a piece of a
// place is to hold about a `budget`th of it.
template <int COLS>
__device__ __forceinline__ bool find_piece(const ChunkArgs& a, int at, int lane, Piece& piece) {
    if (a.plan == nullptr) {
        int begin;
        piece.place = place_of_tile<COLS>(a, at, lane, begin);
        piece.first = start_of(a, piece.place);
        piece.rows = max(start_of(a, piece.place + 1) - piece.first, 0);
        const int tiles = static_cast<int>(tiles_of(static_cast<int64_t>(piece.rows) * a.group, COLS));
        if (at - begin >= tiles) return false;
        piece.tile = tiles - 1 - (at - begin);  // the longest first
        piece.split = 0;
        piece.splits = 1;
        piece.slot = 0;
    } else {
        const int places = a.p.sequences + 2;
        auto tiles_at = [&](int i, uint32_t& most, float& work) {
            const int first = i < places ? start_of(a, i) : 0;
            const int rows = i < places ? max(start_of(a, i + 1) - first, 0) : 0;
            const int length = i < places ? length_of(a, i) : -1;
            const uint32_t tiles = tiles_of(static_cast<int64_t>(rows) * a.group, COLS);
            most = tiles_of(seen_by(a, length, rows - 1), kTile);
            work = static_cast<float>(tiles) * 0.5f * static_cast<float>(most + tiles_of(seen_by(a, length, 0), kTile));
            return tiles;
        };
        float work = 0.0f;
        uint32_t most;
        for (int base = 0; base < places; base += 64) {
            float w;
            tiles_at(base + lane, most, w);
            work += w;
        }
        work = __shfl(plm_wave_sum(work), kSumLane);
        const uint32_t span = max(a.least_span, static_cast<uint32_t>(work * static_cast<float>(a.kv_heads) /
                                                                      static_cast<float>(a.budget)) + 1u);
        uint32_t before = 0, slots = 0;
        bool found = false;
        for (int base = 0; base < places && !found; base += 64) {
            float w;
            const uint32_t tiles = tiles_at(base + lane, most, w);
            const uint32_t splits = max(1u, most / span);
            const uint32_t mine = tiles * splits, parts = splits > 1 ? mine : 0;
            uint32_t upto = mine, part_upto = parts;
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t u = __shfl_up(upto, off), v = __shfl_up(part_upto, off);
                if (lane >= off) upto += u, part_upto += v;
            }
            const unsigned long long past = __ballot(before + upto > static_cast<uint32_t>(at));
            if (past != 0) {
                const int l = __ffsll(past) - 1;
                const uint32_t n = __shfl(tiles, l), s = __shfl(splits, l);
                const uint32_t begin = before + __shfl(upto, l) - n * s;
                const uint32_t in = static_cast<uint32_t>(at) - begin;
                piece.place = base + l;
                piece.tile = static_cast<int>(n - 1 - in / s);
                piece.split = static_cast<int>(in % s);
                piece.splits = static_cast<int>(s);
                piece.slot = static_cast<int>(slots + __shfl(part_upto, l) - (s > 1 ? n * s : 0));
                found = true;
            }
            before += __shfl(upto, 63);
            slots += __shfl(part_upto, 63);
        }
        if (!found) return false;
        piece.place = __builtin_amdgcn_readfirstlane(piece.place);
        piece.split = __builtin_amdgcn_readfirstlane(piece.split);
        piece.splits = __builtin_amdgcn_readfirstlane(piece.splits);
        piece.slot = __builtin_amdgcn_readfirstlane(piece.slot);
        piece.first = start_of(a, piece.place);
        piece.rows = max(start_of(a, piece.place + 1) - piece.first, 0);
    }
    piece.tile = __builtin_amdgcn_readfirstlane(piece.tile);
    piece.first = __builtin_amdgcn_readfirstlane(piece.first);
    piece.rows = __builtin_amdgcn_readfirstlane(piece.rows);
    piece.length = __builtin_amdgcn_readfirstlane(length_of(a, piece.place));
    return true;
}

// Workgroup -> (piece, head).  Workgroups are dealt to the 8 XCDs in turn: a
// head's are kept on as few of them as there are heads for, so that its keys
// and values lie in few L2s.
__device__ __forceinline__ void block_of(const ChunkArgs& a, int& at, int& kvh) {
    const int id = blockIdx.x;
    if (8 % a.kv_heads == 0) {
        const int x = id & 7;
        kvh = x % a.kv_heads;
        at = (id >> 3) * (8 / a.kv_heads) + x / a.kv_heads;
    } else {
        at = id / a.kv_heads;
        kvh = id - at * a.kv_heads;
    }
}

template <bool BF16>
__device__ __forceinline__ f32x16 mfma32(const u32x4 a, const u32x4 b, const f32x16 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
}

// Over the two lanes of a column.
__device__ __forceinline__ float both_max(float v) {
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
}
__device__ __forceinline__ float both_sum(float v) {
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

// A 16-byte piece of a row of LDS is kept at piece ^ swizzle(row), so that what is
// read together touches every group of banks (a line of 256 bytes) once: the same
// piece of 16 adjacent rows for keys, four adjacent pieces of four rows,
// transposed, for values.  Where a line holds two rows, their lowest bit is one
// of the line's.
template <int DP>
__device__ __forceinline__ int swizzle(int row) {
    return DP == 64 ? (row >> 1 & 1) << 2 | (row >> 2 & 3) : (row & 3) << 2 | (row >> 2 & 3);
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 16 bytes a lane to LDS, the wave's KB in lane order at `to` (see fp8_matmul.hip).  The wait is loads_barrier's.
__device__ __forceinline__ void load_to_lds(const void* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "s"(to) : "m0", "memory");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void loads_barrier() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// One column over positions [begin, end) by a wave, in fp32, reading nothing that
// the column does not see: a lane has a position's score, then the values d =
// lane + 64 i of the sum.  For columns that meet infinities or NaN, so only right,
// not fast.
template <bool BF16, bool E8, int COLS>
__device__ void careful_column(const ChunkArgs& a, const Piece& piece, int kvh, int col, int begin, int end, int lane) {
    const int r = col / a.group, h = col - r * a.group;
    const uint16_t* q = a.q + (piece.first + r) * a.q_row + (kvh * a.group + h) * a.q_head;
    const int* table = a.p.table + static_cast<int64_t>(piece.place - 1) * a.p.table_cols;
    const uint8_t* kbase = reinterpret_cast<const uint8_t*>(a.p.k) + (E8 ? 1 : 2) * kvh * a.p.head_stride;
    const uint8_t* vbase = reinterpret_cast<const uint8_t*>(a.p.v) + (E8 ? 1 : 2) * kvh * a.p.head_stride;
    const int last = min(end, seen_by(a, piece.length, r));
    auto value = [&](const uint8_t* row, int d) {
        if constexpr (E8)
            return __uint_as_float(pair_of<true>(row[d], false) << 16);
        else
            return widen1<BF16>(reinterpret_cast<const uint16_t*>(row)[d]);
    };
    float m = -INFINITY, l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int t0 = begin; t0 < last; t0 += kTile) {
        const int pos = t0 + lane;
        int page = -1;
        uint32_t slot = 0;
        if (pos < last) {
            const uint32_t index = static_cast<uint32_t>(pos) / a.p.page_size;
            page = table[index];
            slot = static_cast<uint32_t>(pos) - index * a.p.page_size;
        }
        const bool there = page >= 0 && static_cast<uint32_t>(page) < a.p.num_pages;
        const uint32_t row = there ? static_cast<uint32_t>(page) * a.p.page_stride + slot * a.p.slot_stride : 0u;
        unsigned long long left = __ballot(there);
        if (left == 0) continue;
        float s = -INFINITY, by = 1.0f;
        if (there) {
            const uint8_t* k = kbase + static_cast<int64_t>(row) * 16;
            s = 0.0f;
#pragma unroll 1
            for (int d = 0; d < a.head_dim; ++d) s = fmaf(widen1<BF16>(q[d] ^ static_cast<uint16_t>(a.flip)), value(k, d), s);
            if constexpr (E8) {
                const int64_t scale = page * a.s.page_stride + kvh * a.s.head_stride + slot;
                s *= a.s.k[scale];
                by = a.s.v[scale];
            }
            s *= a.scale;
        }
        float top = fmaxf(s, there ? -FLT_MAX : -INFINITY);
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off));
        top = fmaxf(top - bias_of(BF16 || E8), m);  // weights of the sizes that they have elsewhere
        const float fade = exp2_from(m, top);
        m = top;
        const float p = there ? exp2f(s - m) : 0.0f;
        float sum = p;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off);
        l = fmaf(l, fade, sum);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= fade;
        for (; left != 0; left &= left - 1) {
            const int at = __ffsll(left) - 1;
            const uint8_t* v = vbase + static_cast<int64_t>(__shfl(row, at)) * 16;
            const float w = __shfl(p, at) * __shfl(by, at);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = lane + 64 * i;
                if (d < a.head_dim) acc[i] = fmaf(w, value(v, d), acc[i]);
            }
        }
    }
    if (piece.splits > 1) {
        const int slot = piece.slot + piece.tile * piece.splits + piece.split;
        if (slot >= a.slots) return;
        const int64_t to = (static_cast<int64_t>(slot) * a.kv_heads + kvh) * COLS + (col - piece.tile * COLS);
        if (lane == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * to) = f32x2{m, l};
        for (int i = 0; i < 4; ++i)
            if (lane + 64 * i < a.head_dim) a.part[to * a.head_dim + lane + 64 * i] = acc[i];
        return;
    }
    uint16_t* out = a.out + (static_cast<int64_t>(piece.first + r) * a.heads + kvh * a.group + h) * a.head_dim;
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < a.head_dim)
            out[lane + 64 * i] = m == -INFINITY ? static_cast<uint16_t>(0) : narrow1<BF16>(acc[i] * (1.0f / l));
}

typedef __attribute__((address_space(3))) char lds_char;
__device__ __forceinline__ u32x4 lds16(const lds_char* base, int at) {
    return *(const __attribute__((address_space(3))) u32x4*)(base + at);
}
__device__ __forceinline__ u32x2 lds_transposed(lds_char* base, int at) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(base + at)));
}

template <int DP, bool E8>
struct Stage {
    static constexpr int kRow = 2 * DP;                     // bytes
    static constexpr int kV = kTile * kRow;                 // values behind the keys
    static constexpr int kScales = 2 * kTile * kRow;        // then the scales
    static constexpr int kBytes = kScales + (E8 ? 2 * kTile * 4 : 0);
    static constexpr int kLds = 2 * kBytes;
};

// Workgroup (piece, key-value head): 4 waves of 32 CB columns each over the
// piece's positions, 64 at a time through LDS, two tiles deep.
//
//   scores  S^T = K Q^T (32 x 32 x 16): a lane has, of column l & 31, the positions
//           8 (j / 4) + 4 (l / 32) + j % 4, so that a column's maximum and sum are
//           its own registers' and one other lane's
//   values  O^T = V^T P^T: the weights go in as they lie, eight registers a step; the
//           values' eight positions are chosen to match, by two transposed reads
//
// Weights are rounded to the values' type once.
//
// E8: keys and values become 16-bit (exactly) on their way to LDS, values and
// weights bf16 whatever the queries' type, scores and weights are multiplied by
// their positions' scales in fp32.
//
// What a row does not see must not reach it, but a weight of 0 times an infinity or
// a NaN left there is NaN.  That shows: such an accumulator stays NaN.  So the
// first pass goes without care, and a wave that ends with a value that is not
// finite and met positions that not every column sees does its columns again, one at
// a time (careful_column).  Positions behind the last one seen, or without a page, are
// never read.
template <bool BF16, bool E8, int DP, int CB>
__global__ __launch_bounds__(64 * kWaves, (DP >= 128 && CB == 2) || DP > 128 ? 1 : 2) void paged_chunk_kernel(
    const ChunkArgs a) {
    using St = Stage<DP, E8>;
    constexpr bool VBF16 = BF16 || E8;
    constexpr int COLS = 32 * CB * kWaves;
    constexpr int KS = DP / 16;   // score steps
    constexpr int DB = DP / 32;   // blocks of head values
    constexpr int kLines = KS < 8 ? KS : 8;  // score steps whose pieces lie in one line of 256 bytes
    constexpr int kAhead = 6;
    constexpr float kBias = bias_of(VBF16);
    extern __shared__ char lds_raw[];
    lds_char* const lds = (lds_char*)lds_raw;
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 31, half = lane >> 5;
    int at, kvh;
    block_of(a, at, kvh);
    Piece piece;
    if (at >= a.pieces || !find_piece<COLS>(a, at, lane, piece)) return;
    if (a.plan != nullptr && kvh == 0 && piece.tile == 0 && piece.split == 0 && threadIdx.x == 0)
        a.plan[piece.place] = make_uint2(piece.slot, piece.splits);

    const int columns = piece.rows * a.group;
    const int col0 = piece.tile * COLS;
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const int seen = uniform(seen_by(a, piece.length, (min(col0 + COLS, columns) - 1) / a.group));
    const int least = uniform(seen_by(a, piece.length, col0 / a.group));  // what every column sees
    const uint32_t units = tiles_of(seen, kTile);
    const int begin = uniform(static_cast<int>(static_cast<uint64_t>(units) * piece.split / piece.splits) * kTile);
    const int end = uniform(
        min(seen, static_cast<int>(static_cast<uint64_t>(units) * (piece.split + 1) / piece.splits) * kTile));
    const int wave0 = col0 + 32 * CB * wave;
    const int wave_least = uniform(seen_by(a, piece.length, min(wave0, columns - 1) / a.group));
    const int wave_seen =
        wave0 < columns ? uniform(seen_by(a, piece.length, (min(wave0 + 32 * CB, columns) - 1) / a.group)) : 0;

    u32x4 q[CB][KS];
    int limit[CB];
#pragma unroll
    for (int t = 0; t < CB; ++t) {
        const int col = wave0 + 32 * t + li;
        const int r = min(col, columns - 1) / a.group, h = min(col, columns - 1) - r * a.group;
        const uint16_t* src = a.q + (piece.first + r) * a.q_row + (kvh * a.group + h) * a.q_head;
        limit[t] = col < columns ? seen_by(a, piece.length, r) : 0;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = 16 * s + 8 * half;
            q[t][s] = *reinterpret_cast<const u32x4*>(src + (d < a.head_dim ? d : 0)) ^ a.flip;
            if (col >= columns || d >= a.head_dim) q[t][s] = u32x4{0, 0, 0, 0};
        }
    }
    if (a.head_dim != DP) {  // the loads leave out what is behind a head's end
        for (int i = threadIdx.x; i < St::kLds / 16; i += 64 * kWaves)
            *(__attribute__((address_space(3))) u32x4*)(lds + 16 * i) = u32x4{0, 0, 0, 0};
        __syncthreads();
    }

    const int* table = a.p.table + static_cast<int64_t>(max(piece.place - 1, 0)) * a.p.table_cols;
    const uint8_t* kbase = reinterpret_cast<const uint8_t*>(a.p.k) + (E8 ? 1 : 2) * kvh * a.p.head_stride;
    const uint8_t* vbase = reinterpret_cast<const uint8_t*>(a.p.v) + (E8 ? 1 : 2) * kvh * a.p.head_stride;

    // lane l looks up position t0 + l of a tile; past the last one it is the last
    auto index_of = [&](int pos) {
        return static_cast<uint32_t>(static_cast<uint64_t>(pos) * a.divide >> 31 >> a.shift);
    };
    auto page_of = [&](int t0) { return table[index_of(min(t0 + lane, seen - 1))]; };

    // LDS addresses of this lane's reads: keys by score step, values by block and half
    constexpr int kMask = DP == 64 ? 7 : 15;
    constexpr int kBlocks = DB < 4 ? DB : 4;  // blocks whose pieces lie in one line
    int kat[kLines], vat[kBlocks][2];
#pragma unroll
    for (int x = 0; x < kLines; ++x) kat[x] = li * St::kRow + (((2 * x + half) ^ swizzle<DP>(li)) & kMask) * 16;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int i16 = lane & 15, row = 8 * z + 4 * half + (i16 >> 2);
            const int chunk = 4 * b + 2 * (lane >> 4 & 1) + (i16 >> 1 & 1);
            vat[b][z] = St::kV + row * St::kRow + ((chunk ^ swizzle<DP>(row)) & kMask) * 16 + (i16 & 1) * 8;
        }

    float m[CB], l[CB];  // weights are exp2(score - m): m is the maximum less the bias, up to kLate behind
    f32x16 acc[CB][DB];

    bool masked = false;  // there was a position that some column does not see
#pragma unroll
        for (int t = 0; t < CB; ++t) {
            m[t] = -INFINITY;
            l[t] = 0.0f;
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[t][b][j] = 0.0f;
        }
    if (begin < end) {
        // rows of a tile, in pieces of 16 bytes; a position without a page reads one that has one, a tile of none
        // is left out
        uint32_t row, slot;
        int page;
        bool there;
        auto find_rows = [&](int t0) {
            const uint32_t pos = static_cast<uint32_t>(min(t0 + lane, seen - 1));
            slot = pos - index_of(static_cast<int>(pos)) * a.p.page_size;
            there = page >= 0 && static_cast<uint32_t>(page) < a.p.num_pages;
            row = static_cast<uint32_t>(page) * a.p.page_stride + slot * a.p.slot_stride;
            const unsigned long long gone = __ballot(!there);
            if (gone != 0 && gone != ~0ull) {
                const uint32_t other = __shfl(row, __ffsll(~gone) - 1);
                if (!there) row = other;
            }
            return gone;
        };
        // 16-bit caches: straight to LDS
        auto load = [&](int stage) {
            constexpr int kPerRow = St::kRow / 16;       // pieces of a row
            constexpr int kLoads = kTile * St::kRow / 1024 / kWaves;
            int64_t from[kLoads];
            bool in[kLoads];
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int r = (wave * kLoads + i) * (64 / kPerRow) + lane / kPerRow;
                const int chunk = (lane % kPerRow) ^ swizzle<DP>(r);
                from[i] = static_cast<int64_t>(__shfl(row, r)) * 16 + chunk * 16;
                in[i] = chunk * 8 < a.head_dim;
            }
            const uint32_t to = __builtin_amdgcn_readfirstlane(lds_at + stage * St::kBytes + wave * kLoads * 1024);
            if (a.head_dim == DP) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    load_to_lds(kbase + from[i], to + i * 1024);
                    load_to_lds(vbase + from[i], to + St::kV + i * 1024);
                }
            } else {
#pragma unroll
                for (int i = 0; i < kLoads; ++i)
                    if (in[i]) {
                        load_to_lds(kbase + from[i], to + i * 1024);
                        load_to_lds(vbase + from[i], to + St::kV + i * 1024);
                    }
            }
        };
        // e4m3 caches: to registers first
        constexpr int kUnits = E8 ? DP / 64 : 1;
        u32x4 kraw[kUnits], vraw[kUnits];
        float scale_raw = 0.0f;
        auto load8 = [&] {
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int u = threadIdx.x + 64 * kWaves * i;
                const int r = u / (DP / 16), c = u % (DP / 16);
                const int64_t from = static_cast<int64_t>(__shfl(row, r)) * 16 + (16 * c < a.head_dim ? 16 * c : 0);
                kraw[i] = *reinterpret_cast<const u32x4*>(kbase + from);
                vraw[i] = *reinterpret_cast<const u32x4*>(vbase + from);
            }
            if (wave < 2)
                scale_raw = there ? (wave == 0 ? a.s.k : a.s.v)[page * a.s.page_stride + kvh * a.s.head_stride + slot] : 0.0f;
        };
        auto store8 = [&](int stage) {
            lds_char* const to = lds + stage * St::kBytes;
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int u = threadIdx.x + 64 * kWaves * i;
                const int r = u / (DP / 16), c = u % (DP / 16);
                if (16 * c < a.head_dim) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int where = r * St::kRow + ((2 * c + x) ^ swizzle<DP>(r)) * 16;
                        *(__attribute__((address_space(3))) u32x4*)(to + where) = eight_of<BF16>(kraw[i], x);
                        *(__attribute__((address_space(3))) u32x4*)(to + St::kV + where) = eight_of<true>(vraw[i], x);
                    }
                }
            }
            if (wave < 2) *(__attribute__((address_space(3))) float*)(to + St::kScales + wave * kTile * 4 + lane * 4) = scale_raw;
        };

        page = page_of(begin);
        unsigned long long gone = find_rows(begin), next_gone = 0;
        if (gone != ~0ull) {
            if constexpr (E8) {
                load8();
                store8(0);
            } else {
                load(0);
            }
        }
        page = page_of(begin + kTile);
        int stage = 0;
        for (int t0 = begin; t0 < end; t0 += kTile, stage ^= 1) {
            if constexpr (E8)
                __syncthreads();
            else
                loads_barrier();
            const bool more = t0 + kTile < end;
            if (more) {
                next_gone = find_rows(t0 + kTile);
                if (next_gone != ~0ull) {
                    if constexpr (E8)
                        load8();
                    else
                        load(stage ^ 1);
                }
                page = page_of(t0 + 2 * kTile);
            }
            lds_char* const tile = lds + stage * St::kBytes;
            masked |= t0 + kTile > least || gone != 0;
            if (t0 < wave_seen && gone != ~0ull) {
                f32x16 s[CB][2];
#pragma unroll
                for (int t = 0; t < CB; ++t)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int j = 0; j < 16; ++j) s[t][b][j] = 0.0f;
#pragma unroll
                for (int x = 0; x < KS; ++x)
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const u32x4 k = lds16(tile, kat[x % kLines] + x / kLines * 256 + b * 32 * St::kRow);
#pragma unroll
                        for (int t = 0; t < CB; ++t) s[t][b] = mfma32<BF16>(k, q[t][x], s[t][b]);
                    }
                // keys kAhead reads in front of their matrix instructions (without this each is waited for)
                __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
                for (int i = 0; i < 2 * KS - kAhead; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x8, CB, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x8, kAhead * CB, 0);
                if constexpr (E8) {
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            const f32x4 by = a.scale *
                                __builtin_bit_cast(f32x4, lds16(tile, St::kScales + (32 * b + 2 * j + 4 * half) * 4));
#pragma unroll
                            for (int t = 0; t < CB; ++t)
#pragma unroll
                                for (int i = 0; i < 4; ++i) s[t][b][j + i] *= by[i];
                        }
                }
                const bool full = t0 + kTile <= wave_least && gone == 0;
                // A row that sees a position has a maximum of at least the lowest number, one that sees none keeps
                // -inf: its result is 0, while scores that are all -inf give 0 / 0.
                float floor[CB];
#pragma unroll
                for (int t = 0; t < CB; ++t) floor[t] = full ? -FLT_MAX : -INFINITY;
                if (!full) {
                    asm volatile("");  // a branch, not selects in every tile
#pragma unroll
                    for (int t = 0; t < CB; ++t)
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            // bit i: position 32 b + 4 half + i of the tile is hidden
                            const int left = limit[t] - t0 - 32 * b - 4 * half;
                            const uint32_t hidden = static_cast<uint32_t>(gone >> 32 * b) >> 4 * half |
                                                    (left >= 32 ? 0u : ~0u << max(left, 0));
                            if ((~hidden & 0x0F0F0F0Fu) != 0) floor[t] = -FLT_MAX;
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                if (hidden >> (8 * (j >> 2) + (j & 3)) & 1) s[t][b][j] = -INFINITY;
                        }
                }
                // 16-bit caches: the scale goes into the weights' exponents as they are formed, in one instruction.
                // The maximum is rounded there and the scores are not, which all weights of a column share, but from
                // 2^22 on it might be large: such scores are multiplied first.
                float times = E8 ? 1.0f : a.scale;
                float top[CB];
                bool late = false, large = false;
#pragma unroll
                for (int t = 0; t < CB; ++t) {
                    float v = s[t][0][0];
#pragma unroll
                    for (int j = 1; j < 32; ++j) v = fmaxf(v, s[t][j >> 4][j & 15]);
                    top[t] = both_max(fmaxf(v * times, floor[t])) - kBias;
                    late |= top[t] > m[t] + kLate;
                    const float to = fmaxf(top[t], m[t]);
                    large |= fabsf(to) > 0x1p22f && to > -0x1p127f;
                }
                if (!E8 && __any(large)) {
                    times = 1.0f;
#pragma unroll
                    for (int t = 0; t < CB; ++t)
#pragma unroll
                        for (int j = 0; j < 32; ++j) s[t][j >> 4][j & 15] *= a.scale;
                }
                if (__any(late)) {
#pragma unroll
                    for (int t = 0; t < CB; ++t) {
                        const float to = fmaxf(m[t], top[t]);
                        const float fade = exp2_from(m[t], to);
                        m[t] = to;
                        l[t] *= fade;
#pragma unroll
                        for (int b = 0; b < DB; ++b)
#pragma unroll
                            for (int j = 0; j < 16; ++j) acc[t][b][j] *= fade;
                    }
                }
                u32x4 w[CB][4];
#pragma unroll
                for (int t = 0; t < CB; ++t) {
                    const float from = m[t] == -INFINITY ? 0.0f : m[t];
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            s[t][b][j] = __builtin_amdgcn_exp2f(fmaf(s[t][b][j], times, -from));
                            sum[j & 3] += s[t][b][j];
                        }
                    l[t] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                }
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        f32x4 by = {1.0f, 1.0f, 1.0f, 1.0f};
                        if constexpr (E8) {
                            by = __builtin_bit_cast(f32x4, lds16(tile, St::kScales + kTile * 4 + (32 * b + 2 * j + 4 * half) * 4));
                        }
#pragma unroll
                        for (int t = 0; t < CB; ++t) {
                            f32x4 v = {s[t][b][j], s[t][b][j + 1], s[t][b][j + 2], s[t][b][j + 3]};
                            if constexpr (E8)
#pragma unroll
                                for (int i = 0; i < 4; ++i) v[i] *= by[i];
                            w[t][2 * b + (j >> 3)][(j & 4) / 2] = pack2<VBF16>(v[0], v[1]);
                            w[t][2 * b + (j >> 3)][(j & 4) / 2 + 1] = pack2<VBF16>(v[2], v[3]);
                        }
                    }
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int b = 0; b < DB; ++b) {
                        const int from = b / kBlocks * 256 + 16 * x * St::kRow;
                        const u32x2 lo = lds_transposed(tile, vat[b % kBlocks][0] + from);
                        const u32x2 hi = lds_transposed(tile, vat[b % kBlocks][1] + from);
                        const u32x4 v = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
                        for (int t = 0; t < CB; ++t) acc[t][b] = mfma32<VBF16>(v, w[t][x], acc[t][b]);
                    }
            }
            if constexpr (E8)
                if (more && next_gone != ~0ull) store8(stage ^ 1);
            gone = next_gone;
        }
    }
#pragma unroll
    for (int t = 0; t < CB; ++t) l[t] = both_sum(l[t]);

    bool odd = false;
#pragma unroll
    for (int t = 0; t < CB; ++t)
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
            for (int j = 0; j < 16; ++j) odd |= !(fabsf(acc[t][b][j]) < INFINITY);
    if (__any(masked && odd)) {
        const int most = min(wave0 + 32 * CB, columns);
        for (int col = wave0; col < most; ++col) careful_column<BF16, E8, COLS>(a, piece, kvh, col, begin, end, lane);
        return;
    }

#pragma unroll
    for (int t = 0; t < CB; ++t) {
        const int in = wave * 32 * CB + 32 * t + li;
        const int col = col0 + in;
        if (col >= columns) continue;
        if (piece.splits > 1) {
            const int slot = piece.slot + piece.tile * piece.splits + piece.split;
            if (slot >= a.slots) continue;
            const int64_t to = (static_cast<int64_t>(slot) * a.kv_heads + kvh) * COLS + in;
            if (half == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * to) = f32x2{m[t], l[t]};
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const int d = 32 * b + 2 * j + 4 * half;
                    if (d < a.head_dim)
                        *reinterpret_cast<f32x4*>(a.part + to * a.head_dim + d) =
                            f32x4{acc[t][b][j], acc[t][b][j + 1], acc[t][b][j + 2], acc[t][b][j + 3]};
                }
            continue;
        }
        // a row that sees nothing is zero
        const int r = col / a.group, h = col - r * a.group;
        const bool empty = m[t] == -INFINITY;
        const float inv = 1.0f / l[t];
        uint16_t* to = a.out + (static_cast<int64_t>(piece.first + r) * a.heads + kvh * a.group + h) * a.head_dim;
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                const int d = 32 * b + 2 * j + 4 * half;
                u32x2 o;
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    o[x] = pack2<BF16>(empty ? 0.0f : acc[t][b][j + 2 * x] * inv,
                                       empty ? 0.0f : acc[t][b][j + 2 * x + 1] * inv);
                if (d < a.head_dim) *reinterpret_cast<u32x2*>(to + d) = o;
            }
    }
}

// Joins the pieces of split tiles: a workgroup for 32 columns of a tile, 8
// threads a column, each every eighth quad of head values.
constexpr int kJoinThreads = 256;
constexpr int kJoinColumns = 32;

template <bool BF16, int COLS>
__global__ __launch_bounds__(kJoinThreads) void paged_chunk_join_kernel(const ChunkArgs a) {
    const int lane = threadIdx.x & 63;
    int begin;
    const int place = place_of_tile<COLS>(a, blockIdx.x, lane, begin);
    const int first = start_of(a, place);
    const int columns = max(start_of(a, place + 1) - first, 0) * a.group;
    const int tile = blockIdx.x - begin;
    const int in = blockIdx.z * kJoinColumns + threadIdx.x / 8;
    const int col = tile * COLS + in;
    if (tile >= static_cast<int>(tiles_of(columns, COLS))) return;
    const uint2 noted = a.plan[place];
    const int splits = static_cast<int>(noted.y);
    const int slot = static_cast<int>(noted.x) + tile * splits;
    if (splits <= 1 || slot + splits > a.slots || col >= columns) return;
    const int kvh = blockIdx.y;
    const int64_t stride = static_cast<int64_t>(a.kv_heads) * COLS;
    const int64_t from = (static_cast<int64_t>(slot) * a.kv_heads + kvh) * COLS + in;
    const f32x2* ml = reinterpret_cast<const f32x2*>(a.part_ml) + from;
    float m = -INFINITY;
    for (int s = 0; s < splits; ++s) m = fmaxf(m, ml[s * stride][0]);
    float sum = 0.0f;
    for (int s = 0; s < splits; ++s) sum = fmaf(ml[s * stride][1], exp2_from(ml[s * stride][0], m), sum);
    const bool empty = m == -INFINITY;
    const float inv = 1.0f / sum;
    const int r = col / a.group, h = col - r * a.group;
    uint16_t* to = a.out + (static_cast<int64_t>(first + r) * a.heads + kvh * a.group + h) * a.head_dim;
    for (int d = 4 * (threadIdx.x & 7); d < a.head_dim; d += 32) {
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < splits; ++s) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(a.part + (from + s * stride) * a.head_dim + d);
            const float w = exp2_from(ml[s * stride][0], m);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = fmaf(x[i], w, acc[i]);
        }
        u32x2 o;
#pragma unroll
        for (int x = 0; x < 2; ++x) o[x] = empty ? 0u : pack2<BF16>(acc[2 * x] * inv, acc[2 * x + 1] * inv);
        *reinterpret_cast<u32x2*>(to + d) = o;
    }
}

// ---------------------------------------------------------------- host side

struct ChunkShape {
    int blocks;        // of 32 columns of a wave
    int64_t tiles;     // of a head, at most
    int64_t pieces;    // of a head, at most
    int64_t slots;     // of partials, at most
    int64_t budget;
    bool split;
    size_t bytes;
};

constexpr int kMostSplitSequences = 256;  // every workgroup reads all their lengths
constexpr int kLeastSpan = 4;

ChunkShape shape_of(int64_t sequences, int64_t rows, int64_t heads, int64_t kv_heads, int64_t head_dim,
                    int64_t capacity) {
    ChunkShape s;
    const int64_t group = heads / kv_heads, cus = plm::cu_count();
    s.blocks = head_dim <= 128 && false ? 2 : 1;
    const int64_t cols = 32 * kWaves * s.blocks;
    s.tiles = rows * group / cols + sequences + 2;
    s.budget = cus * ((head_dim > 64 && s.blocks == 2) || head_dim > 128 ? 1 : 2);
    s.split = sequences <= kMostSplitSequences && rows * heads / cols < 4 * s.budget &&
              capacity >= 2 * kLeastSpan * kTile;
    s.pieces = s.tiles;
    s.slots = 0;
    s.bytes = 0;
    if (s.split) {
        // splits of a place are at most its position tiles over the span, which twice the work bounds
        const int64_t most = std::min(s.tiles * (plm::ceil_div(capacity, kTile) / kLeastSpan),
                                      2 * s.budget / kv_heads + s.budget / 32 + 2);
        s.pieces = s.tiles + most;
        s.slots = most;
        s.bytes = static_cast<size_t>(s.slots) * kv_heads * cols * (head_dim + 2) * sizeof(float) +
                  sizeof(uint2) * (sequences + 2);
    }
    return s;
}

template <bool BF16, bool E8, int DP, int CB>
int launch_kernel(const ChunkArgs& a, const ChunkShape& s, hipStream_t st) {
    constexpr int bytes = Stage<DP, E8>::kLds;
    if (bytes > 64 * 1024) {
        const int code = plm::allow_large_lds(reinterpret_cast<const void*>(&paged_chunk_kernel<BF16, E8, DP, CB>), bytes);
        if (code != 0) return code;
    }
    const int64_t g = 8 % a.kv_heads == 0 ? 8 / a.kv_heads : 1;
    const int64_t blocks = plm::ceil_div(s.pieces, g) * g * a.kv_heads;
    hipLaunchKernelGGL((paged_chunk_kernel<BF16, E8, DP, CB>), dim3(static_cast<unsigned>(blocks)), dim3(64 * kWaves),
                       bytes, st, a);
    if (s.split)
        hipLaunchKernelGGL((paged_chunk_join_kernel<BF16, 32 * CB * kWaves>),
                           dim3(static_cast<unsigned>(s.tiles), static_cast<unsigned>(a.kv_heads),
                                32 * CB * kWaves / kJoinColumns),
                           dim3(kJoinThreads), 0, st, a);
    return 0;
}

template <bool BF16, bool E8>
int launch_chunk(const ChunkArgs& a, const ChunkShape& s, hipStream_t st) {
    if (a.head_dim > 128) return launch_kernel<BF16, E8, 256, 1>(a, s, st);
    if (a.head_dim > 64)
        return s.blocks == 2 ? launch_kernel<BF16, E8, 128, 2>(a, s, st) : launch_kernel<BF16, E8, 128, 1>(a, s, st);
    return s.blocks == 2 ? launch_kernel<BF16, E8, 64, 2>(a, s, st) : launch_kernel<BF16, E8, 64, 1>(a, s, st);
}

bool bad_heads(int64_t rows, int64_t heads, int64_t kv_heads) {
    return rows <= 0 || heads <= 0 || heads > 65535 || kv_heads <= 0 || heads % kv_heads != 0 || rows > kMostInt / heads;
}

// What both entry points check and launch once the caches are known.
template <bool E8>
int run_chunk(ChunkArgs& a, const uint16_t* q, uint16_t* out, const int* row_starts, void* scratch,
              int64_t scratch_bytes, int64_t rows, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t head_dim,
              int64_t q_row_stride, int64_t q_head_stride, float softmax_scale, int dtype_code, const char* name) {
    if (bad_heads(rows, heads, kv_heads)) return plm::fail(-2, "bad dimensions");
    if (!plm::aligned16(q) || !plm::aligned16(out) || q_row_stride < 0 || q_head_stride < 0 || q_row_stride % 8 != 0 ||
        q_head_stride % 8 != 0)
        return plm::fail(-2, "query strides and addresses must be multiples of 16 bytes");
    a.capacity = static_cast<int64_t>(a.p.table_cols) * a.p.page_size;
    const ChunkShape s = shape_of(sequences, rows, heads, kv_heads, head_dim, a.capacity);
    if ((s.pieces + 8) * kv_heads > kMostInt) return plm::fail(-2, "too many rows, heads or sequences");
    void* part = scratch;
    if (s.bytes > 0) {
        if (scratch == nullptr) {
            part = plm::workspace(s.bytes);
            if (part == nullptr) return -3;
        } else if (scratch_bytes < static_cast<int64_t>(s.bytes) || !plm::aligned16(scratch)) {
            return plm::fail(-3, "scratch must hold kv_paged_attention_chunk_scratch_bytes, 16-byte aligned");
        }
    }
    a.q = q;
    a.out = out;
    a.row_starts = row_starts;
    a.q_row = q_row_stride;
    a.q_head = q_head_stride;
    a.rows = static_cast<int>(rows);
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    a.group = static_cast<int>(heads / kv_heads);
    a.head_dim = static_cast<int>(head_dim);
    a.pieces = static_cast<int>(s.pieces);
    a.slots = static_cast<int>(s.slots);
    a.budget = static_cast<uint32_t>(s.budget);
    a.least_span = kLeastSpan;
    const int64_t cols = 32 * kWaves * s.blocks;
    a.part = static_cast<float*>(part);
    a.part_ml = a.part + s.slots * kv_heads * cols * head_dim;
    a.plan = s.split ? reinterpret_cast<uint2*>(a.part_ml + s.slots * kv_heads * cols * 2) : nullptr;
    // position / page_size of positions below 2^31: 2^(31 + shift) / page_size rounded up, 2^shift >= page_size
    a.shift = 0;
    while ((static_cast<uint64_t>(1) << a.shift) < a.p.page_size) ++a.shift;
    a.divide = static_cast<uint32_t>((static_cast<uint64_t>(1) << (31 + a.shift)) / a.p.page_size +
                                     ((static_cast<uint64_t>(1) << (31 + a.shift)) % a.p.page_size != 0 ? 1 : 0));
    // a scale of 0 would make NaN of hidden scores
    a.scale = std::fabs(softmax_scale) * 1.44269504088896340736f;
    if (a.scale == 0.0f) a.scale = 1.4e-45f;
    a.flip = softmax_scale < 0.0f ? 0x80008000u : 0u;
    const hipStream_t st = plm::current_stream();
    const int code = dtype_code == 1 ? launch_chunk<true, E8>(a, s, st) : launch_chunk<false, E8>(a, s, st);
    return code != 0 ? code : plm::check_launch(name);
}

}  // namespace

PLM_EXPORT int64_t kv_paged_attention_chunk_scratch_bytes(int64_t sequences, int64_t rows, int64_t heads,
                                                          int64_t kv_heads, int64_t head_dim, int64_t capacity) {
    if (sequences <= 0 || sequences > 65535 || bad_heads(rows, heads, kv_heads) || head_dim <= 0 || head_dim > 256 ||
        capacity <= 0 || capacity > kMostPositions)
        return plm::fail(-2, "bad dimensions");
    return static_cast<int64_t>(shape_of(sequences, rows, heads, kv_heads, head_dim, capacity).bytes);
}

PLM_EXPORT int kv_paged_attention_chunk_u16(const uint16_t* q, const uint16_t* k_cache, const uint16_t* v_cache,
                                            const int* page_table, const int* lengths, const int* row_starts,
                                            uint16_t* out, void* scratch, int64_t scratch_bytes, int64_t rows,
                                            int64_t sequences, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                            int64_t q_row_stride, int64_t q_head_stride, int64_t table_cols,
                                            int64_t num_pages, int64_t page_size, int64_t page_stride,
                                            int64_t slot_stride, int64_t head_stride, float softmax_scale,
                                            int dtype_code) {
    if (q == nullptr || out == nullptr || row_starts == nullptr) return plm::fail(-1, "null pointer");
    ChunkArgs a = {};
    const int code = pages_of(a.p, const_cast<uint16_t*>(k_cache), const_cast<uint16_t*>(v_cache), page_table, lengths,
                              sequences, table_cols, num_pages, page_size, kv_heads, head_dim, page_stride, slot_stride,
                              head_stride, dtype_code);
    if (code != 0) return code;
    return run_chunk<false>(a, q, out, row_starts, scratch, scratch_bytes, rows, sequences, heads, kv_heads, head_dim,
                            q_row_stride, q_head_stride, softmax_scale, dtype_code, "kv_paged_attention_chunk_u16");
}

PLM_EXPORT int kv_paged_attention_chunk_e4m3(const uint16_t* q, const uint8_t* k_cache, const uint8_t* v_cache,
                                             const float* k_scales, const float* v_scales, const int* page_table,
                                             const int* lengths, const int* row_starts, uint16_t* out, void* scratch,
                                             int64_t scratch_bytes, int64_t rows, int64_t sequences, int64_t heads,
                                             int64_t kv_heads, int64_t head_dim, int64_t q_row_stride,
                                             int64_t q_head_stride, int64_t table_cols, int64_t num_pages,
                                             int64_t page_size, int64_t page_stride, int64_t slot_stride,
                                             int64_t head_stride, int64_t scale_page_stride, int64_t scale_head_stride,
                                             float softmax_scale, int dtype_code) {
    if (q == nullptr || out == nullptr || row_starts == nullptr) return plm::fail(-1, "null pointer");
    ChunkArgs a = {};
    int code = pages_of<16>(a.p, const_cast<uint8_t*>(k_cache), const_cast<uint8_t*>(v_cache), page_table, lengths,
                            sequences, table_cols, num_pages, page_size, kv_heads, head_dim, page_stride, slot_stride,
                            head_stride, dtype_code);
    if (code != 0) return code;
    code = scales_of(a.s, const_cast<float*>(k_scales), const_cast<float*>(v_scales), scale_page_stride,
                     scale_head_stride);
    if (code != 0) return code;
    return run_chunk<true>(a, q, out, row_starts, scratch, scratch_bytes, rows, sequences, heads, kv_heads, head_dim,
                           q_row_stride, q_head_stride, softmax_scale, dtype_code, "kv_paged_attention_chunk_e4m3");
}
