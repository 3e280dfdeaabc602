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

constexpr int kTile = 64;  // positions that work is counted in
// A running maximum is only moved once a score is more than 2^kLate above it: weights grow to 2^kLate, the
// accumulators are multiplied in a few tiles instead of all.
constexpr float kLate = 8.0f;
constexpr int kFewPositions = 512;    // see attend
constexpr float kMuch = 1.0f / 3.0f;
// So bf16 weights are kept times 2^-kLate, which ends them at 1: their sum with values at the end of the range
// leaves fp32 no sooner than the decode kernel's.  fp16 weights are kept times 2^7, so that they end at 2^15 and
// begin at 2^-31.
__host__ __device__ constexpr float bias_of(bool bf16) { return bf16 ? -kLate : 7.0f; }

// n / d of n < 2^31 without a division: n * times >> 31 + shift, where times is
// 2^(31 + shift) / d rounded up and 2^shift >= d, so that its error, less than d,
// times n stays below 2^(31 + shift).
struct Divider {
    uint32_t times;
    uint32_t shift;

    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return __umulhi(2 * n, times) >> shift; }
};

struct ChunkArgs {
    Pages p;
    Scales s;              // of e4m3 caches
    const uint16_t* q;     // [rows][heads][head_dim]
    uint16_t* out;         // the same, contiguous
    const int* row_starts; // [sequences + 1]
    float* part;           // [slot][kv head][column of a tile, of part_columns][head_dim], then the maxima and sums
    float* part_ml;
    int* plan;             // {the run that begins it, the one that ends it} of each tile; null: no tile is split
    struct Found* found;   // of each run, by a kernel of its own; null: each workgroup finds its run
    int* begun;            // with found: the tile that each run begins and does not end, or -1
    int tiles;             // of a head, at most
    int64_t q_row, q_head; // strides, values
    int64_t capacity;      // positions of a table row
    int rows;
    int heads;
    int kv_heads;
    int group;
    int head_dim;
    int columns_log2;      // of a tile
    int part_columns;      // of a tile of the largest sequence that the rows may be
    int pieces;            // tiles of a head, and runs, at most
    int runs;              // at most
    uint32_t work_shift;   // so that a head's work stays in 32 bits
    Divider by_page;       // positions by page_size
    Divider by_group;      // columns by group
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

__device__ __forceinline__ int rows_of(const ChunkArgs& a, int place) {
    return max(start_of(a, place + 1) - start_of(a, place), 0);
}

// Tiles of `count` positions, and of the columns of `rows` rows (rows * heads is below 2^31).
__device__ __forceinline__ uint32_t position_tiles(int count) { return (static_cast<uint32_t>(count) + kTile - 1) / kTile; }
__device__ __forceinline__ int column_tiles(const ChunkArgs& a, int rows) {
    const uint32_t columns = static_cast<uint32_t>(rows) * static_cast<uint32_t>(a.group);
    return static_cast<int>((columns + (1u << a.columns_log2) - 1) >> a.columns_log2);
}
// Positions that row `row` of a sequence sees.
__device__ __forceinline__ int seen_by(const ChunkArgs& a, int length, int row) {
    return length < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(length) + row + 1, a.capacity));
}

// Part of a tile's positions, in tiles of kTile: a workgroup's work until its next one.
struct Piece {
    int place;
    int first;    // row
    int rows;
    int length;
    int tiles;    // of the place's columns
    int tile;
    int seen;     // positions that its last column sees
    int least;    // and that every one sees
    int begin;    // this piece's
    int end;
    bool whole;   // all that the tile sees
    int slot;     // of its partial, where it is not
};

// A tile of a place, whole.
__device__ __forceinline__ Piece piece_of(const ChunkArgs& a, int place, int tile) {
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    Piece p;
    p.place = place;
    p.first = uniform(start_of(a, place));
    p.rows = uniform(rows_of(a, place));
    p.length = uniform(length_of(a, place));
    const int columns = p.rows * a.group;
    p.tiles = column_tiles(a, p.rows);
    p.tile = tile;
    p.seen = uniform(seen_by(a, p.length, a.by_group(max(min((tile + 1) << a.columns_log2, columns), 1) - 1)));
    p.least = uniform(seen_by(a, p.length, a.by_group(min(tile << a.columns_log2, columns))));
    p.begin = 0;
    p.end = p.seen;
    p.whole = true;
    p.slot = 0;
    return p;
}

// Place i's tiles begin at floor(start * group / columns of a tile) + i, which
// leaves room for each place's last, partly filled one.
__device__ __forceinline__ int first_tile_of(const ChunkArgs& a, int place) {
    return static_cast<int>(static_cast<uint32_t>(start_of(a, place) * a.group) >> a.columns_log2) + place;
}
// The place of tile `at`, by a search 64 wide; every lane calls it.
__device__ __forceinline__ int place_of_tile(const ChunkArgs& a, int at, int lane, int& first) {
    int lo = 0, hi = a.p.sequences + 2;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64;
        const int i = lo + lane * step;
        const int count = __popcll(__ballot(i < hi && first_tile_of(a, min(i, hi - 1)) <= at));
        lo += (max(count, 1) - 1) * step;
        hi = min(hi, lo + step);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    first = __builtin_amdgcn_readfirstlane(first_tile_of(a, lo));
    return lo;
}

// Where tiles are few for the device, runs: the places' tiles in their order, a
// tile's work its position tiles (taken to grow evenly from a place's first tile
// to its last) and kTileWork for its queries and results, dealt in equal parts
// whatever the tiles' borders.  A run writes the results of the tiles that it
// holds whole; of the others it leaves two partials at most: of the tile that
// it goes on with (slot 2 run) and of the one that it begins and does not end
// (slot 2 run + 1).
//
// Unless whole tiles take no longer.  They take as many position tiles as the
// longest of them has, or where there are more than the device holds their share
// of the work and a fifth of the longest; runs take their share, kStart for each tile
// that they hold a part of, kJoin, and kJoinRuns where every workgroup leaves
// partials of full tiles (67 MB at a head of 128).  28 and 4 heads of 128, whole / in runs: a prompt
// of 500 rows 29 / 41 us, of 1500 56 / 67, of 2500 81 / 108, 16 of up to 200 rows 33 / 56; 37 rows
// behind 700 positions 34 / 27, 64 times 2 rows behind up to 4000 128 / 110.
constexpr uint32_t kTileWork = 2;
constexpr uint32_t kLeastWork = 4;  // of a run
constexpr float kStart = 3.0f, kJoin = 3.0f, kJoinRuns = 11.0f;

struct Work {
    int tiles;
    uint32_t first, last;  // position tiles of its first and last tile

    // Work of the tiles before `tile`, times 2 max(tiles - 1, 1); about, which every run takes alike.
    __device__ __forceinline__ float before(int tile) const {
        const float t = tile, n = max(tiles - 1, 1);
        return t * (2.0f * n * static_cast<float>(first + kTileWork) +
                    (static_cast<float>(last) - static_cast<float>(first)) * (t - 1.0f));
    }
    __device__ __forceinline__ uint32_t total(uint32_t shift) const {
        const uint64_t twice = static_cast<uint64_t>(tiles) * (static_cast<uint64_t>(first) + last + 2 * kTileWork);
        return tiles > 0 ? max(1u, static_cast<uint32_t>(twice >> (shift + 1))) : 0u;
    }
};

__device__ __forceinline__ Work work_of(const ChunkArgs& a, int place) {
    Work w = {0, 0, 0};
    if (place >= a.p.sequences + 2) return w;
    const int rows = rows_of(a, place);
    if (rows == 0) return w;  // whatever its length
    const int length = length_of(a, place);
    w.tiles = column_tiles(a, rows);
    w.first = position_tiles(seen_by(a, length, min(static_cast<int>(a.by_group(1u << a.columns_log2)), rows) - 1));
    w.last = position_tiles(seen_by(a, length, rows - 1));
    return w;
}

// A border between runs: a place, a tile of it and the share of the tile before the border (of 1).
struct Border {
    int place;
    int tile;
    float share;
};

// The border at work x of a block of 64 places, which begins at work `before`; each lane has a place's work and
// `upto`, the work up to its end, lane l the first place that ends past x.
__device__ __forceinline__ Border border_in(const Work& w, uint32_t total, uint32_t upto, uint32_t x, int base, int l) {
    Work of;
    of.tiles = __builtin_amdgcn_readlane(w.tiles, l);
    of.first = __builtin_amdgcn_readlane(w.first, l);
    of.last = __builtin_amdgcn_readlane(w.last, l);
    const uint32_t size = __builtin_amdgcn_readlane(total, l);
    const uint32_t in = x - (__builtin_amdgcn_readlane(upto, l) - size);
    const float z = static_cast<float>(in) * __builtin_amdgcn_rcpf(static_cast<float>(size)) * of.before(of.tiles);
    int lo = 0, hi = of.tiles;
#pragma unroll 1
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        (of.before(mid) <= z ? lo : hi) = mid;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const float from = of.before(lo);
    const float share = in == 0 ? 0.0f : (z - from) * __builtin_amdgcn_rcpf(of.before(lo + 1) - from);
    return Border{base + l, lo, share};
}

// What workgroup `run` of a head does: kRun and its borders, kTiles (tile `run`, whole) or kNone.  Every lane calls
// it.
// (Kept short, as all that a call does once: a small call waits for its
// instructions.)
enum Dealt { kNone, kTiles, kRun };

// Of the work of all places: the runs, whether they take whole tiles instead, and the work before run r.
struct Deal {
    uint32_t all, runs;
    float per_run;
    bool whole;

    __device__ __forceinline__ Deal(const ChunkArgs& a, uint32_t work, uint32_t longest, uint32_t tiles) : all(work) {
        runs = min(static_cast<uint32_t>(a.runs), max(1u, all / kLeastWork));
        // (what is only about right is the same for both runs of a border)
        const float each = __builtin_amdgcn_rcpf(static_cast<float>(runs));
        per_run = static_cast<float>(all) * each;
        const float filled = static_cast<float>(a.rows) * static_cast<float>(a.group) *
                             __builtin_amdgcn_rcpf(static_cast<float>(tiles << a.columns_log2));
        const float share = __builtin_amdgcn_rcpf(static_cast<float>(a.runs));
        const float scale = static_cast<float>(1u << a.work_shift);
        const float in_runs = per_run * scale + kStart * static_cast<float>(tiles) * each + kJoin +
                              kJoinRuns * static_cast<float>(runs) * share * filled;
        float in_tiles = static_cast<float>(longest);
        if (tiles > static_cast<uint32_t>(a.runs))
            in_tiles = fmaxf(in_tiles, static_cast<float>(all) * share * scale + in_tiles * 0.2f);
        whole = in_tiles <= in_runs;
    }
    __device__ __forceinline__ uint32_t border_at(uint32_t r) const {
        return r == runs ? all : static_cast<uint32_t>(static_cast<float>(r) * per_run);
    }
};

__device__ __forceinline__ Dealt find_run(const ChunkArgs& a, int run, int lane, Border (&border)[2]) {
    const int places = a.p.sequences + 2;
    uint32_t all = 0, longest = 0, tiles = 0;
#pragma unroll 1
    for (int base = 0; base < places; base += 64) {
        const Work w = work_of(a, base + lane);
        all += w.total(a.work_shift);
        longest = max(longest, w.last);
        tiles += w.tiles;
    }
    all = __builtin_amdgcn_readlane(wave_prefix(all), 63);
    longest = wave_max(longest);
    tiles = __builtin_amdgcn_readlane(wave_prefix(tiles), 63);
    const Deal deal(a, all, longest, tiles);
    if (deal.whole) return kTiles;
    if (static_cast<uint32_t>(run) >= deal.runs) return kNone;
    border[0].place = border[1].place = places;
    border[0].tile = border[1].tile = 0;
    border[0].share = border[1].share = 0.0f;
    uint32_t before = 0;
#pragma unroll 1
    for (int base = 0; base < places && border[1].place == places; base += 64) {
        const Work w = work_of(a, base + lane);
        const uint32_t total = w.total(a.work_shift), upto = before + wave_prefix(total);
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
            const uint32_t x = deal.border_at(static_cast<uint32_t>(run + k));
            const unsigned long long past = __ballot(upto > x);
            if (past == 0 || (k == 0 && border[0].place < places)) continue;
            const Border found = border_in(w, total, upto, x, base, __builtin_amdgcn_readfirstlane(__ffsll(past) - 1));
            if (k == 0) border[0] = found;
            if (k == 1) border[1] = found;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return kRun;
}

// The same in a kernel of its own, a workgroup for each run, for calls of many sequences: each workgroup of the
// attention would read all their lengths.  The waves share the places out, blocks of 64 whose work is kept in
// LDS.  (us where calls of more than 256 sequences were never split, and now: 512 of 200 positions but one of 100000
// 1986 and 170, 512 of up to 2000 262 and 277; two launches more, 9 and 5 us.)
constexpr int kFewSequences = 256;  // that each workgroup reads itself
constexpr int kFindThreads = 1024;
struct Found {
    int dealt;
    Border border[2];
};
__global__ __launch_bounds__(kFindThreads) void paged_chunk_find_kernel(const ChunkArgs a) {
    constexpr int kBlocks = (65535 + 2 + 63) / 64;  // of places, at most
    __shared__ uint32_t block_work[kBlocks + 63];
    __shared__ uint32_t sums[kFindThreads / 64][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int places = a.p.sequences + 2, blocks = (places + 63) / 64, run = blockIdx.x;
    uint32_t longest = 0, tiles = 0;
    for (int b = wave; b < blocks; b += kFindThreads / 64) {
        const Work w = work_of(a, 64 * b + lane);
        const uint32_t work = wave_prefix(w.total(a.work_shift));
        if (lane == 63) block_work[b] = work;
        longest = max(longest, w.last);
        tiles += w.tiles;
    }
    longest = wave_max(longest);
    tiles = __builtin_amdgcn_readlane(wave_prefix(tiles), 63);
    if (lane == 0) sums[wave][0] = longest, sums[wave][1] = tiles;
    __syncthreads();
    if (wave > 0) return;
    uint32_t all = 0;
    for (int b = 0; b < blocks; b += 64) all += b + lane < blocks ? block_work[b + lane] : 0;
    all = __builtin_amdgcn_readlane(wave_prefix(all), 63);
    longest = wave_max(lane < kFindThreads / 64 ? sums[lane][0] : 0);
    tiles = __builtin_amdgcn_readlane(wave_prefix(lane < kFindThreads / 64 ? sums[lane][1] : 0), 63);
    const Deal deal(a, all, longest, tiles);
    Found found = {deal.whole ? kTiles : static_cast<uint32_t>(run) < deal.runs ? kRun : kNone,
                   {Border{places, 0, 0.0f}, Border{places, 0, 0.0f}}};
    if (found.dealt == kRun)
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
            const uint32_t x = deal.border_at(static_cast<uint32_t>(run + k));
            uint32_t before = 0;
            int block = -1;
            for (int b = 0; b < blocks && block < 0; b += 64) {
                const uint32_t work = b + lane < blocks ? block_work[b + lane] : 0;
                const uint32_t upto = before + wave_prefix(work);
                const unsigned long long past = __ballot(upto > x);
                const int l = past == 0 ? 63 : __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
                if (past != 0) block = b + l;
                before = __builtin_amdgcn_readlane(upto, l) - (past == 0 ? 0 : __builtin_amdgcn_readlane(work, l));
            }
            if (block < 0) continue;  // the end
            const Work w = work_of(a, 64 * block + lane);
            const uint32_t total = w.total(a.work_shift), upto = before + wave_prefix(total);
            const unsigned long long past = __ballot(upto > x);
            if (past == 0) continue;  // (lengths changed under the kernel)
            found.border[k] =
                border_in(w, total, upto, x, 64 * block, __builtin_amdgcn_readfirstlane(__ffsll(past) - 1));
        }
    if (lane == 0) {
        a.found[run] = found;
        a.begun[run] = -1;
    }
}

// Workgroup -> (tile or run, head).  They are dealt to the 8 XCDs in turn: a
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

// A tile lies in LDS in blocks of 64 head values, a position's 128 bytes after the
// other's, each 16-byte piece at piece ^ swizzle(position), so that what is read
// together touches every group of banks (a line of 256 bytes) once: the same piece
// of 16 adjacent positions for keys, four adjacent pieces of four positions,
// transposed, for values.
__device__ __forceinline__ int swizzle(int position) {
    return (position >> 1 & 1) << 2 | (position >> 2 & 3);
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 16 bytes a lane to LDS, the wave's KB in lane order at `to` (see fp8_matmul.hip).  The wait is `landed`'s.
__device__ __forceinline__ void load_to_lds(const void* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "s"(to) : "m0", "memory");
}
// 4 bytes a lane.
__device__ __forceinline__ void load4_to_lds(const void* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(from), "s"(to) : "m0", "memory");
}
#pragma clang diagnostic pop

typedef __attribute__((address_space(3))) char lds_char;
__device__ __forceinline__ u32x4 lds16(const lds_char* base, int at) {
    return *(const __attribute__((address_space(3))) u32x4*)(base + at);
}
__device__ __forceinline__ u32x2 lds_transposed(lds_char* base, int at) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(base + at)));
}

// LDS of a workgroup: kStages tiles of keys and values (and scales), then for each
// wave the page table's entries of eight tiles, then what has been cleared (see
// attend): the first position of each head value that is NaN, inf or -inf, and
// whether there is any.
template <int DP, bool E8>
struct Layout {
    static constexpr int kWaves = DP > 128 ? 4 : 8;
    static constexpr int kColumns = 32 * kWaves;
    static constexpr int kPositions = DP > 128 ? 32 : 64;   // of a tile
    static constexpr int kBlocks = DP / 64;
    static constexpr int kBlock = kPositions * 128;         // bytes
    static constexpr int kV = kBlocks * kBlock;             // values behind the keys
    static constexpr int kScales = 2 * kV;                  // then the scales
    static constexpr int kStage = kScales + (E8 ? 2 * kPositions * 4 : 0);
    static constexpr int kStages = 4;
    static constexpr int kEntries = kStages * kStage;
    static constexpr int kRing = 8;
    static constexpr int kCleared = kEntries + kWaves * kRing * 256;
    static constexpr int kAnyCleared = kCleared + 3 * DP * 4;
    static constexpr int kBytes = kAnyCleared + 16;
    static_assert(kPositions == 8 * kWaves, "a wave loads eight positions of a tile");
};

template <int DP, bool E8>
__device__ __forceinline__ void reset_cleared(lds_char* lds) {
    using L = Layout<DP, E8>;
    for (int i = threadIdx.x; i <= 3 * DP; i += 64 * L::kWaves)
        *(__attribute__((address_space(3))) int*)(lds + L::kCleared + 4 * i) = i < 3 * DP ? 0x7FFFFFFF : 0;
}

// A piece by a workgroup: waves of 32 columns each over the piece's positions, a
// tile at a time through LDS.
//
//   scores  S^T = K Q^T (32 x 32 x 16): a lane has, of column l & 31, the positions
//           8 (j / 4) + 4 (l / 32) + j % 4, so that a column's maximum and sum are
//           its own registers' and one other lane's
//   values  O^T = V^T P^T: the weights go in as they lie, eight registers a step; the
//           values' eight positions are chosen to match, by two transposed reads
//
// Weights are rounded to the values' type once.  But over e4m3 pages they are
// multiplied by their values' scales, need bf16's range and are not summed as
// they were rounded: so they go in as two values, the second the rest, for fp16
// rows (results within 2.1e-4 of their size, 1.7e-3 with one value, 1.26 ms and
// 0.99 for 2048 rows behind 30000 positions), and for bf16 rows where one weight's
// rounding may be most of the result's: in tiles with a weight of more than kMuch of
// its column's sum so far, and all of those of rows that see few positions (a
// first prompt's rows were off by up to 2.1 times the output's rounding).  Rows of
// 8000 positions whose scores spread by 2 and 4 were off by 1.4 times the output's
// rounding, up to 1.7, and are by 1.02 and 1.00; evenly spread ones, of whose many weights
// each is rounded, by 1.4 (kMuch of 1/8 1.25, but tiles of a call's first positions
// exceed it: six turns of 24 rows behind 5000 50 us instead of 46, 46 with 1/3).
//
// Each wave alternates between the matrix cores (the scores of tile i + 1, then the
// values of tile i) and the vector units (the weights of tile i + 1); the second four
// waves are one step behind the first, so that of the two waves of a SIMD one is in
// each.  A barrier a step keeps them so.  Tile t's keys are read in steps 2 t - 1
// and 2 t (first and second waves), its values in 2 t + 1 and 2 t + 2; a wave loads its
// part of tile t + 3 in the step of tile t's products, when tile t - 1, which lay
// there, has been read.  Loads past the piece's end repeat its last row, so that
// their count is always the same.
//
// E8: keys and values become 16-bit (exactly) on their way to LDS, values and
// weights bf16 whatever the queries' type, scores and weights are multiplied by
// their positions' scales in fp32.
//
// What a row does not see must not reach it, but a weight of 0 times an infinity or
// a NaN left there is NaN.  So where some column of the workgroup does not see all
// of a tile, each wave looks at the values that it has loaded of it (32 bytes a lane
// at a head of 128), clears those that are not finite and notes their first positions;
// at the end the columns that see one get it: whatever a cache holds, a call takes as
// long as without it.  Positions behind the last one seen are never read.
//
// Bound by the matrix cores' power and by the exponentials between them: two
// prompts of up to 8191 rows of 28 and 4 heads of 128, 752 GFLOP, in 717 to 776 us (as
// the card is rested or in a row of calls), 0.97 to 1.05 PFLOP/s (a library product of
// 8192^3 1.05 to 1.2); in step, with tiles three deep, the waves took 818.  Over e4m3
// pages 2048 rows behind 30000 positions, 911 GFLOP, in 966 to 1050 us (1065 with each
// lane's page and scale found anew for each load, against 952).  Small calls wait for
// memory and for the code: 37 rows behind 700 positions 21 us of kernel; the look at
// the tiles of the diagonal is 1 us of a prompt of 500 rows' 29.
template <bool BF16, bool E8, int DP>
__device__ __forceinline__ void attend(const ChunkArgs& a, const Piece& piece, int kvh, lds_char* lds) {
    using L = Layout<DP, E8>;
    constexpr bool VBF16 = BF16 || E8;
    constexpr int KT = L::kPositions;
    constexpr int KB = KT / 32;   // blocks of 32 positions
    constexpr int KS = DP / 16;   // score steps
    constexpr int DB = DP / 32;   // blocks of head values
    constexpr float kBias = bias_of(VBF16);
    constexpr bool kTwo = E8 && !BF16;     // weights of two values
    constexpr bool kDotSum = BF16 && !E8;  // the weights are summed as they were rounded, two an instruction
    constexpr int kOutstanding = 1 + 2 * L::kBlocks;  // loads of a step
    typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
    typedef __attribute__((address_space(3))) const int lds_int;
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
    // (the lane's place anew for each piece: what follows from it is not kept in registers over the others, which
    // took e4m3 kernels of heads of 65 to 128 past their 256)
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool second = wave >= 4;
    const int li = lane & 31, half = lane >> 5;
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const int columns = piece.rows * a.group;
    const int wave0 = piece.tile * L::kColumns + 32 * wave;
    const int col = wave0 + li;
    const int wave_least = uniform(seen_by(a, piece.length, a.by_group(min(wave0, columns - 1))));
    const int wave_seen =
        wave0 < columns ? uniform(seen_by(a, piece.length, a.by_group(min(wave0 + 32, columns) - 1))) : 0;
    const int begin = piece.begin, end = piece.end;
    [[maybe_unused]] const bool few = wave_least < kFewPositions;

    typedef __attribute__((address_space(3))) int lds_word;
    bool cleared = false;
    float m = -INFINITY, l = 0.0f;  // weights are exp2(score - m): m is the maximum less the bias, up to kLate behind
    f32x16 acc[DB];
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[b][j] = 0.0f;

    if (begin < end) {
        u32x4 q[KS];
        int limit;
        {
            const int r = a.by_group(min(col, columns - 1)), h = min(col, columns - 1) - r * a.group;
            const uint16_t* src = a.q + (piece.first + r) * a.q_row + (kvh * a.group + h) * a.q_head;
            limit = col < columns ? seen_by(a, piece.length, r) : 0;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = 16 * s + 8 * half;
                q[s] = *reinterpret_cast<const u32x4*>(src + (d < a.head_dim ? d : 0)) ^ a.flip;
                if (col >= columns || d >= a.head_dim) q[s] = u32x4{0, 0, 0, 0};
            }
        }
        const int* table = a.p.table + static_cast<int64_t>(piece.place - 1) * a.p.table_cols;
        const uint8_t* kbase = reinterpret_cast<const uint8_t*>(a.p.k) + (E8 ? 1 : 2) * kvh * a.p.head_stride;
        const uint8_t* vbase = reinterpret_cast<const uint8_t*>(a.p.v) + (E8 ? 1 : 2) * kvh * a.p.head_stride;

        // LDS addresses of this lane's reads: keys by score step, values by block of 32 and half
        int kat[4], vat[2][2];
#pragma unroll
        for (int x = 0; x < 4; ++x) kat[x] = li * 128 + ((2 * x + half) ^ swizzle(li)) * 16;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const int i16 = lane & 15, row = 8 * z + 4 * half + (i16 >> 2);
                const int chunk = 4 * b + 2 * (lane >> 4 & 1) + (i16 >> 1 & 1);
                vat[b][z] = L::kV + row * 128 + (chunk ^ swizzle(row)) * 16 + (i16 & 1) * 8;
            }

        auto index_of = [&](uint32_t pos) { return a.by_page(pos); };
        // position r of tile t; past the piece's end its last one
        auto position = [&](int t, int r) { return static_cast<uint32_t>(min(begin + KT * t + r, end - 1)); };
        auto slot_of = [&](uint32_t pos) { return pos - index_of(pos) * a.p.page_size; };
        auto row_at = [&](int page, uint32_t slot) {
            return static_cast<uint32_t>(page) * a.p.page_stride + slot * a.p.slot_stride;
        };
        auto is_page = [&](int page) { return page >= 0 && static_cast<uint32_t>(page) < a.p.num_pages; };
        const uint32_t ring = L::kEntries + wave * L::kRing * 256;
        // the page table's entries of tile t, to LDS
        auto load_entries = [&](int t) {
            load4_to_lds(table + index_of(position(t, lane & (KT - 1))), lds_at + ring + (t & (L::kRing - 1)) * 256);
        };
        auto entry = [&](int t, int r) { return *(lds_int*)(lds + ring + (t & (L::kRing - 1)) * 256 + r * 4); };
        // bit r: position r of a tile, whose entries the lanes hold, has no page
        auto gone_of = [&](int page) {
            const unsigned long long gone = __ballot(!is_page(page));
            return KT == 64 ? gone : gone & 0xFFFFFFFFull;
        };
        // what a position without a page reads instead: one of the tile that has one, the cache's first row where none has
        auto other_row = [&](int t, unsigned long long gone) {
            const unsigned long long there = KT == 64 ? ~gone : ~gone & 0xFFFFFFFFull;
            if (there == 0) return 0u;
            const int f = __ffsll(there) - 1;
            return row_at(entry(t, f), slot_of(position(t, f)));
        };
        // A wave loads eight positions of a tile, eight lanes each: this lane's, its page and where it lies.
        const int own = 8 * wave + (lane >> 3), piece8 = lane & 7, chunk = piece8 ^ swizzle(own);
        int own_page = 0;
        uint32_t own_slot = 0;
        const int tiles = (end - begin + KT - 1) / KT;
        // the first tile that some column does not see all of, or where a position of the wave's has no page or a scale
        // that is not finite (times which a weight has no two values)
        int open = max(piece.least - begin, 0) / KT;
        const uint8_t *ksrc = nullptr, *vsrc = nullptr;
        auto find_own = [&](int t) {
            own_slot = slot_of(position(t, own));
            uint32_t row = row_at(own_page, own_slot);
            if (__any(!is_page(own_page))) {
                open = min(open, t);
                const uint32_t instead = other_row(t, gone_of(entry(t, lane)));
                if (!is_page(own_page)) row = instead;
            }
            const int64_t from = static_cast<int64_t>(row) * 16 + (E8 ? (16 * piece8 < a.head_dim ? piece8 : 0) : chunk) * 16;
            ksrc = kbase + from;
            vsrc = vbase + from;
        };
        // 16-bit caches: straight to LDS
        auto load_block = [&](int t, int i) {
            const uint32_t to = uniform(lds_at + (t & (L::kStages - 1)) * L::kStage + i * L::kBlock + wave * 1024);
            if (a.head_dim == DP || 64 * i + 8 * chunk < a.head_dim) {  // (some lanes of every load)
                load_to_lds(ksrc + 128 * i, to);
                load_to_lds(vsrc + 128 * i, to + L::kV);
            }
        };
        // e4m3 caches: to registers first, 16 values a lane and piece, to LDS a step of products later; the first lane of
        // a position has its key scale (times the softmax's), the second its value scale
        // (every lane loads something: a branch around a load is a wait for the ones before it)
        constexpr int kUnits = (DP + 127) / 128;
        struct Raw {
            u32x4 k[kUnits], v[kUnits];
            float scale;
            bool there;
        };
        Raw raw = {};
        const float* const scales = (piece8 == 0 ? a.s.k : a.s.v) + static_cast<uint32_t>(kvh) * a.s.head_stride;
        const int further = 16 * piece8 + 128 < a.head_dim ? 128 : 0;
        auto load8 = [&](Raw& to) {
            to.there = is_page(own_page);
            const uint32_t at = to.there ? static_cast<uint32_t>(own_page) * a.s.page_stride + own_slot : 0u;
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                to.k[i] = *reinterpret_cast<const u32x4*>(ksrc + (i > 0 ? further : 0));
                to.v[i] = *reinterpret_cast<const u32x4*>(vsrc + (i > 0 ? further : 0));
            }
            to.scale = scales[at];
        };
        auto store8 = [&](int t, const Raw& from) {
            lds_char* const to = lds + (t & (L::kStages - 1)) * L::kStage;
#pragma unroll
            for (int i = 0; i < kUnits; ++i)
                if (16 * piece8 + 128 * i < a.head_dim) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int where = (piece8 / 4 + 2 * i) * L::kBlock + own * 128 +
                                          (((2 * piece8 + x) & 7) ^ swizzle(own)) * 16;
                        *(lds_u32x4*)(to + where) = eight_of<BF16>(from.k[i], x);
                        *(lds_u32x4*)(to + L::kV + where) = eight_of<true>(from.v[i], x);
                    }
                }
            if (__any(from.there && !(fabsf(from.scale) < INFINITY))) open = min(open, t);
            if (piece8 < 2)
                *(__attribute__((address_space(3))) float*)(to + L::kScales + (piece8 * KT + own) * 4) =
                    from.there ? (piece8 == 0 ? from.scale * a.scale : from.scale) : 0.0f;
        };

        // The values of the wave's positions of tile t, which have been loaded, from the first open tile on: what is not
        // finite is cleared and noted (not of a position without a page, which has another one's values).
        auto clean = [&](int t) {
            if (t < open || t >= tiles) return;
            int here = lane;
            asm volatile("" : "+v"(here));  // (nothing of this is kept in registers over the tiles)
            lds_char* const tile = lds + (t & (L::kStages - 1)) * L::kStage;
            const int at = L::kV + wave * 1024 + here * 16, position8 = 8 * wave + (here >> 3);
            constexpr uint32_t kInf = VBF16 ? 0x7F80u : 0x7C00u;
            uint32_t high = 0, low = 0;  // largest magnitudes
#pragma unroll
            for (int i = 0; i < L::kBlocks; ++i) {
                const u32x4 piece16 = lds16(tile, at + i * L::kBlock);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    high = max(high, piece16[x] & 0x7FFF0000u);
                    low = max(low, piece16[x] & 0x7FFFu);
                }
            }
            bool odd = max(high >> 16, low) >= kInf;
            float scale = 1.0f;
            __attribute__((address_space(3))) float* const held =
                (__attribute__((address_space(3))) float*)(tile + L::kScales + (KT + position8) * 4);
            if constexpr (E8) {
                scale = *held;
                odd |= !(fabsf(scale) < INFINITY);
            }
            if (!__any(odd)) return;
            const int pos = static_cast<int>(position(t, position8));
            const bool there = is_page(entry(t, position8));
            const int first = 8 * ((here & 7) ^ swizzle(position8));  // head value
#pragma unroll 1
            for (int j = 0; j < 8 * L::kBlocks; ++j) {
                typedef __attribute__((address_space(3))) uint16_t lds_half;
                lds_half* const one = (lds_half*)(tile + at + j / 8 * L::kBlock + j % 8 * 2);
                const float value = widen1<VBF16>(*one);
                if (fabsf(value) < INFINITY && fabsf(scale) < INFINITY) continue;
                *one = 0;
                const float seen = value * scale;
                const int kind = seen != seen ? 0 : seen > 0.0f ? 1 : 2;
                if (there)
                    __hip_atomic_fetch_min((lds_word*)(lds + L::kCleared + (kind * DP + first + j / 8 * 64 + j % 8) * 4), pos,
                                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            }
            if constexpr (E8)
                if (!(fabsf(scale) < INFINITY)) *held = 0.0f;
            if (lane == 0) *(lds_word*)(lds + L::kAnyCleared) = 1;
        };

        f32x16 s[KB];
        u32x4 w[2 * KB], rest[kTwo ? 2 * KB : 1];
        u32x4 ahead_v[DB];
        auto value_piece = [&](lds_char* tile, int x, int b) {
            const int from = b / 2 * L::kBlock + 16 * x * 128;
            const u32x2 lo = lds_transposed(tile, vat[b % 2][0] + from);
            const u32x2 hi = lds_transposed(tile, vat[b % 2][1] + from);
            return u32x4{lo[0], lo[1], hi[0], hi[1]};
        };
        // Scores of tile t + 1, and the first values of tile t for what follows.  Reads of LDS are kept kAhead in
        // front of their matrix instructions: as the compiler orders them each is waited for.  Between them (LOAD) the
        // loads of tile t + 3, in the matrix instructions' shade.
        int tile_page = 0;  // this lane's entry of the tile that is weighed next
        auto scores = [&](int t, auto with_loads) {
            constexpr bool LOAD = decltype(with_loads)::value;
            const lds_char* const tile = lds + ((t + 1) & (L::kStages - 1)) * L::kStage;
            lds_char* const vtile = lds + (t & (L::kStages - 1)) * L::kStage;
            constexpr int kLeast = kTwo ? 4 : 6;  // (registers)
            constexpr int kAhead = DB > kLeast ? DB : kLeast, kSteps = KB * KS;
            u32x4 k[kAhead];
            auto key_piece = [&](int i) {
                const int x = i / KB, b = i % KB;
                return lds16(tile, kat[x % 4] + x / 4 * L::kBlock + b * 32 * 128);
            };
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) s[b][j] = 0.0f;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) k[i] = key_piece(i);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                __builtin_amdgcn_sched_barrier(0);
                s[i % KB] = mfma32<BF16>(k[i % kAhead], q[i / KB], s[i % KB]);
                if (i + kAhead < kSteps)
                    k[i % kAhead] = key_piece(i + kAhead);
                else if (i + kAhead - kSteps < DB)
                    ahead_v[i + kAhead - kSteps] = value_piece(vtile, 0, i + kAhead - kSteps);
                if constexpr (LOAD && E8) {
                    if (i == 1) {
                        store8(t + 3, raw);
                        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the entries of the step before
                        own_page = entry(t + 4, own);
                    }
                    if (i == 3) load_entries(t + 5);
                    if (i == 5) {
                        find_own(t + 4);
                        load8(raw);
                    }
                } else if constexpr (LOAD) {
                    if (i == 0) own_page = entry(t + 3, own);
                    if (i == 1) load_entries(t + 5);
                    if (i == 4) find_own(t + 3);
                    if (i >= 5 && i - 5 < L::kBlocks) load_block(t + 3, i - 5);
                }
                if (i == kSteps - 1) tile_page = entry(t + 1, lane);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        // the values of tile t, after scores(t)
        auto values = [&](int t) {
            lds_char* const tile = lds + (t & (L::kStages - 1)) * L::kStage;
#pragma unroll
            for (int x = 0; x < 2 * KB; ++x)
#pragma unroll
                for (int b = 0; b < DB; ++b) {
                    __builtin_amdgcn_sched_barrier(0);
                    acc[b] = mfma32<VBF16>(ahead_v[b], w[x], acc[b]);
                    if constexpr (kTwo) acc[b] = mfma32<VBF16>(ahead_v[b], rest[x], acc[b]);
                    if (x + 1 < 2 * KB) ahead_v[b] = value_piece(tile, x + 1, b);
                }
            __builtin_amdgcn_sched_barrier(0);
        };
        // the weights of tile t's scores; false: the wave's columns see none of it
        auto weigh = [&](int t) {
            const int t0 = begin + KT * t;
            const unsigned long long gone = gone_of(tile_page);
            if (t0 >= wave_seen || gone == (KT == 64 ? ~0ull : 0xFFFFFFFFull)) return false;
            const lds_char* const tile = lds + (t & (L::kStages - 1)) * L::kStage;
            // scales of this lane's positions, each kind read at once (as the compiler orders them each is waited for)
            f32x4 scale[E8 ? 4 * KB : 1];
            auto read_scales = [&](int kind) {
#pragma unroll
                for (int i = 0; i < 4 * KB; ++i)
                    scale[i] = __builtin_bit_cast(f32x4, lds16(tile, L::kScales + (kind * KT + 8 * i + 4 * half) * 4));
                __builtin_amdgcn_sched_barrier(0);
            };
            if constexpr (E8) {
                read_scales(0);
#pragma unroll
                for (int j = 0; j < 16 * KB; ++j) s[j >> 4][j & 15] *= scale[j >> 2][j & 3];
                __builtin_amdgcn_sched_barrier(0);
                read_scales(1);
            }
            const bool full = t0 + KT <= wave_least && gone == 0;
            // A row that sees a position has a maximum of at least the lowest number, one that sees none keeps
            // -inf: its result is 0, while scores that are all -inf give 0 / 0.
            float floor = full ? -FLT_MAX : -INFINITY;
            if (!full) {
                asm volatile("");  // a branch, not selects in every tile
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    // bit i: position 32 b + 4 half + i of the tile is hidden
                    const int left = limit - t0 - 32 * b - 4 * half;
                    const uint32_t hidden = static_cast<uint32_t>(gone >> 32 * b) >> 4 * half |
                                            (left >= 32 ? 0u : ~0u << max(left, 0));
                    if ((~hidden & 0x0F0F0F0Fu) != 0) floor = -FLT_MAX;
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (hidden >> (8 * (j >> 2) + (j & 3)) & 1) s[b][j] = -INFINITY;
                }
            }
            // 16-bit caches: the scale goes into the weights' exponents as they are formed, in one instruction.
            // The maximum is rounded there and the scores are not, which all weights of a column share, but from
            // 2^22 on it might be large: such scores are multiplied first.
            float times = E8 ? 1.0f : a.scale;
            float top = s[0][0];
#pragma unroll
            for (int j = 1; j < 16 * KB; ++j) top = fmaxf(top, s[j >> 4][j & 15]);
            const float best = both_max(fmaxf(top * times, floor));
            top = fmaxf(m, best - kBias);
            if (!E8 && __any(fabsf(top) > 0x1p22f && top > -0x1p127f)) {
                times = 1.0f;
#pragma unroll
                for (int j = 0; j < 16 * KB; ++j) s[j >> 4][j & 15] *= a.scale;
            }
            if (__any(top > m + kLate)) {
                const float fade = exp2_from(m, top);
                m = top;
                l *= fade;
#pragma unroll
                for (int b = 0; b < DB; ++b)
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[b][j] *= fade;
            }
            const float from = m == -INFINITY ? 0.0f : m;
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    f32x4 v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v[i] = __builtin_amdgcn_exp2f(fmaf(s[b][j + i], times, -from));
                        if constexpr (!kDotSum) sum[i] += v[i];
                    }
                    if constexpr (E8)
                        v = v * scale[4 * b + j / 4];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t two;
                        if constexpr (kTwo) {
                            const uint32_t lo = __float_as_uint(v[2 * i]), hi = __float_as_uint(v[2 * i + 1]) & 0xFFFF0000u;
                            two = hi | lo >> 16;
                            rest[2 * b + (j >> 3)][(j & 4) / 2 + i] =
                                pack2<true>(v[2 * i] - __uint_as_float(lo & 0xFFFF0000u), v[2 * i + 1] - __uint_as_float(hi));
                        } else {
                            two = pack2<VBF16>(v[2 * i], v[2 * i + 1]);
                        }
                        w[2 * b + (j >> 3)][(j & 4) / 2 + i] = two;
                        if constexpr (kDotSum)
                            sum[2 * (j >> 2 & 1) + i] = __builtin_amdgcn_fdot2_f32_bf16(
                                __builtin_bit_cast(bf16x2, two), __builtin_bit_cast(bf16x2, 0x3F803F80u),
                                sum[2 * (j >> 2 & 1) + i], false);
                    }
                }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if constexpr (E8 && BF16) {
                // what the rounding left, formed again: its products at once
                if (few || __any(__builtin_amdgcn_exp2f(best - from) > kMuch * both_sum(l))) {
#pragma unroll
                    for (int x = 0; x < 2 * KB; ++x) {
                        u32x4 left;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float v[2];
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                const int j = 8 * (x & 1) + 2 * i + y;
                                v[y] = __builtin_amdgcn_exp2f(s[x >> 1][j] - from) * scale[4 * (x >> 1) + j / 4][j & 3];
                            }
                            left[i] = pack2<true>(v[0] - __uint_as_float(w[x][i] << 16),
                                                  v[1] - __uint_as_float(w[x][i] & 0xFFFF0000u));
                        }
#pragma unroll
                        for (int b = 0; b < DB; ++b)
                            acc[b] = mfma32<true>(value_piece(const_cast<lds_char*>(tile), x, b), left, acc[b]);
                    }
                }
            }
            return true;
        };
        // This wave's loads but the last step's are there, of tile t the last ones (16-bit caches: the first waves after
        // their weights, the second after their products).
        auto landed = [&](int t) {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kOutstanding) : "memory");
            clean(t);
        };
        auto step_end = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

#pragma unroll 1
        for (int t = 0; t < 5; ++t) load_entries(t);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if constexpr (E8) {
            Raw first[3];  // all on their way at once
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                own_page = entry(t, own);
                find_own(t);
                load8(t < 3 ? first[t] : raw);
            }
#pragma unroll
            for (int t = 0; t < 3; ++t) store8(t, first[t]);
        } else {
#pragma unroll 1
            for (int t = 0; t < 3; ++t) {
                own_page = entry(t, own);
                find_own(t);
#pragma unroll
                for (int i = 0; i < L::kBlocks; ++i) load_block(t, i);
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        for (int t = 0; t < 3; ++t) clean(t);
        step_end();
        if (second) asm volatile("s_barrier" ::: "memory");
        scores(-1, std::false_type{});
        step_end();
        for (int t = 0; t < tiles; ++t) {
            const bool live = weigh(t);
            if constexpr (!E8)
                if (!second) landed(t + 1);
            step_end();
            __builtin_amdgcn_s_setprio(1);
            scores(t, std::true_type{});
            if (live) values(t);
            __builtin_amdgcn_s_setprio(0);
            if constexpr (E8)
                clean(t + 3);
            else if (second)
                landed(t + 2);
            step_end();
        }
        if (!second) asm volatile("s_barrier" ::: "memory");
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // what was loaded past the end
        cleared = __builtin_amdgcn_readfirstlane(*(lds_int*)(lds + L::kAnyCleared)) != 0;
    }
    l = both_sum(l);
    // where column c's results go: a partial's, or the output's
    auto partial_of = [&](int c) {
        return (static_cast<int64_t>(piece.slot) * a.kv_heads + kvh) * a.part_columns + (c - piece.tile * L::kColumns);
    };
    auto output_of = [&](int c, int r) {
        return a.out + (static_cast<int64_t>(piece.first + r) * a.heads + kvh * a.group + c - r * a.group) * a.head_dim + 4 * half;
    };
    if (col < columns && !piece.whole) {
        const int64_t to = partial_of(col);
        if (half == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * to) = f32x2{m, l};
        float* const at = a.part + to * a.head_dim + 4 * half;
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
            for (int j = 0; j < 16; j += 4)
                if (32 * b + 2 * j < a.head_dim)
                    *reinterpret_cast<f32x4*>(at + 32 * b + 2 * j) =
                        f32x4{acc[b][j], acc[b][j + 1], acc[b][j + 2], acc[b][j + 3]};
    } else if (col < columns) {
        // a row that sees nothing is zero
        const float inv = m == -INFINITY ? 0.0f : __builtin_amdgcn_rcpf(l);  // (the accumulators are 0 there too)
        uint16_t* const to = output_of(col, a.by_group(col));
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
            for (int j = 0; j < 16; j += 4)
                if (32 * b + 2 * j < a.head_dim)
                    *reinterpret_cast<u32x2*>(to + 32 * b + 2 * j) = u32x2{
                        pack2<BF16>(acc[b][j] * inv, acc[b][j + 1] * inv), pack2<BF16>(acc[b][j + 2] * inv, acc[b][j + 3] * inv)};
    }
    if (cleared) {
        // what has been cleared, to the results of the columns that see it
        int c = col;
        asm volatile("" : "+v"(c));  // (nothing of this is kept in registers over the rest)
        const int r = a.by_group(min(c, columns - 1));
        const int limit = c < columns ? seen_by(a, piece.length, r) : 0;
        float* const part = a.part + partial_of(c) * a.head_dim + 4 * half;
        uint16_t* const out = output_of(c, r);
#pragma unroll 1
        for (int d = 0; d < a.head_dim - 4 * half; ++d) {
            if (d % 8 >= 4) continue;  // the other half's
            auto sees = [&](int kind) { return limit > *(lds_int*)(lds + L::kCleared + (kind * DP + d + 4 * half) * 4); };
            const float add = (sees(0) ? NAN : 0.0f) + (sees(1) ? INFINITY : 0.0f) + (sees(2) ? -INFINITY : 0.0f);
            if (add == 0.0f) continue;
            if (piece.whole)
                out[d] = narrow1<BF16>(widen1<BF16>(out[d]) + add);
            else
                part[d] += add;
        }
        __syncthreads();  // that has been read
        reset_cleared<DP, E8>(lds);
    }
}

// Workgroup -> (tile or run, key-value head).
template <bool BF16, bool E8, int DP>
__global__ __launch_bounds__(DP > 128 ? 256 : 512, 1) void paged_chunk_kernel(const ChunkArgs a) {
    using L = Layout<DP, E8>;
    extern __shared__ char lds_raw[];
    lds_char* const lds = (lds_char*)lds_raw;
    const int lane = threadIdx.x & 63;
    int at, kvh;
    block_of(a, at, kvh);
    if (at >= a.pieces) return;
    if (a.head_dim != DP)  // the loads leave out what is behind a head's end
        for (int i = threadIdx.x; i < L::kStages * L::kStage / 16; i += 64 * L::kWaves)
            *(__attribute__((address_space(3))) u32x4*)(lds + 16 * i) = u32x4{0, 0, 0, 0};
    reset_cleared<DP, E8>(lds);
    Border border[2];  // of the run: where it goes on, where it ends
    Dealt dealt = kTiles;
    if (a.found != nullptr) {
        auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
        const Found found = a.found[min(at, a.runs - 1)];
        dealt = static_cast<Dealt>(uniform(found.dealt));
        if (dealt == kRun && at >= a.runs) dealt = kNone;
#pragma unroll
        for (int k = 0; k < 2; ++k)
            border[k] = Border{uniform(found.border[k].place), uniform(found.border[k].tile),
                               __int_as_float(uniform(__float_as_int(found.border[k].share)))};
    } else if (a.plan != nullptr) {
        dealt = find_run(a, at, lane, border);
    }
    if (dealt == kNone) return;
    if (dealt == kTiles) {
        int first;
        const int place = place_of_tile(a, at, lane, first);
        const int longest_first = column_tiles(a, rows_of(a, place)) - 1 - (at - first);
        if (longest_first < 0) return;
        border[0] = Border{place, longest_first, 0.0f};
        border[1] = Border{place, longest_first + 1, 0.0f};
    }
    const Border &next = border[0], &last = border[1];
    int place = next.place, tile = next.tile;
    while (place < last.place || (place == last.place && tile <= last.tile)) {
        Piece piece = piece_of(a, place, tile);
        if (tile >= piece.tiles) {
            if (++place > a.p.sequences + 1) return;
            tile = 0;
            continue;
        }
        const int units = static_cast<int>(position_tiles(piece.seen));
        auto unit_at = [&](float share) {
            return __builtin_amdgcn_readfirstlane(min(units, max(0, static_cast<int>(share * static_cast<float>(units)))));
        };
        const bool goes_on = place == next.place && tile == next.tile && next.share > 0.0f;
        const bool ends_here = place == last.place && tile == last.tile;
        if (ends_here && last.share == 0.0f) return;
        const int from = goes_on ? unit_at(next.share) : 0, to = ends_here ? max(from, unit_at(last.share)) : units;
        if (units > 0 && to == 0) return;  // the next run begins it
        // (not what the run before has ended)
        if (units > 0 ? from < units : !goes_on) {
            if (a.plan != nullptr && kvh == 0 && threadIdx.x == 0) {
                int* const noted = a.plan + 2 * (first_tile_of(a, place) + tile);
                if (from == 0) noted[0] = at;
                if (to == units) noted[1] = at;
                if (a.begun != nullptr && from == 0 && to < units) a.begun[at] = first_tile_of(a, place) + tile;
            }
            piece.whole = from == 0 && to == units;
            piece.slot = 2 * at + (from == 0 ? 1 : 0);
            piece.begin = from * kTile;
            piece.end = min(piece.seen, to * kTile);
            __syncthreads();  // the tile before has been read
            attend<BF16, E8, DP>(a, piece, kvh, lds);
        }
        ++tile;
    }
}

// Joins the partials of the tiles that several runs hold: of each tile, or with many
// sequences of the one that each run begins and does not end (2048 sequences have
// 530000 workgroups of tiles, which take 114 us to do nothing).  GROUPS of 16 lanes for a
// column: a lane takes four head values of every GROUPS-th partial.  One group
// where partials are few, a wave's four where they are many (64 partials of 112
// columns of 4 heads: 50 us with one, 16 with four; 4 partials of 10500 columns 13
// and 28).
constexpr int kJoinThreads = 256;
constexpr int kJoinColumns = 4;  // of a workgroup, one a wave; 16 where partials are few
constexpr int kFewPartials = 8;

template <bool BF16, int GROUPS>
__device__ __forceinline__ void join_column(const ChunkArgs& a, int run, int parts, int kvh, int first, int in, int col,
                                            int lane) {
    constexpr int LANES = 16 * GROUPS;
    const int part_lane = lane & (LANES - 1), g = part_lane >> 4, j = lane & 15;
    // partial i: the first is its run's second
    auto slot = [](int i) { return max(2 * i, 1); };
    const int64_t stride = static_cast<int64_t>(a.kv_heads) * a.part_columns;
    const int64_t from = (static_cast<int64_t>(2 * run) * a.kv_heads + kvh) * a.part_columns + in;
    const f32x2* ml = reinterpret_cast<const f32x2*>(a.part_ml) + from;
    float m = -INFINITY;
    for (int i = part_lane; i < parts; i += LANES) m = fmaxf(m, ml[slot(i) * stride][0]);
#pragma unroll
    for (int off = 1; off < LANES; off <<= 1) m = fmaxf(m, __shfl_xor(m, off));
    const float* part = a.part + from * a.head_dim + 4 * j;
    float sum = 0.0f;
    f32x4 acc[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) acc[x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int base = 0; base < parts; base += LANES) {
        const int n = min(LANES, parts - base);
        float weight = 0.0f;
        if (part_lane < n) {
            const f32x2 v = ml[slot(base + part_lane) * stride];
            weight = exp2_from(v[0], m);
            sum = fmaf(v[1], weight, sum);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            if (64 * x >= a.head_dim) break;
            const bool in_head = 4 * j + 64 * x < a.head_dim;
#pragma unroll 4
            for (int i = g; i < n + g; i += GROUPS) {  // as often in every lane
                const float w = __shfl(weight, (lane & ~(LANES - 1)) + min(i, n - 1));
                const f32x4 v = *reinterpret_cast<const f32x4*>(part + slot(base + min(i, n - 1)) * stride * a.head_dim +
                                                                (in_head ? 64 * x : -4 * j));
#pragma unroll
                for (int y = 0; y < 4; ++y) acc[x][y] = i < n ? fmaf(v[y], w, acc[x][y]) : acc[x][y];
            }
        }
    }
#pragma unroll
    for (int off = 1; off < LANES; off <<= 1) sum += __shfl_xor(sum, off);
    if constexpr (GROUPS == 4) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                acc[x][y] += __shfl_xor(acc[x][y], 16);
                acc[x][y] += __shfl_xor(acc[x][y], 32);
            }
    }
    const bool empty = m == -INFINITY;
    const float inv = 1.0f / sum;
    const int r = a.by_group(col), h = col - r * a.group;
    uint16_t* to = a.out + (static_cast<int64_t>(first + r) * a.heads + kvh * a.group + h) * a.head_dim + 4 * j;
#pragma unroll
    for (int x = 0; x < 4; ++x)
        if (g == 0 && 4 * j + 64 * x < a.head_dim) {
            u32x2 o;
#pragma unroll
            for (int y = 0; y < 2; ++y)
                o[y] = empty ? 0u : pack2<BF16>(acc[x][2 * y] * inv, acc[x][2 * y + 1] * inv);
            *reinterpret_cast<u32x2*>(to + 64 * x) = o;
        }
}

template <bool BF16>
__global__ __launch_bounds__(kJoinThreads) void paged_chunk_join_kernel(const ChunkArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int at = blockIdx.x;
    if (a.begun != nullptr) {
        at = a.begun[at];
        if (at < 0 || at >= a.tiles) return;
    }
    // (within the runs also where the lengths were changed under the first kernel)
    const int run = max(a.plan[2 * at], 0);
    const int parts = min(a.plan[2 * at + 1], a.runs - 1) - run + 1;
    if (parts <= 1) return;
    int begin;
    const int place = place_of_tile(a, at, lane, begin);
    const int first = start_of(a, place), rows = rows_of(a, place);
    const int tile = at - begin;
    if (tile < 0 || tile >= column_tiles(a, rows)) return;  // (below 0 where row starts do not ascend)
    const int col0 = tile << a.columns_log2, columns = rows * a.group;
    if (parts > kFewPartials) {
        const int in = blockIdx.z * kJoinColumns + wave;
        if (col0 + in < columns) join_column<BF16, 4>(a, run, parts, blockIdx.y, first, in, col0 + in, lane);
    } else if (blockIdx.z % 4 == 0) {
        // a lane without a column joins the last one again
        const int in = min(blockIdx.z * kJoinColumns + 4 * wave + (lane >> 4), columns - 1 - col0);
        if (blockIdx.z * kJoinColumns < columns - col0)
            join_column<BF16, 1>(a, run, parts, blockIdx.y, first, in, col0 + in, lane);
    }
}

// ---------------------------------------------------------------- host side

struct ChunkShape {
    int64_t columns;   // of a tile
    int64_t part_columns;
    int64_t tiles;     // of a head, at most
    int64_t runs;      // of a head, at most
    bool split;
    uint32_t work_shift;
    size_t bytes;
};

constexpr int64_t kFewTiles = 4;              // for each workgroup that the device holds

ChunkShape shape_of(int64_t sequences, int64_t rows, int64_t heads, int64_t kv_heads, int64_t head_dim,
                    int64_t capacity) {
    ChunkShape s;
    const int64_t group = heads / kv_heads;
    const int64_t resident = plm::cu_count();
    s.columns = head_dim > 128 ? Layout<256, false>::kColumns : Layout<128, false>::kColumns;
    s.part_columns = std::min(s.columns, rows * group);
    s.tiles = rows * group / s.columns + sequences + 2;
    s.split = rows * heads / s.columns < kFewTiles * resident &&
              capacity > kTile * (static_cast<int64_t>(kStart + kJoin) + 1);
    s.runs = 0;
    s.work_shift = 0;
    s.bytes = 0;
    if (s.split) {
        s.runs = std::max<int64_t>(1, resident / kv_heads);
        while (s.tiles * (plm::ceil_div(capacity, kTile) + kTileWork) >> s.work_shift > kMostInt / 2) ++s.work_shift;
        s.bytes = static_cast<size_t>(2 * s.runs) * kv_heads * s.part_columns * (head_dim + 2) * sizeof(float) +
                  2 * sizeof(int) * s.tiles;
        if (sequences > kFewSequences) s.bytes += (sizeof(Found) + sizeof(int)) * s.runs;
    }
    return s;
}

Divider divider_of(uint32_t d) {
    Divider by = {0, 0};
    while ((static_cast<uint64_t>(1) << by.shift) < d) ++by.shift;
    const uint64_t whole = static_cast<uint64_t>(1) << (31 + by.shift);
    by.times = static_cast<uint32_t>(whole / d + (whole % d != 0 ? 1 : 0));
    return by;
}

template <bool BF16, bool E8, int DP>
int launch_kernel(const ChunkArgs& a, const ChunkShape& s, hipStream_t st) {
    using L = Layout<DP, E8>;
    constexpr int bytes = L::kBytes;
    if (bytes > 64 * 1024) {
        const int code = plm::allow_large_lds(reinterpret_cast<const void*>(&paged_chunk_kernel<BF16, E8, DP>), bytes);
        if (code != 0) return code;
    }
    const int64_t g = 8 % a.kv_heads == 0 ? 8 / a.kv_heads : 1;
    const int64_t blocks = plm::ceil_div(a.pieces, g) * g * a.kv_heads;
    if (a.found != nullptr)
        hipLaunchKernelGGL(paged_chunk_find_kernel, dim3(static_cast<unsigned>(s.runs)), dim3(kFindThreads), 0, st, a);
    hipLaunchKernelGGL((paged_chunk_kernel<BF16, E8, DP>), dim3(static_cast<unsigned>(blocks)), dim3(64 * L::kWaves),
                       bytes, st, a);
    if (s.split)
        hipLaunchKernelGGL((paged_chunk_join_kernel<BF16>),
                           dim3(static_cast<unsigned>(a.found != nullptr ? s.runs : s.tiles), static_cast<unsigned>(a.kv_heads),
                                L::kColumns / kJoinColumns),
                           dim3(kJoinThreads), 0, st, a);
    return 0;
}

template <bool BF16, bool E8>
int launch_chunk(const ChunkArgs& a, const ChunkShape& s, hipStream_t st) {
    if (a.head_dim > 192) return launch_kernel<BF16, E8, 256>(a, s, st);
    if (a.head_dim > 128) return launch_kernel<BF16, E8, 192>(a, s, st);
    return a.head_dim > 64 ? launch_kernel<BF16, E8, 128>(a, s, st) : launch_kernel<BF16, E8, 64>(a, s, st);
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
    if ((std::max(s.tiles, s.runs) + 8) * kv_heads > kMostInt) return plm::fail(-2, "too many rows, heads or sequences");
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
    a.columns_log2 = 0;
    while ((1 << a.columns_log2) < s.columns) ++a.columns_log2;
    a.pieces = static_cast<int>(std::max(s.tiles, s.runs));
    a.runs = static_cast<int>(s.runs);
    a.work_shift = s.work_shift;
    a.part = static_cast<float*>(part);
    a.part_columns = static_cast<int>(s.part_columns);
    a.part_ml = a.part + 2 * s.runs * kv_heads * s.part_columns * head_dim;
    a.plan = s.split ? reinterpret_cast<int*>(a.part_ml + 2 * s.runs * kv_heads * s.part_columns * 2) : nullptr;
    a.tiles = static_cast<int>(s.tiles);
    const bool many = s.split && sequences > kFewSequences;
    a.found = many ? reinterpret_cast<Found*>(a.plan + 2 * s.tiles) : nullptr;
    a.begun = many ? reinterpret_cast<int*>(a.found + s.runs) : nullptr;
    a.by_page = divider_of(a.p.page_size);
    a.by_group = divider_of(static_cast<uint32_t>(a.group));
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
    code = scales_of(a.s, a.p, kv_heads, const_cast<float*>(k_scales), const_cast<float*>(v_scales), scale_page_stride,
                     scale_head_stride);
    if (code != 0) return code;
    return run_chunk<true>(a, q, out, row_starts, scratch, scratch_bytes, rows, sequences, heads, kv_heads, head_dim,
                           q_row_stride, q_head_stride, softmax_scale, dtype_code, "kv_paged_attention_chunk_e4m3");
}
