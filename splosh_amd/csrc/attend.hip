// attend.hip -- causal attention of a packed step's rows over the 8-bit paged cache.
//
// With s_j = q . code(k_j), ks_j and vs_j the scales of key and value j, and t_j = s_j ks_j scale log2(e) + log2(vs_j):
//     a_j = 2^(t_j - M),   out = sum_j a_j code(v_j) / sum_j (a_j / vs_j),
// M a running maximum of t. The scale of v_j goes into its weight's exponent, so that a_j is what v_j's codes are
// multiplied with, and lies in [0, 2^8] whatever the scales are: fp16 holds it to 2^-11, and of what is too small for
// it nothing but 2^-25 of the largest is lost. Codes are whole numbers up to 127 and exact in fp16; so are the values of
// a row of q, moved by the power of two that brings its largest to 2^14 (what is below 2^-28 of that is cut at 2^-39 of it).
// Both products run on the fp16 matrix instructions with fp32 sums.
//
// Beside a key whose value has a large scale, a_j of one with a small scale (2^-100 for a value of zeros) may be below what fp32 holds, where
// its a_j / vs_j is not. What is lost so of the sum is below 2^(-126 - log2(vs_j)), and the key that M is from has 2^-log2(vs) of it: below 2^-24 of
// the whole while the scales of a piece are within 2^102 of each other, as they are where none is above 4, or none below 2^-62 and none above 2^40. The loops
// note whether that is so. Where it is not, a piece leaves its vectors to the last launch, which goes through all of their keys by itself
// (apart_vector: 20 to 30 times the time). Made good in these kernels, in the loop, behind it or in an instance of its own, it took registers from the sums, or
// parted what is scheduled together: the verify step took 107 to 168 us instead of 103, with the notes alone 106.
// Where M moves, and where pieces are joined, the sum is scaled by 2^(x / 2) twice: for scales from 2^-100 to 2^122 it is between 2^-122 and 2^108 a key.
//
// Scores are computed transposed, keys by queries: a lane then holds four consecutive keys of one query, and their
// weights are, as they are, its operand of the second product (values' dimensions by queries), whose order of keys is
// free as long as both operands have the same. Nothing but sums over the lanes of a query crosses lanes.
//
// Two kernels share the work out as attend_plan.hpp says. `few` (up to 48 or 64 vectors of a request and key/value head): bound
// by the cache's bytes. Each of a workgroup's four waves goes through blocks of 32 keys of its own for all vectors, each block on
// its way into LDS while the one before is multiplied; the waves are joined at the end. `many`: bound by the matrix instructions
// and what feeds them. Eight waves hold 32 vectors each, and go together through blocks that are widened to fp16 once, in LDS.
#include <climits>
#include <mutex>
#include <type_traits>

#include "attend_plan.hpp"

namespace splosh {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr size_t kAttendCounterBytes = 16384;  // the workspace's first bytes belong to other kernels' counters
constexpr float kLowest = -0x1.fffffep+127f;   // M before the first key: no finite t is lower
constexpr float kSlack = 8.0f;                 // how far t may pass M before M follows
constexpr int kManyThreads = 512, kManyRows = 256;
// (Row, query head) vectors that are joined a wave each; more, sixteen lanes each. (1536 of some 35 pieces: 14 us, sixteen lanes 19; 49152 of two
// or three: 51 us, sixteen lanes 25.)
constexpr int64_t kJoinApart = 4096;
constexpr uint32_t kNoRecord = 0xffe5a7d3;     // in place of a scale: a NaN that no arithmetic gives
constexpr float kFarApart = 0x1p102f;          // the most that scales may lie apart
constexpr float kSmallScale = 0x1p-62f, kLargeScale = 4.0f;             // with one below and one above they may be
constexpr uint32_t kSmallBits = 0x20800000u, kLargeBits = 0x40800000u;  // of these
constexpr float kApart = -1.0f;                // in place of a sum, which is not negative

struct AttendArgs {
    const uint16_t *q;
    int64_t row_stride, head_stride;
    uint16_t *out;
    int64_t ld_out;
    int q_heads, shared, wide, wide_out;  // whether vectors of q are 16-byte aligned, and of out 8-byte
    float factor;               // scale log2(e)
    TileShape tile;
    Divisor by_blocks;          // a page's
    int prefix;                 // the launch over the shared prefix
    int partial;                // whether every piece leaves its partial result
    float *slots;
    int64_t first_slots;        // where the slots begin of pieces that are not their segment's first
    struct Pieces *pieces;      // of every (row, query head)
};

// Where the partial results of one (row, query head) lie, for the launch that joins them.
struct Pieces {
    int slot;       // the first one's
    int workgroup;  // the workgroup that took it; the next ones took the next, and have slots by workgroup
    int count;      // 1 and no prefix: written already; -1: of a whole segment whose scales lie far apart
    int at;         // its vector of the tile
};

// Where a piece's vectors and keys lie.
struct Piece {
    Span span;
    int request, head, tile;
    int first_block, blocks;  // of 32 keys, from the span's first on
    int slot, count;          // count: the segment's pieces, where this is the first of them; 0 else
    bool direct;              // the whole segment, and nothing to join it with
};

// Four codes, kept as code + 128, as fp16: 1024 + byte is 0x6400 | byte.
__device__ __forceinline__ f16x2 as_f16x2(uint32_t v) { return __builtin_bit_cast(f16x2, v); }
__device__ __forceinline__ f16x2 centred(uint32_t v) { return as_f16x2(v) - f16x2{(_Float16)1152, (_Float16)1152}; }
__device__ __forceinline__ void widen4(uint32_t codes, f16x2 &lo, f16x2 &hi) {
    lo = centred(perm_bytes(0x64646464u, codes, 0x04010400u));
    hi = centred(perm_bytes(0x64646464u, codes, 0x04030402u));
}
__device__ __forceinline__ f16x8 join8(f16x2 a, f16x2 b, f16x2 c, f16x2 d) {
    return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2, 3, 4,
                                   5, 6, 7);
}
__device__ __forceinline__ f16x8 widen8(uint32_t lo, uint32_t hi) {
    f16x2 a, b, c, d;
    widen4(lo, a, b);
    widen4(hi, c, d);
    return join8(a, b, c, d);
}
// Four dimensions of eight tokens, transposed: part[c] is dimension c of tokens 0..7.
__device__ __forceinline__ void widen_turned(const uint32_t (&v)[8], f16x8 (&part)[4]) {
    f16x2 of[4][4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const uint32_t low = perm_bytes(v[2 * p + 1], v[2 * p], 0x05040100u), high = perm_bytes(v[2 * p + 1], v[2 * p], 0x07060302u);
        of[0][p] = centred(perm_bytes(0x64646464u, low, 0x04020400u));
        of[1][p] = centred(perm_bytes(0x64646464u, low, 0x04030401u));
        of[2][p] = centred(perm_bytes(0x64646464u, high, 0x04020400u));
        of[3][p] = centred(perm_bytes(0x64646464u, high, 0x04030401u));
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) part[c] = join8(of[c][0], of[c][1], of[c][2], of[c][3]);
}

__device__ __forceinline__ uint32_t f16_pair(float lo, float hi) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

// Eight values of q.
__device__ __forceinline__ u32x4 load_q8(const uint16_t *at, int wide) {
    if (wide) return *reinterpret_cast<const u32x4 *>(at);
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = at[2 * e] | (uint32_t)at[2 * e + 1] << 16;
    return w;
}
__device__ __forceinline__ float largest8(const u32x4 &w) {
    float most = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        most = __builtin_fmaxf(most, __builtin_fmaxf(__builtin_fabsf(bf16_bits_to_f32(w[e])), __builtin_fabsf(__uint_as_float(w[e] & 0xffff0000u))));
    return most;
}
// The power that brings a row's largest value to [2^14, 2^15).
__device__ __forceinline__ int power_of(float most) { return 141 - (int)(__float_as_uint(most) >> 23); }
__device__ __forceinline__ u32x4 moved8(const u32x4 &v, int power) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        w[e] = f16_pair(__builtin_ldexpf(bf16_bits_to_f32(v[e]), power), __builtin_ldexpf(__uint_as_float(v[e] & 0xffff0000u), power));
    return w;
}

// A value that all lanes of the wave have, as a scalar.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ Span uniform(const Span &s) {
    return {uniform(s.begin), uniform(s.n), uniform(s.first), uniform(s.from), uniform(s.to)};
}

// The lane's number, found anew: where every register is taken, a kept one is spilled, and its reload waits for all loads into LDS.
__device__ __forceinline__ int lane_anew() {
    int lane;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
    return lane;
}

// The larger of a lane's value and that of the lane 16 (32) further: two registers' rows swapped, in place of a trip through LDS.
__device__ __forceinline__ float max_rows(float v) {
    typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));
    const u32x2v r = __builtin_bit_cast(u32x2v, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_halves(float v) {
    typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));
    const u32x2v r = __builtin_bit_cast(u32x2v, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// What the sum of a_j is divided by, for the scale of v_j. (1 where it is no scale: t is then NaN, or the key masked.)
__device__ __forceinline__ float inverse_scale(float vs) {
    const float r = __builtin_amdgcn_rcpf(vs);
    return __builtin_fabsf(r) < __builtin_inff() ? r : 1.0f;
}

// A sum against another maximum: v 2^x.
__device__ __forceinline__ float scaled(float v, float x) {
    const float root = __builtin_amdgcn_exp2f(0.5f * x);
    return v * root * root;
}

// The packed row that vector x of a tile's request is of.
__device__ __forceinline__ int row_of(const Piece &p, const TileShape &tile, int x) { return p.span.begin + tile.by_group.of(x); }
// And its query head.
__device__ __forceinline__ int head_of(const Piece &p, const TileShape &tile, int x) {
    return p.head * tile.group + x - tile.by_group.of(x) * tile.group;
}

// The last key that packed row `row` sees, of the launch's.
__device__ __forceinline__ int position_of(const AttendArgs &a, const PackedView &packed, const Piece &p, int row) {
    if (!a.prefix) return p.span.first + row - p.span.begin;
    int low = 0, high = packed.requests;  // the last request that starts at or before the row
    while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (packed.starts[mid] <= row) low = mid;
        else high = mid;
    }
    return position_in(packed, low, row);
}

// The page ids of a request, 64 columns at a time in a wave's lanes.
struct Pages {
    const int32_t *table;
    int columns, base, ids;
    __device__ __forceinline__ Pages(const PackedView &p, int request)
        : table(p.table + request * p.table_stride), columns(p.table_pages), base(-64), ids(-1) {}
    __device__ __forceinline__ int operator()(int column) {
        if (column < base || column >= base + 64) {
            base = column;
            const int c = base + (int)(threadIdx.x & 63);
            ids = c < columns ? table[c] : -1;
        }
        return __builtin_amdgcn_readlane(ids, column - base);
    }
};

// The record of a block of the request's keys; `hole`: it lies in no page (some record is given all the same).
template <int D>
__device__ __forceinline__ const uint8_t *block_record(const AttendArgs &a, const CacheView &cache, Pages &pages, int head, int block, bool &hole) {
    const int column = a.by_blocks.of(block);
    int page = pages(column);
    hole = page < 0 || page >= cache.pages;
    page = hole ? 0 : page;
    return record_of<D>(cache, page, head, block - column * cache.page_blocks);
}

// Over the wave's lanes, the running sum of v, each lane's own included: within rows of sixteen lanes, then from row to row.
__device__ __forceinline__ int running_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}
// The largest of a lane's value and those of the lanes beside it, in groups of N (4, 8 or 16).
template <int N>
__device__ __forceinline__ float group_max(float v) {
    auto other = [](float x, auto ctrl) {
        return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), decltype(ctrl)::value, 0xf, 0xf, false));
    };
    v = __builtin_fmaxf(v, other(v, std::integral_constant<int, 0xb1>{}));                      // lanes 1 0 3 2
    v = __builtin_fmaxf(v, other(v, std::integral_constant<int, 0x4e>{}));                      // lanes 2 3 0 1
    if constexpr (N >= 8) v = __builtin_fmaxf(v, other(v, std::integral_constant<int, 0x141>{}));   // eight lanes turned round
    if constexpr (N >= 16) v = __builtin_fmaxf(v, other(v, std::integral_constant<int, 0x140>{}));  // sixteen
    return v;
}

// A span's units, and the tile that unit `offset` of them is in (offset: then in that tile), 64 tiles at a time in a wave's lanes. (One after the other,
// the 48 tiles of 2048 rows with 24 heads on 4 took every workgroup 13 us.)
__device__ __forceinline__ int wave_units(const Span &span, const TileShape &tile, int tiles) {
    const int lane = threadIdx.x & 63;
    int units = 0;
    for (int base = 0; base < tiles; base += 64) units += base + lane < tiles ? tile_units(span, tile, base + lane) : 0;
    return __builtin_amdgcn_readlane(running_sum(units), 63);
}
__device__ __forceinline__ int wave_tile(const Span &span, const TileShape &tile, int tiles, int &offset) {
    const int lane = threadIdx.x & 63;
    for (int base = 0;; base += 64) {
        const int units = base + lane < tiles ? tile_units(span, tile, base + lane) : 0, units_to = running_sum(units);
        const int all = __builtin_amdgcn_readlane(units_to, 63);
        if (offset < all || base + 64 >= tiles) {
            const int t = __builtin_ctzll(__ballot(offset < units_to) | 1ull << 63);
            offset -= __builtin_amdgcn_readlane(units_to - units, t);
            return base + t;
        }
        offset -= all;
    }
}

// Calls `work` for each piece of the launch's units that workgroup blockIdx.x takes. All threads call it.
template <int THREADS, typename F>
__device__ __forceinline__ void for_pieces(const AttendArgs &a, const CacheView &cache, const PackedView &packed, F work) {
    const TileShape &tile = a.tile;
    const int w = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    // Up to 64 requests lie in a wave's lanes, and every wave sums them up by itself; more of them are runs of the workgroup's threads, which count
    // a request's tiles one after the other (8192 rows of 24 heads on 4 beside 65 single tokens take 1006 us, beside 63 of them 995).
    const bool few = packed.requests <= 64;
    Span mine{};  // the lane's request
    auto span_at = [&](int r) {
        if (!few) return uniform(own_span(packed, cache.page_tokens, a.shared, r));
        return Span{__builtin_amdgcn_readlane(mine.begin, r), __builtin_amdgcn_readlane(mine.n, r), __builtin_amdgcn_readlane(mine.first, r),
                    a.shared, packed.table_pages * cache.page_tokens};
    };
    int request = 0, total, before = 0, segment = 0;
    Span span;
    if (a.prefix) {
        span = uniform(prefix_span(packed, a.shared));
        total = tile.heads * wave_units(span, tile, tiles_of(span, tile));
    } else if (few) {
        int units = 0, segments = 0;
        if (lane < packed.requests) {
            mine = own_span(packed, cache.page_tokens, a.shared, lane);
            segments = tile.heads * tiles_of(mine, tile);
        }
        // (A lane each, or all lanes for one after the other, whichever takes fewer steps.)
        int longest = segments;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) longest = max(longest, __shfl_xor(longest, m));
        if (uniform(longest) > tile.heads * packed.requests) {
            for (int r = 0; r < packed.requests; ++r) {
                const Span s = span_at(r);
                const int all = tile.heads * wave_units(s, tile, tiles_of(s, tile));
                units = lane == r ? all : units;
            }
        } else if (lane < packed.requests) {
            units = tile.heads * units_before(mine, tile, tiles_of(mine, tile));
        }
        const int units_to = running_sum(units), segments_to = running_sum(segments);
        total = __builtin_amdgcn_readlane(units_to, 63);
        const int sharers = sharers_of(total, tile.workgroups);
        if (w >= sharers) return;
        const int first = first_unit(total, sharers, w);
        request = __builtin_ctzll(__ballot(first < units_to));
        before = __builtin_amdgcn_readlane(units_to - units, request), segment = __builtin_amdgcn_readlane(segments_to - segments, request);
        span = span_at(request);
    } else {
        __shared__ int wave_units[THREADS / 64], wave_segments[THREADS / 64], found[3];
        const int run = (packed.requests + THREADS - 1) / THREADS;
        const int low = min(tid * run, packed.requests), high = min(low + run, packed.requests);
        auto units_of = [&](int r, int &segments) {
            const Span s = own_span(packed, cache.page_tokens, a.shared, r);
            const int tiles = tiles_of(s, tile);
            segments = tile.heads * tiles;
            return tile.heads * units_before(s, tile, tiles);
        };
        int units = 0, segments = 0, n;
        bool ascending = true;
        for (int r = low; r < high; ++r) units += units_of(r, n), segments += n, ascending &= ascends(packed, r);
        int units_to = running_sum(units), segments_to = running_sum(segments);
        const bool sound = __all(ascending);
        if (lane == 63) wave_units[wave] = sound ? units_to : -1, wave_segments[wave] = segments_to;
        if (tid == 0) found[0] = -1;
        __syncthreads();
        total = 0;
        for (int i = 0; i < THREADS / 64; ++i) {
            if (wave_units[i] < 0) return;  // (starts that do not ascend: nothing is computed)
            if (i < wave) units_to += wave_units[i], segments_to += wave_segments[i];
            total += wave_units[i];
        }
        total = uniform(total);
        const int sharers = sharers_of(total, tile.workgroups), first = w < sharers ? first_unit(total, sharers, w) : total;
        int at = units_to - units, at_segment = segments_to - segments;
        if (at <= first && first < units_to) {
            for (int r = low; r < high; ++r) {
                const int u = units_of(r, n);
                if (at <= first && first < at + u) found[0] = r, found[1] = at, found[2] = at_segment;
                at += u, at_segment += n;
            }
        }
        __syncthreads();
        request = uniform(found[0]), before = uniform(found[1]), segment = uniform(found[2]);
        if (request < 0) return;
        span = span_at(request);
    }
    const int sharers = sharers_of(total, tile.workgroups);
    if (w >= sharers) return;
    int unit = first_unit(total, sharers, w);
    const int end = first_unit(total, sharers, w + 1);
    const int each = wave_units(span, tile, tiles_of(span, tile));
    int tiles = tiles_of(span, tile), offset = unit - before, head = offset / each;
    offset -= head * each;
    int t = wave_tile(span, tile, tiles, offset);
    segment += head * tiles + t;
    while (true) {
        const Cut cut = cut_of(span, tile, t, segment, offset, unit, end, w, sharers, total, a.partial, a.first_slots);
        Piece p;
        p.span = span, p.request = request, p.head = head, p.tile = t;
        p.first_block = cut.first_block, p.blocks = cut.blocks, p.slot = cut.slot, p.count = cut.count, p.direct = cut.direct;
        // (More segments than slots for them there are only where starts do not ascend.)
        if (cut.any && (!a.partial || segment < a.first_slots)) work(p);
        unit += cut.take;
        if (unit >= end) return;
        offset = 0, ++segment;
        if (++t < tiles) continue;
        t = 0;
        if (++head < tile.heads) continue;
        head = 0;
        do {  // (there is another one: the units say so)
            span = span_at(++request);
            tiles = tiles_of(span, tile);
        } while (tiles == 0 && request + 1 < packed.requests);
    }
}

// The result of vector x, dimensions d .. d + N - 1 of N sums o with maximum M: written, or left in the piece's slot.
template <int D, int N>
__device__ __forceinline__ void write_sums(const AttendArgs &a, const Piece &p, int i, int d, const float *o, float total) {
    const int x = p.tile * a.tile.rows + i;
    if (x >= p.span.n * a.tile.group) return;
    if (p.direct) {
        const int row = row_of(p, a.tile, x), h = head_of(p, a.tile, x);
        const float inv = 1.0f / total;
        uint16_t *at = a.out + row * a.ld_out + (int64_t)h * D + d;
        uint32_t pair[N / 2];
#pragma unroll
        for (int e = 0; e < N / 2; ++e) pair[e] = total == 0.0f ? 0u : f32x2_to_bf16x2(o[2 * e] * inv, o[2 * e + 1] * inv);
        if (a.wide_out) {
#pragma unroll
            for (int e = 0; e < N / 4; ++e) reinterpret_cast<u32x2 *>(at)[e] = u32x2{pair[2 * e], pair[2 * e + 1]};
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) at[e] = (uint16_t)(pair[e / 2] >> 16 * (e & 1));
        }
    } else {
        float *at = a.slots + p.slot * (a.tile.rows * (int64_t)(D + 2)) + (int64_t)i * D + d;
#pragma unroll
        for (int e = 0; e < N; e += 4) *reinterpret_cast<f32x4 *>(at + e) = f32x4{o[e], o[e + 1], o[e + 2], o[e + 3]};
    }
}
// A vector whose piece's scales lie far apart.
template <int D>
__device__ __forceinline__ void write_apart(const AttendArgs &a, const Piece &p, int i) {
    const int x = p.tile * a.tile.rows + i;
    if (x >= p.span.n * a.tile.group) return;
    if (p.count > 0)
        a.pieces[(int64_t)row_of(p, a.tile, x) * a.q_heads + head_of(p, a.tile, x)] = {p.slot, (int)blockIdx.x, p.direct ? -1 : p.count, i};
    if (!p.direct) a.slots[p.slot * (a.tile.rows * (int64_t)(D + 2)) + (int64_t)a.tile.rows * (D + 1) + i] = kApart;
}
// And its maximum and sum, where they are left; with the segment's first piece, where all of its pieces are.
template <int D>
__device__ __forceinline__ void write_total(const AttendArgs &a, const Piece &p, int i, float most, float total) {
    const int x = p.tile * a.tile.rows + i;
    if (x >= p.span.n * a.tile.group) return;
    if (p.count > 0)
        a.pieces[(int64_t)row_of(p, a.tile, x) * a.q_heads + head_of(p, a.tile, x)] = {p.slot, (int)blockIdx.x, p.count, i};
    if (p.direct) return;
    float *at = a.slots + p.slot * (a.tile.rows * (int64_t)(D + 2)) + (int64_t)a.tile.rows * D;
    at[i] = most, at[a.tile.rows + i] = total;
}

// The tile's queries as the first product's operand, 16 dimensions of a vector a thread; the powers that they are moved back by, their positions
// and the least of these.
template <int D, int R, int THREADS>
__device__ __forceinline__ void stage_queries(const AttendArgs &a, const PackedView &packed, const Piece &p, u32x4 *q_parts, float *row_factor,
                                              int *row_position, int *least) {
    constexpr int STEPS = D / 32, CHUNKS = D / 16;
    const int vectors = p.span.n * a.tile.group, tid = threadIdx.x;
    for (int item = tid; item < (R * CHUNKS + THREADS - 1) / THREADS * THREADS; item += THREADS) {
        const int i = item / CHUNKS, c = item % CHUNKS, x = p.tile * R + i;
        const bool valid = i < R && x < vectors;
        const int row = valid ? row_of(p, a.tile, x) : 0;
        u32x4 low = {}, high = {};
        if (valid) {
            const uint16_t *at = a.q + row * a.row_stride + head_of(p, a.tile, x) * a.head_stride + c * 16;
            low = load_q8(at, a.wide), high = load_q8(at + 8, a.wide);
        }
        const float most = group_max<CHUNKS>(__builtin_fmaxf(largest8(low), largest8(high)));
        const int power = power_of(most);
        if (i < R) {
            u32x4 *to = q_parts + (i / 16 * STEPS + c / 4 * 2) * 64 + (c % 4) * 16 + i % 16;
            to[0] = moved8(low, power);
            to[64] = moved8(high, power);
            if (c == 0) {
                row_factor[i] = __builtin_ldexpf(a.factor, -power);
                row_position[i] = valid ? position_of(a, packed, p, row) : -1;
                if (valid && a.prefix) atomicMin(least, row_position[i]);
            }
        }
    }
}

// The groups' sums against the largest of their maxima, added in their order: 32 vectors at a time (what the ring has room for), all threads.
template <int D, int NT, typename S, int HELD>
__device__ __forceinline__ void join_groups(const AttendArgs &a, const Piece &p, f32x4 (&acc)[HELD][NT], const float (&most)[NT], float (&total)[NT],
                                            float *joined, float *wave_most, float *wave_total, int record_group, const int *apart) {
    constexpr int R = S::kRows, GROUPS = S::kGroups, PITCH = S::kPitch;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        total[n] += __shfl_xor(total[n], 16);
        total[n] += __shfl_xor(total[n], 32);
        if (g == 0) wave_most[record_group * R + n * 16 + col] = most[n], wave_total[record_group * R + n * 16 + col] = total[n];
    }
    __syncthreads();
    static_assert(GROUPS == 4, "a word of `apart` each");
    const u32x4 any_apart = *reinterpret_cast<const u32x4 *>(apart);
    if (__builtin_expect(uniform((int)(any_apart[0] | any_apart[1] | any_apart[2] | any_apart[3])), 0)) {
        if (tid < R) write_apart<D>(a, p, tid);
        return;
    }
#pragma unroll
    for (int n0 = 0; n0 < NT; n0 += 2) {
        constexpr int MOST = NT > 1 ? 2 : 1;
        const int here = NT - n0 < MOST ? NT - n0 : MOST;
        if (n0) __syncthreads();  // (the last vectors are read)
#pragma unroll
        for (int k = 0; k < MOST; ++k) {
            const int n = n0 + k;
            if (n >= NT) break;
            float top = kLowest;
#pragma unroll
            for (int w = 0; w < GROUPS; ++w) top = __builtin_fmaxf(top, wave_most[w * R + n * 16 + col]);
            const float keep = __builtin_amdgcn_exp2f(most[n] - top);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int j = 0; j < HELD; j += 4)
                    *reinterpret_cast<f32x4 *>(joined + ((k * GROUPS + record_group) * 16 + col) * PITCH + (4 * g + e) * HELD + j) =
                        f32x4{acc[j][n][e] * keep, acc[j + 1][n][e] * keep, acc[j + 2][n][e] * keep, acc[j + 3][n][e] * keep};
        }
        __syncthreads();
        for (int item = tid; item < here * 256; item += S::kThreads) {
            const int k = item / 256, i = item / 16 % 16, d = item % 16 * (D / 16), row = (n0 + k) * 16 + i;
            float sum[D / 16] = {}, row_total = 0.0f, row_most = kLowest;
#pragma unroll
            for (int w = 0; w < GROUPS; ++w) row_most = __builtin_fmaxf(row_most, wave_most[w * R + row]);
#pragma unroll
            for (int w = 0; w < GROUPS; ++w) {
                row_total += scaled(wave_total[w * R + row], wave_most[w * R + row] - row_most);
#pragma unroll
                for (int e = 0; e < D / 16; e += 4) {
                    const f32x4 part = *reinterpret_cast<const f32x4 *>(joined + ((k * GROUPS + w) * 16 + i) * PITCH + d + e);
#pragma unroll
                    for (int f = 0; f < 4; ++f) sum[e + f] += part[f];
                }
            }
            write_sums<D, D / 16>(a, p, row, d, sum, row_total);
            if (item % 16 == 0) write_total<D>(a, p, row, row_most, row_total);
        }
    }
}

// A lane's eight scores of each vector masked, and the largest of all lanes' of the vector.
template <int NT>
__device__ __forceinline__ void mask_scores(float (&t)[NT][8], bool masked, bool dead, int block, int g, const int (&position)[NT], float (&top)[NT]) {
    if (masked) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                t[n][e] = !dead && block * kBlock + (e / 4) * 16 + 4 * g + e % 4 <= position[n] ? t[n][e] : -__builtin_inff();
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        top[n] = t[n][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top[n] = __builtin_fmaxf(top[n], t[n][e]);
        top[n] = max_halves(max_rows(top[n]));
    }
}

// Their weights against the running maxima, summed with the scales' inverses, and as the second product's operand.
template <int NT>
__device__ __forceinline__ void weigh(const float (&t)[NT][8], const float (&inverse)[8], const float (&most)[NT], float (&total)[NT], f16x8 (&weight)[NT]) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        uint32_t pairs[4];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float a = __builtin_amdgcn_exp2f(t[n][e] - most[n]), b = __builtin_amdgcn_exp2f(t[n][e + 1] - most[n]);
            total[n] = __builtin_fmaf(a, inverse[e], total[n]);
            total[n] = __builtin_fmaf(b, inverse[e + 1], total[n]);
            pairs[e / 2] = f16_pair(a, b);
        }
        const u32x4 four = {pairs[0], pairs[1], pairs[2], pairs[3]};
        weight[n] = __builtin_bit_cast(f16x8, four);
    }
}

// ---- few vectors --------------------------------------------------------------------------------
//
// A wave has two records in LDS: the one it multiplies and the next one, on its way from memory (16 bytes a lane straight into LDS), so
// that what is in flight takes no registers. Nothing is shared between the waves but the queries, and there is no
// barrier while a piece runs. A row of codes lies in LDS with its 16-byte runs exchanged by `turned`: the sixteen keys of an
// operand read then hit different banks.

template <int D>
struct FewRing {
    static constexpr int kRecord = record_bytes(D), kCodeLoads = 2 * kBlock * D / 1024, kLoads = kCodeLoads + 1;
    static constexpr int kRuns = D / 16;  // of 16 bytes, of a row
    static __device__ __forceinline__ int turned(int row, int run) {
        return run ^ (D == 64 ? (row ^ row >> 2) & 3 : row & (kRuns - 1));
    }
};

// (A wave a record. Where a wave's sums take more than 96 registers it has its SIMD for itself, and they lie in accumulation registers.)
constexpr int kFewGroups = 4;
template <int D, int NT>
struct FewShape {
    static constexpr bool kAlone = D / 16 * NT * 4 > 96;
    static constexpr int kGroups = kFewGroups, kThreads = 64 * kGroups, kRows = 16 * NT, kPitch = D + 4;
    static constexpr int kRingBytes = kGroups * 2 * FewRing<D>::kRecord, kQueryBytes = kRows * D * 2;
    static constexpr int kNumbers = kRingBytes + kQueryBytes;  // then: maxima and sums of each group, factors, positions, their least, a word a wave
    static constexpr int kLds = kNumbers + (2 * kGroups + 2) * kRows * 4 + 32;
    static_assert((NT > 1 ? 2 : 1) * kGroups * 16 * kPitch * 4 <= kRingBytes && kLds <= 160 * 1024, "LDS");
    // (LDS is given out in pieces of 1280 bytes; 48 are for_pieces' own.)
    static_assert(D == 256 || kAlone || 2 * ((kLds + 48 + 1279) / 1280 * 1280) <= 160 * 1024, "two workgroups a CU");
};

template <int D, int NT>
__global__ __launch_bounds__((FewShape<D, NT>::kThreads), (FewShape<D, NT>::kAlone ? 1 : 2)) void few_kernel(AttendArgs a, CacheView cache, PackedView packed) {
    typedef FewShape<D, NT> S;
    typedef FewRing<D> Ring;
    constexpr int R = S::kRows, SLABS = D / 64, STEPS = D / 32, GROUPS = S::kGroups, HELD = D / 16;
    extern __shared__ __align__(16) char lds[];
    u32x4 *const q_parts = reinterpret_cast<u32x4 *>(lds + S::kRingBytes);
    float *const joined = reinterpret_cast<float *>(lds);  // [group][16][PITCH], in the ring's place
    float *const wave_most = reinterpret_cast<float *>(lds + S::kNumbers), *const wave_total = wave_most + GROUPS * R;
    float *const row_factor = wave_total + GROUPS * R;
    int *const row_position = reinterpret_cast<int *>(row_factor + R), *const least = row_position + R, *const apart = least + 4;
    const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, col = lane & 15, g = lane >> 4;
    const int record_group = wave, ring = record_group * 2 * Ring::kRecord;  // where the group's two records lie

    // What load j of a record brings to the lane's 16 bytes of LDS: run (l mod kRuns) of row j (1024 / D) + l / kRuns, from where
    // `turned` has it. Only with 256 dimensions does that depend on j, and on j mod 4 alone.
    constexpr int SOURCES = D == 256 ? 4 : 1;
    uint32_t source[SOURCES];
#pragma unroll
    for (int j = 0; j < SOURCES; ++j) {
        const int row = j * (1024 / D) + lane / Ring::kRuns;
        source[j] = (uint32_t)(lane / Ring::kRuns * D + Ring::turned(row, lane % Ring::kRuns) * 16);
    }
    for_pieces<S::kThreads>(a, cache, packed, [&](const Piece &p) {
        __syncthreads();  // (the last piece's LDS is read)
        Pages pages(packed, a.prefix ? 0 : p.request);
        const int from = p.span.from / kBlock + p.first_block, to = from + p.blocks;
        bool hole = false;
        auto load = [&](int block, int buffer) {
            const uint8_t *record = block_record<D>(a, cache, pages, p.head, block, hole);
            const rsrc_t r = make_rsrc(record, Ring::kRecord);
            char *at = lds + uniform(ring + buffer * Ring::kRecord);
#pragma unroll
            for (int j = 0; j < Ring::kCodeLoads; ++j)
                buffer_load_lds16(r, at + j * 1024, source[j % SOURCES] + j * 1024);
            buffer_load_lds4(r, at + 2 * kBlock * D, 2 * kBlock * D + lane * 4);
            __builtin_amdgcn_sched_barrier(0);
        };
        if (from + record_group < to) load(from + record_group, 0);
        if (a.prefix) {
            if (tid == 0) *least = INT_MAX;
            __syncthreads();
        }
        stage_queries<D, R, S::kThreads>(a, packed, p, q_parts, row_factor, row_position, least);
        __syncthreads();
        float factor[NT], most[NT], total[NT];
        int position[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            factor[n] = row_factor[n * 16 + col], position[n] = row_position[n * 16 + col];
            most[n] = kLowest, total[n] = 0.0f;
        }
        const int first_position = a.prefix ? uniform(*least) : p.span.first + a.tile.by_group.of(p.tile * R);
        const int seen_to = tile_end(p.span, a.tile, p.tile);  // (keys that no row of the tile sees were never written)
        f32x4 acc[HELD][NT] = {};
        int buffer = 0;
        bool waited = false, dead = false;
        float least_scale = 1.0f, most_scale = 1.0f;  // of the lane's key of each record
        // Where a maximum moves by more than kSlack the loop over the records is left, the sums scaled, and the record
        // begun again: inside of it nothing but the matrix instructions touches the sums. (Scaled in a branch of the loop, the compiler holds
        // them twice, and copies 192 registers a record: 150 us for the 320 MB of the verify step.)
        for (int block = from + record_group; block < to;) {
        float top[NT];
        bool moved = false;
        do {
            if (!waited) {
                dead = hole;
                if (block + GROUPS < to) {
                    load(block + GROUPS, buffer ^ 1);
                    wait_vmcnt<Ring::kLoads>();  // this record has landed; the next may be in flight
                } else {
                    wait_vmcnt<0>();
                }
                waited = true;
            }
            asm volatile("" ::: "memory");
            const char *const record = lds + ring + buffer * Ring::kRecord;
            const float *const scales = reinterpret_cast<const float *>(record + 2 * kBlock * D) + 4 * g;
            f32x4 s[2][NT] = {};
#pragma unroll
            for (int slab = 0; slab < SLABS; ++slab) {
                u32x4 k[2];
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    k[t] = *reinterpret_cast<const u32x4 *>(record + (t * 16 + col) * D + Ring::turned(t * 16 + col, slab * 4 + g) * 16);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const f16x8 k0 = widen8(k[0][2 * half], k[0][2 * half + 1]), k1 = widen8(k[1][2 * half], k[1][2 * half + 1]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const f16x8 q = __builtin_bit_cast(f16x8, q_parts[(n * STEPS + slab * 2 + half) * 64 + lane]);
                        s[0][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q, s[0][n], 0, 0, 0);
                        s[1][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q, s[1][n], 0, 0, 0);
                    }
                }
            }
            float key_scale[8], value_log[8], inverse[8];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const f32x4 ks = *reinterpret_cast<const f32x4 *>(scales + 16 * t), vs = *reinterpret_cast<const f32x4 *>(scales + kBlock + 16 * t);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    key_scale[4 * t + e] = ks[e];
                    value_log[4 * t + e] = __builtin_amdgcn_logf(vs[e]);
                    inverse[4 * t + e] = inverse_scale(vs[e]);
                }
            }
            const bool masked = dead || block * kBlock + kBlock - 1 > first_position;
            float value_scale = __builtin_fmaxf((scales - 4 * g)[kBlock + (lane & (kBlock - 1))], kLeastScale);
            asm("" : "+v"(value_scale));  // (read whatever the lane: a branch around it parts what is scheduled together)
            const float counted = (lane & (kBlock - 1)) < (dead ? 0 : seen_to - block * kBlock) ? value_scale : 1.0f;
            least_scale = __builtin_fminf(least_scale, counted), most_scale = __builtin_fmaxf(most_scale, counted);
            f16x8 weight[NT];
            float t[NT][8];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 8; ++e) t[n][e] = __builtin_fmaf(s[e / 4][n][e % 4], key_scale[e] * factor[n], value_log[e]);
            mask_scores<NT>(t, masked, dead, block, g, position, top);
#pragma unroll
            for (int n = 0; n < NT; ++n) moved |= top[n] > most[n] + kSlack;
            moved = __any(moved);
            if (moved) {
                if (block != from + record_group) break;
                moved = false;  // (the first record: there are no sums yet)
#pragma unroll
                for (int n = 0; n < NT; ++n) most[n] = __builtin_fmaxf(top[n], most[n]);
            }
            weigh<NT>(t, inverse, most, total, weight);
            uint32_t v[8][SLABS];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int token = kBlock + (e / 4) * 16 + 4 * g + e % 4;
                const char *at = record + token * D + Ring::turned(token, col * Ring::kRuns / 16) * 16 + col * (D / 16) % 16;
                if constexpr (SLABS == 4) {
                    const u32x4 x = *reinterpret_cast<const u32x4 *>(at);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[e][i] = x[i];
                } else if constexpr (SLABS == 2) {
                    const u32x2 x = *reinterpret_cast<const u32x2 *>(at);
                    v[e][0] = x[0], v[e][1] = x[1];
                } else {
                    v[e][0] = *reinterpret_cast<const uint32_t *>(at);
                }
            }
#pragma unroll
            for (int slab = 0; slab < SLABS; ++slab) {
                uint32_t of[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) of[e] = v[e][slab];
                f16x8 part[4];
                widen_turned(of, part);
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        acc[slab * 4 + c][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(part[c], weight[n], acc[slab * 4 + c][n], 0, 0, 0);
            }
            // The record is read before the load after the next overwrites it.
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            block += GROUPS, buffer ^= 1, waited = false;
        } while (block < to);
        if (moved) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float now = __builtin_fmaxf(top[n], most[n]), keep = __builtin_amdgcn_exp2f(most[n] - now);
                total[n] = scaled(total[n], most[n] - now);
                most[n] = now;
#pragma unroll
                for (int j = 0; j < HELD; ++j) acc[j][n] *= keep;
            }
        }
        }
        apart[wave] = __any(most_scale > kSmallScale * kFarApart) | (__any(most_scale > kLargeScale) & __any(least_scale < kSmallScale));
        join_groups<D, NT, S, HELD>(a, p, acc, most, total, joined, wave_most, wave_total, record_group, apart);
    });
}

// ---- many vectors -------------------------------------------------------------------------------

template <int D>
struct ManyShape {
    // Records of a step: what the eight waves widen and multiply in one is the same for every dim. (With one, a step of fewer dimensions
    // is shorter than the way of its loads from memory: 2048 rows on 6144 with 24 heads on 4 took 272 us instead of 247 with 128
    // dimensions, 204 instead of 180 with 64.)
    static constexpr int kRecords = 256 / D;
    static constexpr int kPitch = 1024 + 64;  // of a step of keys: spreads a quad's writes over the banks
    static constexpr int kRaw = kRecords * record_bytes(D), kKeys = 2 * kRaw, kValues = kKeys + 3 * 16 * kPitch, kScales = kValues + 4 * 16 * 1024;
    static constexpr int kEnds = kScales + 4 * kRecords * 3 * kBlock * 4;  // the bits of the least and of the largest scale
    static constexpr int kThreads = kManyThreads, kLds = kEnds + 16;
    static constexpr int kSumPitch = D + 4;
    static_assert(kLds <= 160 * 1024 && 8 * 16 * kSumPitch * 4 <= kLds, "LDS");
};

template <int D>
__global__ __launch_bounds__(kManyThreads) void many_kernel(AttendArgs a, CacheView cache, PackedView packed) {
    constexpr int STEPS = D / 16, TILES = D / 32, K_PITCH = ManyShape<D>::kPitch, RECORDS = ManyShape<D>::kRecords;
    // Operands are read from LDS this many products ahead of their own, and the order is kept: left to the compiler's scheduler, each was
    // read right before its product, and half of a step went by waiting (prompt chunk 462 us instead of 437).
    constexpr int KEYS_AHEAD = D == 256 ? 2 : 4;  // (256: more of them push queries out of the registers)
    typedef ManyShape<D> S;
    extern __shared__ __align__(16) char lds[];  // two steps' records as they are, then three of keys, four of values and of scales as they are used
    uint8_t *const key_parts = reinterpret_cast<uint8_t *>(lds + S::kKeys);
    u32x4 *const value_parts = reinterpret_cast<u32x4 *>(lds + S::kValues);
    float *const scales = reinterpret_cast<float *>(lds + S::kScales);
    uint32_t *const scale_ends = reinterpret_cast<uint32_t *>(lds + S::kEnds);
    const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, col = lane & 31, g = lane >> 5;

    for_pieces<kManyThreads>(a, cache, packed, [&](const Piece &p) {
        const int vectors = p.span.n * a.tile.group;
        const int x = p.tile * kManyRows + wave * 32 + col;
        const bool valid = x < vectors;
        const int row = valid ? row_of(p, a.tile, x) : 0;
        const int position = valid ? position_of(a, packed, p, row) : INT_MAX;
        int first_position = position;  // of the wave's vectors
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) first_position = min(first_position, __shfl_xor(first_position, m));
        first_position = uniform(first_position);
        // The lane's vector, half of its dimensions.
        f16x8 q[STEPS];
        float factor;
        {
            float most = 0.0f;
            const uint16_t *at = a.q + row * a.row_stride + head_of(p, a.tile, valid ? x : 0) * a.head_stride + g * 8;
            u32x4 held[STEPS];
#pragma unroll
            for (int s = 0; s < STEPS; ++s) held[s] = load_q8(at + 16 * s, a.wide);
#pragma unroll
            for (int s = 0; s < STEPS; ++s) most = __builtin_fmaxf(most, largest8(held[s]));
            most = max_halves(most);
            const int power = power_of(most);
            factor = __builtin_ldexpf(a.factor, -power);
#pragma unroll
            for (int s = 0; s < STEPS; ++s) q[s] = __builtin_bit_cast(f16x8, moved8(held[s], power));
        }
        f32x16 acc[TILES] = {};
        float most = kLowest, total = 0.0f;
        Pages pages(packed, a.prefix ? 0 : p.request);
        const int from = p.span.from / kBlock + p.first_block, to = from + p.blocks;

        // A step's records go straight into LDS three steps before they are multiplied, and are widened to fp16 two steps before. Waves 0 to 3
        // do that with the values (a thread four dimensions of eight of them) and the scales, waves 4 to 7 with the keys (16-byte runs).
        const int quarter = wave & 3, record_at = quarter * RECORDS / 4;  // what the wave loads: 2 KiB of codes of this record of a step
        bool none = false, hole = false;  // whether its page is none; whether its record is
        int left = 0;                     // records of the page behind `next`, itself included
        const uint8_t *next = nullptr;
        auto fetch = [&](int first, int buffer) {
            const int lane = lane_anew(), block = first + record_at;
            hole = true;
            if (block >= to) return;
            if (left <= 0) {
                next = block_record<D>(a, cache, pages, p.head, block, none);
                left = cache.page_blocks - (block - a.by_blocks.of(block) * cache.page_blocks);
            }
            hole = none;
            const rsrc_t r = make_rsrc(next, record_bytes(D));
            next += RECORDS * record_bytes(D), left -= RECORDS;
            const int part = (wave < 4 ? kBlock * D : 0) + quarter % (4 / RECORDS) * 2048;
            char *const at = lds + (buffer * RECORDS + record_at) * record_bytes(D);
#pragma unroll
            for (int n = 0; n < 2; ++n) buffer_load_lds16(r, at + part + n * 1024, part + n * 1024 + lane * 16);
            if (wave < 4) buffer_load_lds4(r, at + 2 * kBlock * D, 2 * kBlock * D + lane * 4);
            __builtin_amdgcn_sched_barrier(0);
        };

        // The wave's part of the records in `buffer` widened to place `third` of the keys or `fourth` of the values and scales, and between that
        // (MULTIPLY) the scores of the keys at place `keys`: the products run while the codes are widened (one after the other, the prompt
        // chunk took 437 us instead of 426). `first`: the first of the records' blocks; `dead`: the one whose
        // scales are the wave's is none.
        f32x16 s[RECORDS];
        auto widen_and_score = [&](auto values, auto multiply, int first, int buffer, int third, int fourth, int keys, bool dead) {
            constexpr bool VALUES = decltype(values)::value, MULTIPLY = decltype(multiply)::value;
            const char *const raw = lds + buffer * S::kRaw;
            const int lane = lane_anew(), tid = quarter * 64 + lane;
            const int record = tid / D, combo = tid % D / (D / 4), quad = tid % (D / 4), value_step = combo >> 1, value_g = combo & 1;
            uint32_t v[8];
            u32x4 run[2];
            float scale = 0.0f;
            if constexpr (VALUES) {
                const char *const at = raw + record * record_bytes(D) + (kBlock + 16 * value_step + 4 * value_g) * D + quad * 4;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = *reinterpret_cast<const uint32_t *>(at + (e / 4 * 8 + e % 4) * D);
                scale = reinterpret_cast<const float *>(raw + record_at * record_bytes(D) + 2 * kBlock * D)[lane];
            } else {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int all = tid + 256 * n, item = all % (2 * D);
                    run[n] = *reinterpret_cast<const u32x4 *>(raw + all / (2 * D) * record_bytes(D) + item / 4 % 32 * D + (item / 128 * 4 + item % 4) * 16);
                }
            }
            auto turn = [&] {  // pairs of tokens: v[2p] and v[2p + 1] to their bytes 0, 1 and 2, 3
                if constexpr (VALUES) {
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        const uint32_t low = perm_bytes(v[2 * p + 1], v[2 * p], 0x05040100u), high = perm_bytes(v[2 * p + 1], v[2 * p], 0x07060302u);
                        v[2 * p] = low, v[2 * p + 1] = high;
                    }
                }
            };
            auto piece = [&](int c) {
                if constexpr (VALUES) {
                    f16x2 of[4];
#pragma unroll
                    for (int p = 0; p < 4; ++p) of[p] = centred(perm_bytes(0x64646464u, v[2 * p + c / 2], c % 2 ? 0x04030401u : 0x04020400u));
                    const int t = D == 64 ? c >> 1 : quad / 32 * 4 + c, m = D == 64 ? (c & 1) * 16 + quad : quad % 32;
                    value_parts[(((fourth * RECORDS + record) * TILES + t) * 2 + value_step) * 64 + value_g * 32 + m] =
                        __builtin_bit_cast(u32x4, join8(of[0], of[1], of[2], of[3]));
                } else {
                    const int all = tid + 256 * (c / 2), item = all % (2 * D), half = c % 2;
                    uint8_t *const at = key_parts + ((third * RECORDS + all / (2 * D)) * STEPS + item / 128 * 4 + item % 4) * K_PITCH + item / 4 % 32 * 16;
                    *reinterpret_cast<f16x8 *>(at + 512 * half) = widen8(run[c / 2][2 * half], run[c / 2][2 * half + 1]);
                }
            };
            if constexpr (MULTIPLY) {
                const uint8_t *const at = key_parts + keys * 16 * K_PITCH + lane * 16;
                auto key = [&](int i) { return *reinterpret_cast<const f16x8 *>(at + i * K_PITCH); };
                f16x8 k[KEYS_AHEAD];
#pragma unroll
                for (int i = 0; i < KEYS_AHEAD; ++i) k[i] = key(i);
#pragma unroll
                for (int r = 0; r < RECORDS; ++r) s[r] = f32x16{};
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    __builtin_amdgcn_sched_barrier(0);
                    s[i / STEPS] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[i % KEYS_AHEAD], q[i % STEPS], s[i / STEPS], 0, 0, 0);
                    if (i + KEYS_AHEAD < 16) k[i % KEYS_AHEAD] = key(i + KEYS_AHEAD);
                    if (i == 4) turn();
                    if (i == 5 || i == 7 || i == 10 || i == 13) piece(i / 3 - 1);
                }
                __builtin_amdgcn_sched_barrier(0);
            } else {
                turn();
#pragma unroll
                for (int c = 0; c < 4; ++c) piece(c);
            }
            if constexpr (VALUES) {
                // (A record that is none: a key's scale that no record holds.)
                if (quarter % (4 / RECORDS) == 0) {
                    float *const at = scales + (fourth * RECORDS + record_at) * 3 * kBlock + lane;
                    at[0] = lane >= kBlock ? __builtin_amdgcn_logf(scale) : dead ? __uint_as_float(kNoRecord) : scale;
                    if (lane >= kBlock) at[kBlock] = inverse_scale(scale);
                    const uint32_t bits = __float_as_uint(scale);  // (0, and less than 0 as a float, are not looked at either)
                    if (__builtin_expect(__any((lane >= kBlock) & (bits - kSmallBits > kLargeBits - kSmallBits) & (bits - 1 < 0x7f800000u)), 0)) {
                        if (!dead & (lane >= kBlock) & (bits - 1 < 0x7f800000u) & ((first + record_at) * kBlock + lane - kBlock < tile_end(p.span, a.tile, p.tile)))
                            atomicMin(&scale_ends[0], bits), atomicMax(&scale_ends[1], bits);
                    }
                }
            }
        };
        auto part_of_step = [&](auto multiply, int first, int buffer, int third, int fourth, int keys, bool dead) {
            if (wave < 4) widen_and_score(std::true_type{}, multiply, first, buffer, third, fourth, keys, dead);
            else widen_and_score(std::false_type{}, multiply, first, buffer, third, fourth, keys, dead);
        };

        auto weigh_values = [&](int block, int fourth) {
            constexpr int KEYS = 16 * RECORDS, PRODUCTS = 2 * TILES * RECORDS, GROUPS = 2 * RECORDS;  // a lane's; groups of eight weights
            const int lane = lane_anew(), g = lane >> 5;
            auto value = [&](int n) {  // group n / TILES, tile n % TILES
                return __builtin_bit_cast(f16x8, value_parts[(((fourth * RECORDS + n / TILES / 2) * TILES + n % TILES) * 2 + n / TILES % 2) * 64 + lane]);
            };
            const float *const at = scales + fourth * RECORDS * 3 * kBlock + 4 * g;
            bool masked = (block + RECORDS) * kBlock - 1 > first_position;
            float t[KEYS], top = -__builtin_inff();
            uint32_t seen = ~0u;  // a bit a record
#pragma unroll
            for (int r = 0; r < RECORDS; ++r)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const f32x4 ks = *reinterpret_cast<const f32x4 *>(at + r * 3 * kBlock + 8 * b);
                    const f32x4 lv = *reinterpret_cast<const f32x4 *>(at + r * 3 * kBlock + kBlock + 8 * b);
                    if (b == 0) {
                        const bool dead = (uint32_t)uniform((int)__float_as_uint(ks[0])) == kNoRecord;
                        masked |= dead, seen &= dead ? ~(1u << r) : ~0u;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) t[16 * r + 4 * b + e] = __builtin_fmaf(s[r][4 * b + e], ks[e] * factor, lv[e]);
                }
            if (masked) {
#pragma unroll
                for (int e = 0; e < KEYS; ++e)
                    t[e] = (seen >> e / 16 & 1) && (block + e / 16) * kBlock + e % 16 / 4 * 8 + 4 * g + e % 4 <= position ? t[e] : -__builtin_inff();
            }
#pragma unroll
            for (int e = 0; e < KEYS; ++e) top = __builtin_fmaxf(top, t[e]);
            top = max_halves(top);
            if (__any(top > most + kSlack)) {
                top = __builtin_fmaxf(top, most);
                const float keep = __builtin_amdgcn_exp2f(most - top);
                total = scaled(total, most - top);
                most = top;
#pragma unroll
                for (int j = 0; j < TILES; ++j) acc[j] *= keep;
            }
            // The first eight weights, and each next eight between the products with those before.
            auto weigh = [&](int e, float inverse) {
                t[e] = __builtin_amdgcn_exp2f(t[e] - most);
                total = __builtin_fmaf(t[e], inverse, total);
            };
            auto inverses = [&](int e) { return *reinterpret_cast<const f32x4 *>(at + e / 16 * 3 * kBlock + 2 * kBlock + e % 16 / 4 * 8); };
            u32x4 pairs;
            auto pack = [&](int group) {
#pragma unroll
                for (int e = 0; e < 4; ++e) pairs[e] = f16_pair(t[8 * group + 2 * e], t[8 * group + 2 * e + 1]);
            };
            f16x8 v[PRODUCTS];
            // (How many are read once product n is begun: with 256 dimensions there is room for two ahead until weights are done with.)
            auto read = [](int n) {
                const int ahead = D < 256 ? 4 : n < TILES ? 2 : 4;
                return n + 1 + ahead < PRODUCTS ? n + 1 + ahead : PRODUCTS;
            };
#pragma unroll
            for (int n = 0; n < read(-1); ++n) v[n] = value(n);
            f32x4 inverse[2 * GROUPS];
#pragma unroll
            for (int b = 0; b < 2; ++b) inverse[b] = inverses(4 * b);
#pragma unroll
            for (int e = 0; e < 8; ++e) weigh(e, inverse[e / 4][e % 4]);
            pack(0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int b = 2; b < 4; ++b) inverse[b] = inverses(4 * b);
#pragma unroll
            for (int n = 0; n < PRODUCTS; ++n) {
                constexpr int EACH = 8 / TILES;
                const int group = n / TILES;
                __builtin_amdgcn_sched_barrier(0);
                if (n % TILES == 0 && group > 0) pack(group);
                acc[n % TILES] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[n], __builtin_bit_cast(f16x8, pairs), acc[n % TILES], 0, 0, 0);
#pragma unroll
                for (int m = read(n - 1); m < read(n); ++m) v[m] = value(m);
                if (n % TILES == 0 && group + 2 < GROUPS)  // those of the weights after the next
#pragma unroll
                    for (int b = 2 * group + 4; b < 2 * group + 6; ++b) inverse[b] = inverses(4 * b);
                if (group + 1 < GROUPS) {
#pragma unroll
                    for (int e = 8 * (group + 1) + n % TILES * EACH; e < 8 * (group + 1) + (n % TILES + 1) * EACH; ++e) weigh(e, inverse[e / 4][e % 4]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        };

        lds_barrier();  // (the last piece's LDS is read)
        if (tid == 0) scale_ends[0] = kSmallBits, scale_ends[1] = kLargeBits;
        bool staged_hole = true;  // of the record that is widened next
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            if (from + n * RECORDS < to) fetch(from + n * RECORDS, n);
            if (n == 0) staged_hole = hole;
        }
        wait_vmcnt<0>();
        lds_barrier();
        part_of_step(std::false_type{}, from, 0, 0, 0, 0, staged_hole);
        if (from + RECORDS < to) part_of_step(std::false_type{}, from + RECORDS, 1, 1, 1, 0, hole);
        lds_barrier();
        if (from + 2 * RECORDS < to) fetch(from + 2 * RECORDS, 0);
        staged_hole = hole;
        wait_vmcnt<0>();
        // A step is the scores of its records, while those of the step after the next are widened, and then its values. Waves 4 to 7 are half
        // a step behind: of a SIMD's two waves one has vector instructions where the other has few.
        lds_barrier();
        if (wave >= 4) lds_barrier();
        int third = 0, step = 0;
        for (int block = from; block < to; block += RECORDS, ++step) {
            if (block + 3 * RECORDS < to) fetch(block + 3 * RECORDS, (step + 1) & 1);
            // (Behind the last records something that nothing reads is widened once more.)
            part_of_step(std::true_type{}, block + 2 * RECORDS, step & 1, third == 0 ? 2 : third - 1, (step + 2) & 3, third, staged_hole);
            staged_hole = hole;
            lds_barrier();
            weigh_values(block, step & 3);
            third = third == 2 ? 0 : third + 1;
            wait_vmcnt<0>();
            lds_barrier();
        }
        if (wave < 4) lds_barrier();
        if (__builtin_expect(__uint_as_float(uniform((int)scale_ends[0])) < __uint_as_float(uniform((int)scale_ends[1])) / kFarApart, 0)) {
            if (g == 0) write_apart<D>(a, p, wave * 32 + col);
            return;
        }
        total += __shfl_xor(total, 32);
        // The wave's sums go through its eighth of the LDS, sixteen vectors at a time, and out in whole rows: as the lanes have them, 16 bytes
        // of 32 rows at once, 256 vectors of 256 dimensions took 9.7 us.
        float *const turned = reinterpret_cast<float *>(lds) + wave * 16 * S::kSumPitch;
        constexpr int ROWS = 256 / D;  // at once, 16 bytes a lane
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
            if (col >> 4 == half) {
                float *const at = turned + (col & 15) * S::kSumPitch;
                if constexpr (D > 64) {
#pragma unroll
                    for (int b = 0; b < 4; ++b)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int j = 0; j < TILES; j += 4)
                                *reinterpret_cast<f32x4 *>(at + 4 * (8 * j + 8 * b + 4 * g + e)) =
                                    f32x4{acc[j][4 * b + e], acc[j + 1][4 * b + e], acc[j + 2][4 * b + e], acc[j + 3][4 * b + e]};
                } else {
                    // Tile t, row m holds dimension 4 (m % 16) + 2 t + m / 16: rows m and m + 16 of both tiles are four in a row.
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            *reinterpret_cast<f32x4 *>(at + 4 * (8 * b + 4 * g + e)) =
                                f32x4{acc[0][4 * b + e], acc[0][4 * b + 8 + e], acc[1][4 * b + e], acc[1][4 * b + 8 + e]};
                }
            }
            // (What the wave's lanes wrote for each other: nothing of it is another wave's.)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll 2
            for (int n = 0; n < 16; n += ROWS) {
                const int i = n + lane / (D / 4), d = lane % (D / 4) * 4;
                const f32x4 x = *reinterpret_cast<const f32x4 *>(turned + i * S::kSumPitch + d);
                const float o[4] = {x[0], x[1], x[2], x[3]};
                write_sums<D, 4>(a, p, wave * 32 + 16 * half + i, d, o, __shfl(total, 16 * half + i));
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        if (g == 0) write_total<D>(a, p, wave * 32 + col, most, total);
    });
}

// ---- the pieces joined ----------------------------------------------------------------------------

// LANES lanes a (row, query head): the weights of its pieces, one a lane, and their sums in the order of the keys, BATCH pieces'
// loads at a time. All 64 where there are few vectors, of many pieces each: what it takes is then three loads one after the other.
// Sixteen where there are many: four vectors' loads are under way in a wave at once.
//
// A vector whose scales lie far apart: its keys, LANES at a time, a lane a key for the scores and a lane E dimensions for the sums, with a maximum of the
// scores of its own for what is divided by. (Eight requests of 4096 tokens with 24 heads of 256 on 4: 768 us, 30 where nothing is left to this; 1024 rows on
// 1024 before them: 3.4 ms, 105.)
template <int D, int LANES>
__device__ __forceinline__ void apart_vector(const AttendArgs &a, const CacheView &cache, const PackedView &packed, int row, int h, float (&o)[D / LANES], float &total) {
    constexpr int E = D / LANES;
    struct alignas(E) Codes {
        uint8_t of[E];
    };
    const int lane = threadIdx.x % LANES;
    int request = 0;  // the last that starts at or before the row
    for (int step = 1 << 16; step; step >>= 1)
        if (request + step < packed.requests && packed.starts[request + step] <= row) request += step;
    const Span span = own_span(packed, cache.page_tokens, 0, request);
    const int end = min(span.first + row - span.begin + 1, span.to), head = h / a.tile.group;
    const uint16_t *const q = a.q + row * a.row_stride + h * a.head_stride;
    float largest = 0.0f;
    for (int d = 0; d < D; d += 8) largest = __builtin_fmaxf(largest, largest8(load_q8(q + d, a.wide)));
    const int power = power_of(largest);
    const float factor = __builtin_ldexpf(a.factor, -power);
    float most = kLowest, top = kLowest;  // of the weights' exponents, of the scores
    total = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
    for (int first = 0; first < end; first += LANES) {
        const int key = first + lane;
        const uint8_t *record = nullptr;  // of the lane's key, where it has one
        int page, at, token = 0;
        if (key < end && place_of(cache, packed, key < a.shared ? 0 : request, key, page, at)) record = record_of<D>(cache, page, head, at / kBlock), token = at % kBlock;
        float score = -__builtin_inff(), t = score;
        if (record) {
            float s = 0.0f;
#pragma unroll 4
            for (int d = 0; d < D; d += 8) {
                const u32x4 x = load_q8(q + d, a.wide);
                const u32x2 k = *reinterpret_cast<const u32x2 *>(record + token * D + d);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float v = e % 2 ? __uint_as_float(x[e / 2] & 0xffff0000u) : bf16_bits_to_f32(x[e / 2]);
                    s += __builtin_ldexpf(v, power) * (float)((int)(k[e / 4] >> 8 * (e % 4) & 0xff) - 128);
                }
            }
            const float *const scales = reinterpret_cast<const float *>(record + 2 * kBlock * D) + token;
            score = s * (scales[0] * factor);
            t = score + __builtin_amdgcn_logf(scales[kBlock]);
        }
        float now = __builtin_fmaxf(most, t), now_top = __builtin_fmaxf(top, score);
#pragma unroll
        for (int m = 1; m < LANES; m <<= 1) now = __builtin_fmaxf(now, __shfl_xor(now, m)), now_top = __builtin_fmaxf(now_top, __shfl_xor(now_top, m));
        const float keep = __builtin_amdgcn_exp2f(most - now), weight = __builtin_amdgcn_exp2f(t - now);
        float sum = __builtin_amdgcn_exp2f(score - now_top);
#pragma unroll
        for (int m = 1; m < LANES; m <<= 1) sum += __shfl_xor(sum, m);
        total = total * __builtin_amdgcn_exp2f(top - now_top) + sum;
        most = now, top = now_top;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] *= keep;
        // The values of each key in turn, from where that key's lane found them. (Where it found none its weight is 0.)
        const int64_t where = reinterpret_cast<int64_t>(record ? record + (kBlock + token) * D : cache.data);
#pragma unroll 4
        for (int j = 0; j < LANES; ++j) {
            const Codes codes = reinterpret_cast<const Codes *>(__shfl(where, j, LANES))[lane];
            const float w = __shfl(weight, j, LANES);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += w * (float)((int)codes.of[e] - 128);
        }
    }
    total = scaled(total, top - most);  // (against the same maximum as the sums)
}

template <int D, int LANES>
__global__ __launch_bounds__(256) void join_kernel(AttendArgs own, AttendArgs prefix, CacheView cache, PackedView packed) {
    constexpr int E = D / LANES, BATCH = LANES == 64 ? 16 : 64 / E < 4 ? 64 / E : 4;
    typedef float Sums __attribute__((ext_vector_type(E == 1 ? 2 : E < 4 ? E : 4)));
    const int64_t vector = (long_block() * blockDim.x + threadIdx.x) / LANES;
    if (vector >= (int64_t)packed.rows * own.q_heads) return;
    const int lane = threadIdx.x % LANES, row = (int)(vector / own.q_heads), h = (int)(vector % own.q_heads);
    const int begin = packed.starts[0], end = packed.starts[packed.requests];  // (all four loads at once)
    const Pieces mine = own.pieces[vector], theirs = prefix.pieces[vector];
    if (row >= end | row < begin | (mine.count == 1 && !own.partial)) return;
    float top = kLowest, total = 0.0f, o[E] = {};
    bool apart = mine.count < 0;
    auto join = [&](const AttendArgs &l, const Pieces &p) {
        const int rows = l.tile.rows, last = (int)l.first_slots + l.tile.workgroups;
        const int64_t size = rows * (int64_t)(D + 2);
        // (Of rows that no request has, where starts do not ascend, this is what the workspace happened to hold.)
        if (p.slot < 0 || p.slot >= last || p.workgroup < 0 || p.count < 1 || p.count > l.tile.workgroups - p.workgroup || p.at < 0 || p.at >= rows) return;
        auto slot = [&](int j) { return l.slots + (j == 0 ? p.slot : l.first_slots + p.workgroup + j) * size; };
        for (int base = 0; base < p.count; base += LANES) {
            const int j = base + lane, here = min(LANES, p.count - base);
            float most = kLowest, sum = 0.0f;
            if (j < p.count) {
                const float *at = slot(j) + (int64_t)rows * D + p.at;
                most = at[0], sum = at[rows];
            }
            const uint64_t marked = __ballot(sum == kApart);
            if (__builtin_expect(marked != 0, 0)) apart |= (marked >> (threadIdx.x & 63 & ~(LANES - 1)) & (~0ull >> (64 - LANES))) != 0;
            float part[BATCH][E];
            auto load = [&](int first) {
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                    const float *at = slot(base + min(first + k, here - 1)) + (int64_t)p.at * D + lane * E;
                    if constexpr (E == 1) {
                        part[k][0] = *at;
                    } else {
                        constexpr int RUN = E < 4 ? E : 4;
#pragma unroll
                        for (int e = 0; e < E; e += RUN) {
                            const Sums v = *reinterpret_cast<const Sums *>(at + e);
#pragma unroll
                            for (int f = 0; f < RUN; ++f) part[k][e + f] = v[f];
                        }
                    }
                }
            };
            float now = __builtin_fmaxf(top, most);
#pragma unroll
            for (int m = 1; m < LANES; m <<= 1) now = __builtin_fmaxf(now, __shfl_xor(now, m));
            const float keep = __builtin_amdgcn_exp2f(top - now), weight = __builtin_amdgcn_exp2f(most - now);
            sum = scaled(sum, most - now), total = scaled(total, top - now);
            top = now;
#pragma unroll
            for (int m = 1; m < LANES; m <<= 1) sum += __shfl_xor(sum, m);
            total += sum;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= keep;
            for (int first = 0; first < here; first += BATCH) {
                load(first);
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                    const float w = __shfl(weight, (first + k) % LANES, LANES);
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e] = first + k < here ? o[e] + w * part[k][e] : o[e];
                }
            }
        }
    };
    if (own.partial) join(prefix, theirs);
    join(own, mine);
    if (__builtin_expect(apart, 0)) apart_vector<D, LANES>(own, cache, packed, row, h, o, total);
    uint16_t *at = own.out + row * own.ld_out + (int64_t)h * D + lane * E;
    const float inv = 1.0f / total;
    if constexpr (E >= 4) {
        if (own.wide_out) {
#pragma unroll
            for (int e = 0; e < E; e += 4)
                *reinterpret_cast<u32x2 *>(at + e) = total == 0.0f ? u32x2{} : u32x2{f32x2_to_bf16x2(o[e] * inv, o[e + 1] * inv),
                                                                                    f32x2_to_bf16x2(o[e + 2] * inv, o[e + 3] * inv)};
            return;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) at[e] = total == 0.0f ? 0 : f32_to_bf16(o[e] * inv);
}

// ---- host -----------------------------------------------------------------------------------------

struct AttendPlan {
    bool few;
    TileShape tile;
    int64_t segments;  // at most
    // A workgroup leaves one piece at most that ends before its segment does, and one that does not begin with it; where every
    // segment leaves its sums (a prefix is to be joined), each has a slot.
    int64_t first_slots(bool partial) const { return partial ? segments : tile.workgroups; }
    size_t slot_rows(bool partial) const { return (size_t)((first_slots(partial) + tile.workgroups) * tile.rows); }  // of dim + 2 floats
};

// `vectors`: those of a request and key/value head, on average. (Few and many, eight requests of 8192 tokens with 24 heads on 4, us, at 18, 30,
// 48 and 60 vectors: 256 dimensions 46, 47, 63 and 200, where a wave's sums no longer fit into its registers, against 101 at each of them;
// 128 dimensions 28, 29, 37 and 60 against 66 to 68; 64 dimensions 22, 22, 27 and 31 against 53.)
static AttendPlan plan_launch(int64_t vectors, int64_t requests, int64_t rows, int64_t q_heads, const splosh_cache &cache) {
    AttendPlan p;
    const int cus = device_cus();
    p.few = vectors <= (cache.dim == 256 ? 48 : 64);
    const int nt = (int)((vectors + 15) / 16), keys = (p.few ? kFewGroups : cache.dim == 64 ? 4 : 2) * kBlock;  // (whole steps)
    const int tile = p.few ? 16 * nt : kManyRows, workgroups = p.few && cache.dim < 256 ? 2 * cus : cus;
    p.segments = most_segments(requests, rows, q_heads, cache.heads, tile);
    // What a segment costs beside its keys (its queries, filling the pipeline, its sums out), in units of keys. Few vectors: 3 (with 1 the
    // decode step of 64 requests is 119 us instead of 116, the verify step 108 instead of 106). Many: 5, with dim 64, whose units are
    // twice as long, 3 (with 1 a prompt of 8192 rows of 24 heads on 4 takes 1190 us instead of 944, with 64 dimensions 478 instead of 395; 7 and 10 are
    // level or slower). Where segments are so few that each is cut over four workgroups or more, 1: a unit more or less is a large part of
    // a share then (7 requests of 333 rows, heads of 128: 31.5 us instead of 33.6).
    const int extra = p.few ? 3 : p.segments * 4 < workgroups ? 1 : cache.dim == 64 ? 3 : 5;
    p.tile = tile_shape(tile, keys, extra, (int)(q_heads / cache.heads), (int)cache.heads, workgroups);
    return p;
}
static AttendPlan plan_own(const splosh_cache &cache, int64_t requests, int64_t rows, int64_t q_heads) {
    return plan_launch((rows + requests - 1) / requests * (q_heads / cache.heads), requests, rows, q_heads, cache);
}
static AttendPlan plan_prefix(const splosh_cache &cache, int64_t rows, int64_t q_heads) {
    return plan_launch(rows * (q_heads / cache.heads), 1, rows, q_heads, cache);
}
// Where the vectors' pieces are, of each launch.
static size_t pieces_bytes(int64_t rows, int64_t q_heads) { return (size_t)(rows * q_heads) * sizeof(Pieces); }

// Units are counted in 32 bits: whether a launch of this size can have no more.
bool attend_fits(const splosh_cache &cache, int64_t requests, int64_t rows, int64_t q_heads, int64_t tokens) {
    const AttendPlan p = plan_own(cache, requests, rows, q_heads);
    return p.segments * (tokens / p.tile.keys + 2 + p.tile.extra) < INT32_MAX && p.segments + p.tile.workgroups < INT32_MAX;
}

size_t attend_workspace_bytes(const splosh_cache &cache, int64_t requests, int64_t rows, int64_t q_heads, int64_t shared) {
    size_t slots = plan_own(cache, requests, rows, q_heads).slot_rows(shared > 0);
    if (shared > 0) slots += plan_prefix(cache, rows, q_heads).slot_rows(true);
    return kAttendCounterBytes + (shared > 0 ? 2 : 1) * pieces_bytes(rows, q_heads) + slots * (size_t)(cache.dim + 2) * sizeof(float);
}

// (More dynamic LDS than the default 64 KiB has to be allowed, once a device.)
template <typename S, typename K>
static void launch_lds(K kernel, int grid, hipStream_t stream, const AttendArgs &a, const CacheView &cache, const PackedView &packed) {
    static std::once_flag allowed[64];
    int device = 0;
    (void)hipGetDevice(&device);
    std::call_once(allowed[device & 63], [&] {
        (void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, S::kLds);
    });
    kernel<<<grid, S::kThreads, S::kLds, stream>>>(a, cache, packed);
}

template <int D>
static void launch_part(const AttendPlan &plan, const AttendArgs &a, const CacheView &cache, const PackedView &packed,
                        hipStream_t stream) {
    auto few = [&](auto tiles) {
        constexpr int NT = decltype(tiles)::value;
        launch_lds<FewShape<D, NT>>(few_kernel<D, NT>, plan.tile.workgroups, stream, a, cache, packed);
    };
    if (!plan.few) launch_lds<ManyShape<D>>(many_kernel<D>, plan.tile.workgroups, stream, a, cache, packed);
    else if (plan.tile.rows == 16) few(std::integral_constant<int, 1>{});
    else if (plan.tile.rows == 32) few(std::integral_constant<int, 2>{});
    else if (plan.tile.rows == 48) few(std::integral_constant<int, 3>{});
    else if constexpr (D < 256) few(std::integral_constant<int, 4>{});
}

hipError_t launch_attend(const uint16_t *q, int64_t row_stride, int64_t head_stride, int64_t q_heads,
                         const splosh_cache &cache, const splosh_packed &packed, int64_t rows, int64_t shared,
                         float scale, uint16_t *out, int64_t ld_out, void *workspace, hipStream_t stream) {
    const AttendPlan own = plan_own(cache, packed.requests, rows, q_heads);
    uint8_t *at = static_cast<uint8_t *>(workspace) + kAttendCounterBytes;
    AttendArgs a{};
    a.q = q, a.row_stride = row_stride, a.head_stride = head_stride, a.out = out, a.ld_out = ld_out;
    a.q_heads = (int)q_heads, a.shared = (int)shared;
    a.wide = reinterpret_cast<uintptr_t>(q) % 16 == 0 && row_stride % 8 == 0 && head_stride % 8 == 0;
    a.wide_out = reinterpret_cast<uintptr_t>(out) % 8 == 0 && ld_out % 4 == 0;
    a.by_blocks = divisor((int)(cache.page_tokens / kBlock));
    a.factor = scale * 1.4426950408889634f;
    a.pieces = reinterpret_cast<Pieces *>(at);
    a.slots = reinterpret_cast<float *>(at + (shared > 0 ? 2 : 1) * pieces_bytes(rows, q_heads));
    a.tile = own.tile, a.partial = shared > 0, a.first_slots = own.first_slots(a.partial);
    const CacheView cv = view_of(cache);
    const PackedView pv = view_of(packed, rows);
    AttendArgs b = a;
    AttendPlan prefix = own;
    if (shared > 0) {
        prefix = plan_prefix(cache, rows, q_heads);
        b.tile = prefix.tile, b.first_slots = prefix.first_slots(true), b.prefix = 1;
        b.pieces = a.pieces + rows * q_heads;
        b.slots = a.slots + own.slot_rows(true) * (cache.dim + 2);
    }
    auto run = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        if (shared > 0) launch_part<D>(prefix, b, cv, pv, stream);
        launch_part<D>(own, a, cv, pv, stream);
        if (rows * q_heads <= kJoinApart)  // a workgroup each, so that they spread over the CUs
            join_kernel<D, 64><<<(unsigned)(rows * q_heads), 64, 0, stream>>>(a, b, cv, pv);
        else
            join_kernel<D, 16><<<long_grid((rows * q_heads + 15) / 16), 256, 0, stream>>>(a, b, cv, pv);
    };
    if (cache.dim == 256) run(std::integral_constant<int, 256>{});
    else if (cache.dim == 128) run(std::integral_constant<int, 128>{});
    else run(std::integral_constant<int, 64>{});
    return hipGetLastError();
}

}  // namespace splosh
