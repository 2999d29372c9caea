// attend_plan.hpp -- how a launch of the attention kernels shares a step's work out, as functions of the step's shape that the
// kernels and the host both compile.
#pragma once

#include "cache.hpp"

namespace splosh {

// x / d for 0 <= x < 2^31 as a product: m = ceil(2^(31 + L) / d) for the L with 2^(L - 1) < d <= 2^L is off by e < d / 2^(31 + L)
// relative, which x e < 2^(31 + L) keeps below the next whole number. (m = 0: d is 1.)
struct Divisor {
    uint32_t m;
    int shift;
    __host__ __device__ __forceinline__ int of(int x) const {
        return m == 0 ? x : (int)((uint32_t)(((uint64_t)(uint32_t)x * m) >> 32) >> shift);
    }
};
inline Divisor divisor(int d) {
    if (d <= 1) return {0, 0};
    int log = 1;
    while (((int64_t)1 << log) < d) ++log;
    return {(uint32_t)((((uint64_t)1 << (31 + log)) + d - 1) / d), log - 1};
}

// A tile is `rows` of the (row, query head) vectors of one request that share a key/value head, side by side: vector x
// is row x / group of the request and head x % group of the group. A segment is a tile with all its keys, counted in units of
// `keys` keys, after `extra` units that stand for what a segment costs beside its keys; the segments lie one behind the other (requests,
// then key/value heads, then tiles) and workgroup w of `workgroups` takes the units from total w / workgroups on. So every workgroup has the
// same share, whatever the lengths, and what a segment is cut into follows from the shape alone.
struct TileShape {
    int rows, keys, extra, group, heads, workgroups;
    Divisor by_rows, by_keys, by_group;
};
inline TileShape tile_shape(int rows, int keys, int extra, int group, int heads, int workgroups) {
    return {rows, keys, extra, group, heads, workgroups, divisor(rows), divisor(keys), divisor(group)};
}

// One request's part of a launch: its n rows from packed row `begin` on, the first at position `first`, and the keys
// [from, to) of those that its rows see. A prefix that all requests share is one such part, of all rows.
struct Span {
    int begin, n, first, from, to;
};

__host__ __device__ __forceinline__ Span span_of(const PackedView &p, int page_tokens, int shared, int start, int end, int length) {
    Span s;
    s.begin = start < 0 ? 0 : start;
    s.n = (end > p.rows ? p.rows : end) - s.begin;
    if (s.n < 0) s.n = 0;
    // (Lengths past either end of what a table can hold are as good as these: nothing is seen, or everything.)
    const int least = -(1 << 22), most = (1 << 30) + (1 << 23);
    s.first = (length < least ? least : length > most ? most : length) - s.n;
    s.from = shared;
    s.to = p.table_pages * page_tokens;
    return s;
}
__host__ __device__ __forceinline__ Span own_span(const PackedView &p, int page_tokens, int shared, int request) {
    return span_of(p, page_tokens, shared, p.starts[request], p.starts[request + 1], p.lengths[request]);
}
__host__ __device__ __forceinline__ Span prefix_span(const PackedView &p, int shared) {
    const int end = p.starts[p.requests];
    return {0, end < 0 ? 0 : end > p.rows ? p.rows : end, shared, 0, shared};
}

// Whether a request ends where it begins or later, with starts past the step's rows as those. Where all do, no row is two requests', and the units of all of them are what the host has
// found to fit into 32 bits; where one does not, they can be many times that, and with sums that wrap two requests can have the same unit.
__host__ __device__ __forceinline__ bool ascends(const PackedView &p, int request) {
    const int begin = p.starts[request], end = p.starts[request + 1];
    return begin <= end || begin <= 0 || end >= p.rows;
}

__host__ __device__ __forceinline__ int tiles_of(const Span &s, const TileShape &t) { return t.by_rows.of(s.n * t.group + t.rows - 1); }

// The end of the keys that tile i of a span sees.
__host__ __device__ __forceinline__ int tile_end(const Span &s, const TileShape &t, int i) {
    const int vectors = s.n * t.group, last = ((i + 1) * t.rows < vectors ? (i + 1) * t.rows : vectors) - 1;
    const int end = s.first + t.by_group.of(last) + 1;
    return end < s.to ? end : s.to;
}
// Its units: one of keys at least, so that rows that see nothing are written too.
__host__ __device__ __forceinline__ int tile_units(const Span &s, const TileShape &t, int i) {
    const int keys = tile_end(s, t, i) - s.from;
    return t.extra + (keys <= t.keys ? 1 : t.by_keys.of(keys - 1) + 1);
}
// The units of the tiles before tile i, for one key/value head.
__host__ __device__ __forceinline__ int units_before(const Span &s, const TileShape &t, int i) {
    int units = 0;
    for (int j = 0; j < i; ++j) units += tile_units(s, t, j);
    return units;
}

// The workgroups that get any of `total` units: one a unit where there are fewer units. Their pieces of a segment are consecutive.
__host__ __device__ __forceinline__ int sharers_of(int total, int workgroups) { return total < workgroups ? total : workgroups; }
// Of these, workgroup w's first unit, and the workgroup that unit u belongs to. (Neither's products are near 2^53, and no
// quotient that is not whole is nearer to a whole number than 1 / total.)
__host__ __device__ __forceinline__ int first_unit(int total, int workgroups, int w) {
    return total / workgroups * w + total % workgroups * w / workgroups;
}
__host__ __device__ __forceinline__ int owner_of(int total, int workgroups, int u) {
    return (int)(((double)(u + 1) * workgroups - 1.0) / total);
}

// What workgroup w of `sharers` takes of a segment from unit `offset` on, which is unit `unit` of the launch's `total`.
struct Cut {
    int take;                 // units
    bool any;                 // whether it has keys, or all there is of a segment without: who has nothing but units before the keys leaves the segment to the next
    int first_block, blocks;  // of 32 keys, from the span's first on
    int slot, count;          // where partial results go; of the segment's first piece, how many workgroups have one
    bool direct;              // the whole segment, and nothing to join it with
};
__host__ __device__ __forceinline__ Cut cut_of(const Span &s, const TileShape &t, int i, int segment, int offset, int unit, int end, int w, int sharers, int total,
                                               bool partial, int64_t first_slots) {
    const int units = tile_units(s, t, i), keys = tile_end(s, t, i) - s.from;
    const int blocks = keys > 0 ? (keys + kBlock - 1) / kBlock : 0, per = t.keys / kBlock;
    Cut c;
    c.take = units - offset < end - unit ? units - offset : end - unit;
    c.any = offset + c.take > t.extra;
    const bool first = offset <= t.extra, whole = offset + c.take == units;
    const int from = offset > t.extra ? (offset - t.extra) * per : 0, to = (offset + c.take - t.extra) * per < blocks ? (offset + c.take - t.extra) * per : blocks;
    c.first_block = from, c.blocks = to > from ? to - from : 0;
    c.slot = !first ? (int)first_slots + w : partial ? segment : w;
    c.count = !first ? 0 : whole ? 1 : owner_of(total, sharers, unit + units - offset - 1) - w + 1;
    c.direct = !partial && first && whole;
    return c;
}

// The most segments that a step of so many requests and rows can have.
__host__ __device__ __forceinline__ int64_t most_segments(int64_t requests, int64_t rows, int64_t q_heads, int64_t heads, int tile_rows) {
    return heads * ((requests < rows ? requests : rows) + rows * (q_heads / heads) / tile_rows);
}

}  // namespace splosh
