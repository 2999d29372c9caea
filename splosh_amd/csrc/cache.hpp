// cache.hpp -- the 8-bit paged cache and the rows of a packed step, as the kernels see them.
#pragma once

#include <type_traits>

#include "common.hpp"
#include "launch.hpp"

namespace splosh {

constexpr int kBlock = 32;  // tokens of a record
constexpr float kLeastScale = 7.888609052210118e-31f;  // 2^-100

// A launch has at most 2^32 threads a dimension: this many workgroups of 256 go along x, and more of them in rows of so many along y.
constexpr int kGridLog = 22;
inline dim3 long_grid(int64_t workgroups) {
    const int64_t row = (int64_t)1 << kGridLog;
    return workgroups <= row ? dim3((unsigned)workgroups) : dim3((unsigned)row, (unsigned)((workgroups + row - 1) / row));
}
__device__ __forceinline__ int64_t long_block() { return (int64_t)blockIdx.y << kGridLog | blockIdx.x; }

// A record: codes of 32 keys, of 32 values, their scales; a code is kept as the byte code + 128, which takes one instruction less to
// widen than a signed one. Rows of codes are whole vectors, so that a token is written
// and read back in runs of `dim` bytes, and a matrix instruction's operand is a run of a row (keys: 16 bytes
// of dimensions a lane) or the same run of eight rows (values), transposed in the registers while it is widened to fp16.
constexpr int record_bytes(int dim) { return 2 * kBlock * dim + 2 * kBlock * 4; }

struct CacheView {
    uint8_t *data;
    int64_t page_stride;
    int pages, page_tokens, page_blocks, heads;
};
struct PackedView {
    const int32_t *starts, *lengths, *table;
    int64_t table_stride;
    int table_pages, requests, rows;
};

inline CacheView view_of(const splosh_cache &c) {
    return {c.data, c.page_stride, (int)c.pages, (int)c.page_tokens, (int)(c.page_tokens / kBlock), (int)c.heads};
}
inline PackedView view_of(const splosh_packed &p, int64_t rows) {
    return {p.starts, p.lengths, p.table, p.table_stride, (int)p.table_pages, (int)p.requests, (int)rows};
}

// The request that packed row `row` belongs to, -1: none. All lanes of a wave call it with the same row: 64 starts at a time.
__device__ __forceinline__ int request_of(const int32_t *starts, int requests, int row) {
    const int lane = threadIdx.x & 63;
    int count = 0;  // starts not past the row
    for (int base = 0; base <= requests; base += 64) {
        const int i = base + lane;
        const int n = __popcll(__ballot(i <= requests && starts[i] <= row));
        count += n;
        if (n < 64) break;
    }
    const int r = count - 1;
    return r < requests ? r : -1;
}

// The position of packed row `row`, one of request `request`'s: starts past the step's rows count as those, as everywhere (and those below 0: this one's
// end is past the row), and a position below 32 bits is as good as their least.
__host__ __device__ __forceinline__ int position_in(const PackedView &p, int request, int row) {
    const int end = p.starts[request + 1] < p.rows ? p.starts[request + 1] : p.rows;
    const int64_t position = (int64_t)p.lengths[request] - end + row;
    return position < INT32_MIN ? INT32_MIN : (int)position;
}

// Where token `position` of request `request` lies: its page's id and its place there; false where it has none.
__host__ __device__ __forceinline__ bool place_of(const CacheView &c, const PackedView &p, int request, int position, int &page, int &at) {
    if (request < 0 || position < 0) return false;
    const int column = position / c.page_tokens;
    if (column >= p.table_pages) return false;
    page = p.table[request * p.table_stride + column];
    at = position - column * c.page_tokens;
    return page >= 0 && page < c.pages;
}

template <int D>
__device__ __forceinline__ uint8_t *record_of(const CacheView &c, int page, int head, int block) {
    return c.data + page * c.page_stride + ((int64_t)head * c.page_blocks + block) * record_bytes(D);
}

}  // namespace splosh
