// heads.hip -- the heads of a packed step before its attention: norms of queries and keys over each head and their
// rotation by position in one pass, keys and values into the 8-bit cache, and the cache read back.
//
// All of it is bound by memory or, for few rows, by the launch. A workgroup takes one row: its first threads compute
// the row's cosines and sines, once for all heads, and then each wave takes four heads of one projection at a time,
// sixteen lanes a head with dim / 16 consecutive elements each: what a vector costs once (a root, a division) is
// shared by four, and its sums take four steps within a row of lanes. 2048 rows of 24 + 4 heads of 256 in fp32, 88 MB,
// take 17.4 us (5.0 TB/s, the rate of a large copy); with a wave a head, four elements a lane, it was 23 us, bound by
// instructions, and 2000 rows of 32 queries, 8 keys and 8 values of 128 into the cache were 29 us instead of 14. The two
// halves of a rotated pair meet through the wave's own LDS.
#include "cache.hpp"

namespace splosh {

constexpr int kHeadThreads = 256, kHeadWaves = kHeadThreads / 64;
constexpr int kVectors = 4, kLanes = 64 / kVectors;  // heads of a wave, and lanes of a head

struct HeadPart {
    const void *x;
    int64_t row_stride, head_stride;
    const uint16_t *weight;
    uint16_t *out;
    int64_t ld_out;
    int heads;
    int16_t rotated;  // whether it is turned
    int16_t kept;     // 0: out; 1, 2: keys, values into the cache
    int16_t wide_x, wide_weight, wide_out;  // whether their runs of eight (weight, out: four) bytes and more are aligned to them
};
struct HeadArgs {
    int first[SPLOSH_MAX_GROUP + 1];  // each part's first unit of a row, four heads of one part; and their count
    int parts, chunk;                 // units a workgroup
    int half;
    float eps;
    const int32_t *positions;
    const float *frequencies;
    HeadPart part[SPLOSH_MAX_GROUP];
};

// The sum, and the largest, over the sixteen lanes of a head, in each of them.
template <typename F>
__device__ __forceinline__ float head_fold(float v, F fold) {
    auto step = [&](auto ctrl) {
        const int other = __builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), decltype(ctrl)::value, 0xf, 0xf, false);
        v = fold(v, __uint_as_float((uint32_t)other));
    };
    step(std::integral_constant<int, 0xb1>{});   // lanes 1 0 3 2
    step(std::integral_constant<int, 0x4e>{});   // 2 3 0 1
    step(std::integral_constant<int, 0x141>{});  // eight lanes turned round
    step(std::integral_constant<int, 0x140>{});  // sixteen
    return v;
}
__device__ __forceinline__ float head_sum(float v) {
    return head_fold(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float head_max(float v) {
    return head_fold(v, [](float a, float b) { return __builtin_fmaxf(a, b); });
}

// E elements from `at` on as fp32; wide: in runs of 16 bytes (bf16 of 64 dimensions: 8).
template <int E>
__device__ __forceinline__ void load_elements(const float *at, bool wide, float (&v)[E]) {
    if (wide) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(at + e);
#pragma unroll
            for (int f = 0; f < 4; ++f) v[e + f] = x[f];
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = at[e];
    }
}
template <int E>
__device__ __forceinline__ void load_elements(const uint16_t *at, bool wide, float (&v)[E]) {
    uint32_t pair[E / 2];
    if (wide) {
        constexpr int RUN = E < 8 ? 2 : 4;
        typedef uint32_t Run __attribute__((ext_vector_type(RUN)));
#pragma unroll
        for (int e = 0; e < E / 2; e += RUN) {
            const Run x = *reinterpret_cast<const Run *>(at + 2 * e);
#pragma unroll
            for (int f = 0; f < RUN; ++f) pair[e + f] = x[f];
        }
    } else {
#pragma unroll
        for (int e = 0; e < E / 2; ++e) pair[e] = at[2 * e] | (uint32_t)at[2 * e + 1] << 16;
    }
#pragma unroll
    for (int e = 0; e < E / 2; ++e) v[2 * e] = bf16_bits_to_f32(pair[e]), v[2 * e + 1] = __uint_as_float(pair[e] & 0xffff0000u);
}

template <int E>
__device__ __forceinline__ void store_bf16(uint16_t *at, bool wide, const float (&v)[E]) {
    uint32_t pair[E / 2];
#pragma unroll
    for (int e = 0; e < E / 2; ++e) pair[e] = f32x2_to_bf16x2(v[2 * e], v[2 * e + 1]);
    if (wide) {
        constexpr int RUN = E < 8 ? 2 : 4;
        typedef uint32_t Run __attribute__((ext_vector_type(RUN)));
#pragma unroll
        for (int e = 0; e < E / 2; e += RUN) {
            Run x;
#pragma unroll
            for (int f = 0; f < RUN; ++f) x[f] = pair[e + f];
            *reinterpret_cast<Run *>(at + 2 * e) = x;
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) at[e] = (uint16_t)(pair[e / 2] >> 16 * (e & 1));
    }
}

// The bytes of a vector's codes, E a lane, and its scale. 127 x has 15 bits for a bf16 x, and a quotient of 15 bits by 8 that is not a
// half of an odd number is further from one than its rounding: with the quotient rounded once, a bf16 vector's codes are exact.
// It is: the product with the rounded reciprocal, corrected by what an fma leaves over. Vectors near the upper end of
// fp32 are moved by a power of two before it.
template <int E>
__device__ __forceinline__ void codes_of(const float (&v)[E], float &scale, uint32_t (&codes)[E / 4]) {
    float most = 0.0f, bad = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        most = __builtin_fmaxf(most, __builtin_fabsf(v[e]));
        bad = __builtin_fabsf(v[e]) < __builtin_inff() ? bad : 1.0f;
    }
    most = head_max(most);
    bad = head_max(bad);
    scale = most / 127.0f;
    const bool small = scale < kLeastScale;
    const float move = most > 0x1p100f ? 0x1p-64f : 1.0f;
    const float by = small ? kLeastScale : most * move, times = bad > 0.0f ? 0.0f : small ? 1.0f : 127.0f * move, r = 1.0f / by;
    scale = bad > 0.0f ? __builtin_nanf("") : small ? kLeastScale : scale;
#pragma unroll
    for (int e = 0; e < E; e += 4) {
        codes[e / 4] = 0;
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const float x = bad > 0.0f ? 0.0f : v[e + f] * times, q = x * r, c = __builtin_rintf(__builtin_fmaf(__builtin_fmaf(-q, by, x), r, q));
            codes[e / 4] |= (uint32_t)((int)c + 128) << 8 * f;
        }
    }
}

template <typename T, int D, bool kCache>
__global__ __launch_bounds__(kHeadThreads) void heads_kernel(HeadArgs a, CacheView cache, PackedView packed) {
    constexpr int E = D / kLanes, PITCH = D + 4;
    __shared__ __align__(16) float turn_cos[D / 2 + 4], turn_sin[D / 2 + 4];
    __shared__ __align__(16) float vectors[kHeadWaves][kVectors][PITCH];
    const int row = blockIdx.x, tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int which = lane / kLanes, first = lane % kLanes * E;  // the lane's head of the wave's four, and its elements
    const int units = a.first[a.parts], end = min(units, (int)(blockIdx.y + 1) * a.chunk);
    int unit = blockIdx.y * a.chunk + wave;
    float v[E];
    int part_at = 0, head = 0;
    bool here = false;
    auto load = [&]() {  // (a wave's heads are of one part)
        while (part_at + 1 < a.parts && unit >= a.first[part_at + 1]) ++part_at;
        const HeadPart &part = a.part[part_at];
        head = (unit - a.first[part_at]) * kVectors + which;
        here = head < part.heads;
        if (here) load_elements<E>((const T *)part.x + row * part.row_stride + head * part.head_stride + first, part.wide_x, v);
        else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = 0.0f;
        }
    };
    if (unit < end) load();  // (on its way while the row's place is looked up)
    int position, page = 0, at = 0;
    bool placed = false;
    if (kCache) {
        const int r = request_of(packed.starts, packed.requests, row);
        if (r < 0) return;  // (the same for the whole workgroup)
        position = position_in(packed, r, row);
        placed = place_of(cache, packed, r, position, page, at);
    } else {
        position = a.positions ? a.positions[row] : 0;
    }
    if (tid < a.half) {
        // In turns, so that only a fraction of one is left of a far position's angle: 64 bits up to there.
        const double turns = (double)position * (double)a.frequencies[tid] * 0.15915494309189535;
        sincospif(2.0f * (float)(turns - __builtin_rint(turns)), &turn_sin[tid], &turn_cos[tid]);
    }
    __syncthreads();
    // Whether a pair's two elements are at the same place of two lanes.
    const bool even = a.half % E == 0;
    float *const mine = vectors[wave][which];
    for (; unit < end; ) {
        const HeadPart &part = a.part[part_at];
        if (part.weight) {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) sum += v[e] * v[e];
            const float inv = 1.0f / sqrtf(head_sum(sum) * (1.0f / D) + a.eps);
            float w[E];
            load_elements<E>(part.weight + first, part.wide_weight, w);
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = v[e] * inv * w[e];
        }
        if (part.rotated) {
            if (first < 2 * a.half) {
#pragma unroll
                for (int e = 0; e < E; e += 4) *reinterpret_cast<f32x4 *>(mine + first + e) = f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]};
            }
            // (What the wave's lanes wrote for each other: nothing of it is another wave's.)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (even) {
                if (first < 2 * a.half) {
                    const bool low = first < a.half;
                    const int other = low ? first + a.half : first - a.half, pair = low ? first : other;
#pragma unroll
                    for (int e = 0; e < E; e += 4) {
                        const f32x4 x = *reinterpret_cast<const f32x4 *>(mine + other + e), c = *reinterpret_cast<const f32x4 *>(turn_cos + pair + e),
                                    s = *reinterpret_cast<const f32x4 *>(turn_sin + pair + e);
#pragma unroll
                        for (int f = 0; f < 4; ++f) v[e + f] = v[e + f] * c[f] + x[f] * (low ? -s[f] : s[f]);
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int i = first + e;
                    if (i < a.half) v[e] = v[e] * turn_cos[i] - mine[i + a.half] * turn_sin[i];
                    else if (i < 2 * a.half) v[e] = v[e] * turn_cos[i - a.half] + mine[i - a.half] * turn_sin[i - a.half];
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        if (!kCache || !part.kept) {
            if (here) store_bf16<E>(part.out + row * part.ld_out + (int64_t)head * D + first, part.wide_out, v);
        } else if (placed) {
            float scale;
            uint32_t codes[E / 4];
            codes_of<E>(v, scale, codes);
            if (here) {
                uint8_t *record = record_of<D>(cache, page, head, at / kBlock);
                const int token = at % kBlock, values = part.kept - 1;
                typedef uint32_t Run __attribute__((ext_vector_type(E / 4 > 1 ? E / 4 : 2)));
                uint8_t *to = record + (values * kBlock + token) * D + first;
                if constexpr (E == 4) {
                    *reinterpret_cast<uint32_t *>(to) = codes[0];
                } else {
                    Run x;
#pragma unroll
                    for (int e = 0; e < E / 4; ++e) x[e] = codes[e];
                    *reinterpret_cast<Run *>(to) = x;
                }
                if (first == 0) reinterpret_cast<float *>(record + 2 * kBlock * D)[values * kBlock + token] = scale;
            }
        }
        unit += kHeadWaves;
        if (unit < end) load();
    }
}

struct ReadArgs {
    uint16_t *out[2];  // of keys, of values
    int64_t ld[2];
    int wide[2];
};

// A wave four heads of a row, keys and values: one way through the table for both, and both under way at once.
template <int D>
__global__ __launch_bounds__(kHeadThreads) void cache_read_kernel(ReadArgs a, CacheView cache, PackedView packed) {
    constexpr int E = D / kLanes;
    const int units = (cache.heads + kVectors - 1) / kVectors;
    const int64_t item = long_block() * kHeadWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= (int64_t)packed.rows * units) return;
    const int row = (int)(item / units), lane = threadIdx.x & 63;
    const int head = (int)(item % units) * kVectors + lane / kLanes, first = lane % kLanes * E;
    const int r = request_of(packed.starts, packed.requests, row);
    if (r < 0) return;
    int page = 0, at = 0;
    const bool placed = place_of(cache, packed, r, position_in(packed, r, row), page, at);
    if (head >= cache.heads) return;
    struct alignas(E) Codes {
        uint8_t of[E];
    } codes[2] = {};
    float scale[2] = {};
    const uint8_t *record = record_of<D>(cache, placed ? page : 0, head, placed ? at / kBlock : 0);
    const int token = placed ? at % kBlock : 0;
#pragma unroll
    for (int values = 0; values < 2; ++values) {
        if (!a.out[values]) continue;
        codes[values] = *reinterpret_cast<const Codes *>(record + (values * kBlock + token) * D + first);
        scale[values] = reinterpret_cast<const float *>(record + 2 * kBlock * D)[values * kBlock + token];
    }
#pragma unroll
    for (int values = 0; values < 2; ++values) {
        if (!a.out[values]) continue;
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = placed ? (float)(codes[values].of[e] - 128) * scale[values] : 0.0f;
        store_bf16<E>(a.out[values] + row * a.ld[values] + (int64_t)head * D + first, a.wide[values], v);
    }
}

static bool fits(const void *p, int64_t stride, int64_t size, int64_t bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride * size % bytes == 0;
}
// The runs that a lane's elements are moved in (fp32: 16 bytes; bf16: 16, of 64 dimensions 8).
static int64_t run_bytes(int64_t dim, int64_t size) { return dim / kLanes * size < 16 ? dim / kLanes * size : 16; }

// Units a workgroup takes of a row: all of them where there are rows for every CU, four (one a wave) where there are few.
static int chunk_of(int64_t rows, int units) {
    int chunk = units;
    while (chunk > kHeadWaves && rows * ((units + chunk - 1) / chunk) < 1024) chunk = (chunk + 1) / 2;
    return chunk < kHeadWaves ? kHeadWaves : chunk;
}

template <bool kCache>
static hipError_t launch_heads(HeadArgs &a, int dtype, int64_t rows, int64_t dim, const CacheView &cache,
                               const PackedView &packed, hipStream_t stream) {
    const int64_t size = dtype == SPLOSH_F32 ? 4 : 2;
    for (int i = 0; i < a.parts; ++i) {
        HeadPart &p = a.part[i];
        p.wide_x = fits(p.x, p.row_stride, size, run_bytes(dim, size)) && fits(p.x, p.head_stride, size, run_bytes(dim, size));
        p.wide_weight = fits(p.weight, 0, 2, run_bytes(dim, 2));
        p.wide_out = fits(p.out, p.ld_out, 2, run_bytes(dim, 2));
    }
    const int units = a.first[a.parts];
    a.chunk = chunk_of(rows, units);
    const dim3 grid((unsigned)rows, (unsigned)((units + a.chunk - 1) / a.chunk));
    auto go = [&](auto kernel) { kernel<<<grid, kHeadThreads, 0, stream>>>(a, cache, packed); };
    if (dtype == SPLOSH_F32) {
        if (dim == 256) go(heads_kernel<float, 256, kCache>);
        else if (dim == 128) go(heads_kernel<float, 128, kCache>);
        else go(heads_kernel<float, 64, kCache>);
    } else {
        if (dim == 256) go(heads_kernel<uint16_t, 256, kCache>);
        else if (dim == 128) go(heads_kernel<uint16_t, 128, kCache>);
        else go(heads_kernel<uint16_t, 64, kCache>);
    }
    return hipGetLastError();
}

static void add_part(HeadArgs &a, const splosh_heads &h, bool rotated, int kept) {
    a.part[a.parts] = {h.x, h.row_stride, h.head_stride, h.weight, h.out, h.ld_out, (int)h.heads, rotated, (int16_t)kept, 0, 0, 0};
    a.first[a.parts + 1] = a.first[a.parts] + (int)((h.heads + kVectors - 1) / kVectors);
    ++a.parts;
}

hipError_t launch_rotate_heads(const splosh_heads *parts, int count, int dtype, int64_t rows, int64_t dim,
                               const int32_t *positions, const float *frequencies, int64_t rotary, float eps,
                               hipStream_t stream) {
    HeadArgs a{};
    a.positions = positions, a.frequencies = frequencies, a.half = (int)(rotary / 2), a.eps = eps;
    for (int i = 0; i < count; ++i) add_part(a, parts[i], rotary > 0, 0);
    return launch_heads<false>(a, dtype, rows, dim, CacheView{}, PackedView{}, stream);
}

hipError_t launch_cache_write(const splosh_cache &cache, const splosh_packed &packed, const splosh_heads &k,
                              const splosh_heads &v, const splosh_heads *q, int dtype, int64_t rows,
                              const float *frequencies, int64_t rotary, float eps, hipStream_t stream) {
    HeadArgs a{};
    a.frequencies = frequencies, a.half = (int)(rotary / 2), a.eps = eps;
    add_part(a, k, rotary > 0, 1);
    add_part(a, v, false, 2);
    if (q) add_part(a, *q, rotary > 0, 0);
    return launch_heads<true>(a, dtype, rows, cache.dim, view_of(cache), view_of(packed, rows), stream);
}

hipError_t launch_cache_read(const splosh_cache &cache, const splosh_packed &packed, int64_t rows, uint16_t *k,
                             int64_t ldk, uint16_t *v, int64_t ldv, hipStream_t stream) {
    const int64_t bytes = run_bytes(cache.dim, 2);
    const ReadArgs a{{k, v}, {ldk, ldv}, {fits(k, ldk, 2, bytes), fits(v, ldv, 2, bytes)}};
    auto go = [&](auto kernel) {
        const int64_t items = rows * ((cache.heads + kVectors - 1) / kVectors);
        kernel<<<long_grid((items + kHeadWaves - 1) / kHeadWaves), kHeadThreads, 0, stream>>>(a, view_of(cache), view_of(packed, rows));
    };
    if (cache.dim == 256) go(cache_read_kernel<256>);
    else if (cache.dim == 128) go(cache_read_kernel<128>);
    else go(cache_read_kernel<64>);
    return hipGetLastError();
}

}  // namespace splosh
