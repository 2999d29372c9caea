// heads.hip -- the heads of a packed step before its attention: norms of queries and keys over each head and their
// rotation by position in one pass, keys and values into the 8-bit cache, and the cache read back.
//
// All of it is bound by memory or, for few rows, by the launch. A workgroup takes one row: its first threads compute
// the row's cosines and sines, once for all heads, and then each wave takes four (row, head) vectors at a time, dim / 64
// consecutive elements a lane. The two halves of a rotated pair meet through the wave's own LDS.
#include "cache.hpp"

namespace splosh {

constexpr int kHeadThreads = 256, kHeadWaves = kHeadThreads / 64;

struct HeadPart {
    const void *x;
    int64_t row_stride, head_stride;
    const uint16_t *weight;
    uint16_t *out;
    int64_t ld_out;
    int first;    // its first unit; a row's units are the heads of all parts
    int rotated;  // whether it is turned
    int kept;     // 0: out; 1, 2: keys, values into the cache
    int wide;     // whether vectors of dim / 64 elements may be loaded and stored at once
};
struct HeadArgs {
    HeadPart part[SPLOSH_MAX_GROUP];
    int parts, units, chunk;  // units a workgroup
    const int32_t *positions;
    const float *frequencies;
    int half;
    float eps;
};

template <int E, typename T>
__device__ __forceinline__ void load_elements(const T *at, int wide, float (&v)[E]) {
    T raw[E];
    if (E > 1 && wide) {
        struct alignas(E * sizeof(T)) Vector {
            T of[E];
        };
        const Vector w = *reinterpret_cast<const Vector *>(at);
#pragma unroll
        for (int e = 0; e < E; ++e) raw[e] = w.of[e];
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) raw[e] = at[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if constexpr (sizeof(T) == 2) v[e] = bf16_bits_to_f32((uint32_t)raw[e]);
        else v[e] = (float)raw[e];
    }
}

template <int E>
__device__ __forceinline__ void store_bf16(uint16_t *at, int wide, const float (&v)[E]) {
    if constexpr (E == 1) {
        at[0] = f32_to_bf16(v[0]);
    } else {
        uint32_t pair[E / 2];
#pragma unroll
        for (int e = 0; e < E / 2; ++e) pair[e] = f32x2_to_bf16x2(v[2 * e], v[2 * e + 1]);
        if (wide) {
            typedef uint32_t vec __attribute__((ext_vector_type(E / 2)));
            if constexpr (E == 4) *reinterpret_cast<vec *>(at) = vec{pair[0], pair[1]};
            else *reinterpret_cast<uint32_t *>(at) = pair[0];
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) at[e] = (uint16_t)(pair[e / 2] >> 16 * (e & 1));
        }
    }
}

// The codes of a vector whose elements the wave holds, E a lane, and its scale. x 127 and the division are each rounded
// once, so that a bf16 vector's codes are exact: 127 x has 15 bits, and a quotient of 15 bits by 8 that is not a
// half of an odd number is further from one than its rounding. Vectors near the ends of fp32 are moved by a power of two before it.
template <int E>
__device__ __forceinline__ uint32_t codes_of(const float (&v)[E], float &scale) {
    float most = 0.0f;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        most = __builtin_fmaxf(most, __builtin_fabsf(v[e]));
        bad |= !(__builtin_fabsf(v[e]) < __builtin_inff());
    }
    most = wave_max(most);  // (the same in every lane)
    scale = most / 127.0f;
    const bool small = scale < kLeastScale;
    if (small) scale = kLeastScale;
    bad = __any(bad);
    if (bad) scale = __builtin_nanf("");
    const float move = most > 0x1p100f ? 0x1p-64f : 1.0f;
    const float by = small ? kLeastScale : most * move, times = small ? 1.0f : 127.0f * move;
    uint32_t codes = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = bad ? 0 : (int)__builtin_rintf(v[e] * times / by);
        codes |= (uint32_t)(c + 128) << 8 * e;
    }
    return codes;
}

template <typename T, int D, bool kCache>
__global__ __launch_bounds__(kHeadThreads) void heads_kernel(HeadArgs a, CacheView cache, PackedView packed) {
    constexpr int E = D / 64, BATCH = 4;  // vectors that a wave has in hand at a time
    __shared__ float2 turn[D / 2];
    __shared__ float vector[kHeadWaves][BATCH][D];
    const int row = blockIdx.x, tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int end = min(a.units, (int)(blockIdx.y + 1) * a.chunk);
    int unit = blockIdx.y * a.chunk + wave;
    auto part_of = [&](int u) {
        int which = 0;
        while (which + 1 < a.parts && u >= a.part[which + 1].first) ++which;
        return which;
    };
    float v[BATCH][E];
    auto load = [&]() {
#pragma unroll
        for (int n = 0; n < BATCH; ++n) {
            const int u = unit + n * kHeadWaves;
            if (u >= end) break;
            const HeadPart &part = a.part[part_of(u)];
            load_elements<E>((const T *)part.x + row * part.row_stride + (u - part.first) * part.head_stride + lane * E, part.wide, v[n]);
        }
    };
    load();  // (on its way while the row's place is looked up)
    int position, page = 0, at = 0;
    bool placed = false;
    if (kCache) {
        const int r = request_of(packed.starts, packed.requests, row);
        if (r < 0) return;  // (the same for the whole workgroup)
        position = packed.lengths[r] - packed.starts[r + 1] + row;
        placed = place_of(cache, packed, r, position, page, at);
    } else {
        position = a.positions ? a.positions[row] : 0;
    }
    if (tid < a.half) {
        // In turns, so that only a fraction of one is left of a far position's angle: 64 bits up to there.
        const double turns = (double)position * (double)a.frequencies[tid] * 0.15915494309189535;
        float s, c;
        sincospif(2.0f * (float)(turns - __builtin_rint(turns)), &s, &c);
        turn[tid] = make_float2(c, s);
    }
    __syncthreads();
    while (true) {
#pragma unroll
        for (int n = 0; n < BATCH; ++n) {
            const int u = unit + n * kHeadWaves;
            if (u >= end) break;
            const HeadPart &part = a.part[part_of(u)];
            if (part.weight) {
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) sum += v[n][e] * v[n][e];
                const float inv = 1.0f / sqrtf(wave_sum(sum) * (1.0f / D) + a.eps);
                float w[E];
                load_elements<E>(part.weight + lane * E, 0, w);
#pragma unroll
                for (int e = 0; e < E; ++e) v[n][e] = v[n][e] * inv * w[e];
            }
            if (part.rotated) {
#pragma unroll
                for (int e = 0; e < E; ++e) vector[wave][n][lane * E + e] = v[n][e];
            }
        }
        // (What the wave's lanes wrote for each other: nothing of it is another wave's.)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int n = 0; n < BATCH; ++n) {
            const int u = unit + n * kHeadWaves;
            if (u >= end) break;
            const HeadPart &part = a.part[part_of(u)];
            const int head = u - part.first;
            if (part.rotated) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int i = lane * E + e;
                    if (i < a.half) {
                        const float2 t = turn[i];
                        v[n][e] = v[n][e] * t.x - vector[wave][n][i + a.half] * t.y;
                    } else if (i < 2 * a.half) {
                        const float2 t = turn[i - a.half];
                        v[n][e] = v[n][e] * t.x + vector[wave][n][i - a.half] * t.y;
                    }
                }
            }
            if (!kCache || !part.kept) {
                store_bf16<E>(part.out + row * part.ld_out + head * D + lane * E, part.wide, v[n]);
                continue;
            }
            if (!placed) continue;
            float scale;
            const uint32_t codes = codes_of<E>(v[n], scale);
            uint8_t *record = record_of<D>(cache, page, head, at / kBlock);
            const int token = at % kBlock, values = part.kept - 1;
            uint8_t *to = record + (values * kBlock + token) * D + lane * E;
            if constexpr (E == 4) *reinterpret_cast<uint32_t *>(to) = codes;
            else if constexpr (E == 2) *reinterpret_cast<uint16_t *>(to) = (uint16_t)codes;
            else *to = (uint8_t)codes;
            if (lane == 0) reinterpret_cast<float *>(record + 2 * kBlock * D)[values * kBlock + token] = scale;
        }
        unit += BATCH * kHeadWaves;
        if (unit >= end) return;
        load();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

struct ReadArgs {
    uint16_t *out[2];  // of keys, of values
    int64_t ld[2];
    int wide[2];
};

template <int D>
__global__ __launch_bounds__(kHeadThreads) void cache_read_kernel(ReadArgs a, CacheView cache, PackedView packed) {
    constexpr int E = D / 64;
    const int row = blockIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int r = request_of(packed.starts, packed.requests, row);
    if (r < 0) return;
    int page = 0, at = 0;
    const bool placed = place_of(cache, packed, r, packed.lengths[r] - packed.starts[r + 1] + row, page, at);
#pragma unroll 4
    for (int unit = wave; unit < 2 * cache.heads; unit += kHeadWaves) {
        const int values = unit & 1, head = unit >> 1;
        if (!a.out[values]) continue;
        float v[E] = {};
        if (placed) {
            const uint8_t *record = record_of<D>(cache, page, head, at / kBlock);
            const int token = at % kBlock;
            struct alignas(E) Codes {
                uint8_t of[E];
            };
            const Codes codes = *reinterpret_cast<const Codes *>(record + (values * kBlock + token) * D + lane * E);
            const float scale = reinterpret_cast<const float *>(record + 2 * kBlock * D)[values * kBlock + token];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = (float)(codes.of[e] - 128) * scale;
        }
        store_bf16<E>(a.out[values] + row * a.ld[values] + head * D + lane * E, a.wide[values], v);
    }
}

static bool fits(const void *p, int64_t stride, int64_t size, int64_t bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride * size % bytes == 0;
}

// Units a workgroup takes of a row: all of them where there are rows for every CU, four (one a wave) where there are few.
static int chunk_of(int64_t rows, int units) {
    int chunk = units;
    while (chunk > kHeadWaves && rows * ((units + chunk - 1) / chunk) < 1024) chunk = (chunk + 1) / 2;
    return chunk < kHeadWaves ? kHeadWaves : chunk;
}

template <bool kCache>
static hipError_t launch_heads(HeadArgs &a, int dtype, int64_t rows, int64_t dim, const CacheView &cache,
                               const PackedView &packed, hipStream_t stream) {
    const int64_t size = dtype == SPLOSH_F32 ? 4 : 2, elements = dim / 64;
    for (int i = 0; i < a.parts; ++i) {
        HeadPart &p = a.part[i];
        p.wide = fits(p.x, p.row_stride, size, elements * size) && fits(p.x, p.head_stride, size, elements * size) &&
                 (!p.out || fits(p.out, p.ld_out, 2, elements * 2));
    }
    a.chunk = chunk_of(rows, a.units);
    const dim3 grid((unsigned)rows, (unsigned)((a.units + a.chunk - 1) / a.chunk));
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
    a.part[a.parts++] = {h.x, h.row_stride, h.head_stride, h.weight, h.out, h.ld_out, a.units, rotated, kept, 0};
    a.units += (int)h.heads;
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
    const int64_t bytes = cache.dim / 64 * 2;
    const ReadArgs a{{k, v}, {ldk, ldv}, {fits(k, ldk, 2, bytes), fits(v, ldv, 2, bytes)}};
    auto go = [&](auto kernel) {
        kernel<<<(unsigned)rows, kHeadThreads, 0, stream>>>(a, view_of(cache), view_of(packed, rows));
    };
    if (cache.dim == 256) go(cache_read_kernel<256>);
    else if (cache.dim == 128) go(cache_read_kernel<128>);
    else go(cache_read_kernel<64>);
    return hipGetLastError();
}

}  // namespace splosh
