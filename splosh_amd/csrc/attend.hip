// attend.hip -- causal attention of a packed step's rows over the 8-bit paged cache.
//
// A wave takes one (row, query head): its lanes hold dim / 64 dimensions each and go through the keys one after the
// other with the running maximum and sum of the softmax.
#include "cache.hpp"

namespace splosh {

constexpr int kAttendThreads = 256;

struct AttendArgs {
    const uint16_t *q;
    int64_t row_stride, head_stride;
    uint16_t *out;
    int64_t ld_out;
    int q_heads, group, shared;
    float scale;
};

template <int D>
__global__ __launch_bounds__(kAttendThreads) void attend_kernel(AttendArgs a, CacheView cache, PackedView packed) {
    constexpr int E = D / 64;
    const int row = blockIdx.x, lane = threadIdx.x & 63;
    const int r = request_of(packed.starts, packed.requests, row);
    if (r < 0) return;
    const int position = packed.lengths[r] - packed.starts[r + 1] + row;
    for (int h = threadIdx.x >> 6; h < a.q_heads; h += kAttendThreads / 64) {
        float q[E], o[E] = {}, most = -__builtin_inff(), sum = 0.0f;
        for (int e = 0; e < E; ++e)
            q[e] = bf16_bits_to_f32(a.q[row * a.row_stride + h * a.head_stride + lane * E + e]);
        for (int j = 0; j <= position; ++j) {
            int page, at;
            if (!place_of(cache, packed, j < a.shared ? 0 : r, j, page, at)) continue;
            const uint8_t *record = record_of<D>(cache, page, h / a.group, at / kBlock);
            const int8_t *k = reinterpret_cast<const int8_t *>(record) + at % kBlock * D + lane * E, *v = k + kBlock * D;
            const float *scales = reinterpret_cast<const float *>(record + 2 * kBlock * D) + at % kBlock;
            float s = 0.0f;
            for (int e = 0; e < E; ++e) s += q[e] * (float)k[e];
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m);
            s = s * scales[0] * a.scale * 1.4426950408889634f;
            const float top = __builtin_fmaxf(most, s), keep = exp2f(most - top), w = exp2f(s - top);
            most = top;
            sum = sum * keep + w;
            for (int e = 0; e < E; ++e) o[e] = o[e] * keep + w * scales[kBlock] * (float)v[e];
        }
        for (int e = 0; e < E; ++e)
            a.out[row * a.ld_out + h * D + lane * E + e] = f32_to_bf16(sum == 0.0f ? 0.0f : o[e] / sum);
    }
}

size_t attend_workspace_bytes(const splosh_cache &, int64_t, int64_t, int64_t, int64_t) { return 16384; }

hipError_t launch_attend(const uint16_t *q, int64_t row_stride, int64_t head_stride, int64_t q_heads,
                         const splosh_cache &cache, const splosh_packed &packed, int64_t rows, int64_t shared,
                         float scale, uint16_t *out, int64_t ld_out, void *, hipStream_t stream) {
    const AttendArgs a{q, row_stride, head_stride, out, ld_out, (int)q_heads, (int)(q_heads / cache.heads), (int)shared, scale};
    auto go = [&](auto kernel) {
        kernel<<<(unsigned)rows, kAttendThreads, 0, stream>>>(a, view_of(cache), view_of(packed, rows));
    };
    if (cache.dim == 256) go(attend_kernel<256>);
    else if (cache.dim == 128) go(attend_kernel<128>);
    else go(attend_kernel<64>);
    return hipGetLastError();
}

}  // namespace splosh
