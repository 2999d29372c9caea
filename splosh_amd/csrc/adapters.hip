// adapters.hip -- low-rank adapters of many requests beside a shared projection.
//
// out[m] += c_s b_s (a_s x[m]) for the adapter s = slots[m] of row m, in two launches: the products
// t = a_s x (fp32, in the workspace), then out += c_s b_s t.
#include "common.hpp"
#include "launch.hpp"

namespace splosh {

// The workspace's first 16 KiB belong to the arrival counters of the kernels that have any.
constexpr size_t kAdapterCounterBytes = 16384;

struct AdapterWeight {
    splosh_adapters w;
    void *out;
    int64_t ldc;
    int t_offset;  // its first column of t
};

struct AdapterArgs {
    AdapterWeight w[SPLOSH_MAX_GROUP];
    const uint16_t *x;
    int64_t ldx;
    const int32_t *slots;
    float *t;     // [rows][t_cols]
    int t_cols;
    int64_t rows;
};

// The rank of the row's adapter, 0 for none.
__device__ __forceinline__ int adapter_rank(const splosh_adapters &w, int slot) {
    if (slot < 0 || slot >= w.count) return 0;
    const int rank = w.ranks ? w.ranks[slot] : (int)w.max_rank;
    return rank < (int)w.max_rank ? rank : (int)w.max_rank;
}

// One wave a (row, rank): the dot product of x[m] with one row of a.
__global__ void __launch_bounds__(64) adapter_down_kernel(AdapterArgs args, int which) {
    const AdapterWeight &g = args.w[which];
    const int64_t m = blockIdx.y;
    const int j = blockIdx.x, slot = args.slots[m];
    if (j >= adapter_rank(g.w, slot)) return;
    const uint16_t *a = g.w.a + slot * g.w.a_slot_stride + j * g.w.a_row_stride;
    const uint16_t *x = args.x + m * args.ldx;
    float sum = 0.0f;
    for (int64_t k = threadIdx.x; k < g.w.inner; k += 64)
        sum = __builtin_fmaf(bf16_bits_to_f32(x[k]), bf16_bits_to_f32(a[k]), sum);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
    if (threadIdx.x == 0) args.t[m * args.t_cols + g.t_offset + j] = sum;
}

// One thread an output.
template <typename OUT>
__global__ void __launch_bounds__(256) adapter_up_kernel(AdapterArgs args, int which) {
    const AdapterWeight &g = args.w[which];
    const int64_t m = blockIdx.y, n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int slot = args.slots[m], rank = adapter_rank(g.w, slot);
    if (rank <= 0 || n >= g.w.rows) return;
    const uint16_t *b = g.w.b + slot * g.w.b_slot_stride + n * g.w.b_row_stride;
    const float *t = args.t + m * args.t_cols + g.t_offset;
    float sum = 0.0f;
    for (int j = 0; j < rank; ++j) sum = __builtin_fmaf(t[j], bf16_bits_to_f32(b[j]), sum);
    const float scale = g.w.scales ? g.w.scales[slot] : 1.0f;
    OUT *out = (OUT *)g.out + m * g.ldc + n;
    if constexpr (sizeof(OUT) == 4)
        *out = __builtin_fmaf(scale, sum, *out);
    else
        *out = f32_to_bf16(__builtin_fmaf(scale, sum, bf16_bits_to_f32(*out)));
}

static int t_columns(const splosh_adapters *w, int group) {
    int cols = 0;
    for (int i = 0; i < group; ++i) cols += (int)w[i].max_rank;
    return cols;
}

size_t adapters_workspace_bytes(const splosh_adapters *w, int group, int64_t rows) {
    return kAdapterCounterBytes + (size_t)rows * t_columns(w, group) * sizeof(float);
}

hipError_t launch_adapters(const splosh_adapters *w, int group, const uint16_t *x, int64_t ldx, void *const *outs,
                           const int64_t *ldcs, int out_dtype, const int32_t *slots, int64_t rows, void *workspace,
                           hipStream_t stream) {
    AdapterArgs args{};
    args.x = x;
    args.ldx = ldx;
    args.slots = slots;
    args.t = (float *)((char *)workspace + kAdapterCounterBytes);
    args.t_cols = t_columns(w, group);
    args.rows = rows;
    int at = 0;
    for (int i = 0; i < group; ++i) {
        args.w[i] = AdapterWeight{w[i], outs[i], ldcs[i], at};
        at += (int)w[i].max_rank;
    }
    // (A launch takes 65535 rows.)
    for (int64_t m = 0; m < rows; m += 65535) {
        const unsigned part = (unsigned)(rows - m < 65535 ? rows - m : 65535);
        AdapterArgs p = args;
        p.x += m * ldx;
        p.slots += m;
        p.t += m * args.t_cols;
        for (int i = 0; i < group; ++i) {
            p.w[i].out = (char *)outs[i] + m * ldcs[i] * (out_dtype == SPLOSH_F32 ? 4 : 2);
            hipLaunchKernelGGL(adapter_down_kernel, dim3((unsigned)w[i].max_rank, part), dim3(64), 0, stream, p, i);
        }
        for (int i = 0; i < group; ++i) {
            const dim3 grid((unsigned)((w[i].rows + 255) / 256), part);
            if (out_dtype == SPLOSH_F32)
                hipLaunchKernelGGL(adapter_up_kernel<float>, grid, dim3(256), 0, stream, p, i);
            else
                hipLaunchKernelGGL(adapter_up_kernel<uint16_t>, grid, dim3(256), 0, stream, p, i);
        }
    }
    return hipGetLastError();
}

}  // namespace splosh
