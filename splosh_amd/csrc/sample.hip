// sample.hip -- the next token of each row: temperature, top-k, top-p and min-p from given random
// numbers.
//
// Every filter keeps a run from the start of one total order, larger logits first and of equal ones
// the lower index, so together they keep {element >= cut} of it (min-p a value bound of its own), and
// one cut decides the row. The order is that of a 64-bit key: the logit's bits made monotone, then the
// complement of the index. Weights are integers (2^40 for the largest logit), so that their sums do not
// depend on the order of the additions, whichever way a row's elements are split.
#include "common.hpp"
#include "launch.hpp"

namespace splosh {

constexpr size_t kSampleCounterBytes = 16384;
constexpr int kRowThreads = 1024;
constexpr int kWeightBits = 40;

__device__ __forceinline__ float logit_of(float v) { return v; }
__device__ __forceinline__ float logit_of(uint16_t v) { return bf16_bits_to_f32(v); }

// The logit's place in the order as an unsigned number: 0 for those that are never chosen (NaN, -inf);
// the two zeros are equal.
__device__ __forceinline__ uint32_t logit_key(float v) {
    uint32_t bits = __float_as_uint(v);
    if (bits == 0x80000000u) bits = 0;
    const uint32_t key = bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u);
    return v != v || key <= 0x007fffffu ? 0u : key;
}
__device__ __forceinline__ float key_logit(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ uint64_t order_key(float v, uint32_t index) {
    const uint32_t key = logit_key(v);
    return key ? (uint64_t)key << 32 | (0xffffffffu - index) : 0;
}

// exp((v - top) / T) in units of 2^-40, c = log2(e) / T: the exponent in 64 bits, its fraction's power
// by the hardware's (1 ulp of fp32, 2^-24 .. 2^-23 relative). The largest logit weighs 2^40 also where
// it is infinite.
__device__ __forceinline__ uint64_t logit_weight(float v, float top, double c) {
    if (v == top) return (uint64_t)1 << kWeightBits;
    const double t = ((double)v - (double)top) * c;
    if (!(t > -(kWeightBits + 2.0))) return 0;
    const double n = __builtin_rint(t);
    const uint32_t e = (uint32_t)(__builtin_amdgcn_exp2f((float)(t - n)) * 16777216.0f);
    const int shift = (int)n + kWeightBits - 24;
    return shift >= 0 ? (uint64_t)e << shift : (uint64_t)(((e >> (-shift - 1)) + 1) >> 1);
}

template <typename F>
__device__ __forceinline__ uint64_t block_reduce(uint64_t v, F op, uint64_t *scratch) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = op(v, __shfl_xor((unsigned long long)v, d, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    v = scratch[0];
    for (int i = 1; i < kRowThreads / 64; ++i) v = op(v, scratch[i]);
    return v;
}
struct MaxOp {
    __device__ uint64_t operator()(uint64_t a, uint64_t b) const { return a > b ? a : b; }
};
struct SumOp {
    __device__ uint64_t operator()(uint64_t a, uint64_t b) const { return a + b; }
};

struct SampleArgs {
    const void *logits;
    int64_t ld;
    int vocab;
    SampleParams p;
    uint32_t *tokens;
    float *logprobs;
};

struct RowShared {
    uint64_t reduce[kRowThreads / 64];
    uint64_t weight[256];
    uint32_t count[256];
    uint64_t found_key, found_weight, found_count;
};

// The smallest run from the start of the order, of at most `limit`'s keys on, with `k` elements, or with
// weight >= share where k is 0: the last element's key; *weight the run's weight.
template <typename T>
__device__ uint64_t find_cut(const T *row, int vocab, float top, double c, uint64_t limit, uint64_t k, double share,
                             uint64_t *weight, RowShared &sh) {
    const int tid = threadIdx.x;
    uint64_t prefix = 0, base_weight = 0, base_count = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        if (tid < 256) sh.count[tid] = 0, sh.weight[tid] = 0;
        __syncthreads();
        for (int i = tid; i < vocab; i += kRowThreads) {
            const float v = logit_of(row[i]);
            const uint64_t key = order_key(v, i);
            if (key == 0 || key < limit || (shift < 56 && key >> (shift + 8) != prefix >> (shift + 8))) continue;
            const int d = (int)(key >> shift) & 255;
            atomicAdd(&sh.count[d], 1u);
            atomicAdd((unsigned long long *)&sh.weight[d], (unsigned long long)logit_weight(v, top, c));
        }
        __syncthreads();
        if (tid == 0) {
            uint64_t wsum = base_weight, csum = base_count;
            for (int d = 255; d >= 0; --d) {
                if (sh.count[d] == 0) continue;
                const uint64_t w = wsum + sh.weight[d], n = csum + sh.count[d];
                sh.found_key = prefix | (uint64_t)d << shift;
                sh.found_weight = wsum;
                sh.found_count = csum;
                if (shift == 0) sh.found_weight = w;
                if (k ? n >= k : (double)w >= share) break;
                wsum = w;
                csum = n;
            }
        }
        __syncthreads();
        prefix = sh.found_key;
        base_weight = sh.found_weight;
        base_count = sh.found_count;
    }
    *weight = base_weight;
    return prefix;
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) sample_row_kernel(SampleArgs args) {
    __shared__ RowShared sh;
    const int tid = threadIdx.x, vocab = args.vocab;
    const int64_t r = blockIdx.x;
    const T *row = (const T *)args.logits + r * args.ld;
    uint64_t best = 0;
    for (int i = tid; i < vocab; i += kRowThreads) {
        const uint64_t key = order_key(logit_of(row[i]), i);
        best = key > best ? key : best;
    }
    best = block_reduce(best, MaxOp(), sh.reduce);
    const float temperature = args.p.temperature ? args.p.temperature[r] : 1.0f;
    if (best == 0 || !args.p.uniforms || !(temperature > 0.0f)) {
        if (tid == 0) {
            args.tokens[r] = best ? 0xffffffffu - (uint32_t)best : 0xffffffffu;
            if (args.logprobs) args.logprobs[r] = best ? 0.0f : -__builtin_inff();
        }
        return;
    }
    const float top = key_logit((uint32_t)(best >> 32));
    const double c = 1.4426950408889634074 / (double)temperature;
    // The cut of top-k, then that of top-p among its elements.
    uint64_t cut = 1, weight = 0, valid = 0;
    const int k = args.p.top_k ? args.p.top_k[r] : 0;
    const float p = args.p.top_p ? args.p.top_p[r] : 1.0f, q = args.p.min_p ? args.p.min_p[r] : 0.0f;
    for (int i = tid; i < vocab; i += kRowThreads) {
        const float v = logit_of(row[i]);
        if (logit_key(v)) ++valid, weight += logit_weight(v, top, c);
    }
    valid = block_reduce(valid, SumOp(), sh.reduce);
    weight = block_reduce(weight, SumOp(), sh.reduce);
    if (k > 0 && (uint64_t)k < valid) cut = find_cut(row, vocab, top, c, cut, (uint64_t)k, 0.0, &weight, sh);
    if (p < 1.0f) cut = find_cut(row, vocab, top, c, cut, 0, (double)p * (double)weight, &weight, sh);
    // min-p: w >= q, i.e. (v - top) c >= log2(q).
    const double low = q > 0.0f ? log2((double)(q < 1.0f ? q : 1.0f)) : -__builtin_inf();
    auto kept = [&](int i) -> uint64_t {
        const float v = logit_of(row[i]);
        const uint64_t key = order_key(v, i);
        if (key < cut || (v != top && !(((double)v - (double)top) * c >= low))) return 0;
        return logit_weight(v, top, c);
    };
    uint64_t total = 0;
    for (int i = tid; i < vocab; i += kRowThreads) total += kept(i);
    total = block_reduce(total, SumOp(), sh.reduce);
    // The first index whose running weight exceeds u total.
    const double u = args.p.uniforms[r], at = u * (double)total;
    uint64_t target = at > 0.0 ? (at < (double)total ? (uint64_t)at : total - 1) : 0;
    target = target < total ? target : total - 1;
    uint64_t before = 0;
    for (int base = 0; base < vocab; base += kRowThreads) {
        const uint64_t mine = base + tid < vocab ? kept(base + tid) : 0;
        const uint64_t all = block_reduce(mine, SumOp(), sh.reduce);
        if (before + all <= target) {
            before += all;
            continue;
        }
        uint64_t run = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t up = __shfl_up((unsigned long long)run, d, 64);
            if ((tid & 63) >= d) run += up;
        }
        __syncthreads();
        if ((tid & 63) == 63) sh.reduce[tid >> 6] = run;
        __syncthreads();
        for (int w = 0; w < tid >> 6; ++w) run += sh.reduce[w];
        if (before + run > target && before + run - mine <= target) {
            args.tokens[r] = (uint32_t)(base + tid);
            if (args.logprobs) args.logprobs[r] = (float)log((double)mine / (double)total);
        }
        return;
    }
}

size_t sample_workspace_bytes(int64_t rows, int64_t vocab) {
    (void)rows, (void)vocab;
    return kSampleCounterBytes;
}

hipError_t launch_sample(const void *logits, int64_t ld, int dtype, int64_t rows, int64_t vocab,
                         const SampleParams &params, uint32_t *tokens, float *logprobs, void *workspace,
                         hipStream_t stream) {
    (void)workspace;
    const SampleArgs args{logits, ld, (int)vocab, params, tokens, logprobs};
    if (dtype == SPLOSH_F32)
        hipLaunchKernelGGL(sample_row_kernel<float>, dim3((unsigned)rows), dim3(kRowThreads), 0, stream, args);
    else
        hipLaunchKernelGGL(sample_row_kernel<uint16_t>, dim3((unsigned)rows), dim3(kRowThreads), 0, stream, args);
    return hipGetLastError();
}

}  // namespace splosh
