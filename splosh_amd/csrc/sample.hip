// sample.hip -- the next token of each row: temperature, top-k, top-p and min-p from given random
// numbers.
//
// Every filter keeps a run from the start of one total order, larger logits first and of equal ones
// the lower index, so together they keep {element >= cut} of it (min-p a value bound of its own), and
// one cut decides the row. The order is that of a 64-bit key: the logit's bits made monotone, then the
// complement of the index. Weights are integers (2^40 for the largest logit of what they are measured
// against), so that their sums do not depend on the order of the additions.
//
// Two launches over pieces of 8192 logits, a workgroup each, the last of a row's to arrive going on with
// the row (no workgroup waits for another):
//   scan    -- a piece's largest logit and its weight, and for rows with a cut how many elements and how
//              much weight fall into each of 512 value bins below its largest. The row: greedy ones and
//              those with the temperature alone are settled here, from one piece more; else the bins that
//              the cut can be in.
//   collect -- the weight above these bins, and the elements in them as a list. The row: the list sorted,
//              the cut found on running sums, the piece the draw falls into and the token in it.
// A row whose cut lies below its bins, or in bins of more elements than the list holds, is settled by one
// workgroup with a radix search over the whole row.
#include "common.hpp"
#include "launch.hpp"

namespace splosh {

constexpr size_t kSampleCounterBytes = 16384;
constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kPer = 16;                     // logits a thread
constexpr int kPiece = kThreads * kPer;      // and a workgroup
constexpr int kBins = kThreads;              // value bins of a piece
constexpr int kList = 8192;                  // elements of a row's list
constexpr int kBatchRows = 256;              // rows of one launch
constexpr int kWeightBits = 40;
// A bin's entry: 15 bits of count (a piece has 2^13 elements) over 49 of weight in units of 2^-35.
constexpr int kBinShift = 49, kBinUnit = kWeightBits - 35;

static_assert((int64_t)kPiece * kThreads >= kSampleMaxVocab, "a row's pieces are one a thread");

typedef unsigned long long u64;

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
__device__ __forceinline__ u64 order_key(float v, uint32_t index) {
    const uint32_t key = logit_key(v);
    return key ? (u64)key << 32 | (0xffffffffu - index) : 0;
}

// exp((v - top) / T) in units of 2^-40, c = log2(e) / T: the exponent in 64 bits, its fraction's power
// by the hardware's (1 ulp of fp32, 2^-24 .. 2^-23 relative). The largest logit weighs 2^40 also where
// it is infinite.
__device__ __forceinline__ u64 logit_weight(float v, float top, double c) {
    if (v == top) return (u64)1 << kWeightBits;
    const double t = ((double)v - (double)top) * c;
    if (!(t > -(kWeightBits + 2.0))) return 0;
    const double n = __builtin_rint(t);
    const uint32_t e = (uint32_t)(__builtin_amdgcn_exp2f((float)(t - n)) * 16777216.0f);
    const int shift = (int)n + kWeightBits - 24;
    return shift >= 0 ? (u64)e << shift : (u64)(((e >> (-shift - 1)) + 1) >> 1);
}

// w >= q for min-p, low = log2(q).
__device__ __forceinline__ bool weighs(float v, float top, double c, double low) {
    return v == top || ((double)v - (double)top) * c >= low;
}

// The value bins: 64 an octave of 1 + |logit|, so 1/64 wide about 0 and 1/8 about 10, the same for every
// piece and row. Monotone in the logit.
__device__ __forceinline__ int value_bin(float v) {
    const int bin = (int)(__float_as_uint(__builtin_fabsf(v) + 1.0f) >> 17) - (127 << 6);
    return v >= 0.0f ? bin : -1 - bin;
}

// ---- across a workgroup ---------------------------------------------------------------------------

template <typename V>
__device__ __forceinline__ V shuffle_xor(V v, int d) {
    if constexpr (sizeof(V) == 8) return (V)__shfl_xor((u64)v, d, 64);
    else return __shfl_xor(v, d, 64);
}
struct MaxOp {
    template <typename V> __device__ V operator()(V a, V b) const { return a > b ? a : b; }
};
struct MinOp {
    template <typename V> __device__ V operator()(V a, V b) const { return a < b ? a : b; }
};
struct SumOp {
    template <typename V> __device__ V operator()(V a, V b) const { return a + b; }
};
template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, F op, u64 *scratch) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = op(v, shuffle_xor(v, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = (u64)v;
    __syncthreads();
    v = (V)scratch[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) v = op(v, (V)scratch[i]);
    return v;
}
// The sum over the threads up to this one.
__device__ __forceinline__ u64 block_scan(u64 v, u64 *scratch) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 up = __shfl_up(v, d, 64);
        if (lane >= d) v += up;
    }
    __syncthreads();
    if (lane == 63) scratch[wave] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves - 1; ++i)
        if (i < wave) v += scratch[i];
    return v;
}

// ---- what the launches leave for each other ---------------------------------------------------------
//
// What a workgroup of the same launch reads is written and read past the L2s (agent scope), which are one an
// XCD and not coherent.

__device__ __forceinline__ void put(u64 *p, u64 v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ u64 get(const u64 *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

enum RowState : int { kSettled = 0, kCollect = 1, kSearch = 2 };

struct RowPlan {
    int state, above_bin, low_bin;  // the list takes the bins [low_bin, above_bin)
    uint32_t top_key;
    u64 total;         // the whole row's weight, of the largest logit
    uint32_t above;    // elements in the bins above the list's
    uint32_t listed;   // elements of the list so far
    uint32_t valid, reserved;
};
// A piece. key: its largest logit's << 32 | the index of that.
struct PieceHead {
    u64 key, weight, valid;  // scan: its weight, of its own largest logit; its elements that can be chosen
    u64 above, kept;         // collect: the weight above the list's bins, and of it what min-p leaves
};
struct RowScratch {
    RowPlan plan;
    PieceHead heads[1];  // [pieces], then the bins u64 [pieces][kBins], then the list u64 [kList]
};

struct SampleArgs {
    const void *logits;
    int64_t ld;
    int vocab, pieces;
    SampleParams p;
    uint32_t *tokens;
    float *logprobs;
    int *arrivals;
    char *rows;
    size_t row_bytes;
};

__device__ __forceinline__ RowScratch &row_scratch(const SampleArgs &args, int r) {
    return *(RowScratch *)(args.rows + r * args.row_bytes);
}
__device__ __forceinline__ u64 *row_bins(const SampleArgs &args, RowScratch &row) {
    return (u64 *)&row.heads[args.pieces];
}
__device__ __forceinline__ u64 *row_list(const SampleArgs &args, RowScratch &row) {
    return row_bins(args, row) + (size_t)args.pieces * kBins;
}

struct RowParams {
    bool greedy;
    double c;  // log2(e) / T
    int k;     // 0: off
    float p;   // 1: off
    float q;   // 0: off
    float u;
    // log2(q), the least (v - top) c of what min-p keeps; -inf: off.
    __device__ double low() const { return q > 0.0f ? log2((double)q) : -__builtin_inf(); }
};
__device__ __forceinline__ RowParams row_params(const SampleArgs &args, int64_t r) {
    const float t = args.p.temperature ? args.p.temperature[r] : 1.0f, p = args.p.top_p ? args.p.top_p[r] : 1.0f,
                q = args.p.min_p ? args.p.min_p[r] : 0.0f;
    const int k = args.p.top_k ? args.p.top_k[r] : 0;
    RowParams out;
    out.greedy = !args.p.uniforms || !(t > 0.0f);
    out.c = 1.4426950408889634074 / (double)t;
    out.k = k > 0 ? k : 0;
    out.p = p < 1.0f ? p : 1.0f;
    out.q = q > 0.0f ? (q < 1.0f ? q : 1.0f) : 0.0f;
    out.u = args.p.uniforms ? args.p.uniforms[r] : 0.0f;
    return out;
}

// floor(u total), below total.
__device__ __forceinline__ u64 draw_of(float u, u64 total) {
    const double at = (double)u * (double)total;
    if (!(at > 0.0)) return 0;
    const u64 target = at < (double)total ? (u64)at : total;
    return target < total ? target : total - 1;
}

// The last workgroup of `parts` to arrive. What each has put before is then there for it.
__device__ __forceinline__ bool last_to_arrive(int *counter, int parts, int *shared) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const int old = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (old == parts - 1) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *shared = old;
    }
    __syncthreads();
    return *shared == parts - 1;
}

// A thread's sixteen logits of the piece at `base`: v, and their indexes through index_of. Past the vocabulary
// and NaN: -inf. VECTOR: rows whose 16-byte pieces are aligned.
template <typename T, bool VECTOR>
__device__ __forceinline__ int index_of(int e) {
    constexpr int kRun = VECTOR ? 16 / (int)sizeof(T) : 1;
    return e / kRun * (kThreads * kRun) + (int)threadIdx.x * kRun + e % kRun;
}
template <typename T, bool VECTOR>
__device__ __forceinline__ void load_piece(const T *row, int base, int vocab, float (&v)[kPer]) {
    constexpr int kRun = VECTOR ? 16 / (int)sizeof(T) : 1;
#pragma unroll
    for (int e = 0; e < kPer; e += kRun) {
        const int i = base + index_of<T, VECTOR>(e);
        if (VECTOR && i + kRun <= vocab) {
            const u32x4 w = *(const u32x4 *)(row + i);
#pragma unroll
            for (int j = 0; j < kRun; ++j)
                v[e + j] = sizeof(T) == 4 ? __uint_as_float(w[j & 3])
                                          : bf16_bits_to_f32(j & 1 ? w[(j >> 1) & 3] >> 16 : w[(j >> 1) & 3] & 0xffffu);
        } else {
#pragma unroll
            for (int j = 0; j < kRun; ++j) v[e + j] = i + j < vocab ? logit_of(row[i + j]) : -__builtin_inff();
        }
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] = v[e] != v[e] ? -__builtin_inff() : v[e];
}

struct Shared {
    u64 scratch[kWaves];
    int arrival;
    int chosen;
    u64 rest;
    int cuts[4];
    u64 weights[4];
};

// The token of a settled piece: the first index of the piece whose running weight over the kept elements
// (order key >= cut, weight of `top` at least 2^low) exceeds `target`. probability: its weight times `scale`.
template <typename T>
__device__ __forceinline__ void locate(const SampleArgs &args, int64_t r, const T *row, int piece, float top, double c, u64 cut,
                                       double low, u64 target, double scale, Shared &sh) {
    const int first = piece * kPiece + (int)threadIdx.x * kPer;
    u64 w[kPer], sum = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const float v = first + e < args.vocab ? logit_of(row[first + e]) : -__builtin_inff();
        const u64 key = order_key(v, first + e);
        w[e] = key && key >= cut && weighs(v, top, c, low) ? logit_weight(v, top, c) : 0;
        sum += w[e];
    }
    u64 run = block_scan(sum, sh.scratch) - sum;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        if (run <= target && target < run + w[e]) {
            args.tokens[r] = (uint32_t)(first + e);
            if (args.logprobs) args.logprobs[r] = (float)log((double)w[e] * scale);
        }
        run += w[e];
    }
}

// The piece the draw falls into, from its weight in thread `piece`; the rest of the target there.
__device__ __forceinline__ u64 choose_piece(u64 weight, float u, Shared &sh) {
    const u64 run = block_scan(weight, sh.scratch);
    u64 total = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) total += sh.scratch[i];
    const u64 target = draw_of(u, total);
    if (run > target && run - weight <= target) {
        sh.chosen = (int)threadIdx.x;
        sh.rest = target - (run - weight);
    }
    __syncthreads();
    return total;
}

// ---- the radix search over a whole row ---------------------------------------------------------------

constexpr int kDigitBits = 11;

// The smallest run from the start of the order, of keys >= limit, with `k` elements, or with weight >= share
// where k is 0: its last key; *weight its weight. counts and sums: 2^kDigitBits each.
template <typename T>
__device__ __noinline__ u64 find_cut(const T *row, int vocab, float top, double c, u64 limit, u64 k, double share,
                                     u64 *weight, uint32_t *counts, u64 *sums, Shared &sh) {
    const int tid = threadIdx.x;
    u64 prefix = 0, base_weight = 0, base_count = 0;
    for (int shift = 64 - kDigitBits, bits = kDigitBits;; shift -= bits) {
        const u64 above = shift + bits >= 64 ? 0 : ~(u64)0 << (shift + bits);
        for (int d = tid; d < 1 << bits; d += kThreads) counts[d] = 0, sums[d] = 0;
        __syncthreads();
        for (int i = tid; i < vocab; i += kThreads) {
            const float v = logit_of(row[i]);
            const u64 key = order_key(v, i);
            if (key == 0 || key < limit || ((key ^ prefix) & above)) continue;
            const int d = (int)(key >> shift) & ((1 << bits) - 1);
            atomicAdd(&counts[d], 1u);
            atomicAdd(&sums[d], logit_weight(v, top, c));
        }
        __syncthreads();
        // The digits from the largest down, a run of them a thread; the first that the run can end in, or where
        // rounding leaves none the last there is.
        const int per = (1 << bits) / kThreads, high = (1 << bits) - 1 - tid * per;
        u64 own_count = 0, own_weight = 0;
        for (int d = high; d > high - per; --d) own_count += counts[d], own_weight += sums[d];
        u64 n = base_count + block_scan(own_count, sh.scratch) - own_count;
        u64 w = base_weight + block_scan(own_weight, sh.scratch) - own_weight;
        if (tid == 0) sh.cuts[0] = -1, sh.cuts[1] = 1 << bits;
        __syncthreads();
        for (int pass = 0; pass < 2; ++pass) {
            for (int d = high; d > high - per; --d) {
                if (counts[d] == 0) continue;
                const bool before = (k ? n >= k : (double)w >= share) && n != base_count;
                n += counts[d];
                w += sums[d];
                if (pass == 0) atomicMin(&sh.cuts[1], d);
                if (pass == 0 ? !before && (k ? n >= k : (double)w >= share) : d == sh.cuts[1]) {
                    sh.cuts[0] = d;
                    sh.weights[0] = w - sums[d];
                    sh.weights[1] = n - counts[d];
                    sh.weights[2] = w;
                }
            }
            __syncthreads();
            if (sh.cuts[0] >= 0) break;
        }
        if (tid == 0) sh.rest = prefix | (u64)sh.cuts[0] << shift;
        __syncthreads();
        prefix = sh.rest;
        base_weight = sh.weights[0];
        base_count = sh.weights[1];
        *weight = sh.weights[2];
        if (shift == 0) return prefix;
        if (shift < kDigitBits) bits = shift;
    }
}

template <typename T>
__device__ __noinline__ void search_row(const SampleArgs &args, int64_t r, const T *row, const RowPlan &plan,
                                        const RowParams &rp, u64 *memory, Shared &sh) {
    uint32_t *counts = (uint32_t *)memory;
    u64 *sums = memory + (1 << kDigitBits) / 2;
    const float top = key_logit(plan.top_key);
    const double low = rp.low();
    u64 cut = 1, weight = plan.total;
    if (rp.k && (uint32_t)rp.k < plan.valid)
        cut = find_cut(row, args.vocab, top, rp.c, cut, (u64)rp.k, 0.0, &weight, counts, sums, sh);
    if (rp.p < 1.0f)
        cut = find_cut(row, args.vocab, top, rp.c, cut, 0, (double)rp.p * (double)weight, &weight, counts, sums, sh);
    // The pieces' kept weights, thread by thread.
    u64 mine = 0;
    for (int piece = 0; piece < args.pieces; ++piece) {
        float v[kPer];
        load_piece<T, false>(row, piece * kPiece, args.vocab, v);
        u64 kept = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const u64 key = order_key(v[e], piece * kPiece + index_of<T, false>(e));
            if (key && key >= cut && weighs(v[e], top, rp.c, low)) kept += logit_weight(v[e], top, rp.c);
        }
        kept = block_reduce(kept, SumOp(), sh.scratch);
        if ((int)threadIdx.x == piece) mine = kept;
    }
    const u64 total = choose_piece(mine, rp.u, sh);
    locate<T>(args, r, row, sh.chosen, top, rp.c, cut, low, sh.rest, 1.0 / (double)total, sh);
}

// ---- scan -------------------------------------------------------------------------------------------

// 2^t for t <= 0, in 64 bits.
__device__ __forceinline__ double power_of(double t) { return t > -1000.0 ? exp2(t) : 0.0; }

template <typename T, bool VECTOR>
__global__ void __launch_bounds__(kThreads) sample_scan_kernel(SampleArgs args) {
    __shared__ Shared sh;
    __shared__ u64 bins[kBins];
    const int tid = threadIdx.x, piece = blockIdx.x;
    const int64_t r = blockIdx.y;
    const T *row = (const T *)args.logits + r * args.ld;
    float v[kPer];
    load_piece<T, VECTOR>(row, piece * kPiece, args.vocab, v);
    const RowParams rp = row_params(args, r);
    const bool cut = !rp.greedy && (rp.k || rp.p < 1.0f);
    RowScratch &scratch = row_scratch(args, (int)r);
    bins[tid] = 0;
    uint32_t best = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const uint32_t key = logit_key(v[e]);
        best = best > key ? best : key;
    }
    best = block_reduce(best, MaxOp(), sh.scratch);
    u64 weight = 0, valid = 0, index = 0;
    if (rp.greedy) {
        uint32_t at = 0xffffffffu;
#pragma unroll
        for (int e = kPer - 1; e >= 0; --e)
            if (logit_key(v[e]) == best) at = (uint32_t)(piece * kPiece + index_of<T, VECTOR>(e));
        index = block_reduce(at, MinOp(), sh.scratch);
    } else if (best) {
        const float top = key_logit(best);
        const int top_bin = value_bin(top);
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const u64 w = logit_weight(v[e], top, rp.c);
            weight += w;
            if (cut && logit_key(v[e])) {
                ++valid;
                const int below = top_bin - value_bin(v[e]);
                if (below < kBins) atomicAdd(&bins[below], (u64)1 << kBinShift | w >> kBinUnit);
            }
        }
        // (Sixteen times 512 weights of 2^40 at most, and 2^13 elements: one sum of both.)
        weight = block_reduce(weight, SumOp(), sh.scratch);
        if (cut) valid = block_reduce(valid, SumOp(), sh.scratch);
    }
    if (tid == 0) {
        put(&scratch.heads[piece].key, (u64)best << 32 | index);
        put(&scratch.heads[piece].weight, weight);
        put(&scratch.heads[piece].valid, valid);
    }
    u64 *all_bins = row_bins(args, scratch);
    if (cut) put(&all_bins[(size_t)piece * kBins + tid], bins[tid]);
    if (!last_to_arrive(args.arrivals + r, args.pieces, &sh.arrival)) return;

    // The row: one piece a thread.
    __shared__ float factors[kThreads];  // the pieces' weights in the row's
    __shared__ int top_bins[kThreads];
    const u64 key = tid < args.pieces ? get(&scratch.heads[tid].key) : 0;
    const u64 piece_weight = tid < args.pieces ? get(&scratch.heads[tid].weight) : 0;
    const u64 piece_valid = tid < args.pieces ? get(&scratch.heads[tid].valid) : 0;
    const uint32_t top_key = block_reduce((uint32_t)(key >> 32), MaxOp(), sh.scratch);
    RowPlan &plan = scratch.plan;
    if (rp.greedy || top_key == 0) {
        // The first piece that has the largest has its first index.
        const uint32_t at = block_reduce((uint32_t)(key >> 32) == top_key ? (uint32_t)key : 0xffffffffu, MinOp(), sh.scratch);
        if (tid == 0) {
            args.tokens[r] = top_key ? at : 0xffffffffu;
            if (args.logprobs) args.logprobs[r] = top_key ? 0.0f : -__builtin_inff();
            plan.state = kSettled;
        }
        return;
    }
    const float top = key_logit(top_key), piece_top = key_logit((uint32_t)(key >> 32));
    const double factor = key >> 32 == 0 ? 0.0
                          : piece_top == top ? 1.0 : power_of(((double)piece_top - (double)top) * rp.c);
    const u64 row_weight = (u64)((double)piece_weight * factor);
    if (!cut && rp.q == 0.0f) {  // the temperature alone
        const u64 total = choose_piece(row_weight, rp.u, sh);
        __shared__ double chosen_factor;
        __shared__ u64 chosen_weight, chosen_key;
        if (tid == sh.chosen) chosen_factor = factor, chosen_weight = piece_weight, chosen_key = key;
        __syncthreads();
        u64 target = (u64)((double)sh.rest / chosen_factor);
        target = target < chosen_weight ? target : chosen_weight - 1;
        locate<T>(args, r, row, sh.chosen, key_logit((uint32_t)(chosen_key >> 32)), rp.c, 1, -__builtin_inf(), target,
                  chosen_factor / (double)total, sh);
        if (tid == 0) plan.state = kSettled;
        return;
    }
    const u64 total = block_reduce(row_weight, SumOp(), sh.scratch);
    const u64 all_valid = block_reduce(piece_valid, SumOp(), sh.scratch);
    if (!cut) {  // min-p alone: everything is above the list
        if (tid == 0) plan = {kCollect, -0x7fffffff, -0x7fffffff, top_key, total, 0, 0, (uint32_t)all_valid, 0};
        return;
    }
    // The row's bins: thread j the j-th below that of its largest logit.
    const int top_bin = value_bin(top);
    factors[tid] = (float)factor;
    top_bins[tid] = key >> 32 ? value_bin(piece_top) : -0x40000000;
    __syncthreads();
    u64 count = 0;
    double bin_weight = 0.0;
    constexpr int kAtOnce = 8;
    for (int first = 0; first < args.pieces; first += kAtOnce) {
        u64 entry[kAtOnce];
#pragma unroll
        for (int e = 0; e < kAtOnce; ++e) {
            const int below = first + e < args.pieces ? tid - (top_bin - top_bins[first + e]) : -1;
            entry[e] = below >= 0 ? get(&all_bins[(size_t)(first + e) * kBins + below]) : 0;
        }
#pragma unroll
        for (int e = 0; e < kAtOnce; ++e) {
            count += entry[e] >> kBinShift;
            bin_weight += (double)((entry[e] & (((u64)1 << kBinShift) - 1)) << kBinUnit) *
                          (double)(first + e < args.pieces ? factors[first + e] : 0.0f);
        }
    }
    const u64 own_weight = (u64)bin_weight, run_count = block_scan(count, sh.scratch),
              run_weight = block_scan(own_weight, sh.scratch);
    // cuts: the bins of the k-th element, and those between which the run ends that has the share p.
    if (tid < 4) sh.cuts[tid] = kBins;
    __syncthreads();
    const bool by_count = rp.k && (u64)rp.k < all_valid;
    if (by_count && run_count >= (u64)rp.k && run_count - count < (u64)rp.k) {
        sh.cuts[0] = tid;
        sh.weights[0] = run_weight - own_weight;
        sh.weights[1] = run_weight;
    }
    __syncthreads();
    const bool found = !by_count || sh.cuts[0] < kBins;
    if (rp.p < 1.0f && found) {
        // (The bins' weights are exact to 2^-22 or better: piece factors in fp32, entries in 2^-35.)
        constexpr double kSlack = 1.0 / (1 << 20);
        const double least = (double)rp.p * (double)(by_count ? sh.weights[0] : total) * (1.0 - kSlack);
        const double most = (double)rp.p * (double)(by_count ? sh.weights[1] : total) * (1.0 + kSlack);
        if (count && (double)run_weight >= least && ((double)(run_weight - own_weight) < least || run_count == count))
            sh.cuts[1] = tid;
        if (count && (double)run_weight >= most && ((double)(run_weight - own_weight) < most || run_count == count))
            sh.cuts[2] = tid;
    }
    __syncthreads();
    // The list: from the first bin that the cut can be in to the last that matters.
    const int from = rp.p < 1.0f ? sh.cuts[1] : sh.cuts[0];
    const int to = by_count ? sh.cuts[0] : rp.p < 1.0f ? sh.cuts[2] : sh.cuts[0];
    const bool none = !by_count && !(rp.p < 1.0f);  // k is past what the row has
    if (none) {
        if (tid == 0) plan = {kCollect, -0x7fffffff, -0x7fffffff, top_key, total, 0, 0, (uint32_t)all_valid, 0};
        return;
    }
    if (from < kBins && tid == from) sh.weights[2] = run_count - count;
    if (to < kBins && tid == to) sh.weights[3] = run_count;
    __syncthreads();
    if (tid == 0) {
        const bool fits = from < kBins && to < kBins && sh.weights[3] - sh.weights[2] <= kList;
        plan = {fits ? kCollect : kSearch, top_bin - from + 1, top_bin - to, top_key, total,
                fits ? (uint32_t)sh.weights[2] : 0, 0, (uint32_t)all_valid, 0};
    }
}

// ---- collect ----------------------------------------------------------------------------------------

template <typename T, bool VECTOR>
__global__ void __launch_bounds__(kThreads) sample_collect_kernel(SampleArgs args) {
    __shared__ Shared sh;
    __shared__ u64 list[kList];
    const int tid = threadIdx.x, piece = blockIdx.x, lane = tid & 63;
    const int64_t r = blockIdx.y;
    RowScratch &scratch = row_scratch(args, (int)r);
    const RowPlan plan = scratch.plan;
    const u64 piece_key = scratch.heads[piece].key >> 32;
    if (plan.state == kSettled) return;
    const T *row = (const T *)args.logits + r * args.ld;
    const RowParams rp = row_params(args, r);
    if (plan.state == kSearch) {
        if (piece == 0) search_row<T>(args, r, row, plan, rp, list, sh);
        return;
    }
    const float top = key_logit(plan.top_key), piece_top = key_logit((uint32_t)piece_key);
    const double low = rp.low();
    u64 *row_list_at = row_list(args, scratch);
    u64 above = 0, kept = 0;
    // (A piece whose largest is below the list's bins, or below min-p with no list, has nothing to give.)
    if (piece_key && value_bin(piece_top) >= plan.low_bin &&
        (plan.low_bin != -0x7fffffff || weighs(piece_top, top, rp.c, low))) {
        float v[kPer];
        load_piece<T, VECTOR>(row, piece * kPiece, args.vocab, v);
        int mine = 0;
        uint32_t listed = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            if (logit_key(v[e]) == 0) continue;
            const int bin = value_bin(v[e]);
            if (bin >= plan.above_bin) {
                const u64 w = logit_weight(v[e], top, rp.c);
                above += w;
                if (weighs(v[e], top, rp.c, low)) kept += w;
            } else if (bin >= plan.low_bin) {
                listed |= 1u << e;
                ++mine;
            }
        }
        // Places in the row's list, a wave at a time.
        if (__ballot(mine != 0)) {
            int run = mine;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int up = __shfl_up(run, d, 64);
                if (lane >= d) run += up;
            }
            uint32_t at = 0;
            if (lane == 63)
                at = __hip_atomic_fetch_add(&scratch.plan.listed, (uint32_t)run, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            at = __builtin_amdgcn_readlane(at, 63) + (uint32_t)(run - mine);
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                if (listed >> e & 1) {
                    if (at < kList) put(&row_list_at[at], order_key(v[e], piece * kPiece + index_of<T, VECTOR>(e)));
                    ++at;
                }
        }
        above = block_reduce(above, SumOp(), sh.scratch);
        kept = block_reduce(kept, SumOp(), sh.scratch);
    }
    if (tid == 0) {
        put(&scratch.heads[piece].above, above);
        put(&scratch.heads[piece].kept, kept);
    }
    if (!last_to_arrive(args.arrivals + r, args.pieces, &sh.arrival)) return;

    // The row. The list in order, larger keys first.
    const uint32_t listed = __hip_atomic_load(&scratch.plan.listed, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int n = listed < (uint32_t)kList ? (int)listed : kList;
    u64 piece_kept = tid < args.pieces ? get(&scratch.heads[tid].kept) : 0;
    const u64 piece_above = tid < args.pieces ? get(&scratch.heads[tid].above) : 0;
    u64 cut = 1;
    if (n) {
        int size = 64;
        while (size < n) size *= 2;
        for (int i = tid; i < size; i += kThreads) list[i] = i < n ? get(&row_list_at[i]) : 0;
        for (int width = 2; width <= size; width *= 2)
            for (int step = width / 2; step > 0; step /= 2) {
                __syncthreads();
                for (int i = tid; i < size / 2; i += kThreads) {
                    const int a = 2 * i - (i & (step - 1)), b = a + step;
                    const u64 x = list[a], y = list[b];
                    if ((x < y) == ((a & width) == 0)) list[a] = y, list[b] = x;
                }
            }
        const u64 row_above = block_reduce(piece_above, SumOp(), sh.scratch);
        // Running weights over runs of the list, one a thread.
        const int per = (n + kThreads - 1) / kThreads, first = tid * per;
        u64 sum = 0;
        for (int i = first; i < first + per && i < n; ++i) sum += logit_weight(key_logit((uint32_t)(list[i] >> 32)), top, rp.c);
        const u64 before = row_above + block_scan(sum, sh.scratch) - sum;
        // The k-th element, and the weight up to it.
        const bool by_count = rp.k && (uint32_t)rp.k < plan.valid;
        int last = n - 1;
        if (by_count) {
            const int64_t at = (int64_t)rp.k - plan.above - 1;
            last = at < 0 ? 0 : at < n ? (int)at : n - 1;
        }
        if (tid == 0) sh.cuts[0] = last;
        if (by_count && last >= first && last < first + per) {
            u64 run = before;
            for (int i = first; i <= last; ++i) run += logit_weight(key_logit((uint32_t)(list[i] >> 32)), top, rp.c);
            sh.weights[0] = run;
        }
        __syncthreads();
        if (rp.p < 1.0f) {
            const double share = (double)rp.p * (double)(by_count ? sh.weights[0] : plan.total);
            u64 run = before;
            for (int i = first; i < first + per && i <= last; ++i) {
                const u64 w = logit_weight(key_logit((uint32_t)(list[i] >> 32)), top, rp.c);
                run += w;
                // (The first that reaches the share; where rounding has the elements above reach it, the first.)
                if ((double)run >= share && ((double)(run - w) < share || i == 0)) sh.cuts[0] = i;
            }
        }
        __syncthreads();
        cut = list[sh.cuts[0]];
        // What min-p leaves of the list's kept elements, to their pieces.
        u64 *extra = (u64 *)list;  // (kept apart by the barriers)
        const int end = sh.cuts[0] + 1;
        u64 keys[kList / kThreads];
#pragma unroll
        for (int j = 0; j < kList / kThreads; ++j) {
            const int i = tid + j * kThreads;
            keys[j] = i < end ? list[i] : 0;
        }
        __syncthreads();
        extra[tid] = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kList / kThreads; ++j) {
            const float v = key_logit((uint32_t)(keys[j] >> 32));
            if (keys[j] && weighs(v, top, rp.c, low))
                atomicAdd(&extra[(0xffffffffu - (uint32_t)keys[j]) / kPiece], logit_weight(v, top, rp.c));
        }
        __syncthreads();
        piece_kept += extra[tid];
    }
    const u64 total = choose_piece(piece_kept, rp.u, sh);
    locate<T>(args, r, row, sh.chosen, top, rp.c, cut, low, sh.rest, 1.0 / (double)total, sh);
}

// ---- host -------------------------------------------------------------------------------------------

static int64_t pieces_of(int64_t vocab) { return (vocab + kPiece - 1) / kPiece; }
static size_t row_bytes(int64_t vocab) {
    const int64_t pieces = pieces_of(vocab);
    const size_t bytes = sizeof(RowPlan) + pieces * sizeof(PieceHead) + pieces * kBins * sizeof(u64) + kList * sizeof(u64);
    return (bytes + 255) / 256 * 256;
}

size_t sample_workspace_bytes(int64_t rows, int64_t vocab) {
    return kSampleCounterBytes + (size_t)(rows < kBatchRows ? rows : kBatchRows) * row_bytes(vocab);
}

template <typename T, bool VECTOR>
static void launch_batch(const SampleArgs &args, int rows, hipStream_t stream) {
    const dim3 grid((unsigned)args.pieces, (unsigned)rows);
    hipLaunchKernelGGL((sample_scan_kernel<T, VECTOR>), grid, dim3(kThreads), 0, stream, args);
    if (args.p.uniforms)
        hipLaunchKernelGGL((sample_collect_kernel<T, VECTOR>), grid, dim3(kThreads), 0, stream, args);
}

hipError_t launch_sample(const void *logits, int64_t ld, int dtype, int64_t rows, int64_t vocab,
                         const SampleParams &params, uint32_t *tokens, float *logprobs, void *workspace,
                         hipStream_t stream) {
    const int64_t esize = dtype == SPLOSH_F32 ? 4 : 2;
    const bool vector = (uintptr_t)logits % 16 == 0 && ld * esize % 16 == 0;
    for (int64_t at = 0; at < rows; at += kBatchRows) {
        const int count = (int)(rows - at < kBatchRows ? rows - at : kBatchRows);
        SampleArgs args{};
        args.logits = (const char *)logits + at * ld * esize;
        args.ld = ld;
        args.vocab = (int)vocab;
        args.pieces = (int)pieces_of(vocab);
        auto from = [at](auto *p) { return p ? p + at : p; };
        args.p = {from(params.uniforms), from(params.temperature), from(params.top_k), from(params.top_p), from(params.min_p)};
        args.tokens = tokens + at;
        args.logprobs = from(logprobs);
        args.arrivals = (int *)workspace;
        args.rows = (char *)workspace + kSampleCounterBytes;
        args.row_bytes = row_bytes(vocab);
        if (dtype == SPLOSH_F32) {
            if (vector) launch_batch<float, true>(args, count, stream);
            else launch_batch<float, false>(args, count, stream);
        } else {
            if (vector) launch_batch<uint16_t, true>(args, count, stream);
            else launch_batch<uint16_t, false>(args, count, stream);
        }
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

}  // namespace splosh
