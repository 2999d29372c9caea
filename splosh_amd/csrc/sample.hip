// sample.hip -- the next token of each row: temperature, top-k, top-p and min-p from given random
// numbers.
//
// Every filter keeps a run from the start of one total order, larger logits first and of equal ones
// the lower index, so together they keep {element >= cut} of it (min-p a value bound of its own), and
// one cut decides the row. The order is that of a 64-bit key: the logit's bits made monotone, then the
// complement of the index in as many bits as the vocabulary takes. What decides between elements is summed in
// integers (2^40 for the row's largest logit), so that no order of additions matters.
//
// Four launches; a workgroup takes a piece of 8192 logits, or a row:
//   scan    (pieces) the piece's largest logit, the weight of each wave's strip of 1024 against it, and for
//           rows with a cut how many elements and how much weight fall into each of 512 value bins
//           below it;
//   settle  (rows)   greedy rows and those with the temperature alone are settled, from one strip more;
//           for the others, the bins that the cut can be in;
//   collect (pieces) each strip's weight above these bins, and the elements in them as a list;
//   finish  (rows)   the cut, by ranking a short list or by a radix search in it, the strip the draw falls into and
//           the token in it. A row is searched whole where the bins cannot narrow its cut down to the list: by one
//           workgroup, a pass over the row for each nine bits of key (248320 fp32: 0.4 to 0.9 ms, 64 rows of it 0.6 to
//           1.2; all logits equal 2.1 and 2.3). Which rows those are: see settle.
// The launches over pieces hold nothing but what they stream, so that four workgroups share a CU. The rows' launches
// are chains of a few dependent round trips, about 1.5 us of each the launch's own: one row of 248320 with every
// filter takes 5.2 + 6.4 + 4.9 + 4.8 us, and 64 of them 19 + 7.1 + 7.4 + 5.6. What has to move is the logits, once:
// 64 rows of 248320 fp32, 64 MB, 13 us at the rate of a large copy.
#include "common.hpp"
#include "launch.hpp"

namespace splosh {

// The workspace's first 16 KiB belong to the arrival counters of the kernels that have any.
constexpr size_t kSampleCounterBytes = 16384;
constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kPer = 16;                     // logits a thread
constexpr int kStrip = 64 * kPer;            // a wave
constexpr int kPiece = kThreads * kPer;      // and a workgroup
constexpr int kBins = kThreads;              // value bins of a piece
constexpr int kWeightBits = 40;
// A bin's entry while it is counted: 15 bits of count (a piece has 2^13 elements) over 49 of weight in units of
// 2^-31, so that an element's fits 32 bits; as it is left, the count over the fp32 weight in units of 2^-40.
constexpr int kBinShift = 49, kBinBits = 31;
// Rows whose largest logit is in a bin below this one are searched whole: 512 bins further down NaN and -inf
// (past bin -8192) would be among those that are counted.
constexpr int kLowestBin = -7000;
constexpr int kMaxStrips = (int)(kSampleMaxVocab / kStrip);
constexpr int kList = 8192;                  // elements of a row's list
constexpr int kBatchRows = 256;              // rows of one launch

static_assert((int64_t)kPiece * kThreads >= kSampleMaxVocab && kSampleMaxVocab % kPiece == 0, "a row's pieces are one a thread");

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
// An element's place in the order, 0 for those that are never chosen: its logit's over `bits` bits of its
// index's complement, of a bf16 logit the half that its bits are in.
template <typename T>
struct OrderKeys {
    static constexpr int kLow = sizeof(T) == 2 ? 16 : 0;
    int bits;
    __device__ __forceinline__ explicit OrderKeys(int vocab) : bits(32 - __builtin_clz(vocab)) {}
    __device__ __forceinline__ u64 operator()(float v, int index) const {
        const uint32_t key = logit_key(v) >> kLow;
        return key ? (u64)key << bits | (uint32_t)((1 << bits) - 1 - index) : 0;
    }
    __device__ __forceinline__ float logit(u64 key) const {
        const uint32_t high = (uint32_t)(key >> bits);
        return key_logit(kLow && !(high & 0x8000u) ? high << kLow | 0xffffu : high << kLow);
    }
    // The least and the most that a logit's keys can be.
    __device__ __forceinline__ u64 least(float v) const { return (u64)(logit_key(v) >> kLow) << bits; }
    __device__ __forceinline__ u64 most(float v) const { return least(v) | ((1u << bits) - 1); }
    __device__ __forceinline__ int index(u64 key) const { return (1 << bits) - 1 - (int)((uint32_t)key & ((1u << bits) - 1)); }
};

// exp((v - top) / T) in units of 2^-40, downwards, c = log2(e) / T. The exponent is (v - s) c - (top - s) c, its
// parts kept apart: the whole number nearest to the fp32 product is the shift, what an fma leaves of the product
// past it, the product with c's second fp32 part and top's fraction add up to the fraction, whose power is the
// hardware's (1 ulp). s is 0, and top where the exponent at top is so large that its fraction would be lost:
// then v - top is exact for every v that has weight. Where top is infinite, so is each that has weight.
struct Weights {
    float s, c_high, c_low, shift0, fraction, infinite;

    __device__ __forceinline__ Weights(float top, double c) {
        double at = (double)top * c;
        s = 0.0f;
        if (!(__builtin_fabs(at) < (double)(1 << 21))) s = top, at = 0.0;
        c_high = (float)c;
        c_low = c_high < __builtin_inff() ? (float)(c - (double)c_high) : 0.0f;
        const double n = __builtin_rint(at);
        shift0 = (float)n + (float)(kShift);
        fraction = (float)(at - n);
        infinite = top == __builtin_inff() ? top : __builtin_nanf("");
    }
    // m 2^32 (m: 24 bits and the power's) moved down to m 2^(40 - 24) at the exponent 0, or 1 less where the
    // two whole numbers are rounded apart.
    static constexpr int kShift = 32 - (kWeightBits - 24);
    // 2^f. (Far below top f can be anything, and NaN for a NaN or -inf: none.)
    static __device__ __forceinline__ float power(float f) {
        return __builtin_fminf(__builtin_fmaxf(__builtin_amdgcn_exp2f(f), 0.0f), 4.0f);
    }
    __device__ __forceinline__ u64 operator()(float v) const {
#pragma clang fp contract(off)  // (n is the rounded product's)
        const float d = v - s, n = __builtin_rintf(d * c_high);
        const float f = __builtin_fmaf(d, c_high, -n) + __builtin_fmaf(d, c_low, -fraction);
        float e = power(f);
        e = v == infinite ? 0.5f : e;
        int shift = (int)(shift0 - n);
        shift = shift < kShift - 1 ? kShift - 1 : shift > 63 ? 63 : shift;  // (an infinite one's: the least)
        return (u64)(uint32_t)(e * 16777216.0f) << 32 >> shift;
    }
};

// The same as a number, 1 at top, for sums over a piece: 2^x of the fp32 product x = (v - top) c and, to first
// order, of what the product rounds off. Off by the power's last place and by v - top's half a one (2^-25 x).
// NaN and -inf weigh `none`, which is 0 for all but the largest T. top finite.
struct PieceWeights {
    float top, c_high, c_low, least, none;
    __device__ __forceinline__ PieceWeights(float top, double c)
        : top(top), c_high((float)c), c_low((float)(c - (double)c_high)) {
        // (Past it a weight is 0.)
        least = __builtin_fmaxf(-160.0f / c_high, -__FLT_MAX__);
        none = of(least);
    }
    __device__ __forceinline__ float of(float d) const {
#pragma clang fp contract(off)
        const float x = d * c_high, rest = __builtin_fmaf(d, c_low, __builtin_fmaf(d, c_high, -x));
        const float e = __builtin_amdgcn_exp2f(x);
        return __builtin_fmaf(e, rest * 0.6931471805599453f, e);
    }
    __device__ __forceinline__ float operator()(float v) const { return of(__builtin_fmaxf(v - top, least)); }
};

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

// The smallest value of a bin, to the rounding of 1 + |logit|.
__device__ __forceinline__ float bin_edge(int bin) {
    const int at = bin >= 0 ? bin : -bin;
    const float v = __uint_as_float((uint32_t)((at < 8192 ? at : 8192) + (127 << 6)) << 17) - 1.0f;
    return bin >= 0 ? v : -v;
}

// ---- across a workgroup ---------------------------------------------------------------------------
//
// Reductions and running sums over the lanes by DPP moves (a move within a row of 16, then its last lane to
// the rows after it), over the waves through LDS. Zero is neutral in all of them.

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_move(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_move(u64 v) {
    return (u64)dpp_move<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | dpp_move<CTRL, ROWS>((uint32_t)v);
}
__device__ __forceinline__ u64 lane_of(u64 v, int lane) {
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
struct MaxOp {
    template <typename V> __device__ V operator()(V a, V b) const { return a > b ? a : b; }
};
struct SumOp {
    template <typename V> __device__ V operator()(V a, V b) const { return a + b; }
};
// Over the lanes up to this one; lane 63 has the wave's.
template <typename V, typename F>
__device__ __forceinline__ V wave_scan(V v, F op) {
    v = op(v, dpp_move<0x111, 0xf>(v));
    v = op(v, dpp_move<0x112, 0xf>(v));
    v = op(v, dpp_move<0x114, 0xf>(v));
    v = op(v, dpp_move<0x118, 0xf>(v));
    v = op(v, dpp_move<0x142, 0xa>(v));
    v = op(v, dpp_move<0x143, 0xc>(v));
    return v;
}
template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, F op, u64 *scratch) {
    v = wave_scan(v, op);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) scratch[threadIdx.x >> 6] = (u64)v;
    __syncthreads();
    v = (V)scratch[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) v = op(v, (V)scratch[i]);
    return v;
}
// The sum over the threads up to this one.
__device__ __forceinline__ u64 block_scan(u64 v, u64 *scratch) {
    const int wave = threadIdx.x >> 6;
    v = wave_scan(v, SumOp());
    __syncthreads();
    if ((threadIdx.x & 63) == 63) scratch[wave] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves - 1; ++i)
        if (i < wave) v += scratch[i];
    return v;
}

// ---- what the launches leave for each other ---------------------------------------------------------

constexpr int kNoBin = -0x7fffffff;  // (as low_bin and above_bin: nothing goes to the list)
enum RowState : int { kSettled = 0, kCollect = 1, kSearch = 2 };

struct RowPlan {
    int state, above_bin, low_bin;  // the list takes the bins [low_bin, above_bin)
    uint32_t top_key;
    u64 total;         // the whole row's weight, of the largest logit
    uint32_t above;    // elements in the bins above the list's
    uint32_t listed;   // elements of the list so far
    uint32_t valid, reserved;  // valid: elements that can be chosen
    double c, low;     // log2(e) / T; log2(min_p), -inf where it is off
};
// A wave's strip of a piece.
struct Strip {
    u64 key;          // scan: its largest logit's
    u64 weight;       // scan: its weight, of its piece's largest logit
    u64 above, kept;  // collect: the weight above the list's bins, and of it what min-p leaves
};
struct RowScratch {
    RowPlan plan;
    // [pieces] its largest logit's key << 32 | the index of that (greedy rows); [pieces] elements that can be chosen;
    // [strips] Strip; [pieces][kBins] count << 32 | fp32 weight; [kList] the list.
    u64 heads[1];
};

struct SampleArgs {
    const void *logits;
    int64_t ld;
    int vocab, pieces;
    SampleParams p;
    uint32_t *tokens;
    float *logprobs;
    char *rows;
    size_t row_bytes;
};

__device__ __forceinline__ RowScratch &row_scratch(const SampleArgs &args, int r) {
    return *(RowScratch *)(args.rows + r * args.row_bytes);
}
__device__ __forceinline__ u64 *row_valid(const SampleArgs &args, RowScratch &row) { return row.heads + args.pieces; }
__device__ __forceinline__ Strip *row_strips(const SampleArgs &args, RowScratch &row) {
    return (Strip *)(row_valid(args, row) + args.pieces);
}
__device__ __forceinline__ u64 *row_bins(const SampleArgs &args, RowScratch &row) {
    return (u64 *)(row_strips(args, row) + args.pieces * kWaves);
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
};
__device__ __forceinline__ RowParams row_params(const SampleArgs &args, int64_t r) {
    const float t = args.p.temperature ? args.p.temperature[r] : 1.0f, p = args.p.top_p ? args.p.top_p[r] : 1.0f,
                q = args.p.min_p ? args.p.min_p[r] : 0.0f;
    const int k = args.p.top_k ? args.p.top_k[r] : 0;
    RowParams out;
    out.greedy = !args.p.uniforms || !(t > 0.0f);
    out.c = 1.4426950408889634074 / (double)(t > 0x1p-126f ? t : 0x1p-126f);  // (so that fp32 holds it)
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

// A thread's sixteen logits of the piece at `base`, -inf past the row's end; their indexes are base + index_of(e), a
// wave's a strip. Pieces are counted from the row's first element whatever its alignment, so that which elements
// share a sum does not depend on where the row lies: the 16-byte loads need no more than an element's alignment.
// (Whole pieces without a branch, so that every load is out before the first is waited for.)
template <typename T>
__device__ __forceinline__ int index_of(int e) {
    constexpr int kRun = 16 / (int)sizeof(T);
    return (int)(threadIdx.x >> 6) * kStrip + e / kRun * (64 * kRun) + (int)(threadIdx.x & 63) * kRun + e % kRun;
}
template <typename T>
__device__ __forceinline__ void load_piece(const T *row, int base, int vocab, float (&v)[kPer]) {
    constexpr int kRun = 16 / (int)sizeof(T);
    u32x4 w[kPer / kRun];
    const bool whole = base + kPiece <= vocab;
    if (whole) {
#pragma unroll
        for (int e = 0; e < kPer; e += kRun) __builtin_memcpy(&w[e / kRun], row + base + index_of<T>(e), 16);
    } else {
        constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
#pragma unroll
        for (int e = 0; e < kPer; e += kRun) {
            const int i = base + index_of<T>(e);
            w[e / kRun] = u32x4{kNone, kNone, kNone, kNone};
            if (i + kRun <= vocab) __builtin_memcpy(&w[e / kRun], row + i, 16);
        }
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const uint32_t word = w[e / kRun][e % kRun * sizeof(T) / 4];
        v[e] = sizeof(T) == 4 ? __uint_as_float(word) : bf16_bits_to_f32(e & 1 ? word >> 16 : word & 0xffffu);
    }
    if (!whole) {  // the part that the row ends in
#pragma unroll
        for (int e = 0; e < kPer; e += kRun) {
            const int i = base + index_of<T>(e);
            if (i < vocab && i + kRun > vocab) {
#pragma unroll
                for (int j = 0; j < kRun; ++j)
                    if (i + j < vocab) v[e + j] = logit_of(row[i + j]);
            }
        }
    }
}

struct Shared {
    u64 scratch[kWaves];
    int chosen;
    double fraction;
    u64 rest;
    int cuts[4];
    u64 weights[4];
};

// The strip the draw falls into, strips one after the other (weight_of(s) for s < strips): sh.chosen, and how far
// into its weight. Returns the whole weight.
template <typename F>
__device__ __forceinline__ u64 choose_strip(const F &weight_of, int strips, float u, Shared &sh) {
    const int each = (strips + kThreads - 1) / kThreads, first = (int)threadIdx.x * each;
    u64 mine = 0;
    for (int s = first; s < first + each && s < strips; ++s) mine += weight_of(s);
    if (threadIdx.x == 0) sh.chosen = 0, sh.fraction = 0.0;
    const u64 run = block_scan(mine, sh.scratch);
    u64 total = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) total += sh.scratch[i];
    const u64 target = draw_of(u, total);
    if (run > target && run - mine <= target) {
        u64 rest = target - (run - mine);
        int s = first;
        u64 w = weight_of(s);
        while (rest >= w) {
            rest -= w;
            w = weight_of(++s);
        }
        sh.chosen = s;
        sh.fraction = (double)rest / (double)w;
    }
    __syncthreads();
    return total;
}

// The token of the row: the first index of the strip whose running weight over the kept elements (order key
// >= cut, weight of the row's largest at least 2^low) exceeds `fraction` of the strip's. Its probability: its
// weight times scale.
template <typename T>
__device__ __forceinline__ void locate(const SampleArgs &args, int64_t r, const T *row, int strip, float top, double c,
                                       u64 cut, double low, double fraction, double scale, Shared &sh) {
    constexpr int kEach = kStrip / kThreads;
    const int first = strip * kStrip + (int)threadIdx.x * kEach;
    const Weights weigh(top, c);
    const OrderKeys<T> keys(args.vocab);
    float v[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e)
        v[e] = first + e < args.vocab ? logit_of(row[first + e]) : -__builtin_inff();
    u64 w[kEach], run = 0, total = 0;
    for (int pass = 0; pass < 2 && total == 0; ++pass) {  // (again, by number, where what is left is less than a unit each)
        u64 sum = 0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const u64 key = keys(v[e], first + e);
            w[e] = key && key >= cut && weighs(v[e], top, c, low) ? pass ? 1 : weigh(v[e]) : 0;
            sum += w[e];
        }
        run = block_scan(sum, sh.scratch) - sum;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) total += sh.scratch[i];
    }
    u64 target = (u64)(fraction * (double)total), found = 0;
    target = target < total ? target : total - 1;
    int at = 0;
    float logit = top;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        if (run <= target && target < run + w[e]) at = e, found = w[e], logit = v[e];
        run += w[e];
    }
    if (found) {
        args.tokens[r] = (uint32_t)(first + at);
        // (Below 2^24 units the weight's own unit would be seen in its logarithm: the exponent as it is.)
        constexpr double kLn2 = 0.693147180559945309417;
        const bool small = found >> 24 == 0 && logit != top;
        const double weight = small ? (double)((u64)1 << kWeightBits) : (double)found;
        const double power = small ? ((double)logit - (double)top) * c * kLn2 : 0.0;
        if (args.logprobs) args.logprobs[r] = (float)(power + log(weight * scale));
    }
}

// ---- scan -------------------------------------------------------------------------------------------
//
// Bound by its vector instructions beside the read: 35 an element with bins (an exponential at a quarter of the rate,
// an LDS atomic), 20 without. 64 rows of 248320: fp32 with bins 64 MB in 17-19 us (3.4-3.7 TB/s), greedy 11.8 (5.4),
// bf16 with the temperature alone 32 MB in 12.2 us (2.6 TB/s). 512 threads of sixteen logits each: with 256 or 1024 threads slower.

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_scan_kernel(SampleArgs args) {
    __shared__ u64 scratch[kWaves];
    __shared__ u64 bins[kBins];
    const int tid = threadIdx.x, piece = blockIdx.x;
    const int64_t r = blockIdx.y;
    const T *logits = (const T *)args.logits + r * args.ld;
    const int base = piece * kPiece;
    float v[kPer];
    load_piece(logits, base, args.vocab, v);
    const RowParams rp = row_params(args, r);
    const bool cut = !rp.greedy && (rp.k || rp.p < 1.0f);
    RowScratch &row = row_scratch(args, (int)r);
    if (cut) bins[tid] = 0;
    float best = -__builtin_inff();
#pragma unroll
    for (int e = 0; e < kPer; ++e) best = __builtin_fmaxf(best, __builtin_canonicalizef(v[e]));  // (a signalling NaN quiet)
    const uint32_t strip_key = wave_scan(logit_key(best), MaxOp());  // (in lane 63)
    const uint32_t best_key = block_reduce(logit_key(best), MaxOp(), scratch);
    const float top = key_logit(best_key);
    u64 index = 0, weight = 0;
    uint32_t valid = 0;
    if (rp.greedy) {
        uint32_t at = 0;  // (the complement: the first index is the largest)
#pragma unroll
        for (int e = kPer - 1; e >= 0; --e)
            if (v[e] == top) at = ~(uint32_t)(base + index_of<T>(e));
        index = ~block_reduce(at, MaxOp(), scratch);
    } else if (best_key) {
        if (rp.k) {
#pragma unroll
            for (int e = 0; e < kPer; ++e) valid += __builtin_popcountll(__ballot(v[e] > -__builtin_inff()));
        }
        // Where the largest is infinite, those that are have weight.
        const bool infinite = top == __builtin_inff();
        if (infinite) {
#pragma unroll
            for (int e = 0; e < kPer; ++e) v[e] = v[e] == top ? 0.0f : -__builtin_inff();
        }
        const PieceWeights weigh(infinite ? 0.0f : top, rp.c);
        // A lane's sixteen in fp32, the lanes in integers.
        float sum = 0.0f;
        if (cut) {
            const int top_bin = value_bin(top);
            if (top_bin >= kLowestBin - kBins && !infinite) {
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    const float w = weigh(v[e]);
                    sum += w;
                    const int below = top_bin - value_bin(v[e]);
                    if ((uint32_t)below < (uint32_t)kBins)
                        atomicAdd(&bins[below], (u64)1 << kBinShift | (uint32_t)__builtin_fmaf(w, (float)(1u << kBinBits), 0.5f));
                }
            } else {
#pragma unroll
                for (int e = 0; e < kPer; ++e) sum += weigh(v[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < kPer; ++e) sum += weigh(v[e]);
        }
        if (weigh.none > 0.0f) {  // (added up without them: taken off again, their rounding would be left)
            sum = 0.0f;
#pragma unroll
            for (int e = 0; e < kPer; ++e) sum += v[e] > -__builtin_inff() ? weigh(v[e]) : 0.0f;
        }
        weight = (u64)(sum * (float)((u64)1 << kWeightBits));
        if (rp.k) valid = block_reduce(tid & 63 ? 0u : valid, SumOp(), scratch);
    }
    if (!rp.greedy) {
        weight = wave_scan(weight, SumOp());
        if ((tid & 63) == 63) {
            Strip &strip = row_strips(args, row)[piece * kWaves + (tid >> 6)];
            strip.key = strip_key;
            strip.weight = weight;
        }
    }
    if (tid == 0) {
        row.heads[piece] = (u64)best_key << 32 | index;
        row_valid(args, row)[piece] = valid;
    }
    if (cut) {
        __syncthreads();
        const u64 entry = bins[tid];
        const float w = (float)((entry & (((u64)1 << kBinShift) - 1)) << (kWeightBits - kBinBits));
        row_bins(args, row)[(size_t)piece * kBins + tid] = entry >> kBinShift << 32 | __float_as_uint(w);
    }
}

// ---- settle -----------------------------------------------------------------------------------------
//
// Latency: the pieces' heads, then their bins (sixteen pieces at a time, 4 KB each), then scans over the workgroup;
// 6.4 us for one row of 31 pieces, 7.1 for 64. Loading the bins before the heads are known measured slower.
//
// Rows that are left to be searched whole (measured with vocabularies of 248320, normal logits with a deviation of 2):
//   - a share p that the bins cannot tell from the whole weight: p (1 + 2^-14) and half a bin's unit for each element
//     of the vocabulary exceed it; p from 0.9999 on, 0.9998 with a head of likely tokens;
//   - more than 8192 elements in the bins from the first that a cut can be in to the last that matters: equal logits;
//     the cuts of top-p and of a top-k of ten thousands far apart; and logits about a value far from 0, since the bins
//     are as wide as 1 + |logit| makes them: nuclei of p = 0.9 from an offset of 15 on, of 0.8 from 30 on;
//   - cuts more than 512 bins below the largest logit.

// 2^t for t <= 0, to the hardware's 2^-23.
__device__ __forceinline__ double power_of(double t) {
    const double n = __builtin_rint(t);
    return t > -1000.0 ? __builtin_ldexp((double)__builtin_amdgcn_exp2f((float)(t - n)), (int)n) : 0.0;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_settle_kernel(SampleArgs args) {
    __shared__ Shared sh;
    __shared__ double factors[kThreads];  // the pieces' weights in the row's
    __shared__ int top_bins[kThreads];
    const int tid = threadIdx.x, strips = args.pieces * kWaves;
    const int64_t r = blockIdx.x;
    const T *row = (const T *)args.logits + r * args.ld;
    RowScratch &scratch = row_scratch(args, (int)r);
    const RowParams rp = row_params(args, r);
    const bool cut = !rp.greedy && (rp.k || rp.p < 1.0f);
    // One piece a thread.
    const u64 head = tid < args.pieces ? scratch.heads[tid] : 0;
    const u64 piece_valid = tid < args.pieces ? row_valid(args, scratch)[tid] : 0;
    const u64 strip_weight = tid < strips ? row_strips(args, scratch)[tid].weight : 0;  // (the first 512)
    const uint32_t piece_key = (uint32_t)(head >> 32), top_key = block_reduce(piece_key, MaxOp(), sh.scratch);
    RowPlan &plan = scratch.plan;
    if (rp.greedy || top_key == 0) {
        // Of the pieces that have the largest, the first index.
        const uint32_t at = ~block_reduce(piece_key == top_key ? ~(uint32_t)head : 0u, MaxOp(), sh.scratch);
        if (tid == 0) {
            args.tokens[r] = top_key ? at : 0xffffffffu;
            if (args.logprobs) args.logprobs[r] = top_key ? 0.0f : -__builtin_inff();
            plan.state = kSettled;
        }
        return;
    }
    const float top = key_logit(top_key), piece_top = key_logit(piece_key);
    factors[tid] = piece_key == 0 ? 0.0
                   : piece_key == top_key ? 1.0 : power_of(((double)piece_top - (double)top) * rp.c);
    __syncthreads();
    const auto weight_of = [&](int s) {
        return (u64)((double)(s == tid ? strip_weight : row_strips(args, scratch)[s].weight) * factors[s / kWaves]);
    };
    if (!cut && rp.q == 0.0f) {  // the temperature alone
        const u64 total = choose_strip(weight_of, strips, rp.u, sh);
        const int piece = sh.chosen / kWaves;
        locate<T>(args, r, row, sh.chosen, key_logit((uint32_t)(scratch.heads[piece] >> 32)), rp.c, 1, -__builtin_inf(),
                  sh.fraction, factors[piece] / (double)total, sh);
        if (tid == 0) plan.state = kSettled;
        return;
    }
    u64 row_weight = 0;
    for (int s = tid; s < strips; s += kThreads) row_weight += weight_of(s);
    const u64 total = block_reduce(row_weight, SumOp(), sh.scratch);
    const u64 valid = rp.k ? block_reduce(piece_valid, SumOp(), sh.scratch) : 0;
    // The least (v - top) c of what min-p keeps.
    const double low = rp.q > 0.0f ? log2((double)rp.q) : -__builtin_inf();
    const bool by_count = rp.k && (u64)rp.k < valid, by_share = rp.p < 1.0f;
    if (!by_count && !by_share) {  // min-p alone, or with a k past what the row has: everything is above the list
        if (tid == 0) plan = {kCollect, kNoBin, kNoBin, top_key, total, 0, 0, (uint32_t)valid, 0, rp.c, low};
        return;
    }
    // The row's bins: thread j the j-th below that of its largest logit.
    const int top_bin = value_bin(top);
    constexpr int kNoPiece = -0x4000000;
    top_bins[tid] = piece_key ? value_bin(piece_top) : kNoPiece;
    if (tid < 4) sh.cuts[tid] = kBins;
    __syncthreads();
    // (Lane e has where piece first + e's bins begin and its weight in the row's: a load and its use take a few
    // instructions, and a bin above the piece's own is out of the descriptor's range: zero.)
    const rsrc_t bins = make_rsrc(row_bins(args, scratch), (uint32_t)args.pieces * kBins * sizeof(u64));
    uint32_t count = 0;
    float bin_weight = 0.0f;
    constexpr int kAtOnce = 16;  // (eight: 7.4 us for one row, 32: 6.4 and with four pieces 7.2 for 6.1)
    for (int first = 0; first < args.pieces; first += kAtOnce) {
        const int piece = first + (tid & (kAtOnce - 1));
        const int from = (piece < args.pieces ? top_bins[piece] : kNoPiece) - top_bin;
        const uint32_t factor = __float_as_uint((float)factors[piece & (kThreads - 1)]);
        u32x2 entry[kAtOnce];
#pragma unroll
        for (int e = 0; e < kAtOnce; ++e)
            entry[e] = __builtin_amdgcn_raw_buffer_load_b64(bins, (tid + __builtin_amdgcn_readlane(from, e)) * 8,
                                                            (first + e < args.pieces ? first + e : 0) * kBins * 8, 0);
        __builtin_amdgcn_sched_barrier(0);  // (every load out before the first is waited for)
#pragma unroll
        for (int e = 0; e < kAtOnce; ++e) {
            count += entry[e].y;
            bin_weight = __builtin_fmaf(__uint_as_float(entry[e].x),
                                        __uint_as_float(__builtin_amdgcn_readlane(factor, e)), bin_weight);
        }
    }
    const u64 own_weight = (u64)bin_weight, run_count = block_scan(count, sh.scratch),
              run_weight = block_scan(own_weight, sh.scratch);
    // cuts: the bin of the k-th element, and those between which the run ends that has the share p.
    if (by_count && run_count >= (u64)rp.k && run_count - count < (u64)rp.k) {
        sh.cuts[0] = tid;
        sh.weights[0] = run_weight - own_weight;
        sh.weights[1] = run_weight;
    }
    __syncthreads();
    if (by_share && (!by_count || sh.cuts[0] < kBins)) {
        // (The bins' weights are fp32 sums of one product a piece: 2^-19 for a row of 32, 2^-15 for one of 512;
        // and of elements rounded to their units.)
        constexpr double kSlack = 1.0 / (1 << 14);
        const double rounding = (double)args.vocab * (double)((u64)1 << (kWeightBits - kBinBits - 1));
        const double least = (double)rp.p * (double)(by_count ? sh.weights[0] : total) * (1.0 - kSlack) - rounding;
        const double most = (double)rp.p * (double)(by_count ? sh.weights[1] : total) * (1.0 + kSlack) + rounding;
        const double before = (double)(run_weight - own_weight);
        if (count && (double)run_weight >= least && (before < least || run_count == count)) sh.cuts[1] = tid;
        if (count && (double)run_weight >= most && (before < most || run_count == count)) sh.cuts[2] = tid;
    }
    __syncthreads();
    // The list: from the first bin that the cut can be in to the last that matters.
    const int from = by_share ? sh.cuts[1] : sh.cuts[0], to = by_count ? sh.cuts[0] : sh.cuts[2];
    if (tid == from) sh.weights[2] = run_count - count;
    if (tid == to) sh.weights[3] = run_count;
    __syncthreads();
    if (tid == 0) {
        const bool fits = from < kBins && to < kBins && top_bin >= kLowestBin && top < __builtin_inff() &&
                          sh.weights[3] - sh.weights[2] <= kList;
        plan = {fits ? kCollect : kSearch, top_bin - from + 1, top_bin - to, top_key, total,
                fits ? (uint32_t)sh.weights[2] : 0, 0, (uint32_t)valid, 0, rp.c, low};
    }
}

// ---- collect ----------------------------------------------------------------------------------------
//
// Reads again what can be above the list or in it, strip by strip: nothing but the strips' records for rows that are
// settled, few strips for rows with a peaked head (64 rows of 248320 fp32: 14 of 64 MB, 7.4 us), all of a flat row's
// (16 of 100003 bf16 with top-p: 7.5 us).

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_collect_kernel(SampleArgs args) {
    const int piece = blockIdx.x, lane = threadIdx.x & 63;
    const int64_t r = blockIdx.y;
    RowScratch &row = row_scratch(args, (int)r);
    const RowPlan &plan = row.plan;
    Strip &strip = row_strips(args, row)[piece * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)];
    const int state = plan.state, low_bin = plan.low_bin, above_bin = plan.above_bin;
    const uint32_t strip_key = (uint32_t)strip.key;
    const float top = key_logit(plan.top_key), strip_top = key_logit(strip_key);
    const double c = plan.c, low = plan.low;
    if (state != kCollect) return;
    u64 above = 0, kept = 0;
    // (A strip whose largest is below the list's bins, or below min-p with no list, has nothing to give.)
    const bool listing = low_bin != kNoBin;
    if (strip_key && value_bin(strip_top) >= low_bin && (listing || weighs(strip_top, top, c, low))) {
        const Weights weigh(top, c);
        const T *logits = (const T *)args.logits + r * args.ld;
        const int base = piece * kPiece;
        float v[kPer];
        load_piece(logits, base, args.vocab, v);
        uint32_t listed = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const int bin = value_bin(v[e]);
            if (v[e] > -__builtin_inff() && bin >= low_bin) {
                if (bin >= above_bin) {
                    const bool keep = weighs(v[e], top, c, low);
                    if (keep || listing) {
                        const u64 w = weigh(v[e]);
                        above += w;
                        kept += keep ? w : 0;
                    }
                } else {
                    listed |= 1u << e;
                }
            }
        }
        // Places in the row's list, a wave at a time.
        if (__ballot(listed != 0)) {
            const uint32_t mine = __builtin_popcount(listed), run = wave_scan(mine, SumOp());
            uint32_t at = 0;
            if (lane == 63)
                at = __hip_atomic_fetch_add(&row.plan.listed, run, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            at = __builtin_amdgcn_readlane(at, 63) + run - mine;
            u64 *list = row_list(args, row);
            const OrderKeys<T> keys(args.vocab);
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                if (listed >> e & 1) {
                    if (at < kList) list[at] = keys(v[e], base + index_of<T>(e));
                    ++at;
                }
        }
        above = wave_scan(above, SumOp());
        kept = wave_scan(kept, SumOp());
    }
    if (lane == 63) {
        strip.above = above;
        strip.kept = kept;
    }
}

// ---- finish -----------------------------------------------------------------------------------------
//
// Latency: the plan, the list, the cut, the strip. A list of up to 64 keys, of most rows with a peaked head, is
// ranked at once (4.8 us a row; by digits 7.3); a longer one is searched by digits, and up to 64 keys that share one
// are ranked by one wave, which saves the steps below it (9.5 us with lists of hundreds).

// A step of the search for a cut among keys: how many there are with each digit of nine bits, and their weight.
struct Digits {
    u64 prefix, above;  // the bits above the digit, and where they are
    int shift;
    u64 base_count;     // elements before all of them
    // Of this thread's digit (the largest in thread 0): its elements and weight, and with those before.
    u64 count, weight, run_count, run_weight;
};
constexpr int kDigitBits = 9, kFew = 64;
static_assert(1 << kDigitBits == kThreads, "a digit a thread");

// The keys are those of a source, key(i) for i < n, from `limit` on (limit >= 1; a key of 0 is none).
template <typename Source, typename Keys>
__device__ __forceinline__ void count_digits(Digits &d, const Source &key_at, int n, const Keys &keys, const Weights &weigh,
                                             u64 limit, u64 base_count, u64 base_weight, u64 *memory, Shared &sh) {
    const int tid = threadIdx.x;
    u64 *counts = memory, *sums = memory + kThreads;
    __syncthreads();
    counts[tid] = 0;
    sums[tid] = 0;
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < n; i += kThreads) {
        const u64 key = key_at(i);
        if (key < limit || ((key ^ d.prefix) & d.above)) continue;
        const int digit = (int)((key & ~d.above) >> d.shift);
        atomicAdd(&counts[digit], (u64)1);
        atomicAdd(&sums[digit], weigh(keys.logit(key)));
    }
    __syncthreads();
    d.base_count = base_count;
    d.count = counts[kThreads - 1 - tid];
    d.weight = sums[kThreads - 1 - tid];
    d.run_count = base_count + block_scan(d.count, sh.scratch);
    d.run_weight = base_weight + block_scan(d.weight, sh.scratch);
}

// The smallest run from the start of the order with `k` elements, or with weight >= share where k is 0: its last
// key, of those >= limit; *weight its weight. `d`: the first step. Where rounding has what comes before the keys
// reach the share already, the first key. Where no run reaches it (the pieces' weights, of which it is a share, hold
// more of those below a unit of the row's), 0.
template <typename Source, typename Keys>
__device__ __forceinline__ u64 find_cut(Digits d, const Source &key_at, int n, const Keys &keys, const Weights &weigh, u64 limit,
                                        u64 k, double share, u64 *weight, u64 *memory, Shared &sh) {
    const int tid = threadIdx.x;
    const auto ends = [&](u64 count, u64 sum) { return k ? count >= k : (double)sum >= share; };
    u64 *few = memory;
    for (;;) {
        const u64 count_before = d.run_count - d.count, weight_before = d.run_weight - d.weight;
        if (d.count && ends(d.run_count, d.run_weight) &&
            (count_before == d.base_count || !ends(count_before, weight_before))) {
            sh.cuts[0] = kThreads - 1 - tid;
            sh.weights[0] = count_before;
            sh.weights[1] = weight_before;
            sh.weights[2] = d.run_weight;
            sh.weights[3] = d.count;
        }
        if (tid == 0) sh.cuts[1] = 0;
        __syncthreads();
        if (sh.cuts[0] < 0) return 0;
        const u64 base_count = sh.weights[0], base_weight = sh.weights[1], inside = sh.weights[3];
        d.prefix |= (u64)(uint32_t)sh.cuts[0] << d.shift;
        d.above = ~(u64)0 << d.shift;
        if (d.shift == 0) {
            *weight = sh.weights[2];
            return d.prefix;
        }
        if (inside <= kFew) break;
        d.shift = d.shift < kDigitBits ? 0 : d.shift - kDigitBits;
        count_digits(d, key_at, n, keys, weigh, limit, base_count, base_weight, memory, sh);
    }
    // A wave's worth of keys: each lane counts what comes before its own.
    const u64 base_count = sh.weights[0], base_weight = sh.weights[1];
#pragma unroll 4
    for (int i = tid; i < n; i += kThreads) {
        const u64 key = key_at(i);
        if (key >= limit && ((key ^ d.prefix) & d.above) == 0) {
            const int at = atomicAdd(&sh.cuts[1], 1);
            if (at < kFew) few[at] = key;
        }
    }
    __syncthreads();
    if (tid < 64) {
        const int m = sh.cuts[1] < kFew ? sh.cuts[1] : kFew;
        const u64 key = tid < m ? few[tid] : 0, own = tid < m ? weigh(keys.logit(key)) : 0;
        u64 count = base_count + 1, sum = base_weight + own;
        for (int i = 0; i < m; ++i) {
            const u64 other = few[i], w = lane_of(own, i);
            if (other > key) ++count, sum += w;
        }
        if (tid < m && ends(count, sum) && (count == base_count + 1 || !ends(count - 1, sum - own))) {
            sh.rest = key;
            sh.weights[2] = sum;
        }
    }
    __syncthreads();
    *weight = sh.weights[2];
    return sh.rest;
}

// The cuts of top-k and, among its elements, of top-p; the keys lie in [least, most], after `base_weight`.
template <typename Source, typename Keys>
__device__ __forceinline__ u64 find_cuts(const Source &key_at, int n, const Keys &keys, u64 least, u64 most,
                                         const Weights &weigh, const RowPlan &plan, const RowParams &rp, u64 base_weight,
                                         u64 *memory, Shared &sh) {
    const bool by_count = rp.k && (uint32_t)rp.k < plan.valid, by_share = rp.p < 1.0f;
    u64 cut = 1, weight = plan.total;
    if (!by_count && !by_share) return cut;
    const int top_bit = 63 - __builtin_clzll(most ^ least);
    Digits d;
    d.shift = top_bit < kDigitBits ? 0 : top_bit - kDigitBits + 1;
    d.above = ~(u64)0 << top_bit << 1;
    d.prefix = most & d.above;
    if (threadIdx.x == 0) sh.cuts[0] = -1;
    count_digits(d, key_at, n, keys, weigh, cut, plan.above, base_weight, memory, sh);
    for (int pass = 0; pass < 2; ++pass) {
        if (pass ? !by_share : !by_count) continue;
        cut = find_cut(d, key_at, n, keys, weigh, cut, pass ? 0 : (u64)rp.k, (double)rp.p * (double)weight, &weight, memory, sh);
        __syncthreads();  // (every wave has read its results in sh, which the next one writes before a barrier of its own)
    }
    return cut;
}

// The same for a list of no more keys than a wave has lanes, lane i the i-th, in every wave: each wave counts what an
// eighth of them adds before each key, and all add the eighths up. `above`: this thread's part of the weight above
// the list's bins.
__device__ __forceinline__ u64 rank_few(u64 key, u64 own, int n, u64 above, const RowPlan &plan, const RowParams &rp,
                                        u64 *memory, Shared &sh) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    u64 count = 0, sum = 0;
    for (int i = wave; i < n; i += kWaves) {
        const u64 other = lane_of(key, i), w = lane_of(own, i);  // (of lanes that the branch may leave out: before it)
        if (other > key) ++count, sum += w;
    }
    memory[threadIdx.x] = sum;
    memory[kThreads + threadIdx.x] = count;
    above = wave_scan(above, SumOp());
    if (lane == 63) sh.scratch[wave] = above;
    __syncthreads();
    count = plan.above + 1;
    sum = own;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        sum += memory[w * 64 + lane] + sh.scratch[w];
        count += memory[kThreads + w * 64 + lane];
    }
    const bool any = lane < n;
    u64 cut = 1, weight = plan.total, hit;
    if (rp.k && (uint32_t)rp.k < plan.valid && (hit = __ballot(any && count == (u64)rp.k))) {
        cut = lane_of(key, __builtin_ctzll(hit));
        weight = lane_of(sum, __builtin_ctzll(hit));
    }
    if (rp.p < 1.0f) {
        const double share = (double)rp.p * (double)weight;
        hit = __ballot(any && (double)sum >= share && (count == plan.above + 1 || (double)(sum - own) < share));
        if (!hit) hit = __ballot(any && count == (u64)plan.above + n);  // (no run reaches it: the whole list)
        const u64 last = hit ? lane_of(key, __builtin_ctzll(hit)) : 1;
        cut = last > cut ? last : cut;
    }
    return cut;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_finish_kernel(SampleArgs args) {
    __shared__ Shared sh;
    __shared__ u64 list[kList], memory[2 * kThreads], extra[kMaxStrips];
    const int tid = threadIdx.x, strips = args.pieces * kWaves;
    const int64_t r = blockIdx.x;
    RowScratch &scratch = row_scratch(args, (int)r);
    const RowPlan plan = scratch.plan;
    const Strip *of = row_strips(args, scratch);
    const u64 strip_kept = tid < strips ? of[tid].kept : 0;  // (the first 512)
    u64 above = tid < strips ? of[tid].above : 0;
    const u64 early = row_list(args, scratch)[tid & 63];  // (before it is known how many there are)
    if (plan.state == kSettled) return;
    const T *row = (const T *)args.logits + r * args.ld;
    const RowParams rp = row_params(args, r);
    const float top = key_logit(plan.top_key);
    const double c = plan.c, low = plan.low;
    const Weights weigh(top, c);
    const OrderKeys<T> keys(args.vocab);
    u64 cut = 1;
    const bool listed = plan.state == kCollect;
    const int n = listed ? plan.listed < (uint32_t)kList ? (int)plan.listed : kList : 0;
    for (int s = tid; s < strips; s += kThreads) extra[s] = 0;
    if (n)
        for (int s = tid + kThreads; s < strips; s += kThreads) above += of[s].above;
    const bool few = listed && n <= kFew;
    if (few) {
        if (n) {
            const bool any = (tid & 63) < n;
            const float v = keys.logit(early);
            const u64 own = any ? weigh(v) : 0;
            cut = rank_few(any ? early : 0, own, n, above, plan, rp, memory, sh);
            if (tid < n && early >= cut && weighs(v, top, c, low)) atomicAdd(&extra[keys.index(early) / kStrip], own);
        }
    } else if (n) {
        const u64 *from = row_list(args, scratch);
        for (int i = tid; i < n; i += kThreads) list[i] = from[i];
        const u64 base_weight = block_reduce(above, SumOp(), sh.scratch);
        cut = find_cuts([&](int i) { return list[i]; }, n, keys, keys.least(bin_edge(plan.low_bin - 1)),
                        keys.most(bin_edge(plan.above_bin + 1)), weigh, plan, rp, base_weight, memory, sh);
        if (cut == 0) {  // the whole list
            u64 last = 0;  // (the complement)
            for (int i = tid; i < n; i += kThreads) last = last > ~list[i] ? last : ~list[i];
            cut = ~block_reduce(last, MaxOp(), sh.scratch);
        }
    } else {
        cut = find_cuts([&](int i) { return keys(logit_of(row[i]), i); }, args.vocab, keys, 0, keys.most(__builtin_inff()),
                        weigh, plan, rp, 0, memory, sh);
        cut = cut ? cut : 1;
    }
    // What min-p leaves of the kept elements of the list, or of the row, to their strips.
    __syncthreads();
    for (int i = tid; i < (few ? 0 : listed ? n : args.vocab); i += kThreads) {
        const u64 key = listed ? list[i] : keys(logit_of(row[i]), i);
        const float v = keys.logit(key);
        if (key >= cut && weighs(v, top, c, low)) atomicAdd(&extra[keys.index(key) / kStrip], weigh(v));
    }
    __syncthreads();
    const u64 total = choose_strip(
        [&](int s) { return extra[s] + (!listed ? 0 : s == tid ? strip_kept : of[s].kept); }, strips, rp.u, sh);
    locate<T>(args, r, row, sh.chosen, top, c, cut, low, sh.fraction, 1.0 / (double)total, sh);
}

// ---- host -------------------------------------------------------------------------------------------

static int64_t pieces_of(int64_t vocab) { return (vocab + kPiece - 1) / kPiece; }
static size_t row_bytes(int64_t vocab) {
    const int64_t pieces = pieces_of(vocab);
    const size_t bytes = sizeof(RowPlan) + pieces * (2 * sizeof(u64) + kWaves * sizeof(Strip) + kBins * sizeof(u64)) +
                         kList * sizeof(u64);
    return (bytes + 255) / 256 * 256;
}

size_t sample_workspace_bytes(int64_t rows, int64_t vocab) {
    return kSampleCounterBytes + (size_t)(rows < kBatchRows ? rows : kBatchRows) * row_bytes(vocab);
}

template <typename T>
static void launch_batch(const SampleArgs &args, int rows, hipStream_t stream) {
    const dim3 pieces((unsigned)args.pieces, (unsigned)rows), whole((unsigned)rows);
    hipLaunchKernelGGL(sample_scan_kernel<T>, pieces, dim3(kThreads), 0, stream, args);
    hipLaunchKernelGGL(sample_settle_kernel<T>, whole, dim3(kThreads), 0, stream, args);
    if (!args.p.uniforms || (!args.p.top_k && !args.p.top_p && !args.p.min_p)) return;  // every row is settled
    hipLaunchKernelGGL(sample_collect_kernel<T>, pieces, dim3(kThreads), 0, stream, args);
    hipLaunchKernelGGL(sample_finish_kernel<T>, whole, dim3(kThreads), 0, stream, args);
}

hipError_t launch_sample(const void *logits, int64_t ld, int dtype, int64_t rows, int64_t vocab,
                         const SampleParams &params, uint32_t *tokens, float *logprobs, void *workspace,
                         hipStream_t stream) {
    const int64_t esize = dtype == SPLOSH_F32 ? 4 : 2;
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
        args.rows = (char *)workspace + kSampleCounterBytes;
        args.row_bytes = row_bytes(vocab);
        if (dtype == SPLOSH_F32) launch_batch<float>(args, count, stream);
        else launch_batch<uint16_t>(args, count, stream);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

}  // namespace splosh
