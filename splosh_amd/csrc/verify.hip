// verify.hip -- drafted tokens against the target's probabilities.
//
// A drafted token t is accepted if u q(t) < p(t); where one is not, the next token comes from max(p - q, 0). What has
// to move is the step's logits, once, for the maximum and sum of each row's softmax; of each request one row more of
// logits and draft for the new token. All that decides between two tokens is in 64-bit floating point, added in an
// order that the shape alone gives: the neighbours of a draw on a vocabulary of 250000 lie 4e-6 of the weight apart on average, and
// the sums that lead there are off by as much in fp32.
//
// Three launches; a workgroup takes a piece of 4096 entries of a row, or a request:
//   scan   (pieces of every row)         the piece's largest entry and the weight of its entries against it;
//   rest   (pieces of every request's row) which row ends the request's accepted run, from the pieces' numbers and one
//          probability a row, and the weights max(p - q, 0) and p of that row by strips of 512;
//   finish (requests)                    the strip that the draw falls into, and the token in it.
#include <climits>

#include "cache.hpp"
#include "launch.hpp"

namespace splosh {

constexpr size_t kVerifyCounterBytes = 16384;  // the workspace's first bytes belong to other kernels' counters
constexpr int kThreads = 512, kWaves = kThreads / 64, kPer = 8;  // of the workgroup for a piece of a request's row
constexpr int kStrip = 64 * kPer, kPiece = kThreads * kPer;
// The scan has sixteen entries a thread, so half the threads: 64 rows of 248320 fp32 16.9 us (512 threads of sixteen 18.3, of eight 21.3), where
// the one row a request, mostly round trips, is 9.0 us with eight a thread (sixteen: 9.6, 256 threads of sixteen 11.5).
constexpr int kScanPer = 16, kScanThreads = kPiece / kScanPer, kScanWaves = kScanThreads / 64;

struct PieceStats {
    double sum;
    float most;
    int first;  // the first entry of that value
};
struct Decision {
    int row, last, top;  // the row that ends the accepted run, whether it is the request's last, its first largest entry
    float most;
    double total, by;    // the row's weight; log2(e) / T, 0: greedy
};
struct StripSums {
    double rest, whole;
};

struct VerifyArgs {
    const void *logits;
    int64_t ld;
    int vocab, pieces, requests, rows;
    const int32_t *tokens, *starts;
    const float *uniforms, *temperature;
    const void *draft;
    int64_t ld_draft;
    int draft_f32;
    int32_t *out, *accepted;
    PieceStats *stats;
    Decision *decisions;
    StripSums *strips;
};

// 2^(j / 64): each thread below 64 puts one into LDS.
constexpr int kSteps = 64;
__constant__ const double kPowers[kSteps] = {
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284, 1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418, 1.1387886347566916, 1.1511892299529827, 1.1637248587775775,
    1.1763969916502812, 1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687, 1.241857812073484, 1.255380757024691,
    1.2690509571917332, 1.2828700160787783, 1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303, 1.3542555469368927,
    1.3690024229745905, 1.383909881963832, 1.3989796725383112, 1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384, 1.5422108254079407, 1.559004400237837, 1.5759808451078865,
    1.593142151342267, 1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364, 1.681792830507429, 1.7001063537185235,
    1.718619298122478, 1.7373338352737062, 1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989, 1.8340080864093424,
    1.8539791250833855, 1.8741676341103, 1.8945759815869656, 1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951};

// 2^(x / 64), x <= 0, to 1e-13 of it: x is a whole number and a rest |r| <= 1/2; of the whole number the last six bits are looked up and the
// others are the exponent, and of the rest comes the series in r ln 2 / 64 (the fifth power left out by 4e-14). Borders between tokens lie
// close: with the entries of a draw good to 1e-9, one draw of 8000 over 248320 of them could fall to another token than in 64 bits.
__device__ __forceinline__ double power2(double x, const double *powers) {
    x = __builtin_fmax(x, -128000.0);  // (0 from 2^-1075 on)
    const double shifted = x + 0x1.8p52, r = x - (shifted - 0x1.8p52);  // (the low bits of `shifted` are the whole number)
    const int whole = (int)(uint32_t)__double_as_longlong(shifted);
    const double e = r * __builtin_fma(__builtin_fma(__builtin_fma(5.732851688640402e-10, r, 2.1173137155464776e-07), r, 5.86490495505617e-05), r, 0.010830424696249145);
    const double power = powers[whole & (kSteps - 1)];
    return __builtin_ldexp(__builtin_fma(power, e, power), whole >> 6);
}

// 2^x, x <= 0, to 1e-9 of it, for the sums of the scan, whose errors even out: the whole part as the exponent, and of the fraction (|f| <= 1/2)
// the series in f ln 2, from the third power on in fp32 (that part is below 0.008: off by 5e-10 at most, where it ends with the eighth
// power by 2e-10). 64 rows of 248320 fp32 take 16.9 us so, 19.0 with the function above.
__device__ __forceinline__ double power2_near(double x) {
    x = __builtin_fmax(x, -2000.0);  // (0 from 2^-1075 on)
    const double n = __builtin_rint(x), f = x - n;
    const float g = (float)f;
    float h = 1.3215487e-6f;
    h = __builtin_fmaf(h, g, 1.5252734e-5f);
    h = __builtin_fmaf(h, g, 1.5403530e-4f);
    h = __builtin_fmaf(h, g, 1.3333558e-3f);
    h = __builtin_fmaf(h, g, 9.6181291e-3f);
    h = __builtin_fmaf(h, g, 5.5504109e-2f);
    const double e = __builtin_fma(__builtin_fma(__builtin_fma((double)h, f, 0.24022650695910072), f, 0.6931471805599453), f, 1.0);
    return __builtin_ldexp(e, (int)n);
}

// log2(e) / T; 0 where T asks for the largest entry.
__device__ __forceinline__ double factor_of(const float *temperature, int request) {
    const float t = temperature ? temperature[request] : 1.0f;
    // (An infinite T: all entries alike.)
    return t > 0.0f ? __builtin_fmax(1.4426950408889634 / (double)__builtin_fmaxf(t, 1.1754944e-38f), 1e-300) : 0.0;
}

// The weight of an entry against the largest, `most`; `first`: whether it is the first of that value.
__device__ __forceinline__ double weight_of(float v, float most, double by, bool first, const double *powers) {
    if (!(v > -__builtin_inff())) return 0.0;  // (NaN and -inf)
    if (by == 0.0) return first ? 1.0 : 0.0;
    if (v == most) return 1.0;
    return most == __builtin_inff() ? 0.0 : power2(((double)v - (double)most) * (kSteps * by), powers);
}

// Four entries in a row, of a row of any alignment, the first `here` of which are its.
struct __attribute__((packed, aligned(4))) Four32 {
    float v[4];
};
struct __attribute__((packed, aligned(2))) Four16 {
    uint16_t v[4];
};
__device__ __forceinline__ void entries(const float *p, int here, float (&v)[4]) {
    if (here >= 4) {
        const Four32 x = *reinterpret_cast<const Four32 *>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = x.v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = e < here ? p[e] : -__builtin_inff();
    }
}
__device__ __forceinline__ void entries(const uint16_t *p, int here, float (&v)[4]) {
    if (here >= 4) {
        const Four16 x = *reinterpret_cast<const Four16 *>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = bf16_bits_to_f32(x.v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = e < here ? bf16_bits_to_f32(p[e]) : -__builtin_inff();
    }
}

// The weights of N entries in fours from index `first` on, `step` further the next four. With a finite `most` and a T, NaN and -inf go the way of
// what is far below it: 2^-2000.
template <int N, bool NEAR>
__device__ __forceinline__ void weights_of(const float (&v)[N / 4][4], float most, double by, int first, int step, int top, const double *powers, double (&w)[N]) {
    if (by > 0.0 && __builtin_fabsf(most) < __builtin_inff()) {
#pragma unroll
        for (int k = 0; k < N / 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double x = (double)v[k][e] - (double)most;
                w[4 * k + e] = NEAR ? power2_near(x * by) : power2(x * (kSteps * by), powers);
            }
    } else {
#pragma unroll
        for (int k = 0; k < N / 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool one = by == 0.0 ? first + k * step + e == top : v[k][e] == most;
                w[4 * k + e] = one && v[k][e] > -__builtin_inff() ? 1.0 : 0.0;
            }
    }
}

__device__ __forceinline__ float entry(const float *p) { return *p; }
__device__ __forceinline__ float entry(const uint16_t *p) { return bf16_bits_to_f32(*p); }

// (v, i): the larger value, of equal ones the lower index. NaN is no value.
__device__ __forceinline__ void keep_first(float &v, int &i, float w, int j) {
    if (w > v || (w == v && j < i)) v = w, i = j;
}

template <typename T>
__global__ __launch_bounds__(kScanThreads) void scan_kernel(VerifyArgs a) {
    __shared__ float wave_most[kScanWaves];
    __shared__ int wave_first[kScanWaves];
    __shared__ double wave_total[kScanWaves];
    const int row = blockIdx.y, piece = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int r = request_of(a.starts, a.requests, row);
    if (r < 0) return;
    const T *logits = (const T *)a.logits + row * a.ld;
    const int begin = piece * kPiece + wave * 64 * kScanPer + lane * 4;  // its entries: four in a row, 256 further the next four
    float v[kScanPer / 4][4], most = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < kScanPer / 4; ++k) entries(logits + begin + 256 * k, a.vocab - begin - 256 * k, v[k]);
#pragma unroll
    for (int k = 0; k < kScanPer / 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) most = __builtin_fmaxf(most, v[k][e]);
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) most = __builtin_fmaxf(most, __shfl_xor(most, m));
    if (lane == 0) wave_most[wave] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kScanWaves; ++w) most = __builtin_fmaxf(most, wave_most[w]);
    int first = INT_MAX;
#pragma unroll
    for (int k = 0; k < kScanPer / 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) first = min(first, v[k][e] == most ? begin + 256 * k + e : INT_MAX);
    const double by = factor_of(a.temperature, r);
    double sum = 0.0, w[kScanPer];
    // (Of a greedy row any one entry of the largest value stands for the piece: its first is found below.)
    if (by > 0.0) {
        weights_of<kScanPer, true>(v, most, by, begin, 256, -1, nullptr, w);
#pragma unroll
        for (int e = 0; e < kScanPer; ++e) sum += w[e];
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m), first = min(first, __shfl_xor(first, m));
    if (lane == 0) wave_first[wave] = first;
    if (lane == 0) wave_total[wave] = sum;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kScanWaves; ++w) sum += wave_total[w], first = min(first, wave_first[w]);
        if (by == 0.0) sum = most > -__builtin_inff() ? 1.0 : 0.0;
        a.stats[(int64_t)row * a.pieces + piece] = {sum, most, first};
    }
}

// The whole row from its pieces, by one wave: the largest entry, the first of that value, and the weight against it.
__device__ __forceinline__ PieceStats row_stats(const VerifyArgs &a, int row, double by, const double *powers) {
    const int lane = threadIdx.x & 63;
    const PieceStats *stats = a.stats + (int64_t)row * a.pieces;
    float most = -__builtin_inff();
    int first = INT_MAX;
    for (int i = lane; i < a.pieces; i += 64) keep_first(most, first, stats[i].most, stats[i].first);
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) keep_first(most, first, __shfl_xor(most, m), __shfl_xor(first, m));
    double sum = 0.0;
    for (int i = lane; i < a.pieces; i += 64) sum += stats[i].sum * weight_of(stats[i].most, most, by, stats[i].first == first, powers);
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m);
    return {sum, most, first};
}

__device__ __forceinline__ double draft_of(const VerifyArgs &a, int row, int token, int drafted) {
    if (!a.draft) return token == drafted ? 1.0 : 0.0;
    const int64_t at = row * a.ld_draft + token;
    return a.draft_f32 ? ((const float *)a.draft)[at] : bf16_bits_to_f32(((const uint16_t *)a.draft)[at]);
}

// u of a row: below 0 or NaN as 0.
__device__ __forceinline__ double uniform_of(const VerifyArgs &a, int row) { return __builtin_fmax((double)a.uniforms[row], 0.0); }

// (weight of max(p - q, 0), of p) of N entries of the decided row from `token` on, four in a row and `step` further the next four.
template <typename T, int N>
__device__ __forceinline__ void rests_of(const VerifyArgs &a, const Decision &d, int drafted, int token, int step, const double *powers, StripSums (&w)[N]) {
    float v[N / 4][4], q[N / 4][4];
    const T *logits = (const T *)a.logits + d.row * a.ld;
    const bool whole = d.last || !a.draft;
#pragma unroll
    for (int k = 0; k < N / 4; ++k) entries(logits + token + k * step, a.vocab - token - k * step, v[k]);
    if (!whole) {
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
            const int64_t at = d.row * a.ld_draft + token + k * step;
            if (a.draft_f32) entries((const float *)a.draft + at, a.vocab - token - k * step, q[k]);
            else entries((const uint16_t *)a.draft + at, a.vocab - token - k * step, q[k]);
        }
    }
    const double inv = d.total > 0.0 ? 1.0 / d.total : 0.0;
    double weight[N];
    weights_of<N, false>(v, d.most, d.by, token, step, d.top, powers, weight);
#pragma unroll
    for (int k = 0; k < N / 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = token + k * step + e;
            const double p = weight[4 * k + e] * inv;
            const double taken = d.last ? 0.0 : !a.draft ? (i == drafted ? 1.0 : 0.0) : (double)q[k][e];
            w[4 * k + e] = {p > 0.0 ? __builtin_fmax(p - taken, 0.0) : 0.0, p};  // (past the vocabulary p is 0)
        }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void rest_kernel(VerifyArgs a) {
    constexpr int kKept = 64;
    __shared__ int stop;
    __shared__ PieceStats kept[kKept];
    __shared__ double powers[kSteps];
    const int r = blockIdx.y, piece = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int begin = max(a.starts[r], 0), end = min(a.starts[r + 1], a.rows);
    if (begin >= end) {
        if (piece == 0 && tid == 0) a.accepted[r] = 0, a.decisions[r].row = -1;
        return;
    }
    if (tid == 0) stop = end - 1;
    if (tid < kSteps) powers[tid] = kPowers[tid];
    __syncthreads();
    const double by = factor_of(a.temperature, r);
    // A wave a row; what the deciding row's numbers are is kept for as many rows as there is room for.
    for (int row = begin + wave; row < end; row += kWaves) {
        const int t = row + 1 < end ? a.tokens[row + 1] : -1;
        bool accept = t >= 0 && t < a.vocab;
        const float logit = accept ? entry((const T *)a.logits + row * a.ld + t) : 0.0f;
        const double u = uniform_of(a, row), q = accept ? draft_of(a, row, t, t) : 0.0;
        const PieceStats s = row_stats(a, row, by, powers);
        if (accept) accept = s.sum > 0.0 && u * q < weight_of(logit, s.most, by, t == s.first, powers) / s.sum;
        if (lane == 0) {
            if (!accept) atomicMin(&stop, row);
            if (row - begin < kKept) kept[row - begin] = s;
        }
    }
    __syncthreads();
    const int last = stop;
    PieceStats s;
    if (last - begin < kKept) s = kept[last - begin];
    else s = row_stats(a, last, by, powers);
    const Decision d = {last, last == end - 1, s.first, s.most, s.sum, by};
    const int drafted = d.last ? -1 : a.tokens[d.row + 1];
    if (piece == 0) {
        if (tid == 0) a.decisions[r] = d, a.accepted[r] = d.row - begin;
        for (int row = begin + tid; row < end; row += kThreads)
            if (row != d.row) a.out[row] = row < d.row ? a.tokens[row + 1] : -1;
    }
    StripSums sum{0.0, 0.0}, w[kPer];
    rests_of<T, kPer>(a, d, drafted, piece * kPiece + wave * kStrip + lane * 4, 256, powers, w);
#pragma unroll
    for (int e = 0; e < kPer; ++e) sum.rest += w[e].rest, sum.whole += w[e].whole;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) sum.rest += __shfl_xor(sum.rest, m), sum.whole += __shfl_xor(sum.whole, m);
    if (lane == 0) a.strips[((int64_t)r * a.pieces + piece) * kWaves + wave] = sum;
}

// The wave's running sums over its lanes, each lane's own included.
__device__ __forceinline__ double wave_running(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const double w = __shfl_up(v, m);
        if (lane >= m) v += w;
    }
    return v;
}

// One wave a request. The strips, and then the entries of the one that the draw falls into, lie in runs over the lanes: the lane whose
// run the draw falls into goes through it.
template <typename T>
__global__ __launch_bounds__(64) void finish_kernel(VerifyArgs a) {
    __shared__ double powers[kSteps];
    const int r = blockIdx.x, lane = threadIdx.x;
    const Decision d = a.decisions[r];
    powers[lane] = kPowers[lane];
    __syncthreads();
    const StripSums *strips = a.strips + (int64_t)r * a.pieces * kWaves;
    const int count = a.pieces * kWaves, run = (count + 63) / 64;
    const int low = min(lane * run, count), high = min(low + run, count);
    const double u = uniform_of(a, max(min(a.starts[r + 1], a.rows) - 1, 0));
    double rest = 0.0, whole = 0.0;
#pragma unroll 4
    for (int i = low; i < high; ++i) rest += strips[i].rest, whole += strips[i].whole;
    if (d.row < 0) return;  // (no rows; the loads above do not wait for it)
    const int drafted = d.last ? -1 : a.tokens[d.row + 1];
    const double rests = wave_running(rest), wholes = wave_running(whole);
    const bool from_rest = __shfl(rests, 63) > 0.0;
    const double total = from_rest ? __shfl(rests, 63) : __shfl(wholes, 63);
    // (u >= 1 is past the whole weight. The product would be the sum in one order, which sums in the others' orders pass before the last entry.)
    const double draw = u < 1.0 ? u * total : __builtin_inf();
    // The lane that the draw falls into: the first whose running weight passes it, or, if none does, the last with weight.
    auto lane_of = [&](double own, double running) {
        const uint64_t passed = __ballot(own > 0.0 && running > draw), with = __ballot(own > 0.0);
        return passed ? __builtin_ctzll(passed) : with ? 63 - __builtin_clzll(with) : -1;
    };
    const double mine = from_rest ? rest : whole, running = from_rest ? rests : wholes;
    const int at = lane_of(mine, running);
    int token = -1;
    if (at >= 0) {
        // That lane's strips one by one (all lanes go along with it).
        const int first = __shfl(low, at), end = __shfl(high, at);
        double before = __shfl(running - mine, at), strip_before = before;
        int strip = -1;
        for (int i = first; i < end; ++i) {
            const double w = from_rest ? strips[i].rest : strips[i].whole;
            if (w > 0.0) {
                strip = i, strip_before = before;
                if (before + w > draw) break;
            }
            before += w;
        }
        if (strip >= 0) {
            StripSums w[kPer];
            rests_of<T, kPer>(a, d, drafted, strip * kStrip + lane * kPer, 4, powers, w);
            double own = 0.0;
#pragma unroll
            for (int e = 0; e < kPer; ++e) own += from_rest ? w[e].rest : w[e].whole;
            const double to = strip_before + wave_running(own);
            const int found = lane_of(own, to);
            double sum = to - own;
            int entry_of = -1;
            bool done = false;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const double x = from_rest ? w[e].rest : w[e].whole;
                if (x > 0.0 && !done) entry_of = e;
                sum += x;
                done |= x > 0.0 && sum > draw;
            }
            const int entry_there = __shfl(entry_of, found < 0 ? 0 : found);
            if (found >= 0 && entry_there >= 0) token = strip * kStrip + found * kPer + entry_there;
        }
    }
    if (lane == 0) a.out[d.row] = token;
}

static int64_t pieces_of(int64_t vocab) { return (vocab + kPiece - 1) / kPiece; }

size_t verify_workspace_bytes(int64_t rows, int64_t vocab, int64_t requests) {
    const int64_t pieces = pieces_of(vocab);
    return kVerifyCounterBytes + rows * pieces * sizeof(PieceStats) + requests * sizeof(Decision) +
           requests * pieces * kWaves * sizeof(StripSums);
}

hipError_t launch_verify(const void *logits, int64_t ld, int dtype, int64_t rows, int64_t vocab, const int32_t *tokens,
                         const int32_t *starts, int64_t requests, const float *uniforms, const float *temperature,
                         const void *draft, int64_t ld_draft, int draft_dtype, int32_t *out, int32_t *accepted,
                         void *workspace, hipStream_t stream) {
    static_assert(sizeof(PieceStats) == 16 && sizeof(Decision) % 16 == 0 && sizeof(StripSums) == 16, "aligned arrays");
    VerifyArgs a{logits, ld, (int)vocab, (int)pieces_of(vocab), (int)requests, (int)rows, tokens, starts, uniforms,
                 temperature, draft, ld_draft, draft_dtype == SPLOSH_F32, out, accepted, nullptr, nullptr, nullptr};
    uint8_t *at = static_cast<uint8_t *>(workspace) + kVerifyCounterBytes;
    a.stats = reinterpret_cast<PieceStats *>(at);
    at += rows * a.pieces * sizeof(PieceStats);
    a.decisions = reinterpret_cast<Decision *>(at);
    at += requests * sizeof(Decision);
    a.strips = reinterpret_cast<StripSums *>(at);
    const dim3 rows_grid(a.pieces, (unsigned)rows), requests_grid(a.pieces, (unsigned)requests);
    auto go = [&](auto scan, auto rest, auto finish) {
        scan<<<rows_grid, kScanThreads, 0, stream>>>(a);
        rest<<<requests_grid, kThreads, 0, stream>>>(a);
        finish<<<(unsigned)requests, 64, 0, stream>>>(a);
    };
    if (dtype == SPLOSH_F32) go(scan_kernel<float>, rest_kernel<float>, finish_kernel<float>);
    else go(scan_kernel<uint16_t>, rest_kernel<uint16_t>, finish_kernel<uint16_t>);
    return hipGetLastError();
}

}  // namespace splosh
