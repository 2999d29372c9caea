// adapters.hip -- low-rank adapters of many requests beside a shared projection.
//
// out[m] += c_s b_s (a_s x[m]) for the adapter s = slots[m] of row m, in two launches: the products
// t = a_s x (fp32 partial sums over slices of K, in the workspace), then out += b_s (c_s t).
//
// Both walk the rows in chunks of 64. A chunk's rows are taken adapter by adapter: the lanes of a wave
// hold the chunk's slots, a ballot gives the rows of one adapter, and these meet the adapter's matrix as
// the columns of v_mfma_f32_16x16x32_bf16, sixteen at a time, whatever places they have in the batch. So
// an adapter's matrices are read once a chunk, no sorted order of the rows is asked for, and an adapter
// no row uses costs nothing.
#include "common.hpp"
#include "launch.hpp"

namespace splosh {

// The workspace's first 16 KiB belong to the arrival counters of the kernels that have any.
constexpr size_t kAdapterCounterBytes = 16384;
constexpr int kChunk = 64;       // rows of a chunk
constexpr int kDownRanks = 64;   // rows of a that a workgroup of the first launch takes
constexpr int kUpColumns = 256;  // outputs of a workgroup of the second
constexpr int kUpRanks = 64;     // ranks it stages at a time

struct AdapterWeight {
    splosh_adapters w;
    void *out;
    int64_t ldc;
    int t_offset;  // its first column of t
    int first;     // its first workgroup column of the launch
};

struct AdapterArgs {
    AdapterWeight w[SPLOSH_MAX_GROUP];
    int group;
    const uint16_t *x;
    int64_t ldx;
    const int32_t *slots;
    float *t;     // [slices][rows][t_cols]
    int t_cols, slices;
    int64_t rows;
};

// The projection a workgroup column belongs to.
__device__ __forceinline__ int projection_of(const AdapterArgs &args, int column) {
    int i = 0;
    while (i + 1 < args.group && column >= args.w[i + 1].first) ++i;
    return i;
}

// Elements [0, n) of eight from p, zero past them; ALIGNED: p is 16-byte aligned.
template <bool ALIGNED>
__device__ __forceinline__ u32x4 load8(const uint16_t *p, int n) {
    u32x4 v = {0, 0, 0, 0};
    if (ALIGNED && n >= 8) return *(const u32x4 *)p;
    if (n > 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) v[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
    }
    return v;
}

// The rows of a chunk, adapter by adapter: every lane holds its row's slot and rank (0: no adapter), and
// next() leaves in `mine` the i-th row of the next adapter's for lane i (the other rows after them).
struct ChunkRows {
    int slot, rank, seen, mine, count;
    uint64_t todo;
    int group_slot, group_rank;

    __device__ __forceinline__ ChunkRows(const AdapterArgs &args, const splosh_adapters &w, int64_t base) {
        const int lane = threadIdx.x & 63;
        const int64_t row = base + lane;
        slot = row < args.rows ? args.slots[row] : -1;
        const bool known = slot >= 0 && slot < w.count;
        rank = known ? (w.ranks ? w.ranks[slot] : (int)w.max_rank) : 0;
        rank = rank < (int)w.max_rank ? rank : (int)w.max_rank;
        todo = __ballot(rank > 0);
        seen = 0;
    }

    // The next adapter whose turn is `z` of `turns`; false past the last.
    __device__ __forceinline__ bool next(int z, int turns) {
        while (todo) {
            const int first = __builtin_ctzll(todo);
            group_slot = __builtin_amdgcn_readlane(slot, first);
            const uint64_t rows = __ballot(rank > 0 && slot == group_slot);
            todo &= ~rows;
            if (seen++ % turns != z) continue;
            group_rank = __builtin_amdgcn_readlane(rank, first);
            count = __builtin_popcountll(rows);
            const int lane = threadIdx.x & 63;
            const uint64_t below = ((uint64_t)1 << lane) - 1;
            const int place = rows >> lane & 1 ? __builtin_popcountll(rows & below)
                                               : count + __builtin_popcountll(~rows & below);
            mine = __builtin_amdgcn_ds_permute(place * 4, lane);
            return true;
        }
        return false;
    }

    // The chunk row at place i of the adapter's.
    __device__ __forceinline__ int row_at(int i) const { return __builtin_amdgcn_ds_bpermute(i * 4, mine); }
};

// ---- t = a x --------------------------------------------------------------------------------------
//
// A workgroup: one chunk, up to 64 rows of one projection's a, one slice of K. Its four waves take the
// slice's steps of 32 k in turn, kSteps of them with every load in flight, and add their sums in LDS.
// a's rows are the MFMA's rows and the activation rows its columns: the sum's four registers are then
// four neighbouring ranks of one activation row, a 16-byte store.

constexpr int kSteps = 4;

template <int RB, int P, bool ALIGNED>
__device__ __attribute__((always_inline)) void down_rows(const AdapterArgs &args, const AdapterWeight &g, const ChunkRows &rows,
                                          int64_t base, int rank0, int slice, f32x4 *sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, q = lane >> 4;
    const int inner = (int)g.w.inner, steps = (inner + 31) / 32;
    const int from = (int)((int64_t)steps * slice / args.slices), to = (int)((int64_t)steps * (slice + 1) / args.slices);
    const uint16_t *a = g.w.a + rows.group_slot * g.w.a_slot_stride;
    const uint16_t *xr[RB], *ar[P];
    bool xv[RB], av[P];
    int64_t out_row[RB];
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        xv[i] = i * 16 + m < rows.count;
        const int at = rows.row_at(i * 16 + m);
        out_row[i] = base + (xv[i] ? at : 0);
        xr[i] = args.x + out_row[i] * args.ldx;
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int r = rank0 + p * 16 + m;
        av[p] = r < rows.group_rank;
        ar[p] = a + (av[p] ? r : 0) * g.w.a_row_stride;
    }
    f32x4 acc[RB][P];
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int p = 0; p < P; ++p) acc[i][p] = f32x4{0, 0, 0, 0};
    for (int s = from + wave; s < to; s += 4 * kSteps) {
        u32x4 xs[kSteps][RB], as[kSteps][P];
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            const int step = s + 4 * j, k = step * 32 + q * 8, n = step < to ? inner - k : 0;
#pragma unroll
            for (int i = 0; i < RB; ++i) xs[j][i] = load8<ALIGNED>(xr[i] + k, xv[i] ? n : 0);
#pragma unroll
            for (int p = 0; p < P; ++p) as[j][p] = load8<ALIGNED>(ar[p] + k, av[p] ? n : 0);
        }
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
#pragma unroll
            for (int i = 0; i < RB; ++i)
#pragma unroll
                for (int p = 0; p < P; ++p)
                    acc[i][p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(as[j][p]), as_bf16x8(xs[j][i]),
                                                                         acc[i][p], 0, 0, 0);
    }
    // The waves' sums, panel by panel: [wave][row block][lane].
#pragma unroll
    for (int p = 0; p < P; ++p) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RB; ++i) sums[(wave * RB + i) * 64 + lane] = acc[i][p];
        __syncthreads();
        if (wave < RB) {
            f32x4 v = sums[wave * 64 + lane];
#pragma unroll
            for (int w = 1; w < 4; ++w) v += sums[(w * RB + wave) * 64 + lane];
            const int r = rank0 + p * 16 + q * 4;
            int64_t row = out_row[0];
            bool live = xv[0];
#pragma unroll
            for (int i = 1; i < RB; ++i)
                if (wave == i) row = out_row[i], live = xv[i];
            if (live && r < rows.group_rank)
                *(f32x4 *)(args.t + ((int64_t)slice * args.rows + row) * args.t_cols + g.t_offset + r) = v;
        }
    }
}

template <int RBMAX, int P, bool ALIGNED>
__global__ void __launch_bounds__(256, 2) adapter_down_kernel(AdapterArgs args) {
    __shared__ f32x4 sums[4 * RBMAX * 64];
    const int column = blockIdx.x / args.slices, slice = blockIdx.x % args.slices;
    const AdapterWeight &g = args.w[projection_of(args, column)];
    const int rank0 = (column - g.first) * kDownRanks;
    const int64_t base = (int64_t)blockIdx.y * kChunk;
    ChunkRows rows(args, g.w, base);
    while (rows.next(blockIdx.z, gridDim.z)) {
        if (rank0 >= rows.group_rank) continue;
        if (RBMAX == 1 || rows.count <= 16)
            down_rows<1, P, ALIGNED>(args, g, rows, base, rank0, slice, sums);
        else if (rows.count <= 32)
            down_rows<RBMAX == 1 ? 1 : 2, P, ALIGNED>(args, g, rows, base, rank0, slice, sums);
        else
            down_rows<RBMAX, P, ALIGNED>(args, g, rows, base, rank0, slice, sums);
    }
}

// ---- out += b t -----------------------------------------------------------------------------------
//
// A workgroup: one chunk, 256 outputs of one projection, 64 a wave. t's slices are summed, scaled, and
// laid down in LDS as MFMA operands, in two bf16 pieces for a bf16 output and three for an fp32 one (a
// piece takes eight more bits, so the products keep 16 or 24 of t's); b's rows are the MFMA's rows,
// dealt so that a lane's sixteen sums of one output row are sixteen neighbouring outputs: row 4 q + i of
// block j is output 16 q + 4 j + i.

template <typename OUT>
__device__ __forceinline__ void load_out16(const OUT *p, int n, bool vector, uint32_t (&v)[16 * sizeof(OUT) / 4]) {
    constexpr int kPer = 4 / sizeof(OUT);
    if (vector && n >= 16) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(OUT); ++i) {
            const u32x4 w = *(const u32x4 *)((const char *)p + 16 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * i + e] = w[e];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 16 / kPer; ++i) {
        v[i] = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e)
            if (i * kPer + e < n) {
                if constexpr (sizeof(OUT) == 4) v[i] = __float_as_uint(p[i]);
                else v[i] |= (uint32_t)p[i * kPer + e] << (16 * e);
            }
    }
}

template <int RB, typename OUT, bool ALIGNED>
__device__ __attribute__((always_inline)) void up_rows(const AdapterArgs &args, const AdapterWeight &g, const ChunkRows &rows,
                                        int64_t base, int column0, u32x2 *pieces) {
    constexpr int kPieces = sizeof(OUT) == 4 ? 3 : 2, kPanels = kUpRanks / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, q = lane >> 4;
    const int n0 = column0 + wave * 64, columns = (int)g.w.rows, rank = rows.group_rank;
    // The outputs to add to, asked for first.
    OUT *out[RB];
    bool live[RB];
    uint32_t old[RB][16 * sizeof(OUT) / 4];
    const int left = columns - n0 - q * 16;
    const bool vector = (g.ldc * sizeof(OUT)) % 16 == 0 && ((uintptr_t)g.out & 15) == 0;
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        live[i] = i * 16 + m < rows.count;
        const int at = rows.row_at(i * 16 + m);
        out[i] = (OUT *)g.out + (base + (live[i] ? at : 0)) * g.ldc + n0 + q * 16;
        load_out16<OUT>(out[i], live[i] ? left : 0, vector, old[i]);
    }
    const uint16_t *b = g.w.b + rows.group_slot * g.w.b_slot_stride;
    const float scale = g.w.scales ? g.w.scales[rows.group_slot] : 1.0f;
    f32x4 acc[RB][4];
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    for (int rank0 = 0; rank0 < rank; rank0 += kUpRanks) {
        u32x4 bs[kPanels][4];
#pragma unroll
        for (int p = 0; p < kPanels; ++p)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = n0 + (m >> 2) * 16 + j * 4 + (m & 3), r = rank0 + p * 32 + q * 8;
                bs[p][j] = load8<ALIGNED>(b + (int64_t)n * g.w.b_row_stride + r, n < columns ? rank - r : 0);
            }
        if (rank0) __syncthreads();
        // Four ranks of one row a thread: [piece][panel][row block][lane of the operand] x 16 bytes.
        const int ranks = rank - rank0 < kUpRanks ? rank - rank0 : kUpRanks, quads = (ranks + 31) / 32 * 8;
        for (int item = tid; item < RB * 16 * quads; item += 256) {
            const int i = item / quads, r = (item % quads) * 4;
            f32x4 v = {0, 0, 0, 0};
            const int chunk_row = rows.row_at(i & 63);
            if (i < rows.count && rank0 + r < rank) {
                const float *t = args.t + (base + chunk_row) * args.t_cols + g.t_offset + rank0 + r;
                for (int s = 0; s < args.slices; ++s) v += *(const f32x4 *)(t + (int64_t)s * args.rows * args.t_cols);
            }
            float piece[kPieces][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float rest = rank0 + r + e < rank ? v[e] * scale : 0.0f;
#pragma unroll
                for (int c = 0; c < kPieces; ++c) {
                    piece[c][e] = rest;
                    const float top = bf16_bits_to_f32(f32_to_bf16(rest));
                    rest = __builtin_fabsf(top) < __builtin_inff() ? rest - top : 0.0f;
                }
            }
            const int at = ((r >> 5) * RB + (i >> 4)) * 64 + ((r >> 3) & 3) * 16 + (i & 15);
#pragma unroll
            for (int c = 0; c < kPieces; ++c)
                pieces[(c * kPanels * RB * 64 + at) * 2 + ((r >> 2) & 1)] =
                    u32x2{f32x2_to_bf16x2(piece[c][0], piece[c][1]), f32x2_to_bf16x2(piece[c][2], piece[c][3])};
        }
        __syncthreads();
#pragma unroll
        for (int p = 0; p < kPanels; ++p) {
            if (p * 32 >= ranks) break;
#pragma unroll
            for (int c = 0; c < kPieces; ++c)
#pragma unroll
                for (int i = 0; i < RB; ++i) {
                    const u32x4 t = *(const u32x4 *)&pieces[(((c * kPanels + p) * RB + i) * 64 + lane) * 2];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(bs[p][j]), as_bf16x8(t), acc[i][j],
                                                                             0, 0, 0);
                }
        }
    }
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        if (!live[i]) continue;
        if constexpr (sizeof(OUT) == 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(old[i][4 * j + e]) + acc[i][j][e];
                if (vector && left >= 16) *(f32x4 *)(out[i] + 4 * j) = v;
                else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (4 * j + e < left) out[i][4 * j + e] = v[e];
                }
            }
        } else {
            uint32_t v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = f32x2_to_bf16x2(bf16_bits_to_f32(old[i][e] & 0xffffu) + acc[i][e >> 1][2 * (e & 1)],
                                       bf16_bits_to_f32(old[i][e] >> 16) + acc[i][e >> 1][2 * (e & 1) + 1]);
            if (vector && left >= 16) {
                *(u32x4 *)out[i] = u32x4{v[0], v[1], v[2], v[3]};
                *(u32x4 *)(out[i] + 8) = u32x4{v[4], v[5], v[6], v[7]};
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (e < left) out[i][e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
            }
        }
    }
    __syncthreads();  // (the next adapter stages into the same LDS)
}

template <int RBMAX, typename OUT, bool ALIGNED>
__global__ void __launch_bounds__(256, 2) adapter_up_kernel(AdapterArgs args) {
    __shared__ u32x4 pieces[3 * (kUpRanks / 32) * RBMAX * 64];
    const AdapterWeight &g = args.w[projection_of(args, blockIdx.x)];
    const int column0 = ((int)blockIdx.x - g.first) * kUpColumns;
    const int64_t base = (int64_t)blockIdx.y * kChunk;
    ChunkRows rows(args, g.w, base);
    while (rows.next(blockIdx.z, gridDim.z)) {
        if (RBMAX == 1 || rows.count <= 16)
            up_rows<1, OUT, ALIGNED>(args, g, rows, base, column0, (u32x2 *)pieces);
        else if (rows.count <= 32)
            up_rows<RBMAX == 1 ? 1 : 2, OUT, ALIGNED>(args, g, rows, base, column0, (u32x2 *)pieces);
        else
            up_rows<RBMAX, OUT, ALIGNED>(args, g, rows, base, column0, (u32x2 *)pieces);
    }
}

// ---- host -----------------------------------------------------------------------------------------

static int t_columns(const splosh_adapters *w, int group) {
    int cols = 0;
    for (int i = 0; i < group; ++i) cols += (int)(w[i].max_rank + 15) / 16 * 16;
    return cols;
}

static int down_columns(const splosh_adapters *w, int group) {
    int columns = 0;
    for (int i = 0; i < group; ++i) columns += (int)(w[i].max_rank + kDownRanks - 1) / kDownRanks;
    return columns;
}

// Slices of K: 512 workgroups from the chunks and projections alone, of 16 steps of 32 or more each (four
// a wave).
static int plan_slices(const splosh_adapters *w, int group, int64_t rows) {
    const int64_t chunks = (rows + kChunk - 1) / kChunk, steps = (w[0].inner + 31) / 32;
    const int64_t want = (511 + chunks * down_columns(w, group)) / (chunks * down_columns(w, group));
    int64_t slices = steps / 16 < want ? steps / 16 : want;
    slices = slices < 32 ? slices : 32;
    return slices < 1 ? 1 : (int)slices;
}

size_t adapters_workspace_bytes(const splosh_adapters *w, int group, int64_t rows) {
    return kAdapterCounterBytes + (size_t)plan_slices(w, group, rows) * rows * t_columns(w, group) * sizeof(float);
}

// The adapters of a chunk go to up to this many workgroups: all of its rows' where the launch is small, one
// where it fills the device anyway.
static unsigned turns(const splosh_adapters *w, int group, int64_t rows, int64_t others) {
    int64_t most = rows < kChunk ? rows : kChunk, count = 1;
    for (int i = 0; i < group; ++i) count = w[i].count > count ? w[i].count : count;
    most = count < most ? count : most;
    const int64_t n = 4096 / others;
    return (unsigned)(n < 1 ? 1 : n < most ? n : most);
}

template <int RBMAX, bool ALIGNED>
static void launch_down(const AdapterArgs &args, int panels, dim3 grid, hipStream_t stream) {
    if (panels == 1) hipLaunchKernelGGL((adapter_down_kernel<RBMAX, 1, ALIGNED>), grid, dim3(256), 0, stream, args);
    else if (panels == 2) hipLaunchKernelGGL((adapter_down_kernel<RBMAX, 2, ALIGNED>), grid, dim3(256), 0, stream, args);
    else hipLaunchKernelGGL((adapter_down_kernel<RBMAX, 4, ALIGNED>), grid, dim3(256), 0, stream, args);
}

template <int RBMAX, typename OUT>
static void launch_up(const AdapterArgs &args, bool aligned, dim3 grid, hipStream_t stream) {
    if (aligned) hipLaunchKernelGGL((adapter_up_kernel<RBMAX, OUT, true>), grid, dim3(256), 0, stream, args);
    else hipLaunchKernelGGL((adapter_up_kernel<RBMAX, OUT, false>), grid, dim3(256), 0, stream, args);
}

hipError_t launch_adapters(const splosh_adapters *w, int group, const uint16_t *x, int64_t ldx, void *const *outs,
                           const int64_t *ldcs, int out_dtype, const int32_t *slots, int64_t rows, void *workspace,
                           hipStream_t stream) {
    AdapterArgs args{};
    args.group = group;
    args.x = x;
    args.ldx = ldx;
    args.slots = slots;
    args.t = (float *)((char *)workspace + kAdapterCounterBytes);
    args.t_cols = t_columns(w, group);
    args.slices = plan_slices(w, group, rows);
    args.rows = rows;
    auto aligned16 = [](const void *p, int64_t a, int64_t b) { return (uintptr_t)p % 16 == 0 && a % 8 == 0 && b % 8 == 0; };
    bool down_aligned = aligned16(x, ldx, 0), up_aligned = true;
    int at = 0, columns = 0;
    int64_t most_rank = 0;
    for (int i = 0; i < group; ++i) {
        args.w[i] = AdapterWeight{w[i], outs[i], ldcs[i], at, columns};
        at += (int)(w[i].max_rank + 15) / 16 * 16;
        columns += (int)(w[i].max_rank + kDownRanks - 1) / kDownRanks;
        most_rank = w[i].max_rank > most_rank ? w[i].max_rank : most_rank;
        down_aligned = down_aligned && aligned16(w[i].a, w[i].a_slot_stride, w[i].a_row_stride);
        up_aligned = up_aligned && aligned16(w[i].b, w[i].b_slot_stride, w[i].b_row_stride);
    }
    const unsigned chunks = (unsigned)((rows + kChunk - 1) / kChunk);
    const unsigned down_x = (unsigned)(columns * args.slices);
    const dim3 down(down_x, chunks, turns(w, group, rows, (int64_t)down_x * chunks));
    const int panels = most_rank <= 16 ? 1 : most_rank <= 32 ? 2 : 4;
    if (rows <= 16) {
        if (down_aligned) launch_down<1, true>(args, panels, down, stream);
        else launch_down<1, false>(args, panels, down, stream);
    } else {
        if (down_aligned) launch_down<4, true>(args, panels, down, stream);
        else launch_down<4, false>(args, panels, down, stream);
    }
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    unsigned up_x = 0;
    for (int i = 0; i < group; ++i) {
        args.w[i].first = (int)up_x;
        up_x += (unsigned)((w[i].rows + kUpColumns - 1) / kUpColumns);
    }
    const dim3 up(up_x, chunks, turns(w, group, rows, (int64_t)up_x * chunks));
    if (rows <= 16) {
        if (out_dtype == SPLOSH_F32) launch_up<1, float>(args, up_aligned, up, stream);
        else launch_up<1, uint16_t>(args, up_aligned, up, stream);
    } else {
        if (out_dtype == SPLOSH_F32) launch_up<4, float>(args, up_aligned, up, stream);
        else launch_up<4, uint16_t>(args, up_aligned, up, stream);
    }
    return hipGetLastError();
}

}  // namespace splosh
