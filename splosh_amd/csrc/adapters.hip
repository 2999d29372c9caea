// adapters.hip -- low-rank adapters of many requests beside a shared projection.
//
// out[m] += c_s b_s (a_s x[m]) for the adapter s = slots[m] of row m, in two launches: the products
// t = c_s a_s x (fp32 partial sums over slices of K, in the workspace), then out += b_s t.
//
// Both walk the rows in chunks of 64. A chunk's rows are taken adapter by adapter: the lanes of a wave
// hold the chunk's slots, a ballot gives the rows of one adapter, and these meet the adapter's matrix as
// the columns of v_mfma_f32_16x16x32_bf16, whatever places they have in the batch. So no sorted order of
// the rows is asked for, and an adapter that no row uses costs nothing. a is read once a chunk; b once for each of the
// up to four workgroups that share an adapter's rows, and past 32 ranks once for each sixteen rows. The first launch
// leaves the chunks' lists of adapters and rows for the second.
//
// FAST kernels are for operands whose every 16-byte piece is whole, aligned and within a buffer
// descriptor's reach (the usual case): their loads have no branches, since an offset out of a descriptor's
// range reads zeros and writes nothing. The others load pieces at any alignment, where they are whole, and
// element by element where they are not (both launches on FAST operands: 64 rows, K5120 -> 2 x 17408, fp32: 15.3 us
// FAST, 19.6 not; 2048 rows, K5120 -> N17408, bf16: 44.0 and 57.6, and 66 with the odd sizes K5119 -> N17401).
//
// What has to move is the adapters' matrices in use, x, and out twice; the arithmetic, 2 rank (K + N) a row, is far
// under the matrix core's rate. A step's small calls are two launches of 2 us, each with four dependent round
// trips to memory (slots, ranks, operands, sums): 4.2 + 4.8 us for one row of K5120 -> N5120.
#include "common.hpp"
#include "launch.hpp"

namespace splosh {

// The workspace's first 16 KiB belong to the arrival counters of the kernels that have any.
constexpr size_t kAdapterCounterBytes = 16384;
constexpr int kChunk = 64;       // rows of a chunk
constexpr int kDownRanks = 32;   // rows of a that a workgroup of the first launch takes
constexpr int kUpColumns = 256;  // outputs of a tile of the second
// An offset past every descriptor, and still so with another one added.
constexpr uint32_t kNowhere = 0x40000000u;

// One chunk's adapters for one projection.
struct ChunkList {
    struct Part {
        int32_t slot;
        uint16_t rank;       // 0: past the last part
        uint8_t first, count;  // its rows: order[first ..]
    } part[kChunk];
    uint8_t order[kChunk];
};

struct AdapterWeight {
    splosh_adapters w;
    void *out;
    int64_t ldc;
    int t_offset;  // its first column of t
};

struct AdapterArgs {
    const uint16_t *x;
    int64_t ldx, rows;
    const int32_t *slots;
    ChunkList *lists;  // [projection][chunk]
    float *t;          // [slices][rows][t_cols]
    int t_cols, slices, slice_steps;
    int tiles;    // tiles of outputs a workgroup of the second launch takes
    int turns;    // workgroups that share a chunk's adapters
    int shares;   // workgroups of the second launch that share an adapter's rows, sixteen at a time
    AdapterWeight w[SPLOSH_MAX_GROUP];
};

// Elements [0, n) of the eight at p, of any alignment; zero past them.
__device__ __forceinline__ u32x4 load8(const uint16_t *p, int n) {
    u32x4 v = {0, 0, 0, 0};
    if (n >= 8) {
        __builtin_memcpy(&v, p, 16);
    } else if (n > 0) {
        uint64_t low = 0, high = 0;
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            const uint64_t e = (uint64_t)p[i] << (16 * (i & 3));
            low |= i < 4 ? e : 0;
            high |= i < 4 ? 0 : e;
        }
        v = u32x4{(uint32_t)low, (uint32_t)(low >> 32), (uint32_t)high, (uint32_t)(high >> 32)};
    }
    return v;
}
__device__ __forceinline__ u32x4 keep8(u32x4 v, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = 2 * i + 1 < n ? v[i] : 2 * i < n ? v[i] & 0xffffu : 0u;
    return v;
}

// Orders a wave's own LDS operations for the compiler (the hardware does them in order).
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// ---- t = a x --------------------------------------------------------------------------------------
//
// A workgroup: one adapter's rows of a chunk, up to 32 rows of one projection's a, one slice of K. Its four
// waves take the slice's steps of 32 k in turn, kSteps of them with every load in flight, and add their
// sums in LDS. a's rows are the MFMA's rows and the activation rows its columns: the sum's four registers
// are then four neighbouring ranks of one activation row, a 16-byte store.
//
// A load has the four lanes of a quad read the 64 bytes of one row, and goes through LDS to the MFMA's order,
// in which neighbouring lanes hold neighbouring rows: loaded in that order, every lane is a cache lookup of
// its own.
//
// Bound by the reads of a where they are many, at up to 3.0 TB/s: 64 rows of 32 adapters, K17408, ranks 16 to 64
// 47 MB in 15.7 us, 2 us of it the launch. Ranks of 64, 32, 16 and 8 leave workgroups of very uneven lengths, and the
// longest decides: 36 MB in 15.1 us, and 31 MB in 13.9 where the rows use 27 of the 32 (2.2 TB/s). More loads in flight (the next steps' before this one's products; rows in runs of 128 bytes)
// measured the same. One block of rows a workgroup (RBMAX 1, for up to 16 rows) saves the code and registers of the
// other form: 4.9 us for 5.1 with eight rows on q, k and v. One panel of 16 ranks (P 1): 4.2 us for 4.7 with one row.

constexpr int kDownWaves = 4;

// 16 RB of the adapter's rows: `mine` is the chunk row that lane i holds as the adapter's i-th.
template <int RB, int P, bool FAST>
__device__ __attribute__((always_inline)) void down_rows(const AdapterArgs &args, const AdapterWeight &g, int slot,
                                                         int rank, float scale, int mine, int count, int64_t base,
                                                         int rank0, int slice, u32x4 *memory) {
    constexpr int kSteps = RB == 1 ? 4 : 2;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, q = lane >> 4;
    // Where a lane's 16 bytes of a load lie: row and piece; and, spread over the banks, in LDS.
    const int load_row = lane >> 2, load_piece = lane & 3;
    u32x4 *stage = memory + wave * (RB + P) * 64;
    const int put = lane ^ ((lane >> 4) & 3), get = m * 4 + (q ^ ((m >> 2) & 3));
    const int inner = (int)g.w.inner, steps = (inner + 31) / 32;
    const int from = slice * args.slice_steps, to = from + args.slice_steps < steps ? from + args.slice_steps : steps;
    const uint16_t *a = g.w.a + slot * g.w.a_slot_stride, *x = args.x + base * args.ldx;
    const rsrc_t ra = make_rsrc(a, FAST ? (uint32_t)(g.w.max_rank * g.w.a_row_stride * 2) : 0);
    const rsrc_t rx = make_rsrc(x, FAST ? (uint32_t)(kChunk * args.ldx * 2) : 0);
    uint32_t xo[RB], ao[P];
    const uint16_t *xp[RB], *ap[P];
    bool xv[RB], av[P];
    int xr[RB];
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        xr[i] = __builtin_amdgcn_ds_bpermute(((i * 16 + m) & 63) * 4, mine);
        if (i * 16 + m >= count) xr[i] = -1;
        const int row = __builtin_amdgcn_ds_bpermute(((i * 16 + load_row) & 63) * 4, mine);
        xv[i] = i * 16 + load_row < count;
        xo[i] = xv[i] ? (uint32_t)(row * args.ldx * 2) : kNowhere;
        xp[i] = x + (xv[i] ? row : 0) * args.ldx;
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int r = rank0 + p * 16 + load_row;
        av[p] = r < rank;
        ao[p] = av[p] ? (uint32_t)(r * g.w.a_row_stride * 2) : kNowhere;
        ap[p] = a + (av[p] ? r : 0) * g.w.a_row_stride;
    }
    f32x4 acc[RB][P];
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int p = 0; p < P; ++p) acc[i][p] = f32x4{0, 0, 0, 0};
    for (int s = from + wave; s < to; s += kDownWaves * kSteps) {
        u32x4 xs[kSteps][RB], as[kSteps][P];
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            const int step = s + kDownWaves * j, k = step * 32 + load_piece * 8, n = step < to ? inner - k : 0;
            const uint32_t ko = n > 0 ? (uint32_t)k * 2 : kNowhere;
#pragma unroll
            for (int i = 0; i < RB; ++i)
                xs[j][i] = FAST ? buffer_load16(rx, xo[i] + ko, 0) : load8(xp[i] + k, xv[i] ? n : 0);
#pragma unroll
            for (int p = 0; p < P; ++p)
                as[j][p] = FAST ? buffer_load16(ra, ao[p] + ko, 0) : load8(ap[p] + k, av[p] ? n : 0);
        }
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
#pragma unroll
            for (int i = 0; i < RB; ++i) stage[i * 64 + put] = xs[j][i];
#pragma unroll
            for (int p = 0; p < P; ++p) stage[(RB + p) * 64 + put] = as[j][p];
            wave_fence();
#pragma unroll
            for (int i = 0; i < RB; ++i) xs[j][i] = stage[i * 64 + get];
#pragma unroll
            for (int p = 0; p < P; ++p) as[j][p] = stage[(RB + p) * 64 + get];
            wave_fence();
#pragma unroll
            for (int i = 0; i < RB; ++i)
#pragma unroll
                for (int p = 0; p < P; ++p)
                    acc[i][p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(as[j][p]), as_bf16x8(xs[j][i]),
                                                                         acc[i][p], 0, 0, 0);
        }
    }
    f32x4 *sums = (f32x4 *)memory;
    // The waves' sums, a panel at a time: [row block][wave][lane].
#pragma unroll
    for (int p = 0; p < P; ++p) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RB; ++i) sums[(i * kDownWaves + wave) * 64 + lane] = acc[i][p];
        __syncthreads();
        if (wave >= RB) continue;
        f32x4 v = sums[wave * kDownWaves * 64 + lane];
#pragma unroll
        for (int w = 1; w < kDownWaves; ++w) v += sums[(wave * kDownWaves + w) * 64 + lane];
        int row = xr[0];
#pragma unroll
        for (int i = 1; i < RB; ++i) row = wave == i ? xr[i] : row;
        const int r = rank0 + p * 16 + q * 4;
        if (row >= 0 && r < rank)
            *(f32x4 *)(args.t + ((int64_t)slice * args.rows + base + row) * args.t_cols + g.t_offset + r) = v * scale;
    }
    __syncthreads();  // (the next adapter's operands go where these sums were)
}

template <int RBMAX, int P, bool FAST>
__global__ void __launch_bounds__(64 * kDownWaves, 2) adapter_down_kernel(AdapterArgs args) {
    __shared__ u32x4 memory[(RBMAX + P) * kDownWaves * 64];
    const int which = blockIdx.z / args.turns, turn = blockIdx.z % args.turns;
    const int column = blockIdx.x / args.slices, slice = blockIdx.x % args.slices;
    const AdapterWeight &g = args.w[which];
    const int rank0 = column * kDownRanks, lane = threadIdx.x & 63;
    if (rank0 >= g.w.max_rank) return;
    // Every lane its row's slot, rank (0: no adapter) and scale.
    const int64_t base = (int64_t)blockIdx.y * kChunk, my_row = base + lane;
    const int slot = my_row < args.rows ? args.slots[my_row] : -1;
    const bool known = slot >= 0 && slot < g.w.count;
    int rank = known ? (g.w.ranks ? g.w.ranks[slot] : (int)g.w.max_rank) : 0;
    const float scale = known && g.w.scales ? g.w.scales[slot] : 1.0f;
    rank = rank < (int)g.w.max_rank ? rank : (int)g.w.max_rank;
    const uint64_t all = __ballot(rank > 0), below = ((uint64_t)1 << lane) - 1;
    uint64_t todo = all;
    for (int part = 0; todo; ++part) {
        const int lead = __builtin_ctzll(todo);
        const int group_slot = __builtin_amdgcn_readlane(slot, lead), group_rank = __builtin_amdgcn_readlane(rank, lead);
        const uint64_t rows = __ballot(rank > 0 && slot == group_slot);
        todo &= ~rows;
        if (part % args.turns != turn || rank0 >= group_rank) continue;
        const int count = __builtin_popcountll(rows);
        const int place = rows >> lane & 1 ? __builtin_popcountll(rows & below)
                                           : count + __builtin_popcountll(~rows & below);
        const int mine = __builtin_amdgcn_ds_permute(place * 4, lane);
        const float group_scale = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(scale), lead));
        if (RBMAX == 1 || count <= 16)
            down_rows<1, P, FAST>(args, g, group_slot, group_rank, group_scale, mine, count, base, rank0, slice, memory);
        else
            down_rows<RBMAX, P, FAST>(args, g, group_slot, group_rank, group_scale, mine, count, base, rank0, slice, memory);
    }
    // The list for the second launch, by one wave of the chunk.
    if (blockIdx.x != 0 || turn != 0 || threadIdx.x >= 64) return;
    ChunkList &list = args.lists[which * (int64_t)gridDim.y + blockIdx.y];
    int first = 0, part = 0;
    for (todo = all; todo; ++part) {
        const int lead = __builtin_ctzll(todo), group_slot = __builtin_amdgcn_readlane(slot, lead);
        const uint64_t rows = __ballot(rank > 0 && slot == group_slot);
        todo &= ~rows;
        if (rows >> lane & 1) list.order[first + __builtin_popcountll(rows & below)] = (uint8_t)lane;
        const int count = __builtin_popcountll(rows);
        if (lane == lead) list.part[part] = {group_slot, (uint16_t)rank, (uint8_t)first, (uint8_t)count};
        first += count;
    }
    if (lane >= part) list.part[lane].rank = 0;
}

// ---- out += b t -----------------------------------------------------------------------------------
//
// A workgroup: one adapter's rows of a chunk, a run of tiles of 256 outputs of one projection, 64 outputs
// a wave. t's slices are summed and laid down in LDS as MFMA operands, in three bf16 pieces of eight bits each, so
// that the products keep all of t's 24. (Two pieces are enough for most bf16 outputs and save 0.3 of 41.4 us for 2048 rows,
// N17408, rank 16; but one value in a thousand is then rounded the other way.)
// b's rows are the MFMA's rows and stay in registers while the adapter's rows go by, sixteen at a time. Their
// sums pass through LDS, so that a wave reads and writes runs of 64 neighbouring outputs of a row: with
// the MFMA's own layout, neighbouring lanes hold different rows, and four times the cache lookups.
//
// Bound by out, read and written, where it is large: 2048 rows, N17408, bf16: 160 MB in 34.6 us (4.6 TB/s, near a large
// copy's 4.95); 64 rows, 2 x 17408, fp32, rank 16: 27 MB in 8.7 us (3.1 TB/s).

constexpr int kPieces = 3;
constexpr int kUpSumStride = 68;  // floats of a row of sums in LDS: 64 and a step of four banks

// The rows of t of a workgroup's blocks of sixteen (block j of its own: from the adapter's row 16 (share + j
// shares) on), summed over the slices, as operands in LDS: [piece][panel of 32 ranks][block][lane] x 16 bytes.
// Four ranks of one row a thread.
__device__ __forceinline__ void stage_t(const AdapterArgs &args, const AdapterWeight &g, int mine, int count,
                                        int blocks, int share, int64_t base, int rank, u32x2 *pieces) {
    constexpr int kAtOnce = 8;
    const int panels = (rank + 31) / 32, quads = panels * 8;
    const int64_t slice_floats = args.rows * args.t_cols;
    for (int item = threadIdx.x; item < blocks * 16 * quads; item += 256) {
        const int i = item / quads, r = (item - i * quads) * 4;
        f32x4 v = {0, 0, 0, 0};
        const int place = (share + (i >> 4) * args.shares) * 16 + (i & 15);
        const int chunk_row = __builtin_amdgcn_ds_bpermute((place & 63) * 4, mine);
        if (place < count && r < rank) {
            const float *t = args.t + (base + chunk_row) * args.t_cols + g.t_offset + r;
            for (int s = 0; s < args.slices; s += kAtOnce) {
                f32x4 part[kAtOnce];
#pragma unroll
                for (int e = 0; e < kAtOnce; ++e)
                    part[e] = *(const f32x4 *)(t + (s + e < args.slices ? s + e : s) * slice_floats);
#pragma unroll
                for (int e = 0; e < kAtOnce; ++e)
                    if (s + e < args.slices) v += part[e];
            }
        }
        float piece[kPieces][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float rest = r + e < rank ? v[e] : 0.0f;
#pragma unroll
            for (int c = 0; c < kPieces; ++c) {
                // (Cut off and not rounded: a finite value's piece is finite. Sums' NaNs are quiet ones, which stay NaN.)
                const float top = __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
                piece[c][e] = top;
                rest = __builtin_fabsf(top) < __builtin_inff() ? rest - top : 0.0f;
            }
        }
        const int at = ((r >> 5) * blocks + (i >> 4)) * 64 + ((r >> 3) & 3) * 16 + (i & 15);
#pragma unroll
        for (int c = 0; c < kPieces; ++c)
            pieces[(c * panels * blocks * 64 + at) * 2 + ((r >> 2) & 1)] =
                u32x2{f32x2_to_bf16x2(piece[c][0], piece[c][1]), f32x2_to_bf16x2(piece[c][2], piece[c][3])};
    }
}

// NP 1: ranks up to 32, b held in registers; NP 0: any rank, b read again for each block of rows (2048 rows of rank
// 16: 34.6 us held, 35.6 read again; holding 64 ranks measured level with reading them again).
template <int NP, typename OUT, bool FAST>
__global__ void __launch_bounds__(256, NP == 1 ? 4 : 3) adapter_up_kernel(AdapterArgs args) {
    constexpr int kLoads = sizeof(OUT), kPer = 16 / sizeof(OUT), kHeld = NP ? NP : 1;
    extern __shared__ u32x4 pieces[];
    __shared__ float sums[4][16 * kUpSumStride];
    const int share = blockIdx.z % args.shares, z = blockIdx.z / args.shares;
    const int which = z / args.turns, turn = z % args.turns;
    const AdapterWeight &g = args.w[which];
    const int column0 = (int)blockIdx.x * args.tiles * kUpColumns, columns = (int)g.w.rows;
    if (column0 >= columns) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, q = lane >> 4;
    const int64_t base = (int64_t)blockIdx.y * kChunk;
    const ChunkList &list = args.lists[which * (int64_t)gridDim.y + blockIdx.y];
    const u32x2 record = *(const u32x2 *)&list.part[lane];
    const int order = list.order[lane], parts = __builtin_popcountll(__ballot((record.y & 0xffffu) != 0));
    OUT *out = (OUT *)g.out + base * g.ldc;
    const rsrc_t ro = make_rsrc(out, FAST ? (uint32_t)(kChunk * g.ldc * sizeof(OUT)) : 0);
    for (int part = turn; part < parts; part += args.turns) {
        const int slot = __builtin_amdgcn_readlane(record.x, part);
        const uint32_t rest = __builtin_amdgcn_readlane(record.y, part);
        const int rank = rest & 0xffffu, first = (rest >> 16) & 0xffu, count = rest >> 24;
        const int blocks = ((count + 15) / 16 - share + args.shares - 1) / args.shares, panels = (rank + 31) / 32;
        if (blocks <= 0) continue;
        const int mine = __builtin_amdgcn_ds_bpermute(((first + lane) & 63) * 4, order);
        const uint16_t *b = g.w.b + slot * g.w.b_slot_stride;
        const rsrc_t rb = make_rsrc(b, FAST ? (uint32_t)(g.w.rows * g.w.b_row_stride * 2) : 0);
        for (int tile = 0; tile < args.tiles; ++tile) {
            const int n0 = column0 + tile * kUpColumns + wave * 64;
            if (n0 - wave * 64 >= columns) break;
            u32x4 bs[kHeld][4];
            auto load_b = [&](int p, u32x4(&v)[4]) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = n0 + j * 16 + m, r = p * 32 + q * 8;
                    if constexpr (FAST)
                        v[j] = buffer_load16(
                            rb, n < columns && r < rank ? (uint32_t)((n * g.w.b_row_stride + r) * 2) : kNowhere, 0);
                    else
                        v[j] = load8(b + n * g.w.b_row_stride + r, n < columns ? rank - r : 0);
                }
            };
            auto past_rank = [&](int p, u32x4(&v)[4]) {
                if (FAST && (rank & 7)) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = keep8(v[j], rank - p * 32 - q * 8);
                }
            };
#pragma unroll
            for (int p = 0; p < NP; ++p) load_b(p, bs[p]);
            if (tile == 0) {
                __syncthreads();  // (the operands before them have been read)
                stage_t(args, g, mine, count, blocks, share, base, rank, (u32x2 *)pieces);
                __syncthreads();
            }
#pragma unroll
            for (int p = 0; p < NP; ++p) past_rank(p, bs[p]);
#pragma unroll 1
            for (int i = 0; i < blocks; ++i) {
                // The outputs to add to: 16 bytes a lane, runs of 64 outputs of a row.
                u32x4 old[kLoads];
                uint32_t at[kLoads];
                int row[kLoads];
#pragma unroll
                for (int c = 0; c < kLoads; ++c) {
                    const int place = (share + i * args.shares) * 16 + (c * 64 + lane) * kPer / 64, n = n0 + lane * kPer % 64;
                    row[c] = __builtin_amdgcn_ds_bpermute((place & 63) * 4, mine);
                    if (place >= count) row[c] = -1;
                    if constexpr (FAST) {
                        at[c] = row[c] >= 0 && n < columns ? (uint32_t)((row[c] * g.ldc + n) * sizeof(OUT)) : kNowhere;
                        old[c] = buffer_load16(ro, at[c], 0);
                    } else if (row[c] >= 0 && n + kPer <= columns) {
                        __builtin_memcpy(&old[c], out + row[c] * g.ldc + n, 16);
                    }
                }
                f32x4 acc[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] = f32x4{0, 0, 0, 0};
                // Sixteen bytes of outputs and their sums, rounded once.
                auto added = [](u32x4 o, const f32x4(&v)[kPer / 4]) {
                    u32x4 w;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (sizeof(OUT) == 4)
                            w[e] = __float_as_uint(__uint_as_float(o[e]) + v[0][e]);
                        else
                            w[e] = f32x2_to_bf16x2(bf16_bits_to_f32(o[e] & 0xffffu) + v[e >> 1][2 * (e & 1)],
                                                   bf16_bits_to_f32(o[e] >> 16) + v[e >> 1][2 * (e & 1) + 1]);
                    }
                    return w;
                };
                auto multiply = [&](int p, const u32x4(&v)[4]) {
#pragma unroll
                    for (int c = 0; c < kPieces; ++c) {
                        const u32x4 t = pieces[((c * panels + p) * blocks + i) * 64 + lane];
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(v[j]), as_bf16x8(t), acc[j], 0, 0, 0);
                    }
                };
                if constexpr (NP > 0) {
#pragma unroll
                    for (int p = 0; p < NP; ++p)
                        if (p < panels) multiply(p, bs[p]);
                } else {
                    for (int p = 0; p < panels; ++p) {
                        load_b(p, bs[0]);
                        past_rank(p, bs[0]);
                        multiply(p, bs[0]);
                    }
                }
                // Column m of the MFMA is a row of the sums here, registers j, e its outputs 16 j + 4 q + e. (A
                // wave's LDS operations are done in order.)
                float *mine_sums = sums[wave];
#pragma unroll
                for (int j = 0; j < 4; ++j) *(f32x4 *)(mine_sums + m * kUpSumStride + j * 16 + q * 4) = acc[j];
                wave_fence();
#pragma unroll
                for (int c = 0; c < kLoads; ++c) {
                    const float *from = mine_sums + (c * 64 + lane) * kPer / 64 * kUpSumStride + lane * kPer % 64;
                    f32x4 v[kPer / 4];
#pragma unroll
                    for (int e = 0; e < kPer / 4; ++e) v[e] = *(const f32x4 *)(from + 4 * e);
                    if constexpr (FAST) {
                        const u32x4 w = added(old[c], v);
                        __builtin_amdgcn_raw_buffer_store_b128(w, ro, (int)at[c], 0, 0);
                    } else if (row[c] >= 0) {
                        const int n = n0 + lane * kPer % 64;
                        OUT *p = out + row[c] * g.ldc + n;
                        if (n + kPer <= columns) {
                            const u32x4 w = added(old[c], v);
                            __builtin_memcpy(p, &w, 16);
                        } else {
#pragma unroll
                            for (int e = 0; e < kPer; ++e) {
                                if (n + e >= columns) continue;
                                if constexpr (sizeof(OUT) == 4) p[e] += v[0][e];
                                else p[e] = f32_to_bf16(bf16_bits_to_f32(p[e]) + v[e >> 2][e & 3]);
                            }
                        }
                    }
                }
                wave_fence();
            }
        }
    }
}

// ---- host -----------------------------------------------------------------------------------------

static int t_columns(const splosh_adapters *w, int group) {
    int cols = 0;
    for (int i = 0; i < group; ++i) cols += (int)(w[i].max_rank + 15) / 16 * 16;
    return cols;
}

static int down_columns(const splosh_adapters &w) { return (int)(w.max_rank + kDownRanks - 1) / kDownRanks; }
static int64_t up_tiles(const splosh_adapters &w) { return (w.rows + kUpColumns - 1) / kUpColumns; }

// Steps of 32 k a slice of K, whole rounds of the workgroup's waves: a workgroup a CU from the chunks and
// projections alone, eight slices at most (the second launch adds them up; K17408, 64 rows of 32 adapters,
// both launches: 4 slices 23.1 us, 8 21.1, 16 23.2).
struct SlicePlan {
    int steps, slices;
};
static SlicePlan plan_slices(const splosh_adapters *w, int group, int64_t rows) {
    const int64_t chunks = (rows + kChunk - 1) / kChunk, steps = (w[0].inner + 31) / 32;
    int64_t others = 0;
    for (int i = 0; i < group; ++i) others += chunks * down_columns(w[i]);
    int64_t want = (256 - 1 + others) / others;
    want = want < 8 ? want : 8;
    const int64_t rounds = (steps + kDownWaves - 1) / kDownWaves, per = (rounds + want - 1) / want;
    return {(int)(per * kDownWaves), (int)((rounds + per - 1) / per)};
}

static size_t lists_bytes(int group, int64_t rows) {
    return (size_t)group * ((rows + kChunk - 1) / kChunk) * sizeof(ChunkList);
}

size_t adapters_workspace_bytes(const splosh_adapters *w, int group, int64_t rows) {
    return kAdapterCounterBytes + lists_bytes(group, rows) +
           (size_t)plan_slices(w, group, rows).slices * rows * t_columns(w, group) * sizeof(float);
}

// A chunk has this many adapters at most (rows and slots bound them).
static int64_t most_parts(const splosh_adapters *w, int group, int64_t rows) {
    int64_t count = 1;
    for (int i = 0; i < group; ++i) count = w[i].count > count ? w[i].count : count;
    const int64_t most = rows < kChunk ? rows : kChunk;
    return count < most ? count : most;
}

// The adapters of a chunk go to up to this many workgroups: each its own where the launch is small, several to one
// where it fills the device anyway: eight workgroups a CU (64 rows of eight, K5120 -> 2 x 17408, the second launch:
// 8.4 us, two a CU 12.0).
static int plan_turns(int64_t parts, int64_t others) {
    const int64_t n = 2048 / others;
    return (int)(n < 1 ? 1 : n < parts ? n : parts);
}

template <int RB, bool FAST>
static void launch_down(const AdapterArgs &args, int panels, dim3 grid, hipStream_t stream) {
    if (panels == 1) hipLaunchKernelGGL((adapter_down_kernel<RB, 1, FAST>), grid, dim3(64 * kDownWaves), 0, stream, args);
    else hipLaunchKernelGGL((adapter_down_kernel<RB, 2, FAST>), grid, dim3(64 * kDownWaves), 0, stream, args);
}

// LDS of the operands: their pieces of whole panels of ranks for a chunk's rows; past the default limit of 64 KB with
// what the kernel has of its own, the limit is raised once.
constexpr int kUpMaxLds = kPieces * (SPLOSH_MAX_RANK / 32) * (kChunk / 16) * 1024;

template <int NP, typename OUT, bool FAST>
static hipError_t launch_up(const AdapterArgs &args, int lds, dim3 grid, hipStream_t stream) {
    if (NP == 0) {
        static const hipError_t raised = hipFuncSetAttribute((const void *)adapter_up_kernel<NP, OUT, FAST>,
                                                             hipFuncAttributeMaxDynamicSharedMemorySize, kUpMaxLds);
        if (raised != hipSuccess) return raised;
    }
    hipLaunchKernelGGL((adapter_up_kernel<NP, OUT, FAST>), grid, dim3(256), lds, stream, args);
    return hipGetLastError();
}
template <typename OUT>
static hipError_t launch_up(const AdapterArgs &args, int panels, bool fast, int lds, dim3 grid, hipStream_t stream) {
    if (!fast) return panels == 1 ? launch_up<1, OUT, false>(args, lds, grid, stream)
                                  : launch_up<0, OUT, false>(args, lds, grid, stream);
    if (panels == 1) return launch_up<1, OUT, true>(args, lds, grid, stream);
    return launch_up<0, OUT, true>(args, lds, grid, stream);
}

hipError_t launch_adapters(const splosh_adapters *w, int group, const uint16_t *x, int64_t ldx, void *const *outs,
                           const int64_t *ldcs, int out_dtype, const int32_t *slots, int64_t rows, void *workspace,
                           hipStream_t stream) {
    AdapterArgs args{};
    args.x = x;
    args.ldx = ldx;
    args.slots = slots;
    args.lists = (ChunkList *)((char *)workspace + kAdapterCounterBytes);
    args.t = (float *)((char *)workspace + kAdapterCounterBytes + lists_bytes(group, rows));
    args.t_cols = t_columns(w, group);
    const SlicePlan plan = plan_slices(w, group, rows);
    args.slices = plan.slices;
    args.slice_steps = plan.steps;
    args.rows = rows;
    const int64_t esize = out_dtype == SPLOSH_F32 ? 4 : 2;
    auto aligned16 = [](const void *p, int64_t a, int64_t b) { return (uintptr_t)p % 16 == 0 && a % 8 == 0 && b % 8 == 0; };
    auto near = [](int64_t n, int64_t stride, int64_t size) { return stride < (int64_t)kNowhere / size / n; };
    bool down_fast = aligned16(x, ldx, w[0].inner) && near(kChunk, ldx, 2), up_fast = true;
    int at = 0, columns = 0;
    int64_t most_rank = 0, tiles = 0, most_tiles = 0;
    for (int i = 0; i < group; ++i) {
        args.w[i] = AdapterWeight{w[i], outs[i], ldcs[i], at};
        at += (int)(w[i].max_rank + 15) / 16 * 16;
        columns = columns > down_columns(w[i]) ? columns : down_columns(w[i]);
        most_rank = w[i].max_rank > most_rank ? w[i].max_rank : most_rank;
        tiles += up_tiles(w[i]);
        most_tiles = up_tiles(w[i]) > most_tiles ? up_tiles(w[i]) : most_tiles;
        down_fast = down_fast && aligned16(w[i].a, w[i].a_slot_stride, w[i].a_row_stride) &&
                    near(w[i].max_rank, w[i].a_row_stride, 2);
        up_fast = up_fast && (uintptr_t)outs[i] % 16 == 0 && ldcs[i] % (16 / esize) == 0 && w[i].rows % 16 == 0 &&
                  w[i].max_rank % 8 == 0 && near(kChunk, ldcs[i], esize) &&
                  aligned16(w[i].b, w[i].b_slot_stride, w[i].b_row_stride) && near(w[i].rows, w[i].b_row_stride, 2);
    }
    const unsigned chunks = (unsigned)((rows + kChunk - 1) / kChunk);
    const unsigned down_x = (unsigned)(columns * args.slices);
    const int64_t parts = most_parts(w, group, rows);
    args.turns = plan_turns(parts, (int64_t)down_x * chunks * group);
    const dim3 down(down_x, chunks, (unsigned)(group * args.turns));
    const int panels = most_rank <= 16 ? 1 : 2;
    if (rows <= 16) {
        if (down_fast) launch_down<1, true>(args, panels, down, stream);
        else launch_down<1, false>(args, panels, down, stream);
    } else {
        if (down_fast) launch_down<4, true>(args, panels, down, stream);
        else launch_down<4, false>(args, panels, down, stream);
    }
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    // Tiles a workgroup, for which t is staged once: so many that six workgroups a CU are left (2048 rows,
    // N17408: two tiles 34.1 us, one 40.9, four 34.2; 64 rows, 2 x 17408: one tile 8.2, four 12.0).
    const int64_t share = (tiles * chunks * (chunks == 1 ? parts : 1) + 1535) / 1536;
    args.tiles = (int)(share < most_tiles ? share : most_tiles);
    const unsigned up_x = (unsigned)((most_tiles + args.tiles - 1) / args.tiles);
    // More than 16 rows an adapter: its rows in shares, a block of sixteen each (fp32, K6144 -> N5120: 333 rows of three
    // adapters of rank 64: 9.5 us, one workgroup for all of a chunk's rows 15.2; 500 of two, rank 128: 16.2 and 23.5).
    args.shares = rows <= 16 * parts ? 1 : rows <= 32 ? 2 : 4;
    args.turns = plan_turns(parts, (int64_t)up_x * chunks * group * args.shares);
    const dim3 up(up_x, chunks, (unsigned)(group * args.turns * args.shares));
    const int up_panels = (int)(most_rank + 31) / 32, blocks = rows < kChunk ? (int)(rows + 15) / 16 : kChunk / 16;
    const int lds = kPieces * up_panels * ((blocks + args.shares - 1) / args.shares) * 1024;
    return out_dtype == SPLOSH_F32 ? launch_up<float>(args, up_panels, up_fast, lds, up, stream)
                                   : launch_up<uint16_t>(args, up_panels, up_fast, lds, up, stream);
}

}  // namespace splosh
