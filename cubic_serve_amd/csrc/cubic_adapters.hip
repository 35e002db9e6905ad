// Low-rank adapters of many requests beside a shared projection (gfx950):
//
//   t[i, :]   = A_e x[i, :]                         e = row_slots[i], rank r_e
//   y[i, :]   = round16(base[i, :] + s_e B_e t[i, :])
//
// for up to kMaxGemmMembers projections that share x.  Few rows: one launch
// (adapter_row_kernel).  Else a down kernel writes t as binary32 partial sums over K
// partitions and an up kernel adds them and finishes the rows; where column chunks
// would add them much again, a launch between the two does (adapter_join_kernel).
//
// Rows come in any order, without a grouping launch or any host knowledge of
// the slots.  Batches of some size are tiled in order of adapters, each
// workgroup finding its tile's rows by itself (slot_rows): an adapter is then
// read once per 16 of its rows, wherever they lie.  Else a tile of consecutive
// rows is walked once per distinct adapter in it (a ballot over the tile's slots
// finds the rows of each); a prompt's rows share one.  `groups` workgroups may
// share such a tile's adapters: number j takes those at j, j + groups, ...
//
// Arithmetic order: K partitions of kDownK columns, each a sum of four quarters
// (0 + 1) + (2 + 3), partitions added in ascending order; then the rank in steps
// of 32.  Nothing of it depends on m, on the kernel, on the tile or on the
// other rows, so a row's result is the same bit for bit whichever batch it is in.
#include "cubic_gemm_common.h"

namespace cubic {
namespace {

using gemm::floatx4_t;
using gemm::mfma16;

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kDownK = kAdapterDownK;       // columns of x per K partition
constexpr int kQuarter = kDownK / 4;
constexpr int kSteps = kQuarter / 32;       // MFMA steps of a quarter
constexpr uint32_t kOutside = 0x80000000u;  // added to a byte offset: past every buffer, reads 0

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}

__device__ __forceinline__ uint4 load16(__amdgpu_buffer_rsrc_t r, uint32_t byte_offset) {
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)byte_offset, 0, 0));
}

typedef __attribute__((address_space(3))) void lds_void_t;
// s_waitcnt immediate: at most n vector-memory accesses in flight, no LDS access.
constexpr int vmcnt_and_lds(int n) { return (n & 0xF) | (0x7 << 4) | ((n >> 4) << 14); }
constexpr int kParts = 3;          // 16-bit parts of t in the second product
constexpr int kDownTileRanks = 8;  // 16-rank blocks of the prompts' down kernel

// The tile's adapter slots, one per lane (-1: past the batch, kNone: no
// adapter), the same in every wave: one wave reads them, so that waves cannot
// disagree on the walk (and its barriers) if the caller rewrites them meanwhile.
constexpr int kNone = -2;
__device__ __forceinline__ int row_slot(const AdapterArgs& a, int row0, int rows, int lane) {
    if (lane >= rows || row0 + lane >= a.m) return -1;
    const int slot = a.row_slots[row0 + lane];
    return slot < 0 || slot >= a.slots ? kNone : slot;
}
__device__ __forceinline__ int tile_slots(const AdapterArgs& a, int row0, int rows, int* lds) {
    if (threadIdx.x < 64) lds[threadIdx.x] = row_slot(a, row0, rows, threadIdx.x);
    __syncthreads();
    return lds[threadIdx.x & 63];
}

// Rows in order of adapters (at most 1024 rows, 255 adapters, those without one
// last): item w is the wth tile of up to 16 rows that share an adapter.  Returns
// it (-1: no such item) and leaves the tile's rows in lds.rows, -1 behind them.
// Ranks within an adapter are the rows' order, so that every workgroup finds the
// same tiles.  A barrier has to precede another call.
struct SlotRows { int count[kThreads], sums[kWaves], slot, tile, rows[16]; };
__device__ __forceinline__ int slot_rows(const AdapterArgs& a, int w, SlotRows& lds) {
    constexpr int kRows = 4;  // rows per thread
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    int slot[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int row = wave * 64 * kRows + i * 64 + lane;
        slot[i] = row < a.m ? a.row_slots[row] : -1;
        if (row < a.m && (slot[i] < 0 || slot[i] >= a.slots)) slot[i] = a.slots;
    }
    lds.count[t] = 0;
    if (t < 16) lds.rows[t] = -1;
    if (t == 0) lds.slot = -1;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRows; ++i)
        if (slot[i] >= 0) atomicAdd(&lds.count[slot[i]], 1);
    __syncthreads();
    const int tiles = (lds.count[t] + 15) / 16;
    int before = (int)wave_scan_u32((uint32_t)tiles);
    if (lane == 63) lds.sums[wave] = before;
    before -= tiles;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) before += i < wave ? lds.sums[i] : 0;
    if (before <= w && w < before + tiles) {
        lds.slot = t;
        lds.tile = w - before;
    }
    __syncthreads();
    const int e = lds.slot;
    if (e < 0) return -1;
    uint64_t hits[kRows];
    int held = 0;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        hits[i] = __ballot(slot[i] == e);
        held += __popcll(hits[i]);
    }
    if (lane == 0) lds.sums[wave] = held;
    __syncthreads();
    int at = -16 * lds.tile;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) at += i < wave ? lds.sums[i] : 0;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int mine = at + __popcll(hits[i] & ((1ull << lane) - 1));
        if (slot[i] == e && mine >= 0 && mine < 16) lds.rows[mine] = wave * 64 * kRows + i * 64 + lane;
        at += __popcll(hits[i]);
    }
    __syncthreads();
    return e == a.slots ? kNone : e;
}

// One quarter of t for 16 * MT rows x RT 16-rank tiles, every load in flight at
// once.  MFMA operands straight from memory: the first is A (its rows are the
// ranks), the second x, so a lane ends with four consecutive ranks of one row.
// x goes out ahead of A in runs of four steps (256 bytes of every row).
// behind() runs once they have, before any is waited for.
template <bool F16, int MT, int RT, typename Behind>
__device__ __forceinline__ void quarter_product(__amdgpu_buffer_rsrc_t x, const uint32_t (&xoff)[MT],
                                                __amdgpu_buffer_rsrc_t d, const uint32_t (&doff)[RT], int k0,
                                                int k, floatx4_t (&acc)[MT][RT], Behind&& behind) {
    uint4 xf[kSteps][MT], df[kSteps][RT];
#pragma unroll
    for (int h = 0; h < kSteps; h += 4) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int s = h; s < h + 4; ++s) {
                const int kk = k0 + s * 32;
                xf[s][i] = load16(x, kk < k ? xoff[i] + (uint32_t)kk * 2 : kOutside);
            }
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int s = h; s < h + 4; ++s) {
                const int kk = k0 + s * 32;
                df[s][t] = load16(d, kk < k && doff[t] != kOutside ? doff[t] + (uint32_t)kk * 2 : kOutside);
            }
    }
    __builtin_amdgcn_sched_barrier(0);
    behind();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[i][t] = floatx4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[i][t] = mfma16<F16>(df[s][t], xf[s][i], acc[i][t]);
}

// ---------------------------------------------------------------------------
// t = A x into the partial sums.  Workgroup: 16 * MT rows x RT rank tiles x one K
// partition, a quarter per wave.
// ---------------------------------------------------------------------------
template <bool F16, int MT, int RT>
__global__ __launch_bounds__(kThreads) void adapter_down_kernel(AdapterArgs a) {
    constexpr int kRows = 16 * MT;
    __shared__ union {
        int slots[64];
        SlotRows rows;
    } walk;
    __shared__ floatx4_t red[2][MT * RT][64];
    const AdapterMember& mb = a.member[blockIdx.z];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, q = lane >> 4;
    // K partitions first: workgroups that run together spread over all of a
    // row (tiles first, they meet on the few memory channels of one column
    // range: 4096 x 8192 at rank 128, 76 -> 57 us)
    const int part = blockIdx.x % a.split, item = blockIdx.x / a.split;
    const int tile = item / a.down_groups, group = item % a.down_groups;
    const int rank0 = blockIdx.y * RT * 16;
    if (rank0 >= mb.max_rank) return;
    // this lane's row, 16 i + col of the tile, from row0 on
    int row0 = tile * kRows, rows = min(kRows, a.m - row0), slot, row[MT];
    if (MT == 1 && a.items) {
        const int e = slot_rows(a, item, walk.rows);
        if (e < 0) return;  // no such tile, or one without an adapter
        row0 = 0;
        rows = a.m;
        slot = lane < 16 && walk.rows.rows[lane] >= 0 ? e : -1;
        row[0] = walk.rows.rows[col];
    } else {
        slot = tile_slots(a, row0, kRows, walk.slots);
#pragma unroll
        for (int i = 0; i < MT; ++i) row[i] = 16 * i + col;
    }
    const auto x = buffer(a.x + (int64_t)row0 * a.ldx, ((int64_t)(rows - 1) * a.ldx + a.k) * 2);
    const int k0 = part * kDownK + wave * kQuarter + q * 8;
    uint64_t left = __ballot(slot >= 0);
    for (int order = 0; left; ++order) {
        const int lead = __builtin_ctzll(left);
        const int e = __builtin_amdgcn_readlane(slot, lead);
        const uint64_t mine = __ballot(slot == e);
        left &= ~mine;
        if (order % a.down_groups != group) continue;
        const int first = MT == 1 ? __builtin_amdgcn_readlane(row[0], lead) : lead;
        // rows of other adapters repeat the first row: their columns of the
        // product are not stored
        uint32_t xoff[MT], doff[RT];
#pragma unroll
        for (int i = 0; i < MT; ++i)
            xoff[i] = (uint32_t)((mine >> (16 * i + col)) & 1 ? row[i] : first) * (uint32_t)(a.ldx * 2);
        // the first tile does not wait for the slot's rank (what lies past it
        // the up kernel leaves out); the others are read only below it
        const int rank = RT > 1 || rank0 ? min(mb.ranks[e], mb.max_rank) : mb.max_rank;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int r = rank0 + 16 * t + col;
            doff[t] = r < (rank0 + t == 0 ? mb.max_rank : rank) ? (uint32_t)r * (uint32_t)(a.k * 2) : kOutside;
        }
        const auto d = buffer(mb.down + (int64_t)e * mb.max_rank * a.k, (int64_t)mb.max_rank * a.k * 2);
        floatx4_t acc[MT][RT];
        quarter_product<F16, MT, RT>(x, xoff, d, doff, k0, a.k, acc, [] {});
        // (0 + 1) + (2 + 3); the walk's next turn writes red only after the
        // last barrier, which follows every read of it
        if (wave & 1)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int t = 0; t < RT; ++t) red[wave >> 1][i * RT + t][lane] = acc[i][t];
        __syncthreads();
        if (!(wave & 1))
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int t = 0; t < RT; ++t) acc[i][t] += red[wave >> 1][i * RT + t][lane];
        __syncthreads();
        if (wave == 2)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int t = 0; t < RT; ++t) red[0][i * RT + t][lane] = acc[i][t];
        __syncthreads();
        if (wave == 0)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if (!((mine >> (16 * i + col)) & 1)) continue;
                float* out = a.partial + ((int64_t)part * a.m + row0 + row[i]) * a.width + mb.rank0 + rank0 + 4 * q;
#pragma unroll
                for (int t = 0; t < RT; ++t)
                    if (rank0 + 16 * t < mb.max_rank)
                        *(floatx4_t*)(out + 16 * t) = acc[i][t] + red[0][i * RT + t][lane];
            }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// t = A x for prompts: the same sums over tiles of 64 rows and 128 ranks, x and A
// staged through LDS by direct loads, blocks of 64 columns, three deep (72 KB:
// two workgroups per CU).  The kernel above has each wave read A from the caches for
// its own 32 rows: at K = 8192, rank 128, 4096 rows that is 0.4 GB into the CUs
// beside 0.07 from memory.  Here waves share the ranks in halves and the rows in
// halves, and A is read once per 64 rows: 54 -> 27.5 us with one adapter.  A tile on a
// boundary is done once per adapter, at the end alone on its CU: with two requests
// and up 39 to 52 (workgroups of their own for the second adapter wait for a place
// until the others end: 44 and 41 with three requests).  Four blocks make a
// quarter; quarters add as above, bit for bit.  LDS image of a 16-row block: 16-byte
// chunk c of row r in slot 8 r + (c ^ (r / 2) mod 8), so that the 16 rows of a
// fragment read lie in distinct banks.
// ---------------------------------------------------------------------------
template <bool F16>
__global__ __launch_bounds__(kThreads) void adapter_down_tile_kernel(AdapterArgs a) {
    constexpr int RT = kDownTileRanks, S = 3;  // two blocks in flight; 72 KB: two workgroups per CU
    constexpr int kBlock = 64, kBlocks = kDownK / kBlock, kBytes = 16 * kBlock * 2;
    constexpr int kStage = (4 + RT) * kBytes;  // four row blocks, RT rank blocks
    constexpr int kDown = RT / 2;              // 1 KB loads of A per wave and stage; two of x
    constexpr int RW = RT / 2;                 // rank blocks per wave; two row blocks
    __shared__ int slots_lds[64];
    __shared__ __attribute__((aligned(16))) uint8_t stage[S * kStage];
    const AdapterMember& mb = a.member[blockIdx.z];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, q = lane >> 4;
    const int wr = wave >> 1, wc = wave & 1;
    const int part = blockIdx.x % a.split, row0 = (int)(blockIdx.x / a.split) * 64;
    const int rank0 = blockIdx.y * RT * 16;
    if (rank0 >= mb.max_rank) return;
    const int slot = tile_slots(a, row0, 64, slots_lds);

    const int rows = min(64, a.m - row0);
    const __amdgpu_buffer_rsrc_t x = buffer(a.x + (int64_t)row0 * a.ldx, ((int64_t)(rows - 1) * a.ldx + a.k) * 2);
    // this lane's place in a 1 KB load: rows 8 i + lane / 8 of a block
    const int dr = lane >> 3;
    auto chunk_of = [&](int r) { return (lane & 7) ^ (r >> 1 & 7); };

    uint64_t left = __ballot(slot >= 0);
    while (left) {
        const int e = __builtin_amdgcn_readlane(slot, __builtin_ctzll(left));
        const uint64_t mine = __ballot(slot == e);
        left &= ~mine;
        const int rank = min(mb.ranks[e], mb.max_rank);
        const __amdgpu_buffer_rsrc_t d = buffer(mb.down + (int64_t)e * mb.max_rank * a.k, (int64_t)mb.max_rank * a.k * 2);
        // x: wave w's loads are the two halves of row block w; a block without a
        // row of this adapter is not read
        const bool need = (mine >> (16 * wave) & 0xffff) != 0;
        uint32_t xoff[2], doff[kDown];
#pragma unroll
        for (int i = 0; i < 2; ++i) xoff[i] = need ? (uint32_t)(16 * wave + 8 * i + dr) * (uint32_t)(a.ldx * 2) : kOutside;
#pragma unroll
        for (int i = 0; i < kDown; ++i) {
            const int r = rank0 + 8 * (wave * kDown + i) + dr;
            doff[i] = r < rank ? (uint32_t)r * (uint32_t)(a.k * 2) : kOutside;
        }
        // K block b into stage b % S; past the partition: reads nothing, writes 0
        auto issue = [&](int b) {
            auto* to = (__attribute__((address_space(3))) uint8_t*)(void*)(stage + b % S * kStage);
            // (named operands: the host pass drops a kernel that passes array elements here)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int kk = part * kDownK + b * kBlock + chunk_of(8 * i + dr) * 8;
                const uint32_t off = b < kBlocks && kk < a.k && xoff[i] != kOutside ? xoff[i] + (uint32_t)kk * 2 : kOutside;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(x, (lds_void_t*)(to + (2 * wave + i) * 1024), 16, off, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < kDown; ++i) {
                const int at = wave * kDown + i;  // half block of A
                const int kk = part * kDownK + b * kBlock + chunk_of(8 * (at & 1) + dr) * 8;
                const uint32_t off = b < kBlocks && kk < a.k && doff[i] != kOutside ? doff[i] + (uint32_t)kk * 2 : kOutside;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (lds_void_t*)(to + 4 * kBytes + at * 1024), 16, off, 0, 0, 0);
            }
        };
        floatx4_t sum[2][RW], even[2][RW], acc[2][RW];
#pragma unroll
        for (int b = 0; b < S - 1; ++b) {
            issue(b);
            __builtin_amdgcn_sched_barrier(0);  // in the order in which they are waited for
        }
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            // this wave's loads of block b have landed (S - 2 younger blocks may
            // be in flight); after the barrier every wave's have, and every wave
            // is done with the stage that block b + S - 1 takes
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(vmcnt_and_lds((S - 2) * (2 + kDown)));
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            issue(b + S - 1);
            __builtin_amdgcn_sched_barrier(0);
            const uint8_t* from = stage + b % S * kStage + col * 128;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int at = ((4 * s + q) ^ (col >> 1)) * 16;
                uint4 xf[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) xf[i] = *(const uint4*)(from + (2 * wr + i) * kBytes + at);
#pragma unroll
                for (int t = 0; t < RW; ++t) {
                    const uint4 df = *(const uint4*)(from + (4 + wc * RW + t) * kBytes + at);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (b % 4 == 0 && s == 0) acc[i][t] = floatx4_t{0.f, 0.f, 0.f, 0.f};
                        acc[i][t] = mfma16<F16>(df, xf[i], acc[i][t]);
                    }
                }
            }
            if (b % 4 == 3)  // a quarter is whole
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int t = 0; t < RW; ++t) {
                        if (b % 8 == 3) even[i][t] = acc[i][t];
                        else if (b == 7) sum[i][t] = even[i][t] + acc[i][t];
                        else sum[i][t] += even[i][t] + acc[i][t];
                    }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 16 * (2 * wr + i) + col;
            if (!((mine >> r) & 1)) continue;
            float* out = a.partial + ((int64_t)part * a.m + row0 + r) * a.width + mb.rank0 + rank0 + 4 * q;
#pragma unroll
            for (int t = 0; t < RW; ++t) {
                const int f = 16 * (wc * RW + t);
                if (rank0 + f < mb.max_rank) *(floatx4_t*)(out + f) = sum[i][t];
            }
        }
        // no load into LDS is left when the next adapter's, or the kernel's end, comes
        __builtin_amdgcn_s_waitcnt(vmcnt_and_lds(0));
        __syncthreads();
    }
}

// t itself, the partitions added in ascending order, in place of the first: every
// column chunk of the up kernel would read them all (8192 columns, 8 partitions:
// 0.16 GB of partitions beside the 0.13 of base and y).
__global__ __launch_bounds__(kThreads) void adapter_join_kernel(AdapterArgs a) {
    const int64_t words = (int64_t)a.m * a.width;
    const int64_t at = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 4;
    if (at >= words) return;
    constexpr int kAhead = 8;
    floatx4_t v = *(const floatx4_t*)(a.partial + at);
    for (int part = 1; part < a.split; part += kAhead) {
        floatx4_t in[kAhead];
#pragma unroll
        for (int p = 0; p < kAhead; ++p) in[p] = *(const floatx4_t*)(a.partial + at + min(part + p, a.split - 1) * words);
#pragma unroll
        for (int p = 0; p < kAhead; ++p)
            if (part + p < a.split) v += in[p];
    }
    *(floatx4_t*)(a.partial + at) = v;
}

// ---------------------------------------------------------------------------
// y = base + s B t.  A wave takes 16 rows x kTurn columns per turn; the four
// waves of a workgroup stand side by side over columns (WR = 1: few rows) or
// one below the other (WR = 4: they read the same B, which their CU's cache
// holds).  The first MFMA operand is B, so a lane ends with four consecutive
// columns of one row; the product passes through LDS (the wave's own, no
// barrier) so that base and y move as whole 256-byte pieces of rows: a copy in
// that pattern runs at 4.6 - 4.8 TB/s where 64-byte pieces of 16 rows, which
// the product's own layout gives, run at 3.1 - 3.7 (2048 x 24576 and 4096 x 8192).
//
// t is split into three 16-bit parts whose sum is all its 24 bits, so that the only
// rounding to 16 bits is y's: with two, 2^-17 of t, what is left where the base
// cancels the adapter is off by up to eleven times what binary32 allows.  The third
// product and the longer split cost 0 to 2 %, at rank 128 1 to 4 % (4096 rows x 8192
// columns, K = 8192, 104 -> 108 us; 2048 rows, K = 4096 39.9 -> 40.3).  All parts of a
// value have its sign and none is 0 unless it is, so that a product with an
// infinity of B is that infinity in each, as in the formula.  fp16 parts are taken of
// t scaled by a power of two, its row's largest into [2^14, 2^15), which fp16's range
// needs and which changes no digit of the product.
// ---------------------------------------------------------------------------
// Eight values t into their parts: each is what is left of t, cut to 16 bits
// towards 0, so that all have t's sign, and at least a trifle (2^-30 of t, fp16:
// 2^-24), so that none is 0 unless t is.
template <bool F16>
__device__ __forceinline__ void split_parts(const float* t, uint4 (&part)[kParts]) {
    uint32_t h[kParts][4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        float rest[2], least[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const float x = t[2 * p + c];
            least[c] = F16 ? __builtin_amdgcn_fmed3f(x * 0x1p60f, -0x1p-24f, 0x1p-24f) : x * 0x1p-30f;
            rest[c] = F16 ? x + least[c] : x;
        }
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            float cut[2];
            if constexpr (F16) {
                h[i][p] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(rest[0], rest[1]));
                cut[0] = half_bits_to_float(h[i][p] & 0xffffu);
                cut[1] = half_bits_to_float(h[i][p] >> 16);
            } else {
                cut[0] = __uint_as_float(__float_as_uint(rest[0]) & 0xffff0000u);
                cut[1] = __uint_as_float(__float_as_uint(rest[1]) & 0xffff0000u);
                h[i][p] = __builtin_amdgcn_perm(__float_as_uint(rest[1]), __float_as_uint(rest[0]), 0x07060302u);
            }
            if (i == kParts - 1) break;
            // the middle one: least <= rest - cut <= t in size; of an infinity the
            // difference is NaN, and the result the smaller of the other two, itself
#pragma unroll
            for (int c = 0; c < 2; ++c) rest[c] = __builtin_amdgcn_fmed3f(rest[c] - cut[c], least[c], t[2 * p + c]);
        }
    }
#pragma unroll
    for (int i = 0; i < kParts; ++i) part[i] = uint4{h[i][0], h[i][1], h[i][2], h[i][3]};
}

// The parts of a row of t (this lane's eight ranks of every step; lanes of one
// column hold the row): scaled, cut at the rank; returns what the product has
// to be multiplied by.
template <bool F16, int KS>
__device__ __forceinline__ float split_row(const floatx4_t (&v)[KS][2], int rank, float scale, int q,
                                           uint4 (&t16)[KS][kParts]) {
    float t[KS][8];
    float top = 0.f, back = 1.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            t[s][c] = s * 32 + q * 8 + c < rank ? v[s][c >> 2][c & 3] * scale : 0.f;
            top = fmaxf(top, fabsf(t[s][c]));
        }
    if constexpr (F16) {
        top = fmaxf(top, __uint_as_float(xor16_u32(__float_as_uint(top))));
        top = fmaxf(top, __uint_as_float(xor32_u32(__float_as_uint(top))));
        // the row's largest into [2^14, 2^15), the scale kept within normal numbers
        int ex = (int)(__float_as_uint(top) >> 23) - 126;
        ex = top == 0.f || !__builtin_isfinite(top) ? 15 : max(ex, -105);
        const float down = __uint_as_float((uint32_t)(127 + 15 - ex) << 23);
        back = __uint_as_float((uint32_t)(127 - 15 + ex) << 23);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int c = 0; c < 8; ++c) t[s][c] *= down;
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) split_parts<F16>(t[s], t16[s]);
    return back;
}

// The parts of t of this lane's row (row0 + row, if own; rows of them from row0 on
// are there): the partitions in ascending order, kAhead requested together (four
// of 32 ranks: 26.0 us of 256 rows, rank 64, K = 12288, with eight 26.3, sixteen 27.5; what
// the registers cost is more than the wait); what is not there (another row, past
// the rank) reads as 0.
template <bool F16, int KS, int kAhead>
__device__ __forceinline__ float row_parts(const AdapterArgs& a, const AdapterMember& mb, int row0, int rows, int row,
                                           bool own, int rank, float scale, int q, uint4 (&t16)[KS][kParts]) {
    uint32_t off[KS][2];
    floatx4_t v[KS][2];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int f = s * 32 + q * 8 + 4 * c;
            off[s][c] = own && f < rank ? (uint32_t)(row * a.width + mb.rank0 + f) * 4 : kOutside;
            v[s][c] = floatx4_t{0.f, 0.f, 0.f, 0.f};
        }
    for (int part = 0; part < a.split; part += kAhead) {
        floatx4_t in[kAhead][KS][2];
#pragma unroll
        for (int p = 0; p < kAhead; ++p) {
            const int64_t at = ((int64_t)min(part + p, a.split - 1) * a.m + row0) * a.width;
            const auto buf = buffer(a.partial + at, part + p < a.split ? (int64_t)rows * a.width * 4 : 0);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int c = 0; c < 2; ++c) in[p][s][c] = __builtin_bit_cast(floatx4_t, load16(buf, off[s][c]));
        }
#pragma unroll
        for (int p = 0; p < kAhead; ++p)
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int c = 0; c < 2; ++c) v[s][c] += in[p][s][c];
    }
    return split_row<F16, KS>(v, rank, scale, q, t16);
}

// Rows of base or y from the tile's first on, and eight 16-bit values of one (its
// byte offset, or kOutside: reads what is not used, writes nothing) at column c.
// VEC: rows and columns in 16-byte words, past the row reads 0 and is not written.  Else
// the words lie anywhere: one access all the same, a row's last word read where
// it ends and moved into place; element by element (1218 rows x 27723 columns 117 us
// against 66) only to write that and where a row is shorter than a word.
struct __attribute__((packed, aligned(2))) AnyWord { uint32_t w[4]; };
template <bool VEC>
struct Rows {
    __amdgpu_buffer_rsrc_t r;
    uint8_t* p;
    __device__ __forceinline__ Rows(const uint16_t* first, int64_t bytes) : r(buffer(first, bytes)), p((uint8_t*)first) {}
};
template <bool VEC>
__device__ __forceinline__ uint4 load8(const Rows<VEC>& rows, uint32_t row, int c, int n) {
    if constexpr (VEC) {
        return load16(rows.r, row + 2 * c);
    } else {
        const uint8_t* from = rows.p + (row == kOutside ? 0 : row);
        if (n < 8) {
            uint32_t v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = c + i < n ? ((const uint16_t*)from)[c + i] : 0;
            return uint4{v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16};
        }
        const int past = max(c - (n - 8), 0);
        const AnyWord w = *(const AnyWord*)(from + 2 * (c - past));
        if (past <= 0 || past >= 8) return uint4{w.w[0], w.w[1], w.w[2], w.w[3]};
        unsigned __int128 x = ((unsigned __int128)((uint64_t)w.w[3] << 32 | w.w[2]) << 64) | ((uint64_t)w.w[1] << 32 | w.w[0]);
        x >>= 16 * past;
        return uint4{(uint32_t)x, (uint32_t)(x >> 32), (uint32_t)(x >> 64), (uint32_t)(x >> 96)};
    }
}

template <bool VEC>
__device__ __forceinline__ void store8(const Rows<VEC>& rows, uint32_t row, int c, int n, uint4 v) {
    if constexpr (VEC) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_dev_t, v), rows.r, (int)(row + 2 * c), 0, 0);
    } else {
        if (row == kOutside) return;
        uint8_t* to = rows.p + row;
        if (c + 8 <= n) {
            *(AnyWord*)(to + 2 * c) = AnyWord{{v.x, v.y, v.z, v.w}};
            return;
        }
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < n) ((uint16_t*)to)[c + i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
    }
}

// Eight values of LDS at column c = 0, 8, ...: every other four lanes take their
// second half first, so that the eight lanes of a pass lie in distinct banks.
__device__ __forceinline__ void eight_of(const float* from, int c, floatx4_t& d0, floatx4_t& d1) {
    const int first = c >> 3 & 4;
    const floatx4_t a = *(const floatx4_t*)(from + first), b = *(const floatx4_t*)(from + (first ^ 4));
    d0 = first ? b : a;
    d1 = first ? a : b;
}

// Two 16-bit values plus two binary32 ones, each sum rounded once.
template <bool F16>
__device__ __forceinline__ uint32_t add_pair(uint32_t in, float lo, float hi) {
    if constexpr (F16) return gemm::pack_level2<true>(half_bits_to_float(in & 0xffffu) + lo, half_bits_to_float(in >> 16) + hi);
    else return gemm::pack_level2<false>(bf16_bits_to_float(in & 0xffffu) + lo, __uint_as_float(in & 0xffff0000u) + hi);
}

template <bool F16, int KS, int WR, bool VEC>
// (two waves per SIMD, 256 registers; fp16 prompts of more than 128 ranks do not fit them)
__global__ __launch_bounds__(kThreads, F16 && KS == 8 && WR == 4 ? 1 : 2) void adapter_up_kernel(AdapterArgs a) {
    constexpr int kColWaves = kWaves / WR;  // waves side by side
    constexpr int kTurn = kAdapterUpTurn, kPitch = kTurn + 4;
    __shared__ __attribute__((aligned(16))) float product[kWaves][16][kPitch];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, q = lane >> 4;
    const int chunk = blockIdx.x % a.chunks, item = blockIdx.x / a.chunks;
    const int tile = item / a.up_groups, group = item % a.up_groups;
    // every wave walks its own rows, or all the item's: row0 + row_of(0 .. 15)
    int row0 = (tile * WR + wave / kColWaves) * 16, rows = 16, slot;
    __shared__ SlotRows walk;
    if (WR == 1 && a.items) {
        const int e = slot_rows(a, item, walk);
        if (e == -1) return;
        row0 = 0;
        rows = a.m;
        slot = lane < 16 && walk.rows[lane] >= 0 ? e : -1;
    } else {
        slot = row_slot(a, row0, 16, lane);
    }
    auto row_of = [&](int r) { return WR == 1 && a.items ? max(walk.rows[r], 0) : r; };
    // the member of this column chunk (a grid of members x the widest one's
    // chunks leaves workgroups that only end: m = 64, q k v: 7.4 -> 13 us)
    int j = 0;
#pragma unroll
    for (int i = 0; i < kMaxGemmMembers; ++i) j += chunk >= a.chunk_end[i];
    const AdapterMember& mb = a.member[j];
    const int n = mb.n, max_rank = mb.max_rank;
    const int c_begin = (chunk - mb.chunk0) * a.chunk_cols + wave % kColWaves * kTurn;
    const int c_end = min(n, (chunk - mb.chunk0 + 1) * a.chunk_cols);
    const uint32_t ldbase = (uint32_t)mb.ldbase * 2, ldy = (uint32_t)mb.ldy * 2;  // bytes
    const Rows<VEC> base(mb.base + (int64_t)row0 * mb.ldbase, (int64_t)(rows - 1) * ldbase + 2 * n);
    const Rows<VEC> y(mb.y + (int64_t)row0 * mb.ldy, (int64_t)(rows - 1) * ldy + 2 * n);
    const bool in_place = mb.base == mb.y;

    uint64_t left = __ballot(slot != -1);
    for (int order = 0; left; ++order) {
        const int lead = __builtin_ctzll(left);
        const int e = __builtin_amdgcn_readlane(slot, lead);
        const uint64_t mine = __ballot(slot == e);
        left &= ~mine;
        if (order % a.up_groups != group) continue;
        const int rank = e >= 0 ? min(mb.ranks[e], max_rank) : 0;
        if (rank <= 0 && in_place) continue;
        const float scale = e >= 0 ? mb.scales[e] : 0.f;
        uint4 t16[KS][kParts];
        const float back = row_parts<F16, KS, KS < 4 ? 4 / KS : 1>(a, mb, row0, rows, row_of(col), (mine >> col) & 1, rank, scale, q, t16);
        const auto up = buffer(mb.up + (e >= 0 ? (int64_t)e * n * max_rank : 0), (int64_t)n * max_rank * 2);
        for (int c0 = c_begin; c0 < c_end; c0 += kColWaves * kTurn) {
            // base and y: rows q, q + 4, ..., eight columns per lane; what is
            // not this turn's reads 0 and is not written
            const int cy = c0 + 8 * col;
            uint4 in[4];
            uint32_t at[4];  // row offsets are the caller's strides times this lane's rows
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool own = ((mine >> (4 * i + q)) & 1) && cy < n;
                at[i] = own ? (uint32_t)row_of(4 * i + q) : kOutside;
                in[i] = load8<VEC>(base, own ? at[i] * ldbase : kOutside, cy, n);
            }
            if (rank > 0) {
                constexpr int kTiles = kTurn / 16, kHalf = kTiles / 2;
                auto fetch = [&](int h, int s, uint4 (&b)[kHalf]) {
#pragma unroll
                    for (int u = 0; u < kHalf; ++u) {
                        const int c = c0 + 16 * (h * kHalf + u) + col, r = s * 32 + q * 8;
                        b[u] = load16(up, r < rank && c < n ? (uint32_t)(c * max_rank + r) * 2 : kOutside);
                    }
                };
                uint4 b[2][kHalf];
                fetch(0, 0, b[0]);
                floatx4_t acc[kHalf];
#pragma unroll
                for (int v = 0; v < 2 * KS; ++v) {  // half v / KS, rank step v % KS
                    const int s = v % KS;
                    if (v + 1 < 2 * KS) fetch((v + 1) / KS, (v + 1) % KS, b[(v + 1) & 1]);
                    __builtin_amdgcn_sched_barrier(0);  // the next loads go out before these are waited for
#pragma unroll
                    for (int u = 0; u < kHalf; ++u) {
                        if (s == 0) acc[u] = floatx4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int i = 0; i < kParts; ++i) acc[u] = mfma16<F16>(b[v & 1][u], t16[s][i], acc[u]);
                        if (s == KS - 1)
                            *(floatx4_t*)&product[wave][col][16 * (v / KS * kHalf + u) + 4 * q] = acc[u] * back;
                    }
                }
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    floatx4_t d0, d1;
                    eight_of(&product[wave][4 * i + q][8 * col], 8 * col, d0, d1);
                    in[i].x = add_pair<F16>(in[i].x, d0[0], d0[1]);
                    in[i].y = add_pair<F16>(in[i].y, d0[2], d0[3]);
                    in[i].z = add_pair<F16>(in[i].z, d1[0], d1[1]);
                    in[i].w = add_pair<F16>(in[i].w, d1[2], d1[3]);
                }
                __builtin_amdgcn_wave_barrier();
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) store8<VEC>(y, at[i] == kOutside ? kOutside : at[i] * ldy, cy, n, in[i]);
        }
    }
}

// ---------------------------------------------------------------------------
// y = base + s B t for prompts.  Workgroup: 64 rows, 16 per wave, x a column
// chunk, kTurn columns per turn.  The turn's B lies in LDS for all four waves
// (direct loads, the next turn's under way): what bounds the kernel above at many
// rows is what its waves read of B, each for its 16 rows (8192 columns, rank
// 128, 4096 rows: 0.31 GB beside the 0.13 of base and y, 88 us).  LDS image of
// 32 ranks of B: 16-byte chunk q of column c in slot 4 c + (q ^ (c / 2) mod 4), so that
// eight columns of a fragment read, what one pass takes, lie in distinct banks.
// ---------------------------------------------------------------------------
template <bool F16, int KS, int kTurn, bool VEC>
__global__ __launch_bounds__(kThreads) void adapter_up_tile_kernel(AdapterArgs a) {
    constexpr int kPitch = kTurn + 4, kTiles = kTurn / 16;
    constexpr int kRowsAt = 512 / kTurn, kPieces = 16 / kRowsAt;  // rows per access of base and y, accesses per turn
    constexpr int kDma = kTurn / 64;                              // 1 KB pieces of a slab per wave
    const int rr = (threadIdx.x & 63) / (kTurn / 8), rc = 8 * ((threadIdx.x & 63) % (kTurn / 8));  // row, column of an access
    constexpr int kSlab = kTurn * 64;  // bytes of 32 ranks of a turn's columns
    __shared__ int slots_lds[64];
    __shared__ __attribute__((aligned(16))) uint8_t stage[2 * KS * kSlab];
    __shared__ __attribute__((aligned(16))) float product[kWaves][16][kPitch];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, q = lane >> 4;
    const int chunk = blockIdx.x % a.chunks, tile0 = (int)(blockIdx.x / a.chunks) * 64;
    const int row0 = tile0 + 16 * wave;
    int j = 0;
#pragma unroll
    for (int i = 0; i < kMaxGemmMembers; ++i) j += chunk >= a.chunk_end[i];
    const AdapterMember& mb = a.member[j];
    const int n = mb.n, max_rank = mb.max_rank;
    const int c_begin = (chunk - mb.chunk0) * a.chunk_cols, c_end = min(n, c_begin + a.chunk_cols);
    const uint32_t ldbase = (uint32_t)mb.ldbase * 2, ldy = (uint32_t)mb.ldy * 2;  // bytes
    // (a wave past the last row reads none of its own)
    const int64_t first = min(row0, a.m - 1);
    const Rows<VEC> base(mb.base + first * mb.ldbase, 15 * (int64_t)ldbase + 2 * n);
    const Rows<VEC> y(mb.y + first * mb.ldy, 15 * (int64_t)ldy + 2 * n);
    const bool in_place = mb.base == mb.y;
    const int slot = tile_slots(a, tile0, 64, slots_lds);
    // this lane's part of a slab's 1 KB pieces (two per wave): column, chunk
    const int dc = lane >> 2, dq = (lane & 3) ^ (dc >> 1 & 3);
    uint64_t left = __ballot(slot != -1);
    while (left) {
        const int e = __builtin_amdgcn_readlane(slot, __builtin_ctzll(left));
        const uint64_t all = __ballot(slot == e);
        left &= ~all;
        if (e < 0 && in_place) continue;
        const uint32_t mine = (uint32_t)(all >> (16 * wave)) & 0xffffu;
        const int rank = e >= 0 ? min(mb.ranks[e], max_rank) : 0;
        const float scale = e >= 0 ? mb.scales[e] : 0.f;
        const __amdgpu_buffer_rsrc_t up = buffer(mb.up + (e >= 0 ? (int64_t)e * n * max_rank : 0), (int64_t)n * max_rank * 2);
        // B of the turn at c0 into stage half h, and the turn's base
        auto issue = [&](int c0, int h) {
            auto* to = (__attribute__((address_space(3))) uint8_t*)(void*)(stage + h * KS * kSlab + wave * kDma * 1024);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int p = 0; p < kDma; ++p) {
                    const int c = c0 + 16 * (kDma * wave + p) + dc, r = s * 32 + dq * 8;
                    const uint32_t off = r < rank && c < n ? (uint32_t)(c * max_rank + r) * 2 : kOutside;
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(up, (lds_void_t*)(to + s * kSlab + p * 1024), 16, off, 0, 0, 0);
                }
        };
        auto row_at = [&](int i, int c0, uint32_t ld) {  // row kRowsAt i + rr, eight columns per lane
            return (mine >> (kRowsAt * i + rr)) & 1 && c0 + rc < c_end ? (uint32_t)(kRowsAt * i + rr) * ld : kOutside;
        };
        uint4 next[kPieces];
        issue(c_begin, 0);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) next[i] = load8<VEC>(base, row_at(i, c_begin, ldbase), c_begin + rc, n);
        uint4 t16[KS][kParts];
        const float back = row_parts<F16, KS, 1>(a, mb, row0, 16, col, (mine >> col) & 1, rank, scale, q, t16);
        int h = 0;
        for (int c0 = c_begin; c0 < c_end; c0 += kTurn, h ^= 1) {
            // this wave's loads of the turn have landed (the last turn's
            // stores may be under way); after the barrier every wave's have, and
            // every wave is done with the other half
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(vmcnt_and_lds(kPieces));
            if (c0 == c_begin) __builtin_amdgcn_s_waitcnt(vmcnt_and_lds(0));
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            uint4 in[kPieces];
#pragma unroll
            for (int i = 0; i < kPieces; ++i) in[i] = next[i];
            if (c0 + kTurn < c_end) {
                issue(c0 + kTurn, h ^ 1);
                __builtin_amdgcn_sched_barrier(0);  // what is waited for with kPieces left goes out first
#pragma unroll
                for (int i = 0; i < kPieces; ++i) next[i] = load8<VEC>(base, row_at(i, c0 + kTurn, ldbase), c0 + kTurn + rc, n);
            }
            __builtin_amdgcn_sched_barrier(0);
            const uint8_t* from = stage + h * KS * kSlab + col * 64 + ((q ^ (col >> 1)) & 3) * 16;
#pragma unroll
            for (int u0 = 0; u0 < kTiles; u0 += 4) {
                // four column tiles side by side: one's products wait for each other
                // (4096 rows x 8192 columns, rank 128: one by one 61 us, so 56)
                floatx4_t acc[4];
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    uint4 b[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) b[u] = *(const uint4*)(from + s * kSlab + (u0 + u) * 1024);
#pragma unroll
                    for (int i = 0; i < kParts; ++i)
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            if (s == 0 && i == 0) acc[u] = floatx4_t{0.f, 0.f, 0.f, 0.f};
                            acc[u] = mfma16<F16>(b[u], t16[s][i], acc[u]);
                        }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) *(floatx4_t*)&product[wave][col][16 * (u0 + u) + 4 * q] = acc[u] * back;
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                floatx4_t d0, d1;
                eight_of(&product[wave][kRowsAt * i + rr][rc], rc, d0, d1);
                if (rank > 0) {
                    in[i].x = add_pair<F16>(in[i].x, d0[0], d0[1]);
                    in[i].y = add_pair<F16>(in[i].y, d0[2], d0[3]);
                    in[i].z = add_pair<F16>(in[i].z, d1[0], d1[1]);
                    in[i].w = add_pair<F16>(in[i].w, d1[2], d1[3]);
                }
                store8<VEC>(y, row_at(i, c0, ldy), c0 + rc, n, in[i]);
            }
            __builtin_amdgcn_wave_barrier();
        }
        // the next adapter's first loads go into a half that may still be read
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Few rows, ranks of at most 16: both products in one launch.  Workgroup: one adapter's rows of a
// 16-row tile x a column chunk; its sixteen waves make t, a quarter of a K
// partition each, in LDS, then 64 columns of y per turn, whose B and base
// (TURNS turns of them) are on the way since A is.  Every column chunk reads A
// again.  What bounds it is the chain of dependent loads (slot, A and rank) and
// what one CU takes in (30 - 60 GB/s); two launches have that chain twice: q k v
// of 64 rows, each its own adapter, rank 16: 15.9 us in two, 12.5 in one.  B's
// rows are permuted so that a lane ends with eight consecutive columns of one
// row: of two 16-row tiles, row 4 p + s of tile u stands for column 8 p + 4 u + s.
// ---------------------------------------------------------------------------
template <bool F16, int TURNS, bool VEC>
__global__ __launch_bounds__(kAdapterRowWaves * 64) void adapter_row_kernel(AdapterArgs a) {
    constexpr int kW = kAdapterRowWaves, kTurn = kAdapterRowTurn;
    __shared__ int slots_lds[64];
    __shared__ floatx4_t quarters[kW][64];
    const AdapterMember& mb = a.member[blockIdx.z];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, q = lane >> 4;
    const int n = mb.n, max_rank = mb.max_rank;
    const int row0 = (int)(blockIdx.x / a.down_groups) * 16;
    const int c_begin = blockIdx.y * a.chunk_cols + wave * kTurn, c_end = min(n, (int)(blockIdx.y + 1) * a.chunk_cols);
    if ((int)blockIdx.y * a.chunk_cols >= n) return;
    const int slot = tile_slots(a, row0, 16, slots_lds);
    // this workgroup's adapter: number blockIdx.x % groups of the tile's
    uint64_t left = __ballot(slot != -1), mine = 0;
    int lead = 0, e = 0;
    for (int order = (int)(blockIdx.x % a.down_groups); order >= 0; --order) {
        if (!left) return;
        lead = __builtin_ctzll(left);
        e = __builtin_amdgcn_readlane(slot, lead);
        mine = __ballot(slot == e);
        left &= ~mine;
    }
    const bool in_place = mb.base == mb.y;
    if (e < 0 && in_place) return;
    const int rank = e >= 0 ? min(mb.ranks[e], max_rank) : 0;
    const float scale = e >= 0 ? mb.scales[e] : 0.f;
    const int es = max(e, 0), parts = 4 * a.split;
    const uint32_t ldbase = (uint32_t)mb.ldbase * 2, ldy = (uint32_t)mb.ldy * 2;  // bytes
    const Rows<VEC> base(mb.base + (int64_t)row0 * mb.ldbase, 15 * (int64_t)ldbase + 2 * n);
    const Rows<VEC> y(mb.y + (int64_t)row0 * mb.ldy, 15 * (int64_t)ldy + 2 * n);
    const auto up = buffer(mb.up + (int64_t)es * n * max_rank, (int64_t)n * max_rank * 2);
    const bool own = (mine >> col) & 1;
    uint4 b[TURNS][kTurn / 16], in[TURNS][kTurn / 32];
    auto fetch = [&](int c0) {
#pragma unroll
        for (int v = 0; v < TURNS; ++v)
#pragma unroll
            for (int g = 0; g < kTurn / 32; ++g) {
                const int first = c0 + v * kW * kTurn + 32 * g;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int c = first + 8 * (col >> 2) + 4 * u + (col & 3);
                    b[v][2 * g + u] = load16(up, q * 8 < rank && c < c_end ? (uint32_t)(c * max_rank + q * 8) * 2 : kOutside);
                }
                const int cy = first + 8 * q;
                in[v][g] = load8<VEC>(base, own && cy < c_end ? col * ldbase : kOutside, cy, n);
            }
    };
    {
        const int rows = min(16, a.m - row0);
        const auto x = buffer(a.x + (int64_t)row0 * a.ldx, ((int64_t)(rows - 1) * a.ldx + a.k) * 2);
        const auto d = buffer(mb.down + (int64_t)es * max_rank * a.k, e >= 0 ? (int64_t)max_rank * a.k * 2 : 0);
        const uint32_t xoff[1] = {(uint32_t)(own ? col : lead) * (uint32_t)(a.ldx * 2)};
        // (not waiting for the rank: what lies past it split_row leaves out)
        const uint32_t doff[1] = {col < max_rank ? (uint32_t)col * (uint32_t)(a.k * 2) : kOutside};
        floatx4_t acc[1][1];
        if (wave < parts) {
            quarter_product<F16, 1, 1>(x, xoff, d, doff, wave * kQuarter + q * 8, a.k, acc, [&] { fetch(c_begin); });
            quarters[wave][lane] = acc[0][0];
        } else {
            fetch(c_begin);
        }
    }
    __syncthreads();
    // t of row col, ranks 8 q .. 8 q + 7 (q < 2): lane 16 (rank / 4) + col holds
    // four ranks; quarters and partitions in order
    uint4 t16[1][kParts];
    floatx4_t t8[1][2];
    t8[0][0] = t8[0][1] = floatx4_t{0.f, 0.f, 0.f, 0.f};
    if (q < 2)
        for (int j = 0; j < parts; j += 4)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int at = 16 * (2 * q + c) + col;
                t8[0][c] += (quarters[j][at] + quarters[j + 1][at]) + (quarters[j + 2][at] + quarters[j + 3][at]);
            }
    const float back = split_row<F16, 1>(t8, rank, scale, q, t16);
    if (rank <= 0 && in_place) return;
    for (int c0 = c_begin; c0 < c_end; c0 += TURNS * kW * kTurn) {
        if (c0 != c_begin) fetch(c0);
#pragma unroll
        for (int v = 0; v < TURNS; ++v)
#pragma unroll
            for (int g = 0; g < kTurn / 32; ++g) {
                if (rank > 0) {
                    floatx4_t acc[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        acc[u] = floatx4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int i = 0; i < kParts; ++i) acc[u] = mfma16<F16>(b[v][2 * g + u], t16[0][i], acc[u]);
                        acc[u] *= back;
                    }
                    in[v][g].x = add_pair<F16>(in[v][g].x, acc[0][0], acc[0][1]);
                    in[v][g].y = add_pair<F16>(in[v][g].y, acc[0][2], acc[0][3]);
                    in[v][g].z = add_pair<F16>(in[v][g].z, acc[1][0], acc[1][1]);
                    in[v][g].w = add_pair<F16>(in[v][g].w, acc[1][2], acc[1][3]);
                }
                const int cy = c0 + v * kW * kTurn + 32 * g + 8 * q;
                store8<VEC>(y, own && cy < c_end ? col * ldy : kOutside, cy, n, in[v][g]);
            }
    }
}

template <bool F16, int MT, int RT>
void start_down(const AdapterArgs& a, hipStream_t s) {
    const dim3 grid((a.items ? a.items : (a.m + 16 * MT - 1) / (16 * MT) * a.down_groups) * a.split,
                    (a.rank_tiles + RT - 1) / RT, a.members);
    adapter_down_kernel<F16, MT, RT><<<grid, kThreads, 0, s>>>(a);
}

template <bool F16, int MT>
void start_down_tiles(const AdapterArgs& a, hipStream_t s) {
    if (a.rank_tiles == 1) start_down<F16, MT, 1>(a, s);
    else if (a.rank_tiles == 2) start_down<F16, MT, 2>(a, s);
    else start_down<F16, MT, 4>(a, s);
}

template <bool F16, int KS, int WR>
void start_up(const AdapterArgs& a, hipStream_t s) {
    const dim3 grid((a.items ? a.items : (a.m + 16 * WR - 1) / (16 * WR) * a.up_groups) * a.chunks);
    if (a.vectors) adapter_up_kernel<F16, KS, WR, true><<<grid, kThreads, 0, s>>>(a);
    else adapter_up_kernel<F16, KS, WR, false><<<grid, kThreads, 0, s>>>(a);
}

template <bool F16, int KS>
void start_up_rows(const AdapterArgs& a, hipStream_t s) {
    if constexpr (KS <= 4)
        if (a.up_tile) {
            constexpr int kTurn = KS == 4 ? 64 : kAdapterUpTurn;
            const int grid = (a.m + 63) / 64 * a.chunks;
            if (a.vectors) adapter_up_tile_kernel<F16, KS, kTurn, true><<<grid, kThreads, 0, s>>>(a);
            else adapter_up_tile_kernel<F16, KS, kTurn, false><<<grid, kThreads, 0, s>>>(a);
            return;
        }
    if (a.up_rows == 1) start_up<F16, KS, 1>(a, s);
    else start_up<F16, KS, 4>(a, s);
}

template <bool F16, int TURNS, bool VEC>
void start_row(const AdapterArgs& a, hipStream_t s) {
    const dim3 grid((a.m + 15) / 16 * a.down_groups, a.chunks, a.members);
    adapter_row_kernel<F16, TURNS, VEC><<<grid, kAdapterRowWaves * 64, 0, s>>>(a);
}

template <bool F16>
hipError_t start(const AdapterArgs& a, hipStream_t s) {
    if (a.fused) {
        if (!a.vectors) start_row<F16, 1, false>(a, s);
        else if (a.chunk_cols <= kAdapterRowWaves * kAdapterRowTurn) start_row<F16, 1, true>(a, s);
        else start_row<F16, 2, true>(a, s);
        return hipGetLastError();
    }
    if (a.down_rows == 4) {
        const dim3 grid((a.m + 63) / 64 * a.split, (a.rank_tiles + kDownTileRanks - 1) / kDownTileRanks, a.members);
        adapter_down_tile_kernel<F16><<<grid, kThreads, 0, s>>>(a);
    } else if (a.down_rows == 1) start_down_tiles<F16, 1>(a, s);
    else start_down_tiles<F16, 2>(a, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    AdapterArgs u = a;
    if (a.join) {
        adapter_join_kernel<<<(unsigned)(((int64_t)a.m * a.width / 4 + kThreads - 1) / kThreads), kThreads, 0, s>>>(a);
        u.split = 1;
    }
    const int steps = (a.rank_tiles + 1) / 2;
    if (steps == 1) start_up_rows<F16, 1>(u, s);
    else if (steps == 2) start_up_rows<F16, 2>(u, s);
    else if (steps <= 4) start_up_rows<F16, 4>(u, s);
    else start_up_rows<F16, 8>(u, s);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_adapters(const AdapterArgs& a, hipStream_t s) {
    return a.f16 ? start<true>(a, s) : start<false>(a, s);
}

}  // namespace cubic
