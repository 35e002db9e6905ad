// Block-scaled 8-bit products for gfx950:
//
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} xq[m, k] wq[n, k]
//
// over e4m3 values and blocks of 128 columns.  Each block's product starts from zero
// and is added to the 32-bit accumulator under its scale.
//
// Outputs in 16 bits: one v_mfma_f32_16x16x128_f8f6f4 (unscaled form: the plain products
// of its 8-bit operands, at twice the rate of the K = 32 ones) is one block of a 16 x 16
// tile.  The instruction adds eight neighbouring products at 14 bits below the largest's
// exponent, and those sums in 32 bits.  That is the one rounding below 32 bits here,
// taken for its rate: of N(0, 1) operands it leaves y 1.5e-5 off (root mean
// square), a hundredth of bf16's rounding and a fourteenth of fp16's; at most 7 * 2^-13 of an
// eight's largest |x| times its largest |w|.
// Outputs in 32 bits (FULL): the K = 32 instructions of 8-bit operands cut in the same way (2^16 + 2^e
// keeps 2^e to e = 3 in both, to e = -7 with 16-bit operands), so the values go to
// fp16, which holds all of e4m3, and four v_mfma_f32_16x16x32_f16 make a block: sums in 32 bits.
//
// Weights are its first operand: a lane then holds four columns n of one row m, the
// scale is one number per lane, and outputs leave four columns at a time.
//
// Any order of k inside a block serves as long as both operands have it.  Here
// lane l of an operand has row l % 16 and the 16 bytes at 16 (l / 16) of each half
// block: loads of 64 contiguous bytes per row of x.  Weights are laid out once as
// [128 rows][block][tile of 16 rows][half][lane][16 bytes]: 2 KB per tile and block, 16 KB
// in one piece for all columns that share a scale.
#include <type_traits>

#include "cubic_capi_internal.h"
#include "cubic_device.h"

namespace cubic {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
constexpr int kBlockBytes = 2048;              // one tile and block
constexpr int kGroupBytes = 8 * kBlockBytes;   // 128 rows of one block
constexpr uint32_t kPastEnd = 0x80000000u;     // a buffer offset past every extent
constexpr int kStreamWaves = 8;

__device__ __forceinline__ v8i join(u32x4_dev_t a, u32x4_dev_t b) {
    return v8i{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

// 32 values of a row in fp16, as four operands of 8.
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
struct Halves {
    v8h c[4];
};
__device__ __forceinline__ Halves to_halves(v8i v) {
    Halves h;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const v2h p = e & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[2 * c + e / 2], 1.0f, true)
                                : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[2 * c + e / 2], 1.0f, false);
            h.c[c][2 * e] = p[0];
            h.c[c][2 * e + 1] = p[1];
        }
    return h;
}

// 16 x 16 products over one block from zero: rows of w by rows of x.
__device__ __forceinline__ v4f block_product(const Halves& w, const Halves& x) {
    v4f p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 4; ++c) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.c[c], x.c[c], p, 0, 0, 0);
    return p;
}
__device__ __forceinline__ v4f block_product(v8i w, v8i x) {
    const v4f zero = {0.f, 0.f, 0.f, 0.f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, zero, 0, 0, 0, 0, 0, 0);
}

// 32 values of a row as block_product takes them.
template <bool FULL>
__device__ __forceinline__ auto operand(v8i v) {
    if constexpr (FULL) return to_halves(v);
    else return v;
}

// Four outputs in 16 bits.
__device__ __forceinline__ v2u pack4(const BlockGemmArgs& a, v4f v) {
    if (a.out == 1)
        return v2u{float_to_f16_bits(v[0]) | float_to_f16_bits(v[1]) << 16, float_to_f16_bits(v[2]) | float_to_f16_bits(v[3]) << 16};
    return v2u{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}

// Four columns of one row of y (global memory takes 8 or 16 bytes at any element's address).
// LINES: past the caches where rows of y are whole lines, which a wave then writes whole: 64 rows
// of 151936 x 4096 in 124 and 117 us, 2048 x 24576 x 4096 185 and 179; rows that share lines
// (333 of 1521 x 2064) lose by it, 9.1 and 9.5.
template <bool FULL, bool LINES = false>
__device__ __forceinline__ void store4(const BlockGemmArgs& a, const BlockMember& w, int64_t m, int n, v4f v) {
    if (n >= w.n) return;
    if constexpr (FULL) {
        float* y = static_cast<float*>(w.y) + m * w.ldy + n;
        if (LINES && w.lines) {
            __builtin_nontemporal_store(v, reinterpret_cast<v4f*>(y));
        } else if (n + 4 <= w.n) {
            __builtin_memcpy(y, &v, sizeof v);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < w.n) y[i] = v[i];
        }
    } else {
        const v2u u = pack4(a, v);
        uint16_t* y = static_cast<uint16_t*>(w.y) + m * w.ldy + n;
        if (n + 4 <= w.n) {
            __builtin_memcpy(y, &u, sizeof u);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < w.n) y[i] = (uint16_t)(u[i >> 1] >> (16 * (i & 1)));
        }
    }
}

// Eight columns in 16 bits, past the caches as above.
__device__ __forceinline__ void store8(const BlockGemmArgs& a, const BlockMember& w, int64_t m, int n, v4f lo, v4f hi) {
    if (n + 8 > w.n) {
        store4<false>(a, w, m, n, lo);
        store4<false>(a, w, m, n + 4, hi);
        return;
    }
    const v2u l = pack4(a, lo), h = pack4(a, hi);
    const u32x4_dev_t u = {l[0], l[1], h[0], h[1]};
    uint16_t* y = static_cast<uint16_t*>(w.y) + m * w.ldy + n;
    if (w.lines) __builtin_nontemporal_store(u, reinterpret_cast<u32x4_dev_t*>(y));
    else __builtin_memcpy(y, &u, sizeof u);
}

// The member and its first tile of a column group.
__device__ __forceinline__ int find_member(const BlockGemmArgs& a, int group) {
    int j = 0;
    for (int i = 0; i + 1 < a.members; ++i) j += group >= a.group_end[i];
    return j;
}

// ---------------------------------------------------------------------------
// Up to 8 rows: the weight stream bounds it.  A workgroup has NT tiles of columns; its
// waves take the blocks of K in turn, each block's weights and activations straight
// into registers, DEPTH blocks ahead, no barrier until the waves' sums are added
// through LDS, in the order of the waves.  1 row, 20000 x 16384: 61 us, 5.4 TB/s.
// ---------------------------------------------------------------------------
template <int NT, int DEPTH, bool FULL>
__global__ __launch_bounds__(kStreamWaves * 64) void block_stream_kernel(BlockGemmArgs a) {
    __shared__ v4f sums[kStreamWaves][NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int quarter = lane >> 4, row = lane & 15;
    const int j = find_member(a, blockIdx.x);
    const BlockMember& w = a.member[j];
    const int tile0 = (blockIdx.x - (j ? a.group_end[j - 1] : 0)) * NT;

    // buffers of x and of the workgroup's 128 rows of w: what lies past them reads as zero
    const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(a.x), 0, (int)((a.m - 1) * a.ldx) + a.k, 0x00020000);
    const uint32_t x_at = (uint32_t)(row * a.ldx) + 16u * quarter;
    const float* sx = a.x_scales + (int64_t)min(row, a.m - 1) * a.scale_row;
    const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(w.codes + (int64_t)(tile0 >> 3) * a.blocks * kGroupBytes), 0, a.blocks * kGroupBytes, 0x00020000);
    const uint32_t w_at = (tile0 & 7) * kBlockBytes + lane * 16;
    const float* sw = w.scales + (int64_t)(tile0 >> 3) * a.blocks;

    struct Stage {
        u32x4_dev_t w[NT][2], x[2];
        float sx, sw;
    };
    Stage st[DEPTH];
    auto load = [&](Stage& s, int b) {
        const bool some = b < a.blocks;
        const uint32_t from = some ? (uint32_t)b * kGroupBytes : kPastEnd;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                s.w[t][h] = __builtin_amdgcn_raw_buffer_load_b128(wr, from + w_at + t * kBlockBytes + h * 1024, 0, 2);  // nt
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = b * kScaleBlock + h * 64;
            s.x[h] = __builtin_amdgcn_raw_buffer_load_b128(
                xr, some && row < a.m && k + 16 * quarter < a.k ? x_at + (uint32_t)k : kPastEnd, 0, 0);
        }
        const int at = min(b, a.blocks - 1);
        s.sx = sx[(int64_t)at * a.scale_group];
        s.sw = sw[at];
    };
    v4f acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};

#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(st[d], wave + d * kStreamWaves);
    for (int b = wave; b < a.blocks; b += DEPTH * kStreamWaves) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (b + d * kStreamWaves < a.blocks) {
                Stage& s = st[d];
                const float scale = s.sx * s.sw;
                const auto xv = operand<FULL>(join(s.x[0], s.x[1]));
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const v4f p = block_product(operand<FULL>(join(s.w[t][0], s.w[t][1])), xv);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(scale, p[e], acc[t][e]);
                }
                load(s, b + (d + DEPTH) * kStreamWaves);
            }
        }
    }

#pragma unroll
    for (int t = 0; t < NT; ++t) sums[wave][t][lane] = acc[t];
    __syncthreads();
    if (wave < NT && tile0 + wave < w.tiles && row < a.m) {
        v4f v = sums[0][wave][lane];
        for (int o = 1; o < kStreamWaves; ++o) v += sums[o][wave][lane];
        store4<FULL>(a, w, row, (tile0 + wave) * 16 + quarter * 4, v);
    }
}

// ---------------------------------------------------------------------------
// Many rows: the matrix cores bound it.  A workgroup has a tile of 16 NTW WN columns
// by 16 MTW WM rows, WN x WM waves of 16 NTW x 16 MTW.  Both operands of a
// block, and its row scales, go straight to LDS (buffer and global loads to LDS)
// while the block before is multiplied (PAST: weights past the caches).
//
// LDS order: weights as they were laid out, 16 bytes per lane in lane order.  x: of
// a tile of 16 rows 128 slots of 16 bytes, row r's chunk c at slot 8 r + (c ^ turn(r)):
// eight neighbouring lanes of a load take one line of a row, and eight rows (in 128
// bytes of banks) or sixteen (in 256) that read a chunk together lie on different banks.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int turn(int r) { return (r >> 1 & 3) | ((r ^ r >> 3) & 1) << 2; }

typedef __attribute__((address_space(3))) void lds_void_t;
typedef const __attribute__((address_space(1))) void global_void_t;

// s_waitcnt vmcnt(n) lgkmcnt(0), and vmcnt(n) alone
constexpr int step_waits(int n) { return (n & 0xF) | (0x7 << 4) | ((n >> 4) << 14); }
constexpr int vm_waits(int n) { return (n & 0xF) | (0x7 << 4) | (0xF << 8) | ((n >> 4) << 14); }

constexpr int leave_pitch(int ntw) { return 16 * ntw + 4; }  // of 32-bit sums

// Workgroups go round robin over the eight XCDs; an XCD takes consecutive items of an
// order that goes through 8 column groups for a row group, then the next rows, so that
// those it has at one time share operands in its L2.
__device__ __forceinline__ int xcd_item(int id, int total) {
    const int per = total >> 3, rest = total & 7, xcd = id & 7;
    return xcd * per + min(xcd, rest) + (id >> 3);
}

struct TileAt {
    int m0, tile0, member;  // first row, first tile of 16 columns of that member
};

__device__ __forceinline__ TileAt tile_at(const BlockGemmArgs& a, int id, int row_groups, int M, int N) {
    const int cols = a.group_end[a.members - 1], band = id / (8 * row_groups), wide = min(8, cols - 8 * band);
    id -= band * 8 * row_groups;
    const int group = 8 * band + id % wide, j = find_member(a, group);
    return {id / wide * (16 * M), (group - (j ? a.group_end[j - 1] : 0)) * N, j};
}

// A wave's sums, 16 rows at a time through a run of LDS of its own (`out`), to leave in whole lines.
template <bool FULL, int NTW, int MTW>
__device__ __forceinline__ void leave(const BlockGemmArgs& a, const BlockMember& w, int m_first, int n0, const v4f (&acc)[NTW][MTW], float* out) {
    constexpr int kPitch = leave_pitch(NTW);
    const int lane = threadIdx.x & 63, quarter = lane >> 4, row = lane & 15;
#pragma unroll
    for (int i = 0; i < MTW; ++i) {
#pragma unroll
        for (int t = 0; t < NTW; ++t) *reinterpret_cast<v4f*>(out + row * kPitch + t * 16 + quarter * 4) = acc[t][i];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if constexpr (!FULL) {  // (eight columns a lane: 2048 x 24576 x 4096 in 174 us by four, and 166)
#pragma unroll
            for (int at = lane; at < 32 * NTW; at += 64) {
                const int r = at / (2 * NTW), c = at % (2 * NTW) * 8, m = m_first + i * 16 + r;
                const v4f lo = *reinterpret_cast<const v4f*>(out + r * kPitch + c), hi = *reinterpret_cast<const v4f*>(out + r * kPitch + c + 4);
                if (m < a.m) store8(a, w, m, n0 + c, lo, hi);
            }
        } else {
#pragma unroll 1
            for (int at = lane; at < 64 * NTW; at += 64) {
                const int r = at / (4 * NTW), c = at % (4 * NTW) * 4, m = m_first + i * 16 + r;
                if (m < a.m) store4<true, true>(a, w, m, n0 + c, *reinterpret_cast<const v4f*>(out + r * kPitch + c));
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

template <int NTW, int MTW, int WN, int WM, int S, int G, int EU, bool SPLIT, bool PAST, bool FULL>
__global__ __launch_bounds__(G * WN * WM * 64) __attribute__((amdgpu_waves_per_eu(EU, EU)))
void block_tile_kernel(BlockGemmArgs a) {
    constexpr int W = WN * WM, N = NTW * WN, M = MTW * WM;  // waves of a group; tiles of 16
    static_assert(8 % NTW == 0, "a wave's columns share a scale");
    static_assert(M == W && N % W == 0 && (S == 3 || S == 4), "a wave loads a tile of x, the scales of its rows, whole tiles of w");
    // A stage is x and w of G blocks, one per group; the rows' scales are for S blocks of a
    // group, four places a row.  Each is an object of its own: a load into one then does not wait
    // for reads of another.
    constexpr int kW = M * kBlockBytes, kStage = kW + N * kBlockBytes;
    __shared__ __attribute__((aligned(1024))) uint8_t stage0[G * kStage], stage1[G * kStage], stage2[G * kStage], stage3[G * kStage];
    __shared__ __attribute__((aligned(1024))) uint8_t row_scales[G * W * 256];
    auto stage_of = [&](auto stage) -> uint8_t* {
        constexpr int P = decltype(stage)::value;
        if constexpr (P == 0) return stage0; else if constexpr (P == 1) return stage1; else if constexpr (P == 2) return stage2; else return stage3;
    };
    constexpr int kWt = N / W, kLoads = 2 + 2 * kWt;  // tiles of w, and loads to LDS, per wave and block
    const int lane = threadIdx.x & 63, wave_of_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = wave_of_all % W, k_group = wave_of_all / W;
    const int quarter = lane >> 4, row = lane & 15;
    const int wn = wave % WN, wm = wave / WN;

    const int row_groups = (a.m + 16 * M - 1) / (16 * M), tiles = a.group_end[a.members - 1] * row_groups;
    int id = xcd_item(blockIdx.x, SPLIT ? tiles * a.split : tiles);
    const int part = SPLIT ? id / tiles : 0;  // of K
    if constexpr (SPLIT) id -= part * tiles;
    const int tile_id = id;
    const TileAt at_tile = tile_at(a, id, row_groups, M, N);
    const int m0 = at_tile.m0, tile0 = at_tile.tile0;
    const BlockMember& w = a.member[at_tile.member];

    // --- loads to LDS -------------------------------------------------------------------
    // Every tile of rows has a buffer of its own, moved on by the block: what a lane
    // adds to it is one number.  Rows past the last, columns past K and blocks past
    // the last read as zero.
    const int load_row = lane >> 3;  // of a tile's first half, or second
    const int load_chunk[2] = {(lane & 7) ^ turn(load_row), (lane & 7) ^ turn(load_row + 8)};
    const uint32_t w_at = lane * 16;
    const uint32_t x_at[2] = {(uint32_t)(load_row * a.ldx) + 16u * load_chunk[0], (uint32_t)((load_row + 8) * a.ldx) + 16u * load_chunk[1]};
    const int x_columns[2] = {a.k - 16 * load_chunk[0], a.k - 16 * load_chunk[1]};
    const float* sx = a.x_scales + (int64_t)min(m0 + wave * 16 + (lane >> 2), a.m - 1) * a.scale_row;
    // a wave's tiles' starts and extents
    const int x_first = m0 + 16 * wave, x_left = min(a.m - x_first, 16);
    const uint8_t *const x_from = a.x + (int64_t)x_first * a.ldx, *w_from[kWt];
    const int x_bytes = x_left <= 0 ? 0 : (int)((x_left - 1) * a.ldx) + a.k;
    int w_bytes[kWt];
#pragma unroll
    for (int p = 0; p < kWt; ++p) {
        const int tile = tile0 + wave * kWt + p;
        w_from[p] = w.codes + (int64_t)(tile >> 3) * a.blocks * kGroupBytes + (tile & 7) * kBlockBytes;
        w_bytes[p] = tile < w.tiles ? kBlockBytes : 0;
    }
    const int b_first = SPLIT ? part * a.part_blocks : 0;
    const int blocks = SPLIT ? min(a.blocks, b_first + a.part_blocks) : a.blocks;  // up to there
    const int64_t scale_group = a.scale_group;
    auto dma = [&](int b, auto stage) {
        uint8_t* to = stage_of(stage) + k_group * kStage;
        __attribute__((address_space(3))) uint8_t* xl = (__attribute__((address_space(3))) uint8_t*)(void*)to;
        __attribute__((address_space(3))) uint8_t* wl = xl + kW;
        const int k = b * kScaleBlock;
        const bool some = !SPLIT || b < blocks;
        const uint32_t off[2] = {some && k < x_columns[0] ? x_at[0] : kPastEnd, some && k < x_columns[1] ? x_at[1] : kPastEnd};
        const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(x_from + k), 0, max(x_bytes - k, 0), 0x00020000);
#pragma unroll
        for (int h = 0; h < 2; ++h)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_void_t*)(xl + wave * kBlockBytes + h * 1024), 16, off[h], 0, 0, 0);
#pragma unroll
        for (int p = 0; p < kWt; ++p) {
            const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<uint8_t*>(w_from[p] + (int64_t)b * kGroupBytes), 0, b < blocks ? w_bytes[p] : 0, 0x00020000);
#pragma unroll
            for (int h = 0; h < 2; ++h)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (lds_void_t*)(wl + (wave * kWt + p) * kBlockBytes + h * 1024), 16, w_at + h * 1024, 0, 0, PAST ? 2 : 0);
        }
    };
    // Those of a group's next S blocks at a time: where a row's lie together, four lanes
    // are one access (a block at a time, 64 x 151936 x 4096 takes 134 us and not 129; PAST 125)
    auto load_scales = [&](int b) {
        __builtin_amdgcn_global_load_lds((global_void_t*)(sx + (int64_t)min(b + (lane & 3) * G, blocks - 1) * scale_group),
                                         (lds_void_t*)((__attribute__((address_space(3))) uint8_t*)(void*)row_scales + (k_group * W + wave) * 256), 4, 0, 0);
    };

    v4f acc[NTW][MTW];
#pragma unroll
    for (int t = 0; t < NTW; ++t)
#pragma unroll
        for (int i = 0; i < MTW; ++i) acc[t][i] = v4f{0.f, 0.f, 0.f, 0.f};
    // (the constant address space: one scalar load per wave)
    const __attribute__((address_space(4))) float* sw = (const __attribute__((address_space(4))) float*)(
        w.scales + (int64_t)(min(tile0 + wn * NTW, w.tiles - 1) >> 3) * a.blocks);
    const uint32_t x_slot = (uint32_t)(wm * MTW * kBlockBytes) + (uint32_t)(8 * row + (quarter ^ turn(row))) * 16;
    const uint32_t x_half = x_slot ^ 64;  // of its second half block
    const uint32_t w_slot = (uint32_t)(wn * NTW * kBlockBytes) + lane * 16;
    const float* const row_scale = reinterpret_cast<const float*>(row_scales + k_group * W * 256) + (wm * MTW * 16 + row) * 4;
    auto fragment = [](const uint8_t* at) {
        return join(*reinterpret_cast<const u32x4_dev_t*>(at), *reinterpret_cast<const u32x4_dev_t*>(at + 1024));
    };

    // A product is added to its sum kLag products later, in the shadow of theirs (1024 x 8192 x 4096:
    // 43.6 us for 2, 41.8 for 3).
    constexpr int kLag = 3;
    // S - 1 steps' blocks are on their way.  A step begins where its blocks have landed and
    // every wave is done with the step before, into whose place the next load goes.
    v4f scales[MTW];  // of a row's next S blocks
    auto step = [&](int at, auto stage) {
        constexpr int P = decltype(stage)::value;
        const int b = b_first + at * G + k_group;
        const uint8_t *xs = stage_of(stage) + k_group * kStage, *ws = xs + kW;
        float scale[MTW];
        v8i wv[2];
        decltype(operand<FULL>(wv[0])) xv[MTW], of_w;
        v4f p[kLag + 1];
        // (S - 2 steps' loads may be on their way, and the scales' that step 1 of S sends)
        __builtin_amdgcn_s_waitcnt(vm_waits((S - 2) * kLoads + (P >= 2 ? 1 : 0)));
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        const float block_scale = sw[G == 1 ? b : min(b, blocks - 1)];
#pragma unroll
        for (int i = 0; i < MTW; ++i)
            xv[i] = operand<FULL>(join(*reinterpret_cast<const u32x4_dev_t*>(xs + x_slot + i * kBlockBytes),
                                       *reinterpret_cast<const u32x4_dev_t*>(xs + x_half + i * kBlockBytes)));
        wv[0] = fragment(ws + w_slot);
#pragma unroll
        for (int i = 0; i < MTW; ++i) {
            if constexpr (P == 0) scales[i] = *reinterpret_cast<const v4f*>(row_scale + i * 64);
            scale[i] = scales[i][P] * block_scale;
            if constexpr (G > 1) {  // groups past the last block add products of zeros under scale 0
                asm("" : "+v"(scale[i]));
                scale[i] = b < blocks ? scale[i] : 0.0f;
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        dma(b + (S - 1) * G, std::integral_constant<int, (P + S - 1) % S>{});
        if constexpr (P == 1) load_scales(b + (S - 1) * G);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < NTW * MTW + kLag; ++q) {
            const int t = q / MTW, i = q % MTW;
            if (i == 0 && t + 1 < NTW) wv[(t + 1) & 1] = fragment(ws + w_slot + (t + 1) * kBlockBytes);
            if (i == 0 && t < NTW) of_w = operand<FULL>(wv[t & 1]);
            if (t < NTW) p[q % (kLag + 1)] = block_product(of_w, xv[i]);
            if (q >= kLag) {
                const int of = q - kLag;
                v4f& sum = acc[of / MTW][of % MTW];
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] = fmaf(scale[of % MTW], p[of % (kLag + 1)][e], sum[e]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        // the sums stay in this step (the compiler would move additions to the next one)
#pragma unroll
        for (int t = 0; t < NTW; ++t)
#pragma unroll
            for (int i = 0; i < MTW; ++i) asm volatile("" : "+v"(acc[t][i]));
    };
    load_scales(b_first + k_group);
    auto first = [&](auto... stages) { (dma(b_first + decltype(stages)::value * G + k_group, stages), ...); };
    typedef std::integral_constant<int, 0> I0;
    typedef std::integral_constant<int, 1> I1;
    typedef std::integral_constant<int, 2> I2;
    typedef std::integral_constant<int, 3> I3;
    if constexpr (S == 3) first(I0{}, I1{});
    else first(I0{}, I1{}, I2{});
    // Whole rounds of the stages, then the rest: a loop of one exit, through which the
    // compiler follows which loads are on their way (with more it waits for all).
    const int steps = (blocks - b_first + G - 1) / G;
    int at = 0;
    for (; at + S <= steps; at += S) {
        step(at, I0{});
        step(at + 1, I1{});
        step(at + 2, I2{});
        if constexpr (S > 3) step(at + 3, I3{});
    }
    if (at < steps) step(at, I0{});
    if (at + 1 < steps) step(at + 1, I1{});
    if constexpr (S > 3) {
        if (at + 2 < steps) step(at + 2, I2{});
    }
    __syncthreads();  // the last loads (of nothing) have landed, all is read
    if constexpr (G > 1) {  // the groups' sums, in order
        static_assert((G - 1) * W * NTW * MTW * 1024 <= G * kStage, "the other groups' sums fit a stage");
        v4f* sums = reinterpret_cast<v4f*>(stage0) + wave * NTW * MTW * 64 + lane;
        constexpr int kGroup = W * NTW * MTW * 64;
        if (k_group) {
#pragma unroll
            for (int t = 0; t < NTW; ++t)
#pragma unroll
                for (int i = 0; i < MTW; ++i) sums[(k_group - 1) * kGroup + (t * MTW + i) * 64] = acc[t][i];
        }
        __syncthreads();
        if (!SPLIT && k_group) return;
        if (k_group == 0) {
#pragma unroll
            for (int t = 0; t < NTW; ++t)
#pragma unroll
                for (int i = 0; i < MTW; ++i)
#pragma unroll
                    for (int g = 0; g + 1 < G; ++g) acc[t][i] += sums[g * kGroup + (t * MTW + i) * 64];
        }
    }
    if constexpr (SPLIT) {
        // The parts' sums through memory; the workgroup that arrives last adds them, in
        // the order of the parts.
        __shared__ uint32_t last;
        constexpr int kTileBytes = W * NTW * MTW * 1024;
        const __amdgpu_buffer_rsrc_t r = device_rsrc(a.partial + (int64_t)tile_id * a.split * (kTileBytes / 4));
        const int at = wave * NTW * MTW * 1024 + lane * 16;
        if (k_group == 0) {
#pragma unroll
            for (int t = 0; t < NTW; ++t)
#pragma unroll
                for (int i = 0; i < MTW; ++i) store_device4(r, part * kTileBytes + at + (t * MTW + i) * 1024, acc[t][i]);
        }
        if (!arrive_last(&a.counters[tile_id], a.split, &last)) return;
        if (threadIdx.x == 0) store_device(&a.counters[tile_id], 0u);
        if (k_group) return;
#pragma unroll
        for (int t = 0; t < NTW; ++t)
#pragma unroll
            for (int i = 0; i < MTW; ++i) acc[t][i] = load_device4(r, at + (t * MTW + i) * 1024);
        for (int o = 1; o < a.split; ++o)
#pragma unroll
            for (int t = 0; t < NTW; ++t)
#pragma unroll
                for (int i = 0; i < MTW; ++i) acc[t][i] += load_device4(r, o * kTileBytes + at + (t * MTW + i) * 1024);
    }

    constexpr int kRun = 16 * leave_pitch(NTW);
    static_assert((G > 1 ? W : W / 2) * kRun * 4 <= G * kStage, "the waves' rows fit one stage, or two");
    float* out = G > 1 ? reinterpret_cast<float*>(stage1) + wave * kRun
                       : reinterpret_cast<float*>(wave & 1 ? stage1 : stage0) + (wave >> 1) * kRun;
    leave<FULL>(a, w, m0 + wm * MTW * 16, (tile0 + wn * NTW) * 16, acc, out);
}

// ---------------------------------------------------------------------------
// The largest tile, 256 columns by 256 rows: eight waves of 128 x 64, K block by block.
// 4096 x 8192 x 8192 in 207 to 223 us, 2.5 P operations a second; the matrix cores are busy for 62 % of
// its cycles, and its loads bound it (262 us below are 180 without them, 255 without three quarters of its
// additions), then the stores of y, two bursts of all CUs.  160 KB hold two blocks of both operands, so a place is loaded
// again as soon as it is read: a wave has all of x in registers at a block's start, and half of the
// weights' columns at the half, where a second barrier lets the loads of the block after
// next go; the other half's go at the next block's start.  Each is on its way for one and a half
// blocks.  The rows' scales come four blocks at a time, 16 bytes of a row.  With one
// barrier, loads a block ahead and scales by the block, which are then a third of the lines
// asked for: 262 us (of column-major scales 240, and 233 with loads as here).  The two
// waves of a SIMD half a block apart, one reading while the other multiplies: 240.
// ---------------------------------------------------------------------------
constexpr int kWideTiles = 16, kScaleBlocks = 4;  // of 16 rows, or columns; scales of a row at a time

__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))
void block_wide_kernel(BlockGemmArgs a) {
    constexpr int NTW = 8, MTW = 4, WN = 2;
    // objects of their own: a load into one does not wait for reads of another
    __shared__ __attribute__((aligned(1024))) uint8_t x0[32768], x1[32768], lo0[16384], lo1[16384], hi0[16384], hi1[16384];
    __shared__ __attribute__((aligned(1024))) uint8_t row_scales[256 * kScaleBlocks * 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int quarter = lane >> 4, row = lane & 15, wn = wave % WN, wm = wave / WN;
    const int row_groups = (a.m + 255) / 256;
    const TileAt at_tile = tile_at(a, xcd_item(blockIdx.x, a.group_end[a.members - 1] * row_groups), row_groups, kWideTiles, kWideTiles);
    const int m0 = at_tile.m0, tile0 = at_tile.tile0;
    const BlockMember& w = a.member[at_tile.member];
    const int blocks = a.blocks;

    // --- loads: two tiles of x per wave, a tile of each half of the columns, 32 rows' scales
    // (extents and rows as in the kernel above)
    const int load_row = lane >> 3;
    const int load_chunk[2] = {(lane & 7) ^ turn(load_row), (lane & 7) ^ turn(load_row + 8)};
    const uint32_t x_at[2] = {(uint32_t)(load_row * a.ldx) + 16u * load_chunk[0], (uint32_t)((load_row + 8) * a.ldx) + 16u * load_chunk[1]};
    const int x_columns[2] = {a.k - 16 * load_chunk[0], a.k - 16 * load_chunk[1]};
    const uint8_t *x_from[2], *w_from[2];
    int x_bytes[2], w_bytes[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const int first = m0 + 16 * (2 * wave + p), left = min(a.m - first, 16);
        x_from[p] = a.x + (int64_t)first * a.ldx;
        x_bytes[p] = left <= 0 ? 0 : (int)((left - 1) * a.ldx) + a.k;
        const int tile = tile0 + (wave >> 2) * 8 + p * 4 + (wave & 3);
        w_from[p] = w.codes + (int64_t)(tile >> 3) * blocks * kGroupBytes + (tile & 7) * kBlockBytes;
        w_bytes[p] = tile < w.tiles ? kBlockBytes : 0;
    }
    const float* sx[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) sx[h] = a.x_scales + (int64_t)min(m0 + wave * 32 + h * 16 + (lane >> 2), a.m - 1) * a.scale_row;
    typedef __attribute__((address_space(3))) uint8_t lds_t;
    auto load_x = [&](int b, uint8_t* to, int p) {
        const int k = b * kScaleBlock;
        const uint32_t off[2] = {k < x_columns[0] ? x_at[0] : kPastEnd, k < x_columns[1] ? x_at[1] : kPastEnd};
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(x_from[p] + k), 0, max(x_bytes[p] - k, 0), 0x00020000);
#pragma unroll
        for (int h = 0; h < 2; ++h)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t*)((lds_t*)(void*)to + (2 * wave + p) * kBlockBytes + h * 1024), 16, off[h], 0, 0, 0);
    };
    auto load_w = [&](int b, uint8_t* to, int half) {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(w_from[half] + (int64_t)b * kGroupBytes), 0, b < blocks ? w_bytes[half] : 0, 0x00020000);
#pragma unroll
        for (int h = 0; h < 2; ++h)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t*)((lds_t*)(void*)to + wave * kBlockBytes + h * 1024), 16, (uint32_t)lane * 16 + h * 1024, 0, 0, 0);
    };
    auto load_scales = [&](int b) {
        const int64_t at = (int64_t)min(b + (lane & 3), blocks - 1) * a.scale_group;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            __builtin_amdgcn_global_load_lds((global_void_t*)(sx[h] + at), (lds_void_t*)((lds_t*)(void*)row_scales + wave * 512 + h * 256), 4, 0, 0);
    };

    // (w lies past the 64 KB that an LDS read's constant reaches: from a base beyond them all
    // its places are constants, 30 registers fewer)
    constexpr uint32_t kFar = 65536;
    v4f acc[NTW][MTW];
#pragma unroll
    for (int t = 0; t < NTW; ++t)
#pragma unroll
        for (int i = 0; i < MTW; ++i) acc[t][i] = v4f{0.f, 0.f, 0.f, 0.f};
    const __attribute__((address_space(4))) float* sw = (const __attribute__((address_space(4))) float*)(
        w.scales + (int64_t)(min(tile0 + wn * NTW, w.tiles - 1) >> 3) * blocks);
    const uint32_t x_slot = (uint32_t)(wm * MTW * kBlockBytes) + (uint32_t)(8 * row + (quarter ^ turn(row))) * 16;
    uint32_t w_slot = kFar + (uint32_t)(wn * 4 * kBlockBytes) + lane * 16;
    asm("" : "+v"(w_slot));
    auto fragment = [&](const uint8_t* of, int t) {
        return join(*reinterpret_cast<const u32x4_dev_t*>(of + (w_slot - kFar + t * kBlockBytes)), *reinterpret_cast<const u32x4_dev_t*>(of + (w_slot - kFar + t * kBlockBytes + 1024)));
    };

    // Per block b a wave loads, in this order: at its start hi(b + 1) (2 loads), at its half
    // x(b + 2), lo(b + 2) (6) and, every fourth, the scales from b + 2 on (2).  The start needs the
    // half's before last, the half the last start's: either way a start's and a half's may stay on their way.
    constexpr int kLag = 3;  // (as above: 240 us for 2, 257 for 1)
    float block_scale = sw[0];
    v2f scales[MTW];  // of a block and the next
    auto step = [&](int b, auto turn_of) {
        constexpr int J = decltype(turn_of)::value, kAway = 8 + (J == 3 ? 2 : 0);
        uint8_t *const xs = J & 1 ? x1 : x0, *const lo = J & 1 ? lo1 : lo0, *const hi = J & 1 ? hi1 : hi0;
        float scale[MTW], next_scale = 0.0f;
        v8i xv[MTW], wv[2];
        v4f p[kLag + 1];
        __builtin_amdgcn_s_waitcnt(step_waits(kAway));
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        wv[0] = fragment(lo, 0);
#pragma unroll
        for (int i = 0; i < MTW; ++i)
            xv[i] = join(*reinterpret_cast<const u32x4_dev_t*>(xs + x_slot + i * kBlockBytes),
                         *reinterpret_cast<const u32x4_dev_t*>(xs + (x_slot ^ 64) + i * kBlockBytes));
        if constexpr (J % 2 == 0) {
#pragma unroll
            for (int i = 0; i < MTW; ++i) scales[i] = *reinterpret_cast<const v2f*>(row_scales + ((wm * MTW + i) * 16 + row) * 16 + J * 4);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < NTW * MTW + kLag; ++q) {
            const int t = q / MTW, i = q % MTW;
            if (q == 3 * MTW) {
                __builtin_amdgcn_s_waitcnt(step_waits(kAway));
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_sched_barrier(0);
            }
            if (i == 0 && t + 1 < NTW) wv[(t + 1) & 1] = fragment(t + 1 < 4 ? lo : hi, (t + 1) % 4);
            if (t < NTW) p[q % (kLag + 1)] = block_product(wv[t & 1], xv[i]);
            if (q == kLag) {
#pragma unroll
                for (int j = 0; j < MTW; ++j) scale[j] = scales[j][J & 1] * block_scale;
            }
            if (q >= kLag) {
                const int of = q - kLag;
                v4f& sum = acc[of / MTW][of % MTW];
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] = fmaf(scale[of % MTW], p[of % (kLag + 1)][e], sum[e]);
            }
            // (here, so that no scalar load is on its way beside the LDS reads of a start:
            // they share a counter, and it could only be waited to 0)
            if (q == NTW * MTW - 1) next_scale = sw[min(b + 1, blocks - 1)];
            if (q == 1) load_w(b + 1, J & 1 ? hi0 : hi1, 1);
            if (q == 3 * MTW + 3) load_x(b + 2, xs, 0);
            if (q == 4 * MTW+3) load_x(b + 2, xs, 1);
            if (q == 5 * MTW + 3) load_w(b + 2, lo, 0);
            if (J == 2 && q == 6 * MTW) load_scales(b + 2);
            __builtin_amdgcn_sched_barrier(0);
        }
        block_scale = next_scale;
        // the sums stay in this step (the compiler would move additions to the next one)
#pragma unroll
        for (int t = 0; t < NTW; ++t)
#pragma unroll
            for (int i = 0; i < MTW; ++i) asm volatile("" : "+v"(acc[t][i]));
    };
    load_scales(0);
    load_x(0, x0, 0);
    load_x(0, x0, 1);
    load_w(0, lo0, 0);
    __builtin_amdgcn_sched_barrier(0);
    load_w(0, hi0, 1);
    __builtin_amdgcn_sched_barrier(0);
    load_x(1, x1, 0);
    load_x(1, x1, 1);
    load_w(1, lo1, 0);
    __builtin_amdgcn_sched_barrier(0);
    typedef std::integral_constant<int, 0> I0;
    typedef std::integral_constant<int, 1> I1;
    typedef std::integral_constant<int, 2> I2;
    typedef std::integral_constant<int, 3> I3;
    int b = 0;
    for (; b + 4 <= blocks; b += 4) {
        step(b, I0{});
        step(b + 1, I1{});
        step(b + 2, I2{});
        step(b + 3, I3{});
    }
    if (b < blocks) step(b, I0{});
    if (b + 1 < blocks) step(b + 1, I1{});
    if (b + 2 < blocks) step(b + 2, I2{});
    __builtin_amdgcn_s_waitcnt(0);  // the last loads (of nothing) have landed
    __syncthreads();
    constexpr int kRun = 16 * leave_pitch(NTW);
    static_assert(3 * kRun * 4 <= 32768 && kRun * 4 <= 16384, "three waves' rows fit x0 or x1, one's the others");
    uint8_t* const out = wave < 3 ? x0 + wave * kRun * 4 : wave < 6 ? x1 + (wave - 3) * kRun * 4 : wave < 7 ? lo0 : lo1;
    leave<false>(a, w, m0 + wm * MTW * 16, (tile0 + wn * NTW) * 16, acc, reinterpret_cast<float*>(out));
}
// Values [n, k] of any row stride to tiles; rows past n and columns past k are 0.
__global__ __launch_bounds__(256) void block_prepare_kernel(const uint8_t* values, int64_t ld, int64_t n, int k,
                                                            int blocks, int64_t chunks, uint8_t* out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * 256) {
        const int lane = i & 63, half = (i >> 6) & 1;
        const int64_t at = i >> 10, group = at / blocks;
        const int64_t r = group * kScaleBlock + (i >> 7 & 7) * 16 + (lane & 15);
        const int c = (int)(at - group * blocks) * kScaleBlock + half * 64 + (lane >> 4) * 16;
        uint8_t v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = r < n && c + e < k ? values[r * ld + c + e] : 0;
        uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            u[e] = v[4 * e] | (uint32_t)v[4 * e + 1] << 8 | (uint32_t)v[4 * e + 2] << 16 | (uint32_t)v[4 * e + 3] << 24;
        *reinterpret_cast<uint4*>(out + i * 16) = make_uint4(u[0], u[1], u[2], u[3]);
    }
}

// The members' column groups of so many tiles.
unsigned count_groups(BlockGemmArgs& a, int tiles) {
    unsigned groups = 0;
    for (int j = 0; j < kMaxGemmMembers; ++j) {
        if (j < a.members) groups += (a.member[j].tiles + tiles - 1) / tiles;
        a.group_end[j] = (int)groups;
    }
    return groups;
}

template <int NT, bool FULL>
hipError_t launch_stream(BlockGemmArgs a, hipStream_t s) {
    block_stream_kernel<NT, 4, FULL><<<count_groups(a, NT), kStreamWaves * 64, 0, s>>>(a);
    return hipGetLastError();
}

template <bool FULL, int NTW, int MTW, int WN, int WM, int S, int G, int EU, bool SPLIT = false, bool PAST = false>
hipError_t launch_tile(BlockGemmArgs a, hipStream_t s) {
    const unsigned tiles = count_groups(a, NTW * WN) * ((a.m + 16 * MTW * WM - 1) / (16 * MTW * WM));
    block_tile_kernel<NTW, MTW, WN, WM, S, G, EU, SPLIT, PAST, FULL><<<SPLIT ? tiles * a.split : tiles, G * WN * WM * 64, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_wide(BlockGemmArgs a, hipStream_t s) {
    block_wide_kernel<<<count_groups(a, kWideTiles) * ((a.m + 255) / 256), 512, 0, s>>>(a);
    return hipGetLastError();
}

template <bool FULL>
hipError_t launch_any(const BlockGemmArgs& a, hipStream_t s) {
    int64_t tiles = 0;
    for (int j = 0; j < a.members; ++j) tiles += a.member[j].tiles;
    // Weights that the 256 MB cache cannot hold, read by one workgroup each, are read past
    // it: 64 rows of 151936 x 4096 131 and 125 us, 128 rows 156 and 147; 64 rows of 65536 x 4096, which
    // it all but holds, 45 and 56; by two workgroups, 128 rows of 24576 x 4096 in 64-row tiles, 39 and 41.
    const bool large = tiles * a.blocks * kBlockBytes > kPastCacheBytes;
    switch (a.tile) {
        case 1: return launch_tile<FULL, 2, 2, 2, 2, 3, 1, 3>(a, s);
        case 2:
            return large && a.m <= 64 ? launch_tile<FULL, 4, 2, 2, 2, 3, 1, 2, false, true>(a, s) : launch_tile<FULL, 4, 2, 2, 2, 3, 1, 2>(a, s);
        case 3:
            return large && a.m <= 128 ? launch_tile<FULL, 4, 4, 4, 2, 3, 1, 2, false, true>(a, s) : launch_tile<FULL, 4, 4, 4, 2, 3, 1, 2>(a, s);
        case 4: return FULL ? hipErrorInvalidValue : launch_wide(a, s);
        case 5: return a.split > 1 ? launch_tile<FULL, 2, 2, 2, 2, 4, 2, 2, true>(a, s) : launch_tile<FULL, 2, 2, 2, 2, 4, 2, 2>(a, s);
        default: break;
    }
    // the more columns there are, the fewer times x is read
    if (tiles >= 2048) return launch_stream<4, FULL>(a, s);
    return tiles >= 1024 ? launch_stream<2, FULL>(a, s) : launch_stream<1, FULL>(a, s);
}

}  // namespace

hipError_t launch_block_gemm(const BlockGemmArgs& a, hipStream_t s) {
    return a.out == 2 ? launch_any<true>(a, s) : launch_any<false>(a, s);
}

hipError_t launch_block_prepare(const uint8_t* values, int64_t ld, int64_t n, int64_t k, uint8_t* out, hipStream_t s) {
    const int blocks = (int)((k + kScaleBlock - 1) / kScaleBlock);
    const int64_t chunks = (n + kScaleBlock - 1) / kScaleBlock * blocks * 1024, groups = (chunks + 255) / 256;
    block_prepare_kernel<<<(unsigned)(groups < (1 << 20) ? groups : (1 << 20)), 256, 0, s>>>(values, ld, n, (int)k, blocks,
                                                                                           chunks, out);
    return hipGetLastError();
}

}  // namespace cubic
