// Low-rank adapters of many requests beside a shared projection (gfx950):
//
//   t[i, :]   = A_e x[i, :]                         e = row_slots[i], rank r_e
//   y[i, :]   = round16(base[i, :] + s_e B_e t[i, :])
//
// for up to kMaxGemmMembers projections that share x, in two launches: the
// down kernel writes t as binary32 partial sums over K partitions, the up
// kernel adds the partitions in ascending order and finishes the rows.
//
// Rows come in any order.  A tile of consecutive rows is walked once per
// distinct adapter in it (a ballot over the tile's slots finds the rows of
// each), so a prompt's rows, which share an adapter, are one matrix product and
// a decode batch whose rows all differ reads each adapter once, without a
// grouping launch or any host knowledge of the slots.
//
// Arithmetic order: K partitions of kDownK columns, a quarter per wave, the
// quarters added as (0 + 1) + (2 + 3); then the rank in steps of 32.  Nothing
// of it depends on m, on the tile or on the other rows, so a row's result is
// the same bit for bit whichever batch it is in.
#include "cubic_gemm_common.h"

namespace cubic {
namespace {

using gemm::floatx4_t;
using gemm::mfma16;

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kDownK = kAdapterDownK;       // columns of x per workgroup
constexpr int kWaveK = kDownK / kWaves;     // ... per wave
constexpr int kSteps = kWaveK / 32;         // MFMA steps per wave
constexpr uint32_t kOutside = 0x80000000u;  // added to a byte offset: past every buffer, reads 0

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}

__device__ __forceinline__ uint4 load16(__amdgpu_buffer_rsrc_t r, uint32_t byte_offset) {
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)byte_offset, 0, 0));
}

// The tile's adapter slots, one per lane (-1: past the batch, kNone: no
// adapter), the same in every wave: one wave reads them, so that waves cannot
// disagree on the walk (and its barriers) if the caller rewrites them meanwhile.
constexpr int kNone = -2;
template <int ROWS>
__device__ __forceinline__ int tile_slots(const AdapterArgs& a, int row0, int* lds) {
    if (threadIdx.x < 64) {
        int slot = -1;
        if ((int)threadIdx.x < ROWS && row0 + (int)threadIdx.x < a.m) {
            slot = a.row_slots[row0 + threadIdx.x];
            if (slot < 0 || slot >= a.slots) slot = kNone;
        }
        lds[threadIdx.x] = slot;
    }
    __syncthreads();
    return lds[threadIdx.x & 63];
}

// ---------------------------------------------------------------------------
// t = A x.  Workgroup: 16 * MT rows x RT 16-rank tiles x kDownK columns.  MFMA
// operands straight from memory: the first is A (its rows are the ranks), the
// second x, so a lane ends with four consecutive ranks of one row.
// ---------------------------------------------------------------------------
template <bool F16, int MT, int RT, int S>
__global__ __launch_bounds__(kThreads) void adapter_down_kernel(AdapterArgs a) {
    constexpr int kRows = 16 * MT;
    __shared__ int slots_lds[64];
    __shared__ floatx4_t red[2][MT * RT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, q = lane >> 4;
    const int tile = blockIdx.x / a.down_groups, group = blockIdx.x % a.down_groups;
    const int row0 = tile * kRows;
    const int slot = tile_slots<kRows>(a, row0, slots_lds);

    const int rows = min(kRows, a.m - row0);
    const auto x = buffer(a.x + (int64_t)row0 * a.ldx, ((int64_t)(rows - 1) * a.ldx + a.k) * 2);
    const int k0 = blockIdx.y * kDownK + wave * kWaveK + q * 8;
    // the rank tiles of this workgroup: member and first rank of each
    const uint16_t* down[RT];
    const int32_t* ranks[RT];
    int max_rank[RT], first[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int v = blockIdx.z * RT + t;
        down[t] = a.member[0].down;
        ranks[t] = a.member[0].ranks;
        max_rank[t] = 0;
        first[t] = 0;
#pragma unroll
        for (int j = 0; j < kMaxGemmMembers; ++j)
            if (v >= a.member[j].tile0 && v < a.member[j].tile1) {
                down[t] = a.member[j].down;
                ranks[t] = a.member[j].ranks;
                max_rank[t] = a.member[j].max_rank;
                first[t] = (v - a.member[j].tile0) * 16;
            }
    }

    uint64_t left = __ballot(slot >= 0);
    for (int order = 0; left; ++order) {
        const int lead = __builtin_ctzll(left);
        const int e = __builtin_amdgcn_readlane(slot, lead);
        const uint64_t mine = __ballot(slot == e);
        left &= ~mine;
        if (order % a.down_groups != group) continue;
        uint32_t xoff[MT], doff[RT];
        __amdgpu_buffer_rsrc_t d[RT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            // rows of other adapters repeat the first row: their columns of
            // the product are not stored
            const int r = (mine >> (16 * i + col)) & 1 ? 16 * i + col : lead;
            xoff[i] = (uint32_t)r * (uint32_t)(a.ldx * 2);
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int rank = max_rank[t] ? min(ranks[t][e], max_rank[t]) : 0;
            d[t] = buffer(down[t] + (int64_t)e * max_rank[t] * a.k, (int64_t)max_rank[t] * a.k * 2);
            doff[t] = first[t] + col < rank ? (uint32_t)(first[t] + col) * (uint32_t)(a.k * 2) : kOutside;
        }
        uint4 xf[S][MT], df[S][RT];
        auto issue = [&](int s) {
            const int kk = k0 + s * 32;
            const uint32_t ko = kk < a.k ? (uint32_t)kk * 2 : kOutside;
#pragma unroll
            for (int t = 0; t < RT; ++t) df[s % S][t] = load16(d[t], doff[t] == kOutside ? kOutside : doff[t] + ko);
#pragma unroll
            for (int i = 0; i < MT; ++i) xf[s % S][i] = load16(x, xoff[i] + ko);
        };
        floatx4_t acc[MT][RT];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[i][t] = floatx4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < S; ++s) issue(s);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int t = 0; t < RT; ++t) acc[i][t] = mfma16<F16>(df[s % S][t], xf[s % S][i], acc[i][t]);
            if (s + S < kSteps) issue(s + S);
        }
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
                float* out = a.partial + ((int64_t)blockIdx.y * a.m + row0 + 16 * i + col) * a.width +
                             blockIdx.z * RT * 16 + 4 * q;
#pragma unroll
                for (int t = 0; t < RT; ++t)
                    if (blockIdx.z * RT + t < a.tiles)
                        *(floatx4_t*)(out + 16 * t) = acc[i][t] + red[0][i * RT + t][lane];
            }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// y = base + s B t.  Workgroup: 16 * MT rows x a chunk of one member's columns,
// 32 columns per wave and turn.  The first MFMA operand is B with its rows
// (columns of y) permuted so that a lane ends with eight consecutive columns of
// one row: two 16-row tiles, row 4 q + s of tile u standing for column 8 q + 4 u
// + s.  t is split into two 16-bit parts, t = hi + lo with an error below 2^-17
// (bf16) or 2^-22 of the row's largest (fp16) of t, so that the only rounding
// to 16 bits that counts is y's; the operator is bound by y's bytes, and the
// second product costs matrix time that is idle.  fp16 parts are taken of t
// scaled by a power of two to at most 1, which fp16's range needs and which
// changes no digit of the product.
// ---------------------------------------------------------------------------
template <bool F16>
__device__ __forceinline__ void split_parts(const float* t, uint4& hi, uint4& lo) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const float a = t[2 * p], b = t[2 * p + 1];
        h[p] = gemm::pack_level2<F16>(a, b);
        float ha, hb;
        if constexpr (F16) {
            ha = half_bits_to_float(h[p] & 0xffffu);
            hb = half_bits_to_float(h[p] >> 16);
        } else {
            ha = bf16_bits_to_float(h[p] & 0xffffu);
            hb = bf16_bits_to_float(h[p] >> 16);
        }
        // an infinity or NaN is whole in its first part
        l[p] = gemm::pack_level2<F16>(__builtin_isfinite(ha) ? a - ha : 0.f, __builtin_isfinite(hb) ? b - hb : 0.f);
    }
    hi = uint4{h[0], h[1], h[2], h[3]};
    lo = uint4{l[0], l[1], l[2], l[3]};
}

template <bool F16, int MT, int KS, bool VEC>
__global__ __launch_bounds__(kThreads) void adapter_up_kernel(AdapterArgs a) {
    constexpr int kRows = 16 * MT, kPitch = KS * 32 + 4;
    __shared__ int slots_lds[64];
    __shared__ __attribute__((aligned(16))) float tl[kRows][kPitch];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, q = lane >> 4;
    const int tile = blockIdx.x / a.up_groups, group = blockIdx.x % a.up_groups;
    const int row0 = tile * kRows;
    const int slot = tile_slots<kRows>(a, row0, slots_lds);

    // member of this column chunk
    AdapterMember mb = a.member[0];
#pragma unroll
    for (int j = 1; j < kMaxGemmMembers; ++j)
        if ((int)blockIdx.y >= a.member[j].chunk0 && (int)blockIdx.y < a.member[j].chunk1) mb = a.member[j];
    const int c_begin = ((int)blockIdx.y - mb.chunk0) * a.chunk_cols;
    const int c_end = min(mb.n, c_begin + a.chunk_cols);

    uint64_t left = __ballot(slot != -1);
    for (int order = 0; left; ++order) {
        const int lead = __builtin_ctzll(left);
        const int e = __builtin_amdgcn_readlane(slot, lead);
        const uint64_t mine = __ballot(slot == e);
        left &= ~mine;
        if (order % a.up_groups != group) continue;
        const int rank = e >= 0 ? min(mb.ranks[e], mb.max_rank) : 0;
        const float scale = e >= 0 ? mb.scales[e] : 0.f;
        __syncthreads();  // the last turn's reads of tl
        for (int i = threadIdx.x; i < kRows * KS * 8; i += kThreads) {
            const int r = i / (KS * 8), f = (i % (KS * 8)) * 4;
            floatx4_t v = {0.f, 0.f, 0.f, 0.f};
            if (f < rank && ((mine >> r) & 1)) {
                const float* p = a.partial + (int64_t)(row0 + r) * a.width + mb.tile0 * 16 + f;
                for (int s = 0; s < a.split; ++s) v += *(const floatx4_t*)(p + (int64_t)s * a.m * a.width);
#pragma unroll
                for (int c = 0; c < 4; ++c) v[c] = f + c < rank ? v[c] * scale : 0.f;
            }
            *(floatx4_t*)&tl[r][f] = v;
        }
        __syncthreads();
        uint4 hi[MT][KS], lo[MT][KS];
        float back[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            float t[KS][8];
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int c = 0; c < 8; c += 4) {
                    const floatx4_t v = *(const floatx4_t*)&tl[16 * i + col][s * 32 + q * 8 + c];
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        t[s][c + d] = v[d];
                        top = fmaxf(top, fabsf(v[d]));
                    }
                }
            back[i] = 1.f;
            if constexpr (F16) {
                top = fmaxf(top, __uint_as_float(xor16_u32(__float_as_uint(top))));
                top = fmaxf(top, __uint_as_float(xor32_u32(__float_as_uint(top))));
                // 2^-(exponent + 1) of the row's largest, kept within normal numbers
                int ex = (int)(__float_as_uint(top) >> 23) - 126;
                ex = top == 0.f || !__builtin_isfinite(top) ? 0 : min(max(ex, -120), 120);
                const float down = __uint_as_float((uint32_t)(127 - ex) << 23);
                back[i] = __uint_as_float((uint32_t)(127 + ex) << 23);
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int c = 0; c < 8; ++c) t[s][c] *= down;
            }
#pragma unroll
            for (int s = 0; s < KS; ++s) split_parts<F16>(t[s], hi[i][s], lo[i][s]);
        }
        const auto up = buffer(mb.up + (e >= 0 ? (int64_t)e * mb.n * mb.max_rank : 0), (int64_t)mb.n * mb.max_rank * 2);
        for (int c0 = c_begin + wave * 32; c0 < c_end; c0 += kWaves * 32) {
            floatx4_t acc[MT][2];
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i][0] = acc[i][1] = floatx4_t{0.f, 0.f, 0.f, 0.f};
            if (rank > 0) {
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int c = c0 + 8 * (col >> 2) + 4 * u + (col & 3), r = s * 32 + q * 8;
                        const uint4 b = load16(up, r < rank && c < mb.n ? (uint32_t)(c * mb.max_rank + r) * 2 : kOutside);
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            acc[i][u] = mfma16<F16>(b, lo[i][s], acc[i][u]);
                            acc[i][u] = mfma16<F16>(b, hi[i][s], acc[i][u]);
                        }
                    }
            }
            const int cy = c0 + 8 * q;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if (!((mine >> (16 * i + col)) & 1) || cy >= mb.n) continue;
                const int64_t row = row0 + 16 * i + col;
                const uint16_t* base = mb.base + row * mb.ldbase + cy;
                uint16_t* y = mb.y + row * mb.ldy + cy;
                uint16_t in[8], out[8];
                if constexpr (VEC) {
                    *(uint4*)in = *(const uint4*)base;
                } else {
#pragma unroll
                    for (int c = 0; c < 8; ++c) in[c] = cy + c < mb.n ? base[c] : 0;
                }
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const float b = F16 ? half_bits_to_float(in[c]) : bf16_bits_to_float(in[c]);
                    const float d = acc[i][c >> 2][c & 3] * back[i];
                    out[c] = rank > 0 ? gemm::out_bits<F16>(b + d) : in[c];
                }
                if constexpr (VEC) {
                    *(uint4*)y = *(const uint4*)out;
                } else {
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        if (cy + c < mb.n) y[c] = out[c];
                }
            }
        }
    }
}

template <bool F16, int MT, int RT, int S>
void start_down(const AdapterArgs& a, hipStream_t s) {
    const dim3 grid((a.m + 16 * MT - 1) / (16 * MT) * a.down_groups, a.split, (a.tiles + RT - 1) / RT);
    adapter_down_kernel<F16, MT, RT, S><<<grid, kThreads, 0, s>>>(a);
}

template <bool F16, int MT>
void start_down_tiles(const AdapterArgs& a, hipStream_t s) {
    if (a.tiles == 1) start_down<F16, MT, 1, 8>(a, s);
    else if (a.tiles == 2) start_down<F16, MT, 2, MT == 4 ? 4 : 8>(a, s);
    else if (a.tiles <= 4) start_down<F16, MT, 4, 4>(a, s);
    else start_down<F16, MT, 8, MT == 4 ? 2 : 4>(a, s);
}

template <bool F16, int MT, int KS>
void start_up(const AdapterArgs& a, hipStream_t s) {
    const dim3 grid((a.m + 16 * MT - 1) / (16 * MT) * a.up_groups, a.chunks);
    if (a.vectors) adapter_up_kernel<F16, MT, KS, true><<<grid, kThreads, 0, s>>>(a);
    else adapter_up_kernel<F16, MT, KS, false><<<grid, kThreads, 0, s>>>(a);
}

template <bool F16, int MT>
void start_up_steps(const AdapterArgs& a, hipStream_t s) {
    if (a.rank_steps == 1) start_up<F16, MT, 1>(a, s);
    else if (a.rank_steps == 2) start_up<F16, MT, 2>(a, s);
    else if (a.rank_steps <= 4) start_up<F16, MT, 4>(a, s);
    else if constexpr (MT < 4) start_up<F16, MT, 8>(a, s);
}

template <bool F16>
hipError_t start(const AdapterArgs& a, hipStream_t s) {
    if (a.down_rows == 1) start_down_tiles<F16, 1>(a, s);
    else if (a.down_rows == 2) start_down_tiles<F16, 2>(a, s);
    else start_down_tiles<F16, 4>(a, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.up_rows == 1) start_up_steps<F16, 1>(a, s);
    else if (a.up_rows == 2) start_up_steps<F16, 2>(a, s);
    else start_up_steps<F16, 4>(a, s);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_adapters(const AdapterArgs& a, hipStream_t s) {
    return a.f16 ? start<true>(a, s) : start<false>(a, s);
}

}  // namespace cubic
