// Row norms and 8-bit activations for gfx950.
//
//   norm      h = x + r,  y = h * (offset + w) / sqrt(mean(h^2) + eps)
//   quantise  y = x,  or  y = silu(g) x = g x / (1 + exp(-g))
//
// y leaves in 16 bits, and / or per group of 128 columns as a 32-bit scale
// s = max(max |y|, 2^-96) / 448 and values q = e4m3(y * (448 / max(max |y|, 2^-96))),
// so that q s stands for y (448: the largest e4m3 value; 2^-96, small beside any
// activation, keeps 448 / top and what is scaled by it far from the largest number).  h leaves in 16 bits too.  All is
// held in 32 bits and each output rounded once: y is computed from h as added, not
// from the rounded one.  A NaN or an infinity makes all of its group NaN.
//
// What bounds it: the bytes of the rows.  A row is read once, its columns stay in
// registers, eight to a vector, between the sum of squares and the outputs.  A
// group of 128 columns is the vectors of 16 lanes, one DPP row: its maximum
// takes four lane exchanges and no LDS.
#include "cubic_capi_internal.h"
#include "cubic_device.h"

namespace cubic {
namespace {

constexpr int kVec = 8;          // columns of a thread's vector
constexpr float kTop = 448.0f;   // largest e4m3 value
constexpr float kSmallest = 0x1p-96f;

template <bool F16>
__device__ __forceinline__ float from_bits(uint32_t b) {
    return F16 ? half_bits_to_float(b) : bf16_bits_to_float(b);
}
template <bool F16>
__device__ __forceinline__ uint32_t to_bits(float f) {
    return F16 ? float_to_f16_bits(f) : float_to_bf16_bits(f);
}

// Columns c..c+7 of a row; the ones past k read as zero.  Global memory takes 16 bytes at any
// element's address: 2000 rows of 4097 columns by single elements take 44 us, by vectors 16.
template <bool F16>
__device__ __forceinline__ void load8(const uint16_t* row, int c, int k, float (&v)[kVec]) {
    if (c + kVec <= k) {
        uint32_t u[4];
        __builtin_memcpy(u, row + c, sizeof u);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = from_bits<F16>(u[i] & 0xFFFFu);
            v[2 * i + 1] = from_bits<F16>(u[i] >> 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[i] = c + i < k ? from_bits<F16>(row[c + i]) : 0.0f;
    }
}

typedef u32x4_dev_t any_u32x4_t __attribute__((aligned(2)));

// PAST: past the caches.
template <bool F16, bool PAST>
__device__ __forceinline__ void store8(uint16_t* row, int c, int k, const float (&v)[kVec]) {
    if (c + kVec <= k) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            u[i] = F16 ? to_bits<F16>(v[2 * i]) | to_bits<F16>(v[2 * i + 1]) << 16 : pack_bf16x2(v[2 * i], v[2 * i + 1]);
        const u32x4_dev_t w = {u[0], u[1], u[2], u[3]};
        if constexpr (PAST) __builtin_nontemporal_store(w, reinterpret_cast<any_u32x4_t*>(row + c));
        else *reinterpret_cast<any_u32x4_t*>(row + c) = w;
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
            if (c + i < k) row[c + i] = (uint16_t)to_bits<F16>(v[i]);
    }
}

// silu(g) x, from exp(-|g|) = 2^t with t = -|g| log2(e) in two parts, so that the error
// does not grow with |g|.  Past 64 below zero silu(g) = g exp(g), under 2^128, which x brings
// back to the 32-bit numbers: half of those powers of two are taken off x, half off the product.
__device__ __forceinline__ float gated(float g, float x) {
    constexpr float kHi = 1.44269502162933349609375f, kLo = 1.92596299112661746887e-8f;  // log2(e)
    const float a = fabsf(g), t = -a * kHi;
    const float rest = fmaf(-a, kHi, -t) + -a * kLo;
    const bool far = a > 64.0f;
    float e = __builtin_amdgcn_exp2f(far ? t + 128.0f : t);
    e = e > 0.0f ? fmaf(e, rest * 0.693147182464599609375f, e) : e;  // (the rest of an infinite t is none)
    const float down = far && g < 0.0f ? 0x1p-64f : 1.0f;
    return (g < 0.0f ? g * e : g) * __builtin_amdgcn_rcpf(1.0f + (far ? 0.0f : e)) * (x * down) * down;
}

// Quantises the eight columns of every lane; the 16 lanes of a DPP row hold a
// group.  Every lane of the wave calls it.
template <bool PAST>
__device__ __forceinline__ void quantise8(const RowArgs& a, int64_t row, int c, const float (&y)[kVec]) {
    uint32_t most = 0;  // of the magnitudes' bits: a NaN is above an infinity
#pragma unroll
    for (int i = 0; i < kVec; ++i) most = max(most, __float_as_uint(y[i]) & 0x7FFFFFFFu);
    most = max(most, dpp_u32<0xB1>(most));
    most = max(most, dpp_u32<0x4E>(most));
    most = max(most, dpp_u32<0x141>(most));
    most = max(most, dpp_u32<0x140>(most));
    if (c >= a.k) return;
    const float top = __uint_as_float(max(most, __float_as_uint(kSmallest)));
    const float inverse = kTop / top;
    if ((threadIdx.x & 15) == 0) a.scales[row * a.scale_row + (int64_t)(c >> 7) * a.scale_group] = top / kTop;
    uint32_t lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * inverse, y[1] * inverse, lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] * inverse, y[3] * inverse, lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4] * inverse, y[5] * inverse, hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6] * inverse, y[7] * inverse, hi, true);
    uint8_t* q = a.q + row * a.ldq + c;
    if (c + kVec <= a.k) {
        typedef uint32_t any_u32x2_t __attribute__((ext_vector_type(2), aligned(1)));
        const any_u32x2_t u = {lo, hi};
        if constexpr (PAST) __builtin_nontemporal_store(u, reinterpret_cast<any_u32x2_t*>(q));
        else *reinterpret_cast<any_u32x2_t*>(q) = u;
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
            if (c + i < a.k) q[i] = (uint8_t)((i < 4 ? lo : hi) >> (8 * (i & 3)));
    }
}

// The sum over a workgroup's threads, in a fixed order; `sums` is reused by the
// next row after a barrier.
template <bool WAVE>
__device__ __forceinline__ float row_sum(float part, float* sums) {
    part = wave_butterfly_sum(part, 64);
    if constexpr (WAVE) return part;
    const int waves = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = part;
    __syncthreads();
    const int of = threadIdx.x & 15;  // every 16 lanes add all waves' sums
    return wave_butterfly_sum(of < waves ? sums[of] : 0.0f, 16);
}

// One row per workgroup, or per wave (WAVE: blockDim.x == 64, four rows to a
// workgroup); NV vectors per thread cover it.  NV = 0: any length, the row is read
// again (from the caches) for the outputs, and a thread's many additions carry their rounding.
template <bool F16, int NV, bool WAVE, bool PAST>
__global__ __launch_bounds__(1024) void row_norm_kernel(RowArgs a) {
    __shared__ float sums[16];
    constexpr int N = NV ? NV : 1;
    const int turns = (a.k + blockDim.x * kVec - 1) / (blockDim.x * kVec);
    const uint16_t* x = static_cast<const uint16_t*>(a.x);
    const uint16_t* other = static_cast<const uint16_t*>(a.other);
    const uint16_t* weight = static_cast<const uint16_t*>(a.weight);
    for (int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; row < a.m; row += (int64_t)gridDim.x * blockDim.y) {
        float v[N][kVec];
        auto read = [&](int i, float (&h)[kVec]) {
            const int c = (i * blockDim.x + threadIdx.x) * kVec;
            load8<F16>(x + row * a.ldx, c, a.k, h);
            if (other) {
                float o[kVec];
                load8<F16>(other + row * a.ldother, c, a.k, o);
#pragma unroll
                for (int e = 0; e < kVec; ++e) h[e] += o[e];
            }
        };
        auto write = [&](int i, float shift, float factor, float (&h)[kVec]) {
            const int c = (i * blockDim.x + threadIdx.x) * kVec;
            // (the sum is read again a layer later: 4096 x 8192 in 55.9 and 52.1 us past the caches)
            if (a.sum) store8<F16, true>(static_cast<uint16_t*>(a.sum) + row * a.ldsum, c, a.k, h);
            float w[kVec];
            load8<F16>(weight, c, a.k, w);
#pragma unroll
            for (int e = 0; e < kVec; ++e) h[e] = h[e] * shift * factor * (a.offset + w[e]);
            if (a.y) store8<F16, PAST>(static_cast<uint16_t*>(a.y) + row * a.ldy, c, a.k, h);
            if (a.q) quantise8<PAST>(a, row, c, h);
        };
        if constexpr (NV != 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) read(i, v[i]);
        }
        auto squares = [&](float shift) __attribute__((always_inline)) {  // of h * shift, over the row
            float part = 0.0f, rest = 0.0f;
            if constexpr (NV != 0) {
#pragma unroll
                for (int i = 0; i < N; ++i)
#pragma unroll
                    for (int e = 0; e < kVec; ++e) part = fmaf(v[i][e] * shift, v[i][e] * shift, part);
            }
            for (int i = 0; i < (NV ? 0 : turns); ++i) {  // what an addition rounds off goes into the next
                read(i, v[0]);
                float eight = 0.0f;
#pragma unroll
                for (int e = 0; e < kVec; ++e) eight = fmaf(v[0][e] * shift, v[0][e] * shift, eight);
                const float more = eight - rest, next = part + more;
                rest = next < __builtin_huge_valf() ? (next - part) - more : 0.0f;
                part = next;
            }
            return row_sum<WAVE>(part, sums);
        };
        // Where the sum leaves the 32-bit numbers the squares are taken of h times a power of two
        // (of at most 2^48 then, 2^24 of them; of at least 2^-53).  Small ones matter beside a
        // small epsilon only.  (4096 x 8192 to 8 bits: 48.2 us without this, and 48.6.)
        float sum = squares(1.0f), shift = 1.0f;
        const bool large = sum > 0x1.fffffep127f, small = sum < 0x1p-100f && a.epsilon < 0x1p-76f;
        if (__builtin_expect(large || small, 0)) {
            if constexpr (!WAVE) __syncthreads();  // the sums are read
            shift = large ? 0x1p-80f : 0x1p80f;
            sum = squares(shift);
        }
        const float factor = 1.0f / sqrtf(sum / (float)a.k + a.epsilon * shift * shift);
        if constexpr (NV != 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) write(i, shift, factor, v[i]);
        } else {
            for (int i = 0; i < turns; ++i) {
                read(i, v[0]);
                write(i, shift, factor, v[0]);
            }
        }
        if constexpr (!WAVE) __syncthreads();  // the sums are read
    }
}

// 2048 columns per workgroup and turn: blockDim.x vectors of blockDim.y rows.
// blockDim.x is a multiple of 16, so a group's lanes are one DPP row.
template <bool F16, bool GATED, bool PAST>
__global__ __launch_bounds__(256) void quantize_kernel(RowArgs a) {
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * kVec;
    for (int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; row < a.m; row += (int64_t)gridDim.x * blockDim.y) {
        float y[kVec];
        load8<F16>(static_cast<const uint16_t*>(a.x) + row * a.ldx, c, a.k, y);
        if constexpr (GATED) {
            float g[kVec];
            load8<F16>(static_cast<const uint16_t*>(a.other) + row * a.ldother, c, a.k, g);
#pragma unroll
            for (int e = 0; e < kVec; ++e) y[e] = gated(g[e], y[e]);
        }
        quantise8<PAST>(a, row, c, y);
    }
}

template <bool F16, bool PAST>
hipError_t launch_norm(const RowArgs& a, hipStream_t s) {
    const int vectors = (a.k + kVec - 1) / kVec;
    const int64_t most = 1 << 18;  // workgroups; the rest of the rows in turns
    if (vectors <= 128) {
        const dim3 block(64, 4), grid((unsigned)((a.m + 3) / 4 < most ? (a.m + 3) / 4 : most));
        if (vectors <= 64) row_norm_kernel<F16, 1, true, PAST><<<grid, block, 0, s>>>(a);
        else row_norm_kernel<F16, 2, true, PAST><<<grid, block, 0, s>>>(a);
        return hipGetLastError();
    }
    const dim3 grid((unsigned)(a.m < most ? a.m : most));
    auto threads = [&](int nv) { return (unsigned)((vectors + nv * 64 - 1) / (nv * 64) * 64); };
    if (vectors <= 512 || (vectors <= 1024 && a.m <= 512)) row_norm_kernel<F16, 1, false, PAST><<<grid, threads(1), 0, s>>>(a);
    else if (vectors <= 2048) row_norm_kernel<F16, 2, false, PAST><<<grid, threads(2), 0, s>>>(a);
    else if (vectors <= 4096) row_norm_kernel<F16, 4, false, PAST><<<grid, threads(4), 0, s>>>(a);
    else row_norm_kernel<F16, 0, false, PAST><<<grid, 1024, 0, s>>>(a);
    return hipGetLastError();
}

template <bool F16, bool PAST>
hipError_t launch_quantize(const RowArgs& a, hipStream_t s) {
    // a row's vectors evenly over as few workgroups as hold them (1999 x 4104: 6.6 us, and
    // 7.7 with a second workgroup per row for what 256 threads leave)
    const int vectors = (a.k + kVec - 1) / kVec, chunks = (vectors + 255) / 256;
    const unsigned across = ((vectors + chunks - 1) / chunks + 15) / 16 * 16, down = 256 / across;
    const int64_t rows = (a.m + down - 1) / down, most = 1 << 16;
    const dim3 block(across, down), grid((unsigned)(rows < most ? rows : most), (vectors + across - 1) / across);
    if (a.other) quantize_kernel<F16, true, PAST><<<grid, block, 0, s>>>(a);
    else quantize_kernel<F16, false, PAST><<<grid, block, 0, s>>>(a);
    return hipGetLastError();
}

template <bool PAST>
hipError_t launch_any(const RowArgs& a, hipStream_t s) {
    if (a.norm) return a.f16 ? launch_norm<true, PAST>(a, s) : launch_norm<false, PAST>(a, s);
    return a.f16 ? launch_quantize<true, PAST>(a, s) : launch_quantize<false, PAST>(a, s);
}

}  // namespace

hipError_t launch_rows(const RowArgs& a, hipStream_t s) {
    // Outputs of 16 Mi elements and more leave past the caches: 4096 x 8192 to 8 bits in 50 and 42 us,
    // to 16 bits in 53 and 41 (with a product of 8192 columns and a norm behind it the same, 330);
    // 1024 x 4096, whose 8 bits the product behind finds in a cache, 42 us without and 45 with.
    return a.m * a.k >= (int64_t)1 << 24 ? launch_any<true>(a, s) : launch_any<false>(a, s);
}

}  // namespace cubic
