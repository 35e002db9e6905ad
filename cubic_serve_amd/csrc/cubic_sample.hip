// Sampling from the whole vocabulary (gfx950): per row one token under
// temperature T, top-k, top-p and min-p, from a given uniform number u.
//
// Order of a row: logit descending, column ascending on ties (-0 == +0).  Weight
// of a column: w = 2^((l - max) log2(e) / T), in 64-bit fixed point with 2^43 for
// the maximum (so up to 2^20 columns sum below 2^63 and sums do not depend on
// their order; a weight is off by at most half a unit, 2^-44 of the maximum's).
// What top-k, top-p and min-p keep is a prefix of the order each, and a prefix is
// as good as its mass:
//   S_k  mass of the first k
//   S_p  mass through the first position whose inclusive mass reaches top_p S_k
//   S_m  mass of the weights of at least min_p
//   S = min(S_k, S_p, S_m); the token is the first position whose inclusive mass
//   exceeds u S; its log-probability ln(w / S).
// So a row takes at most three searches "first position whose inclusive count or
// mass reaches X", each a descent over the bits of the logits' ordered keys.
#include "cubic_device.h"
#include "cubic_capi_internal.h"

namespace cubic {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 4096;
constexpr double kOne = 8796093022208.0;  // 2^43

// Keys order as the logits do: larger logit, larger key; NaN keys lie past
// both infinities' (negative NaN below, positive above).
__device__ __forceinline__ uint32_t ordered(uint32_t bits) {
    if (bits == 0x80000000u) bits = 0;  // -0 is +0
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ uint32_t unordered(uint32_t key) {
    return key & 0x80000000u ? key & 0x7fffffffu : ~key;
}

// TYPE: CUBIC_DTYPE_BF16 / _F16 / _F32.  A 16-bit logit's key fills the upper
// half of a 32-bit one, so that the descents share their code.
template <int TYPE>
__device__ __forceinline__ uint32_t key_of(uint32_t bits) {
    if constexpr (TYPE == 2) return ordered(bits);
    else return ordered(bits << 16) & 0xffff0000u;
}
template <int TYPE>
__device__ __forceinline__ double value_of(uint32_t key) {
    if constexpr (TYPE == 1) {
        const uint32_t low = key & 0x80000000u ? key & 0x7fff0000u : ~key & 0xffff0000u;
        return (double)half_bits_to_float(low >> 16);
    } else if constexpr (TYPE == 0) {
        const uint32_t low = key & 0x80000000u ? key & 0x7fff0000u : ~key & 0xffff0000u;
        return (double)__uint_as_float(low);
    } else {
        return (double)__uint_as_float(unordered(key));
    }
}
template <int TYPE>
struct Limits {  // keys of +inf and -inf
    static constexpr uint32_t kInf = TYPE == 1 ? 0xfc000000u : 0xff800000u;
    static constexpr uint32_t kNegInf = TYPE == 2 ? ~0xff800000u : TYPE == 0 ? ~0xff800000u & 0xffff0000u
                                                                           : ~0xfc000000u & 0xffff0000u;
};

// 2^t for t <= 0 in fixed point (2^43 at t = 0): 2^t = 2^n 2^f, |f| <= 1/2, the
// second factor by the Taylor polynomial of e^(f ln 2) of degree 11 (off by
// less than 1e-14).
__device__ __forceinline__ uint64_t fixed_weight(double t) {
    if (!(t > -46.0)) return 0;
    const double n = __builtin_rint(t);
    const double x = (t - n) * 0.69314718055994530942;
    double p = 1.0 / 39916800.0;
    p = __builtin_fma(p, x, 1.0 / 3628800.0);
    p = __builtin_fma(p, x, 1.0 / 362880.0);
    p = __builtin_fma(p, x, 1.0 / 40320.0);
    p = __builtin_fma(p, x, 1.0 / 5040.0);
    p = __builtin_fma(p, x, 1.0 / 720.0);
    p = __builtin_fma(p, x, 1.0 / 120.0);
    p = __builtin_fma(p, x, 1.0 / 24.0);
    p = __builtin_fma(p, x, 1.0 / 6.0);
    p = __builtin_fma(p, x, 0.5);
    p = __builtin_fma(p, x, 1.0);
    p = __builtin_fma(p, x, 1.0);
    return (uint64_t)__builtin_rint(__builtin_ldexp(p, (int)n + 43));
}

__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v, int lane) {  // inclusive
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint64_t o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}

// Calls f(column, key) for this wave's columns [begin, end) of the row, in
// ascending order per lane; whole 16-byte words where the row holds them.
template <int TYPE, typename F>
__device__ __forceinline__ void each_column(const void* row, int begin, int end, int lane, F&& f) {
    constexpr int kBytes = TYPE == 2 ? 4 : 2, kPer = 16 / kBytes;
    const uint8_t* base = (const uint8_t*)row;
    // first column of the 16-byte word that holds `begin`
    const int head = (int)((((uintptr_t)base + (uintptr_t)begin * kBytes) & 15) / kBytes);
    for (int c0 = begin - head + lane * kPer; c0 < end; c0 += 64 * kPer) {
        uint32_t bits[kPer];
        if (c0 >= begin && c0 + kPer <= end) {
            const uint4 v = *(const uint4*)(base + (int64_t)c0 * kBytes);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                bits[i] = TYPE == 2 ? w[i & 3] : (i & 1 ? w[i / 2 & 3] >> 16 : w[i / 2 & 3] & 0xffffu);
#pragma unroll
            for (int i = 0; i < kPer; ++i) f(c0 + i, key_of<TYPE>(bits[i]));
        } else {
            for (int i = 0; i < kPer; ++i) {
                const int c = c0 + i;
                if (c < begin || c >= end) continue;
                f(c, key_of<TYPE>(TYPE == 2 ? ((const uint32_t*)row)[c] : ((const uint16_t*)row)[c]));
            }
        }
    }
}

struct Shared {
    uint32_t count[2][kBins];   // [0]: the first digit's, kept for every search; [1]: deeper digits'
    unsigned long long mass[2][kBins];
    uint64_t wave_sum[kWaves];
    uint32_t wave_key[kWaves];
    uint32_t wave_flag[kWaves];
    uint64_t totals[2][kWaves];
    // a search's answer: the bin, and the sums above it
    uint32_t digit;
    uint64_t before_count, before_mass;
};

// First bin in descending order whose inclusive sum (counts, or masses) plus
// `before` reaches x; the sums before it, in both measures.  Called by all.
__device__ __forceinline__ void descend(Shared& sh, int set, bool by_mass, uint64_t x, uint64_t before_count,
                                        uint64_t before_mass) {
    constexpr int kPer = kBins / kThreads;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    // thread t owns bins kBins - 1 - t kPer - i
    uint64_t c[kPer], m[kPer], cs = 0, ms = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        c[i] = sh.count[set][kBins - 1 - t * kPer - i];
        m[i] = sh.mass[set][kBins - 1 - t * kPer - i];
        cs += c[i];
        ms += m[i];
    }
    const uint64_t ci = wave_scan_u64(cs, lane), mi = wave_scan_u64(ms, lane);
    if (lane == 63) {
        sh.totals[0][wave] = ci;
        sh.totals[1][wave] = mi;
    }
    __syncthreads();
    uint64_t cb = before_count + ci - cs, mb = before_mass + mi - ms;
    for (int w = 0; w < wave; ++w) {
        cb += sh.totals[0][w];
        mb += sh.totals[1][w];
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const uint64_t lo = by_mass ? mb : cb, add = by_mass ? m[i] : c[i];
        if (lo < x && lo + add >= x) {  // one bin at most
            sh.digit = kBins - 1 - t * kPer - i;
            sh.before_count = cb;
            sh.before_mass = mb;
        }
        cb += c[i];
        mb += m[i];
    }
    __syncthreads();
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void vocab_sample_kernel(VocabSampleArgs a) {
    __shared__ Shared sh;
    const int row = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    if (row >= (a.live_count ? *a.live_count : a.live_rows)) return;
    const uint8_t* logits = (const uint8_t*)a.logits + (int64_t)row * a.row_stride * (TYPE == 2 ? 4 : 2);
    const float temperature = a.temperatures[row], top_p = a.top_ps[row], min_p = a.min_ps[row], u = a.uniforms[row];
    const int64_t top_k = a.top_ks[row];
    const int seg = ((a.width + kWaves - 1) / kWaves + 7) / 8 * 8;
    const int begin = min(a.width, wave * seg), end = min(a.width, begin + seg);

    // the largest finite key, and whether a NaN or +inf is there
    uint32_t top = 0, bad = 0;
    each_column<TYPE>(logits, begin, end, lane, [&](int, uint32_t key) {
        bad |= key >= Limits<TYPE>::kInf || key < Limits<TYPE>::kNegInf;
        top = max(top, key);
    });
    top = wave_max_u32(top);
    bad = __ballot(bad) != 0;
    if (lane == 0) {
        sh.wave_key[wave] = top;
        sh.wave_flag[wave] = bad;
    }
    for (int i = t; i < kBins; i += kThreads) {
        sh.count[0][i] = 0;
        sh.mass[0][i] = 0;
    }
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) {
        top = max(top, sh.wave_key[w]);
        bad |= sh.wave_flag[w];
    }
    const bool valid = !bad && top > Limits<TYPE>::kNegInf && temperature >= 0.f &&
                       __builtin_isfinite(temperature) && top_p > 0.f && top_p <= 1.f && min_p >= 0.f &&
                       min_p <= 1.f && u >= 0.f && u < 1.f;
    if (!valid) {
        if (t == 0) {
            a.tokens[row] = -1;
            a.valid[row] = 0;
            if (a.logprobs) a.logprobs[row] = __builtin_nanf("");
        }
        return;
    }
    uint32_t key = top;
    uint64_t nth = 1;  // the token is the nth column of that key
    double logprob = 0.0;
    if (temperature > 0.f) {
        const double largest = value_of<TYPE>(top), scale = 1.4426950408889634074 / (double)temperature;
        auto power = [&](uint32_t k) { return (value_of<TYPE>(k) - largest) * scale; };
        const double least = min_p > 0.f ? log2((double)min_p) : -__builtin_inf();
        uint64_t likely = 0;
        each_column<TYPE>(logits, begin, end, lane, [&](int, uint32_t k) {
            const double p = power(k);
            const uint64_t w = fixed_weight(p);
            atomicAdd(&sh.count[0][k >> 20], 1u);
            if (w) atomicAdd(&sh.mass[0][k >> 20], (unsigned long long)w);
            if (p >= least) likely += w;
        });
        likely = wave_scan_u64(likely, lane);
        if (lane == 63) sh.wave_sum[wave] = likely;
        __syncthreads();
        uint64_t kept = 0;
        for (int w = 0; w < kWaves; ++w) kept += sh.wave_sum[w];
        uint64_t head = ~0ull;  // mass of what the stages so far keep; all of it at first
        for (int stage = 0; stage < 3; ++stage) {  // top-k, top-p, the token
            uint64_t x;
            if (stage == 0) {
                if (top_k <= 0 || top_k >= a.width) continue;
                x = (uint64_t)top_k;
            } else if (stage == 1) {
                if (top_p >= 1.f) continue;
                if (head == ~0ull) {
                    uint64_t total = 0;
                    for (int i = lane; i < kBins; i += 64) total += sh.mass[0][i];
                    head = __shfl(wave_scan_u64(total, lane), 63, 64);
                }
                x = max((uint64_t)1, min(head, (uint64_t)__builtin_ceil((double)top_p * (double)head)));
            } else {
                kept = min(kept, head);
                x = min(kept, (uint64_t)((double)u * (double)kept) + 1);
            }
            // the key at which the inclusive count or mass reaches x
            descend(sh, 0, stage > 0, x, 0, 0);
            uint32_t prefix = sh.digit;
            int shift = 20;
            while (shift > (TYPE == 2 ? 0 : 16)) {
                const int bits = shift == 20 ? 12 : 8;
                const uint64_t bc = sh.before_count, bm = sh.before_mass;
                for (int i = t; i < kBins; i += kThreads) {
                    sh.count[1][i] = 0;
                    sh.mass[1][i] = 0;
                }
                __syncthreads();
                each_column<TYPE>(logits, begin, end, lane, [&](int, uint32_t k) {
                    if (k >> shift != prefix) return;
                    const uint32_t d = (k >> (shift - bits)) & ((1u << bits) - 1);
                    atomicAdd(&sh.count[1][d], 1u);
                    atomicAdd(&sh.mass[1][d], (unsigned long long)fixed_weight(power(k)));
                });
                __syncthreads();
                descend(sh, 1, stage > 0, x, bc, bm);
                prefix = prefix << bits | sh.digit;
                shift -= bits;
            }
            key = prefix << shift;
            const uint64_t w = fixed_weight(power(key)), above = sh.before_mass;
            if (stage == 0) head = above + (x - sh.before_count) * w;
            else nth = (x - above + w - 1) / w;
            if (stage == 1) head = min(head, above + nth * w);
            __syncthreads();
        }
        logprob = power(key) * 0.69314718055994530942 - log((double)kept / kOne);
    }
    // the nth column of that key, in ascending order
    uint64_t found = 0;
    each_column<TYPE>(logits, begin, end, lane, [&](int, uint32_t k) { found += k == key; });
    found = wave_scan_u64(found, lane);
    __syncthreads();
    if (lane == 63) sh.wave_sum[wave] = found;
    __syncthreads();
    uint64_t before = 0;
    for (int w = 0; w < wave; ++w) before += sh.wave_sum[w];
    if (before < nth && before + sh.wave_sum[wave] >= nth) {
        // this wave holds it: 64 columns at a time
        for (int c0 = begin; c0 < end; c0 += 64) {
            const int c = c0 + lane;
            bool hit = false;
            if (c < end)
                hit = key_of<TYPE>(TYPE == 2 ? ((const uint32_t*)logits)[c] : ((const uint16_t*)logits)[c]) == key;
            const uint64_t mask = __ballot(hit);
            const int here = __builtin_popcountll(mask);
            if (before + here >= nth) {
                const int below = __builtin_popcountll(mask & ((1ull << lane) - 1));
                if (hit && before + below + 1 == nth) {
                    a.tokens[row] = c;
                    a.valid[row] = 1;
                    if (a.logprobs) a.logprobs[row] = (float)logprob;
                }
                break;
            }
            before += here;
        }
    }
}

template <int TYPE>
hipError_t start(const VocabSampleArgs& a, hipStream_t s) {
    vocab_sample_kernel<TYPE><<<a.rows, kThreads, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_vocab_sample(const VocabSampleArgs& a, hipStream_t s) {
    return a.dtype == 2 ? start<2>(a, s) : a.dtype == 1 ? start<1>(a, s) : start<0>(a, s);
}

}  // namespace cubic
