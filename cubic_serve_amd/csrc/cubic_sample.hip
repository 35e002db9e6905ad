// Sampling from the whole vocabulary (gfx950): per row one token under
// temperature T, top-k, top-p and min-p, from a given uniform number u.
//
// Order of a row: logit descending, column ascending on ties (-0 == +0).  Weight
// of a column: w = 2^((l - max) log2(e) / T), in 64-bit fixed point with 2^43 for
// the maximum (so up to 2^20 columns sum below 2^63 and sums do not depend on
// their order; a weight is off by at most half a unit, 2^-44 of the maximum's, and a
// sum over 151936 columns by 2^-26 of it, below the 2^-24 steps of u).
// What top-k, top-p and min-p keep is a prefix of the order each, and a prefix is
// as good as its mass:
//   S_k  mass of the first k
//   S_p  mass through the first position whose inclusive mass reaches top_p S_k
//   S_m  mass of the weights of at least min_p
//   S = min(S_k, S_p, S_m); the token is the first position whose inclusive mass
//   exceeds u S; its log-probability ln(w / S).
// So a row takes at most three searches "first position whose inclusive count or
// mass reaches X", each a descent over the bits of the logits' ordered keys.
#include <algorithm>

#include "cubic_device.h"
#include "cubic_capi_internal.h"

namespace cubic {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
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

// Inclusive scan over the 64 lanes (as wave_scan_u32).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {
    v += dpp_u64<0x111, 0xF>(v);
    v += dpp_u64<0x112, 0xF>(v);
    v += dpp_u64<0x114, 0xF>(v);
    v += dpp_u64<0x118, 0xF>(v);
    v += dpp_u64<0x142, 0xA>(v);
    v += dpp_u64<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int l) {  // wave-uniform l
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
}
// Sums of the waves' values before this wave, and of all; lds: one per wave.
// A barrier lies between the values and the sums, none behind.
__device__ __forceinline__ uint64_t before_wave(uint64_t value, uint64_t* lds, int lane, int wave, uint64_t& all) {
    if (lane == 0) lds[wave] = value;
    __syncthreads();
    const uint64_t upto = wave_scan_u64(lane < kWaves ? lds[lane] : 0);
    all = lane_u64(upto, 63);
    return wave ? lane_u64(upto, wave - 1) : 0;
}

// Columns [c0, c0 + 8) (four of 32 bits) of a row of `width` columns as their
// bits, c0 a multiple of as many; columns past the row read as -inf.  One load at
// any alignment, without a branch before it, so that loads of several words go
// out together: the row's last word is read where it ends and moved into place.
struct __attribute__((packed, aligned(2))) AnyWord { uint32_t w[4]; };
template <int TYPE>
__device__ __forceinline__ uint4 load_word(const uint8_t* row, int c0, int width) {
    constexpr int kBytes = TYPE == 2 ? 4 : 2, kPer = 16 / kBytes;
    if (width < kPer) {  // a row shorter than a word, element by element
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint32_t e = i >= width ? (TYPE == 2 ? 0xff800000u : TYPE == 1 ? 0xfc00u : 0xff80u)
                               : TYPE == 2 ? ((const uint32_t*)row)[i] : ((const uint16_t*)row)[i];
            if constexpr (TYPE == 2) w[i] = e;
            else w[i / 2] |= e << (16 * (i & 1));
        }
        return uint4{w[0], w[1], w[2], w[3]};
    }
    const AnyWord v = *(const AnyWord*)(row + (int64_t)min(c0, width - kPer) * kBytes);
    return uint4{v.w[0], v.w[1], v.w[2], v.w[3]};
}
template <int TYPE>
__device__ __forceinline__ uint4 place_word(uint4 v, int c0, int width) {
    constexpr int kBytes = TYPE == 2 ? 4 : 2, kPer = 16 / kBytes;
    constexpr uint32_t kFill = TYPE == 2 ? 0xff800000u : TYPE == 1 ? 0xfc00fc00u : 0xff80ff80u;
    const int past = width < kPer ? c0 : c0 - (width - kPer);  // columns to move by
    if (past <= 0) return v;
    if (past >= kPer) return uint4{kFill, kFill, kFill, kFill};
    typedef unsigned __int128 u128;
    const u128 fill = ((u128)((uint64_t)kFill << 32 | kFill) << 64) | ((uint64_t)kFill << 32 | kFill);
    const u128 x = ((u128)((uint64_t)v.w << 32 | v.z) << 64) | ((uint64_t)v.y << 32 | v.x);
    const u128 y = x >> (past * kBytes * 8) | fill << (128 - past * kBytes * 8);
    return uint4{(uint32_t)y, (uint32_t)(y >> 32), (uint32_t)(y >> 64), (uint32_t)(y >> 96)};
}
template <int TYPE>
__device__ __forceinline__ uint32_t word_key(const uint4& v, int i) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (TYPE == 2) return key_of<2>(w[i]);
    else return key_of<TYPE>(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu);
}
// Calls f(column, key) for columns [begin, end) of the row, begin a multiple of 8
// (and for -infs past its end), the workgroup's threads taking words in turn,
// several in flight each.
template <int TYPE, typename F>
__device__ __forceinline__ void each_column(const uint8_t* row, int begin, int end, int width, F&& f) {
    constexpr int kEach = TYPE == 2 ? 4 : 8, kAhead = 4;
    for (int c0 = begin + (int)threadIdx.x * kEach; c0 < end; c0 += kAhead * kThreads * kEach) {
        uint4 word[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) word[i] = load_word<TYPE>(row, c0 + i * kThreads * kEach, width);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int c = c0 + i * kThreads * kEach;
            if (c >= end) break;
            const uint4 v = place_word<TYPE>(word[i], c, width);
#pragma unroll
            for (int j = 0; j < kEach; ++j) f(c + j, word_key<TYPE>(v, j));
        }
    }
}

// ---------------------------------------------------------------------------
// The searches, by one workgroup, over items (key, number of columns with it):
// the columns themselves, or the distinct keys of a row's chunks.
// ---------------------------------------------------------------------------
constexpr int kTable = 128;  // 2^(i / 128)
constexpr uint32_t kNoDigit = ~0u;

struct Choice {
    uint32_t key;   // the token is the nth column (from 1) of this key
    uint64_t nth;
    uint64_t kept;  // mass of the kept columns
};

template <int TYPE>
struct Search {
    // bins: the first digit, 11 of a 16-bit key's bits or 12 of 32; then (32 bits)
    // twice 10
    static constexpr int kBins = TYPE == 2 ? 4096 : 2048, kShift = TYPE == 2 ? 20 : 21;
    static constexpr int kPer = kBins / kThreads;  // bins per thread
    static constexpr int kDeepBins = TYPE == 2 ? 1024 : 1;
    // items held in LDS: key's upper half | number; or (32 bits) the columns of
    // one first digit, key and column
    static constexpr int kCached = TYPE == 2 ? 8192 : 28672;
    alignas(16) uint32_t items[TYPE == 2 ? 2 * kCached : kCached];
    uint32_t count[kBins], deep_count[kDeepBins];
    unsigned long long mass[kBins], deep_mass[kDeepBins];
    uint32_t cursor[TYPE == 2 ? kBins : 1];  // where a bin's next column goes (32 bits)
    uint32_t gathered;          // columns of the first digit (32 bits)
    int starts[kMaxSampleChunks + 1], held[kMaxSampleChunks], number[kMaxSampleChunks];
    uint64_t sums[4][kWaves];   // before_wave's
    uint32_t count_sums[kWaves];
    // 32 bits: a search's digit, the sums before it, what it looks for
    uint32_t digit;
    uint64_t before_count, before_mass, want;
    // each search's digit; 16 bits: the counts of that digit's keys
    uint32_t digits[3], keys[3][32], columns;
    uint32_t split[TYPE == 2 ? 1 : 32][kMaxSampleChunks];  // the token's digit's by chunk
    Choice choice;
    float logprob;
};

// A row's parameters, read by one thread (waves that read them by themselves
// could take different ways through the barriers if a caller rewrites them).
struct Row {
    float temperature, top_p, min_p, u;
    int64_t top_k;
    double scale, least;  // of Weights; by the one thread
    __device__ __forceinline__ void read(const VocabSampleArgs& a, int row) {
        temperature = a.temperatures[row];
        top_p = a.top_ps[row];
        min_p = a.min_ps[row];
        u = a.uniforms[row];
        top_k = a.top_ks[row];
    }
    // As words of a chunk's head, for a launch that follows.
    __device__ __forceinline__ void put(uint32_t* head) const {
        head[0] = __float_as_uint(temperature);
        head[1] = __float_as_uint(top_p);
        head[2] = __float_as_uint(min_p);
        head[3] = __float_as_uint(u);
        head[4] = (uint32_t)top_k;
        head[5] = (uint32_t)((uint64_t)top_k >> 32);
    }
    __device__ __forceinline__ void get(const uint32_t* head) {
        temperature = __uint_as_float(head[0]);
        top_p = __uint_as_float(head[1]);
        min_p = __uint_as_float(head[2]);
        u = __uint_as_float(head[3]);
        top_k = (int64_t)((uint64_t)head[5] << 32 | head[4]);
    }
    __device__ __forceinline__ void prepare() {
        scale = 128.0 * 1.4426950408889634074 / (double)temperature;
        least = min_p > 0.f ? 128.0 * log2((double)min_p) : -__builtin_inf();
    }
    __device__ __forceinline__ bool admitted() const {
        return temperature >= 0.f && __builtin_isfinite(temperature) && top_p > 0.f && top_p <= 1.f &&
               min_p >= 0.f && min_p <= 1.f && u >= 0.f && u < 1.f;
    }
};

// Weight of a key in fixed point: with t = 128 log2(e) (l - max) / T and n = rint(t),
// 2^(t / 128) = 2^(n / 128 rounded down) * table[n mod 128] * e^((t - n) ln 2 / 128), the
// last by its Taylor polynomial of degree 4 (off by less than 2e-15), rounded to an
// integer by adding 2^52.
template <int TYPE>
struct Weights {
    double largest, scale, least;
    const double* table;
    __device__ __forceinline__ Weights(const double* lds, uint32_t top, const Row& r)
        : largest(value_of<TYPE>(top)), scale(r.scale), least(r.least), table(lds) {}
    __device__ __forceinline__ double exponent(uint32_t key) const { return (value_of<TYPE>(key) - largest) * scale; }
    __device__ __forceinline__ uint64_t at(double t) const {
        const double n = __builtin_rint(fmax(t, -46.0 * 128.0));
        const int k = (int)n;
        const double x = (t - n) * (0.69314718055994530942 / 128.0);
        const double f = table[k & (kTable - 1)];
        const double p = x * __builtin_fma(x, __builtin_fma(x, __builtin_fma(x, 1.0 / 24.0, 1.0 / 6.0), 0.5), 1.0);
        const double w = __builtin_ldexp(__builtin_fma(f, p, f), (k >> 7) + 43) + 4503599627370496.0;
        return t > -46.0 * 128.0 ? __builtin_bit_cast(uint64_t, w) & 0xfffffffffffffull : 0;
    }
    __device__ __forceinline__ uint64_t of(uint32_t key) const { return at(exponent(key)); }
};

// Sums of this thread's items.
struct Tally {
    uint64_t likely = 0;  // mass of the weights of at least min_p
};

__device__ __forceinline__ void fill_table(double* table) {
    if (threadIdx.x < kTable) table[threadIdx.x] = exp2((double)threadIdx.x / kTable);
}

// Called by the whole workgroup; a barrier has to follow.
template <int TYPE>
__device__ __forceinline__ void clear(Search<TYPE>& sh) {
    const int t = threadIdx.x;
#pragma unroll
    for (int i = 0; i < Search<TYPE>::kPer; ++i) {
        sh.count[t + i * kThreads] = 0;
        sh.mass[t + i * kThreads] = 0;
    }
    if constexpr (TYPE != 2) {
        if (t < 96) (&sh.keys[0][0])[t] = 0;
        for (int i = t; i < 32 * kMaxSampleChunks; i += kThreads) (&sh.split[0][0])[i] = 0;
    }
}
template <int TYPE>
__device__ __forceinline__ void add(Search<TYPE>& sh, const Weights<TYPE>& weights, Tally& tally, uint32_t key,
                                    uint32_t number) {
    const double t = weights.exponent(key);
    const uint64_t w = weights.at(t) * number;
    if (!w) return;
    atomicAdd(&sh.count[key >> Search<TYPE>::kShift], number);
    atomicAdd(&sh.mass[key >> Search<TYPE>::kShift], (unsigned long long)w);
    if (t >= weights.least) tally.likely += w;
}

// The chunk c whose part [starts[c], starts[c + 1]) holds i.
template <int TYPE>
__device__ __forceinline__ int chunk_of(const Search<TYPE>& sh, int chunks, int i) {
    int c = 0;
    for (int step = 1 << (31 - __builtin_clz(chunks)); step; step >>= 1)
        if (c + step < chunks && sh.starts[c + step] <= i) c += step;
    return c;
}

// First of the bins in descending order whose inclusive sum (of counts, or of
// masses) reaches x: its thread calls found(digit, count before, mass before).
// Thread t owns bins BINS - 1 - t PER - i with c, m in them; cb, mb lie before.
template <int PER, typename Found>
__device__ __forceinline__ void pick(const uint32_t (&c)[PER], const uint64_t (&m)[PER], uint64_t cb, uint64_t mb,
                                     bool by_mass, uint64_t x, Found&& found) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const uint64_t lo = by_mass ? mb : cb, add = by_mass ? m[i] : c[i];
        if (lo < x && lo + add >= x) found(PER * kThreads - 1 - threadIdx.x * PER - i, cb, mb);  // one bin at most
        cb += c[i];
        mb += m[i];
    }
}
// The thread's bins, the sums before them and the mass of all.
template <int TYPE, int PER>
__device__ __forceinline__ void bins_before(Search<TYPE>& sh, const uint32_t* count, const unsigned long long* mass,
                                            uint32_t (&c)[PER], uint64_t (&m)[PER], uint64_t& cb, uint64_t& mb,
                                            uint64_t& all) {
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    uint32_t cs = 0;
    uint64_t ms = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        c[i] = count[PER * kThreads - 1 - t * PER - i];
        m[i] = mass[PER * kThreads - 1 - t * PER - i];
        cs += c[i];
        ms += m[i];
    }
    const uint32_t ci = wave_scan_u32(cs);
    const uint64_t mi = wave_scan_u64(ms);
    if (lane == 63) sh.count_sums[wave] = ci;
    mb = before_wave(lane_u64(mi, 63), sh.sums[0], lane, wave, all) + mi - ms;
    const uint32_t upto = wave_scan_u32(lane < kWaves ? sh.count_sums[lane] : 0);
    cb = (wave ? (uint32_t)__builtin_amdgcn_readlane((int)upto, wave - 1) : 0) + ci - cs;
}

// ceil(want / w), a number of columns (at most 2^20): by a reciprocal, off by
// less than a half, which rounding down leaves at most two short.
__device__ __forceinline__ uint64_t columns_to(uint64_t want, uint64_t w) {
    uint64_t n = (uint32_t)((double)want * __builtin_amdgcn_rcp((double)max(w, (uint64_t)1)));
    if (n * w < want) ++n;
    if (n * w < want) ++n;
    return n;
}

// What the searches look for, in turn: x for top-k (a count), top-p and the token
// (masses); head: mass of what they keep so far, kept: of min-p.  False: the
// search leaves nothing out.
__device__ __forceinline__ bool wanted(int stage, const Row& r, int width, uint64_t head, uint64_t& kept, uint64_t& x) {
    if (stage == 0) {
        x = (uint64_t)r.top_k;
        return r.top_k > 0 && r.top_k < width;
    }
    if (stage == 1) {
        x = max((uint64_t)1, min(head, (uint64_t)__builtin_ceil((double)r.top_p * (double)head)));
        return r.top_p < 1.f;
    }
    kept = min(kept, head);
    x = min(kept, (uint64_t)((double)r.u * (double)kept) + 1);
    return true;
}

// The bins' sums become the sums before them, sh.columns all columns; head: all
// mass, kept: that of min-p.  By the whole workgroup, a barrier before and behind.
template <int TYPE>
__device__ __forceinline__ void sums_before(Search<TYPE>& sh, const Tally& tally, const Row& r, uint64_t& head, uint64_t& kept) {
    constexpr int kPer = Search<TYPE>::kPer, kBins = Search<TYPE>::kBins;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    uint32_t c[kPer];
    uint64_t m[kPer], cb, mb;
    bins_before<TYPE, kPer>(sh, sh.count, sh.mass, c, m, cb, mb, head);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        sh.count[kBins - 1 - t * kPer - i] = (uint32_t)cb;
        sh.mass[kBins - 1 - t * kPer - i] = mb;
        cb += c[i];
        mb += m[i];
    }
    if (t == kThreads - 1) sh.columns = (uint32_t)cb;
    kept = head;
    if (r.min_p > 0.f) before_wave(lane_u64(wave_scan_u64(tally.likely), 63), sh.sums[2], lane, wave, kept);
    __syncthreads();
}

// The last bin in descending order before which the sum (of masses, of counts) is
// below x, and the sums before it.  By one wave.
template <int TYPE>
__device__ __forceinline__ int bin_of(const Search<TYPE>& sh, bool by_mass, uint64_t x, uint64_t& count, uint64_t& mass) {
    constexpr int kBins = Search<TYPE>::kBins, kRun = kBins / 64;
    const int lane = threadIdx.x & 63;
    auto before = [&](int d) { return by_mass ? (uint64_t)sh.mass[kBins - 1 - d] : (uint64_t)sh.count[kBins - 1 - d]; };
    const int run = max(__popcll(__ballot(before(lane * kRun) < x)) - 1, 0);
    const int d = run * kRun + max(__popcll(__ballot(lane < kRun && before(run * kRun + min(lane, kRun - 1)) < x)) - 1, 0);
    count = sh.count[kBins - 1 - d];
    mass = sh.mass[kBins - 1 - d];
    return kBins - 1 - d;
}

// The searches of a row of 16-bit logits.  Called by the whole workgroup once
// the items are added, after a barrier; items(f) calls f(key, number, chunk()) for
// this thread's share of them; columns whose weight is 0 may be left out.  What is
// serial is done by one wave: sixteen that do it side by side share four issue
// ports (a search 4700 cycles, 3000 to 4300 so).
template <int TYPE, typename Items>
__device__ __forceinline__ Choice choose_narrow(Search<TYPE>& sh, const Weights<TYPE>& weights, const Tally& tally,
                                                const Row& r, int width, Items&& items) {
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    uint64_t head, kept;
    sums_before(sh, tally, r, head, kept);
    uint32_t key = 0;
    uint64_t nth = 1;
    for (int stage = 0; stage < 3; ++stage) {
        uint64_t x = 0;
        if (!wanted(stage, r, width, head, kept, x)) continue;  // (the same in every wave)
        uint64_t count = 0, mass = 0;
        if (wave == 0) {
            const int d = bin_of(sh, stage > 0, x, count, mass);
            // (fewer than top_k columns may weigh anything)
            if (lane == 0) sh.digits[stage] = stage == 0 && sh.columns < x ? kNoDigit : (uint32_t)d;
        }
        __syncthreads();
        const uint32_t digit = sh.digits[stage];
        if (digit == kNoDigit) continue;
        items([&](uint32_t k, uint32_t number, auto&& chunk) {
            if (k >> 21 != digit) return;
            atomicAdd(&sh.keys[stage][k >> 16 & 31], number);
            if (stage == 2) atomicAdd(&sh.split[k >> 16 & 31][chunk()], number);
        });
        __syncthreads();
        if (wave != 0) continue;
        const uint32_t mine = (digit << 5 | (31 - (lane & 31))) << 16;
        const uint32_t number = lane < 32 ? sh.keys[stage][31 - lane] : 0;
        const uint64_t w = weights.of(mine), all = w * number;
        count += wave_scan_u32(number) - number;
        mass += wave_scan_u64(all) - all;
        const uint64_t lo = stage ? mass : count, more = stage ? all : number;
        const uint64_t hit = __ballot(lo < x && lo + more >= x);
        const int at = hit ? __builtin_ctzll(hit) : 0;
        const uint64_t weight = lane_u64(w, at);
        key = (uint32_t)__builtin_amdgcn_readlane((int)mine, at);
        x -= lane_u64(lo, at);
        nth = stage ? columns_to(x, weight) : x;
        head = min(head, lane_u64(mass, at) + nth * weight);  // (of the token's own search: not used)
    }
    if (t == 0) sh.choice = {key, nth, kept};
    __syncthreads();
    return sh.choice;
}

// The searches of a row of 32-bit logits: gather(digit) leaves the columns of a
// first digit in sh.items (key and column) and their number in sh.gathered (past
// kCached only that), barriers before and behind included; columns(f) calls f(key)
// for this thread's share of them (and of any other columns).
template <typename Gather, typename Columns>
__device__ __forceinline__ Choice choose_wide(Search<2>& sh, const Weights<2>& weights, const Tally& tally,
                                              const Row& r, int width, Gather&& gather, Columns&& columns) {
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    constexpr int kFew = 128;
    uint32_t held = kNoDigit, key = 0;  // held: the digit whose columns are gathered
    uint64_t head, kept, nth = 1;
    sums_before(sh, tally, r, head, kept);
    for (int stage = 0; stage < 3; ++stage) {
        uint64_t x = 0;
        if (!wanted(stage, r, width, head, kept, x)) continue;  // (the same in every wave)
        uint64_t count = 0, mass = 0;
        if (wave == 0) {
            const int d = bin_of(sh, stage > 0, x, count, mass);
            if (lane == 0) {
                // (fewer than top_k columns may weigh anything)
                sh.digits[stage] = stage == 0 && sh.columns < x ? kNoDigit : (uint32_t)d;
                sh.want = x;
                sh.before_count = count;
                sh.before_mass = mass;
            }
        }
        __syncthreads();
        uint32_t prefix = sh.digits[stage];
        if (prefix == kNoDigit) continue;
        if (prefix != held) gather(prefix);
        held = prefix;
        const int gathered = (int)sh.gathered;
        uint64_t weight = 0;
        if (gathered <= kFew) {
            // every column against every other: the sums over larger keys (from 0
            // on) and over equal ones (from kFew on).  31 columns: 2400 cycles, by bins
            // 7100; 119: 6100 and 7700.
            const int lanes = gathered <= 64 ? 64 : kFew, i = t & (lanes - 1);
            const uint32_t mine = i < gathered ? sh.items[2 * i] : 0;
            if (t < 2 * kFew) sh.deep_count[t] = 0, sh.deep_mass[t] = 0;
            if (t >= kThreads - lanes) sh.deep_mass[2 * kFew + i] = i < gathered ? weights.of(mine) : 0;
            __syncthreads();
            uint32_t over = 0, equal = 0;
            uint64_t overs = 0, equals = 0;
            for (int j = t / lanes; j < gathered; j += kThreads / lanes) {
                const uint32_t other = sh.items[2 * j];
                const uint64_t w = sh.deep_mass[2 * kFew + j];
                over += other > mine;
                overs += other > mine ? w : 0;
                equal += other == mine;
                equals += other == mine ? w : 0;
            }
            if (over) atomicAdd(&sh.deep_count[i], over), atomicAdd(&sh.deep_mass[i], (unsigned long long)overs);
            if (equal) atomicAdd(&sh.deep_count[kFew + i], equal), atomicAdd(&sh.deep_mass[kFew + i], (unsigned long long)equals);
            __syncthreads();
            if (wave != 0) continue;
            for (int from = 0; from < gathered; from += 64) {
                const int k = from + lane;
                const uint64_t c = count + sh.deep_count[k], m = mass + sh.deep_mass[k];
                const uint64_t lo = stage ? m : c, more = stage ? sh.deep_mass[kFew + k] : sh.deep_count[kFew + k];
                const uint64_t hit = __ballot(k < gathered && lo < x && lo + more >= x);
                if (!hit && from + 64 < gathered) continue;
                const int at = hit ? __builtin_ctzll(hit) : 0;
                key = sh.items[2 * (from + at)];
                weight = sh.deep_mass[2 * kFew + from + at];
                mass = lane_u64(m, at);
                count = lane_u64(c, at);
                break;
            }
        } else {
            x = sh.want;
            for (int shift = 20; shift > 0; shift -= 10) {
                const uint64_t bc = sh.before_count, bm = sh.before_mass;
                sh.deep_count[t] = 0;
                sh.deep_mass[t] = 0;
                __syncthreads();
                auto deepen = [&](uint32_t k) {
                    if (k >> shift != prefix) return;
                    const uint32_t d = k >> (shift - 10) & 1023u;
                    atomicAdd(&sh.deep_count[d], 1u);
                    atomicAdd(&sh.deep_mass[d], (unsigned long long)weights.of(k));
                };
                if (gathered <= Search<2>::kCached)
                    for (int i = t; i < gathered; i += kThreads) deepen(sh.items[2 * i]);
                else
                    columns(deepen);
                __syncthreads();
                uint32_t dc[1];
                uint64_t dm[1], dcb, dmb, all;
                bins_before<2, 1>(sh, sh.deep_count, sh.deep_mass, dc, dm, dcb, dmb, all);
                pick<1>(dc, dm, bc + dcb, bm + dmb, stage > 0, x, [&](uint32_t digit, uint64_t c, uint64_t m) {
                    sh.digit = digit;
                    sh.before_count = c;
                    sh.before_mass = m;
                });
                __syncthreads();
                prefix = prefix << 10 | (sh.digit & 1023u);
            }
            key = prefix;
            weight = weights.of(prefix);
            count = sh.before_count;
            mass = sh.before_mass;
            __syncthreads();  // (the next search's sums before its bin)
        }
        nth = stage ? columns_to(x - mass, weight) : x - count;
        head = min(head, mass + nth * weight);  // (of the token's own search: not used)
    }
    if (t == 0) sh.choice = {key, nth, kept};
    __syncthreads();
    return sh.choice;
}

__device__ __forceinline__ void refuse(const VocabSampleArgs& a, int row) {
    if (threadIdx.x == 0) {
        a.tokens[row] = -1;
        a.valid[row] = 0;
        if (a.logprobs) a.logprobs[row] = __builtin_nanf("");
    }
}

template <int TYPE>
__device__ __forceinline__ float logprob_of(const Row& r, uint32_t top, const Choice& choice) {
    if (!(r.temperature > 0.f)) return 0.f;
    return (float)((value_of<TYPE>(choice.key) - value_of<TYPE>(top)) / (double)r.temperature -
                   log((double)choice.kept / kOne));
}

// By the thread that holds the token.
__device__ __forceinline__ void publish(const VocabSampleArgs& a, int row, int column, float logprob) {
    a.tokens[row] = column;
    a.valid[row] = 1;
    if (a.logprobs) a.logprobs[row] = logprob;
}

// The bit pattern of a key's logit (+0 for zero).
template <int TYPE>
__device__ __forceinline__ uint32_t pattern_of(uint32_t key) {
    if constexpr (TYPE == 2) return unordered(key);
    else return (key & 0x80000000u ? key & 0x7fff0000u : ~key & 0xffff0000u) >> 16;
}

// Bit j: element j of the word has the pattern (its sign aside where that is 0).
template <int TYPE>
__device__ __forceinline__ uint32_t word_hits(const uint4& v, uint32_t pattern) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t hits = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (TYPE == 2) {
            hits |= (uint32_t)((pattern ? w[j] : w[j] & 0x7fffffffu) == pattern) << j;
        } else {
            const uint32_t x = pattern ? w[j] : w[j] & 0x7fff7fffu;
            hits |= (uint32_t)((x & 0xffffu) == pattern) << (2 * j) | (uint32_t)(x >> 16 == pattern) << (2 * j + 1);
        }
    }
    return hits;
}

// The nth column of the key among [begin, end) is the token: WORDS words per
// thread at a time, each wave a run of them, in order.  There is one, unless the
// caller has rewritten the logits meanwhile: the row is refused then.
template <int TYPE, int WORDS>
__device__ __forceinline__ void locate(Search<TYPE>& sh, const VocabSampleArgs& a, int row, const uint8_t* logits,
                                       int begin, int end, const Row& r, uint32_t top, const Choice& choice) {
    constexpr int kEach = TYPE == 2 ? 4 : 8;  // columns per word
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t pattern = pattern_of<TYPE>(choice.key);
    const bool ragged = end == a.width && a.width % kEach != 0;  // a word reaches past the row
    const uint64_t nth = max(choice.nth, (uint64_t)1);
    uint64_t past = 0;  // columns of the key so far
    for (int c0 = begin; c0 < end; c0 += kThreads * WORDS * kEach) {
        // the words of a pass, evenly over the waves
        const int each = min(WORDS, ((end - c0 + kEach - 1) / kEach + kThreads - 1) / kThreads);
        const int first = c0 + (wave * each * 64 + lane) * kEach;
        uint4 word[WORDS];
#pragma unroll
        for (int i = 0; i < WORDS; ++i)
            if (i < each) word[i] = load_word<TYPE>(logits, first + i * 64 * kEach, a.width);
        if (c0 == begin && t == kThreads - 1) {  // while they come (a barrier follows)
            __builtin_amdgcn_sched_barrier(0);
            sh.logprob = logprob_of<TYPE>(r, top, choice);
        }
        uint32_t hits[WORDS];
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            hits[i] = 0;
            const int c = first + i * 64 * kEach;
            if (i >= each) continue;
            if (ragged) word[i] = place_word<TYPE>(word[i], c, a.width);
            if (c < end) hits[i] = word_hits<TYPE>(word[i], pattern);
            mine += __builtin_popcount(hits[i]);
        }
        const uint32_t here = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan_u32(mine), 63);
        uint64_t all;
        uint64_t from = past + before_wave(here, sh.sums[0], lane, wave, all);
        if (from < nth && from + here >= nth) {  // this wave holds it
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
                if (__ballot(hits[i] != 0) == 0) continue;
                const uint32_t number = __builtin_popcount(hits[i]), sum = wave_scan_u32(number);
                const uint64_t before = from + sum - number;
                if (before < nth && before + number >= nth) {
                    uint32_t left = hits[i];
                    for (uint64_t k = before + 1; k < nth; ++k) left &= left - 1;
                    publish(a, row, first + i * 64 * kEach + __builtin_ctz(left), sh.logprob);
                }
                from += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
            }
        }
        past += all;
        if (past >= nth) return;
        __syncthreads();  // the sums are free again
    }
    refuse(a, row);
}

template <int TYPE>
__device__ __forceinline__ const uint8_t* row_of(const VocabSampleArgs& a, int row) {
    return (const uint8_t*)a.logits + (int64_t)row * a.row_stride * (TYPE == 2 ? 4 : 2);
}

// Whether the row is sampled, read once for the workgroup (as Row is).
__device__ __forceinline__ bool row_lives(const VocabSampleArgs& a, int row, uint32_t* lds) {
    if (!a.live_count) return row < a.live_rows;
    if (threadIdx.x == 0) *lds = row < *a.live_count;
    __syncthreads();
    return *lds != 0;
}

// ---------------------------------------------------------------------------
// 16-bit logits.  A row is cut into chunks, a workgroup each, which reads its
// chunk once and counts every bit pattern in LDS (65536 counters of 16 bits).  What is then worth searching of a row is its
// distinct logits, some thousands for any number of columns: exponentials are
// taken, and keys formed, per distinct logit and not per column.  The row's last
// workgroup to arrive searches.
// ---------------------------------------------------------------------------
// The largest key below which weights beside a largest logit `top` are 0 (below
// 2^-44: more than 30.5 T away; 32 T here, rounded down).
template <int TYPE>
__device__ __forceinline__ uint32_t least_key(uint32_t top, float temperature) {
    const double d = value_of<TYPE>(top) - 32.0 * (double)temperature;
    const float f = __double2float_rd(d);
    if constexpr (TYPE == 2) return max(key_of<2>(__float_as_uint(f)), Limits<2>::kNegInf + 1);
    else if constexpr (TYPE == 1) return key_of<1>(__half_as_ushort(__float2half_rd(f)));
    else return key_of<0>(__float_as_uint(f) >> 16) - (f < 0.f && (__float_as_uint(f) & 0xffffu) ? 0x10000u : 0u);
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void vocab_sample_kernel(VocabSampleArgs a) {
    constexpr int kWords = 8;  // 16-byte words per thread in flight
    constexpr uint32_t kInfBits = TYPE == 1 ? 0x7c00u : 0x7f80u, kNegInfBits = kInfBits | 0x8000u;
    __shared__ union {
        uint32_t counts[32768];  // bit pattern k: half k & 1 of word k / 2
        Search<TYPE> search;
    } sh;
    __shared__ uint32_t wave_top[kWaves], wave_bad[kWaves], wave_lost[kWaves], listed, last;
    __shared__ double table[kTable];
    __shared__ Row r;
    const int row = a.row0 + blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    if (!row_lives(a, row, &last)) {
        // (all of a row's workgroups arrive or none: a count rewritten meanwhile would
        // leave the row's counter between its ends)
        if (a.live_count && arrive_last(a.counters + row, a.chunks, &last) && t == 0) store_device(a.counters + row, 0u);
        return;
    }
    const uint8_t* logits = row_of<TYPE>(a, row);
    uint32_t counted = 0;  // this thread's columns, -inf left out
    {
        const int begin = chunk * a.chunk, end = min(a.width, begin + a.chunk);
        const bool ragged = end == a.width && a.width % 8 != 0;
        Row params;  // (ahead of the words: what waits for it would wait for them)
        params.read(a, row);
        for (int first = begin + t * 8;; first += kWords * kThreads * 8) {
            uint4 word[kWords];
#pragma unroll
            for (int i = 0; i < kWords; ++i) word[i] = load_word<TYPE>(logits, first + i * kThreads * 8, a.width);
            if (first - t * 8 == begin) {
                if (t == 0) {
                    r = params;
                    r.prepare();
                    listed = 0;
                }
                fill_table(table);
#pragma unroll
                for (int i = 0; i < 8; ++i) ((uint4*)sh.counts)[t + i * kThreads] = uint4{0, 0, 0, 0};
                __syncthreads();
            }
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const int c0 = first + i * kThreads * 8;
                if (c0 >= end) break;
                const uint4 v = ragged ? place_word<TYPE>(word[i], c0, a.width) : word[i];
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t lo = w[j] & 0xffffu, hi = w[j] >> 16;
                    // -inf weighs nothing, and a mask makes it most of a row
                    if (lo != kNegInfBits) atomicAdd(&sh.counts[lo >> 1], 1u << (lo << 4 & 16)), ++counted;
                    if (hi != kNegInfBits) atomicAdd(&sh.counts[hi >> 1], 1u << (hi << 4 & 16)), ++counted;
                }
            }
            if (first - t * 8 + kWords * kThreads * 8 >= end) break;
        }
    }
    __syncthreads();
    // this thread's patterns that occur: bit 8 i + 2 j + b stands for pattern
    // 2 (4 (t + 1024 i) + j) + b, so that bits ascend with patterns; the lower
    // half of the bits are positive numbers, the upper half negative ones
    uint64_t there = 0;
    uint32_t found = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint4 v = ((const uint4*)sh.counts)[t + i * kThreads];
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if (__ballot((v.x | v.y | v.z | v.w) != 0) == 0) continue;
        uint32_t bits = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            bits |= (uint32_t)((w[j] & 0xffffu) != 0) << (2 * j) | (uint32_t)(w[j] > 0xffffu) << (2 * j + 1);
        there |= (uint64_t)bits << (8 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) found += (w[j] & 0xffffu) + (w[j] >> 16);
    }
    auto pattern = [&](int bit) { return (uint32_t)(8 * (t + (bit >> 3) * kThreads) + (bit & 7)); };
    const uint32_t plus = (uint32_t)there, minus = (uint32_t)(there >> 32);
    uint32_t top = 0, bad = 0;
    if (plus) {
        const uint32_t p = pattern(31 - __builtin_clz(plus));
        bad = p >= kInfBits;
        top = key_of<TYPE>(p);
    } else if (minus) {
        top = key_of<TYPE>(pattern(32 + __builtin_ctz(minus)));
    }
    if (minus) bad |= pattern(63 - __builtin_clz(minus)) > kNegInfBits;
    // a counter that overflows (more than 65535 columns of one logit, in a chunk
    // that long) takes 65535 or 65536 off the counters' sum
    top = wave_max_u32(top);
    bad = __ballot(bad) != 0;
    const uint32_t lost = wave_scan_u32(counted - found);
    if (lane == 63) {
        wave_top[wave] = top;
        wave_bad[wave] = bad;
        wave_lost[wave] = lost;
    }
    __syncthreads();
    top = wave_max_u32(lane < kWaves ? wave_top[lane] : 0);
    bad = __ballot(lane < kWaves && wave_bad[lane]) != 0;
    const bool overflow = __builtin_amdgcn_readlane((int)wave_scan_u32(lane < kWaves ? wave_lost[lane] : 0), 63) != 0;
    if (overflow) {
        // the counters tell neither the largest nor whether there is a NaN: a lower
        // half has carried into its neighbour's, an upper one lost 65536
        const int begin = chunk * a.chunk, end = min(a.width, begin + a.chunk);
        top = 0;
        bad = 0;
        each_column<TYPE>(logits, begin, end, a.width, [&](int, uint32_t key) {
            bad |= key >= Limits<TYPE>::kInf || key < Limits<TYPE>::kNegInf;
            top = max(top, key);
        });
        top = wave_max_u32(top);
        bad = __ballot(bad) != 0;
        __syncthreads();  // (the waves' first values are read)
        if (lane == 63) {
            wave_top[wave] = top;
            wave_bad[wave] = bad;
        }
        __syncthreads();
        top = wave_max_u32(lane < kWaves ? wave_top[lane] : 0);
        bad = __ballot(lane < kWaves && wave_bad[lane]) != 0;
    }
    // list those that can weigh anything beside the chunk's largest (at
    // temperature 0 the largest itself): patterns from `low` on among the
    // positive, up to `high` among the negative ones
    const uint32_t least = r.temperature > 0.f ? least_key<TYPE>(top, r.temperature) : top;
    const bool signs = least < 0x80000000u;  // negative ones too
    const int low = signs ? 0 : (int)pattern_of<TYPE>(least);
    const int high = signs ? (int)pattern_of<TYPE>(least) : low == 0 ? 0x8000 : 0;  // (-0)
    uint32_t* const lists = a.lists + (int64_t)row * a.chunks * a.list_words;
    uint32_t* const heads = a.heads + (int64_t)row * a.chunks * kSampleHead;
    const __amdgpu_buffer_rsrc_t shared = device_rsrc(lists);
    // how many of this thread's patterns of one sign lie below p
    auto below = [&](int p) {
        const int x = max(p - 8 * t, 0);
        return min(8 * (x >> 13) + min(x & 8191, 8), 32);
    };
    const uint64_t keep_plus = 0xffffffffull << below(low) & 0xffffffffull;
    const uint64_t keep_minus = (1ull << below(high + 1 - 0x8000)) - 1;
    there &= keep_minus << 32 | keep_plus;
    const uint32_t mine = (uint32_t)__builtin_popcountll(there);
    const uint32_t wave_mine = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan_u32(mine), 63);
    int base = 0;
    if (lane == 0 && wave_mine) base = (int)atomicAdd(&listed, wave_mine);
    base = __builtin_amdgcn_readfirstlane(base);
    uint32_t* const list = lists + (int64_t)chunk * a.list_words;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t bits = (uint32_t)(there >> (8 * i)) & 0xffu;
        if (__ballot(bits) == 0) continue;
        const uint4 v = ((const uint4*)sh.counts)[t + i * kThreads];
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool in = bits >> j & 1;
            const uint64_t who = __ballot(in);
            const int at = base + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
            if (in && at < a.list_words)
                store_device(list + at, key_of<TYPE>((uint32_t)(8 * (t + i * kThreads) + j)) |
                                            (j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu));
            base += __builtin_popcountll(who);
        }
    }
    __syncthreads();
    if (t == 0) {
        store_device(heads + chunk * kSampleHead, overflow ? ~0u : listed);  // (~0: no list holds it)
        store_device(heads + chunk * kSampleHead + 1, top);
        store_device(heads + chunk * kSampleHead + 2, bad);
    }
    if (!arrive_last(a.counters + row, a.chunks, &last)) return;
    // this workgroup searches the row (the counters' place is free)
    Search<TYPE>& s = sh.search;
    if (t == 0) store_device(a.counters + row, 0u);
    clear<TYPE>(s);
    if (wave == 0) {
        uint32_t number = 0, key = 0, flag = 0;
        if (lane < a.chunks) {
            number = load_device(heads + lane * kSampleHead);
            key = load_device(heads + lane * kSampleHead + 1);
            flag = load_device(heads + lane * kSampleHead + 2);
        }
        // (lists begin at multiples of four items)
        const uint32_t words = min(number, (uint32_t)a.list_words), sum = wave_scan_u32((words + 3) & ~3u);
        if (lane < a.chunks) {
            s.starts[lane + 1] = (int)sum;
            s.number[lane] = (int)words;
        }
        if (lane == 0) s.starts[0] = 0;
        key = wave_max_u32(key);
        const uint32_t over = __ballot(number > (uint32_t)a.list_words) != 0 ? 2u : 0u;
        flag = __ballot(flag != 0) != 0 ? 1u : 0u;
        if (lane == 0) {
            wave_top[0] = key;
            wave_bad[0] = flag | over;
        }
    }
    __syncthreads();
    top = wave_top[0];
    const bool whole = !(wave_bad[0] & 2);  // no list overflowed
    if ((wave_bad[0] & 1) || top <= Limits<TYPE>::kNegInf || !r.admitted()) {
        refuse(a, row);
        return;
    }
    const int items = s.starts[a.chunks];
    constexpr int kCached = Search<TYPE>::kCached;
    // f(i, v): the items from i on, four at a time (0: there is none), for the
    // fours from number `from` on; a load of four words each, four in flight
    auto each_listed = [&](int from, auto&& f) {
        constexpr int kAhead = 4;
        for (int q0 = from / 4 + t; 4 * q0 < items; q0 += kAhead * kThreads) {
            uint4 v[kAhead];
            int rest[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int i = 4 * (q0 + j * kThreads), c = chunk_of<TYPE>(s, a.chunks, i), k = i - s.starts[c];
                rest[j] = i < items ? s.number[c] - k : 0;
                // (past the end: an offset that reads nothing)
                v[j] = __builtin_bit_cast(uint4, load_device4(shared, rest[j] > 0 ? (c * a.list_words + k) * 4 : -16));
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (rest[j] <= 0) continue;
                if (rest[j] < 4) v[j].w = 0;
                if (rest[j] < 3) v[j].z = 0;
                if (rest[j] < 2) v[j].y = 0;
                f(4 * (q0 + j * kThreads), v[j]);
            }
        }
    };
    // f(i, v): item i of all (v = 0: none); the first kCached lie in LDS, four to a read
    auto each_item = [&](auto&& f) {
        auto four = [&](int i, const uint4& v) { f(i, v.x), f(i + 1, v.y), f(i + 2, v.z), f(i + 3, v.w); };
        for (int i = 4 * t; i < min(items, kCached); i += 4 * kThreads) four(i, *(const uint4*)&s.items[i]);
        if (items > kCached) each_listed(kCached, four);
    };
    Choice choice = {top, 1, 0};
    if (r.temperature > 0.f) {
        const Weights<TYPE> weights(table, top, r);
        Tally tally;
        if (whole) {
            each_listed(0, [&](int i, const uint4& v) {
                if (i < kCached) *(uint4*)&s.items[i] = v;
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (w[k]) add<TYPE>(s, weights, tally, w[k] & 0xffff0000u, w[k] & 0xffffu);
            });
        } else {
            each_column<TYPE>(logits, 0, a.width, a.width, [&](int, uint32_t key) { add<TYPE>(s, weights, tally, key, 1u); });
        }
        __syncthreads();
        choice = choose_narrow<TYPE>(s, weights, tally, r, a.width, [&](auto&& f) {
            if (whole) each_item([&](int i, uint32_t v) { f(v & 0xffff0000u, v & 0xffffu, [&] { return chunk_of<TYPE>(s, a.chunks, i); }); });
            else each_column<TYPE>(logits, 0, a.width, a.width, [&](int c, uint32_t key) { f(key, 1u, [&] { return min(c / a.chunk, a.chunks - 1); }); });
        });
    } else if (whole) {
        // one item per chunk: its largest (two for +0 and -0)
        each_listed(0, [&](int i, const uint4& v) {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if ((w[k] & 0xffff0000u) == top) atomicAdd(&s.split[top >> 16 & 31][chunk_of<TYPE>(s, a.chunks, i)], w[k] & 0xffffu);
        });
        __syncthreads();
    }
    // the chunk that holds the nth column of the key
    int b = 0, e = a.width;
    if (a.chunks > 1 && (whole || r.temperature > 0.f)) {
        const uint32_t number = lane < a.chunks ? s.split[choice.key >> 16 & 31][lane] : 0, upto = wave_scan_u32(number);
        const uint64_t hit = __ballot(upto >= choice.nth);
        const int c = hit ? __builtin_ctzll(hit) : a.chunks - 1;
        choice.nth -= (uint32_t)__builtin_amdgcn_readlane((int)(upto - number), c);
        b = c * a.chunk;
        e = min(a.width, b + a.chunk);
    }
    locate<TYPE, kWords>(s, a, row, logits, b, e, r, top, choice);
}

// ---------------------------------------------------------------------------
// 32-bit logits: nearly every column a logit of its own.  A first launch takes
// the chunks' largest, so that the second can weigh its columns against the
// row's: each chunk's masses by the keys' first 12 bits, joined by the row's last
// workgroup to arrive, which gathers the columns of the bin in which a search
// ends and finishes the search among those.  Where a row has several chunks (of at
// most 32768 columns then), each leaves its columns' numbers in order of bins, so that
// a bin is a run of each chunk's: 128001 columns, 48 rows, three searches, 78 -> 50 us
// against scans of the row by the one workgroup (17 us each, what one CU reads).
// With a chunk per row there is nothing to share out, and the scans stay.
// The first launch also reads a row's settings and whether it lives, into the first
// chunk's head: the second one's workgroups, which meet at the row's counter, all
// go by that, whatever a caller rewrites meanwhile.
// ---------------------------------------------------------------------------
constexpr int kHeadLives = 8, kHeadRow = 9;  // words of the first chunk's head
__global__ __launch_bounds__(kThreads) void vocab_top_f32_kernel(VocabSampleArgs a) {
    __shared__ uint32_t wave_top[kWaves], wave_bad[kWaves], live;
    const int row = a.row0 + blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    uint32_t* const head = a.heads + ((int64_t)row * a.chunks + chunk) * kSampleHead;
    const bool lives = row_lives(a, row, &live);
    if (chunk == 0 && t == 0) {
        head[kHeadLives] = lives;
        Row r;
        r.read(a, row);
        r.put(head + kHeadRow);
    }
    if (!lives) {
        if (t == 0) head[1] = 1;  // (where only some of its workgroups saw it live)
        return;
    }
    const int begin = chunk * a.chunk, end = min(a.width, begin + a.chunk);
    uint32_t top = 0, bad = 0;
    each_column<2>(row_of<2>(a, row), begin, end, a.width, [&](int, uint32_t key) {
        bad |= key >= Limits<2>::kInf || key < Limits<2>::kNegInf;
        top = max(top, key);
    });
    top = wave_max_u32(top);
    bad = __ballot(bad) != 0;
    if (lane == 0) {
        wave_top[wave] = top;
        wave_bad[wave] = bad;
    }
    __syncthreads();
    if (t >= 64) return;
    top = wave_max_u32(lane < kWaves ? wave_top[lane] : 0);
    bad = __ballot(lane < kWaves && wave_bad[lane]) != 0;
    if (t == 0) {
        head[0] = top;
        head[1] = bad;
    }
}

// The columns whose keys begin with the digit, into s.items.  The logits' own
// first bits are compared, a word's four at a time: forming every column's key
// cost the scan a sixth more (it is bound by what one CU reads).
__device__ __forceinline__ void gather(Search<2>& s, const uint8_t* logits, int width, uint32_t digit) {
    constexpr int kShift = Search<2>::kShift, kAhead = 4;
    const uint32_t first = digit >> 11 ? digit ^ 0x800u : ~digit & 0xfffu;
    for (int c0 = (int)threadIdx.x * 4; c0 < width; c0 += kAhead * kThreads * 4) {
        uint4 word[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) word[i] = load_word<2>(logits, c0 + i * kThreads * 4, width);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int c = c0 + i * kThreads * 4;
            if (c >= width) break;
            const uint4 v = place_word<2>(word[i], c, width);
            bool any = v.x >> kShift == first || v.y >> kShift == first || v.z >> kShift == first || v.w >> kShift == first;
            // -0 begins as the negative numbers do and has +0's key
            if (first == 0) any |= v.x == 0x80000000u || v.y == 0x80000000u || v.z == 0x80000000u || v.w == 0x80000000u;
            if (!any) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t key = word_key<2>(v, j);
                if (key >> kShift != digit) continue;
                const uint32_t at = atomicAdd(&s.gathered, 1u);
                if (at >= Search<2>::kCached) continue;
                s.items[2 * at] = key;
                s.items[2 * at + 1] = (uint32_t)(c + j);
            }
        }
    }
}

__global__ __launch_bounds__(kThreads) void vocab_sample_f32_kernel(VocabSampleArgs a) {
    __shared__ Search<2> s;
    __shared__ uint32_t row_top, row_bad, listed, last;
    __shared__ double table[kTable];
    __shared__ Row r;
    constexpr int kPer = Search<2>::kPer;
    const int row = a.row0 + blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint8_t* logits = row_of<2>(a, row);
    uint32_t* const heads = a.heads + (int64_t)row * a.chunks * kSampleHead;
    if (!heads[kHeadLives]) return;
    if (wave == 0) {
        if (t == 0) {
            r.get(heads + kHeadRow);
            r.prepare();
            listed = 0;
        }
        const uint32_t key = lane < a.chunks ? heads[lane * kSampleHead] : 0;
        const uint32_t bad = lane < a.chunks ? heads[lane * kSampleHead + 1] : 0;
        const uint32_t top = wave_max_u32(key);
        const bool any = __ballot(bad != 0) != 0;
        if (t == 0) {
            row_top = top;
            row_bad = any;
        }
    }
    clear<2>(s);
    fill_table(table);
    __syncthreads();
    const uint32_t top = row_top;
    if (row_bad || top <= Limits<2>::kNegInf || !r.admitted()) {
        if (chunk == 0) refuse(a, row);
        return;
    }
    Choice choice = {top, 1, 0};
    if (!(r.temperature > 0.f)) {
        if (chunk == 0) locate<2, 4>(s, a, row, logits, 0, a.width, r, top, choice);
        return;
    }
    const Weights<2> weights(table, top, r);
    Tally tally;
    const int begin = chunk * a.chunk, end = min(a.width, begin + a.chunk);
    const uint32_t least = least_key<2>(top, r.temperature);
    each_column<2>(logits, begin, end, a.width, [&](int, uint32_t key) {
        if (key < least) return;
        const double e = weights.exponent(key);
        const uint64_t w = weights.at(e);
        atomicAdd(&s.count[key >> Search<2>::kShift], 1u);
        atomicAdd(&s.mass[key >> Search<2>::kShift], (unsigned long long)w);
        if (e >= weights.least) tally.likely += w;
    });
    __syncthreads();
    uint32_t* const lists = a.lists + (int64_t)row * a.chunks * a.list_words;
    const __amdgpu_buffer_rsrc_t shared = device_rsrc(lists);
    const int runs = 4 * min(a.chunk, kSampleBins), columns = runs + kSampleBins / 2;  // words into a chunk's list
    if (a.chunks > 1) {
        // the chunk's bins that hold anything: bin, columns, mass
        const int list = chunk * a.list_words;
        uint64_t likely;
        before_wave(lane_u64(wave_scan_u64(tally.likely), 63), s.sums[2], lane, wave, likely);
        uint32_t number[kPer], before = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int b = t * kPer + i;
            number[i] = s.count[b];
            before += number[i];
            if (!number[i]) continue;
            const uint64_t m = s.mass[b];
            const uint32_t at = atomicAdd(&listed, 1u) * 4;
            store_device4(shared, (list + (int)at) * 4, __builtin_bit_cast(floatx4_dev_t, uint4{(uint32_t)b, number[i], (uint32_t)m, (uint32_t)(m >> 32)}));
        }
        // where each bin's columns begin, and the columns, in order of bins
        const uint32_t scan = wave_scan_u32(before);
        if (lane == 63) s.count_sums[wave] = scan;
        __syncthreads();
        const uint32_t upto = wave_scan_u32(lane < kWaves ? s.count_sums[lane] : 0);
        before = (wave ? (uint32_t)__builtin_amdgcn_readlane((int)upto, wave - 1) : 0) + scan - before;
        const int held = __builtin_amdgcn_readlane((int)upto, kWaves - 1);
        uint64_t begins = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            s.cursor[t * kPer + i] = before;
            begins |= (uint64_t)before << (16 * i);
            before += number[i];
        }
        store_device((uint64_t*)(lists + list + runs) + t, begins);
        __syncthreads();
        uint16_t* const order = (uint16_t*)s.items;
        each_column<2>(logits, begin, end, a.width, [&](int c, uint32_t key) {
            if (key < least) return;
            // (within the list also if the caller rewrites the logits meanwhile)
            const uint32_t at = atomicAdd(&s.cursor[key >> Search<2>::kShift], 1u);
            if (at < (uint32_t)held) order[at] = (uint16_t)(c - begin);
        });
        __syncthreads();
        for (int i = t; i < (held + 7) / 8; i += kThreads)
            store_device4(shared, (list + columns) * 4 + 16 * i, ((const floatx4_dev_t*)order)[i]);
        __syncthreads();
        if (t == 0) {
            store_device(heads + chunk * kSampleHead + 2, listed);
            store_device(heads + chunk * kSampleHead + 3, (uint32_t)likely);
            store_device(heads + chunk * kSampleHead + 4, (uint32_t)(likely >> 32));
        }
        if (!arrive_last(a.counters + row, a.chunks, &last)) return;
        if (t == 0) store_device(a.counters + row, 0u);
        // this workgroup searches the row: the others' bins on top of its own
        tally.likely = 0;
        if (wave == 0) {
            uint32_t items = 0;
            if (lane < a.chunks) {
                const uint32_t* h = heads + lane * kSampleHead;
                items = lane == chunk ? 0 : load_device(h + 2);
                tally.likely = (uint64_t)load_device(h + 4) << 32 | load_device(h + 3);
            }
            const uint32_t scan = wave_scan_u32(items);
            s.starts[lane + 1] = (int)scan;
            if (lane == 0) s.starts[0] = 0;
        }
        __syncthreads();
        constexpr int kAhead = 4;
        const int all = s.starts[kMaxSampleChunks];
        for (int i0 = t; i0 < all; i0 += kAhead * kThreads) {
            uint4 v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int at = i0 + i * kThreads, c = chunk_of<2>(s, a.chunks, at);
                v[i] = __builtin_bit_cast(uint4, load_device4(shared, at < all ? (c * a.list_words + 4 * (at - s.starts[c])) * 4 : -16));
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (i0 + i * kThreads >= all) break;
                atomicAdd(&s.count[v[i].x], v[i].y);
                atomicAdd(&s.mass[v[i].x], (unsigned long long)((uint64_t)v[i].w << 32 | v[i].z));
            }
        }
        __syncthreads();
    }
    // f(key, column) for this thread's share of the runs that s.starts and s.held tell
    auto each_run = [&](int number, auto&& f) {
        constexpr int kAhead = 4;
        for (int i0 = t; i0 < number; i0 += kAhead * kThreads) {
            int c[kAhead];
            uint32_t bits[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int at = min(i0 + i * kThreads, number - 1);
                const int h = chunk_of<2>(s, a.chunks, at);
                const uint16_t* from = (const uint16_t*)(lists + (int64_t)h * a.list_words + columns);
                c[i] = min(h * a.chunk + (int)load_device(from + s.held[h] + at - s.starts[h]), a.width - 1);
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) bits[i] = ((const uint32_t*)logits)[c[i]];
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (i0 + i * kThreads < number) f(i0 + i * kThreads, key_of<2>(bits[i]), c[i]);
        }
    };
    choice = choose_wide(s, weights, tally, r, a.width, [&](uint32_t digit) {
        __syncthreads();
        if (a.chunks == 1) {
            if (t == 0) s.gathered = 0;
            __syncthreads();
            gather(s, logits, a.width, digit);
            __syncthreads();
            return;
        }
        if (wave == 0) {
            uint32_t number = 0;
            if (lane < a.chunks) {
                // (no finite number's digit is the last; within the list also if the
                // caller rewrites the logits meanwhile)
                const uint16_t* from = (const uint16_t*)(lists + (int64_t)lane * a.list_words + runs) + digit;
                const uint32_t run = min((uint32_t)load_device(from), (uint32_t)a.chunk);
                const uint32_t next = digit + 1 < kSampleBins ? min((uint32_t)load_device(from + 1), (uint32_t)a.chunk) : run;
                number = next > run ? next - run : 0;
                s.held[lane] = (int)run;
            }
            const uint32_t scan = wave_scan_u32(number);
            s.starts[lane + 1] = (int)scan;
            if (lane == 0) s.starts[0] = 0;
            if (lane == 63) s.gathered = scan;
        }
        __syncthreads();
        if (s.gathered <= Search<2>::kCached)
            each_run((int)s.gathered, [&](int i, uint32_t key, int c) {
                s.items[2 * i] = key;
                s.items[2 * i + 1] = (uint32_t)c;
            });
        __syncthreads();
    }, [&](auto&& f) {
        if (a.chunks > 1) each_run((int)s.gathered, [&](int, uint32_t key, int) { f(key); });
        else each_column<2>(logits, 0, a.width, a.width, [&](int, uint32_t key) { f(key); });
    });
    // the last search's columns are gathered: where few have the key, the token
    // is that of them which as many precede as it takes
    const int gathered = (int)s.gathered;
    if (t == 0) listed = 0;
    __syncthreads();
    if (gathered <= Search<2>::kCached) {
        if (t == kThreads - 1) s.logprob = logprob_of<2>(r, top, choice);
        constexpr uint32_t kFew = 256;
        for (int i = t; i < gathered; i += kThreads)
            if (s.items[2 * i] == choice.key) {
                const uint32_t at = atomicAdd(&listed, 1u);
                if (at < kFew) s.deep_count[at] = s.items[2 * i + 1];
            }
        __syncthreads();
        if (listed <= kFew) {
            if (t < (int)listed) {
                const uint32_t mine = s.deep_count[t];
                uint32_t before = 0;
                for (uint32_t i = 0; i < listed; ++i) before += s.deep_count[i] < mine;
                if (before + 1 == choice.nth) publish(a, row, (int)mine, s.logprob);
            }
            if (choice.nth < 1 || choice.nth > listed) refuse(a, row);  // (as in locate)
            return;
        }
    }
    locate<2, 4>(s, a, row, logits, 0, a.width, r, top, choice);
}

}  // namespace

// In runs of rows whose workgroups fit a grid (fewer than 2^32 threads).
hipError_t launch_vocab_sample(const VocabSampleArgs& args, hipStream_t s) {
    VocabSampleArgs a = args;
    const int most = (int)(((1ull << 32) / kThreads - 1) / a.chunks);
    for (; a.row0 < a.rows; a.row0 += most) {
        const int grid = std::min(a.rows - a.row0, most) * a.chunks;
        if (a.dtype == 2) {
            vocab_top_f32_kernel<<<grid, kThreads, 0, s>>>(a);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
            vocab_sample_f32_kernel<<<grid, kThreads, 0, s>>>(a);
        } else if (a.dtype == 1) {
            vocab_sample_kernel<1><<<grid, kThreads, 0, s>>>(a);
        } else {
            vocab_sample_kernel<0><<<grid, kThreads, 0, s>>>(a);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace cubic
