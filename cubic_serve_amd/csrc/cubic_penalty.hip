// Penalties for repeated tokens, biases and grammar masks on logits, and the
// history of tokens that they read.
//
// Of a request, with c the number of times token t is among its outputs (a row of a
// verify step counts the drafts before its depth too):
//   l = l > 0 ? l / repetition : l * repetition     where t is in the prompt or c > 0
//   l = l - frequency * c - (c > 0 ? presence : 0)
//   l = l + bias[t];   -infinity where the grammar's bit is 0
// in 32 bits, in this order, each step rounded (an unfused plain form has the same
// bits), and once to the output's type.
//
// A history keeps per slot a table of each token's mark (outputs counted, in the
// prompt, listed) and bias, and for every kHistoryBucket tokens of the vocabulary a list
// of those that have either.  A list's order is that of atomics; nothing depends on
// it, since each listed token is taken by itself.
//
// What bounds the penalties: reading and writing the logits.  Listed tokens are a few
// thousand of 10^5 columns, so each is looked up by itself, by the workgroup that has
// its column: it reads the lists of its own columns only, and changes their logits in
// LDS on their way.  256 rows of 151936 (64 sequences), 3700 tokens listed for each: 38 us (37
// under a grammar, which admits 2 % of them), where a copy takes 31 and a history of no tokens 26.  In
// place 34, and 69 under a grammar that admits half: whole vectors are written where nothing of
// them is admitted, the masked columns one by one in the others.
// What else was built, when this took 44 (its outputs went through the caches): listed tokens
// changed in memory after the rest 69, one list per slot, which every workgroup of a row
// has to search, 95, four rows of a sequence one after the other in a workgroup, for their common
// list, 81 (too few loads on their way).
#include <type_traits>

#include "cubic_capi_internal.h"
#include "cubic_device.h"

namespace cubic {
namespace {

constexpr uint32_t kListed = 1u << 30, kPrompt = 1u << 31, kCount = kListed - 1;
constexpr int kThreads = 256;

// Puts a token on its bucket's list unless it is there.
__device__ __forceinline__ void list_token(const HistoryArgs& h, int64_t slot, int t, uint32_t mark) {
    if (mark & kListed) return;
    if (atomicOr(&h.state[slot * h.vocab + t].x, kListed) & kListed) return;
    const int bucket = t / kHistoryBucket;
    const int at = atomicAdd(&h.sizes[slot * history_buckets(h.vocab) + bucket], 1);
    h.listed[slot * h.vocab + bucket * kHistoryBucket + at] = t;
}

__global__ __launch_bounds__(kThreads) void history_append_kernel(HistoryArgs h, HistoryTokens a) {
    const int live = a.live_count ? min(max(*a.live_count, 0), a.live_rows) : a.live_rows;
    const int64_t all = (int64_t)live * a.length;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < all; i += (int64_t)gridDim.x * kThreads) {
        const int64_t row = i / a.length, at = row * a.ld + (i - row * a.length);
        const int64_t t = a.token_bytes == 8 ? static_cast<const int64_t*>(a.tokens)[at] : static_cast<const int32_t*>(a.tokens)[at];
        const int slot = a.row_slots[row];
        if (slot < 0 || slot >= h.slots || t < 0 || t >= h.vocab) continue;
        uint32_t* mark = &h.state[(int64_t)slot * h.vocab + t].x;
        const uint32_t old = a.prompt ? atomicOr(mark, kPrompt) : atomicAdd(mark, 1u);
        list_token(h, slot, (int)t, old);
    }
}

// One workgroup per row, a wave per bucket: the tables' listed places back to zero
// (biases_only: those of the biases), then the list.
__global__ __launch_bounds__(1024) void history_clear_kernel(HistoryArgs h, const int32_t* row_slots, int rows, int only_slot,
                                                             int biases_only) {
    const int lane = threadIdx.x & 63, buckets = history_buckets(h.vocab);
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        const int slot = row_slots ? row_slots[row] : only_slot;
        if (slot < 0 || slot >= h.slots) continue;
        const int64_t base = (int64_t)slot * h.vocab;
        for (int b = threadIdx.x >> 6; b < buckets; b += 16) {
            int32_t* size = &h.sizes[(int64_t)slot * buckets + b];
            const int n = min(*size, min(kHistoryBucket, h.vocab - b * kHistoryBucket));
            for (int i = lane; i < n; i += 64) {
                const int t = h.listed[base + b * kHistoryBucket + i];
                h.state[base + t].y = 0;
                if (!biases_only) h.state[base + t].x = 0;
            }
            if (!biases_only && lane == 0 && n) *size = 0;
        }
    }
}

__global__ __launch_bounds__(kThreads) void history_bias_kernel(HistoryArgs h, int slot, const int32_t* ids, const float* values, int n) {
    const int i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= n) return;
    const int t = ids[i];
    if (t < 0 || t >= h.vocab) return;
    h.state[(int64_t)slot * h.vocab + t].y = __float_as_uint(values[i]);
    list_token(h, slot, t, 0);
}

// ---------------------------------------------------------------------------
template <int TYPE>
__device__ __forceinline__ float value_of(const void* p, int64_t i) {
    if constexpr (TYPE == 2) return static_cast<const float*>(p)[i];
    const uint32_t b = static_cast<const uint16_t*>(p)[i];
    return TYPE == 1 ? half_bits_to_float(b) : bf16_bits_to_float(b);
}
template <int TYPE>
__device__ __forceinline__ void set_value(void* p, int64_t i, float v) {
    if constexpr (TYPE == 2) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = (uint16_t)(TYPE == 1 ? float_to_f16_bits(v) : float_to_bf16_bits(v));
}

struct Settings {
    float repetition, presence, frequency;
    bool valid;
};
__device__ __forceinline__ Settings settings_of(const PenaltyArgs& a, int sequence) {
    Settings s;
    s.repetition = a.repetition ? a.repetition[sequence] : 1.0f;
    s.presence = a.presence ? a.presence[sequence] : 0.0f;
    s.frequency = a.frequency ? a.frequency[sequence] : 0.0f;
    const float inf = __builtin_huge_valf();
    s.valid = s.repetition > 0.0f && s.repetition < inf && fabsf(s.presence) < inf && fabsf(s.frequency) < inf;
    return s;
}

__device__ __forceinline__ float penalised(float l, uint32_t mark, int ahead, float bias, const Settings& s) {
    const uint32_t count = (mark & kCount) + (uint32_t)ahead;
    if ((mark & kPrompt) || count) l = l > 0.0f ? l / s.repetition : l * s.repetition;
    if (count) {
        l = l - s.frequency * (float)count;
        l = l - s.presence;
    }
    return l + bias;
}

__device__ __forceinline__ bool admitted(const uint32_t* mask, int column) {
    return !mask || (mask[column >> 5] >> (column & 31) & 1);
}

// Eight columns from any element on, as the words they lie in: global memory takes 16
// bytes at any element's address.
template <int TYPE>
struct Eight {
    uint32_t u[TYPE == 2 ? 8 : 4];
};
template <int TYPE>
__device__ __forceinline__ Eight<TYPE> load8(const void* p, int64_t i) {
    Eight<TYPE> v;
    __builtin_memcpy(&v, static_cast<const uint8_t*>(p) + i * (TYPE == 2 ? 4 : 2), sizeof v);
    return v;
}
template <int TYPE>
__device__ __forceinline__ void store8(void* p, int64_t i, const Eight<TYPE>& v) {
    __builtin_memcpy(static_cast<uint8_t*>(p) + i * (TYPE == 2 ? 4 : 2), &v, sizeof v);
}
// Past the caches: 256 rows of 151936 in 48 and 38 us; with a sampler behind them the same, 81.
template <int TYPE>
__device__ __forceinline__ void store8_past(void* p, int64_t i, const Eight<TYPE>& v) {
    typedef uint32_t any_u32x4_t __attribute__((ext_vector_type(4), aligned(2)));
    any_u32x4_t* to = reinterpret_cast<any_u32x4_t*>(static_cast<uint8_t*>(p) + i * (TYPE == 2 ? 4 : 2));
#pragma unroll
    for (int w = 0; w < (int)(sizeof v / 16); ++w)
        __builtin_nontemporal_store(any_u32x4_t{v.u[4 * w], v.u[4 * w + 1], v.u[4 * w + 2], v.u[4 * w + 3]}, to + w);
}
// The same in another type (16 bits to 32).
template <int IN, int OUT>
__device__ __forceinline__ Eight<OUT> to_type(const Eight<IN>& v) {
    if constexpr (IN == OUT) return v;
    else {
        Eight<OUT> w;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t b = v.u[e >> 1] >> (16 * (e & 1)) & 0xFFFFu;
            w.u[e] = __float_as_uint(IN == 1 ? half_bits_to_float(b) : bf16_bits_to_float(b));
        }
        return w;
    }
}
// Columns whose bit is 0 become `other` (a 16-bit value in both halves).
template <int TYPE>
__device__ __forceinline__ void keep8(Eight<TYPE>& v, uint32_t bits, uint32_t other) {
#pragma unroll
    for (int w = 0; w < (int)(sizeof v / 4); ++w) {
        uint32_t keep;
        if constexpr (TYPE == 2) keep = 0u - (bits >> w & 1);
        else keep = ((0u - (bits >> (2 * w) & 1)) & 0xFFFFu) | (0u - (bits >> (2 * w + 1) & 1)) << 16;
        v.u[w] = (v.u[w] & keep) | (other & ~keep);
    }
}
template <int TYPE>
__device__ __forceinline__ void store_some(void* p, int64_t i, const Eight<TYPE>& v, uint32_t some) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (some >> e & 1) {
            if constexpr (TYPE == 2) static_cast<uint32_t*>(p)[i + e] = v.u[e];
            else static_cast<uint16_t*>(p)[i + e] = (uint16_t)(v.u[e >> 1] >> (16 * (e & 1)));
        }
}
template <int TYPE>
constexpr uint32_t minus_infinity() { return TYPE == 2 ? 0xFF800000u : TYPE == 1 ? 0xFC00FC00u : 0xFF80FF80u; }
template <int TYPE>
constexpr uint32_t not_a_number() { return TYPE == 2 ? 0x7FC00000u : TYPE == 1 ? 0x7E007E00u : 0x7FC07FC0u; }

// A (row, chunk of columns) per workgroup.
// Out of place: the chunk goes from logits to outputs through registers, eight columns
// per thread and access, and where its columns have listed tokens or drafts through
// LDS, in the output's type (16 KB), where those are changed; then the mask is applied.
// A last vector that the columns do not fill starts earlier, over columns that another
// thread writes too, with the same values.
// In place (INPLACE): listed tokens and masked columns are written by themselves. A
// token whose bit is 0 is left to the mask, so no column is written with two values.
template <int IN, int OUT, bool INPLACE>
// (eight waves per SIMD: with four the copy alone takes 45 us)
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(8, 8))) void penalty_kernel(PenaltyArgs a) {
    constexpr int kChunk = kPenaltyBytes / (OUT == 2 ? 4 : 2), kTurns = kChunk / (8 * kThreads), kLists = kChunk / kHistoryBucket;
    static_assert(kChunk % kHistoryBucket == 0, "a list is one workgroup's");
    __shared__ __attribute__((aligned(16))) uint8_t staged[INPLACE ? 16 : kPenaltyBytes];
    __shared__ int drafts[kMaxPenaltyDepth], taken[kLists + 1];
    // (all rows' first chunks first: vocabularies begin with the tokens that come often, so
    // those have the long lists and should not come last)
    // The rows of a sequence, eight sequences at a time, on one XCD (workgroups go round robin
    // over the eight): its lists and marks come from one L2 (38 us, and 42 without).
    int row = blockIdx.x;
    const int chunk = blockIdx.y, band = 8 * (a.depth + 1), within = row % band;
    if (row - within + band <= (int)gridDim.x) row = row - within + (within & 7) * (a.depth + 1) + (within >> 3);
    const int live = a.live_count ? min(max(*a.live_count, 0), a.live_sequences) : a.live_sequences;
    const int buckets = history_buckets(a.history.vocab);
    const int sequence = row / (a.depth + 1), ahead = row - sequence * (a.depth + 1);
    if (sequence >= live) return;
    const int c0 = chunk * kChunk, columns = min(kChunk, a.width - c0);
    const uint32_t* mask = a.mask ? a.mask + (int64_t)row * a.mask_words : nullptr;
    const int64_t in_at = (int64_t)row * a.ld + c0, out_at = (int64_t)row * a.ldout + c0;
    const bool whole = columns >= 8;  // else one column per thread
    auto start = [&](int i) { return min((i * kThreads + (int)threadIdx.x) * 8, columns - 8); };
    auto mine = [&](int i) { return whole && (i * kThreads + (int)threadIdx.x) * 8 < columns; };
    auto bits_of = [&](int c) -> uint32_t {  // of eight columns, at any place of the mask's bytes
        if (!mask) return 0xFFu;
        const int first = c0 + c, byte = min(first >> 3, (int)min(a.mask_words, (int64_t)1 << 28) * 4 - 2);
        uint16_t two;
        __builtin_memcpy(&two, reinterpret_cast<const uint8_t*>(mask) + byte, 2);
        return (uint32_t)two >> (first - 8 * byte) & 0xFFu;
    };

    int64_t draft = -1;
    if ((int)threadIdx.x < ahead) draft = a.drafts[(int64_t)threadIdx.x * a.sequences + sequence] - c0;
    const int slot = a.row_slots[sequence];
    const bool slotted = slot >= 0 && slot < a.history.slots;
    const int64_t base = slotted ? (int64_t)slot * a.history.vocab : 0;
    const uint2* state = a.history.state + base + c0;
    const int32_t* listed = a.history.listed + base + c0;
    // Each thread's first token of every list, and what is kept of it, before it is
    // known how many there are: a place past a list's end holds an older token, or 0.
    int early[kLists];
    uint2 early_of[kLists];
#pragma unroll
    for (int l = 0; l < kLists; ++l) {
        const int at = l * kHistoryBucket + (int)threadIdx.x;
        early[l] = slotted && c0 + at < a.history.vocab ? listed[at] - c0 : -1;
    }
    // all loads of the chunk before the first store: the compiler does not move a
    // load up over a store that may be to its place
    Eight<IN> in[kTurns] = {};
    uint32_t bits[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
        bits[i] = 0xFFu;
        if (mine(i)) {
            bits[i] = bits_of(start(i));
            if constexpr (!INPLACE) in[i] = load8<IN>(a.logits, in_at + start(i));
        }
    }
#pragma unroll
    for (int l = 0; l < kLists; ++l) {
        const bool in_chunk = early[l] >= 0 && early[l] < columns && admitted(mask, c0 + early[l]);
        early[l] = in_chunk ? early[l] : -1;
        early_of[l] = in_chunk ? state[early[l]] : make_uint2(0, 0);
    }
    const Settings s = settings_of(a, sequence);
    const bool known = s.valid && slotted;
    // What is listed, and whether a draft is a column of this chunk, as the first wave finds it: the
    // barriers below are met by all of a workgroup or by none, whatever becomes of memory meanwhile.
    if ((int)threadIdx.x < kLists) {
        const int bucket = c0 / kHistoryBucket + (int)threadIdx.x;
        taken[threadIdx.x] = known && bucket < buckets ? min(a.history.sizes[(int64_t)slot * buckets + bucket], kHistoryBucket) : 0;
    }
    const bool drafted = (int)threadIdx.x < ahead && known && draft >= 0 && draft < columns;
    if ((int)threadIdx.x < ahead) drafts[threadIdx.x] = drafted ? (int)draft : -1;
    const bool any_drafted = __ballot(drafted) != 0;
    if (threadIdx.x == 0) taken[kLists] = any_drafted;
    __syncthreads();
    int sizes[kLists], some = __builtin_amdgcn_readfirstlane(taken[kLists]);
#pragma unroll
    for (int l = 0; l < kLists; ++l) some += sizes[l] = __builtin_amdgcn_readfirstlane(taken[l]);
    if (some || !whole) {
        if constexpr (!INPLACE) {
#pragma unroll
            for (int i = 0; i < kTurns; ++i)
                if (mine(i)) store8<OUT>(staged, start(i), to_type<IN, OUT>(in[i]));
            if (!whole && (int)threadIdx.x < columns)
                set_value<OUT>(staged, threadIdx.x, value_of<IN>(a.logits, in_at + threadIdx.x));
        }
        __syncthreads();
        auto change = [&](int c, uint2 mark) {
            int more = 0;
            for (int j = 0; j < ahead; ++j) more += drafts[j] == c;
            const float l = INPLACE ? value_of<IN>(a.logits, in_at + c) : value_of<OUT>(staged, c);
            const float to = penalised(l, mark.x, more, __uint_as_float(mark.y), s);
            if constexpr (INPLACE) set_value<OUT>(a.out, out_at + c, to);
            else set_value<OUT>(staged, c, to);
        };
#pragma unroll
        for (int l = 0; l < kLists; ++l) {
            if ((int)threadIdx.x < sizes[l] && early[l] >= 0) change(early[l], early_of[l]);
            // the others two at a time, whose loads are on their way together
            for (int i = kThreads + threadIdx.x; i < sizes[l]; i += 2 * kThreads) {
                const int j = i + kThreads;
                int c = listed[l * kHistoryBucket + i] - c0, d = j < sizes[l] ? listed[l * kHistoryBucket + j] - c0 : -1;
                if (c >= columns || !admitted(mask, c0 + c)) c = -1;
                if (d >= columns || (d >= 0 && !admitted(mask, c0 + d))) d = -1;
                const uint2 of_c = c >= 0 ? state[c] : make_uint2(0, 0), of_d = d >= 0 ? state[d] : make_uint2(0, 0);
                if (c >= 0) change(c, of_c);
                if (d >= 0) change(d, of_d);
            }
        }
        if ((int)threadIdx.x < ahead) {  // drafts that are new to the request
            const int c = drafts[threadIdx.x];
            bool first = c >= 0;
            for (int j = 0; j < (int)threadIdx.x; ++j) first = first && drafts[j] != c;
            if (first && admitted(mask, c0 + c) && !(state[c].x & kListed)) change(c, make_uint2(0, 0));
        }
        __syncthreads();
    }
    if (!INPLACE || mask || !s.valid) {
        const uint32_t other = s.valid ? minus_infinity<OUT>() : not_a_number<OUT>();
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            if (!mine(i)) continue;
            Eight<OUT> out = to_type<IN, OUT>(in[i]);
            if constexpr (!INPLACE) {
                if (some) out = load8<OUT>(staged, start(i));
            }
            const uint32_t keep = s.valid ? bits[i] : 0u;
            keep8<OUT>(out, keep, other);
            if constexpr (!INPLACE) store8_past<OUT>(a.out, out_at + start(i), out);
            else if (keep == 0u) store8<OUT>(a.out, out_at + start(i), out);
            else if (keep != 0xFFu) store_some<OUT>(a.out, out_at + start(i), out, ~keep);
        }
        if (!whole && (int)threadIdx.x < columns) {
            const bool keep = s.valid && admitted(mask, c0 + threadIdx.x);
            if (!keep) set_value<OUT>(a.out, out_at + threadIdx.x, s.valid ? -__builtin_huge_valf() : __builtin_nanf(""));
            else if constexpr (!INPLACE) set_value<OUT>(a.out, out_at + threadIdx.x, value_of<OUT>(staged, threadIdx.x));
        }
    }
}

template <int IN, int OUT>
hipError_t launch_typed(const PenaltyArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.live_sequences * (a.depth + 1)), (unsigned)a.chunks);
    if (a.inplace) penalty_kernel<IN, IN, true><<<grid, kThreads, 0, s>>>(a);
    else penalty_kernel<IN, OUT, false><<<grid, kThreads, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_penalties(const PenaltyArgs& a, hipStream_t s) {
    if (a.live_sequences < 1) return hipSuccess;
    if (a.in == 2) return launch_typed<2, 2>(a, s);
    if (a.in == 1) return a.out_type == 2 ? launch_typed<1, 2>(a, s) : launch_typed<1, 1>(a, s);
    return a.out_type == 2 ? launch_typed<0, 2>(a, s) : launch_typed<0, 0>(a, s);
}

hipError_t launch_history_append(const HistoryArgs& h, const HistoryTokens& a, hipStream_t s) {
    const int64_t groups = ((int64_t)a.live_rows * a.length + kThreads - 1) / kThreads, most = 1 << 16;
    if (groups < 1) return hipSuccess;
    history_append_kernel<<<(unsigned)(groups < most ? groups : most), kThreads, 0, s>>>(h, a);
    return hipGetLastError();
}

hipError_t launch_history_clear(const HistoryArgs& h, const int32_t* row_slots, int rows, int only_slot, int biases_only, hipStream_t s) {
    history_clear_kernel<<<rows < (1 << 16) ? rows : 1 << 16, 1024, 0, s>>>(h, row_slots, rows, only_slot, biases_only);
    return hipGetLastError();
}

hipError_t launch_history_bias(const HistoryArgs& h, int slot, const int32_t* ids, const float* values, int n, hipStream_t s) {
    history_bias_kernel<<<(n + kThreads - 1) / kThreads, kThreads, 0, s>>>(h, slot, ids, values, n);
    return hipGetLastError();
}

}  // namespace cubic
