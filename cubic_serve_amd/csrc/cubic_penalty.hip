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
// A history keeps per slot a table of marks (outputs counted, in the prompt,
// listed), a table of biases, and the list of the tokens that have either, in
// the order of their arrival.  The list's order is that of atomics; nothing depends on
// it, since each listed token is taken by itself.
//
// What bounds the penalties: reading and writing the logits.  Listed tokens are a few
// thousand of 10^5 columns, so each is looked up by itself.
#include <type_traits>

#include "cubic_capi_internal.h"
#include "cubic_device.h"

namespace cubic {
namespace {

constexpr uint32_t kListed = 1u << 30, kPrompt = 1u << 31, kCount = kListed - 1;
constexpr int kThreads = 256;

// Puts a token on its slot's list unless it is there.
__device__ __forceinline__ void list_token(const HistoryArgs& h, int64_t slot, int t, uint32_t mark) {
    if (mark & kListed) return;
    if (atomicOr(&h.marks[slot * h.vocab + t], kListed) & kListed) return;
    h.listed[slot * h.vocab + atomicAdd(&h.sizes[slot], 1)] = t;
}

__global__ __launch_bounds__(kThreads) void history_append_kernel(HistoryArgs h, HistoryTokens a) {
    const int live = a.live_count ? min(max(*a.live_count, 0), a.live_rows) : a.live_rows;
    const int64_t all = (int64_t)live * a.length;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < all; i += (int64_t)gridDim.x * kThreads) {
        const int64_t row = i / a.length, at = row * a.ld + (i - row * a.length);
        const int64_t t = a.token_bytes == 8 ? static_cast<const int64_t*>(a.tokens)[at] : static_cast<const int32_t*>(a.tokens)[at];
        const int slot = a.row_slots[row];
        if (slot < 0 || slot >= h.slots || t < 0 || t >= h.vocab) continue;
        uint32_t* mark = &h.marks[(int64_t)slot * h.vocab + t];
        const uint32_t old = a.prompt ? atomicOr(mark, kPrompt) : atomicAdd(mark, 1u);
        list_token(h, slot, (int)t, old);
    }
}

// One workgroup per row: the tables' listed places back to zero (biases_only:
// those of the biases), then the list.
__global__ __launch_bounds__(1024) void history_clear_kernel(HistoryArgs h, const int32_t* row_slots, int rows, int only_slot,
                                                             int biases_only) {
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        const int slot = row_slots ? row_slots[row] : only_slot;
        if (slot < 0 || slot >= h.slots) continue;
        const int64_t base = (int64_t)slot * h.vocab;
        const int n = min(h.sizes[slot], h.vocab);
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            const int t = h.listed[base + i];
            h.biases[base + t] = 0.0f;
            if (!biases_only) h.marks[base + t] = 0;
        }
        __syncthreads();
        if (!biases_only && threadIdx.x == 0) h.sizes[slot] = 0;
    }
}

__global__ __launch_bounds__(kThreads) void history_bias_kernel(HistoryArgs h, int slot, const int32_t* ids, const float* values, int n) {
    const int i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= n) return;
    const int t = ids[i];
    if (t < 0 || t >= h.vocab) return;
    h.biases[(int64_t)slot * h.vocab + t] = values[i];
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

// A (row, chunk of kPenaltyChunk columns) per workgroup and turn.
// Out of place: the chunk is staged in LDS in the output's type, the listed tokens
// in it are changed there, and it leaves with the mask applied: every output line is
// written once.  In place (INPLACE): listed tokens, shared out over the
// row's workgroups, and masked columns are written by themselves; a token
// whose bit is 0 is left to the mask, so no two threads write one column.
template <int IN, int OUT, bool INPLACE>
__global__ __launch_bounds__(kThreads) void penalty_kernel(PenaltyArgs a) {
    typedef typename std::conditional<OUT == 2, float, uint16_t>::type out_t;
    __shared__ __attribute__((aligned(16))) out_t staged[INPLACE ? 8 : kPenaltyChunk];
    __shared__ int drafts[kMaxPenaltyDepth];
    const int live = a.live_count ? min(max(*a.live_count, 0), a.live_sequences) : a.live_sequences;
    const int64_t items = (int64_t)live * (a.depth + 1) * a.chunks;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int row = (int)(item / a.chunks), chunk = (int)(item - (int64_t)row * a.chunks);
        const int sequence = row / (a.depth + 1), ahead = row - sequence * (a.depth + 1);
        const int c0 = chunk * kPenaltyChunk, columns = min(kPenaltyChunk, a.width - c0);
        const uint32_t* mask = a.mask ? a.mask + (int64_t)row * a.mask_words : nullptr;
        const int64_t in_row = (int64_t)row * a.ld, out_row = (int64_t)row * a.ldout;
        const int slot = a.row_slots[sequence];
        const Settings s = settings_of(a, sequence);
        const bool known = slot >= 0 && slot < a.history.slots;
        const int64_t base = known ? (int64_t)slot * a.history.vocab : 0;
        if ((int)threadIdx.x < ahead) {
            const int64_t t = a.drafts[(int64_t)threadIdx.x * a.sequences + sequence];
            drafts[threadIdx.x] = t >= 0 && t < a.width ? (int)t : -1;
        }
        if constexpr (!INPLACE) {
            for (int c = threadIdx.x; c < columns; c += kThreads) set_value<OUT>(staged, c, value_of<IN>(a.logits, in_row + c0 + c));
        }
        __syncthreads();
        // a token of this chunk (in place: of this workgroup's share)
        auto change = [&](int t, uint32_t mark, float bias) {
            if constexpr (INPLACE) {
                if (!admitted(mask, t)) return;
            }
            int more = 0;
            for (int j = 0; j < ahead; ++j) more += drafts[j] == t;
            const float v = penalised(value_of<IN>(a.logits, in_row + t), mark, more, bias, s);
            if constexpr (INPLACE) set_value<OUT>(a.out, out_row + t, v);
            else set_value<OUT>(staged, t - c0, v);
        };
        if (known && s.valid) {
            const uint32_t* marks = a.history.marks + base;
            const int n = min(a.history.sizes[slot], a.history.vocab);
            if constexpr (INPLACE) {
                for (int i = chunk * kThreads + threadIdx.x; i < n; i += a.chunks * kThreads) {
                    const int t = a.history.listed[base + i];
                    if (t < a.width) change(t, marks[t], a.history.biases[base + t]);
                }
            } else {
                for (int i = threadIdx.x; i < n; i += kThreads) {
                    const int t = a.history.listed[base + i];
                    if (t >= c0 && t < c0 + columns) change(t, marks[t], a.history.biases[base + t]);
                }
            }
            if ((int)threadIdx.x < ahead) {  // drafts that are new to the request
                const int t = drafts[threadIdx.x];
                bool first = t >= 0;
                for (int j = 0; j < (int)threadIdx.x; ++j) first = first && drafts[j] != t;
                if (first && (INPLACE ? chunk == 0 : t >= c0 && t < c0 + columns) && !(marks[t] & kListed)) change(t, 0, 0.0f);
            }
        }
        __syncthreads();
        if constexpr (INPLACE) {
            if (mask || !s.valid)
                for (int c = c0 + threadIdx.x; c < c0 + columns; c += kThreads) {
                    if (!s.valid) set_value<OUT>(a.out, out_row + c, __builtin_nanf(""));
                    else if (!admitted(mask, c)) set_value<OUT>(a.out, out_row + c, -__builtin_huge_valf());
                }
        } else {
            for (int c = threadIdx.x; c < columns; c += kThreads) {
                const float v = !s.valid ? __builtin_nanf("") : !admitted(mask, c0 + c) ? -__builtin_huge_valf() : value_of<OUT>(staged, c);
                set_value<OUT>(a.out, out_row + c0 + c, v);
            }
        }
        __syncthreads();  // the staged chunk and the drafts are read
    }
}

template <int IN, int OUT>
hipError_t launch_typed(const PenaltyArgs& a, hipStream_t s) {
    const int64_t items = (int64_t)a.live_sequences * (a.depth + 1) * a.chunks, most = 1 << 22;
    const unsigned grid = (unsigned)(items < most ? items : most);
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
