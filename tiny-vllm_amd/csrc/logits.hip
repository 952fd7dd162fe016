// Logit controls in front of the sampler: penalties for tokens that a request
// has seen, additive biases, and masks of allowed tokens.
//
// For row r and token i, x = logits[r, i] in fp32, c the number of times i
// stands in the answer part of the row's history, and seen whether it stands
// in the history at all (prompt or answer):
//   seen:  x = x > 0 ? x / repetition : x * repetition
//   x = x - frequency * c - presence * [c > 0]
//   x = x + bias(r, i)
//   x = -inf where the mask bit of i is 0
// rounded once to the output's type. The reference has no counterpart (its
// sampler takes the logits as they are: tinyvllm/sampling.py:21-72).
//
// MI355X design: one pass over the vocabulary, a workgroup per row and span of
// 8192 tokens, 8 to a thread. The history is a list of token ids by position
// (what a decode step can append to on the device, where the newest token
// still is when the next step starts); each workgroup scans its row's list and
// counts the ids of its own span in LDS, so no table of counts per request and
// token has to be kept, cleared or read. The spans of a row sit on one XCD, so
// its L2 serves the list to all but the first.
#include "common.h"

#include <type_traits>

namespace tvllm {
namespace {

constexpr int kThreads = 1024;
constexpr int kPer = 8;                  // tokens per thread
constexpr int kSpan = kThreads * kPer;   // tokens per workgroup
constexpr uint32_t kPrompt = 0x80000000u;  // the token stands in the prompt part

struct Args {
    const void* logits;
    void* out;
    int64_t stride, out_stride;  // elements
    int64_t vocab, spans, grid;
    bool in_place;
    const float* repetition;
    const float* presence;
    const float* frequency;
    int32_t* history;  // [slots][capacity]
    int64_t num_slots, capacity;
    const int64_t* slots;
    const int64_t* lengths;
    const int64_t* prompts;
    const int64_t* newest;
    const int32_t* bias_tokens;
    const float* bias_values;
    const int64_t* bias_offsets;
    int64_t num_bias;
    const uint32_t* mask;  // [mask_count][mask_stride] words
    int64_t mask_count, mask_stride;
    const int64_t* mask_rows;
};

// VEC: rows of both tensors are 16-byte aligned, a thread's tokens are 8
// neighbours; otherwise neighbouring threads hold neighbouring tokens.
template <typename TI, typename TO, bool VEC>
__global__ void __launch_bounds__(kThreads)
logit_controls(Args a) {
    __shared__ uint32_t count[kSpan];
    const int tid = threadIdx.x;
    int64_t bid = blockIdx.x;
    // Block ids are dealt to 8 XCDs in turn: give each a contiguous range.
    const int64_t per = a.grid / 8, rest = a.grid % 8, xcd = bid % 8;
    bid = xcd * per + min(xcd, rest) + bid / 8;
    const int64_t r = bid / a.spans;
    const int64_t base = (bid - r * a.spans) * kSpan;
    const int64_t left = a.vocab - base;  // tokens of the span
    auto at = [&](int e) { return VEC ? tid * kPer + e : e * kThreads + tid; };

    // What the row asks for (all uniform).
    int64_t slot = a.history ? a.slots[r] : -1, n = 0, prompt = 0;
    float rho = 1.f, pres = 0.f, freq = 0.f;
    if (slot >= 0 && slot < a.num_slots) {
        n = a.lengths[r];
        prompt = a.prompts[r];
        if (a.repetition) rho = a.repetition[r];
        if (a.presence) pres = a.presence[r];
        if (a.frequency) freq = a.frequency[r];
    }
    int32_t* const list = a.history + (n > 0 ? slot * a.capacity : 0);
    // The newest token: it takes the last position, which nobody reads here.
    int64_t last = -1;
    if (n > 0 && a.newest) {
        last = a.newest[r];
        if (last < 0 || last >= a.vocab) last = -1;
        --n;
        if (base == 0 && tid == 0 && n < a.capacity) list[n] = int32_t(last);
    }
    const int64_t stored = min(n, a.capacity);
    const bool penal = (stored > 0 || last >= 0) && (rho != 1.f || pres != 0.f || freq != 0.f);
    int64_t b0 = 0, b1 = 0;
    if (a.bias_offsets) {
        b0 = max(int64_t(0), a.bias_offsets[r]);
        b1 = min(a.num_bias, a.bias_offsets[r + 1]);
    }
    const bool biased = b0 < b1;
    const int64_t mrow = a.mask_rows ? a.mask_rows[r] : -1;
    const bool masked = mrow >= 0 && mrow < a.mask_count;
    if (a.in_place && !penal && !biased && !masked) return;

    const TI* const src = static_cast<const TI*>(a.logits) + r * a.stride + base;
    TO* const dst = static_cast<TO*>(a.out) + r * a.out_stride + base;
    float x[kPer];
    auto load = [&]() {
        if (VEC && at(0) + kPer <= left) {
            if constexpr (sizeof(TI) == 2) {
                unpack8<TI>(*reinterpret_cast<const U16x8*>(src + at(0)), x);
            } else {
                const float4 lo = *reinterpret_cast<const float4*>(src + at(0));
                const float4 hi = *reinterpret_cast<const float4*>(src + at(0) + 4);
                x[0] = lo.x; x[1] = lo.y; x[2] = lo.z; x[3] = lo.w;
                x[4] = hi.x; x[5] = hi.y; x[6] = hi.z; x[7] = hi.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < kPer; ++e) x[e] = at(e) < left ? to_f<TI>(src[at(e)]) : 0.f;
        }
    };
    // Out of place every token is copied: the loads go out ahead of the counting.
    if (!a.in_place) load();

    uint32_t c[kPer] = {};
    uint32_t which[kPer] = {};  // 1 + the token's last entry in the row's biases
    auto clear = [&]() {
        for (int i = tid; i < kSpan; i += kThreads) count[i] = 0u;
        __syncthreads();
    };
    auto read = [&](uint32_t (&to)[kPer]) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kPer; ++e) to[e] = count[at(e)];
    };
    if (penal) {
        clear();
        auto add = [&](int64_t token, int64_t position) {
            const int64_t i = token - base;
            if (i >= 0 && i < kSpan) {
                if (position < prompt) atomicOr(&count[i], kPrompt);
                else atomicAdd(&count[i], 1u);
            }
        };
        for (int64_t p = tid; p < stored; p += kThreads) add(list[p], p);
        if (tid == 0 && last >= 0) add(last, n);
        read(c);
    }
    if (biased) {
        __syncthreads();  // the counts are read
        clear();
        for (int64_t p = b0 + tid; p < b1; p += kThreads) {
            const int64_t i = a.bias_tokens[p] - base;
            if (i >= 0 && i < kSpan) atomicMax(&count[i], uint32_t(p - b0 + 1));
        }
        read(which);
    }

    bool touched = masked;
#pragma unroll
    for (int e = 0; e < kPer; ++e) touched |= c[e] != 0u || which[e] != 0u;
    if (a.in_place) {
        if (!touched) return;
        load();
    }
    if (touched) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            if (c[e]) {
                x[e] = x[e] > 0.f ? x[e] / rho : x[e] * rho;
                const uint32_t times = c[e] & ~kPrompt;
                x[e] -= freq * float(times);
                if (times) x[e] -= pres;
            }
            if (which[e]) x[e] += a.bias_values[b0 + which[e] - 1];
        }
        if (masked) {
            const uint32_t* const words = a.mask + mrow * a.mask_stride;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const int64_t i = base + at(e);
                if (at(e) < left && !((words[i >> 5] >> (i & 31)) & 1u)) x[e] = -INFINITY;
            }
        }
    }
    if (VEC && at(0) + kPer <= left) {
        if constexpr (sizeof(TO) == 2) {
            U16x8 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w.w[e] = pack2<TO>(x[2 * e], x[2 * e + 1]);
            *reinterpret_cast<U16x8*>(dst + at(0)) = w;
        } else {
            *reinterpret_cast<float4*>(dst + at(0)) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(dst + at(0) + 4) = make_float4(x[4], x[5], x[6], x[7]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e)
            if (at(e) < left) dst[at(e)] = static_cast<TO>(x[e]);
    }
}

}  // namespace
}  // namespace tvllm

using namespace tvllm;

extern "C" int tvllm_logit_controls(
    const void* logits, int64_t rows, int64_t vocab, int64_t row_stride, const float* repetition,
    const float* presence, const float* frequency, int32_t* history, int64_t num_slots,
    int64_t capacity, const int64_t* slots, const int64_t* lengths, const int64_t* prompt_lens,
    const int64_t* newest, const int32_t* bias_tokens, const float* bias_values,
    const int64_t* bias_offsets, int64_t num_bias, const int32_t* mask, int64_t mask_count,
    int64_t mask_stride, const int64_t* mask_rows, void* out, int64_t out_stride, int dtype,
    int out_dtype, tvllm_stream_t stream) {
    TVLLM_CHECK(dtype == TVLLM_BF16 || dtype == TVLLM_F16 || dtype == TVLLM_F32,
                "logit_controls: logits must be float16, bfloat16 or float32");
    TVLLM_CHECK(out_dtype == dtype || out_dtype == TVLLM_F32,
                "logit_controls: the output has the logits' type or float32");
    TVLLM_CHECK(rows >= 0 && vocab > 0 && vocab <= INT32_MAX, "logit_controls: invalid sizes");
    TVLLM_CHECK(row_stride >= vocab && out_stride >= vocab,
                "logit_controls: rows must not overlap");
    TVLLM_CHECK(num_slots >= 0 && capacity >= 0 && num_bias >= 0 && num_bias <= INT32_MAX &&
                    mask_count >= 0,
                "logit_controls: negative sizes");
    TVLLM_CHECK(capacity <= INT32_MAX, "logit_controls: at most 2^31-1 tokens of history");
    TVLLM_CHECK(!mask_rows || mask_count == 0 || mask_stride >= (vocab + 31) / 32,
                "logit_controls: a mask row has a bit for every token");
    if (rows == 0) {
        clear_error();
        return TVLLM_OK;
    }
    TVLLM_CHECK(logits && out, "logit_controls: null pointer");
    TVLLM_CHECK(!history || (slots && lengths && prompt_lens), "logit_controls: null pointer");
    TVLLM_CHECK(!bias_offsets || num_bias == 0 || (bias_tokens && bias_values),
                "logit_controls: null pointer");
    TVLLM_CHECK(!mask_rows || mask_count == 0 || mask, "logit_controls: null pointer");
    TVLLM_CHECK(logits != out || (out_dtype == dtype && out_stride == row_stride),
                "logit_controls: in place, the output has the logits' type and rows");
    Args a{};
    a.logits = logits;
    a.out = out;
    a.stride = row_stride;
    a.out_stride = out_stride;
    a.vocab = vocab;
    a.spans = (vocab + kSpan - 1) / kSpan;
    a.grid = rows * a.spans;
    a.in_place = logits == out;
    a.repetition = repetition;
    a.presence = presence;
    a.frequency = frequency;
    a.history = history;
    a.num_slots = num_slots;
    a.capacity = capacity;
    a.slots = slots;
    a.lengths = lengths;
    a.prompts = prompt_lens;
    a.newest = newest;
    a.bias_tokens = bias_tokens;
    a.bias_values = bias_values;
    a.bias_offsets = num_bias ? bias_offsets : nullptr;
    a.num_bias = num_bias;
    a.mask = reinterpret_cast<const uint32_t*>(mask);
    a.mask_count = mask_count;
    a.mask_stride = mask_stride;
    a.mask_rows = mask_count ? mask_rows : nullptr;
    TVLLM_CHECK(a.grid <= INT32_MAX, "logit_controls: grid too large");
    const int64_t unit = dtype == TVLLM_F32 ? 4 : 8, out_unit = out_dtype == TVLLM_F32 ? 4 : 8;
    const bool vec = aligned16(logits) && aligned16(out) && row_stride % unit == 0 &&
                     out_stride % out_unit == 0;
    hipStream_t s = as_hip(stream);
    return dispatch_float(dtype, [&]<int DT>() {
        using T = typename Elem<DT>::T;
        auto go = [&]<typename TO>() {
            if (vec) logit_controls<T, TO, true><<<int(a.grid), kThreads, 0, s>>>(a);
            else logit_controls<T, TO, false><<<int(a.grid), kThreads, 0, s>>>(a);
        };
        if (out_dtype == dtype) go.template operator()<T>();
        else go.template operator()<float>();
        return launch_status("logit_controls");
    });
}
