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
// 8192 tokens, 16 to a thread. The history is a list of token ids by position
// (what a decode step can append to on the device, where the newest token
// still is when the next step starts); each workgroup scans its row's list and
// counts the ids of its own span in LDS, so no table of counts per request and
// token has to be kept, cleared or read. The spans of a row sit on one XCD, so
// its L2 serves the list to all but the first.
//
// Measured on one MI355X (kernel trace), 151936 tokens: 256 rows fp32, lists of
// 2048-32768 ids, biases and masks 102 us, 3.3 TB/s of logits in and out and
// lists; 64 rows bf16, lists up to 4096 15.5 us; one row 6.2 us. The first is
// bound by the scans: without controls it takes 71 us (torch's copy 59), with
// lists of at most 8192 ids 83, every span's workgroup looking at every id.
// Threads and tokens per thread, us for the first two: 512 x 16 107 / 15.6
// (when chosen), 512 x 8 134 / 20.7, 1024 x 8 147 / 25.0, 256 x 16 119 / 15.0,
// 1024 x 16 117 / 19.2, 512 x 32 110 / 17.0.
#include "common.h"

#include <type_traits>

namespace tvllm {
namespace {

constexpr int kThreads = 512;
constexpr int kPer = 16;                 // tokens per thread
constexpr int kSpan = kThreads * kPer;   // tokens per workgroup
constexpr uint32_t kPrompt = 0x80000000u;  // the token stands in the prompt part

struct Args {
    const void* logits;
    void* out;
    int64_t stride, out_stride;  // elements
    int64_t vocab, spans, grid;
    bool in_place, list4;  // list4: the history's rows are 16-byte aligned
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

// VEC: rows of both tensors are 16-byte aligned, a thread's tokens are runs of 8
// neighbours; otherwise neighbouring threads hold neighbouring tokens.
template <typename TI, typename TO, bool VEC>
__global__ void __launch_bounds__(kThreads)
logit_controls(Args a) {
    __shared__ __align__(16) uint32_t count[kSpan];
    __shared__ int met[2];
    const int tid = threadIdx.x;
    int64_t bid = blockIdx.x;
    // Block ids are dealt to 8 XCDs in turn: give each a contiguous range.
    const int64_t share = a.grid / 8, rest = a.grid % 8, xcd = bid % 8;
    bid = xcd * share + min(xcd, rest) + bid / 8;
    const int64_t r = bid / a.spans;
    const int64_t base = (bid - r * a.spans) * kSpan;
    const int64_t left = a.vocab - base;  // tokens of the span
    auto at = [&](int e) {
        return VEC ? (e / 8 * kThreads + tid) * 8 + e % 8 : e * kThreads + tid;
    };

    // What the row asks for: all uniform, and all loaded at once.
    int64_t slot = a.history ? a.slots[r] : -1;
    int64_t n = a.history ? a.lengths[r] : 0, prompt = a.history ? a.prompts[r] : 0;
    const float rho = a.repetition ? a.repetition[r] : 1.f;
    const float pres = a.presence ? a.presence[r] : 0.f;
    const float freq = a.frequency ? a.frequency[r] : 0.f;
    int64_t last = a.newest ? a.newest[r] : -1;
    int64_t b0 = a.bias_offsets ? a.bias_offsets[r] : 0;
    int64_t b1 = a.bias_offsets ? a.bias_offsets[r + 1] : 0;
    const int64_t mrow = a.mask_rows ? a.mask_rows[r] : -1;
    const TI* const src = static_cast<const TI*>(a.logits) + r * a.stride + base;
    TO* const dst = static_cast<TO*>(a.out) + r * a.out_stride + base;
    float x[kPer];
    auto load = [&]() {
        if constexpr (VEC) {
#pragma unroll
            for (int g = 0; g < kPer / 8; ++g) {
                float (&y)[8] = reinterpret_cast<float (&)[8]>(x[8 * g]);
                if (at(8 * g) + 8 <= left) {
                    if constexpr (sizeof(TI) == 2) {
                        unpack8<TI>(*reinterpret_cast<const U16x8*>(src + at(8 * g)), y);
                    } else {
                        const float4 lo = *reinterpret_cast<const float4*>(src + at(8 * g));
                        const float4 hi = *reinterpret_cast<const float4*>(src + at(8 * g) + 4);
                        y[0] = lo.x; y[1] = lo.y; y[2] = lo.z; y[3] = lo.w;
                        y[4] = hi.x; y[5] = hi.y; y[6] = hi.z; y[7] = hi.w;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        y[e] = at(8 * g + e) < left ? to_f<TI>(src[at(8 * g + e)]) : 0.f;
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < kPer; ++e) x[e] = at(e) < left ? to_f<TI>(src[at(e)]) : 0.f;
        }
    };
    // Out of place every token is copied: the loads go out ahead of the counting.
    if (!a.in_place) load();

    if (slot < 0 || slot >= a.num_slots || n <= 0) {
        n = 0;
        last = -1;
        slot = 0;
    }
    int32_t* const list = a.history + slot * a.capacity;
    // The newest token: it takes the last position, which nobody reads here.
    if (n > 0 && a.newest) {
        if (last < 0 || last >= a.vocab) last = -1;
        --n;
        if (base == 0 && tid == 0 && n < a.capacity) list[n] = int32_t(last);
    }
    const int stored = int(min(n, a.capacity));
    const bool penal = (stored > 0 || last >= 0) && (rho != 1.f || pres != 0.f || freq != 0.f);
    b0 = max(int64_t(0), b0);
    b1 = min(a.num_bias, b1);
    const bool biased = b0 < b1;
    const bool masked = mrow >= 0 && mrow < a.mask_count;
    if (a.in_place && !penal && !biased && !masked) return;

    // Cells that a scan of a list has marked are read by the threads that keep
    // their tokens, and only if the scan met the span at all.
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < kPer / 4; ++i)
            reinterpret_cast<uint4*>(count)[i * kThreads + tid] = make_uint4(0, 0, 0, 0);
        if (tid < 2) met[tid] = 0;
        __syncthreads();
    };
    uint32_t c[kPer];
    auto read = [&]() {  // whether one of the thread's cells is marked
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < kPer / 4; ++i) {
                const uint4 w = *reinterpret_cast<const uint4*>(&count[at(4 * i)]);
                c[4 * i] = w.x;
                c[4 * i + 1] = w.y;
                c[4 * i + 2] = w.z;
                c[4 * i + 3] = w.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < kPer; ++e) c[e] = count[at(e)];
        }
        uint32_t any = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) any |= c[e];
        return any != 0;
    };
    bool loaded = !a.in_place;  // else a thread loads what it will change
    auto need = [&]() {
        if (!loaded) load();
        loaded = true;
    };
    if (penal || biased) clear();
    if (penal) {
        const uint32_t low = uint32_t(base);
        bool found = false;
        const int split = int(min(max(prompt, int64_t(0)), int64_t(stored)));
        auto mark = [&](int32_t token, bool in_prompt) {
            const uint32_t i = uint32_t(token) - low;  // (ids below the span wrap past it)
            if (i < uint32_t(kSpan)) {
                found = true;
                if (in_prompt) atomicOr(&count[i], kPrompt);
                else atomicAdd(&count[i], 1u);
            }
        };
        int p = 0;  // where the loop over single ids begins
        if (a.list4) {
            // Quads of ids, several loads of a thread at once. The quad that the
            // prompt ends in, and what is left of the list, are single ids of
            // the first threads.
            const int quads = stored / 4, mixed = split % 4 ? split / 4 : -1;
            p = 4 * quads;
            const int4* const list4 = reinterpret_cast<const int4*>(list);
            constexpr int kAhead = 4;
            if (mixed >= 0 && mixed < quads && tid < 4)
                mark(list[4 * mixed + tid], 4 * mixed + tid < split);
            for (int q0 = 0; q0 < quads; q0 += kAhead * kThreads) {
                int4 t[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int q = q0 + k * kThreads + tid;
                    t[k] = q < quads && q != mixed ? list4[q] : make_int4(-1, -1, -1, -1);
                }
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    auto four = [&](bool in_prompt) {
                        mark(t[k].x, in_prompt);
                        mark(t[k].y, in_prompt);
                        mark(t[k].z, in_prompt);
                        mark(t[k].w, in_prompt);
                    };
                    if (q0 + k * kThreads + tid < split / 4) four(true);
                    else four(false);
                }
            }
        }
        for (p += tid; p < stored; p += kThreads) mark(list[p], p < split);
        if (tid == 0 && last >= 0) mark(int32_t(last), n < prompt);
        if (found) met[0] = 1;
        __syncthreads();
        if (met[0] && read()) {
            need();
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                if (c[e]) {
                    x[e] = x[e] > 0.f ? x[e] / rho : x[e] * rho;
                    const uint32_t times = c[e] & ~kPrompt;
                    x[e] -= freq * float(times);
                    if (times) x[e] -= pres;
                    if (biased) count[at(e)] = 0;  // the biases find it cleared
                }
        }
    }
    if (biased) {
        if (penal) __syncthreads();
        bool found = false;
        for (int64_t p = b0 + tid; p < b1; p += kThreads) {
            const int64_t i = a.bias_tokens[p] - base;
            if (i >= 0 && i < kSpan) {  // 1 + the token's last entry in the row's list
                found = true;
                atomicMax(&count[i], uint32_t(p - b0 + 1));
            }
        }
        if (found) met[1] = 1;
        __syncthreads();
        if (met[1] && read()) {
            need();
#pragma unroll
            for (int e = 0; e < kPer; e += 4)
                if (c[e] | c[e + 1] | c[e + 2] | c[e + 3]) {
                    float y[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = a.bias_values[b0 + max(c[e + i], 1u) - 1];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[e + i] = c[e + i] ? x[e + i] + y[i] : x[e + i];
                }
        }
    }
    if (masked) {
        need();
        const uint32_t* const words = a.mask + mrow * a.mask_stride;
        if constexpr (VEC) {
#pragma unroll
            for (int g = 0; g < kPer / 8; ++g)
                if (at(8 * g) < left) {
                    const int64_t i = base + at(8 * g);
                    const uint32_t bits = words[i >> 5] >> (i & 31);  // 8 of one word
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (!((bits >> e) & 1u)) x[8 * g + e] = -INFINITY;
                }
        } else {
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const int64_t i = base + at(e);
                if (at(e) < left && !((words[i >> 5] >> (i & 31)) & 1u)) x[e] = -INFINITY;
            }
        }
    }
    if (!loaded) return;
    if constexpr (VEC) {
#pragma unroll
        for (int g = 0; g < kPer / 8; ++g) {
            const float (&y)[8] = reinterpret_cast<const float (&)[8]>(x[8 * g]);
            TO* const to = dst + at(8 * g);
            if (at(8 * g) + 8 <= left) {
                if constexpr (sizeof(TO) == 2) {
                    U16x8 w;
#pragma unroll
                    for (int e = 0; e < 4; ++e) w.w[e] = pack2<TO>(y[2 * e], y[2 * e + 1]);
                    *reinterpret_cast<U16x8*>(to) = w;
                } else {
                    *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
                    *reinterpret_cast<float4*>(to + 4) = make_float4(y[4], y[5], y[6], y[7]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (at(8 * g + e) < left) to[e] = static_cast<TO>(y[e]);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e)
            if (at(e) < left) dst[at(e)] = static_cast<TO>(x[e]);
    }
}

// Whether `rows` rows of a_width bytes at stride a_stride from a share bytes with
// rows of b's (columns of one buffer, at one stride, may lie between each other).
bool rows_overlap(const void* a, int64_t a_stride, int64_t a_width, const void* b,
                  int64_t b_stride, int64_t b_width, int64_t rows) {
    const int64_t x = reinterpret_cast<int64_t>(a), y = reinterpret_cast<int64_t>(b);
    if (x + (rows - 1) * a_stride + a_width <= y || y + (rows - 1) * b_stride + b_width <= x)
        return false;
    if (a_stride != b_stride) return true;
    const int64_t d = ((y - x) % a_stride + a_stride) % a_stride;
    return d < a_width || d + b_width > a_stride;
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
    TVLLM_CHECK(capacity <= INT32_MAX - 65536, "logit_controls: at most 2^31-65537 tokens of history");
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
    const int64_t unit_in = dtype == TVLLM_F32 ? 4 : 2, unit_out = out_dtype == TVLLM_F32 ? 4 : 2;
    TVLLM_CHECK(logits != out || (out_dtype == dtype && out_stride == row_stride),
                "logit_controls: in place, the output has the logits' type and rows");
    TVLLM_CHECK(logits == out || !rows_overlap(logits, row_stride * unit_in, vocab * unit_in, out,
                                               out_stride * unit_out, vocab * unit_out, rows),
                "logit_controls: the output must be the logits or not overlap them");
    Args a{};
    a.logits = logits;
    a.out = out;
    a.stride = row_stride;
    a.out_stride = out_stride;
    a.vocab = vocab;
    a.spans = (vocab + kSpan - 1) / kSpan;
    a.grid = rows * a.spans;
    a.in_place = logits == out;
    a.list4 = aligned16(history) && capacity % 4 == 0;
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
