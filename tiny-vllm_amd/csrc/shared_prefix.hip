// Decode attention for batches whose rows share a long prefix, computed once
// for all of them.
//
// For decode row r and query head h,
//   out[rows[r], h] = sum_t softmax_t(scale * q . k_t) v_t,  t < lengths[r],
// exactly as paged decode, but the first prefix_lens[g] tokens of the rows of
// group g lie in the same pages. The softmax splits over any partition X of
// the keys: with m_X = max s, l_X = sum e^(s - m_X), a_X = sum e^(s - m_X) v,
//   out = sum_X e^(m_X - m) a_X / sum_X e^(m_X - m) l_X,  m = max_X m_X,
// so a group's shared keys are one part that every query of the group takes
// from one read of K and V, and each row's own keys are others.
//
// The reference has no counterpart (its decode reads a shared page once per
// row: tinyvllm/kernels/paged_decode.cu:92-466).
//
// MI355X design:
//  * A host-side planner cuts the work into tasks - (KV head, range of keys,
//    up to 128 query vectors) for shared keys, (row, KV head, range of keys)
//    for own ones - of about equal length, 512 of them (two workgroups on each
//    of 256 CUs) where the keys allow. One launch runs them all, so the
//    compute-bound shared part and the memory-bound own parts overlap; a
//    second merges the parts of each (row, head).
//  * Wide tasks (above 16 query vectors): K/V tiles of 32 tokens in LDS, 32
//    queries per wave on the 32x32x16 MFMA: S^T = K Q^T leaves a lane with 16
//    tokens of its own query, which are the k values of its column in O^T +=
//    V^T P^T, so P never moves. V is read from LDS through the transposing
//    load, so it is staged as it lies in the cache. A step multiplies the next
//    tile's scores, works out this tile's weights and multiplies the last
//    tile's values: three chains that do not wait for each other, their
//    instructions interleaved one matrix instruction at a time (without that
//    order a step takes 1.29 times as long).
//  * Narrow tasks (up to 16 query vectors; a row's own keys at GQA groups up
//    to 16): each of four waves streams its quarter of the keys straight into
//    registers (or the waves take the KV heads of a short range), Q.K^T and P.V
//    on 16-wide MFMAs, and the waves merge in LDS.
//
// Measured on one MI355X (kernel trace; tasks + merge, bf16 and 32 / 8 heads of
// 128 if not said otherwise):
//   64 rows behind 2048 shared tokens, 64-512 own           22.8 + 4.1 us
//   256 rows behind 32768, 1-1024 own                        210 + 10.7 us
//   16 rows behind 32768, 64 / 8 heads, FP8 cache             33.6 + 8.2 us
//   own keys alone, 256 rows of 2048         6.3 TB/s (5.2 TB/s from FP8)
// What bounds them: the wide path's step, 32 tokens by 2 x 128 queries in
// 1.2 us on a CU, about 835 TFLOP/s over the card where a large matrix product
// reaches 1375. No unit is full (matrix 34 %, vector 42 %, LDS 27 % busy); left
// out one at a time, staging is 21 % of it, the products with V 23 %, with K
// 17 %, the loads 9 %, the exponentials 3 %. Short calls are bound by chains of
// dependent loads (plan, page, row) and by the second launch.
// 64 queries per wave at one workgroup per CU halve the staging and were
// slower (one wave per SIMD has nothing to run while it waits: with 32 queries
// 453 us instead of 340 for 256 rows behind 65536); so were narrow tasks ahead
// of the wide ones or between them (64 rows behind 2048: 26.2 and 26.6 us; 256
// behind 32768: 284 and 294).
#include "common.h"

#include <algorithm>
#include <type_traits>
#include <vector>

namespace tvllm {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;
constexpr int kWide = 128;    // query vectors of a wide task (32 per wave)
// Query vectors of a narrow one: one 16-wide matrix instruction takes them. A
// second pass over the keys costs more than a wide task with idle columns: 20
// vectors a KV head, 8 heads behind 4096 keys 9.6 us wide, 13.2 narrow; 32 of
// them behind 32768 31.5 and 47.7; 64 33.3 and 90.2.
constexpr int kNarrow = 16;
constexpr float kLog2e = 1.4426950408889634f;
// Running maxima of the wide path rise only when a tile's maximum exceeds them
// by more than this (log2 units), so most tiles skip the rescale.
constexpr float kSlack = 8.f;
// P enters the products as fp16: weights are carried at 2^kShift times their
// value, so that with the slack they stay below 2^15 and keep all 11 bits down
// to 2^-21 of the running maximum, a part of 2^-32 of it below.
constexpr float kShift = 7.f;

// ------------------------------------------------------------------ plan --
// int32 words: header | per row (first part, parts) | members | tasks.
constexpr int kHeader = 16;
constexpr int kTaskWords = 8;
enum Header { H_TASKS, H_ROWS, H_HEADS, H_KV_HEADS, H_DIM, H_BLOCK, H_PARTS, H_MERGE };
// A task's queries are number q_begin .. + q_count - 1 of its group's (T_QUERIES:
// q_begin / 16 above, q_count in the lower 8 bits), query i
// being head i % group (of the KV head) of row members[member + i / group]; its
// keys are tokens k0 .. k1 - 1 of the table of row T_ROW, the first of them.
// T_HEADS (1, 2 or 4; above 1 in narrow tasks only): that many KV heads from T_KVH
// on, each with its queries and keys.
enum Task { T_MEMBER, T_QUERIES, T_KVH, T_HEADS, T_K0, T_K1, T_PART, T_ROW };

constexpr int64_t kSlots = 512;     // workgroups at once: two on each of 256 CUs
constexpr int64_t kKeyUnit = 64;    // tasks' key ranges are multiples of this
constexpr int64_t kMaxParts = 64;   // splits of one unit
constexpr int64_t kMaxContext = INT32_MAX - 4096;  // token numbers past a tile's end fit in 32 bits
constexpr int64_t kMaxSplits = 1024;  // tasks that splitting adds, all units together
// What a task costs beside its keys (its chain of first loads, the merge in LDS
// and the write of its part), in keys. At 32 / 128 / 512: 64 rows behind 2048
// 24.3 / 23.7 / 24.1 us, 49 rows in 6 groups 41.6 / 38.3 / 37.8, 256 rows behind
// 512 20.0 / 20.1 / 21.6.
constexpr int64_t kTaskCost = 128;
// Contexts (at head dims up to 128) and keys of all units up to which rows are
// not cut at all (see below).
constexpr int64_t kDirectKeys = 640;
constexpr int64_t kDirectTotal = 1 << 17;

struct PlanLayout {
    int64_t rows_at, members_at, tasks_at, max_tasks, words;
};

PlanLayout plan_layout(int64_t max_rows, int64_t heads, int64_t kv_heads) {
    const int64_t group = heads / kv_heads;
    PlanLayout p;
    // Every unit (KV head, tile of queries) of keys K makes at most K / chunk
    // + 1 tasks, and chunk >= all units' keys / kMaxSplits.
    const int64_t own = max_rows * ((group + kWide - 1) / kWide);
    const int64_t shared = (max_rows * group + kWide - 1) / kWide + max_rows / 2;
    p.max_tasks = kMaxSplits + kv_heads * (own + shared);
    p.rows_at = kHeader;
    p.members_at = p.rows_at + 2 * max_rows;
    p.tasks_at = p.members_at + max_rows;
    p.words = p.tasks_at + kTaskWords * p.max_tasks;
    return p;
}

// (row part, query head) results of one call at most: a unit of q queries and
// K keys makes q (K / chunk + 1) of them.
int64_t max_entries(int64_t max_rows, int64_t heads) {
    return 2 * max_rows * heads + kWide * kMaxSplits;
}

// ---------------------------------------------------------------- device --

template <typename T>
struct Args {
    const T* q;
    int64_t qts, qhs;
    const void* k;  // cache rows: T elements, or FP8 E4M3 bytes
    const void* v;
    int64_t css, chs;  // cache slot / head strides (elements)
    T* out;
    int64_t ots, ohs;
    const int64_t* rows;
    const int64_t* blocks;
    const int64_t* offsets;
    const int32_t* plan;
    int rows_at, members_at, tasks_at;
    int num_rows, heads, kv_heads, group, head_dim, block_size;
    uint32_t page_mul;  // t / block_size == (2 t * page_mul >> 32) >> page_shift, t < 2^31
    int page_shift;
    float scale_log2;  // softmax scale * log2(e) (* k_scale for an FP8 cache)
    float v_scale;     // FP8 cache: V dequantisation scale (1 otherwise)
    float* part_o;     // [entries][head_dim], unnormalised
    float2* part_ml;   // [entries]: (max, sum) in base 2
    int64_t entries;   // room in the two
};

// Asks for the 64-byte lines that the arguments lie in, all at once.
template <typename T>
__device__ __forceinline__ void touch(const Args<T>& a) {
    asm volatile("" ::"s"(a.q), "s"(a.plan), "s"(a.entries));
}

// The plan's header, in one load, and whether the call is what it was made for.
struct PlanHead {
    int32_t w[8];
    template <typename T>
    __device__ bool fits(const Args<T>& a) const {
        return (w[H_ROWS] == a.num_rows) & (w[H_HEADS] == a.heads) &
               (w[H_KV_HEADS] == a.kv_heads) & (w[H_DIM] == a.head_dim) &
               (w[H_BLOCK] == a.block_size) & (w[H_PARTS] <= a.entries) &
               (w[H_MERGE] <= (a.part_o != nullptr));
    }
};
__device__ __forceinline__ PlanHead load_head(const int32_t* plan) {
    PlanHead h;
    const int4 lo = *reinterpret_cast<const int4*>(plan);
    const int4 hi = *reinterpret_cast<const int4*>(plan + 4);
    h.w[0] = lo.x;
    h.w[1] = lo.y;
    h.w[2] = lo.z;
    h.w[3] = lo.w;
    h.w[4] = hi.x;
    h.w[5] = hi.y;
    h.w[6] = hi.z;
    h.w[7] = hi.w;
    return h;
}

template <int I, int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<I + 1, N>(f);
    }
}

__device__ __forceinline__ float as_f(uint32_t x) { return __uint_as_float(x); }
__device__ __forceinline__ uint32_t as_u(float x) { return __float_as_uint(x); }

// D[32x32] += A[32x16] B[16x32]. Lane l: A row l%32 and B column l%32 with
// k = 8*(l/32)..+7; D column l%32, rows 8*(v/4) + 4*(l/32) + v%4 for v < 16.
template <typename T>
__device__ __forceinline__ f32x16 mfma_32x32x16(const U16x8& a, const U16x8& b, f32x16 c) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    if constexpr (std::is_same_v<T, __bf16>) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(t8, a),
                                                       __builtin_bit_cast(t8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(t8, a),
                                                      __builtin_bit_cast(t8, b), c, 0, 0, 0);
    }
}

// D[16x16] += A[16x16] B[16x16]: lane l supplies A row l%16 and B column l%16
// with k = 4*(l/16)..+3; D column l%16, rows 4*(l/16) + v.
template <typename T>
__device__ __forceinline__ f32x4 mfma_16x16x16(uint2 a, uint2 b, f32x4 c) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    if constexpr (std::is_same_v<T, __bf16>) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(
            __builtin_bit_cast(s4, a), __builtin_bit_cast(s4, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(
            __builtin_bit_cast(h4, a), __builtin_bit_cast(h4, b), c, 0, 0, 0);
    }
}

// Transposing LDS read: lanes 16b + 4r + c of each 16-lane block b point at 4
// consecutive 16-bit elements, row r, columns 4c..4c+3 of a 4 x 16 block; lane
// 16b + x gets column x, rows 0..3.
__device__ __forceinline__ uint2 read_transposed(const uint16_t* p) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    return __builtin_bit_cast(
        uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                   (lds_s4*)(const __attribute__((address_space(3))) uint16_t*)p));
}

// Lanes l and l + 32 hold the same query: combine them with one row swap.
__device__ __forceinline__ float pair_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(as_u(x), as_u(x), false, false);
    return fmaxf(as_f(r[0]), as_f(r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(as_u(x), as_u(x), false, false);
    return as_f(r[0]) + as_f(r[1]);
}

// N bytes from memory as they lie there. STREAM: lines that an instruction takes
// whole and nobody else reads go past the caches (V of the narrow path; where an
// instruction takes half a line of each row, the other half would be fetched
// again: own keys of 256 rows x 2048, 375 us with K through the caches, 401 past
// them).
template <int N>
struct Bytes {
    uint32_t w[(N + 3) / 4];
};

template <int N, bool STREAM>
__device__ __forceinline__ Bytes<N> load_bytes(const char* p) {
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    Bytes<N> r;
    if constexpr (!STREAM) {
        if constexpr (N == 16) {
            const u4 t = *reinterpret_cast<const u4*>(p);
            r.w[0] = t[0];
            r.w[1] = t[1];
            r.w[2] = t[2];
            r.w[3] = t[3];
        } else {
            static_assert(N == 8);
            const u2 t = *reinterpret_cast<const u2*>(p);
            r.w[0] = t[0];
            r.w[1] = t[1];
        }
    } else if constexpr (N == 2) {
        r.w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint16_t*>(p));
    } else if constexpr (N == 4) {
        r.w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
    } else if constexpr (N == 8) {
        const u2 t = __builtin_nontemporal_load(reinterpret_cast<const u2*>(p));
        r.w[0] = t[0];
        r.w[1] = t[1];
    } else {
        static_assert(N == 16);
        const u4 t = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p));
        r.w[0] = t[0];
        r.w[1] = t[1];
        r.w[2] = t[2];
        r.w[3] = t[3];
    }
    return r;
}

// Two E4M3 bytes (the low or high half of w) -> two T elements, exact.
template <typename T, bool HI>
__device__ __forceinline__ uint32_t widen2(uint32_t w) {
    if constexpr (std::is_same_v<T, __bf16>) {
        return __builtin_bit_cast(uint32_t,
                                  __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HI));
    } else {
        return __builtin_bit_cast(uint32_t,
                                  __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HI));
    }
}

// The order of a wide step's instructions: the first operands from LDS, the
// weights' arithmetic, then one matrix instruction at a time, each followed by
// the read of the operand four further on and a share of the vector work.
// Without it the compiler puts each read right before the instruction that
// waits for it (a step takes 1.29 times as long). Vector instructions ahead of
// the first matrix one, 256 rows behind 32768: 1 218 us, 8 212, 12 210, 20 215,
// 30 214; per matrix instruction 4 213, 5 and 6 210.
template <int NC, int ND>
__device__ __forceinline__ void interleave() {
    constexpr int kValu = 0x2, kMfma = 0x8, kRead = 0x100;
    constexpr int kAll = NC + 2 * ND, kAhead = 4;  // operands: K one read each, V two
    static_for<0, kAhead>([&](auto m) {
        __builtin_amdgcn_sched_group_barrier(kRead, m < NC ? 1 : 2, 0);
    });
    __builtin_amdgcn_sched_group_barrier(kValu, 12, 0);
    static_for<0, kAll>([&](auto m) {
        __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
        if constexpr (m + kAhead < kAll)
            __builtin_amdgcn_sched_group_barrier(kRead, m + kAhead < NC ? 1 : 2, 0);
        __builtin_amdgcn_sched_group_barrier(kValu, 5, 0);
    });
}

template <typename T, int DP, bool F8>
__global__ void __launch_bounds__(kThreads, DP == 256 ? 1 : 2)
shared_prefix_tasks(Args<T> a) {
    constexpr int EB = F8 ? 1 : 2;             // bytes per cached element
    constexpr int BK = 32;                     // tokens per wide tile
    constexpr int K_LD = DP + 8;               // LDS row strides (elements): 16-byte reads
    constexpr int V_LD = DP == 32 ? 32 : DP + 32;  // and transposing reads without conflicts
    constexpr int K_TILE = BK * K_LD, V_TILE = BK * V_LD;
    constexpr int kTileBytes = 2 * 2 * (K_TILE + V_TILE);
    constexpr int kMergeBytes = 4 * kNarrow * (4 * DP + 8);
    __shared__ __align__(16) char lds[kTileBytes > kMergeBytes ? kTileBytes : kMergeBytes];
    __shared__ int2 spots[kWide];

    // A chain of loads leads to the keys: the plan's header and the task, the
    // row's offset, its pages, their rows. What can goes out together (the plan
    // holds max_tasks tasks whatever the header says).
    const int32_t* const plan = a.plan;
    const int32_t* const task = plan + a.tasks_at + int64_t(blockIdx.x) * kTaskWords;
    const int t_member = task[T_MEMBER], t_queries = task[T_QUERIES], kvh = task[T_KVH];
    const int t_heads = task[T_HEADS], k0 = task[T_K0], k1 = task[T_K1];
    const int part = task[T_PART], t_row = task[T_ROW];
    const PlanHead head = load_head(plan);
    asm volatile("" ::"s"(t_member), "s"(t_queries), "s"(kvh), "s"(t_heads), "s"(k0), "s"(k1),
                 "s"(part), "s"(t_row), "s"(head.w[0]), "s"(head.w[7]));
    if (int(blockIdx.x) >= head.w[H_TASKS] || !head.fits(a)) return;
    const int32_t* const members = plan + a.members_at + t_member;
    const int q_begin = (t_queries >> 8) * kNarrow, q_count = t_queries & 0xff;
    const int D = a.head_dim;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t table = a.offsets[t_row];
    const uint32_t* const ids = reinterpret_cast<const uint32_t*>(a.blocks + table);
    const uint32_t row_bytes = uint32_t(a.css * EB);
    const char* const kbase = static_cast<const char*>(a.k) + int64_t(kvh) * a.chs * EB;
    const char* const vbase = static_cast<const char*>(a.v) + int64_t(kvh) * a.chs * EB;

    auto page_of = [&](uint32_t t) { return __umulhi(2 * t, a.page_mul) >> a.page_shift; };
    auto slot_of = [&](uint32_t id, uint32_t t, uint32_t page) {
        return id * uint32_t(a.block_size) + (t - page * uint32_t(a.block_size));
    };
    // Query i of the task, of KV head kvh + x: its row, and its head.
    auto query = [&](int i, int x, int& row, int& head) {
        const int g = (q_begin + i) / a.group;
        row = members[g];
        head = (kvh + x) * a.group + (q_begin + i - g * a.group);
    };
    // Where a row's part goes: (first part, parts) of the row, looked up ahead
    // and kept in LDS. Rows of one part are written to the output.
    auto spot_of = [&](int row) {
        return *reinterpret_cast<const int2*>(plan + a.rows_at + 2 * row);
    };
    auto entry_of = [&](int2 spot, int head, bool& direct) -> int64_t {
        direct = spot.y == 1;
        return (int64_t(spot.x) + part) * a.heads + head;
    };

    // ------------------------------------------------------------- wide --
    // Returns whether the outputs are not what fp16 V can give (see below).
    auto wide = [&]() -> bool {
        constexpr int PPR = DP / 8;  // 8-element pieces per row
        constexpr int NC = DP / 16, ND = DP / 32;
        constexpr int EBP = 8 * EB;
        // A bf16 cache's V enters the products as fp16 (P needs its 11 bits: a
        // bf16 P is 2^-9 off, as much as the output's own rounding). That is
        // exact below 65536 in magnitude, to 2^-25 below 2^-14; beyond, the
        // outputs it reaches end non-finite and the task is done again by the
        // narrow path, which takes V as it is.
        constexpr bool kConvert = std::is_same_v<T, __bf16> && !F8;
        uint16_t* const ks = reinterpret_cast<uint16_t*>(lds);
        uint16_t* const vs = ks + 2 * K_TILE;
        const int col = lane & 31, half = lane >> 5;
        // Waves past the queries take the last one along: a second path through
        // the loop for them would make the others wait for its loads.
        const int qi = wave * 32 + col;
        U16x8 qv[NC];
        const int ntiles = (k1 - k0 + BK - 1) / BK;
        const uint32_t last = uint32_t(k1 - 1);
        // Staging: LPR lanes side by side load a row's whole 128-byte lines
        // (its first 64 bytes where it has fewer), each thread PT pieces of each
        // of its JT tokens, so a page is looked up once for those. Two sets of
        // registers, a tile each: rows are loaded two tiles ahead of the step
        // that stores them in LDS.
        constexpr int LPR = PPR < 8 ? PPR : 8;
        constexpr int TSTEP = kThreads / LPR;  // tokens that one round covers
        constexpr int JT = BK > TSTEP ? BK / TSTEP : 1, PT = PPR / LPR;
        const int tok0 = tid / LPR, piece0 = tid % LPR;
        struct Stage {
            Bytes<EBP> k[JT][PT], v[JT][PT];
            uint64_t off[JT];
        };
        Stage st0, st1;
        uint32_t id[JT];
        auto token_of = [&](int i, int j) {  // past the end: the last token again
            return min(uint32_t(k0 + i * BK + tok0 + j * TSTEP), last);
        };
        auto load_ids = [&](uint32_t (&id)[JT], int i) {
#pragma unroll
            for (int j = 0; j < JT; ++j) id[j] = ids[2 * uint64_t(page_of(token_of(i, j)))];
        };
        auto locate = [&](uint64_t (&off)[JT], const uint32_t (&id)[JT], int i) {  // tile i's rows
#pragma unroll
            for (int j = 0; j < JT; ++j) {
                const uint32_t t = token_of(i, j);
                off[j] = uint64_t(slot_of(id[j], t, page_of(t))) * row_bytes;
            }
        };
        auto load = [&](Bytes<EBP> (&to)[JT][PT], const uint64_t (&off)[JT], const char* base) {
#pragma unroll
            for (int j = 0; j < JT; ++j)
#pragma unroll
                for (int x = 0; x < PT; ++x) {
                    const int d = 8 * (piece0 + LPR * x);
                    to[j][x] = load_bytes<EBP, false>(base + off[j] + (d < D ? d : 0) * EB);
                }
        };
        // Rows past the end and dims past the head's are zeros in LDS.
        auto trim = [&](Bytes<EBP> (&to)[JT][PT], int i) {
            const int left = k1 - k0 - i * BK;
            if (left < BK || D < DP) {
                asm volatile("");  // (rare: a branch, not selects)
#pragma unroll
                for (int j = 0; j < JT; ++j)
#pragma unroll
                    for (int x = 0; x < PT; ++x)
                        if (tok0 + j * TSTEP >= left || 8 * (piece0 + LPR * x) >= D)
                            to[j][x] = Bytes<EBP>{};
            }
        };
        auto store_k = [&](const Bytes<EBP> (&k)[JT][PT], int i) {
            uint16_t* const kt = ks + (i & 1) * K_TILE;
            if (TSTEP > BK && tok0 >= BK) return;
#pragma unroll
            for (int j = 0; j < JT; ++j)
#pragma unroll
                for (int x = 0; x < PT; ++x) {
                    U16x8 w8;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        if constexpr (F8)
                            w8.w[w] = (w & 1) ? widen2<T, true>(k[j][x].w[w >> 1])
                                              : widen2<T, false>(k[j][x].w[w >> 1]);
                        else
                            w8.w[w] = k[j][x].w[w];
                    }
                    *reinterpret_cast<U16x8*>(kt + (tok0 + j * TSTEP) * K_LD +
                                              8 * (piece0 + LPR * x)) = w8;
                }
        };
        auto store_v = [&](const Bytes<EBP> (&v)[JT][PT], int i) {
            uint16_t* const vt = vs + (i & 1) * V_TILE;
            if (TSTEP > BK && tok0 >= BK) return;
#pragma unroll
            for (int j = 0; j < JT; ++j)
#pragma unroll
                for (int x = 0; x < PT; ++x) {
                    U16x8 w8;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        if constexpr (F8)
                            w8.w[w] = (w & 1) ? widen2<_Float16, true>(v[j][x].w[w >> 1])
                                              : widen2<_Float16, false>(v[j][x].w[w >> 1]);
                        else if constexpr (kConvert)
                            w8.w[w] = pack2<_Float16>(half_lo<T>(v[j][x].w[w]),
                                                      half_hi<T>(v[j][x].w[w]));
                        else
                            w8.w[w] = v[j][x].w[w];
                    }
                    *reinterpret_cast<U16x8*>(vt + (tok0 + j * TSTEP) * V_LD +
                                              8 * (piece0 + LPR * x)) = w8;
                }
        };

        f32x16 o[ND];  // O^T: lane = (dims 32n + 8g + 4*half + i, query col)
#pragma unroll
        for (int n = 0; n < ND; ++n) o[n] = f32x16{};
        float m_run = -INFINITY, l_run = 0.f;
        // Weights of the last tile, not yet multiplied with its V (two sets: a
        // step reads one and writes the other): step s's token 16s + 8jj +
        // 4*half + i at k = 4jj + i.
        U16x8 pa[2] = {}, pb[2];
        // S^T of a tile: token 8(v/4) + 4*half + v%4 of the lane's query.
        auto scores = [&](int i, f32x16& sc) {
            const uint16_t* const kt = ks + (i & 1) * K_TILE + col * K_LD + 8 * half;
            sc = f32x16{};
#pragma unroll
            for (int c = 0; c < NC; ++c)
                sc = mfma_32x32x16<T>(*reinterpret_cast<const U16x8*>(kt + 16 * c), qv[c], sc);
        };
        const int vlane = (4 * half + ((lane & 15) >> 2)) * V_LD + 16 * ((lane >> 4) & 1) +
                          4 * (lane & 3);
        auto values = [&](int i, const U16x8 (&p)[2]) {  // O^T += V^T P^T of tile i
            const uint16_t* const vt = vs + (i & 1) * V_TILE + vlane;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int n = 0; n < ND; ++n) {
                    const uint2 lo = read_transposed(vt + (16 * s) * V_LD + 32 * n);
                    const uint2 hi = read_transposed(vt + (16 * s + 8) * V_LD + 32 * n);
                    const U16x8 va = {{lo.x, lo.y, hi.x, hi.y}};
                    o[n] = mfma_32x32x16<_Float16>(va, p[s], o[n]);
                }
        };
        // Step i. LDS holds K of two tiles and V of two: K of i + 1 is read while
        // K of i + 2 is written (over i's), V of i - 1 read and V of i written
        // (over i - 2's).
        // Loads come back in order, so the ids go out ahead of the rows: the next
        // step waits for them and not for rows.
        auto stage = [&](Stage& st, int i) {
            store_k(st.k, i + 2);
            store_v(st.v, i);
            uint64_t voff[JT];
#pragma unroll
            for (int j = 0; j < JT; ++j) voff[j] = st.off[j];  // tile i + 2's rows
            locate(st.off, id, i + 4);
            load_ids(id, i + 5);
            load(st.v, voff, vbase);
            load(st.k, st.off, kbase);
        };
        // The scores of the next tile, the weights of this one and the products
        // of the last one have nothing to wait for in each other, so the matrix
        // cores work while the vector units do.
        float cm;  // the tile's maximum score of the lane's query, in base-2 units
        auto maximum = [&](const f32x16& sc) {
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int v = 0; v < 16; ++v) mx[v & 1] = fmaxf(mx[v & 1], sc[v]);
            return pair_max(fmaxf(mx[0], mx[1])) * a.scale_log2;
        };
        auto step = [&](Stage& st, int i, f32x16& sc, f32x16& next, U16x8 (&pl)[2],
                        U16x8 (&pn)[2]) {
            __syncthreads();
            trim(st.k, i + 2);
            trim(st.v, i);
            const int left = k1 - k0 - i * BK;
            if (left < BK) {
                asm volatile("");  // a branch, not selects
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    if (8 * (v >> 2) + 4 * half + (v & 3) >= left) sc[v] = -INFINITY;
                cm = maximum(sc);
            }
            const bool grow = cm > m_run + kSlack;  // also: a first finite maximum
            if (i == 0) {  // (nothing to rescale yet)
                m_run = cm;
            } else if (__builtin_amdgcn_ballot_w64(grow)) {
                values(i - 1, pl);  // at the old maximum
                pl[0] = pl[1] = U16x8{};
                const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - cm) : 1.f;
                m_run = grow ? cm : m_run;
                l_run *= alpha;
#pragma unroll
                for (int n = 0; n < ND; ++n) o[n] *= alpha;
            }
            // What follows stays one block: weights worked out in the arms of the
            // branch above, or put off to the next step, which uses them, would
            // not run beside the products.
            asm volatile("" : "+v"(m_run));
            scores(i + 1, next);
            const float m_use = m_run == -INFINITY ? 0.f : m_run - kShift;
            float ps[2] = {0.f, 0.f};
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p0 = __builtin_amdgcn_exp2f(
                        __builtin_fmaf(sc[8 * s + 2 * e], a.scale_log2, -m_use));
                    const float p1 = __builtin_amdgcn_exp2f(
                        __builtin_fmaf(sc[8 * s + 2 * e + 1], a.scale_log2, -m_use));
                    const uint32_t hw = pack2<_Float16>(p0, p1);
                    pn[s].w[e] = hw;
                    // The denominator sums the fp16 weights that P.V uses.
                    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                    const h2 ones = {1.f16, 1.f16};
                    ps[s] = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, hw), ones, ps[s], false);
                }
            l_run += ps[0] + ps[1];
            values(i - 1, pl);
            stage(st, i);
            cm = maximum(next);
#pragma unroll
            for (int w = 0; w < 4; ++w) asm volatile("" : "+v"(pn[0].w[w]), "+v"(pn[1].w[w]));
            asm volatile("" : "+v"(cm), "+v"(l_run));
            interleave<NC, ND>();
        };

        // Everything the first steps need goes out before anything is waited for,
        // in the order in which it is needed (the loop's waits count on what is
        // behind a load on every way in).
        f32x16 sa, sb;
        {
            auto keep_order = []() { __builtin_amdgcn_sched_barrier(0); };
            uint32_t id0[JT], id1[JT], id2[JT], id3[JT];
            uint64_t off0[JT], off1[JT];
            Bytes<EBP> first[JT][PT], second[JT][PT];
            load_ids(id0, 0);
            load_ids(id1, 1);
            load_ids(id2, 2);
            load_ids(id3, 3);
            load_ids(id, 4);
            int row, head;
            query(min(qi, q_count - 1), 0, row, head);
            keep_order();
            const int64_t qtoken = a.rows[row];
            const int2 spot = spot_of(row);
            locate(off0, id0, 0);
            locate(off1, id1, 1);
            locate(st0.off, id2, 2);
            locate(st1.off, id3, 3);
            keep_order();
            load(first, off0, kbase);
            load(second, off1, kbase);
            keep_order();
            const T* const qrow = a.q + qtoken * a.qts + head * a.qhs;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int d = 16 * c + 8 * half;
                qv[c] = d < D ? *reinterpret_cast<const U16x8*>(qrow + d) : U16x8{};
            }
            keep_order();
            load(st0.v, off0, vbase);
            load(st0.k, st0.off, kbase);
            keep_order();
            load(st1.v, off1, vbase);
            load(st1.k, st1.off, kbase);
            keep_order();
            // Step 0 multiplies what stands in place of tile -1's V with weights
            // of 0: zeros, as LDS may hold NaNs.
            for (int x = tid; x < V_TILE / 8; x += kThreads)
                reinterpret_cast<U16x8*>(vs + V_TILE)[x] = U16x8{};
            if (half == 0) spots[qi] = spot;
            trim(first, 0);
            store_k(first, 0);
            trim(second, 1);
            store_k(second, 1);
        }
        __syncthreads();
        scores(0, sa);
        cm = maximum(sa);
        // Two steps a round, the second past the end where the tiles are odd in
        // number (its weights are 0): a way around it would lead the loop's
        // waits to expect the first one's loads at once.
        const int steps = (ntiles + 1) & ~1;
        for (int i = 0; i < steps; i += 2) {
            step(st0, i, sa, sb, pa, pb);
            step(st1, i + 1, sb, sa, pb, pa);
        }
        __syncthreads();  // V of the last tile
        values(steps - 1, pa);

        bool again = false;
        if constexpr (kConvert) {
            float total = 0.f;  // inf or NaN if any accumulator is
#pragma unroll
            for (int n = 0; n < ND; ++n)
#pragma unroll
                for (int v = 0; v < 16; ++v) total += o[n][v];
            again = !(__builtin_fabsf(total) < INFINITY);
        }
        // Every wave is past its reads of LDS behind this.
        if (__syncthreads_or(again)) return true;
        const float l = pair_sum(l_run);
        if (qi >= q_count) return false;
        int row, head;
        query(qi, 0, row, head);
        bool direct;
        const int64_t entry = entry_of(spots[qi], head, direct);
        if (direct) {
            const float inv = a.v_scale / l;
            T* orow = a.out + a.rows[row] * a.ots + head * a.ohs + 4 * half;
#pragma unroll
            for (int n = 0; n < ND; ++n)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    if (32 * n + 8 * g < D) {
                        uint2 w;
                        w.x = pack2<T>(o[n][4 * g] * inv, o[n][4 * g + 1] * inv);
                        w.y = pack2<T>(o[n][4 * g + 2] * inv, o[n][4 * g + 3] * inv);
                        *reinterpret_cast<uint2*>(orow + 32 * n + 8 * g) = w;
                    }
        } else {
            float* prow = a.part_o + entry * D + 4 * half;
#pragma unroll
            for (int n = 0; n < ND; ++n)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    if (32 * n + 8 * g < D)
                        *reinterpret_cast<float4*>(prow + 32 * n + 8 * g) = make_float4(
                            o[n][4 * g], o[n][4 * g + 1], o[n][4 * g + 2], o[n][4 * g + 3]);
            if (half == 0)
                a.part_ml[entry] =
                    make_float2(m_run == -INFINITY ? m_run : m_run - kShift, l);
        }
        return false;
    };

    // ----------------------------------------------------------- narrow --
    // Queries q0 .. q0 + qn - 1 (qn <= 16) of the task over its keys.
    auto narrow = [&](int q0, int qn) {
        // 16-token tiles per chunk: 16 KB of K and V in flight per wave
        constexpr int NT = DP == 256 ? 1 : DP == 128 ? (F8 ? 4 : 2) : 4;
        constexpr int CH = 16 * NT;
        constexpr int KS = DP / 32;            // k-steps of Q.K^T
        constexpr int E = DP / 16;             // V elements per lane and token
        constexpr int VL = DP == 256 ? 2 : 1;  // loads that hold them
        constexpr int VB = E * EB / VL;        // bytes of one
        // A thread id of its own: nothing derived from it is worked out ahead of
        // the wide path, whose registers it would take.
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
        const int col = lane & 15, quad = lane >> 4;
        f32x4 acc[E];  // query 4*quad + v, this lane's dim e
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m_run = -INFINITY, l_run = 0.f;

        // The waves of a head take its keys in equal, consecutive shares.
        const int heads = t_heads, shares = 4 / heads;
        const int x = wave / shares;  // this wave's KV head, of the task's
        const char* const kbase = static_cast<const char*>(a.k) + int64_t(kvh + x) * a.chs * EB;
        const char* const vbase = static_cast<const char*>(a.v) + int64_t(kvh + x) * a.chs * EB;
        int2 spot;  // wave 0, which always has keys: where its lanes' results go
        const int per = ((k1 - k0 + shares - 1) / shares + 15) & ~15;
        const int t_begin = k0 + (wave - x * shares) * per, t_end = min(k1, t_begin + per);
        if (t_begin < t_end) {
            // This lane's dims: E * col .. (DP 256: 8 * col .. and 128 + 8 * col ..);
            // lanes past the head's dims read dim 0 and write nothing.
            auto dim_of = [&](int half) { return DP == 256 ? 128 * half + 8 * col : E * col; };
            Bytes<8 * EB> kreg[NT][KS];
            Bytes<VB> vreg[NT][4][VL];
            const uint32_t last = uint32_t(t_end - 1);
            auto load_id = [&](int t0) {
                return ids[2 * uint64_t(page_of(min(uint32_t(t0 + lane % CH), last)))];
            };
            auto resolve = [&](int t0, uint32_t id) {
                const uint32_t t = min(uint32_t(t0 + lane % CH), last);
                return slot_of(id, t, page_of(t));
            };
            auto load_k = [&](uint32_t slot) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const uint32_t s = uint32_t(__shfl(int(slot), 16 * j + col, 64));
                    const char* p = kbase + uint64_t(s) * row_bytes;
#pragma unroll
                    for (int c = 0; c < KS; ++c) {
                        const int d = 32 * c + 8 * quad;
                        kreg[j][c] = load_bytes<8 * EB, false>(p + (d < D ? d : 0) * EB);
                    }
                }
            };
            auto load_v = [&](uint32_t slot) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t s = uint32_t(__shfl(int(slot), 16 * j + 4 * quad + i, 64));
                        const char* p = vbase + uint64_t(s) * row_bytes;
#pragma unroll
                        for (int x = 0; x < VL; ++x) {
                            const int d = dim_of(x);
                            vreg[j][i][x] = load_bytes<VB, true>(p + (d < D ? d : 0) * EB);
                        }
                    }
            };

            uint32_t id = load_id(t_begin);
            uint32_t id2 = load_id(t_begin + CH);
            U16x8 qb[KS];  // B operand: query col, dims 32c + 8*quad ..
            {
                int row, head;
                query(q0 + min(col, qn - 1), x, row, head);
                if (wave == 0 && lane < heads * qn) {
                    int r, h;
                    query(q0 + lane % qn, 0, r, h);
                    spot = spot_of(r);
                }
                const T* qrow = a.q + a.rows[row] * a.qts + head * a.qhs;
#pragma unroll
                for (int c = 0; c < KS; ++c) {
                    const int d = 32 * c + 8 * quad;
                    qb[c] = d < D ? *reinterpret_cast<const U16x8*>(qrow + d) : U16x8{};
                }
            }
            {
                const uint32_t slot = resolve(t_begin, id);
                id = id2;
                load_k(slot);
                load_v(slot);
            }
            for (int t0 = t_begin; t0 < t_end; t0 += CH) {
                const uint32_t next = resolve(t0 + CH, id);
                id = load_id(t0 + 2 * CH);

                float s[NT][4];  // token 16j + 4*quad + i, query col
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < KS; ++c) {
                        U16x8 kk;
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            if constexpr (F8)
                                kk.w[w] = (w & 1) ? widen2<T, true>(kreg[j][c].w[w >> 1])
                                                  : widen2<T, false>(kreg[j][c].w[w >> 1]);
                            else
                                kk.w[w] = kreg[j][c].w[w];
                        }
                        // Dims past the head's: zeros on both sides.
                        if (D < DP && 32 * c + 8 * quad >= D) kk = U16x8{};
                        d = mfma32<T>(kk, qb[c], d);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[j][i] = d[i] * a.scale_log2;
                }
                load_k(next);
                if (t0 + CH > t_end) {
                    asm volatile("");  // a branch, not selects
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (t0 + 16 * j + 4 * quad + i >= t_end) s[j][i] = -INFINITY;
                }

                float cmax = -INFINITY;
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) cmax = fmaxf(cmax, s[j][i]);
                cmax = fmaxf(cmax, __shfl_xor(cmax, 16, 64));
                cmax = fmaxf(cmax, __shfl_xor(cmax, 32, 64));
                const float m_new = fmaxf(m_run, cmax);
                const float m_use = m_new == -INFINITY ? 0.f : m_new;
                const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
                m_run = m_new;
                float pw[NT][4];
                float psum = 0.f;
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        pw[j][i] = __builtin_amdgcn_exp2f(s[j][i] - m_use);
                        psum += pw[j][i];
                    }
                l_run = l_run * alpha + psum;
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const float av = __shfl(alpha, 4 * quad + v, 64);
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[e][v] *= av;
                }
                // Rows past the end hold the last token again: their weight is
                // 0, but 0 * inf is not.
                if (t0 + CH > t_end) {
                    asm volatile("");
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (t0 + 16 * j + 4 * quad + i >= t_end)
#pragma unroll
                                for (int x = 0; x < VL; ++x) vreg[j][i][x] = Bytes<VB>{};
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    // P as a rounded value and its rounded remainder: 16 bits of
                    // it in bf16, 22 in fp16 (weights from 2^-14 of the largest).
                    uint2 pa, pl;
                    pa.x = pack2<T>(pw[j][0], pw[j][1]);
                    pa.y = pack2<T>(pw[j][2], pw[j][3]);
                    pl.x = pack2<T>(pw[j][0] - half_lo<T>(pa.x), pw[j][1] - half_hi<T>(pa.x));
                    pl.y = pack2<T>(pw[j][2] - half_lo<T>(pa.y), pw[j][3] - half_hi<T>(pa.y));
                    uint32_t vw[4][E / 2];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int w = 0; w < E / 2; ++w) {
                            constexpr int WPL = E / 2 / VL;  // T words per load
                            const Bytes<VB>& b = vreg[j][i][w / WPL];
                            if constexpr (F8)
                                vw[i][w] = (w & 1) ? widen2<T, true>(b.w[(w % WPL) >> 1])
                                                   : widen2<T, false>(b.w[(w % WPL) >> 1]);
                            else
                                vw[i][w] = b.w[w % WPL];
                        }
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const uint32_t sel = (e & 1) ? 0x07060302u : 0x05040100u;
                        uint2 vb;  // element e of tokens 4*quad + 0..3
                        vb.x = __builtin_amdgcn_perm(vw[1][e >> 1], vw[0][e >> 1], sel);
                        vb.y = __builtin_amdgcn_perm(vw[3][e >> 1], vw[2][e >> 1], sel);
                        acc[e] = mfma_16x16x16<T>(pl, vb, acc[e]);
                        acc[e] = mfma_16x16x16<T>(pa, vb, acc[e]);
                    }
                }
                load_v(next);
            }
        }
        l_run += __shfl_xor(l_run, 16, 64);
        l_run += __shfl_xor(l_run, 32, 64);

        // The waves' parts, merged through LDS.
        float* const so = reinterpret_cast<float*>(lds);                 // [4][16][DP]
        float2* const sml = reinterpret_cast<float2*>(so + 4 * kNarrow * DP);  // [4][16]
        __syncthreads();  // a repeated call: the last one's reads are done
        if (quad == 0) sml[wave * kNarrow + col] = make_float2(m_run, l_run);
        if (wave == 0 && lane < heads * qn) spots[lane] = spot;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int h = 4 * quad + v;
            if (h < qn) {
                float* dst = so + (wave * kNarrow + h) * DP;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int d = DP == 256 ? 128 * (e / 8) + 8 * col + e % 8 : E * col + e;
                    dst[d] = acc[e][v];
                }
            }
        }
        __syncthreads();
        constexpr int Q4 = DP / 4;
        for (int i = tid; i < heads * qn * Q4; i += kThreads) {
            const int y = i / (qn * Q4), h = i / Q4 - y * qn, d = 4 * (i % Q4);
            if (d >= D) continue;
            const int w0 = y * shares;  // the first of the head's waves
            float mx = -INFINITY;
            for (int w = w0; w < w0 + shares; ++w) mx = fmaxf(mx, sml[w * kNarrow + h].x);
            const float m_use = mx == -INFINITY ? 0.f : mx;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            float l = 0.f;
            for (int w = w0; w < w0 + shares; ++w) {
                const float2 ml = sml[w * kNarrow + h];
                const float f = __builtin_amdgcn_exp2f(ml.x - m_use);
                const float4 p = *reinterpret_cast<const float4*>(so + (w * kNarrow + h) * DP + d);
                l += f * ml.y;
                sum.x += f * p.x;
                sum.y += f * p.y;
                sum.z += f * p.z;
                sum.w += f * p.w;
            }
            int row, head;
            query(q0 + h, y, row, head);
            bool direct;
            const int64_t entry = entry_of(spots[y * qn + h], head, direct);
            if (direct) {
                const float inv = a.v_scale / l;
                uint2 w;
                w.x = pack2<T>(sum.x * inv, sum.y * inv);
                w.y = pack2<T>(sum.z * inv, sum.w * inv);
                *reinterpret_cast<uint2*>(a.out + a.rows[row] * a.ots + head * a.ohs + d) = w;
            } else {
                *reinterpret_cast<float4*>(a.part_o + entry * D + d) = sum;
                if (d == 0) a.part_ml[entry] = make_float2(mx, l);
            }
        }
    };

    if (q_count > kNarrow && !wide()) return;
    for (int q0 = 0; q0 < q_count; q0 += kNarrow) narrow(q0, min(kNarrow, q_count - q0));
}

// out = v_scale * sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over the parts
// of a (row, head); rows without keys are zeros, rows of one part are already
// written. A wave each: DP / 4 lanes hold a part's dims, so 64 / (DP / 4)
// parts load at once, eight rounds of them ahead of their use, and lane s
// holds the (max, sum) of part s.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads)
shared_prefix_merge(Args<T> a) {
    constexpr int LPH = DP / 4, PAR = 64 / LPH, B = 8;
    touch(a);
    const uint32_t item = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (item >= uint32_t(a.num_rows) * uint32_t(a.heads)) return;
    const int r = int(item / uint32_t(a.heads)), h = int(item - uint32_t(r) * uint32_t(a.heads));
    const int lane = threadIdx.x & 63, sub = lane / LPH, d = 4 * (lane % LPH);
    // The row's parts and its output row are asked for along with the header.
    const int32_t* const plan = a.plan;
    const int2 spot = *reinterpret_cast<const int2*>(plan + a.rows_at + 2 * r);
    const int64_t out_row = a.rows[r];
    const PlanHead head = load_head(plan);
    asm volatile("" ::"v"(spot.x), "v"(spot.y), "v"(out_row), "s"(head.w[0]), "s"(head.w[7]));
    if (!head.fits(a)) return;
    const int parts = spot.y;
    if (parts == 1) return;
    const bool has = d < a.head_dim;
    const int64_t first = int64_t(spot.x) * a.heads + h;
    const float2* const pml = a.part_ml + first;
    const float* const po = a.part_o + first * a.head_dim + (has ? d : 0);
    const int64_t step = int64_t(a.heads) * a.head_dim;
    auto load = [&](int s0, float4 (&o)[B]) {  // past the last part: that again, at weight 0
#pragma unroll
        for (int i = 0; i < B; ++i)
            o[i] = *reinterpret_cast<const float4*>(po +
                                                    min(s0 + i * PAR + sub, parts - 1) * step);
    };
    float4 o[B];
    if (parts) load(0, o);
    float mx = -INFINITY;
    for (int s0 = 0; s0 < parts; s0 += 64)
        if (s0 + lane < parts) mx = fmaxf(mx, pml[int64_t(s0 + lane) * a.heads].x);
    mx = wave_max(mx);
    const float m_use = mx == -INFINITY ? 0.f : mx;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    for (int s0 = 0; s0 < parts; s0 += 64) {
        float w = 0.f;
        if (s0 + lane < parts) {
            const float2 ml = pml[int64_t(s0 + lane) * a.heads];
            w = __builtin_amdgcn_exp2f(ml.x - m_use);
            l += w * ml.y;
        }
        for (int s1 = s0; s1 < min(s0 + 64, parts); s1 += B * PAR) {
            if (s1 > 0) load(s1, o);
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const int s = s1 + i * PAR + sub;
                float f = __shfl(w, (s - s0) & 63, 64);
                f = s < min(s0 + 64, parts) ? f : 0.f;
                sum.x += f * o[i].x;
                sum.y += f * o[i].y;
                sum.z += f * o[i].z;
                sum.w += f * o[i].w;
            }
        }
    }
    l = wave_sum(l);
#pragma unroll
    for (int off = LPH; off < 64; off <<= 1) {
        sum.x += __shfl_xor(sum.x, off, 64);
        sum.y += __shfl_xor(sum.y, off, 64);
        sum.z += __shfl_xor(sum.z, off, 64);
        sum.w += __shfl_xor(sum.w, off, 64);
    }
    if (sub != 0 || !has) return;
    const float inv = parts == 0 ? 0.f : a.v_scale / l;
    uint2 w;
    w.x = pack2<T>(sum.x * inv, sum.y * inv);
    w.y = pack2<T>(sum.z * inv, sum.w * inv);
    *reinterpret_cast<uint2*>(a.out + out_row * a.ots + h * a.ohs + d) = w;
}

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool plan_geometry_ok(int64_t max_rows, int64_t heads, int64_t kv_heads) {
    // (so that a plan's words and its parts' numbers fit in 32 bits)
    return max_rows > 0 && max_rows <= (1 << 20) && heads > 0 && heads <= (1 << 12) &&
           max_rows * heads <= (1 << 26) && kv_heads > 0 && heads % kv_heads == 0;
}

}  // namespace
}  // namespace tvllm

using namespace tvllm;

extern "C" int64_t tvllm_shared_prefix_plan_words(int64_t max_rows, int64_t num_heads,
                                                  int64_t num_kv_heads) {
    if (!plan_geometry_ok(max_rows, num_heads, num_kv_heads)) return 0;
    return plan_layout(max_rows, num_heads, num_kv_heads).words;
}

extern "C" int64_t tvllm_shared_prefix_max_tasks(int64_t max_rows, int64_t num_heads,
                                                 int64_t num_kv_heads) {
    if (!plan_geometry_ok(max_rows, num_heads, num_kv_heads)) return 0;
    return plan_layout(max_rows, num_heads, num_kv_heads).max_tasks;
}

extern "C" int64_t tvllm_shared_prefix_workspace_size(int64_t max_rows, int64_t num_heads,
                                                      int64_t num_kv_heads, int64_t head_dim) {
    if (!plan_geometry_ok(max_rows, num_heads, num_kv_heads) || head_dim <= 0) return 0;
    return max_entries(max_rows, num_heads) * (head_dim + 2) * 4;
}

extern "C" int tvllm_shared_prefix_plan(const int64_t* lengths, const int64_t* groups,
                                        const int64_t* prefix_lens, int64_t num_rows,
                                        int64_t num_groups, int64_t max_rows, int64_t num_heads,
                                        int64_t num_kv_heads, int64_t head_dim,
                                        int64_t block_size, int32_t* plan, int64_t plan_words,
                                        int64_t* num_tasks, int64_t* workspace_bytes) {
    TVLLM_CHECK(plan_geometry_ok(max_rows, num_heads, num_kv_heads),
                "shared_prefix_plan: invalid geometry");
    TVLLM_CHECK(head_dim > 0 && head_dim <= 256 && head_dim % 8 == 0,
                "shared_prefix_plan: head_dim must be a multiple of 8 up to 256");
    TVLLM_CHECK(block_size > 0 && block_size <= INT32_MAX, "shared_prefix_plan: invalid block size");
    TVLLM_CHECK(num_rows >= 0 && num_rows <= max_rows && num_groups >= 0,
                "shared_prefix_plan: more rows than the plan holds");
    const PlanLayout lay = plan_layout(max_rows, num_heads, num_kv_heads);
    TVLLM_CHECK(plan && num_tasks && workspace_bytes && plan_words >= lay.words,
                "shared_prefix_plan: the plan buffer is too small");
    TVLLM_CHECK(num_rows == 0 || (lengths && groups), "shared_prefix_plan: null pointer");
    TVLLM_CHECK(num_groups == 0 || prefix_lens, "shared_prefix_plan: null pointer");
    for (int64_t g = 0; g < num_groups; ++g)
        TVLLM_CHECK(prefix_lens[g] >= 0 && prefix_lens[g] <= kMaxContext &&
                        prefix_lens[g] % block_size == 0,
                    "shared_prefix_plan: prefix lengths must be whole blocks");
    const int64_t group = num_heads / num_kv_heads;
    struct Group {
        int64_t count = 0, first = 0, prefix = 0, splits = 0, per = 0;
    };
    try {
        std::vector<Group> gs(static_cast<size_t>(num_groups));
        for (int64_t r = 0; r < num_rows; ++r) {
            TVLLM_CHECK(lengths[r] >= 0 && lengths[r] <= kMaxContext,
                        "shared_prefix_plan: invalid context length");
            TVLLM_CHECK(groups[r] >= -1 && groups[r] < num_groups,
                        "shared_prefix_plan: group index out of range");
            if (groups[r] < 0) continue;
            TVLLM_CHECK(lengths[r] >= prefix_lens[groups[r]],
                        "shared_prefix_plan: a row is shorter than its group's prefix");
            ++gs[groups[r]].count;
        }
        // Members: the groups' rows side by side, then the others. A prefix
        // that only one row has is that row's own keys.
        int64_t at = 0;
        for (int64_t g = 0; g < num_groups; ++g) {
            gs[g].first = at;
            at += gs[g].count;
            gs[g].prefix = gs[g].count > 1 ? prefix_lens[g] : 0;
        }
        std::vector<int64_t> next(static_cast<size_t>(num_groups)), place(static_cast<size_t>(num_rows)),
            own(static_cast<size_t>(num_rows));
        for (int64_t g = 0; g < num_groups; ++g) next[g] = gs[g].first;
        int32_t* const rows = plan + lay.rows_at;
        int32_t* const members = plan + lay.members_at;
        int32_t* const tasks = plan + lay.tasks_at;
        int64_t cost = 0;
        const int64_t own_tiles = div_up(group, kWide);
        // Few short rows: each is one task a KV head that writes its output, with
        // nothing shared, no parts and no second launch, which costs what some
        // 500 keys of a task do (one after the other, 107 a microsecond). us a
        // call from Python, shared -> so: 2 rows behind 512 tokens 17.5 -> 13.2,
        // 24 behind 608 16.8 -> 14.0, 64 behind 224 17.5 -> 13.4, but 2 behind
        // 1008 17.1 -> 17.7; head dim 256, 4 behind 288 17.4 -> 15.4, behind 512
        // 17.6 -> 18.0. On the card alone 10.6 and a gap -> 11.4 for the first.
        int64_t most_keys = 0, all_keys = 0, filled = 0;
        for (int64_t r = 0; r < num_rows; ++r) {
            most_keys = std::max(most_keys, lengths[r]);
            all_keys += own_tiles * num_kv_heads * lengths[r];
            filled += lengths[r] > 0;
        }
        const bool direct = most_keys * std::max<int64_t>(head_dim, 128) <= kDirectKeys * 128 &&
                            all_keys <= kDirectTotal &&
                            filled * own_tiles * num_kv_heads <= kSlots;
        if (direct)
            for (Group& g : gs) g.prefix = 0;
        for (int64_t r = 0; r < num_rows; ++r) {
            const int64_t g = groups[r];
            place[r] = g >= 0 ? next[g]++ : at++;
            members[place[r]] = int32_t(r);
            own[r] = lengths[r] - (g >= 0 ? gs[g].prefix : 0);
            cost += own_tiles * num_kv_heads * own[r];
        }
        for (const Group& g : gs) cost += div_up(g.count * group, kWide) * num_kv_heads * g.prefix;
        auto cut = [](int64_t keys, int64_t chunk, int64_t& splits, int64_t& per) {
            splits = std::min(kMaxParts, div_up(keys, chunk));
            per = splits ? div_up(div_up(keys, splits), kKeyUnit) * kKeyUnit : 0;
            if (per) splits = div_up(keys, per);
        };
        // KV heads of one task over a row's own keys: short ones share a task, a
        // wave or two for each, so that its cost beside the keys is paid once
        // (256 rows behind 512 with up to 64 own keys: 29.6 -> 20.1 us; 64
        // behind 2048 25.1 -> 23.7; 33 rows in 2 groups, heads of 64, 13.4 ->
        // 13.6-14.4).
        auto heads_of = [&](int64_t keys, int64_t chunk) -> int64_t {
            if (group > kNarrow) return 1;
            for (int64_t h : {4, 2})
                if (num_kv_heads % h == 0 && h * keys <= chunk) return h;
            return 1;
        };
        // The length of a task: the one that ends soonest by a simple estimate.
        // Tasks run on the card's slots, longest first: all at once where they are
        // that few, otherwise the slots' mean share and half of a last, short
        // task; and the parts are written and read again, an entry of 128 dims
        // in about the time of 4 keys of a slot (8 bytes a dim, 512 bytes a key).
        // Head dims above 128 leave one workgroup to a CU. With 512 -> 256 slots,
        // both kernels at head dim 256: 128 rows behind 16384 100 -> 91 us, 48
        // behind 2048 (FP8) 37.2 -> 34.8, 24 behind 1024 21.3 -> 20.6, but 64
        // behind 8192 36.9 -> 39.6.
        const int64_t slots = head_dim > 128 ? kSlots / 2 : kSlots;
        const int64_t least = std::max(kKeyUnit, div_up(cost, kMaxSplits));
        int64_t chunk = 0;
        double best = 0;
        for (int64_t c = div_up(least, kKeyUnit) * kKeyUnit;; c += div_up(c, 4 * kKeyUnit) * kKeyUnit) {
            int64_t count = 0, sum = 0, longest = 0, shortest = INT64_MAX, entries = 0, most = 0;
            int64_t splits, per;
            auto add = [&](int64_t units, int64_t queries, int64_t keys) {
                cut(keys, c, splits, per);
                count += units * splits;
                sum += units * (keys + splits * kTaskCost);
                longest = std::max(longest, std::min(per, keys) + kTaskCost);
                shortest = std::min(shortest, std::min(per, keys) + kTaskCost);
                entries += queries * splits;
                most = std::max(most, keys);
            };
            for (const Group& g : gs)
                if (g.prefix)
                    add(div_up(g.count * group, kWide) * num_kv_heads, g.count * num_heads, g.prefix);
            for (int64_t r = 0; r < num_rows; ++r)
                if (own[r]) {
                    const int64_t h = heads_of(own[r], c);
                    add(own_tiles * num_kv_heads / h, num_heads, own[r] * h);
                }
            const double time =
                (count <= slots ? double(longest)
                                : std::max(double(longest), double(sum) / double(slots) +
                                                                0.5 * double(shortest))) +
                double(entries) * double(head_dim) / 32 / double(slots);
            if (!chunk || time < best) {
                chunk = c;
                best = time;
            }
            if (c >= 4 * most) break;
        }
        if (direct) chunk = std::max(kKeyUnit, div_up(most_keys, kKeyUnit) * kKeyUnit);
        int64_t n = 0;
        auto emit = [&](int64_t member, int64_t q0, int64_t count, int64_t kvh, int64_t heads,
                        int64_t k0, int64_t k1, int64_t part) {
            int32_t* t = tasks + n++ * kTaskWords;
            t[T_MEMBER] = int32_t(member);
            t[T_QUERIES] = int32_t(q0 / kNarrow << 8 | count);
            t[T_KVH] = int32_t(kvh);
            t[T_HEADS] = int32_t(heads);
            t[T_K0] = int32_t(k0);
            t[T_K1] = int32_t(k1);
            t[T_PART] = int32_t(part);
            t[T_ROW] = members[member + q0 / group];
        };
        // Shared keys first, the longest tasks ahead. Workgroups are dealt to
        // the 8 XCDs in turn: the query tiles of one (KV head, range of keys)
        // go 8 apart, onto one XCD, whose L2 they share.
        struct Column {
            int64_t g, kvh, split;
        };
        std::vector<int64_t> order;
        for (int64_t g = 0; g < num_groups; ++g) {
            cut(gs[g].prefix, chunk, gs[g].splits, gs[g].per);
            if (gs[g].splits) order.push_back(g);
        }
        std::sort(order.begin(), order.end(), [&](int64_t x, int64_t y) {
            return gs[x].per != gs[y].per ? gs[x].per > gs[y].per : x < y;
        });
        std::vector<Column> columns;
        for (int64_t g : order) {
            columns.clear();
            for (int64_t s = 0; s < gs[g].splits; ++s)
                for (int64_t h = 0; h < num_kv_heads; ++h) columns.push_back({g, h, s});
            const int64_t queries = gs[g].count * group, tiles = div_up(queries, kWide);
            const int64_t tile = div_up(div_up(queries, tiles), 32) * 32;
            for (size_t c0 = 0; c0 < columns.size(); c0 += 8)
                for (int64_t t = 0; t < tiles; ++t)
                    for (size_t c = c0; c < std::min(columns.size(), c0 + 8); ++c) {
                        const int64_t k0 = columns[c].split * gs[g].per;
                        const int64_t q0 = t * tile;
                        if (q0 < queries)
                            emit(gs[g].first, q0, std::min(tile, queries - q0), columns[c].kvh, 1, k0,
                                 std::min(gs[g].prefix, k0 + gs[g].per), columns[c].split);
                    }
        }
        order.resize(static_cast<size_t>(num_rows));
        for (int64_t r = 0; r < num_rows; ++r) order[r] = r;
        std::sort(order.begin(), order.end(), [&](int64_t x, int64_t y) {
            return own[x] != own[y] ? own[x] > own[y] : x < y;
        });
        std::vector<int64_t> parts(static_cast<size_t>(num_rows));
        for (int64_t r : order) {
            const int64_t g = groups[r], shared = g >= 0 ? gs[g].splits : 0;
            const int64_t begin = g >= 0 ? gs[g].prefix : 0;
            int64_t splits, per;
            const int64_t heads = heads_of(own[r], chunk);
            cut(own[r], chunk, splits, per);
            parts[r] = shared + splits;
            for (int64_t s = 0; s < splits; ++s)
                for (int64_t t = 0; t < own_tiles; ++t)
                    for (int64_t h = 0; h < num_kv_heads; h += heads) {
                        const int64_t k0 = begin + s * per;
                        emit(place[r], t * kWide, std::min<int64_t>(kWide, group - t * kWide), h,
                             heads, k0, std::min(lengths[r], k0 + per), shared + s);
                    }
        }
        int64_t entries = 0;
        for (int64_t r = 0; r < num_rows; ++r) {
            rows[2 * r] = int32_t(entries);
            rows[2 * r + 1] = int32_t(parts[r]);
            if (parts[r] > 1) entries += parts[r];
        }
        std::fill(plan, plan + kHeader, 0);
        plan[H_TASKS] = int32_t(n);
        plan[H_ROWS] = int32_t(num_rows);
        plan[H_HEADS] = int32_t(num_heads);
        plan[H_KV_HEADS] = int32_t(num_kv_heads);
        plan[H_DIM] = int32_t(head_dim);
        plan[H_BLOCK] = int32_t(block_size);
        plan[H_PARTS] = int32_t(entries * num_heads);
        plan[H_MERGE] = entries > 0 || filled < num_rows;  // (which fills rows without keys)
        *num_tasks = n;
        *workspace_bytes = entries * num_heads * (head_dim + 2) * 4;
        clear_error();
        return TVLLM_OK;
    } catch (const std::exception&) {  // no memory for the lists
        set_error("shared_prefix_plan: out of host memory");
        return TVLLM_EINVAL;
    }
}

extern "C" int tvllm_paged_decode_shared_prefix(
    const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k_cache,
    const void* v_cache, void* out, int64_t out_token_stride, int64_t out_head_stride,
    const int64_t* rows, const int64_t* blocks, const int64_t* offsets, const int32_t* plan,
    int64_t num_rows, int64_t max_rows, int64_t num_tasks, int64_t num_heads,
    int64_t num_kv_heads, int64_t head_dim, int64_t num_slots, int64_t cache_slot_stride,
    int64_t cache_head_stride, int64_t block_size, float scale, void* workspace,
    int64_t workspace_bytes, int dtype, int cache_dtype, float k_scale, float v_scale,
    tvllm_stream_t stream) {
    const bool f8 = cache_dtype == TVLLM_FP8_E4M3;
    TVLLM_CHECK(dtype == TVLLM_BF16 || dtype == TVLLM_F16,
                "shared_prefix: Q must be float16 or bfloat16");
    TVLLM_CHECK(f8 || cache_dtype == dtype,
                "shared_prefix: KV cache dtype must match Q or be FP8 E4M3");
    TVLLM_CHECK(k_scale > 0.f && v_scale > 0.f && k_scale < INFINITY && v_scale < INFINITY,
                "shared_prefix: KV scales must be positive and finite");
    TVLLM_CHECK(f8 || (k_scale == 1.f && v_scale == 1.f),
                "shared_prefix: KV scales apply to an FP8 cache only");
    TVLLM_CHECK(plan_geometry_ok(max_rows, num_heads, num_kv_heads),
                "shared_prefix: invalid GQA geometry");
    TVLLM_CHECK(head_dim > 0 && head_dim <= 256 && head_dim % 8 == 0,
                "shared_prefix: head_dim must be a multiple of 8 up to 256");
    TVLLM_CHECK(block_size > 0 && num_slots > 0 && num_slots % block_size == 0,
                "shared_prefix: invalid block geometry");
    TVLLM_CHECK(num_slots <= INT32_MAX, "shared_prefix: at most 2^31-1 cache slots");
    TVLLM_CHECK(cache_layout_ok(num_slots, num_kv_heads, head_dim, cache_slot_stride,
                                cache_head_stride),
                "shared_prefix: cache strides must give non-overlapping head rows");
    TVLLM_CHECK(scale > 0.f && scale < INFINITY, "shared_prefix: scale must be positive");
    TVLLM_CHECK(num_rows >= 0 && num_rows <= max_rows && workspace_bytes >= 0,
                "shared_prefix: negative sizes, or more rows than the plan holds");
    const PlanLayout lay = plan_layout(max_rows, num_heads, num_kv_heads);
    TVLLM_CHECK(num_tasks >= 0 && num_tasks <= lay.max_tasks,
                "shared_prefix: more tasks than the plan holds");
    if (num_rows == 0) {
        clear_error();
        return TVLLM_OK;
    }
    TVLLM_CHECK(q && k_cache && v_cache && out && rows && blocks && offsets && plan,
                "shared_prefix: null pointer");
    TVLLM_CHECK(workspace || workspace_bytes == 0, "shared_prefix: null workspace");
    TVLLM_CHECK(cache_slot_stride % 8 == 0 && cache_head_stride % 8 == 0 &&
                    cache_slot_stride * (f8 ? 1 : 2) <= int64_t(UINT32_MAX) &&
                    (f8 ? aligned8(k_cache) && aligned8(v_cache)
                        : aligned16(k_cache) && aligned16(v_cache)),
                "shared_prefix: cache rows must be whole, aligned 8-element units "
                "(slot stride below 2^32 bytes)");
    TVLLM_CHECK(aligned16(q) && q_token_stride % 8 == 0 && q_head_stride % 8 == 0,
                "shared_prefix: Q rows must be 16-byte aligned");
    TVLLM_CHECK(aligned8(out) && out_token_stride % 4 == 0 && out_head_stride % 4 == 0,
                "shared_prefix: output rows must be 8-byte aligned");
    TVLLM_CHECK(aligned16(plan), "shared_prefix: the plan must be 16-byte aligned");
    TVLLM_CHECK(aligned16(workspace), "shared_prefix: the workspace must be 16-byte aligned");
    TVLLM_CHECK(q != out, "shared_prefix: the output must not be Q (tasks of a row read Q while "
                          "others write its output)");
    hipStream_t s = as_hip(stream);
    return dispatch_half(dtype, [&]<int DT>() {
        using T = typename Elem<DT>::T;
        Args<T> a{};
        a.q = static_cast<const T*>(q);
        a.qts = q_token_stride;
        a.qhs = q_head_stride;
        a.k = k_cache;
        a.v = v_cache;
        a.css = cache_slot_stride;
        a.chs = cache_head_stride;
        a.out = static_cast<T*>(out);
        a.ots = out_token_stride;
        a.ohs = out_head_stride;
        a.rows = rows;
        a.blocks = blocks;
        a.offsets = offsets;
        a.plan = plan;
        a.rows_at = int(lay.rows_at);
        a.members_at = int(lay.members_at);
        a.tasks_at = int(lay.tasks_at);
        a.num_rows = int(num_rows);
        a.heads = int(num_heads);
        a.kv_heads = int(num_kv_heads);
        a.group = int(num_heads / num_kv_heads);
        a.head_dim = int(head_dim);
        a.block_size = int(block_size);
        // With 2^(s-1) < d <= 2^s, m = ceil(2^(31+s) / d) fits in 32 bits and
        // (t m) >> (31 + s) is t / d for every t < 2^31.
        int sh = 0;
        while ((int64_t(1) << sh) < block_size) ++sh;
        a.page_shift = sh;
        a.page_mul = uint32_t(((uint64_t(1) << (31 + sh)) + uint64_t(block_size) - 1) /
                              uint64_t(block_size));
        a.scale_log2 = scale * kLog2e * k_scale;
        a.v_scale = v_scale;
        a.entries = workspace_bytes / ((head_dim + 2) * 4);
        a.part_o = static_cast<float*>(workspace);
        if (workspace) a.part_ml = reinterpret_cast<float2*>(a.part_o + a.entries * head_dim);
        auto go = [&]<int DP>() {
            if (num_tasks) {
                if (f8) shared_prefix_tasks<T, DP, true><<<int(num_tasks), kThreads, 0, s>>>(a);
                else shared_prefix_tasks<T, DP, false><<<int(num_tasks), kThreads, 0, s>>>(a);
            }
            if (workspace)
                shared_prefix_merge<T, DP>
                    <<<int(div_up(num_rows * num_heads, kThreads / 64)), kThreads, 0, s>>>(a);
        };
        if (head_dim <= 32) go.template operator()<32>();
        else if (head_dim <= 64) go.template operator()<64>();
        else if (head_dim <= 128) go.template operator()<128>();
        else go.template operator()<256>();
        return launch_status("shared_prefix");
    });
}
