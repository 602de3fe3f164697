// The best continuations of a beam search's step: over every beam of a request and the whole vocabulary
//
//   c(r, v) = score_r + x[r][v] - log sum_u exp(x[r][u])
//
// the `keep` largest in descending order, the lowest (beam, token) first among equals.  A row that has no softmax (a NaN, an infinite maximum, nothing
// above -inf) or whose score is not finite offers its tokens at -inf, in their order.
//
// One launch, one read of the logits.  A block walks a stretch of a row, 4,096 values at a time in registers (float32, as the logits come) with the next ones on their way, and leaves
// the values' maximum, their sum of exponentials against it and their `keep` best in order: within a row c and x have the same order, so neither needs the row's sum.
// The block that completes a request joins the sums and merges its lists; c is computed there, in float64, for the few values that are left, so that a row's candidates keep the
// order of its values and none is lost to the rounding of score + x.  Across rows the order is as good as the rows' log sums, whose sums of exponentials are float32: off by 5e-7 at most in
// what was measured (512 to 262,144 tokens, values that are normal, equal, rising, flat, a few hundred far above the rest), and by less than 2^-15 whatever the values are (up to 128 terms added
// one after the other by a thread, 8 times a new maximum, some 26 joins, each exponential to 2^-22 and 2^-24 of its argument): candidates of two rows that lie closer may change places.
//
// Choosing `keep` of many, without sorting them: the block's threads make 32 to 256 groups, at least twice as many as are kept; the keep-th largest of the groups'
// best is a bound that at least `keep` values reach and few others do (17 values of 4,096 normal ones above the bound for keep = 8, 150 for 64).  Every thread knows its largest value of each
// round of loads, so only the sixteens that hold such a value are read again; the values are put in a list in shared memory and each counts how many of the list are larger: its
// place.  The merge does the same with the lists' first entries, and goes on down a list whose last one of those still reaches the bound.  Where too many reach
// the bound (many equal values, values laid out against the groups) the choice is made by value and token together, and at last the bound raised bit by bit to the keep-th largest itself.
//
// What bounds it.  Two requests of 32 beams over 131,072 tokens, 64 kept (34 MB): 22.4 us; the walk is 4 (the reading alone 5 at the copy rate, and half the values were in the second-level cache),
// what follows it in every block 6, the last block's merge 8: chains of barriers and dependent trips, in one block for each request.  Eight requests of eight beams over 49,152 tokens (13 MB):
// 13.2 us; one request of four (0.8 MB): 8.5.  On the way: a bound and a list after every round of loads 28.5 us, ranks counted by value and token together 34, every row merged before its
// request 72.
#include "common.cuh"

#include <cuda_fp16.h>

namespace vk {

constexpr int BS_THREADS = 256, BS_VALUES = 16, BS_MAX_KEEP = 128, BS_MAX_BEAMS = 64, BS_LIST = 1024, BS_MAX_PARTS = 64, BS_MAX_ROWS = 1024, BS_HELD = 2048, BS_ROUND = BS_THREADS * BS_VALUES, BS_MAX_ROUNDS = 8;

typedef unsigned long long u64;

// A candidate as one number whose order is "larger value first, then lower token": 0 is below all of them.
__device__ __forceinline__ uint32_t bs_order(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);                 // -0 becomes +0
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float bs_value(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o); }
__device__ __forceinline__ u64 bs_pack(float v, uint32_t token) { return ((u64)bs_order(v) << 32) | (0xffffffffu - token); }
__device__ __forceinline__ u64 bs_order64(double v) {
    const u64 b = (u64)__double_as_longlong(v + 0.0);
    return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double bs_value64(u64 o) { return __longlong_as_double((long long)((o >> 63) ? (o & 0x7fffffffffffffffull) : ~o)); }

// A candidate of a request: c in float64 as an ordered number, and beam * vocab + token turned round.
struct BsPair {
    u64 hi;
    uint32_t lo;
};
__device__ __forceinline__ bool bs_above(const BsPair& a, const BsPair& b) { return a.hi > b.hi || (a.hi == b.hi && a.lo > b.lo); }
__device__ __forceinline__ bool bs_above(u64 a, u64 b) { return a > b; }
__device__ __forceinline__ u64 bs_shfl_xor(u64 v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }
__device__ __forceinline__ BsPair bs_shfl_xor(const BsPair& v, int o) { return BsPair{__shfl_xor_sync(0xffffffffu, v.hi, o), __shfl_xor_sync(0xffffffffu, v.lo, o)}; }
__device__ __forceinline__ bool bs_is_none(u64 v) { return v == 0; }
__device__ __forceinline__ bool bs_is_none(const BsPair& v) { return v.lo == 0; }      // flat places are below 2^32 - 1
template <typename K> __device__ __forceinline__ K bs_none();
template <> __device__ __forceinline__ u64 bs_none<u64>() { return 0; }
template <> __device__ __forceinline__ BsPair bs_none<BsPair>() { return BsPair{0, 0}; }
// the number with bit b set on top of t's higher bits (bits counted from the top: 0 .. bits - 1)
__device__ __forceinline__ u64 bs_with_bit(u64 t, int b) { return t | (1ull << (63 - b)); }
__device__ __forceinline__ BsPair bs_with_bit(const BsPair& t, int b) { return b < 64 ? BsPair{t.hi | (1ull << (63 - b)), t.lo} : BsPair{t.hi, t.lo | (1u << (95 - b))}; }
template <typename K> struct BsBits;
template <> struct BsBits<u64> { static constexpr int N = 64; };
template <> struct BsBits<BsPair> { static constexpr int N = 96; };

template <typename K> struct BsPick {
    K group[BS_THREADS];
    K list[BS_LIST];
    K bound;
    int count;
};

__device__ __forceinline__ int bs_lanes(int keep) { return keep <= 16 ? 8 : keep <= 32 ? 4 : keep <= 64 ? 2 : 1; }

// The `keep` largest of the block's candidates into out[0 .. keep), in descending order, none where there are fewer.  each(f) calls f(candidate) for every
// candidate of this thread.  out is shared memory.  Every thread of the block calls it.  The way for candidates that the quick ones do not tell apart: by all of a candidate.
template <typename K, typename Each>
__device__ __noinline__ void bs_pick(BsPick<K>& s, int keep, K* out, const Each& each) {
    const int tid = threadIdx.x, lane = tid & 31;
    K best = bs_none<K>();
    each([&](const K& c) { if (bs_above(c, best)) best = c; });
    const int lanes = bs_lanes(keep), groups = BS_THREADS / lanes;
    for (int o = 1; o < lanes; o <<= 1) {
        const K other = bs_shfl_xor(best, o);
        if (bs_above(other, best)) best = other;
    }
    __syncthreads();
    if (lane % lanes == 0) s.group[tid / lanes] = best;
    if (tid == 0) { s.bound = bs_none<K>(); s.count = 0; }
    for (int i = tid; i < keep; i += BS_THREADS) out[i] = bs_none<K>();
    __syncthreads();
    if (tid < groups) {
        const K mine = s.group[tid];
        int above = 0;
        for (int i = 0; i < groups; i++) above += bs_above(s.group[i], mine);
        if (above == keep - 1 && !bs_is_none(mine)) s.bound = mine;          // groups' best are different candidates
    }
    __syncthreads();
    K bound = s.bound;
    each([&](const K& c) {
        if (!bs_is_none(c) && !bs_above(bound, c)) {
            const int at = atomicAdd(&s.count, 1);
            if (at < BS_LIST) s.list[at] = c;
        }
    });
    __syncthreads();
    int n = s.count;
    if (n > BS_LIST) {                                                       // the bound is raised to the keep-th largest
        bound = bs_none<K>();
        for (int b = 0; b < BsBits<K>::N; b++) {
            const K trial = bs_with_bit(bound, b);
            __syncthreads();
            if (tid == 0) s.count = 0;
            __syncthreads();
            int mine = 0;
            each([&](const K& c) { mine += !bs_is_none(c) && !bs_above(trial, c); });
            if (mine) atomicAdd(&s.count, mine);
            __syncthreads();
            if (s.count >= keep) bound = trial;
        }
        __syncthreads();
        if (tid == 0) s.count = 0;
        __syncthreads();
        each([&](const K& c) {
            if (!bs_is_none(c) && !bs_above(bound, c)) s.list[atomicAdd(&s.count, 1)] = c;       // exactly `keep`: candidates differ
        });
        __syncthreads();
        n = s.count;
    }
    for (int i = tid; i < n; i += BS_THREADS) {
        const K mine = s.list[i];
        int above = 0;
        for (int j = 0; j < n; j++) above += bs_above(s.list[j], mine);
        if (above < keep) out[above] = mine;
    }
    __syncthreads();
}

struct BsArgs {
    const float* logits;      // [rows][ld]
    const float* scores;      // [rows]
    float* out_score;         // [requests][keep]
    int32_t* out_parent;
    int32_t* out_token;
    int* arrived;             // [requests]: zero between launches
    float2* sums;             // [rows][parts] maximum and sum of exponentials
    u64* lists;               // [rows][parts][keep]
    long long ld;
    int beams, vocab, keep, parts, stretch;
};

__device__ __forceinline__ float bs_exp(float x) {           // relative error 2^-22 and 2^-24 |x|
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}

// Maximum and sum of the warp's lanes: one exponential a lane.
__device__ __forceinline__ void bs_join_warp(float& m, float& s) {
    const float top = bs_value(__reduce_max_sync(0xffffffffu, bs_order(m))), r = top == -INFINITY ? 0.0f : top;
    s = warp_sum(s * bs_exp(m - r));
    m = top;
}

// (m, s) and (om, os) together: maximum, and sum of exponentials against it.  Of nothing above -inf the sum is 0; a NaN stays one.
__device__ __forceinline__ void bs_join(float& m, float& s, float om, float os) {
    const float both = fmaxf(m, om), r = both == -INFINITY ? 0.0f : both;
    s = s * bs_exp(m - r) + os * bs_exp(om - r);
    m = both;
}

// The bound: the largest number that at least `keep` of the block's 256 threads reach together with their neighbours, from the groups of threads' largest values rounded down to 11 bits (a
// bound may be lower, and two of those are compared in an instruction).  -inf where there is none.  group: BS_THREADS halves; bound: an ordered number, 0 before.  Two barriers.
__device__ __forceinline__ float bs_bound(float best, int lanes, int keep, __half* group, uint32_t* bound) {
    const int tid = threadIdx.x, lane = tid & 31, groups = BS_THREADS / lanes;
    for (int o = 1; o < lanes; o <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane % lanes == 0) group[tid / lanes] = __float2half_rd(best);
    __syncthreads();
    if (tid < groups) {
        const __half mine = group[tid];
        const __half2 pair = __half2half2(mine);
        __half2 reach = __float2half2_rn(0.0f);
#pragma unroll 2
        for (int i = 0; i < groups; i += 8) {
            const uint4 g = *reinterpret_cast<const uint4*>(group + i);
            reach = __hadd2(reach, __hadd2(__hadd2(__hge2(*reinterpret_cast<const __half2*>(&g.x), pair), __hge2(*reinterpret_cast<const __half2*>(&g.y), pair)),
                                           __hadd2(__hge2(*reinterpret_cast<const __half2*>(&g.z), pair), __hge2(*reinterpret_cast<const __half2*>(&g.w), pair))));
        }
        const uint32_t can = __low2float(reach) + __high2float(reach) >= (float)keep ? bs_order(__half2float(mine)) : 0u;
        const uint32_t most = __reduce_max_sync(0xffffffffu, can);
        if (lane == 0) atomicMax(bound, most);
    }
    __syncthreads();
    return *bound ? bs_value(*bound) : -INFINITY;
}

__global__ void __launch_bounds__(BS_THREADS, 4) beam_select_kernel(const BsArgs a) {
    __shared__ union {
        struct {                                       // this block's values that reach the bound, and their tokens
            float value[BS_LIST + 4];
            int token[BS_LIST], slot[BS_LIST];
        } part;
        struct {                                       // the request's entries, and those of them that reach the bound
            u64 entry[BS_HELD];
            uint32_t place[BS_HELD];
            u64 value[BS_LIST];
            uint32_t flat[BS_LIST];
        } merge;
        BsPick<u64> one;
        BsPick<BsPair> two;
    } sm;
    __shared__ union { u64 one[BS_MAX_KEEP]; BsPair two[BS_MAX_KEEP]; } top;
    __shared__ double base[BS_MAX_BEAMS];
    __shared__ __align__(16) __half group[BS_THREADS];
    __shared__ float2 warp_sums[BS_THREADS / 32];
    __shared__ uint32_t bound_s;
    __shared__ int taken[BS_MAX_KEEP], slots, count, done;
    float* best = reinterpret_cast<float*>(sm.merge.entry) + sizeof(sm.part) / 4;      // a thread's largest value of every round: behind the list
    static_assert(sizeof(sm.part) + BS_MAX_ROUNDS * BS_THREADS * 4 <= sizeof(sm.merge), "the rounds' largest values lie behind the list");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, part = blockIdx.x, row = blockIdx.y, keep = a.keep;
    if (tid == 0) { bound_s = 0; slots = 0; count = 0; }
    if (tid < keep) { taken[tid] = 0; top.one[tid] = 0; }
    dependency_wait();
    let_dependents_start();

    // ---- this block's values: thread t has four neighbours of every 1,024 (wherever the row begins, so that equal rows have equal sums)
    const float* x = a.logits + (size_t)row * a.ld;
    const bool aligned = (uintptr_t)x % 16 == 0;
    const int from = part * a.stretch, to = min(a.vocab, from + a.stretch);
    float v[BS_VALUES], next[BS_VALUES];
    auto load = [&](int first) {
#pragma unroll
        for (int j = 0; j < BS_VALUES / 4; j++) {
            const int i = first + (j * BS_THREADS + tid) * 4;
            if (aligned && i + 3 < to) {
                const float4 f = __ldcs(reinterpret_cast<const float4*>(x + i));
                next[4 * j] = f.x; next[4 * j + 1] = f.y; next[4 * j + 2] = f.z; next[4 * j + 3] = f.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) next[4 * j + e] = i + e < to ? x[i + e] : -INFINITY;
            }
        }
    };
    load(from);
    float m = -INFINITY, s = 0.0f;
#pragma unroll 1
    for (int at = from, round = 0; at < to; at += BS_ROUND, round++) {
#pragma unroll
        for (int j = 0; j < BS_VALUES; j++) v[j] = next[j];
        if (at + BS_ROUND < to) load(at + BS_ROUND);
        float here = v[0];
#pragma unroll
        for (int j = 1; j < BS_VALUES; j++) here = fmaxf(here, v[j]);
        best[round * BS_THREADS + tid] = here;
        // the sum of exponentials: of nothing above -inf nothing; a NaN stays one
        const float more = fmaxf(m, here), ref = more == -INFINITY ? 0.0f : more;
        s *= bs_exp(m - ref);
        m = more;
#pragma unroll
        for (int j = 0; j < BS_VALUES; j++) s += bs_exp(v[j] - ref);
    }
    const float bound = bs_bound(m, bs_lanes(keep), keep, group, &bound_s), enough = fmaxf(bound, -3.402823466e38f);      // -inf comes in behind, if at all
    bs_join_warp(m, s);
    if (lane == 0) warp_sums[warp] = make_float2(m, s);
    // ---- the sixteens that hold a value that reaches the bound, and then those values
    for (int at = from, slot = tid; at < to; at += BS_ROUND, slot += BS_THREADS)
        if (best[slot] >= enough) {
            const int place = atomicAdd(&slots, 1);
            if (place < BS_LIST) sm.part.slot[place] = slot;
        }
    __syncthreads();
    const int fours = min(slots, BS_LIST) * (BS_VALUES / 4);
    for (int c = tid; c < fours; c += BS_THREADS) {
        const int slot = sm.part.slot[c / (BS_VALUES / 4)], i = from + slot / BS_THREADS * BS_ROUND + (c % (BS_VALUES / 4) * BS_THREADS + slot % BS_THREADS) * 4;
        float f[4];
        if (aligned && i + 3 < to) {
            const float4 g = *reinterpret_cast<const float4*>(x + i);
            f[0] = g.x; f[1] = g.y; f[2] = g.z; f[3] = g.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) f[e] = i + e < to ? x[i + e] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (f[e] >= enough) {
                const int place = atomicAdd(&count, 1);
                if (place < BS_LIST) {
                    sm.part.value[place] = f[e];
                    sm.part.token[place] = i + e;
                }
            }
    }
    if (warp == 0) {
        const float2 o = lane < BS_THREADS / 32 ? warp_sums[lane] : make_float2(-INFINITY, 0.0f);
        m = o.x;
        s = o.y;
        bs_join_warp(m, s);
        if (lane == 0) a.sums[(size_t)row * a.parts + part] = make_float2(m, s);
    }
    __syncthreads();
    int n = slots > BS_LIST ? BS_LIST + 1 : count;
    if (n < keep) {
        // everything above -inf is in the list: behind it come the first tokens that are -inf
        if (warp == 0) {
            int have = n;
            for (int i = from + lane; have < keep && i - lane < to; i += 32) {
                const bool none = i < to && x[i] == -INFINITY;
                const uint32_t all = __ballot_sync(0xffffffffu, none);
                const int place = have + __popc(all & ((1u << lane) - 1));
                if (none && place < keep) { sm.part.value[place] = -INFINITY; sm.part.token[place] = i; }
                have += __popc(all);
            }
            if (lane == 0) done = min(have, keep);
        }
        __syncthreads();
        n = done;
    }
    if (n <= BS_LIST) {
        // each counts the larger ones: its place; where several have the same place they have the same value, and are told apart by their tokens
        if (tid < 4) sm.part.value[n + tid] = -INFINITY;
        __syncthreads();
        for (int i = tid; i < n; i += BS_THREADS) {
            const float mine = sm.part.value[i];
            int above = 0;
#pragma unroll 4
            for (int j = 0; j < n; j += 4) {
                const float4 f = *reinterpret_cast<const float4*>(sm.part.value + j);
                above += (f.x > mine) + (f.y > mine) + (f.z > mine) + (f.w > mine);
            }
            if (above < keep && atomicAdd(&taken[above], 1) == 0) top.one[above] = bs_pack(mine, (uint32_t)sm.part.token[i]);
        }
        __syncthreads();
        bool equal = false;
        if (tid < keep) equal = taken[tid] > 1;
        if (__syncthreads_or(equal))
            for (int i = tid; i < n; i += BS_THREADS) {
                const float mine = sm.part.value[i];
                int above = 0, before = 0;
                for (int j = 0; j < n; j++) {
                    above += sm.part.value[j] > mine;
                    before += sm.part.value[j] == mine && sm.part.token[j] < sm.part.token[i];
                }
                if (above + before < keep) top.one[above + before] = bs_pack(mine, (uint32_t)sm.part.token[i]);
            }
    } else {
        bs_pick(sm.one, keep, top.one, [x, from, to, tid](auto&& take) {      // from memory again
            for (int i = from + tid; i < to; i += BS_THREADS) {
                const float f = x[i];
                take(f == f ? bs_pack(f, (uint32_t)i) : bs_pack(-INFINITY, (uint32_t)i));
            }
        });
    }
    __syncthreads();
    for (int i = tid; i < keep; i += BS_THREADS) a.lists[((size_t)row * a.parts + part) * keep + i] = top.one[i];

    // ---- the block that completes the request goes on
    const int request = row / a.beams;
    __syncthreads();
    if (tid == 0) {
        int old;
        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(old) : "l"(a.arrived + request) : "memory");
        done = old == a.beams * a.parts - 1;
        if (done) a.arrived[request] = 0;                     // ready for the next launch
    }
    __syncthreads();
    if (!done) return;

    // ---- its rows' lists: of each the first entries, as many as can be held, are asked for now
    const int n_lists = a.beams * a.parts, held = min(keep, BS_HELD / n_lists), entries = n_lists * held;
    const u64* mine = a.lists + (size_t)request * n_lists * keep;
    auto over = [](int x, float by) { return (int)(((float)x + 0.5f) * by); };        // x / n for x below 2^22
    const float per_list = 1.0f / (float)held, per_row = 1.0f / (float)a.parts;
    {
        u64 raw[BS_HELD / BS_THREADS];
#pragma unroll
        for (int j = 0; j < BS_HELD / BS_THREADS; j++) {
            const int e = tid + j * BS_THREADS, list = over(e, per_list);
            raw[j] = e < entries ? __ldcg(mine + list * keep + e - list * held) : 0;
        }
#pragma unroll
        for (int j = 0; j < BS_HELD / BS_THREADS; j++) sm.merge.entry[tid + j * BS_THREADS] = raw[j];
    }
    // ---- its rows' sums: 4 to 32 threads a row.  base = score - log sum exp; -inf for a row that has no softmax or does not live
    {
        int each = 32;
        while (each * a.beams > BS_THREADS) each >>= 1;
        const int b = tid / each, sub = tid % each;
        const float score = b < a.beams ? a.scores[request * a.beams + b] : 0.0f;
        m = -INFINITY;
        s = 0.0f;
        if (b < a.beams)
            for (int i = sub; i < a.parts; i += each) {
                const float2 o = __ldcg(a.sums + ((size_t)request * a.beams + b) * a.parts + i);
                bs_join(m, s, o.x, o.y);
            }
#pragma unroll 1
        for (int o = 1; o < each; o <<= 1) bs_join(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
        if (b < a.beams && sub == 0) {
            const double lse = (double)m + log((double)s);
            base[b] = isfinite(score) && isfinite(lse) ? (double)score - lse : (double)-INFINITY;
        }
        if (tid == 0) { count = 0; bound_s = 0; }
        if (tid < keep) { taken[tid] = 0; top.two[tid] = bs_none<BsPair>(); }
    }
    __syncthreads();
    // ---- the best of its rows' lists
    auto of_entry = [&](u64 c, int list, int rank) {
        const int b = over(list, per_row);
        if (base[b] == (double)-INFINITY)                       // the row's tokens in their order, once a row
            return list == b * a.parts && rank < a.vocab ? BsPair{bs_order64((double)-INFINITY), 0xffffffffu - ((uint32_t)b * (uint32_t)a.vocab + (uint32_t)rank)} : bs_none<BsPair>();
        if (c == 0) return bs_none<BsPair>();
        return BsPair{bs_order64(base[b] + (double)bs_value((uint32_t)(c >> 32))), 0xffffffffu - ((uint32_t)b * (uint32_t)a.vocab + (0xffffffffu - (uint32_t)c))};
    };
    auto candidate = [&](int list, int rank) { return of_entry(__ldcg(mine + (size_t)list * keep + rank), list, rank); };
    auto into_list = [&](u64 value, uint32_t flat) {
        const int at = atomicAdd(&count, 1);
        if (at < BS_LIST) {
            sm.merge.value[at] = value;
            sm.merge.flat[at] = flat;
        }
    };
    auto rounded = [](const BsPair& c) { return bs_is_none(c) ? -INFINITY : __double2float_rd(bs_value64(c.hi)); };
    float reaches = -INFINITY;
#pragma unroll 1
    for (int e = tid; e < entries; e += BS_THREADS) {
        const int list = over(e, per_list);
        const BsPair c = of_entry(sm.merge.entry[e], list, e - list * held);
        sm.merge.entry[e] = c.hi;
        sm.merge.place[e] = c.lo;
        reaches = fmaxf(reaches, rounded(c));
    }
    const float lowest = bs_bound(reaches, 1, keep, group, &bound_s);
    const u64 least = lowest == -INFINITY ? 0 : bs_order64((double)lowest);
#pragma unroll 1
    for (int e = tid; e < entries; e += BS_THREADS) {
        if (sm.merge.place[e] == 0 || sm.merge.entry[e] < least) continue;
        into_list(sm.merge.entry[e], sm.merge.place[e]);
        const int list = over(e, per_list);
        if (e - list * held + 1 == held)                        // a list's last held entry reaches the bound: on from there
#pragma unroll 1
            for (int rank = held; rank < keep; rank += 8) {
                BsPair c[8];
#pragma unroll
                for (int f = 0; f < 8; f++) c[f] = rank + f < keep ? candidate(list, rank + f) : bs_none<BsPair>();
#pragma unroll
                for (int f = 0; f < 8; f++)
                    if (!bs_is_none(c[f]) && c[f].hi >= least) into_list(c[f].hi, c[f].lo);
                if (bs_is_none(c[7]) || c[7].hi < least) break;
            }
    }
    __syncthreads();
    int n2 = count;
    if (n2 <= BS_LIST && n2 > 2 * keep && n2 > 64) {
        // a second bound, of the list itself, where the first let many through (beams far apart): the list moves to where the entries were
        float mine_best = -INFINITY;
        for (int i = tid; i < n2; i += BS_THREADS) mine_best = fmaxf(mine_best, __double2float_rd(bs_value64(sm.merge.value[i])));
        __syncthreads();
        if (tid == 0) { count = 0; bound_s = 0; }
        __syncthreads();
        const float second = bs_bound(mine_best, 1, keep, group, &bound_s);
        const u64 least2 = second == -INFINITY ? 0 : bs_order64((double)second);
        for (int i = tid; i < n2; i += BS_THREADS)
            if (sm.merge.value[i] >= least2) {
                const int at = atomicAdd(&count, 1);
                sm.merge.entry[at] = sm.merge.value[i];
                sm.merge.place[at] = sm.merge.flat[i];
            }
        __syncthreads();
        n2 = count;
        for (int i = tid; i < n2; i += BS_THREADS) { sm.merge.value[i] = sm.merge.entry[i]; sm.merge.flat[i] = sm.merge.place[i]; }
        __syncthreads();
    }
    if (n2 <= BS_LIST) {
        for (int i = tid; i < n2; i += BS_THREADS) {
            const u64 value = sm.merge.value[i];
            int above = 0;
#pragma unroll 4
            for (int j = 0; j < n2; j++) above += sm.merge.value[j] > value;
            if (above < keep && atomicAdd(&taken[above], 1) == 0) top.two[above] = BsPair{value, sm.merge.flat[i]};
        }
        __syncthreads();
        bool equal = false;
        if (tid < keep) equal = taken[tid] > 1;
        if (__syncthreads_or(equal))
            for (int i = tid; i < n2; i += BS_THREADS) {
                const BsPair c = {sm.merge.value[i], sm.merge.flat[i]};
                int above = 0;
                for (int j = 0; j < n2; j++) above += bs_above(BsPair{sm.merge.value[j], sm.merge.flat[j]}, c);
                if (above < keep) top.two[above] = c;
            }
        __syncthreads();
    } else {
        bs_pick(sm.two, keep, top.two, [&](auto&& take) {
            for (int e = tid; e < n_lists * keep; e += BS_THREADS) {
                const BsPair c = candidate(e / keep, e % keep);
                if (!bs_is_none(c)) take(c);
            }
        });
    }
    for (int i = tid; i < keep; i += BS_THREADS) {
        const BsPair c = top.two[i];
        const uint32_t flat = 0xffffffffu - c.lo;
        const size_t at = (size_t)request * keep + i;
        a.out_score[at] = (float)bs_value64(c.hi);
        a.out_parent[at] = (int)(flat / (uint32_t)a.vocab);
        a.out_token[at] = (int)(flat % (uint32_t)a.vocab);
    }
}

// How long a block's stretch of a row is, in values, and how many make a row: as many rounds of loads a block as keep all blocks running at once (four a multiprocessor), at
// most eight.
struct BsShape { int stretch, parts; };
static BsShape bs_shape(int rows, int vocab) {
    const int rounds = (vocab + BS_ROUND - 1) / BS_ROUND;
    const long long fit = ((long long)rows * rounds + 4 * 148 - 1) / (4 * 148);
    const int each = fit > BS_MAX_ROUNDS ? BS_MAX_ROUNDS : (int)fit;
    return BsShape{each * BS_ROUND, (rounds + each - 1) / each};
}

}  // namespace vk

using namespace vk;

VK_API size_t vk_beam_select_scratch_bytes(int rows, int vocab, int keep) {
    // the shortest stretches' parts, whatever the rows
    const size_t parts = (size_t)(vocab + BS_THREADS * BS_VALUES - 1) / (BS_THREADS * BS_VALUES);
    return (size_t)BS_MAX_ROWS * 4 + rows * parts * 8 + (size_t)rows * parts * keep * 8;
}

// scratch: vk_beam_select_scratch_bytes bytes for at least as many rows, as large a vocabulary and as many kept; its first BS_MAX_ROWS words were zero
// at first use and are zero again after every launch.
VK_API int vk_beam_select(const float* logits, const float* scores, float* out_score, int32_t* out_parent, int32_t* out_token, void* scratch, size_t scratch_bytes,
                          int rows, int beams, int vocab, long long ld, int keep, cudaStream_t stream) {
    if (rows <= 0) return VK_OK;
    if (beams <= 0 || rows % beams || vocab <= 0 || ld < vocab || keep <= 0 || !scratch) return VK_BAD_SHAPE;
    if (beams > BS_MAX_BEAMS || keep > BS_MAX_KEEP || vocab > BS_MAX_PARTS * BS_THREADS * 16 || rows > BS_MAX_ROWS) return VK_TOO_LARGE;
    if ((long long)beams * vocab < keep) return VK_BAD_SHAPE;
    if ((uintptr_t)logits % 4 || (uintptr_t)scratch % 16) return VK_BAD_ALIGNMENT;
    if (scratch_bytes < vk_beam_select_scratch_bytes(rows, vocab, keep)) return VK_SMALL_SCRATCH;
    const BsShape s = bs_shape(rows, vocab);
    BsArgs a;
    a.logits = logits; a.scores = scores; a.out_score = out_score; a.out_parent = out_parent; a.out_token = out_token;
    char* at = (char*)scratch;
    a.arrived = (int*)at; at += (size_t)BS_MAX_ROWS * 4;
    a.lists = (u64*)at; at += (size_t)rows * s.parts * keep * 8;
    a.sums = (float2*)at;
    a.ld = ld; a.beams = beams; a.vocab = vocab; a.keep = keep; a.parts = s.parts; a.stretch = s.stretch;
    return launch_dependent(beam_select_kernel, dim3(s.parts, rows), dim3(BS_THREADS), 0, stream, a);
}
