// The best continuations of a beam search's step: over every beam of a request and the whole vocabulary
//
//   c(r, v) = score_r + x[r][v] - log sum_u exp(x[r][u])
//
// the `keep` largest in descending order, the lowest (beam, token) first among equals.  A row that has no softmax (a NaN, an infinite maximum, nothing
// above -inf) or whose score is not finite offers its tokens at -inf, in their order.
//
// One launch, one read of the logits.  A block holds 4,096 or 8,192 values of a row in registers (float32, as the logits come) and leaves the values'
// maximum, their sum of exponentials against it and their `keep` best in order: within a row c and x have the same order, so neither needs the row's sum.
// The block that completes a request joins the sums in float64 and merges its lists; c is computed there, in float64, for the few values that are left,
// so that two beams' candidates are told apart where float32 sums would tie.  Where the lists are long together, the block that completes a row
// merges that row's lists first.
//
// Choosing `keep` of many, without sorting them: the block's threads make 32 to 256 groups, at least twice as many as are kept; the keep-th largest of the groups'
// best is a bound that at least `keep` values reach and few others do (17 values of 4,096 normal ones above the bound for keep = 8, 150 for 64).  Those are put in a list
// in shared memory and each counts how many of the list are larger: its place.  Where too many reach the bound (values laid out against the groups) it is raised bit by bit
// to the keep-th largest itself.
#include "common.cuh"

namespace vk {

constexpr int BS_THREADS = 256, BS_MAX_KEEP = 128, BS_MAX_BEAMS = 64, BS_LIST = 1024, BS_MAX_PARTS = 64, BS_MAX_ROWS = 1024;

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

// The `keep` largest of the block's candidates into out[0 .. keep), in descending order, none where there are fewer.  each(f) calls f(candidate) for every
// candidate of this thread.  out is shared memory.  Every thread of the block calls it.
template <typename K, typename Each>
__device__ __forceinline__ void bs_pick(BsPick<K>& s, int keep, K* out, const Each& each) {
    const int tid = threadIdx.x, lane = tid & 31;
    K best = bs_none<K>();
    each([&](const K& c) { if (bs_above(c, best)) best = c; });
    const int lanes = keep <= 16 ? 8 : keep <= 32 ? 4 : keep <= 64 ? 2 : 1, groups = BS_THREADS / lanes;
    for (int o = 1; o < lanes; o <<= 1) {
        const K other = bs_shfl_xor(best, o);
        if (bs_above(other, best)) best = other;
    }
    if (lane % lanes == 0) s.group[tid / lanes] = best;
    if (tid == 0) { s.bound = bs_none<K>(); s.count = 0; }
    for (int i = tid; i < keep; i += BS_THREADS) out[i] = bs_none<K>();
    __syncthreads();
    if (tid < groups) {
        const K mine = s.group[tid];
        int above = 0;
#pragma unroll 8
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
#pragma unroll 8
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
    int* arrived;             // [BS_MAX_ROWS] of the rows and, behind them, as many of the requests: zero between launches
    float2* sums;             // [rows][parts] maximum and sum of exponentials
    u64* lists;               // [rows][parts][keep]
    u64* row_lists;           // [rows][keep], where a row's lists are merged first
    long long ld;
    int beams, vocab, keep, parts, merge_rows;
};

template <int VALUES>
__global__ void __launch_bounds__(BS_THREADS) beam_select_kernel(const BsArgs a) {
    __shared__ union { BsPick<u64> one; BsPick<BsPair> two; } pick;
    __shared__ union { u64 one[BS_MAX_KEEP]; BsPair two[BS_MAX_KEEP]; } top;
    __shared__ double base[BS_MAX_BEAMS];
    __shared__ float2 warp_sums[BS_THREADS / 32];
    __shared__ int done;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, part = blockIdx.x, row = blockIdx.y;
    dependency_wait();

    // ---- this block's values: thread t has four neighbours of every 1,024 (wherever the row begins, so that equal rows have equal sums)
    const float* x = a.logits + (size_t)row * a.ld;
    const bool aligned = (uintptr_t)x % 16 == 0;
    const int first = part * (BS_THREADS * VALUES) + tid * 4;
    float v[VALUES];
#pragma unroll
    for (int j = 0; j < VALUES / 4; j++) {
        const int i = first + j * BS_THREADS * 4;
        if (aligned && i + 3 < a.vocab) {
            const float4 f = __ldcs(reinterpret_cast<const float4*>(x + i));
            v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) v[4 * j + e] = i + e < a.vocab ? x[i + e] : -INFINITY;
        }
    }
    float m = -INFINITY, s = 0.0f;
#pragma unroll
    for (int j = 0; j < VALUES; j++) m = fmaxf(m, v[j]);
    const float ref = m == -INFINITY ? 0.0f : m;              // -inf - 0: nothing; a NaN stays one
#pragma unroll
    for (int j = 0; j < VALUES; j++) s += expf(v[j] - ref);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o), both = fmaxf(m, om), r = both == -INFINITY ? 0.0f : both;
        s = s * expf(m - r) + os * expf(om - r);
        m = both;
    }
    if (lane == 0) warp_sums[warp] = make_float2(m, s);
    bs_pick(pick.one, a.keep, top.one, [&](auto&& take) {
#pragma unroll
        for (int j = 0; j < VALUES; j++) {
            const int i = first + j / 4 * BS_THREADS * 4 + j % 4;
            if (i < a.vocab) take(bs_pack(v[j], (uint32_t)i));
        }
    });
    if (tid == 0) {
        for (int w = 0; w < BS_THREADS / 32; w++) {
            const float2 o = warp_sums[w];
            const float both = w ? fmaxf(m, o.x) : o.x, r = both == -INFINITY ? 0.0f : both;
            s = (w ? s * expf(m - r) : 0.0f) + o.y * expf(o.x - r);
            m = both;
        }
        a.sums[(size_t)row * a.parts + part] = make_float2(m, s);
    }
    for (int i = tid; i < a.keep; i += BS_THREADS) a.lists[((size_t)row * a.parts + part) * a.keep + i] = top.one[i];

    // ---- the block that completes the row merges its lists, where they are merged row by row
    const int request = row / a.beams;
    const u64* lists = a.lists;
    int per_row = a.parts;
    auto count = [&](int* counter, int want) {
        __syncthreads();
        if (tid == 0) {
            int old;
            asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
            done = old == want - 1;
            if (done) *counter = 0;                           // ready for the next launch
        }
        __syncthreads();
        return done != 0;
    };
    if (a.merge_rows) {
        if (!count(a.arrived + row, a.parts)) return;
        const u64* mine = a.lists + (size_t)row * a.parts * a.keep;
        // rank by rank over the parts: the groups' best are then the parts' first ones
        bs_pick(pick.one, a.keep, top.one, [&](auto&& take) {
            for (int e = tid; e < a.parts * a.keep; e += BS_THREADS) take(__ldcg(mine + (size_t)(e % a.parts) * a.keep + e / a.parts));
        });
        for (int i = tid; i < a.keep; i += BS_THREADS) a.row_lists[(size_t)row * a.keep + i] = top.one[i];
        if (!count(a.arrived + BS_MAX_ROWS + request, a.beams)) return;
        lists = a.row_lists;
        per_row = 1;
    } else if (!count(a.arrived + BS_MAX_ROWS + request, a.beams * a.parts)) {
        return;
    }

    // ---- the block that completes the request: the rows' sums, then the best of the rows' lists
    for (int b = warp; b < a.beams; b += BS_THREADS / 32) {
        const float2* ms = a.sums + ((size_t)request * a.beams + b) * a.parts;
        float rm = -INFINITY;
        for (int i = lane; i < a.parts; i += 32) rm = fmaxf(rm, __ldcg(ms + i).x);
        rm = warp_max(rm);
        double sum = 0.0;
        for (int i = lane; i < a.parts; i += 32) {
            const float2 o = __ldcg(ms + i);
            sum += o.x == rm ? (double)o.y : (double)o.y * exp((double)o.x - (double)rm);      // a part without a value above -inf has the sum 0, or NaN
        }
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            const double score = (double)a.scores[request * a.beams + b], lse = (double)rm + log(sum);
            base[b] = isfinite(score) && isfinite(lse) ? score - lse : (double)-INFINITY;
        }
    }
    __syncthreads();
    const int n_lists = a.beams * per_row;
    const u64* mine = lists + (size_t)request * n_lists * a.keep;
    bs_pick(pick.two, a.keep, top.two, [&](auto&& take) {
        for (int e = tid; e < n_lists * a.keep; e += BS_THREADS) {
            const int l = e % n_lists, rank = e / n_lists, b = l / per_row;
            const u64 c = __ldcg(mine + (size_t)l * a.keep + rank);
            uint32_t token = 0xffffffffu - (uint32_t)c;
            double value = base[b] + (double)bs_value((uint32_t)(c >> 32));
            bool there = c != 0;
            if (base[b] == (double)-INFINITY) {                  // its tokens in their order, once a row
                token = (uint32_t)rank;
                value = (double)-INFINITY;
                there = l == b * per_row && rank < a.vocab;
            }
            if (there) take(BsPair{bs_order64(value), 0xffffffffu - ((uint32_t)b * (uint32_t)a.vocab + token)});
        }
    });
    for (int i = tid; i < a.keep; i += BS_THREADS) {
        const BsPair c = top.two[i];
        const uint32_t flat = 0xffffffffu - c.lo;
        const size_t at = (size_t)request * a.keep + i;
        a.out_score[at] = (float)bs_value64(c.hi);
        a.out_parent[at] = (int)(flat / (uint32_t)a.vocab);
        a.out_token[at] = (int)(flat % (uint32_t)a.vocab);
    }
}

struct BsShape { int values, parts, merge_rows; };

// Values a thread holds, blocks a row, and whether rows are merged first; by sizes alone, so that the scratch can be asked for without a device.
static BsShape bs_shape(long long rows, int vocab, int keep, int beams) {
    BsShape s;
    const int small = BS_THREADS * 16, large = BS_THREADS * 32;
    s.values = rows * ((vocab + small - 1) / small) <= 4 * 148 ? 16 : 32;
    const int chunk = s.values == 16 ? small : large;
    s.parts = (vocab + chunk - 1) / chunk;
    s.merge_rows = (long long)beams * s.parts * keep > 4096;
    return s;
}

}  // namespace vk

using namespace vk;

VK_API size_t vk_beam_select_scratch_bytes(int rows, int vocab, int keep) {
    // rows of either shape: as many parts as the shorter chunks make
    const size_t parts = (size_t)(vocab + BS_THREADS * 16 - 1) / (BS_THREADS * 16);
    return (size_t)2 * BS_MAX_ROWS * 4 + rows * parts * 8 + ((size_t)rows * parts * keep + (size_t)rows * keep) * 8;
}

// scratch: vk_beam_select_scratch_bytes bytes for at least as many rows, as large a vocabulary and as many kept; its first 2 * BS_MAX_ROWS words were zero
// at first use and are zero again after every launch.
VK_API int vk_beam_select(const float* logits, const float* scores, float* out_score, int32_t* out_parent, int32_t* out_token, void* scratch, int rows,
                          int beams, int vocab, long long ld, int keep, cudaStream_t stream) {
    if (rows <= 0) return VK_OK;
    if (beams <= 0 || rows % beams || vocab <= 0 || ld < vocab || keep <= 0 || !scratch) return VK_BAD_SHAPE;
    if (beams > BS_MAX_BEAMS || keep > BS_MAX_KEEP || vocab > BS_MAX_PARTS * BS_THREADS * 16 || rows > BS_MAX_ROWS) return VK_TOO_LARGE;
    if ((long long)beams * vocab < keep) return VK_BAD_SHAPE;
    if ((uintptr_t)logits % 4 || (uintptr_t)scratch % 16) return VK_BAD_ALIGNMENT;
    const BsShape s = bs_shape(rows, vocab, keep, beams);
    BsArgs a;
    a.logits = logits; a.scores = scores; a.out_score = out_score; a.out_parent = out_parent; a.out_token = out_token;
    char* at = (char*)scratch;
    a.arrived = (int*)at; at += (size_t)2 * BS_MAX_ROWS * 4;
    a.lists = (u64*)at; at += (size_t)rows * s.parts * keep * 8;
    a.row_lists = (u64*)at; at += (size_t)rows * keep * 8;
    a.sums = (float2*)at;
    a.ld = ld; a.beams = beams; a.vocab = vocab; a.keep = keep; a.parts = s.parts; a.merge_rows = s.merge_rows;
    if (s.values == 16) return launch_dependent(beam_select_kernel<16>, dim3(s.parts, rows), dim3(BS_THREADS), 0, stream, a);
    return launch_dependent(beam_select_kernel<32>, dim3(s.parts, rows), dim3(BS_THREADS), 0, stream, a);
}
