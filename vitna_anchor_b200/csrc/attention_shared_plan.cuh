// How a launch of the shared-prefix decode attention is cut into pieces of equal length, worked out on the device.
//
// A family is a run of the member list; its members' block tables agree on the family's first `shared` positions.  Two
// kinds of units are walked, each a key-value head and a run of keys:
//
//   prefix   a tile of up to PREFIX_ROWS rows (members x the heads that read one key-value head) of one family over the
//            family's shared keys [0, P); P is at most the smallest position of its members, and 0 for a family of one
//   own      one member's heads (up to OWN_ROWS of them) over the keys [P, position] that only it reads
//
// The prefix units' keys, one unit after the other, are one line of Wp keys; worker b walks [b Lp, (b+1) Lp) of it.  The
// own units are another line of Wo keys with workers and a length Lo of their own.  So every worker has the same number of
// keys whatever the families look like, a unit is cut into at most ceil(P / Lp) + 1 parts, and a part's place among its
// unit's parts is the worker's number minus that of the unit's first worker.  A part leaves an unnormalised output, a
// maximum and a sum for each of its rows; whoever brings a (member, key-value head) its last part joins them.
//
// Lengths are read from the step's metadata on the device, so that a captured graph follows them.
#pragma once

#include "common.cuh"

namespace vk {

constexpr int SA_MAX_TOKENS = 256, SA_THREADS = 256, SA_PREFIX_ROWS = 64, SA_OWN_ROWS = 16, SA_MAX_KV_HEADS = 128;

struct SaArgs {
    const void* q;                 // [tokens][nh][hd]
    const void* cache;             // [pages][2][nkv][page_size][hd]
    const int32_t* block_tables;   // [segments][max_blocks]
    const int32_t* token_seg;      // [tokens]
    const int32_t* positions;      // [tokens]
    const int32_t* members;        // [n] tokens, family after family
    const int32_t* starts;         // [families + 1]
    const int32_t* shared;         // [families]
    void* out;                     // [tokens][nh][hd]
    int* counters;                 // [SA_MAX_TOKENS][nkv], zero between launches
    float2* part_ml;               // [rows] maximum (base 2) and sum
    float* part_o;                 // [rows][hd]
    int n, families, tokens, segments, pages, nh, nkv, gq, hd, page_size, page_shift, max_blocks;
    int prefix_workers, own_workers, min_prefix, min_own;
    float scale_log2;
};

struct SaPlan {
    long long pbase[SA_MAX_TOKENS + 1], obase[SA_MAX_TOKENS + 1];      // where a family's, a member's units begin on their line
    int start[SA_MAX_TOKENS + 1], first[SA_MAX_TOKENS], shared[SA_MAX_TOKENS];
    int prow[SA_MAX_TOKENS + 1], orow[SA_MAX_TOKENS + 1];              // where their parts' rows begin
    int tok[SA_MAX_TOKENS], pos[SA_MAX_TOKENS], grp[SA_MAX_TOKENS];    // of a member; pos -1: not there
    int count[SA_MAX_TOKENS], least[SA_MAX_TOKENS];
    int lp, lo, tile_members, own_tiles;
    long long scan[2][SA_THREADS / 32];
};

// The most parts that a unit of `keys` keys is cut into.
__device__ __forceinline__ int sa_parts(int keys, int length) { return (keys + length - 1) / length + 1; }

// Exclusive scans of two numbers a thread over the block; both totals to every thread.
__device__ __forceinline__ void sa_scan2(long long (*warps)[SA_THREADS / 32], long long& a, long long& b, long long& ta, long long& tb) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x = a, y = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) { x += u; y += v; }
    }
    __syncthreads();
    if (lane == 31) { warps[0][warp] = x; warps[1][warp] = y; }
    __syncthreads();
    long long px = 0, py = 0;
    ta = tb = 0;
#pragma unroll
    for (int w = 0; w < SA_THREADS / 32; w++) {
        if (w < warp) { px += warps[0][w]; py += warps[1][w]; }
        ta += warps[0][w];
        tb += warps[1][w];
    }
    a = px + x - a;
    b = py + y - b;
}

// The last i of [0, n) with base[i] <= at (base ascends and base[0] <= at): of units of no length, the one behind them.
__device__ __forceinline__ int sa_find(const long long* base, int n, long long at) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (base[mid] <= at) lo = mid; else hi = mid;
    }
    return lo;
}

// Filled by all SA_THREADS threads of a block.  Numbers that cannot be (a member beyond the batch, a negative position, starts
// that go back) are taken as members that are not there and runs of no length: nothing is read or written for them.
__device__ __forceinline__ void sa_make_plan(const SaArgs& a, SaPlan& p) {
    const int i = threadIdx.x, lane = i & 31, warp = i >> 5;
    // starts, made to ascend: a running maximum
    int s = i < a.families ? min(max(a.starts[i], 0), a.n) : 0;
    const int token = i < a.n ? a.members[i] : -1;
    const int shared_i = i < a.families ? a.shared[i] : 0;
    const bool there = token >= 0 && token < a.tokens;
    const int seg = there ? a.token_seg[token] : -1;
    int pos = there && seg >= 0 && seg < a.segments ? a.positions[token] : -1;
    pos = (int)min((long long)pos, (long long)a.max_blocks * a.page_size - 1);
    p.tok[i] = token;
    p.pos[i] = pos;
    p.count[i] = 0;
    p.first[i] = SA_MAX_TOKENS;
    p.least[i] = 0x7fffffff;
    int* tops = reinterpret_cast<int*>(p.scan);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s = max(s, v);
    }
    if (lane == 31) tops[warp] = s;
    __syncthreads();
    for (int w = 0; w < warp; w++) s = max(s, tops[w]);
    if (i < a.families) p.start[i] = s;
    if (i == a.families - 1) p.start[a.families] = max(s, min(a.starts[a.families], a.n));
    __syncthreads();
    int g = -1;
    if (pos >= 0 && i >= p.start[0] && i < p.start[a.families]) {        // the last family that begins at or before the member
        int lo = 0, hi = a.families;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.start[mid] <= i) lo = mid; else hi = mid;
        }
        g = lo;
        atomicAdd(&p.count[g], 1);
        atomicMin(&p.first[g], i);
        atomicMin(&p.least[g], pos);
    }
    p.grp[i] = g;
    if (i == 0) {
        p.tile_members = max(1, SA_PREFIX_ROWS / a.gq);
        p.own_tiles = (a.gq + SA_OWN_ROWS - 1) / SA_OWN_ROWS;
    }
    __syncthreads();
    const int P = i < a.families && p.count[i] > 1 ? max(0, min(shared_i, p.least[i])) : 0;
    p.shared[i] = P;
    const int width = i < a.families ? p.start[i + 1] - p.start[i] : 0;
    const int tiles = (width + p.tile_members - 1) / p.tile_members;
    __syncthreads();
    const int own = g >= 0 ? pos + 1 - p.shared[g] : 0;
    long long wp = (long long)P * tiles * a.nkv, wo = (long long)own * p.own_tiles * a.nkv, tp, to;
    sa_scan2(p.scan, wp, wo, tp, to);
    p.pbase[i] = wp;
    p.obase[i] = wo;
    if (i == 0) {
        p.pbase[SA_MAX_TOKENS] = tp;
        p.obase[SA_MAX_TOKENS] = to;
        // a multiple of 16 keys, so that a part's products are whole
        const long long lp = (tp + a.prefix_workers - 1) / a.prefix_workers, lo = (to + a.own_workers - 1) / a.own_workers;
        p.lp = (int)min(max((lp + 15) / 16 * 16, (long long)a.min_prefix), 0x7ffffff0ll);
        p.lo = (int)min(max((lo + 15) / 16 * 16, (long long)a.min_own), 0x7ffffff0ll);
    }
    __syncthreads();
    long long rp = P > 0 ? (long long)width * a.nh * sa_parts(P, p.lp) : 0, ro = own > 0 ? (long long)a.nh * sa_parts(own, p.lo) : 0;
    sa_scan2(p.scan, rp, ro, tp, to);
    p.prow[i] = (int)rp;
    p.orow[i] = (int)(tp + ro);          // behind the prefix rows
    __syncthreads();
}

// A part of a unit: what a worker walks before it leaves rows behind.
struct SaPart {
    int g, i0, i1;        // the family and the unit's members [i0, i1)
    int kvh, h0, heads;   // the first of the heads (counted inside the key-value head's) and how many of each member's
    int k0, k1;           // its keys
    int row0, stride;     // row of (member i0, head h0) and rows between neighbours: a row's parts lie together
    const int32_t* table;
};

__device__ __forceinline__ SaPart sa_prefix_part(const SaArgs& a, const SaPlan& p, long long at, long long end, int worker) {
    SaPart r;
    r.g = sa_find(p.pbase, SA_MAX_TOKENS, at);
    const int P = p.shared[r.g], width = p.start[r.g + 1] - p.start[r.g];
    const int tiles = (width + p.tile_members - 1) / p.tile_members;
    const long long rel = at - p.pbase[r.g];
    const int u = (int)(rel / P);
    r.kvh = u / tiles;
    const int tile = u - r.kvh * tiles;
    r.i0 = p.start[r.g] + tile * p.tile_members;
    r.i1 = min(r.i0 + p.tile_members, p.start[r.g + 1]);
    r.h0 = 0;
    r.heads = a.gq;
    r.k0 = (int)(rel - (long long)u * P);
    r.k1 = (int)min((long long)P, r.k0 + (end - at));
    r.stride = sa_parts(P, p.lp);
    const int first = (int)((p.pbase[r.g] + (long long)u * P) / p.lp);
    r.row0 = p.prow[r.g] + (r.kvh * width + r.i0 - p.start[r.g]) * a.gq * r.stride + (worker - first);
    r.table = a.block_tables + (size_t)a.token_seg[p.tok[p.first[r.g]]] * a.max_blocks;
    return r;
}

// `parts`: of how many parts the unit is one.
__device__ __forceinline__ SaPart sa_own_part(const SaArgs& a, const SaPlan& p, long long at, long long end, int worker, int& parts) {
    SaPart r;
    r.i0 = sa_find(p.obase, SA_MAX_TOKENS, at);
    r.i1 = r.i0 + 1;
    r.g = p.grp[r.i0];
    const int P = p.shared[r.g], own = p.pos[r.i0] + 1 - P;
    const long long rel = at - p.obase[r.i0];
    const int u = (int)(rel / own);
    r.kvh = u / p.own_tiles;
    r.h0 = (u - r.kvh * p.own_tiles) * SA_OWN_ROWS;
    r.heads = min(SA_OWN_ROWS, a.gq - r.h0);
    const int k = (int)(rel - (long long)u * own);
    r.k0 = P + k;
    r.k1 = P + (int)min((long long)own, k + (end - at));
    r.stride = sa_parts(own, p.lo);
    const long long off = p.obase[r.i0] + (long long)u * own;
    const int first = (int)(off / p.lo);
    parts = (int)((off + own - 1) / p.lo) - first + 1;
    r.row0 = p.orow[r.i0] + (r.kvh * a.gq + r.h0) * r.stride + (worker - first);
    r.table = a.block_tables + (size_t)a.token_seg[p.tok[r.i0]] * a.max_blocks;
    return r;
}

// How many parts the rows of (member, key-value head) get from the family's prefix, and from the member's own tile of heads.
__device__ __forceinline__ int sa_prefix_parts(const SaPlan& p, int i, int kvh) {
    const int g = p.grp[i], P = p.shared[g];
    if (P == 0) return 0;
    const int width = p.start[g + 1] - p.start[g], tiles = (width + p.tile_members - 1) / p.tile_members;
    const long long off = p.pbase[g] + (long long)(kvh * tiles + (i - p.start[g]) / p.tile_members) * P;
    return (int)((off + P - 1) / p.lp) - (int)(off / p.lp) + 1;
}
__device__ __forceinline__ int sa_own_parts(const SaPlan& p, int i, int kvh, int tile) {
    const int own = p.pos[i] + 1 - p.shared[p.grp[i]];
    const long long off = p.obase[i] + (long long)(kvh * p.own_tiles + tile) * own;
    return (int)((off + own - 1) / p.lo) - (int)(off / p.lo) + 1;
}

__device__ __forceinline__ float sa_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Counts one part of (member i, key-value head); true for the caller that brings the last one, which then sees the others' rows.
// The caller's own rows are written by threads of its block or warp that have met (__syncthreads, __syncwarp) since.
__device__ __forceinline__ bool sa_last(const SaArgs& a, const SaPlan& p, int i, int kvh) {
    int want = sa_prefix_parts(p, i, kvh);
    for (int tile = 0; tile < p.own_tiles; tile++) want += sa_own_parts(p, i, kvh, tile);
    int* counter = a.counters + i * a.nkv + kvh;
    int old;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
    const bool last = old == want - 1;
    if (last) *counter = 0;              // ready for the next launch
    return last;
}

// A warp joins the parts of head h of (member i, key-value head): weights exp(own maximum - row maximum), in the parts' order, prefix first.
// Lane j reads the j-th part's maximum and sum, and dims j, j + 32, ... of every part.
template <typename T, int DIMS>
__device__ __forceinline__ void sa_join(const SaArgs& a, const SaPlan& p, int i, int kvh, int h) {
    const int lane = threadIdx.x & 31;
    const int g = p.grp[i], P = p.shared[g], own = p.pos[i] + 1 - P, width = p.start[g + 1] - p.start[g];
    const int np = sa_prefix_parts(p, i, kvh), no = sa_own_parts(p, i, kvh, h / SA_OWN_ROWS);
    const int prow = P > 0 ? p.prow[g] + ((kvh * width + i - p.start[g]) * a.gq + h) * sa_parts(P, p.lp) : 0;
    const int orow = p.orow[i] + (kvh * a.gq + h) * sa_parts(own, p.lo);
    float m = -INFINITY, l = 0.0f, o[DIMS];
#pragma unroll
    for (int d = 0; d < DIMS; d++) o[d] = 0.0f;
    for (int j0 = 0; j0 < np + no; j0 += 32) {
        const int j = j0 + lane;
        const bool on = j < np + no;
        const int row = j < np ? prow + j : orow + j - np;
        const float2 ml = on ? __ldcg(a.part_ml + row) : make_float2(-INFINITY, 0.0f);
        const float top = fmaxf(m, warp_max(ml.x)), ref = top == -INFINITY ? 0.0f : top;      // no score above -inf so far: every weight is 0
        const float keep = sa_ex2(m - ref), w = sa_ex2(ml.x - ref);
        l = l * keep + warp_sum(on ? ml.y * w : 0.0f);
#pragma unroll
        for (int d = 0; d < DIMS; d++) o[d] *= keep;
        m = top;
        const int count = min(32, np + no - j0);
#pragma unroll 4
        for (int c = 0; c < count; c++) {
            const float wc = __shfl_sync(0xffffffffu, w, c);
            const float* po = a.part_o + (size_t)__shfl_sync(0xffffffffu, row, c) * a.hd;
#pragma unroll
            for (int d = 0; d < DIMS; d++)
                if (lane + 32 * d < a.hd) o[d] += __ldcg(po + lane + 32 * d) * wc;
        }
    }
    T* out = static_cast<T*>(a.out) + ((size_t)p.tok[i] * a.nh + kvh * a.gq + h) * a.hd;
#pragma unroll
    for (int d = 0; d < DIMS; d++)
        if (lane + 32 * d < a.hd) out[lane + 32 * d] = from_f32<T>(o[d] / l);
}

}  // namespace vk
