// How a launch of the shared-prefix decode attention is cut into pieces of equal length, worked out on the device.
//
// A family is a run of the member list; its members' block tables agree on the family's first `shared` positions.  Two
// kinds of units are walked, each a key-value head and a run of keys:
//
//   prefix   a tile of up to prefix_rows rows (members x the heads that read one key-value head) of one family over the
//            family's shared keys [0, P); P is at most the smallest position of its members, and 0 for a family of one
//   own      one member's heads (up to own_rows of them) over the keys [P, position] that only it reads
//
// The launch's blocks are divided between the two by what they have to do, so that a block walks one kind only: what limits the prefixes of large families (products) and what limits
// the own keys (memory) is then busy at the same time, and where there is little to do neither waits for the other.  The prefix units, each as its tiles of 16 keys and a number of
// empty tiles that stands for what a unit costs besides its keys, lie one after the other on a line; worker b walks the tiles [b lp, (b+1) lp) of it.  The own units lie on another
// line with workers and a length lo of their own.  So every worker has the same to do whatever the families look like, a unit is cut into at most tiles / l + 2 parts, and a part's
// place among its unit's parts is the worker's number minus that of the unit's first worker.  A part leaves an unnormalised output, a
// maximum and a sum for each of its rows, and a second launch joins a row's parts.
//
// Lengths are read from the step's metadata on the device, so that a captured graph follows them.  They are read, and the parts found, while the kernel before this one may still run (2 us that
// nobody waits for).  What that kernel writes can be seen only behind the wait for it, so the lists are read again there, past the first-level cache, and the parts are found again if any of
// them has changed: a trip to the second-level cache and a barrier for every launch, and right whoever writes the lists.
#pragma once

#include "common.cuh"

namespace vk {

constexpr int SA_MAX_TOKENS = 256, SA_THREADS = 256, SA_MAX_HEADS = 64, SA_MAX_OWN_ROWS = 16, SA_MAX_KV_HEADS = 128;

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
    int4* rows;                    // [n][nh] where a row's parts are: SaRow
    float2* part_ml;               // [rows] maximum (base 2) and sum
    float* part_o;                 // [rows][hd]
    int n, families, tokens, segments, pages, nh, nkv, gq, hd, page_size, page_shift, max_blocks;
    int prefix_rows, own_rows, blocks, own_per_block, min_prefix, min_own, prefix_cost, own_cost;      // own workers a block; the last four in tiles of keys
    float scale_log2, row_unit, tensor_unit;      // row_unit: the rows of a prefix's tile that cost as much as an own tile; tensor_unit: what a tile of tensor_rows or more rows costs, in own tiles
    int tensor_rows;
};

// A row's parts: prefix_parts from prefix_row on and own_parts from own_row on; none: the row was written when it was walked, or its member is not there.
struct SaRow { int prefix_row, prefix_parts, own_row, own_parts; };

struct SaPlan {
    int pbase[SA_MAX_TOKENS + 1], obase[SA_MAX_TOKENS + 1];            // where a family's, a member's units begin on their line, in tiles
    __align__(16) int start[SA_MAX_TOKENS + 4];
    int begin[SA_MAX_TOKENS], width[SA_MAX_TOKENS], first[SA_MAX_TOKENS], shared[SA_MAX_TOKENS];      // of a family: its members, the first that is there, P; start: as given
    int prow[SA_MAX_TOKENS], orow[SA_MAX_TOKENS];                      // where their parts' rows begin
    int tok[SA_MAX_TOKENS], seg[SA_MAX_TOKENS], pos[SA_MAX_TOKENS], grp[SA_MAX_TOKENS];    // of a member; pos -1: not there
    int count[SA_MAX_TOKENS], least[SA_MAX_TOKENS];
    int lp, lo, prefix_blocks, tile_members, own_tiles;
    float weight[SA_THREADS / 32];
    int scan[2][2][SA_THREADS / 32];
};

constexpr int SA_TILE = 16;            // keys: a part's products are whole
__device__ __forceinline__ int sa_tiles(int keys) { return (keys + SA_TILE - 1) / SA_TILE; }
// The most parts that a unit of `keys` keys is cut into.
__device__ __forceinline__ int sa_parts(int keys, int length) { return (sa_tiles(keys) + length - 1) / length + 1; }

// Exclusive scans of two numbers a thread over the block; both totals to every thread.  `warps` is this scan's own.  One barrier.
__device__ __forceinline__ void sa_scan2(int (*warps)[SA_THREADS / 32], int& a, int& b, int& ta, int& tb) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = a, y = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) { x += u; y += v; }
    }
    if (lane == 31) { warps[0][warp] = x; warps[1][warp] = y; }
    __syncthreads();
    int px = 0, py = 0;
    ta = tb = 0;
#pragma unroll
    for (int w = 0; w < SA_THREADS / 32; w++) {
        const int u = warps[0][w], v = warps[1][w];
        if (w < warp) { px += u; py += v; }
        ta += u;
        tb += v;
    }
    a = px + x - a;
    b = py + y - b;
}

// The last i of [0, n) with base[i] <= at (base ascends and base[0] <= at): of units of no length, the one behind them.
__device__ __forceinline__ int sa_find(const int* base, int n, int at) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (base[mid] <= at) lo = mid; else hi = mid;
    }
    return lo;
}

// What a thread has of the lists: of member, family and start threadIdx.x (thread 0 the 257th start too).
struct SaLists { int token, seg, at, shared, start, last; };

__device__ __forceinline__ bool sa_there(const SaArgs& a, int token) { return token >= 0 && token < a.tokens; }
__device__ __forceinline__ SaLists sa_read_lists(const SaArgs& a) {
    const int i = threadIdx.x;
    SaLists l;
    l.token = i < a.n ? __ldcg(a.members + i) : -1;
    l.shared = i < a.families ? __ldcg(a.shared + i) : 0;
    l.start = i <= a.families ? __ldcg(a.starts + i) : 0;
    l.last = i == 0 && a.families == SA_MAX_TOKENS ? __ldcg(a.starts + SA_MAX_TOKENS) : 0;
    l.seg = sa_there(a, l.token) ? __ldcg(a.token_seg + l.token) : -1;
    l.at = sa_there(a, l.token) ? __ldcg(a.positions + l.token) : -1;
    return l;
}
// Whether the lists are still what they were, for the whole block alike.  All of it is asked for at once: a token that has changed says so by itself.
__device__ __forceinline__ bool sa_same_lists(const SaArgs& a, const SaLists& l) {
    const int i = threadIdx.x;
    const int token = i < a.n ? __ldcg(a.members + i) : -1, shared = i < a.families ? __ldcg(a.shared + i) : 0, start = i <= a.families ? __ldcg(a.starts + i) : 0;
    const int last = i == 0 && a.families == SA_MAX_TOKENS ? __ldcg(a.starts + SA_MAX_TOKENS) : 0;
    const int seg = sa_there(a, l.token) ? __ldcg(a.token_seg + l.token) : -1, at = sa_there(a, l.token) ? __ldcg(a.positions + l.token) : -1;
    return !__syncthreads_or((token != l.token) | (shared != l.shared) | (start != l.start) | (last != l.last) | (seg != l.seg) | (at != l.at));
}

// Filled by all SA_THREADS threads of a block.  Numbers that cannot be (a member beyond the batch, a negative position, starts
// that go back) are taken as members that are not there and runs of no length: nothing is read or written for them.
__device__ __forceinline__ void sa_find_parts(const SaArgs& a, const SaLists& lists, SaPlan& p) {
    const int i = threadIdx.x, lane = i & 31, seg = lists.seg, at = lists.at;
    p.start[i] = lists.start;               // zeros behind the last, so that groups of four count no more
    if (i < 4) p.start[SA_MAX_TOKENS + i] = lists.last;
    p.shared[i] = lists.shared;
    p.tok[i] = lists.token;
    p.count[i] = p.width[i] = 0;
    p.begin[i] = p.first[i] = SA_MAX_TOKENS;
    p.least[i] = 0x7fffffff;
    if (i == 0) {
        p.tile_members = a.prefix_rows / a.gq;
        p.own_tiles = (a.gq + a.own_rows - 1) / a.own_rows;
    }
    __syncthreads();
    // the member's family: as many as begin at or before it, the first aside (so families are runs of members even where starts go back); none: before the
    // first or behind all
    int before = 0, behind = 0;
    if (i < a.n) {
#pragma unroll 2
        for (int k = 0; k <= a.families; k += 4) {
            const int4 f = *reinterpret_cast<const int4*>(p.start + k);
            behind |= (f.x > i) | (f.y > i) | (f.z > i) | (f.w > i);
            before += (f.x <= i) + (f.y <= i) + (f.z <= i) + (f.w <= i);
        }
        before -= (a.families / 4 + 1) * 4 - (a.families + 1) + (p.start[a.families] <= i);      // without the zeros, and the end
    }
    const int g = i < a.n && p.start[0] <= i && behind ? before - 1 : -1;
    const bool valid = g >= 0 && seg >= 0 && seg < a.segments && at >= 0;
    const int pos = valid ? (int)min((long long)at, (long long)a.max_blocks * a.page_size - 1) : -1;
    p.seg[i] = seg;
    p.pos[i] = pos;
    p.grp[i] = valid ? g : -1;
    {   // a family's neighbours in the warp count together
        const unsigned same = __match_any_sync(0xffffffffu, g), live = __ballot_sync(0xffffffffu, valid) & same;
        const int least = __reduce_min_sync(same, valid ? pos : 0x7fffffff);
        if (g >= 0 && lane == __ffs(same) - 1) {
            atomicAdd(&p.width[g], __popc(same));
            atomicMin(&p.begin[g], i);
            if (live) {
                atomicAdd(&p.count[g], __popc(live));
                atomicMin(&p.first[g], i - lane + __ffs(live) - 1);
                atomicMin(&p.least[g], least);
            }
        }
    }
    __syncthreads();
    auto common = [&](int f) { return p.count[f] > 1 ? max(0, min(p.shared[f], p.least[f])) : 0; };
    const int P = i < a.families ? common(i) : 0, width = p.width[i], tiles = (width + p.tile_members - 1) / p.tile_members;
    const int own = valid ? pos + 1 - common(g) : 0;
    int wp = P > 0 ? (sa_tiles(P) + a.prefix_cost) * tiles * a.nkv : 0, wo = own > 0 ? (sa_tiles(own) + a.own_cost) * p.own_tiles * a.nkv : 0, tp, to;
    const int rows = min(width, p.tile_members) * a.gq;
    const float weight = warp_sum((float)wp * (rows >= a.tensor_rows ? a.tensor_unit : fmaxf(1.0f, (float)rows / a.row_unit)));
    if (lane == 0) p.weight[i >> 5] = weight;
    sa_scan2(p.scan[0], wp, wo, tp, to);
    p.shared[i] = P;                        // behind the barrier: until then it is what was claimed
    p.pbase[i] = wp;
    p.obase[i] = wo;
    float all = 0.0f;
#pragma unroll
    for (int w = 0; w < SA_THREADS / 32; w++) all += p.weight[w];
    const int blocks = tp > 0 ? min(max((int)((float)a.blocks * all / (all + (float)to) + 0.5f), 1), a.blocks - 1) : 0, own_workers = (a.blocks - blocks) * a.own_per_block;
    const int lp = max(blocks > 0 ? (tp + blocks - 1) / blocks : 1, a.min_prefix), lo = max((to + own_workers - 1) / own_workers, a.min_own);
    if (i == 0) {
        p.pbase[SA_MAX_TOKENS] = tp;
        p.obase[SA_MAX_TOKENS] = to;
        p.prefix_blocks = blocks;
        p.lp = lp;
        p.lo = lo;
    }
    int rp = P > 0 ? width * a.nh * sa_parts(P, lp) : 0, ro = own > 0 ? a.nh * sa_parts(own, lo) : 0;
    sa_scan2(p.scan[1], rp, ro, tp, to);
    p.prow[i] = rp;
    p.orow[i] = tp + ro;          // behind the prefix rows
    __syncthreads();
}

// The plan, and the wait for the kernel before this one.
__device__ __forceinline__ void sa_make_plan(const SaArgs& a, SaPlan& p) {
#pragma unroll 1
    for (int again = 0; again < 2; again++) {
        const SaLists lists = sa_read_lists(a);
        sa_find_parts(a, lists, p);
        if (again == 0) {
            dependency_wait();
            if (sa_same_lists(a, lists)) break;
        }
    }
}

// A part of a unit: what a worker walks before it leaves rows behind.
struct SaPart {
    int g, i0, i1;        // the family and the unit's members [i0, i1)
    int kvh, h0, heads;   // the first of the heads (counted inside the key-value head's) and how many of each member's
    int k0, k1;           // its keys
    int row0, stride;     // row of (member i0, head h0) and rows between neighbours: a row's parts lie together
    const int32_t* table;
};

// The part of a prefix unit at tile `at` of the line, for the worker that walks up to `end`; `at` moves behind it.  False: the unit's keys end before `at`.
__device__ __forceinline__ bool sa_prefix_part(const SaArgs& a, const SaPlan& p, int& at, int end, int worker, SaPart& r) {
    r.g = sa_find(p.pbase, SA_MAX_TOKENS, at);
    const int P = p.shared[r.g], width = p.width[r.g], full = sa_tiles(P), length = full + a.prefix_cost;
    const int tiles = (width + p.tile_members - 1) / p.tile_members;
    const int rel = at - p.pbase[r.g], u = rel / length, t = rel - u * length, off = at - t;
    at = min(end, off + length);
    if (t >= full) return false;
    r.kvh = u / tiles;
    r.i0 = p.begin[r.g] + (u - r.kvh * tiles) * p.tile_members;
    r.i1 = min(r.i0 + p.tile_members, p.begin[r.g] + width);
    r.h0 = 0;
    r.heads = a.gq;
    r.k0 = t * SA_TILE;
    r.k1 = min(P, (at - off) * SA_TILE);
    r.stride = sa_parts(P, p.lp);
    r.row0 = p.prow[r.g] + (r.kvh * width + r.i0 - p.begin[r.g]) * a.gq * r.stride + (worker - off / p.lp);
    r.table = a.block_tables + (size_t)p.seg[p.first[r.g]] * a.max_blocks;
    return true;
}

// The same of an own unit; `parts`: of how many parts the unit is one.
__device__ __forceinline__ bool sa_own_part(const SaArgs& a, const SaPlan& p, int& at, int end, int worker, SaPart& r, int& parts) {
    r.i0 = sa_find(p.obase, SA_MAX_TOKENS, at);
    r.i1 = r.i0 + 1;
    r.g = p.grp[r.i0];
    const int P = p.shared[r.g], own = p.pos[r.i0] + 1 - P, full = sa_tiles(own), length = full + a.own_cost;
    const int rel = at - p.obase[r.i0], u = rel / length, t = rel - u * length, off = at - t;
    at = min(end, off + length);
    if (t >= full) return false;
    r.kvh = u / p.own_tiles;
    r.h0 = (u - r.kvh * p.own_tiles) * a.own_rows;
    r.heads = min(a.own_rows, a.gq - r.h0);
    r.k0 = P + t * SA_TILE;
    r.k1 = P + min(own, (at - off) * SA_TILE);
    r.stride = sa_parts(own, p.lo);
    const int first = off / p.lo;
    parts = (off + full - 1) / p.lo - first + 1;
    r.row0 = p.orow[r.i0] + (r.kvh * a.gq + r.h0) * r.stride + (worker - first);
    r.table = a.block_tables + (size_t)p.seg[r.i0] * a.max_blocks;
    return true;
}

// How many parts the rows of (member, key-value head) get from the family's prefix, and from the member's own tile of heads.
__device__ __forceinline__ int sa_prefix_parts(const SaArgs& a, const SaPlan& p, int i, int kvh) {
    const int g = p.grp[i], P = p.shared[g];
    if (P == 0) return 0;
    const int width = p.width[g], tiles = (width + p.tile_members - 1) / p.tile_members, full = sa_tiles(P);
    const int off = p.pbase[g] + (kvh * tiles + (i - p.begin[g]) / p.tile_members) * (full + a.prefix_cost);
    return (off + full - 1) / p.lp - off / p.lp + 1;
}
__device__ __forceinline__ int sa_own_parts(const SaArgs& a, const SaPlan& p, int i, int kvh, int tile) {
    const int full = sa_tiles(p.pos[i] + 1 - p.shared[p.grp[i]]);
    const int off = p.obase[i] + (kvh * p.own_tiles + tile) * (full + a.own_cost);
    return (off + full - 1) / p.lo - off / p.lo + 1;
}

// A block's share of the rows' table, by one thread a row.
__device__ __forceinline__ void sa_write_rows(const SaArgs& a, const SaPlan& p) {
    for (int r = blockIdx.x + threadIdx.x * gridDim.x; r < a.n * a.nh; r += gridDim.x * SA_THREADS) {
        const int i = r / a.nh, head = r - i * a.nh, kvh = head / a.gq, h = head - kvh * a.gq, g = p.grp[i];
        int4 row = make_int4(0, 0, 0, 0);
        if (g >= 0) {
            const int P = p.shared[g], own = p.pos[i] + 1 - P, width = p.width[g];
            const int np = sa_prefix_parts(a, p, i, kvh), no = sa_own_parts(a, p, i, kvh, h / a.own_rows);
            if (np > 0 || no > 1)
                row = make_int4(np > 0 ? p.prow[g] + ((kvh * width + i - p.begin[g]) * a.gq + h) * sa_parts(P, p.lp) : 0, np,
                                p.orow[i] + head * sa_parts(own, p.lo), no);
        }
        a.rows[r] = row;
    }
}

__device__ __forceinline__ float sa_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// For the launches that walk every member by itself, in clusters: what another block of the cluster has in its shared memory.
__device__ __forceinline__ uint32_t sa_of_rank(const void* p, int rank) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return at;
}
__device__ __forceinline__ float sa_remote(uint32_t at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void sa_cluster_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The member, tile of `rows` heads and run of keys of a block of such a launch (grid: blocks of a cluster, tiles of heads of every key-value head, members); false: nothing of it is there, for the
// whole cluster alike.  The lists are read behind the wait for the kernel before this one, which may have written them (before it and once more behind it, as for the plan, is the slower way here, 11.2 us
// against ten for six requests of five beams; before it alone was 9.6).
__device__ __forceinline__ bool sa_each_part(const SaArgs& a, int rows, SaPart& part, int& token) {
    const int i = blockIdx.z, tid = threadIdx.x, ranks = gridDim.x;
    dependency_wait();
    token = a.members[i];
    const bool there = token >= 0 && token < a.tokens;
    const int seg = there ? a.token_seg[token] : -1, at = there ? a.positions[token] : -1, first = a.starts[0];
    bool behind = false;
    for (int f = tid; f < a.families; f += blockDim.x) behind |= a.starts[f + 1] > i;
    behind = __syncthreads_or(behind);
    if (!behind || first > i || seg < 0 || seg >= a.segments || at < 0) return false;
    const int keys = (int)min((long long)at, (long long)a.max_blocks * a.page_size - 1) + 1;
    const int tiles = (a.gq + rows - 1) / rows, run = (sa_tiles(keys) + ranks - 1) / ranks * SA_TILE;
    part.kvh = blockIdx.y / tiles;
    part.h0 = (blockIdx.y - part.kvh * tiles) * rows;
    part.heads = min(rows, a.gq - part.h0);
    part.k0 = min((int)blockIdx.x * run, keys);
    part.k1 = min(part.k0 + run, keys);
    part.table = a.block_tables + (size_t)seg * a.max_blocks;
    return true;
}

// The outputs of a block's warps ([warps][rows][ld], maxima and sums [warps][rows]) meet, and then the cluster's blocks': `whole` [rows][hd], row_m and row_l [rows] are this block's for the others.
// No score above -inf anywhere: every weight is 0, and the result no number.
template <typename T, int WARPS>
__device__ __forceinline__ void sa_each_join(const SaArgs& a, const SaPart& part, int token, int rows, int ld, const float* out, const float2* ml, float* whole, float* row_m, float* row_l) {
    const int tid = threadIdx.x, ranks = gridDim.x, hd = a.hd, values = part.heads * hd;
    T* to = static_cast<T*>(a.out) + ((size_t)token * a.nh + part.kvh * a.gq + part.h0) * hd;
#pragma unroll 1
    for (int c = tid; c < values; c += WARPS * 32) {
        const int row = c / hd, d = c - row * hd;
        float m = -INFINITY, l = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) m = fmaxf(m, ml[w * rows + row].x);
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float e = sa_ex2(ml[w * rows + row].x - ref);
            l += ml[w * rows + row].y * e;
            o += out[(w * rows + row) * ld + d] * e;
        }
        if (ranks == 1) {
            to[c] = from_f32<T>(o / l);
        } else {
            whole[c] = o;
            if (d == 0) {
                row_m[row] = m;
                row_l[row] = l;
            }
        }
    }
    if (ranks == 1) return;
    sa_cluster_meet();
#pragma unroll 1
    for (int c = blockIdx.x * WARPS * 32 + tid; c < values; c += ranks * WARPS * 32) {      // every block a share of the values
        const int row = c / hd;
        float m = -INFINITY, l = 0.0f, o = 0.0f, rm[8];
#pragma unroll
        for (int r = 0; r < 8; r++) {
            rm[r] = r < ranks ? sa_remote(sa_of_rank(&row_m[row], r)) : -INFINITY;
            m = fmaxf(m, rm[r]);
        }
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int r = 0; r < 8; r++) {
            if (r >= ranks) break;
            const float e = sa_ex2(rm[r] - ref);
            l += sa_remote(sa_of_rank(&row_l[row], r)) * e;
            o += sa_remote(sa_of_rank(&whole[c], r)) * e;
        }
        to[c] = from_f32<T>(o / l);
    }
    sa_cluster_meet();                                        // nobody leaves while another reads its shared memory
}

constexpr int SA_MAX_MULTIPROCESSORS = 160;         // of the sm_100a parts; the scratch is laid out for this many

// Allows a kernel more than 48 KB of shared memory on the current device, asked for again only where a launch needs more than was allowed before.
template <typename... Args> inline int sa_allow_smem(void (*kernel)(Args...), size_t bytes) {
    struct Allowed { void (*kernel)(Args...); int device; size_t bytes; };
    static thread_local Allowed known[8];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    Allowed* slot = nullptr;
    for (Allowed& k : known) {
        if (k.kernel == kernel && k.device == dev) { slot = &k; break; }
        if (!slot && !k.kernel) slot = &k;
    }
    if (slot && slot->kernel == kernel && slot->bytes >= bytes) return VK_OK;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && slot) *slot = Allowed{kernel, dev, bytes};
    return (int)e;
}

// attention_shared_mma.cu
bool attention_shared_mma_takes(const SaArgs& a, int dtype);
int launch_attention_shared_mma(SaArgs a, int multiprocessors, int* error, cudaStream_t stream);
bool attention_each_mma_takes(const SaArgs& a);
int launch_attention_each_mma(const SaArgs& a, int multiprocessors, cudaStream_t stream);

}  // namespace vk
