// Decode attention of requests that hold their first pages in common: beams of one prompt, requests behind one prefix.
//
//   out[t][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[t][h] . k_j),  j = 0 .. position(t) over t's block table
//
// Attention over separate block tables reads the common keys once a request.  Here a family's members are the rows of one product over
// the keys they share, which are read once, and the keys that a member has alone are walked by themselves; the two meet by their maxima
// and sums, which stay in float32 like everything between the scores and the output's rounding.  How the walks are cut: attention_shared_plan.cuh.
//
// This file has the entry point, the launch that joins the parts, and the kernel that takes every size and both types, on the float32 units.
// attention_shared_mma.cu has bfloat16 heads of 64 and 128 on the tensor cores.
//
// The float32 kernel: a warp holds up to eight rows against 32 keys.  Lane j has key j's scores of all the rows (a piece of its key is read once for the eight, the queries come as
// broadcasts), the weights go through shared memory, and then the lane has dims j, j + 32, ... of the rows' outputs (a value once for the eight, the weights as broadcasts of four keys).
// Of the scores 9 reads of 16 bytes from shared memory then serve 32 multiply-adds a lane; a row at a time takes 2 for 4.
// R = 1, 2, 4 or 8 warps that cover a prefix's rows share the tiles of their keys; own keys are walked by single warps.
#include "attention_shared_plan.cuh"

#include <atomic>

namespace vk {

constexpr int SG_KEYS = 32, SG_ROWS = 8, SG_WARPS = SA_THREADS / 32, SG_PREFIX_ROWS = SG_ROWS * SG_WARPS;      // of a warp's tile; rows a block

// Tiles of keys and values that a block holds, for as many warps that walk keys of their own: heads of up to 64 leave room for two blocks a multiprocessor with four each.
__host__ __device__ inline int sg_slots(int hd) { return hd <= 128 ? 4 : 2; }
static int sg_blocks(int hd) { return hd <= 64 ? 2 : 1; }
// Shared memory: the plan; the rows' queries [64][hd], where the groups' outputs meet later, and their maxima and sums [64]; the warps' weights [8][8][32]; the slots' keys and values [32][hd + 4].
__host__ __device__ inline size_t sg_plan_bytes() { return (sizeof(SaPlan) + 15) / 16 * 16; }
static size_t sg_smem(int hd) {
    return sg_plan_bytes() + (size_t)SG_PREFIX_ROWS * (hd * 4 + 8) + (size_t)SG_WARPS * SG_ROWS * SG_KEYS * 4 + (size_t)sg_slots(hd) * 2 * SG_KEYS * (hd + 4) * 4;
}

struct SgRows {
    float *q, *weights, *k, *v;      // the warp's queries [8][hd], weights [8][32], and its group's tile
    int warps, place;                // of the group, and this warp's place in it
    int barrier;                     // the group's, where it has more warps than one
};

// A row's reference maximum is moved only when a score is more than 8 (in base 2) above it, see attention_shared_mma.cu.
constexpr float SG_AHEAD = 8.0f;

// A group of warps walks tiles tile0, tile0 + step, ... of 32 keys of a part; this warp for its NR rows, whose queries are in w.q.
template <typename T, int DIMS, int NR>
__device__ __forceinline__ void sg_walk(const SaArgs& a, const SaPart& part, int tile0, int step, const SgRows& w, float (&m)[NR], float (&l)[NR], float (&o)[NR][DIMS]) {
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x & 31, hd = a.hd, ld = hd + 4, vec = hd / N;
    auto meet = [&]() {
        if (w.warps == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(w.barrier), "r"(w.warps * 32) : "memory");
    };
#pragma unroll
    for (int r = 0; r < NR; r++) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int d = 0; d < DIMS; d++) o[r][d] = 0.0f;
    }
    for (int kb = part.k0 + tile0 * SG_KEYS; kb < part.k1; kb += step * SG_KEYS) {
        meet();                                             // the group is past the tile before
#pragma unroll 4
        for (int c = w.place * 32 + lane; c < SG_KEYS * vec; c += w.warps * 32) {
            const int kl = c / vec, d = c % vec * N, key = kb + kl;
            const T* src = nullptr;
            if (key < part.k1) {
                const int block = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size, page = part.table[block];
                if (page >= 0 && page < a.pages) src = static_cast<const T*>(a.cache) + (((size_t)page * 2 * a.nkv + part.kvh) * a.page_size + key - block * a.page_size) * hd + d;
            }
            const size_t to_value = (size_t)a.nkv * a.page_size * hd;
            if (sizeof(T) == 4) {                           // no key: nothing of it may be read, not even a NaN
                copy16_or_zero(w.k + kl * ld + d, reinterpret_cast<const float*>(src ? src : static_cast<const T*>(a.cache)), src != nullptr);
                copy16_or_zero(w.v + kl * ld + d, reinterpret_cast<const float*>(src ? src + to_value : static_cast<const T*>(a.cache)), src != nullptr);
            } else {
                float fk[N], fv[N];
#pragma unroll
                for (int e = 0; e < N; e++) fk[e] = fv[e] = 0.0f;
                if (src) {
                    load16<T>(src, fk);
                    load16<T>(src + to_value, fv);
                }
#pragma unroll
                for (int e = 0; e < N; e++) { w.k[kl * ld + d + e] = fk[e]; w.v[kl * ld + d + e] = fv[e]; }
            }
        }
        if (sizeof(T) == 4) asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
        meet();
        float s[NR];
#pragma unroll
        for (int r = 0; r < NR; r++) s[r] = 0.0f;
#pragma unroll 2
        for (int d = 0; d < hd; d += 4) {
            const float4 k = *reinterpret_cast<const float4*>(w.k + lane * ld + d);
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const float4 q = *reinterpret_cast<const float4*>(w.q + r * hd + d);
                s[r] += q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
            }
        }
        bool ahead = false;
#pragma unroll
        for (int r = 0; r < NR; r++) {
            if (kb + lane >= part.k1) s[r] = -INFINITY;
            ahead |= s[r] > m[r] + SG_AHEAD;
        }
        if (__any_sync(0xffffffffu, ahead)) {
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const float top = fmaxf(m[r], warp_max(s[r])), keep = top == -INFINITY ? 0.0f : exp2f(m[r] - top);
                m[r] = top;
                l[r] *= keep;
#pragma unroll
                for (int d = 0; d < DIMS; d++) o[r][d] *= keep;
            }
        }
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const float p = exp2f(s[r] - (m[r] == -INFINITY ? 0.0f : m[r]));       // no score above -inf so far: nothing
            l[r] += p;
            w.weights[r * SG_KEYS + lane] = p;
        }
        __syncwarp();
        const int keys = min(SG_KEYS, part.k1 - kb);
        for (int k = 0; k < keys; k += 4) {                 // behind the last key weights and values are zeros
            float v[4][DIMS];
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int d = 0; d < DIMS; d++) v[e][d] = lane + 32 * d < hd ? w.v[(k + e) * ld + lane + 32 * d] : 0.0f;
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const float4 p = *reinterpret_cast<const float4*>(w.weights + r * SG_KEYS + k);
#pragma unroll
                for (int d = 0; d < DIMS; d++) o[r][d] += p.x * v[0][d] + p.y * v[1][d] + p.z * v[2][d] + p.w * v[3][d];
            }
        }
    }
#pragma unroll
    for (int r = 0; r < NR; r++) l[r] = warp_sum(l[r]);
}

// The warp's rows' queries, scaled, into w.q; zeros where there is no such row, or its member is not there.
template <typename T> __device__ __forceinline__ void sg_queries(const SaArgs& a, const SaPlan& p, const SaPart& part, int row0, int rows, const SgRows& w) {
    constexpr int N = Vec16<T>::N;
    const int vec = a.hd / N;
    for (int c = threadIdx.x & 31; c < SG_ROWS * vec; c += 32) {
        const int r = c / vec, d = c % vec * N, row = row0 + r, i = part.i0 + row / part.heads;
        float f[N];
        if (row < rows && p.pos[i] >= 0) load16<T>(static_cast<const T*>(a.q) + ((size_t)p.tok[i] * a.nh + part.kvh * a.gq + part.h0 + row % part.heads) * a.hd + d, f);
        else
#pragma unroll
            for (int e = 0; e < N; e++) f[e] = 0.0f;
#pragma unroll
        for (int e = 0; e < N; e++) w.q[r * a.hd + d + e] = f[e] * a.scale_log2;
    }
    __syncwarp();
}

// A block's part of a prefix: groups of R warps, 8 rows a warp; the groups' outputs meet over the queries.
template <typename T, int DIMS, int NR>
__device__ __forceinline__ void sg_prefix(const SaArgs& a, const SaPlan& p, const SaPart& part, float* sq, float2* ml, const SgRows& mine) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hd = a.hd, rows = (part.i1 - part.i0) * part.heads;
    const int R = rows <= SG_ROWS ? 1 : rows <= 2 * SG_ROWS ? 2 : rows <= 4 * SG_ROWS ? 4 : 8, groups = min(SG_WARPS / R, sg_slots(hd)), group = warp / R, place = warp % R;
    SgRows w = mine;
    w.warps = R;
    w.place = place;
    w.barrier = 1 + group;
    float m[NR], l[NR], o[NR][DIMS];
    __syncthreads();                                        // everybody is past the part before
    if (group < groups) {
        w.k = mine.k + (size_t)group * 2 * SG_KEYS * (hd + 4);
        w.v = w.k + SG_KEYS * (hd + 4);
        sg_queries<T>(a, p, part, place * SG_ROWS, rows, w);
        sg_walk<T, DIMS, NR>(a, part, group, groups, w, m, l, o);
    }
    __syncthreads();                                        // and past the queries
    if (group < groups) {
#pragma unroll
        for (int r = 0; r < NR; r++) {
#pragma unroll
            for (int d = 0; d < DIMS; d++)
                if (lane + 32 * d < hd) sq[(warp * SG_ROWS + r) * hd + lane + 32 * d] = o[r][d];
            if (lane == 0) ml[warp * SG_ROWS + r] = make_float2(m[r], l[r]);
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < rows * hd; c += SA_THREADS) {
        const int row = c / hd, d = c - row * hd, i = part.i0 + row / part.heads;
        if (p.pos[i] < 0) continue;
        float top = -INFINITY, sum = 0.0f, out = 0.0f;
        for (int g = 0; g < groups; g++) top = fmaxf(top, ml[g * R * SG_ROWS + row].x);
        const float ref = top == -INFINITY ? 0.0f : top;
        for (int g = 0; g < groups; g++) {
            const float2 s = ml[g * R * SG_ROWS + row];
            const float e = exp2f(s.x - ref);
            sum += s.y * e;
            out += sq[(g * R * SG_ROWS + row) * hd + d] * e;
        }
        const int at = part.row0 + ((i - part.i0) * a.gq + row % part.heads) * part.stride;
        a.part_o[(size_t)at * hd + d] = out;
        if (d == 0) a.part_ml[at] = make_float2(top, sum);
    }
}

// A warp's part of own keys; `alone`: it is all there is of the unit, and the result is written.
template <typename T, int DIMS, int NR>
__device__ __forceinline__ void sg_own(const SaArgs& a, const SaPlan& p, const SaPart& part, bool alone, const SgRows& w) {
    const int lane = threadIdx.x & 31, hd = a.hd;
    float m[NR], l[NR], o[NR][DIMS];
    __syncwarp();
    sg_queries<T>(a, p, part, 0, part.heads, w);
    sg_walk<T, DIMS, NR>(a, part, 0, 1, w, m, l, o);
#pragma unroll
    for (int r = 0; r < NR; r++) {
        if (r >= part.heads) break;
        T* out = static_cast<T*>(a.out) + ((size_t)p.tok[part.i0] * a.nh + part.kvh * a.gq + part.h0 + r) * hd;
        const int at = part.row0 + r * part.stride;
#pragma unroll
        for (int d = 0; d < DIMS; d++)
            if (lane + 32 * d < hd) {
                if (alone) out[lane + 32 * d] = from_f32<T>(o[r][d] / l[r]);
                else a.part_o[(size_t)at * hd + lane + 32 * d] = o[r][d];
            }
        if (!alone && lane == 0) a.part_ml[at] = make_float2(m[r], l[r]);
    }
}

template <typename T, int DIMS>
__global__ void __launch_bounds__(SA_THREADS, DIMS == 2 ? 2 : 1) attention_shared_kernel(const SaArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    SaPlan& p = *reinterpret_cast<SaPlan*>(smem);
    float* sq = reinterpret_cast<float*>(smem + sg_plan_bytes());
    float2* ml = reinterpret_cast<float2*>(sq + SG_PREFIX_ROWS * a.hd);
    float* weights = reinterpret_cast<float*>(ml + SG_PREFIX_ROWS);
    const int warp = threadIdx.x >> 5;
    SgRows w;
    w.q = sq + warp * SG_ROWS * a.hd;
    w.weights = weights + warp * SG_ROWS * SG_KEYS;
    w.k = weights + SG_WARPS * SG_ROWS * SG_KEYS;
    w.v = nullptr;
    w.warps = 1;
    w.place = w.barrier = 0;
    sa_make_plan(a, p);                       // and the wait for the kernel before this one
    let_dependents_start();
    SaPart r;
    const bool prefix = (int)blockIdx.x < p.prefix_blocks;
    int at = blockIdx.x * p.lp, end = prefix ? min(at + p.lp, p.pbase[SA_MAX_TOKENS]) : 0;
    while (at < end) {
        if (!sa_prefix_part(a, p, at, end, blockIdx.x, r)) continue;
        const int rows = (r.i1 - r.i0) * r.heads;
        if (rows <= 2) sg_prefix<T, DIMS, 2>(a, p, r, sq, ml, w);
        else if (rows <= 4) sg_prefix<T, DIMS, 4>(a, p, r, sq, ml, w);
        else sg_prefix<T, DIMS, 8>(a, p, r, sq, ml, w);
    }
    if (!prefix && warp < a.own_per_block) {
        const int worker = warp * ((int)gridDim.x - p.prefix_blocks) + (int)blockIdx.x - p.prefix_blocks;
        w.k += (size_t)warp * 2 * SG_KEYS * (a.hd + 4);
        w.v = w.k + SG_KEYS * (a.hd + 4);
        at = worker * p.lo;
        end = min(at + p.lo, p.obase[SA_MAX_TOKENS]);
        while (at < end) {
            int parts;
            if (!sa_own_part(a, p, at, end, worker, r, parts)) continue;
            const bool alone = parts == 1 && p.shared[r.g] == 0;      // a unit that needs nobody else
            if (r.heads == 1) sg_own<T, DIMS, 1>(a, p, r, alone, w);
            else if (r.heads <= 4) sg_own<T, DIMS, 4>(a, p, r, alone, w);
            else sg_own<T, DIMS, 8>(a, p, r, alone, w);
        }
    }
    sa_write_rows(a, p);
}

// ---- every member by itself, see attention_shared_mma.cu: a block of four warps, eight heads, a run of its keys ------------------------------------------------------

constexpr int SE_WARPS = 4;
// Shared memory: the queries [8][hd], the warps' weights [4][8][32], the warps' keys and values [32][hd + 4] (the warps' outputs [4][8][hd] later), the block's output [8][hd].
__host__ __device__ inline int se_walkers(int hd) { return hd <= 128 ? 4 : 2; }
static size_t se_smem(int hd) { return (size_t)2 * SG_ROWS * hd * 4 + SE_WARPS * SG_ROWS * SG_KEYS * 4 + (size_t)se_walkers(hd) * 2 * SG_KEYS * (hd + 4) * 4; }

template <typename T, int DIMS, int NR>
__device__ __forceinline__ void se_walk(const SaArgs& a, const SaPart& part, const SgRows& w, float* out, float2* ml) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, walkers = se_walkers(a.hd);
    float m[NR], l[NR], o[NR][DIMS];
#pragma unroll
    for (int r = 0; r < NR; r++) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int d = 0; d < DIMS; d++) o[r][d] = 0.0f;
    }
    if (warp < walkers) sg_walk<T, DIMS, NR>(a, part, warp, walkers, w, m, l, o);
    __syncthreads();                                        // everybody is past the keys and values
#pragma unroll
    for (int r = 0; r < NR; r++) {
#pragma unroll
        for (int d = 0; d < DIMS; d++)
            if (lane + 32 * d < a.hd) out[(warp * SG_ROWS + r) * a.hd + lane + 32 * d] = o[r][d];
        if (lane == 0) ml[warp * SG_ROWS + r] = make_float2(m[r], l[r]);
    }
    __syncthreads();
}

template <typename T, int DIMS>
__global__ void __launch_bounds__(SE_WARPS * 32) attention_each_kernel(const SaArgs a) {
    constexpr int N = Vec16<T>::N;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float row_m[SG_ROWS], row_l[SG_ROWS];
    __shared__ float2 ml[SE_WARPS * SG_ROWS];
    float* sq = reinterpret_cast<float*>(smem);
    float* whole = sq + SG_ROWS * a.hd;
    float* weights = whole + SG_ROWS * a.hd;
    float* tiles = weights + SE_WARPS * SG_ROWS * SG_KEYS;
    const int warp = threadIdx.x >> 5, vec = a.hd / N;
    SaPart part;
    int token;
    if (!sa_each_part(a, SG_ROWS, part, token)) return;     // the wait for the kernel before this one is in there
    let_dependents_start();
    const T* q = static_cast<const T*>(a.q) + ((size_t)token * a.nh + part.kvh * a.gq + part.h0) * a.hd;
    for (int c = threadIdx.x; c < SG_ROWS * vec; c += SE_WARPS * 32) {
        const int r = c / vec, d = c % vec * N;
        float f[N];
        if (r < part.heads) load16<T>(q + r * a.hd + d, f);
        else
#pragma unroll
            for (int e = 0; e < N; e++) f[e] = 0.0f;
#pragma unroll
        for (int e = 0; e < N; e++) sq[r * a.hd + d + e] = f[e] * a.scale_log2;
    }
    __syncthreads();
    SgRows w;
    w.q = sq;
    w.weights = weights + warp * SG_ROWS * SG_KEYS;
    w.k = tiles + (size_t)min(warp, se_walkers(a.hd) - 1) * 2 * SG_KEYS * (a.hd + 4);
    w.v = w.k + SG_KEYS * (a.hd + 4);
    w.warps = 1;
    w.place = w.barrier = 0;
    if (part.heads == 1) se_walk<T, DIMS, 1>(a, part, w, tiles, ml);
    else if (part.heads <= 4) se_walk<T, DIMS, 4>(a, part, w, tiles, ml);
    else se_walk<T, DIMS, 8>(a, part, w, tiles, ml);
    sa_each_join<T, SE_WARPS>(a, part, token, SG_ROWS, a.hd, tiles, ml, whole, row_m, row_l);
}

// A row's parts meet: weights 2^(own maximum - row maximum), sums in the parts' order within a lane, then over the lanes, then over the warps, the same in every launch of
// the same lengths.  WARPS warps a row: one where the rows alone fill the machine, four, eight (up to 256 rows) or sixteen (up to 128) where few rows have many parts, whole calls with 4 / 8 /
// 16: 256 rows of 70 parts 30.0 / 27.5 / 27.5 us, of 4 parts 11.6 / 11.8 / 12.7, 512 rows 19.9 / 20.6 / 22.7, 128 rows 17.4 / 16.1 / 15.5, 80 rows 19.7 / 17.4 / 16.6.  A part's row is read as 16-byte pieces by
// L = 2, 4 .. 32 neighbouring lanes, 32 / L parts at once and four of those in flight.  (No pointer is __restrict__: what the walk, or a kernel before it, has written is not constant for a launch that
// begins beside it, and a load that may be taken for one need not stay behind the wait.)
template <typename T, int WARPS>
__global__ void __launch_bounds__(WARPS > 4 ? WARPS * 32 : 128) attention_shared_join_kernel(const SaRow* rows, const float2* part_ml, const float* part_o,
                                                                    const int32_t* members, T* out, int n_rows, int nh, int hd, int lanes) {
    constexpr int PIECES = 2, FLIGHT = 4;          // pieces of 16 bytes a lane has of a row of up to 256
    constexpr int ROWS = WARPS > 4 ? 1 : 4 / WARPS;      // of a block
    __shared__ float2 warp_ml[ROWS * WARPS];
    __shared__ float4 warp_o[ROWS * WARPS][32 * PIECES];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WARPS, r = blockIdx.x * ROWS + warp / WARPS;
    dependency_wait();
    let_dependents_start();
    SaRow row = {0, 0, 0, 0};
    if (r < n_rows) row = rows[r];
    const int parts = row.prefix_parts + row.own_parts;
    if (parts == 0) return;                                       // with several warps a row the whole block
    const int at_once = 32 / lanes, slot = lane / lanes, piece = lane % lanes, vec = hd / 4;
    float m = -INFINITY, l = 0.0f;
    float4 o[PIECES];
#pragma unroll
    for (int d = 0; d < PIECES; d++) o[d] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int j0 = sub * at_once + slot; j0 < parts; j0 += FLIGHT * WARPS * at_once) {
        float2 ml[FLIGHT];
        float4 v[FLIGHT][PIECES];
#pragma unroll
        for (int f = 0; f < FLIGHT; f++) {
            const int j = j0 + f * WARPS * at_once;
            const bool on = j < parts;
            const int from = j < row.prefix_parts ? row.prefix_row + j : row.own_row + j - row.prefix_parts;
            ml[f] = on ? __ldcg(part_ml + from) : make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int d = 0; d < PIECES; d++)
                v[f][d] = on && piece + d * lanes < vec ? __ldcg(reinterpret_cast<const float4*>(part_o + (size_t)from * hd) + piece + d * lanes) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        float top = m;
#pragma unroll
        for (int f = 0; f < FLIGHT; f++) top = fmaxf(top, ml[f].x);
        const float ref = top == -INFINITY ? 0.0f : top, keep = sa_ex2(m - ref);       // no score above -inf so far: every weight is 0
        l *= keep;
#pragma unroll
        for (int d = 0; d < PIECES; d++) { o[d].x *= keep; o[d].y *= keep; o[d].z *= keep; o[d].w *= keep; }
#pragma unroll
        for (int f = 0; f < FLIGHT; f++) {
            const float w = sa_ex2(ml[f].x - ref);
            l += ml[f].y * w;
#pragma unroll
            for (int d = 0; d < PIECES; d++) { o[d].x += v[f][d].x * w; o[d].y += v[f][d].y * w; o[d].z += v[f][d].z * w; o[d].w += v[f][d].w * w; }
        }
        m = top;
    }
    __syncwarp();
    for (int x = lanes; x < 32; x <<= 1) {                        // the lanes that had other parts of the same piece
        const float om = __shfl_xor_sync(0xffffffffu, m, x), top = fmaxf(m, om), ref = top == -INFINITY ? 0.0f : top, wa = sa_ex2(m - ref), wb = sa_ex2(om - ref);
        l = l * wa + __shfl_xor_sync(0xffffffffu, l, x) * wb;
#pragma unroll
        for (int d = 0; d < PIECES; d++) {
            o[d].x = o[d].x * wa + __shfl_xor_sync(0xffffffffu, o[d].x, x) * wb;
            o[d].y = o[d].y * wa + __shfl_xor_sync(0xffffffffu, o[d].y, x) * wb;
            o[d].z = o[d].z * wa + __shfl_xor_sync(0xffffffffu, o[d].z, x) * wb;
            o[d].w = o[d].w * wa + __shfl_xor_sync(0xffffffffu, o[d].w, x) * wb;
        }
        m = top;
    }
    if (WARPS > 1) {
        if (slot == 0) {
            if (piece == 0) warp_ml[warp] = make_float2(m, l);
#pragma unroll
            for (int d = 0; d < PIECES; d++) warp_o[warp][piece + d * lanes] = o[d];
        }
        __syncthreads();
        if (warp != 0) return;
        m = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; w++) m = fmaxf(m, warp_ml[w].x);
        const float ref = m == -INFINITY ? 0.0f : m;
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < PIECES; d++) o[d] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float e = sa_ex2(warp_ml[w].x - ref);
            l += warp_ml[w].y * e;
#pragma unroll
            for (int d = 0; d < PIECES; d++) {
                const float4 v = warp_o[w][piece + d * lanes];
                o[d].x += v.x * e; o[d].y += v.y * e; o[d].z += v.z * e; o[d].w += v.w * e;
            }
        }
    }
    if (slot != 0) return;
    const int i = r / nh;
    T* to = out + ((size_t)members[i] * nh + r - i * nh) * hd;
#pragma unroll
    for (int d = 0; d < PIECES; d++) {
        const int at = (piece + d * lanes) * 4;
        if (at >= hd) continue;
        if (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(to + at) = make_float4(o[d].x / l, o[d].y / l, o[d].z / l, o[d].w / l);
        } else {
            const __nv_bfloat162 x = __floats2bfloat162_rn(o[d].x / l, o[d].y / l), y = __floats2bfloat162_rn(o[d].z / l, o[d].w / l);
            *reinterpret_cast<uint2*>(to + at) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
        }
    }
}

static int launch_join(const SaArgs& a, int dtype, cudaStream_t stream) {
    const int rows = a.n * a.nh;
    int lanes = 2;
    while (lanes < 32 && lanes * 4 < a.hd) lanes *= 2;
    const SaRow* table = reinterpret_cast<const SaRow*>(a.rows);
#define GO(T, WARPS)                                                                                                                                          \
    return launch_dependent(attention_shared_join_kernel<T, WARPS>, dim3(WARPS > 1 ? rows : (rows + 3) / 4), dim3(WARPS > 4 ? WARPS * 32 : 128), 0, stream, table, a.part_ml, a.part_o, a.members, \
                            static_cast<T*>(a.out), rows, a.nh, a.hd, lanes)
    if (rows >= 1024) {
        if (dtype == 0) GO(float, 1);
        GO(__nv_bfloat16, 1);
    }
    if (rows > 256) {
        if (dtype == 0) GO(float, 4);
        GO(__nv_bfloat16, 4);
    }
    if (rows > 128) {
        if (dtype == 0) GO(float, 8);
        GO(__nv_bfloat16, 8);
    }
    if (dtype == 0) GO(float, 16);
    GO(__nv_bfloat16, 16);
#undef GO
}

// Where: tables of up to 64 MB together at their full width, none longer than 256 positions a block of the largest cluster.  Measured in float32, this way against the other: 8 members of 512
// common and up to 64 own positions at 3 key-value heads of 64 (7 MB) 9.7 us against 16.6, 64 of 512 (58 MB) 29.8 / 30.7, 24 of 512 and up to 600 (42 MB) 24.0 / 25.9, 64 of 512 at 5 heads
// (97 MB) 55 / 37; 8 of 512 at 32 heads (78 MB) 25 / 27, 24 of 512 (233 MB) 72 / 37; 2 of 2,048 at 3 heads (6 MB) 16.3 / 14.4, of 8,000 (25 MB) 41 / 17; 8 of 512 at 2 heads of 128, eight queries
// each (10 MB), 23 / 38, of 2,048 (35 MB) 52 / 39.
static int each_most(const SaArgs& a) { return a.hd <= 64 ? 8 : 4; }
static bool each_takes(const SaArgs& a, int dtype) {
    const long long reach = (long long)a.max_blocks * a.page_size;
    return reach <= 256 * each_most(a) && a.n * reach * a.nkv * a.hd * 2 * (dtype == 0 ? 4 : 2) <= 64ll << 20;
}
static int launch_each(const SaArgs& a, int dtype, int multiprocessors, cudaStream_t stream) {
    const int tiles = a.nkv * ((a.gq + SG_ROWS - 1) / SG_ROWS), room = multiprocessors * (a.hd <= 64 ? 2 : 1);
    int ranks = 1;
    while (ranks < each_most(a) && ranks * 128 < (long long)a.max_blocks * a.page_size && 2 * ranks * tiles * a.n <= room) ranks *= 2;
    const size_t smem = se_smem(a.hd);
#define GO(T, DIMS)                                                                                                                      \
    do {                                                                                                                                 \
        const int e = sa_allow_smem(attention_each_kernel<T, DIMS>, smem);                                                               \
        if (e != VK_OK) return e;                                                                                                        \
        return launch_dependent_cluster(attention_each_kernel<T, DIMS>, dim3(ranks, tiles, a.n), dim3(SE_WARPS * 32), ranks, smem, stream, a); \
    } while (0)
    if (dtype == 0) {
        if (a.hd <= 64) GO(float, 2);
        if (a.hd <= 128) GO(float, 4);
        GO(float, 8);
    }
    if (a.hd <= 64) GO(__nv_bfloat16, 2);
    if (a.hd <= 128) GO(__nv_bfloat16, 4);
    GO(__nv_bfloat16, 8);
#undef GO
}

// The current device's multiprocessors, asked for once a device.
static int sa_multiprocessors() {
    static std::atomic<int> known[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
    return n;
}

static int launched(int status, int kernels) { return status == VK_OK ? VK_LAUNCHED + kernels : status; }

// Rows of parts that a launch can need: a unit of so many tiles of keys and up to R rows leaves at most R (tiles / L + 2), L is at least the line's
// length / workers, and the units' rows are n nh together.  R is 128 for prefixes here and the workers a multiprocessor's blocks (2) and warps (16), which covers
// both kernels.
static size_t sa_part_rows(int tokens, int nh) { return (size_t)(128 * 2 + SA_MAX_OWN_ROWS * 16) * SA_MAX_MULTIPROCESSORS + 4 * (size_t)tokens * nh; }

}  // namespace vk

using namespace vk;

VK_API size_t vk_attention_shared_scratch_bytes(int tokens, int nh, int, int hd) {
    return sa_part_rows(tokens, nh) * ((size_t)hd * 4 + 8) + (size_t)tokens * nh * 16;
}

// The arguments of vk_attention_shared, in one piece.  dtype 0 = float32, 1 = bfloat16.  scratch: vk_attention_shared_scratch_bytes(n, ...) bytes, whatever they hold.
struct VkAttentionShared {
    const void *q, *cache;
    const int32_t *block_tables, *token_seg, *positions, *members, *starts, *shared;
    void *out, *scratch;
    uint64_t scratch_bytes;
    int32_t tokens, segments, n, families, pages, nh, nkv, hd, page_size, max_blocks;
    float scale;
    int32_t dtype;
    int* error;                    // set where a wait inside the kernel runs out
};

// Returns VK_LAUNCHED + 1 (every member by itself) or + 2 (the walk, and the launch that joins the parts); VK_OK where nobody asks for anything.

VK_API int vk_attention_shared(const VkAttentionShared* args, cudaStream_t stream) {
    const auto [q, cache, block_tables, token_seg, positions, members, starts, shared, out, scratch, scratch_bytes, tokens, segments, n, families, pages, nh, nkv, hd, page_size,
                max_blocks, scale, dtype, error] = *args;
    if (n <= 0 || families <= 0) return VK_OK;
    if (n > SA_MAX_TOKENS || families > SA_MAX_TOKENS || nkv > SA_MAX_KV_HEADS || hd > 256) return VK_TOO_LARGE;
    const int vec = dtype == 0 ? 4 : 8;
    if (nkv <= 0 || nh <= 0 || nh % nkv || nh / nkv > SA_MAX_HEADS || hd <= 0 || hd % vec || page_size <= 0 || max_blocks <= 0 || pages <= 0 || !error) return VK_BAD_SHAPE;
    // positions, the lines' tiles and the parts' rows are counted in 31 bits: a walk asks a few tiles behind its part's end and a unit's empty tiles stand behind its keys, the last worker
    // begins up to a tile a worker behind the line's end, so half of what 31 bits hold
    const long long reach = (long long)max_blocks * page_size, tiles = reach / SA_TILE + 64, units = (long long)n * nh;
    if (reach > 1 << 30 || tiles * units > 1 << 30 || units * 4 * hd > 0x7fffffffLL) return VK_TOO_LARGE;
    if (((uintptr_t)q | (uintptr_t)cache | (uintptr_t)out | (uintptr_t)scratch) % 16) return VK_BAD_ALIGNMENT;
    if (scratch_bytes < vk_attention_shared_scratch_bytes(n, nh, nkv, hd)) return VK_SMALL_SCRATCH;
    const int sms = sa_multiprocessors();
    if (sms > SA_MAX_MULTIPROCESSORS) return VK_TOO_LARGE;
    SaArgs a;
    a.q = q; a.cache = cache; a.block_tables = block_tables; a.token_seg = token_seg; a.positions = positions;
    a.members = members; a.starts = starts; a.shared = shared; a.out = out;
    const size_t rows = sa_part_rows(n, nh);
    a.rows = (int4*)scratch;
    a.part_o = (float*)(a.rows + (size_t)n * nh);
    a.part_ml = (float2*)(a.part_o + rows * hd);
    a.n = n; a.families = families; a.tokens = tokens; a.segments = segments; a.pages = pages;
    a.nh = nh; a.nkv = nkv; a.gq = nh / nkv; a.hd = hd; a.page_size = page_size; a.max_blocks = max_blocks;
    a.page_shift = -1;
    for (int b = 0; b < 30; b++) if ((1 << b) == page_size) a.page_shift = b;
    a.scale_log2 = scale * 1.4426950408889634f;
    if (attention_shared_mma_takes(a, dtype)) {
        if (attention_each_mma_takes(a)) return launched(launch_attention_each_mma(a, sms, stream), 1);
        const int status = launch_attention_shared_mma(a, sms, error, stream);
        return status != VK_OK ? status : launched(launch_join(a, dtype, stream), 2);
    }
    if (each_takes(a, dtype)) return launched(launch_each(a, dtype, sms, stream), 1);
    a.prefix_rows = SG_PREFIX_ROWS;
    a.own_rows = SG_ROWS;
    a.row_unit = 16.0f;
    a.tensor_rows = 0x7fffffff;
    a.tensor_unit = 1.0f;
    a.blocks = sms * sg_blocks(hd);
    a.own_per_block = sg_slots(hd);
    a.min_prefix = a.min_own = 4;
    a.prefix_cost = a.own_cost = 4;
    const size_t smem = sg_smem(hd);
#define GO(T, DIMS)                                                                                                                     \
    do {                                                                                                                                \
        auto kern = attention_shared_kernel<T, DIMS>;                                                                                   \
        const int e = sa_allow_smem(kern, smem);                                                                                        \
        if (e != VK_OK) return e;                                                                                                       \
        const int status = launch_dependent(kern, dim3(a.blocks), dim3(SA_THREADS), smem, stream, a);                                        \
        return status != VK_OK ? status : launched(launch_join(a, dtype, stream), 2);                                                   \
    } while (0)
    if (dtype == 0) {
        if (hd <= 64) GO(float, 2);
        if (hd <= 128) GO(float, 4);
        GO(float, 8);
    }
    if (hd <= 64) GO(__nv_bfloat16, 2);
    if (hd <= 128) GO(__nv_bfloat16, 4);
    GO(__nv_bfloat16, 8);
#undef GO
}
