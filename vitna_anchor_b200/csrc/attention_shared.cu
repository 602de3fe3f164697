// Decode attention of requests that hold their first pages in common: beams of one prompt, requests behind one prefix.
//
//   out[t][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[t][h] . k_j),  j = 0 .. position(t) over t's block table
//
// Attention over separate block tables reads the common keys once a request.  Here a family's members are the rows of one product over
// the keys they share, which are read once, and the keys that a member has alone are walked by themselves; the two meet by their maxima
// and sums, which stay in float32 like everything between the scores and the output's rounding.  How the walks are cut: attention_shared_plan.cuh.
//
// This file has the entry point and the kernel that takes every size and both types: a part at a time by a block of eight warps, 32 keys
// and values at a time in shared memory as float32, a warp's lanes 32 keys of a score and then 32 dims of the output.
// attention_shared_mma.cu has bfloat16 heads of 64 and 128 on the tensor cores.
#include "attention_shared_plan.cuh"

#include <atomic>

namespace vk {

constexpr int SG_KEYS = 32, SG_PREFIX_ROWS = 64, SG_ROWS = SG_PREFIX_ROWS / (SA_THREADS / 32);      // rows a block, rows a warp

// Shared memory: the plan, then the rows' queries [64][hd] and the keys' and values' tiles [32][hd + 4].
__host__ __device__ inline size_t sg_plan_bytes() { return (sizeof(SaPlan) + 15) / 16 * 16; }
static size_t sg_smem(int hd) { return sg_plan_bytes() + (size_t)(SG_PREFIX_ROWS * hd + 2 * SG_KEYS * (hd + 4)) * 4; }

// A block walks a part and leaves its rows; `alone`: they are all there is of the unit, and the result is written.
template <typename T, int DIMS>
__device__ __forceinline__ void sg_walk(const SaArgs& a, const SaPlan& p, const SaPart& r, bool alone, float* sq, float* sk, float* sv) {
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hd = a.hd, ld = hd + 4, vec = hd / N;
    const int rows = (r.i1 - r.i0) * r.heads;
    __syncthreads();                                    // the part before is done with the tiles
    for (int c = threadIdx.x; c < rows * vec; c += SA_THREADS) {
        const int row = c / vec, d = c % vec * N, i = r.i0 + row / r.heads;
        float f[N];
        if (p.pos[i] >= 0) load16<T>(static_cast<const T*>(a.q) + ((size_t)p.tok[i] * a.nh + r.kvh * a.gq + r.h0 + row % r.heads) * hd + d, f);
        else for (int e = 0; e < N; e++) f[e] = 0.0f;
#pragma unroll
        for (int e = 0; e < N; e++) sq[row * hd + d + e] = f[e] * a.scale_log2;
    }
    float m[SG_ROWS], l[SG_ROWS], o[SG_ROWS][DIMS];
#pragma unroll
    for (int x = 0; x < SG_ROWS; x++) {
        m[x] = -INFINITY;
        l[x] = 0.0f;
#pragma unroll
        for (int d = 0; d < DIMS; d++) o[x][d] = 0.0f;
    }
    for (int kb = r.k0; kb < r.k1; kb += SG_KEYS) {
        __syncthreads();
        for (int c = threadIdx.x; c < SG_KEYS * vec; c += SA_THREADS) {
            const int kl = c / vec, d = c % vec * N, key = kb + kl;
            float fk[N], fv[N];
#pragma unroll
            for (int e = 0; e < N; e++) fk[e] = fv[e] = 0.0f;       // no key: nothing of it may be read, not even a NaN
            if (key < r.k1) {
                const int block = key / a.page_size, page = r.table[block];
                if (page >= 0 && page < a.pages) {
                    const T* src = static_cast<const T*>(a.cache) + (((size_t)page * 2 * a.nkv + r.kvh) * a.page_size + key - block * a.page_size) * hd + d;
                    load16<T>(src, fk);
                    load16<T>(src + (size_t)a.nkv * a.page_size * hd, fv);
                }
            }
#pragma unroll
            for (int e = 0; e < N; e++) { sk[kl * ld + d + e] = fk[e]; sv[kl * ld + d + e] = fv[e]; }
        }
        __syncthreads();
        const int keys = min(SG_KEYS, r.k1 - kb);
#pragma unroll
        for (int x = 0; x < SG_ROWS; x++) {
            const int row = warp + x * (SA_THREADS / 32);
            if (row >= rows) continue;
            float s = 0.0f;
            for (int d = 0; d < hd; d += 4) {
                const float4 u = *reinterpret_cast<const float4*>(sq + row * hd + d), v = *reinterpret_cast<const float4*>(sk + lane * ld + d);
                s += u.x * v.x + u.y * v.y + u.z * v.z + u.w * v.w;
            }
            if (lane >= keys) s = -INFINITY;
            const float top = fmaxf(m[x], warp_max(s)), ref = top == -INFINITY ? 0.0f : top;
            const float keep = exp2f(m[x] - ref), w = exp2f(s - ref);
            m[x] = top;
            l[x] = l[x] * keep + warp_sum(w);
#pragma unroll
            for (int d = 0; d < DIMS; d++) o[x][d] *= keep;
            for (int k = 0; k < keys; k++) {
                const float wk = __shfl_sync(0xffffffffu, w, k);
#pragma unroll
                for (int d = 0; d < DIMS; d++)
                    if (lane + 32 * d < hd) o[x][d] += wk * sv[k * ld + lane + 32 * d];
            }
        }
    }
#pragma unroll
    for (int x = 0; x < SG_ROWS; x++) {
        const int row = warp + x * (SA_THREADS / 32), i = r.i0 + row / r.heads;
        if (row >= rows || p.pos[i] < 0) continue;
        if (alone) {
            T* out = static_cast<T*>(a.out) + ((size_t)p.tok[i] * a.nh + r.kvh * a.gq + r.h0 + row % r.heads) * hd;
#pragma unroll
            for (int d = 0; d < DIMS; d++)
                if (lane + 32 * d < hd) out[lane + 32 * d] = from_f32<T>(o[x][d] / l[x]);
        } else {
            const int at = r.row0 + ((i - r.i0) * a.gq + row % r.heads) * r.stride;
#pragma unroll
            for (int d = 0; d < DIMS; d++)
                if (lane + 32 * d < hd) a.part_o[(size_t)at * hd + lane + 32 * d] = o[x][d];
            if (lane == 0) a.part_ml[at] = make_float2(m[x], l[x]);
        }
    }
}

template <typename T, int DIMS>
__global__ void __launch_bounds__(SA_THREADS) attention_shared_kernel(const SaArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    SaPlan& p = *reinterpret_cast<SaPlan*>(smem);
    float* sq = reinterpret_cast<float*>(smem + sg_plan_bytes());
    float* sk = sq + SG_PREFIX_ROWS * a.hd;
    float* sv = sk + SG_KEYS * (a.hd + 4);
    sa_make_plan(a, p);                       // from the step's metadata, which no kernel writes
    dependency_wait();
    let_dependents_start();
    SaPart r;
    const bool prefix = (int)blockIdx.x < p.prefix_blocks;
    const int worker = (int)blockIdx.x - (prefix ? 0 : p.prefix_blocks);
    int at = worker * p.lp, end = prefix ? min(at + p.lp, p.pbase[SA_MAX_TOKENS]) : 0;
    while (at < end) {
        if (!sa_prefix_part(a, p, at, end, worker, r)) continue;
        sg_walk<T, DIMS>(a, p, r, false, sq, sk, sv);
    }
    at = worker * p.lo;
    end = prefix ? 0 : min(at + p.lo, p.obase[SA_MAX_TOKENS]);
    while (at < end) {
        int parts;
        if (!sa_own_part(a, p, at, end, worker, r, parts)) continue;
        sg_walk<T, DIMS>(a, p, r, parts == 1 && p.shared[r.g] == 0, sq, sk, sv);      // a unit that needs nobody else writes its result
    }
    sa_write_rows(a, p);
}

// A row's parts meet: weights 2^(own maximum - row maximum), sums in the parts' order within a lane, then over the lanes, then over the warps, the same in every launch of
// the same lengths.  WARPS warps a row: one where the rows alone fill the machine, four where few rows have many parts.  A part's row is read as 16-byte pieces by
// L = 2, 4 .. 32 neighbouring lanes, 32 / L parts at once and four of those in flight.
template <typename T, int WARPS>
__global__ void __launch_bounds__(128) attention_shared_join_kernel(const SaRow* __restrict__ rows, const float2* __restrict__ part_ml, const float* __restrict__ part_o,
                                                                    const int32_t* __restrict__ members, T* __restrict__ out, int n_rows, int nh, int hd, int lanes) {
    constexpr int PIECES = 2, FLIGHT = 4;          // pieces of 16 bytes a lane has of a row of up to 256
    __shared__ float2 warp_ml[4];
    __shared__ float4 warp_o[4][32 * PIECES];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WARPS, r = blockIdx.x * (4 / WARPS) + warp / WARPS;
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
    return launch_dependent(attention_shared_join_kernel<T, WARPS>, dim3((rows + 4 / WARPS - 1) / (4 / WARPS)), dim3(128), 0, stream, table, a.part_ml, a.part_o, a.members, \
                            static_cast<T*>(a.out), rows, a.nh, a.hd, lanes)
    if (rows >= 1024) {
        if (dtype == 0) GO(float, 1);
        GO(__nv_bfloat16, 1);
    }
    if (dtype == 0) GO(float, 4);
    GO(__nv_bfloat16, 4);
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

// Rows of parts that a launch can need: a unit of so many tiles of keys and up to R rows leaves at most R (tiles / L + 2), L is at least the line's
// length / workers, and the units' rows are n nh together.  R is 128 for prefixes here and the workers a multiprocessor's blocks (2) and warps (16), which covers
// both kernels.
static size_t sa_part_rows(int tokens, int nh) { return (size_t)(128 * 2 + SA_OWN_ROWS * 16) * SA_MAX_MULTIPROCESSORS + 4 * (size_t)tokens * nh; }

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
};

VK_API int vk_attention_shared(const VkAttentionShared* args, cudaStream_t stream) {
    const auto [q, cache, block_tables, token_seg, positions, members, starts, shared, out, scratch, scratch_bytes, tokens, segments, n, families, pages, nh, nkv, hd, page_size,
                max_blocks, scale, dtype] = *args;
    if (n <= 0 || families <= 0) return VK_OK;
    if (n > SA_MAX_TOKENS || families > SA_MAX_TOKENS || nkv > SA_MAX_KV_HEADS || hd > 256) return VK_TOO_LARGE;
    const int vec = dtype == 0 ? 4 : 8;
    if (nkv <= 0 || nh <= 0 || nh % nkv || nh / nkv > SA_MAX_HEADS || hd <= 0 || hd % vec || page_size <= 0 || max_blocks <= 0 || pages <= 0) return VK_BAD_SHAPE;
    if ((long long)max_blocks * page_size > 0x7fffffffLL) return VK_TOO_LARGE;
    // the lines' tiles and the parts' rows are counted in 31 bits
    const long long tiles = (long long)max_blocks * page_size / SA_TILE + 64, units = (long long)n * nh;
    if (tiles * units > 0x7fffffffLL || units * 4 * hd > 0x7fffffffLL) return VK_TOO_LARGE;
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
        const int status = launch_attention_shared_mma(a, sms, stream);
        return status != VK_OK ? status : launch_join(a, dtype, stream);
    }
    a.prefix_rows = SG_PREFIX_ROWS;
    a.blocks = sms;
    a.own_per_block = 1;
    a.min_prefix = a.min_own = 4;
    a.prefix_cost = a.own_cost = 4;
    const size_t smem = sg_smem(hd);
#define GO(T, DIMS)                                                                                                                     \
    do {                                                                                                                                \
        auto kern = attention_shared_kernel<T, DIMS>;                                                                                   \
        const int e = sa_allow_smem(kern, smem);                                                                                        \
        if (e != VK_OK) return e;                                                                                                       \
        const int status = launch_dependent(kern, dim3(sms), dim3(SA_THREADS), smem, stream, a);                                        \
        return status != VK_OK ? status : launch_join(a, dtype, stream);                                                                \
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
