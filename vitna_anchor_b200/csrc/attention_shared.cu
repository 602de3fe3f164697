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

namespace vk {

constexpr int SG_KEYS = 32, SG_ROWS = SA_PREFIX_ROWS / (SA_THREADS / 32);      // rows a warp

// Shared memory: the plan, then the rows' queries [64][hd] and the keys' and values' tiles [32][hd + 4].
__host__ __device__ inline size_t sg_plan_bytes() { return (sizeof(SaPlan) + 15) / 16 * 16; }
static size_t sg_smem(int hd) { return sg_plan_bytes() + (size_t)(SA_PREFIX_ROWS * hd + 2 * SG_KEYS * (hd + 4)) * 4; }

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
    float* sk = sq + SA_PREFIX_ROWS * a.hd;
    float* sv = sk + SG_KEYS * (a.hd + 4);
    __shared__ int last[SA_PREFIX_ROWS];
    const int warp = threadIdx.x >> 5, worker = blockIdx.x;
    dependency_wait();
    let_dependents_start();
    sa_make_plan(a, p);
    long long at = (long long)worker * p.lp, end = min(at + p.lp, p.pbase[SA_MAX_TOKENS]);
    while (at < end) {
        const SaPart r = sa_prefix_part(a, p, at, end, worker);
        sg_walk<T, DIMS>(a, p, r, false, sq, sk, sv);
        __syncthreads();
        if ((int)threadIdx.x < r.i1 - r.i0) last[threadIdx.x] = p.pos[r.i0 + threadIdx.x] >= 0 && sa_last(a, p, r.i0 + threadIdx.x, r.kvh);
        __syncthreads();
        for (int i = r.i0; i < r.i1; i++)
            if (last[i - r.i0])
                for (int h = warp; h < a.gq; h += SA_THREADS / 32) sa_join<T, DIMS>(a, p, i, r.kvh, h);
        at += r.k1 - r.k0;
    }
    at = (long long)worker * p.lo;
    end = min(at + p.lo, p.obase[SA_MAX_TOKENS]);
    while (at < end) {
        int parts;
        const SaPart r = sa_own_part(a, p, at, end, worker, parts);
        const bool alone = parts == 1 && p.shared[r.g] == 0;      // then the unit's rows need nobody else
        sg_walk<T, DIMS>(a, p, r, alone, sq, sk, sv);
        __syncthreads();
        if (threadIdx.x == 0) last[0] = sa_last(a, p, r.i0, r.kvh);
        __syncthreads();
        if (last[0])
            for (int h = warp; h < a.gq; h += SA_THREADS / 32)
                if (!(p.shared[r.g] == 0 && sa_own_parts(p, r.i0, r.kvh, h / SA_OWN_ROWS) == 1)) sa_join<T, DIMS>(a, p, r.i0, r.kvh, h);
        at += r.k1 - r.k0;
    }
}

static int sa_multiprocessors() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    return n;
}

constexpr int SA_MAX_MULTIPROCESSORS = 160;         // of the sm_100a parts; the scratch is laid out for this many

// Rows of parts that a launch can need: a unit of `keys` keys and up to R rows leaves at most R (keys / L + 2), L is at least the line's
// length / workers, and the units' rows are n nh together.
static size_t sa_part_rows(int tokens, int nh, int nkv) {
    const size_t gq = nh / nkv, prefix_rows = gq > SA_PREFIX_ROWS ? gq : SA_PREFIX_ROWS, own_rows = gq < SA_OWN_ROWS ? gq : SA_OWN_ROWS;
    return prefix_rows * SA_MAX_MULTIPROCESSORS + own_rows * SA_MAX_MULTIPROCESSORS * 8 + 4 * (size_t)tokens * nh;
}


}  // namespace vk

using namespace vk;

VK_API size_t vk_attention_shared_scratch_bytes(int tokens, int nh, int nkv, int hd) {
    return (size_t)SA_MAX_TOKENS * SA_MAX_KV_HEADS * 4 + sa_part_rows(tokens, nh, nkv) * ((size_t)hd * 4 + 8);
}

// dtype 0 = float32, 1 = bfloat16.  scratch: vk_attention_shared_scratch_bytes(n, ...) bytes whose counters (the first SA_MAX_TOKENS *
// SA_MAX_KV_HEADS words) were zero at first use; the kernel leaves them zero.
VK_API int vk_attention_shared(const void* q, const void* cache, const int32_t* block_tables, const int32_t* token_seg, const int32_t* positions,
                               const int32_t* members, const int32_t* starts, const int32_t* shared, void* out, void* scratch, int tokens, int segments,
                               int n, int families, int pages, int nh, int nkv, int hd, int page_size, int max_blocks, float scale, int dtype,
                               cudaStream_t stream) {
    if (n <= 0 || families <= 0) return VK_OK;
    if (n > SA_MAX_TOKENS || families > SA_MAX_TOKENS || nkv > SA_MAX_KV_HEADS || hd > 256) return VK_TOO_LARGE;
    const int vec = dtype == 0 ? 4 : 8;
    if (nkv <= 0 || nh <= 0 || nh % nkv || nh / nkv > SA_PREFIX_ROWS || hd <= 0 || hd % vec || page_size <= 0 || max_blocks <= 0 || pages <= 0) return VK_BAD_SHAPE;
    if ((long long)max_blocks * page_size > 0x7fffffffLL) return VK_TOO_LARGE;
    if (((uintptr_t)q | (uintptr_t)cache | (uintptr_t)out | (uintptr_t)scratch) % 16) return VK_BAD_ALIGNMENT;
    const int sms = sa_multiprocessors();
    if (sms > SA_MAX_MULTIPROCESSORS) return VK_TOO_LARGE;
    SaArgs a;
    a.q = q; a.cache = cache; a.block_tables = block_tables; a.token_seg = token_seg; a.positions = positions;
    a.members = members; a.starts = starts; a.shared = shared; a.out = out;
    const size_t rows = sa_part_rows(n, nh, nkv);
    a.counters = (int*)scratch;
    a.part_o = (float*)((char*)scratch + (size_t)SA_MAX_TOKENS * SA_MAX_KV_HEADS * 4);
    a.part_ml = (float2*)(a.part_o + rows * hd);
    a.n = n; a.families = families; a.tokens = tokens; a.segments = segments; a.pages = pages;
    a.nh = nh; a.nkv = nkv; a.gq = nh / nkv; a.hd = hd; a.page_size = page_size; a.max_blocks = max_blocks;
    a.page_shift = -1;
    for (int b = 0; b < 30; b++) if ((1 << b) == page_size) a.page_shift = b;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.prefix_workers = a.own_workers = sms;
    a.min_prefix = 64;
    a.min_own = 64;
    const size_t smem = sg_smem(hd);
#define GO(T, DIMS)                                                                                                                     \
    do {                                                                                                                                \
        auto kern = attention_shared_kernel<T, DIMS>;                                                                                   \
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);                             \
        if (e != cudaSuccess) return (int)e;                                                                                            \
        return launch_dependent(kern, dim3(sms), dim3(SA_THREADS), smem, stream, a);                                                    \
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
