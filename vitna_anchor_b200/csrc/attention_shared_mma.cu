// Decode attention over pages held in common, bfloat16 heads of 64 and 128, on the tensor cores.
//
// The mathematics and the cut into parts are attention_shared.cu's and attention_shared_plan.cuh's.  A part's rows (a family's members times the heads
// that read one key-value head) are the 16-row operands of m16n8k16 products, 16 rows a warp; R = 1, 2, 4 or 8 warps that cover a part's rows
// make a group that works through the same keys, and the block's 8 / R groups take turns at the tiles of 16 R keys (heads of 128: R up to 4, more rows go to tcgen05, see below).  So a block holds up to 128 rows
// against keys that are read once, and with few rows all eight warps still read keys of their own.  Up to eight rows turn the products over: the keys are the 16 rows and
// the rows the eight columns, half the products and half the exponentials.
//
//   copy      three stages of 128 keys and values a block by cp.async, each warp asks for 16 keys of its group's tile and the group meets once a tile; the page of the tile after
//             next is asked for a tile before its number is used.  16-byte pieces are stored at piece ^ (key & 7), so that ldmatrix meets no bank twice
//   scores    S = Q K^T, the queries in registers
//   softmax   against a reference maximum that follows only when a score is 2^8 above it, sums in float32
//   p v       the weights go from the score registers into the next product's operand as a high and a low bfloat16 part (p to 2^-17): one part alone would double the error
//             that the output's own rounding makes
//
// A member's own keys are walked by single warps with the same routines (R = 1): up to 16 rows of heads.
//
// What bounds it.  64 requests behind 6,000 positions with up to 700 of their own, 32 heads of 64 (214 MB): 48.5 us, 4.4 TB/s; the common keys' blocks do 64 rows a key, 16,000 cycles of the tensor
// cores' legacy path, and take 37,000 (a group's warps do scores, softmax and p v in step, 4 warps a scheduler), while the own keys' blocks beside them wait for memory.  One kind after the
// other in every block: 57 us.  Eight beams of 2,048 positions, 32 heads of 64 (20 MB): 12.1 us, of which finding the parts is 2 (it runs before the wait for the kernel
// before), looking behind the wait whether they hold 0.3, and joining them 3.
#include "attention_shared_plan.cuh"
#include "tcgen05_common.cuh"

namespace vk {

constexpr int SM_STAGES = 3, SM_WARP_KEYS = 16, SM_KEYS = SM_WARP_KEYS * (SA_THREADS / 32), SM_PREFIX_ROWS = 128;

template <int HD> struct SmSmem {
    static constexpr int HALF = SM_KEYS * HD * 2;                                     // bytes of a stage's keys, or values
    static constexpr int STAGE = 2 * HALF;
    static constexpr int OUT = (SA_THREADS / 32) * 16 * (HD + 4) * 4;                 // the warps' outputs where a part's groups meet: over the stages
    static constexpr int PLAN = (sizeof(SaPlan) + 127) / 128 * 128;
    static constexpr size_t BYTES = PLAN + (size_t)SM_STAGES * STAGE;
    static constexpr int ML = (SA_THREADS / 32) * 16 * 8;                             // and, behind them, their maxima and sums
    static_assert(OUT + ML <= SM_STAGES * STAGE, "the warps' outputs lie over the stages");
};

__device__ __forceinline__ uint32_t sm_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void sm_copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void sm_copy16_or_zero(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void sm_ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void sm_ldsm4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void sm_mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t sm_turn(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t sm_pack(float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// Two weights as a high and a low pair of bfloat16: x = high + low to 2^-17.
__device__ __forceinline__ void sm_split(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = sm_pack(x, y);
    lo = sm_pack(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
}

// How a group of R warps brings tiles tile0, tile0 + step, ... of 16 R keys of a part into its place in the stages: every warp 16 keys of each.
template <int HD, int R> struct SmCopy {
    static constexpr int TK = SM_WARP_KEYS * R, CH = HD / 8, AT_ONCE = 32 / CH, PIECES = SM_WARP_KEYS / AT_ONCE;      // 16-byte pieces a row; rows and pieces a warp asks for at once
    const SaArgs& a;
    const SaPart& part;
    const __nv_bfloat16* lane_src;      // this lane's piece of its row of a page's first AT_ONCE
    uint32_t lane_dst, stages;          // where it goes in a stage
    size_t to_values;                   // elements from a key to its value
    int key, step_keys, mine;           // the warp's first key of tile 0, keys from one tile to the next, tiles
    bool whole_pages;                   // sixteen keys lie in one page

    __device__ __forceinline__ SmCopy(const SaArgs& a_, const SaPart& part_, int tile0, int step, int first_row, uint32_t stages_) : a(a_), part(part_), stages(stages_) {
        const int lane = threadIdx.x & 31, row = lane / CH, piece = lane % CH;
        const int tiles = (part.k1 - part.k0 + TK - 1) / TK;
        mine = tile0 < tiles ? (tiles - tile0 + step - 1) / step : 0;
        key = part.k0 + tile0 * TK + first_row % TK;
        step_keys = step * TK;
        whole_pages = a.page_size % SM_WARP_KEYS == 0 && part.k0 % SM_WARP_KEYS == 0;
        to_values = (size_t)a.nkv * a.page_size * HD;
        lane_src = static_cast<const __nv_bfloat16*>(a.cache) + row * HD + piece * 8;
        lane_dst = (first_row + row) * (HD * 2) + ((piece ^ row) << 4);
    }
    // The page of key `lane % 16` of this warp's keys of the n-th tile; none: -1.  Only asked for: what hangs on it is worked out a tile later, so that nobody waits for it.
    __device__ __forceinline__ int page_of(int n) const {
        const int k = key + n * step_keys + (threadIdx.x & 15);
        return n < mine && k < part.k1 ? part.table[a.page_shift >= 0 ? k >> a.page_shift : k / a.page_size] : -1;
    }
    // The row of the pool that holds the key; none: ~0.
    __device__ __forceinline__ uint32_t row_of(int n, int page) const {
        const int k = key + n * step_keys + (threadIdx.x & 15), block = a.page_shift >= 0 ? k >> a.page_shift : k / a.page_size;
        return (uint32_t)page < (uint32_t)a.pages ? ((uint32_t)page * 2u * a.nkv + part.kvh) * a.page_size + (k - block * a.page_size) : 0xffffffffu;
    }
    __device__ __forceinline__ void issue(int n, int page) const {
        if (n < mine) {
            const uint32_t rows = row_of(n, page);
            const uint32_t stage = stages + (n % SM_STAGES) * SmSmem<HD>::STAGE;
            const uint32_t first = __shfl_sync(0xffffffffu, rows, 0);
            if (whole_pages && key + n * step_keys + SM_WARP_KEYS <= part.k1 && first != 0xffffffffu) {      // sixteen neighbouring rows
                const __nv_bfloat16* src = lane_src + (size_t)first * HD;
                const __nv_bfloat16* val = src + to_values;
#pragma unroll
                for (int i = 0; i < PIECES; i++) {
                    const uint32_t dst = stage + (lane_dst ^ ((i * AT_ONCE & 7) << 4)) + i * AT_ONCE * HD * 2;
                    sm_copy16(dst, src + i * AT_ONCE * HD);
                    sm_copy16(dst + SmSmem<HD>::HALF, val + i * AT_ONCE * HD);
                }
            } else {
#pragma unroll
                for (int i = 0; i < PIECES; i++) {
                    const uint32_t row = __shfl_sync(0xffffffffu, rows, i * AT_ONCE + (threadIdx.x & 31) / CH);
                    const bool there = row != 0xffffffffu;
                    const __nv_bfloat16* src = lane_src + ((there ? (size_t)row : 0) - (threadIdx.x & 31) / CH) * HD;
                    const uint32_t dst = stage + (lane_dst ^ ((i * AT_ONCE & 7) << 4)) + i * AT_ONCE * HD * 2;
                    sm_copy16_or_zero(dst, there ? src : static_cast<const __nv_bfloat16*>(a.cache), there);
                    sm_copy16_or_zero(dst + SmSmem<HD>::HALF, there ? src + to_values : static_cast<const __nv_bfloat16*>(a.cache), there);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
};

// A row's reference: scores count as 2^(score - reference), and the reference is moved to the largest score so far only when one is more than 8 above it: a weight
// is at most 2^8, float32 has room for that, and most tiles need no maximum over the row's lanes.
constexpr float SM_AHEAD = 8.0f;

// What a warp has of its 16 rows: lane (gq, qd) = (lane / 4, lane % 4) rows gq and gq + 8, dims 8 b + 2 qd and the next; the sums over this lane's keys alone.
template <int HD> struct SmRows {
    float o[HD / 8][4], m[2], l[2];
};

// A warp's walk over tiles tile0, tile0 + step, ... of 16 R keys of a part, for the rows whose queries are in qf.  `group` is the group's place among the block's, `wr` the
// warp's in the group.
template <int HD, int R>
__device__ __forceinline__ void sm_walk(const SaArgs& a, const SaPart& part, int tile0, int step, int group, int wr, const uint32_t (&qf)[HD / 16][4], SmRows<HD>& x, uint32_t stages) {
    constexpr int TK = SM_WARP_KEYS * R, CH = HD / 8, SUB = R == 1 ? 16 : 32, NB = SUB / 8;
    const int lane = threadIdx.x & 31, base_row = group * TK;
    const SmCopy<HD, R> copy(a, part, tile0, step, base_row + wr * SM_WARP_KEYS, stages);
    const float scale = a.scale_log2;
#pragma unroll
    for (int b = 0; b < HD / 8; b++) { x.o[b][0] = x.o[b][1] = x.o[b][2] = x.o[b][3] = 0.0f; }
    x.m[0] = x.m[1] = -INFINITY;
    x.l[0] = x.l[1] = 0.0f;
    const int page0 = copy.page_of(0), page1 = copy.page_of(1);
    int page = copy.page_of(2);
    copy.issue(0, page0);
    copy.issue(1, page1);
    for (int n = 0; n < copy.mine; n++) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        if (R == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(R * 32) : "memory");
        copy.issue(n + 2, page);                           // into the stage of the tile before, which the whole group is past
        page = copy.page_of(n + 3);
        const uint32_t sk = stages + (n % SM_STAGES) * SmSmem<HD>::STAGE, sv = sk + SmSmem<HD>::HALF;
        const int key0 = part.k0 + (tile0 + n * step) * TK;
#pragma unroll 1                                           // four copies of the body would not stay in the instruction cache
        for (int sub = 0; sub < TK; sub += SUB) {
            if (key0 + sub >= part.k1) break;
            float s[NB][4];
#pragma unroll
            for (int nb = 0; nb < NB; nb++) { s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.0f; }
#pragma unroll
            for (int ks = 0; ks < HD / 16; ks++)
#pragma unroll
                for (int nb = 0; nb < NB; nb += 2) {
                    const int kl = sub + nb * 8 + (lane & 7) + ((lane >> 4) << 3);
                    uint32_t b[4];
                    sm_ldsm4(b, sk + ((base_row + kl) * CH + ((ks * 2 + ((lane >> 3) & 1)) ^ (kl & 7))) * 16);
                    sm_mma(s[nb], qf[ks], b[0], b[1]);
                    sm_mma(s[nb + 1], qf[ks], b[2], b[3]);
                }
            if (key0 + sub + SUB > part.k1) {
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (key0 + sub + nb * 8 + (lane & 3) * 2 + (e & 1) >= part.k1) s[nb][e] = -INFINITY;
            }
            float top[2];
#pragma unroll
            for (int r = 0; r < 2; r++) {
                top[r] = fmaxf(s[0][2 * r], s[0][2 * r + 1]);
#pragma unroll
                for (int nb = 1; nb < NB; nb++) top[r] = fmaxf(top[r], fmaxf(s[nb][2 * r], s[nb][2 * r + 1]));
                top[r] *= scale;
            }
            if (__any_sync(0xffffffffu, top[0] > x.m[0] + SM_AHEAD || top[1] > x.m[1] + SM_AHEAD)) {
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    top[r] = fmaxf(x.m[r], top[r]);
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                    const float keep = top[r] == -INFINITY ? 0.0f : sa_ex2(x.m[r] - top[r]);
                    x.l[r] *= keep;
#pragma unroll
                    for (int b = 0; b < HD / 8; b++) { x.o[b][2 * r] *= keep; x.o[b][2 * r + 1] *= keep; }
                    x.m[r] = top[r];
                }
            }
            const float ref[2] = {x.m[0] == -INFINITY ? 0.0f : x.m[0], x.m[1] == -INFINITY ? 0.0f : x.m[1]};       // no score above -inf so far: p = 0
            uint32_t ph[NB / 2][4], pl[NB / 2][4];
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const float p0 = sa_ex2(fmaf(s[nb][2 * r], scale, -ref[r])), p1 = sa_ex2(fmaf(s[nb][2 * r + 1], scale, -ref[r]));
                    x.l[r] += p0 + p1;
                    sm_split(p0, p1, ph[nb >> 1][(nb & 1) * 2 + r], pl[nb >> 1][(nb & 1) * 2 + r]);
                }
#pragma unroll
            for (int kk = 0; kk < NB / 2; kk++)
#pragma unroll
                for (int db = 0; db < HD / 8; db += 2) {
                    const int kl = sub + kk * 16 + (lane & 15);
                    uint32_t b[4];
                    sm_ldsm4_trans(b, sv + ((base_row + kl) * CH + ((db + (lane >> 4)) ^ (kl & 7))) * 16);
                    sm_mma(x.o[db], ph[kk], b[0], b[1]);
                    sm_mma(x.o[db + 1], ph[kk], b[2], b[3]);
                    sm_mma(x.o[db], pl[kk], b[0], b[1]);
                    sm_mma(x.o[db + 1], pl[kk], b[2], b[3]);
                }
        }
    }
#pragma unroll
    for (int r = 0; r < 2; r++) {
        x.l[r] += __shfl_xor_sync(0xffffffffu, x.l[r], 1);
        x.l[r] += __shfl_xor_sync(0xffffffffu, x.l[r], 2);
    }
}

// The same for at most eight rows, with the keys as the 16 rows of the products: S^T = K Q^T, and O^T = V^T P^T with the weights turned over in registers
// (movmatrix).  Half the products and half the exponentials.  Lane (gq, qd): rows 2 qd and 2 qd + 1, dims 16 b + gq and + 8; the sums over this lane's keys alone.
template <int HD> struct SmFew {
    float o[HD / 16][4], m[2], l[2];
};
template <int HD>
__device__ __forceinline__ void sm_walk_few(const SaArgs& a, const SaPart& part, int tile0, int step, int warp, const uint32_t (&qb)[HD / 16][2], SmFew<HD>& x, uint32_t stages) {
    constexpr int CH = HD / 8;
    const int lane = threadIdx.x & 31, base_row = warp * SM_WARP_KEYS;
    const SmCopy<HD, 1> copy(a, part, tile0, step, base_row, stages);
    const float scale = a.scale_log2;
#pragma unroll
    for (int b = 0; b < HD / 16; b++) { x.o[b][0] = x.o[b][1] = x.o[b][2] = x.o[b][3] = 0.0f; }
    x.m[0] = x.m[1] = -INFINITY;
    x.l[0] = x.l[1] = 0.0f;
    const uint32_t at_k = ((base_row + (lane & 15)) * CH) * 16, at_v = ((base_row + (lane & 7) + ((lane >> 4) << 3)) * CH) * 16;      // this lane's rows for ldmatrix
    const int page0 = copy.page_of(0), page1 = copy.page_of(1);
    int page = copy.page_of(2);
    copy.issue(0, page0);
    copy.issue(1, page1);
    for (int n = 0; n < copy.mine; n++) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        copy.issue(n + 2, page);
        page = copy.page_of(n + 3);
        const uint32_t sk = stages + (n % SM_STAGES) * SmSmem<HD>::STAGE, sv = sk + SmSmem<HD>::HALF;
        const int key0 = part.k0 + (tile0 + n * step) * SM_WARP_KEYS;
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < HD / 16; ks++) {
            uint32_t k[4];
            sm_ldsm4(k, sk + at_k + (((ks * 2 + (lane >> 4)) ^ (lane & 7)) << 4));
            sm_mma(s, k, qb[ks][0], qb[ks][1]);
        }
        if (key0 + SM_WARP_KEYS > part.k1) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (key0 + (lane >> 2) + (e >> 1) * 8 >= part.k1) s[e] = -INFINITY;
        }
        float top[2] = {fmaxf(s[0], s[2]) * scale, fmaxf(s[1], s[3]) * scale};
        if (__any_sync(0xffffffffu, top[0] > x.m[0] + SM_AHEAD || top[1] > x.m[1] + SM_AHEAD)) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                top[h] = fmaxf(x.m[h], top[h]);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], d));
                const float keep = top[h] == -INFINITY ? 0.0f : sa_ex2(x.m[h] - top[h]);
                x.l[h] *= keep;
#pragma unroll
                for (int b = 0; b < HD / 16; b++) { x.o[b][h] *= keep; x.o[b][2 + h] *= keep; }
                x.m[h] = top[h];
            }
        }
        const float ref[2] = {x.m[0] == -INFINITY ? 0.0f : x.m[0], x.m[1] == -INFINITY ? 0.0f : x.m[1]};
        uint32_t ph[2], pl[2];
#pragma unroll
        for (int half = 0; half < 2; half++) {             // keys gq and gq + 8
            const float p0 = sa_ex2(fmaf(s[2 * half], scale, -ref[0])), p1 = sa_ex2(fmaf(s[2 * half + 1], scale, -ref[1]));
            x.l[0] += p0;
            x.l[1] += p1;
            uint32_t hi, lo;
            sm_split(p0, p1, hi, lo);
            ph[half] = sm_turn(hi);                        // [key][rows 2 qd, 2 qd + 1] -> [row][keys 2 qd, 2 qd + 1]
            pl[half] = sm_turn(lo);
        }
#pragma unroll
        for (int b = 0; b < HD / 16; b++) {
            uint32_t v[4];
            sm_ldsm4_trans(v, sv + at_v + (((b * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4));
            sm_mma(x.o[b], v, ph[0], ph[1]);
            sm_mma(x.o[b], v, pl[0], pl[1]);
        }
    }
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) x.l[h] += __shfl_xor_sync(0xffffffffu, x.l[h], d);
}

// The queries of up to eight rows as the 8-column operand: lane (gq, qd) has row gq, dims 2 qd, the next and + 8 of each k step.  at(row): where its query lies, null for none (zeros).
template <int HD, typename At>
__device__ __forceinline__ void sm_queries_few(const At& at, uint32_t (&qb)[HD / 16][2]) {
    const int lane = threadIdx.x & 31;
    const __nv_bfloat16* q = at(lane >> 2);
#pragma unroll
    for (int ks = 0; ks < HD / 16; ks++) {
        qb[ks][0] = q ? *reinterpret_cast<const uint32_t*>(q + 2 * (lane & 3) + ks * 16) : 0u;
        qb[ks][1] = q ? *reinterpret_cast<const uint32_t*>(q + 2 * (lane & 3) + ks * 16 + 8) : 0u;
    }
}

// The same of rows row0 + gq and row0 + gq + 8 as the 16-row operand.
template <int HD, typename At>
__device__ __forceinline__ void sm_queries(const At& at, int row0, uint32_t (&qf)[HD / 16][4]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < 2; r++) {
        const __nv_bfloat16* q = at(row0 + (lane >> 2) + 8 * r);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ks++) {
            qf[ks][r] = q ? *reinterpret_cast<const uint32_t*>(q + 2 * (lane & 3) + ks * 16) : 0u;
            qf[ks][r + 2] = q ? *reinterpret_cast<const uint32_t*>(q + 2 * (lane & 3) + ks * 16 + 8) : 0u;
        }
    }
}

// Where the query of a part's row lies; null: no such row, or its member is not there.
struct SmQueryOf {
    const SaArgs& a;
    const SaPlan& p;
    const SaPart& part;
    int hd;
    __device__ __forceinline__ const __nv_bfloat16* operator()(int row) const {
        const int i = part.i0 + row / part.heads;
        if (row >= (part.i1 - part.i0) * part.heads || p.pos[i] < 0) return nullptr;
        return static_cast<const __nv_bfloat16*>(a.q) + ((size_t)p.tok[i] * a.nh + part.kvh * a.gq + part.h0 + row % part.heads) * hd;
    }
};

// The outputs that a block's groups of R warps left in shared memory ([8 warps][16][HD + 4], maxima and sums behind them) meet, and the part's rows are written.
template <int HD, int R>
__device__ __forceinline__ void sm_meet(const SaArgs& a, const SaPart& part, const unsigned char* stages) {
    constexpr int GROUPS = (SA_THREADS / 32) / R, LD = HD + 4;
    const float* out = reinterpret_cast<const float*>(stages);
    const float2 (*ml)[16] = reinterpret_cast<const float2 (*)[16]>(stages + SmSmem<HD>::OUT);
    const int rows = (part.i1 - part.i0) * part.heads;
    __syncthreads();
#pragma unroll 1
    for (int c = threadIdx.x; c < rows * (HD / 4); c += SA_THREADS) {
        const int row = c / (HD / 4), d = c % (HD / 4) * 4, w0 = row / 16, rr = row % 16;
        float m = -INFINITY;
#pragma unroll
        for (int g = 0; g < GROUPS; g++) m = fmaxf(m, ml[g * R + w0][rr].x);
        const float ref = m == -INFINITY ? 0.0f : m;
        float l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int g = 0; g < GROUPS; g++) {
            const float2 s = ml[g * R + w0][rr];
            const float w = sa_ex2(s.x - ref);
            const float4 v = *reinterpret_cast<const float4*>(out + ((g * R + w0) * 16 + rr) * LD + d);
            l += s.y * w;
            o.x += v.x * w; o.y += v.y * w; o.z += v.z * w; o.w += v.w * w;
        }
        const int at = part.row0 + row * part.stride;
        *reinterpret_cast<float4*>(a.part_o + (size_t)at * HD + d) = o;
        if (d == 0) a.part_ml[at] = make_float2(m, l);
    }
}

// A block's part of a family's prefix: 8 / R groups of R warps; their outputs meet in shared memory and the part's rows are written.
template <int HD, int R>
__device__ __forceinline__ void sm_prefix(const SaArgs& a, const SaPlan& p, const SaPart& part, unsigned char* stages) {
    constexpr int GROUPS = (SA_THREADS / 32) / R, LD = HD + 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = warp / R, wr = warp % R;
    const int rows = (part.i1 - part.i0) * part.heads;
    uint32_t qf[HD / 16][4];
    sm_queries<HD>(SmQueryOf{a, p, part, HD}, wr * 16, qf);
    SmRows<HD> x;
    sm_walk<HD, R>(a, part, group, GROUPS, group, wr, qf, x, sm_addr(stages));
    if (GROUPS == 1) {
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int row = wr * 16 + (lane >> 2) + 8 * r;
            if (row >= rows) continue;
            const int at = part.row0 + row * part.stride;
#pragma unroll
            for (int b = 0; b < HD / 8; b++) *reinterpret_cast<float2*>(a.part_o + (size_t)at * HD + b * 8 + 2 * (lane & 3)) = make_float2(x.o[b][2 * r], x.o[b][2 * r + 1]);
            if ((lane & 3) == 0) a.part_ml[at] = make_float2(x.m[r], x.l[r]);
        }
        return;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                                       // every group is past its tiles
    float* out = reinterpret_cast<float*>(stages);
    float2 (*ml)[16] = reinterpret_cast<float2 (*)[16]>(stages + SmSmem<HD>::OUT);
#pragma unroll
    for (int r = 0; r < 2; r++) {
        const int row = (lane >> 2) + 8 * r;
#pragma unroll
        for (int b = 0; b < HD / 8; b++) *reinterpret_cast<float2*>(out + (warp * 16 + row) * LD + b * 8 + 2 * (lane & 3)) = make_float2(x.o[b][2 * r], x.o[b][2 * r + 1]);
        if ((lane & 3) == 0) ml[warp][row] = make_float2(x.m[r], x.l[r]);
    }
    sm_meet<HD, R>(a, part, stages);
}

// The same of at most eight rows: every warp by itself.
template <int HD>
__device__ __forceinline__ void sm_prefix_few(const SaArgs& a, const SaPlan& p, const SaPart& part, unsigned char* stages) {
    constexpr int LD = HD + 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t qb[HD / 16][2];
    sm_queries_few<HD>(SmQueryOf{a, p, part, HD}, qb);
    SmFew<HD> x;
    sm_walk_few<HD>(a, part, warp, SA_THREADS / 32, warp, qb, x, sm_addr(stages));
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    float* out = reinterpret_cast<float*>(stages);
    float2 (*ml)[16] = reinterpret_cast<float2 (*)[16]>(stages + SmSmem<HD>::OUT);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int row = 2 * (lane & 3) + h;
#pragma unroll
        for (int b = 0; b < HD / 16; b++) {
            out[(warp * 16 + row) * LD + b * 16 + (lane >> 2)] = x.o[b][h];
            out[(warp * 16 + row) * LD + b * 16 + (lane >> 2) + 8] = x.o[b][2 + h];
        }
        if (lane < 4) ml[warp][row] = make_float2(x.m[h], x.l[h]);
    }
    sm_meet<HD, 1>(a, part, stages);
}

// ---- prefixes of many rows, on the fifth-generation tensor cores ---------------------------------------------------------------------------------
//
// The part's rows (up to 128) are the lanes of tensor memory.  Two groups of four warps walk tiles of 64 keys in turn, each by itself: scores S[128 x 64] = Q K^T out of shared memory, a
// thread a row takes them out, and puts the weights back in their place as high and low parts (32 keys in 16 + 16 columns); O[128 x HD] += P V has them from there and stays in
// tensor memory.  Keys and values come by cp.async into rows of 128 bytes, 16-byte pieces at piece ^ (key & 7) (the 128-byte swizzle): keys two tiles ahead, values one, each into the
// stage that the product before is known to have read.  While one group's weights are worked out the other's products run.
//
// Where: heads of 128 and 65 rows or more.  16 members of 16 heads over 2 of 128 (128 rows) behind 32,000 positions, whole call, 28.0 us against 36.1 with mma.sync, behind 8,000 19.3 / 20.0;
// 32 members behind 4,000 18.2 / 18.4 (the launch that joins the parts has become faster since, for both).  Between 64 and 128 rows, eight of them a member: over 2 heads behind 16,000 and 32,000
// 72 rows 20.6 / 22.7 and 26.0 / 31.6, 96 rows 20.1 / 23.5 and 26.8 / 32.3, 120 rows 20.6 / 24.0 and 26.6 / 33.6, over 8 heads 34.5 / 48.9 and 51.4 / 79.4, 36.9 / 49.7 and 51.9 / 79.7, 36.8 / 50.2
// and 54.8 / 89.4; behind 4,000 both the same within 3 %, but 120 rows over 8 heads 25.1 / 22.8.  With up to 64 rows the lanes that stand for none cost as much as the others (40 rows behind
// 16,000: 19.9 / 19.4; 64 behind 8,000, 8 key-value heads: 24.3 / 22.7), and heads of 64 have half the products for the same exponentials: 64 rows behind 2,000, 32 heads, 27.7 / 24.3; 96 rows
// behind 4,000, 5 heads, 17.0 / 15.6.
//
// What bounds it.  A tile takes its group 2,800 cycles (S 220 from its issue, a thread's 64 weights 1,500, P V 700 until the next S may begin), two groups beside one another, and in the first of
// these cases (26.6 us now) a group has four tiles.  Before them are the plan, 5,000, and the queries, pages and first keys, behind them the groups' meeting, 4,000, and the join: a short
// chain that meets most of its instructions for the first time (4.6 warps wait for them for each that issues; the tensor pipe is at 10 %).
constexpr int SM_TENSOR_ROWS = 65;

template <int HD> struct SmTc {
    static constexpr int KEYS = 64, ROWS = 128, PANELS = HD / 64, PANEL = KEYS * 128, TILE = PANELS * PANEL, Q_PANEL = ROWS * 128, Q = PANELS * Q_PANEL;      // panels of 64 dims
    static constexpr int GROUP = 4 * TILE;                                            // a group's keys, two stages, and values, two
    static constexpr int OUT = 2 * ROWS * (HD + 4) * 4, ML = 2 * ROWS * 8;            // where the groups' outputs meet
    static constexpr uint32_t O_COL = 2 * KEYS, TMEM = 512;                           // columns: the groups' scores, their outputs
    static_assert(1024 + Q + 2 * GROUP <= SM_STAGES * SmSmem<HD>::STAGE && OUT + ML <= SM_STAGES * SmSmem<HD>::STAGE && O_COL + 2 * HD <= TMEM, "it lies over the stages");
};

// Of a block: the tensor memory, the groups' barriers (scores done, output done) and their phases, and whether a wait has run out.
struct SmTcBlock {
    uint32_t tmem;
    uint64_t* bars;
    int phase;
    bool lost;
};

// The product with the first operand in tensor memory (128 lanes, two bfloat16 values a column).
__device__ __forceinline__ void sm_umma_ts(uint32_t d, uint32_t at, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tmov.b64 db, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}"
        ::"r"(d), "r"(at), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(UMMA_DESC_HI_SW128));
}
__device__ __forceinline__ void sm_tmem_st16(uint32_t at, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                 "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}

template <int HD>
__device__ __forceinline__ void sm_prefix_tc(const SaArgs& a, const SaPlan& p, const SaPart& part, unsigned char* stages, SmTcBlock& block, const WaitCtl& wc, int* failed) {
    typedef SmTc<HD> S;
    constexpr int CH = HD / 8, AT_ONCE = 128 / CH, PIECES = S::KEYS / AT_ONCE, RW = 32 / CH, LD = HD + 4;      // 16-byte pieces a row; rows a group, a warp copies at once
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = warp >> 2, w = warp & 3, r = tid & 127, rows = (part.i1 - part.i0) * part.heads;
    unsigned char* base = stages + ((1024 - (sm_addr(stages) & 1023)) & 1023);
    const int tiles = (part.k1 - part.k0 + S::KEYS - 1) / S::KEYS, mine = (tiles - group + 1) / 2;      // this group's: group, group + 2, ...
    const uint32_t ring = sm_addr(base) + S::Q + group * S::GROUP;
    const int crow = r / CH, piece = r % CH, my_key = w * RW + lane % RW + (lane & 15) / RW * AT_ONCE;      // the key of a tile whose page this lane asks for
    const uint32_t lane_dst = (piece >> 3) * S::PANEL + crow * 128 + (((piece & 7) ^ (crow & 7)) << 4);
    const size_t to_values = (size_t)a.nkv * a.page_size * HD;
    const __nv_bfloat16* cache = static_cast<const __nv_bfloat16*>(a.cache);
    auto page_of = [&](int n) -> int {
        const int k = part.k0 + (group + 2 * n) * S::KEYS + my_key;
        return n < mine && k < part.k1 ? part.table[a.page_shift >= 0 ? k >> a.page_shift : k / a.page_size] : -1;
    };
    auto row_of = [&](int n, int page) -> uint32_t {           // the row of the pool that holds the key; none: ~0
        const int k = part.k0 + (group + 2 * n) * S::KEYS + my_key, in_page = a.page_shift >= 0 ? k & (a.page_size - 1) : k % a.page_size;
        return (uint32_t)page < (uint32_t)a.pages ? ((uint32_t)page * 2u * a.nkv + part.kvh) * a.page_size + in_page : 0xffffffffu;
    };
    auto copy = [&](int n, uint32_t from, uint32_t stage, size_t more) {      // a tile's keys, or values
        if (n >= mine) return;
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const uint32_t row = __shfl_sync(0xffffffffu, from, i * RW + lane / CH);
            const bool there = row != 0xffffffffu;
            sm_copy16_or_zero(stage + lane_dst + i * AT_ONCE * 128, there ? cache + (size_t)row * HD + piece * 8 + more : cache, there);
        }
    };
    auto landed = [&]() {                                      // all but the newest of this thread's copies have, and the tensor core may read them behind the group's meeting
        asm volatile("cp.async.wait_group 1;\nfence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
    };
    auto wait = [&](uint64_t* bar, int phase) {                // once a wait has run out there are no more
        if (!block.lost && !__all_sync(0xffffffffu, mbar_wait(bar, (uint32_t)phase & 1, wc.cycles))) {
            block.lost = true;
            if (lane == 0) give_up(wc.error, failed, 81);
        }
        tc_fence_after();
    };
    uint64_t *s_done = block.bars + group, *o_done = block.bars + 2 + group;
    const uint32_t lanes = (uint32_t)(w * 32) << 16, s_at = block.tmem + group * S::KEYS, o_at = block.tmem + S::O_COL + group * HD;
    const uint32_t s_desc = umma_idesc_bf16(S::ROWS, S::KEYS), o_desc = umma_idesc_bf16(S::ROWS, HD) | (1u << 16);      // (the values are N-major)
    const float scale = a.scale_log2;
    float m = -INFINITY, l = 0.0f;

    // what the first tiles and the queries hang on is asked for before any of it is used
    const int page0 = page_of(0), page1 = page_of(1);
    int page = page_of(2);
    const SmQueryOf query_of{a, p, part, HD};
    uint4 queries[S::ROWS * CH / SA_THREADS];
#pragma unroll
    for (int i = 0; i < S::ROWS * CH / SA_THREADS; i++) {
        const __nv_bfloat16* q = query_of(tid / CH + i * (SA_THREADS / CH));
        queries[i] = q ? *reinterpret_cast<const uint4*>(q + tid % CH * 8) : make_uint4(0, 0, 0, 0);
    }
    uint32_t now = row_of(0, page0), next = row_of(1, page1);
    copy(0, now, ring, 0);
    asm volatile("cp.async.commit_group;" ::: "memory");
    copy(1, next, ring + S::TILE, 0);
    copy(0, now, ring + 2 * S::TILE, to_values);
    asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
    for (int i = 0; i < S::ROWS * CH / SA_THREADS; i++) {
        const int row = tid / CH + i * (SA_THREADS / CH), piece = tid % CH;
        *reinterpret_cast<uint4*>(base + (piece >> 3) * S::Q_PANEL + row * 128 + (((piece & 7) ^ (row & 7)) << 4)) = queries[i];
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
#pragma unroll 1
    for (int n = 0; n < mine; n++) {
        landed();
        if (w == 0) {
            if (n > 0) wait(o_done, block.phase + n - 1);      // the scores take the place of weights that the tensor core has read
            if (elect_one()) {
                const uint32_t q_lo = umma_desc_lo(sm_addr(base)), k_lo = umma_desc_lo(ring + (n & 1) * S::TILE);
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < HD / 16; k++) umma_bf16_lo(s_at, q_lo + (k / 4) * (S::Q_PANEL >> 4) + 2 * (k % 4), k_lo + (k / 4) * (S::PANEL >> 4) + 2 * (k % 4), s_desc, k != 0);
                if (n != wc.skip_stage) umma_commit(s_done);   // (a tile named by wc.skip_stage is never told of: a test of the give-up path)
            }
            __syncwarp();
        }
        const uint32_t after = row_of(n + 2, page);
        page = page_of(n + 3);
        wait(s_done, block.phase + n);                         // and so the keys' stage and the values' other one have been read
        copy(n + 2, after, ring + (n & 1) * S::TILE, 0);
        copy(n + 1, next, ring + (2 + ((n + 1) & 1)) * S::TILE, to_values);
        asm volatile("cp.async.commit_group;" ::: "memory");
        next = after;
        // 32 scores at a time, in loops that are not unrolled: a block walks few tiles, and instructions that it meets for the first time cost it more than the second reading
        const int left = part.k1 - (part.k0 + (group + 2 * n) * S::KEYS);
        float top = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < S::KEYS; c += 32) {
            uint32_t s[32];
            tmem_ld32(s_at + lanes + c, s);
            tmem_loaded(s);
            if (left < c + 32) {
#pragma unroll
                for (int j = 0; j < 32; j++)
                    if (c + j >= left) s[j] = 0xff800000u;
                tmem_st32(s_at + lanes + c, s);
                tmem_wait_st();
            }
#pragma unroll
            for (int j = 0; j < 32; j++) top = fmaxf(top, __uint_as_float(s[j]));
        }
        top *= scale;
        const bool ahead = top > m + SM_AHEAD;
        if (__any_sync(0xffffffffu, ahead)) {
            const float keep = ahead ? sa_ex2(m - top) : 1.0f;
            l *= keep;
            if (ahead) m = top;
            if (n > 0) {
#pragma unroll 1
                for (int c = 0; c < HD; c += 16) {
                    uint32_t o[16];
                    tmem_ld16(o_at + lanes + c, o);
#pragma unroll
                    for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
                    sm_tmem_st16(o_at + lanes + c, o);
                }
            }
        }
        const float ref = m == -INFINITY ? 0.0f : m;           // no score above -inf so far: p = 0
        float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll 1
        for (int c = 0; c < S::KEYS; c += 32) {
            uint32_t s[32], hi[16], lo[16];
            tmem_ld32(s_at + lanes + c, s);
            tmem_loaded(s);
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const float p0 = sa_ex2(fmaf(__uint_as_float(s[2 * j]), scale, -ref)), p1 = sa_ex2(fmaf(__uint_as_float(s[2 * j + 1]), scale, -ref));
                sum0 += p0;
                sum1 += p1;
                sm_split(p0, p1, hi[j], lo[j]);
            }
            sm_tmem_st16(s_at + lanes + c, hi);
            sm_tmem_st16(s_at + lanes + c + 16, lo);
        }
        l += sum0 + sum1;
        tmem_wait_st();
        tc_fence_before();
        landed();
        if (w == 0) {
            if (elect_one()) {
                const uint32_t v_lo = ((ring + (2 + (n & 1)) * S::TILE) >> 4) | ((uint32_t)(S::PANEL >> 4) << 16);      // the panels' distance is the leading byte offset
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < S::KEYS / 16; k++) sm_umma_ts(o_at, s_at + 32 * (k / 2) + 8 * (k % 2), v_lo + k * (2048 >> 4), o_desc, n > 0 || k != 0);
#pragma unroll
                for (int k = 0; k < S::KEYS / 16; k++) sm_umma_ts(o_at, s_at + 32 * (k / 2) + 16 + 8 * (k % 2), v_lo + k * (2048 >> 4), o_desc, 1);
                umma_commit(o_done);
            }
            __syncwarp();
        }
    }
    if (mine > 0) wait(o_done, block.phase + mine - 1);
    block.phase += mine;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                                           // both groups are past their tiles
    float* out = reinterpret_cast<float*>(stages);
    float2* ml = reinterpret_cast<float2*>(stages + S::OUT);
#pragma unroll 1
    for (int c = 0; c < HD; c += 16) {
        uint32_t o[16];
        tmem_ld16(o_at + lanes + c, o);
#pragma unroll
        for (int j = 0; j < 16; j += 4)                        // a group without a tile has nothing
            *reinterpret_cast<uint4*>(out + tid * LD + c + j) = mine > 0 ? make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]) : make_uint4(0, 0, 0, 0);
    }
    ml[tid] = make_float2(m, l);
    tc_fence_before();
    __syncthreads();
#pragma unroll 1
    for (int c = tid; c < rows * (HD / 4); c += SA_THREADS) {
        const int row = c / (HD / 4), d = c % (HD / 4) * 4;
        const float2 x = ml[row], y = ml[S::ROWS + row];
        const float most = fmaxf(x.x, y.x), ref = most == -INFINITY ? 0.0f : most, wx = sa_ex2(x.x - ref), wy = sa_ex2(y.x - ref);
        const float4 u = *reinterpret_cast<const float4*>(out + row * LD + d), v = *reinterpret_cast<const float4*>(out + (S::ROWS + row) * LD + d);
        const int at = part.row0 + row * part.stride;
        *reinterpret_cast<float4*>(a.part_o + (size_t)at * HD + d) = make_float4(u.x * wx + v.x * wy, u.y * wx + v.y * wy, u.z * wx + v.z * wy, u.w * wx + v.w * wy);
        if (d == 0) a.part_ml[at] = make_float2(most, x.y * wx + y.y * wy);
    }
}

// What a warp's walk of an own part leaves: the result where the unit needs nobody else, else the part's row.
template <int HD>
__device__ __forceinline__ void sm_leave(const SaArgs& a, const SaPlan& p, const SaPart& part, bool alone, int row, int d, float x, float y) {
    if (alone) *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.out) + ((size_t)p.tok[part.i0] * a.nh + part.kvh * a.gq + part.h0 + row) * HD + d) = sm_pack(x, y);
    else *reinterpret_cast<float2*>(a.part_o + (size_t)(part.row0 + row * part.stride) * HD + d) = make_float2(x, y);
}

template <int HD>
__global__ void __launch_bounds__(SA_THREADS, HD == 64 ? 2 : 1) attention_shared_mma_kernel(const SaArgs a, const WaitCtl wc) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint64_t bars[4];
    __shared__ uint32_t tmem_at;
    __shared__ int failed;
    constexpr bool TENSOR = HD == 128;
    SaPlan& p = *reinterpret_cast<SaPlan*>(smem);
    unsigned char* stages = smem + SmSmem<HD>::PLAN;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    sa_make_plan(a, p);                       // and the wait for the kernel before this one
    const bool prefix = (int)blockIdx.x < p.prefix_blocks;
    // tensor memory where some prefix has many rows, before the kernel after this one may come and want some
    const bool tensor = TENSOR && prefix && __syncthreads_or(p.shared[threadIdx.x] > 0 && min(p.width[threadIdx.x], p.tile_members) * a.gq >= SM_TENSOR_ROWS);
    SmTcBlock block = {0, bars, 0, false};
    if (tensor) {
        if (threadIdx.x == 0) {
            failed = 0;
            for (int b = 0; b < 4; b++) mbar_init(&bars[b], 1);
            asm volatile("fence.mbarrier_init.release.cluster;\nfence.proxy.async.shared::cta;" ::: "memory");
        }
        if (warp == 0) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm_addr(&tmem_at)), "r"(SmTc<HD>::TMEM) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        block.tmem = tmem_at;
    }
    let_dependents_start();
    SaPart part;
    int at = blockIdx.x * p.lp, end = prefix ? min(at + p.lp, p.pbase[SA_MAX_TOKENS]) : 0;
    while (at < end) {
        if (!sa_prefix_part(a, p, at, end, blockIdx.x, part)) continue;
        const int rows = (part.i1 - part.i0) * part.heads;
        if (rows <= 8) sm_prefix_few<HD>(a, p, part, stages);
        else if (rows <= 16) sm_prefix<HD, 1>(a, p, part, stages);
        else if (rows <= 32) sm_prefix<HD, 2>(a, p, part, stages);
        else if (rows <= 64) sm_prefix<HD, 4>(a, p, part, stages);
        else if constexpr (TENSOR) sm_prefix_tc<HD>(a, p, part, stages, block, wc, &failed);
        else sm_prefix<HD, 8>(a, p, part, stages);
        __syncthreads();
    }
    if (TENSOR && tensor && warp == 0) {
        if (failed) __nanosleep(200000);      // after a failed wait: let products in flight end
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(block.tmem), "r"(SmTc<HD>::TMEM) : "memory");
    }
    // every warp by itself; neighbouring parts of the own keys go to different multiprocessors
    const int worker = prefix ? 0 : warp * ((int)gridDim.x - p.prefix_blocks) + (int)blockIdx.x - p.prefix_blocks;
    at = worker * p.lo;
    end = prefix ? 0 : min(at + p.lo, p.obase[SA_MAX_TOKENS]);
    while (at < end) {
        int parts;
        if (!sa_own_part(a, p, at, end, worker, part, parts)) continue;
        const bool alone = parts == 1 && p.shared[part.g] == 0;      // the unit needs nobody else
        __syncwarp();                                      // the lanes are past the tiles of the part before
        if (part.heads <= 8) {
            uint32_t qb[HD / 16][2];
            sm_queries_few<HD>(SmQueryOf{a, p, part, HD}, qb);
            SmFew<HD> x;
            sm_walk_few<HD>(a, part, 0, 1, warp, qb, x, sm_addr(stages));
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int row = 2 * (lane & 3) + h, gq = lane >> 2;
                const float w = alone ? 1.0f / x.l[h] : 1.0f;
#pragma unroll
                for (int b = 0; b < HD / 16; b++) {        // neighbouring dims lie in neighbouring lanes' registers: even lanes take the lower eight, odd ones the upper
                    const float lo = x.o[b][h] * w, up = x.o[b][2 + h] * w;
                    const float got = __shfl_xor_sync(0xffffffffu, gq & 1 ? lo : up, 4);
                    if (row < part.heads) sm_leave<HD>(a, p, part, alone, row, b * 16 + (gq & 1 ? 8 + gq - 1 : gq), gq & 1 ? got : lo, gq & 1 ? up : got);
                }
                if (!alone && lane < 4 && row < part.heads) a.part_ml[part.row0 + row * part.stride] = make_float2(x.m[h], x.l[h]);
            }
        } else {
            uint32_t qf[HD / 16][4];
            sm_queries<HD>(SmQueryOf{a, p, part, HD}, 0, qf);
            SmRows<HD> x;
            sm_walk<HD, 1>(a, part, 0, 1, warp, 0, qf, x, sm_addr(stages));
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int row = (lane >> 2) + 8 * r;
                if (row >= part.heads) continue;
                const float w = alone ? 1.0f / x.l[r] : 1.0f;
#pragma unroll
                for (int b = 0; b < HD / 8; b++) sm_leave<HD>(a, p, part, alone, row, b * 8 + 2 * (lane & 3), x.o[b][2 * r] * w, x.o[b][2 * r + 1] * w);
                if (!alone && (lane & 3) == 0) a.part_ml[part.row0 + row * part.stride] = make_float2(x.m[r], x.l[r]);
            }
        }
    }
    sa_write_rows(a, p);
}

// ---- every member by itself ---------------------------------------------------------------------------------------------------------------
//
// Where the members' tables are short and few, reading common keys once is worth less than what it takes to find out who has which in common and to bring the two kinds of parts
// together: a cluster of blocks walks a member's whole table for one tile of heads, a run of its keys a block, its eight warps in turn, and the blocks' outputs meet through
// each other's shared memory.  One launch, nothing in scratch memory.  Four beams of 512 positions, 9 heads over 3 of 64: 4.7 us in a captured graph, caches cold (with the lists read before the wait 4.2, and 8.2 the other way); the launch, six dependent trips to
// memory and the cluster's two meetings are all of it.

template <int HD>
__global__ void __launch_bounds__(SA_THREADS, HD == 64 ? 2 : 1) attention_each_mma_kernel(const SaArgs a) {
    extern __shared__ __align__(128) unsigned char stages[];
    constexpr int LD = HD + 4;
    __shared__ float row_m[16], row_l[16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    SaPart part;
    int token;
    if (!sa_each_part(a, 16, part, token)) return;                                        // the wait for the kernel before this one is in there
    const __nv_bfloat16* queries = static_cast<const __nv_bfloat16*>(a.q) + ((size_t)token * a.nh + part.kvh * a.gq + part.h0) * HD;
    auto query_of = [&](int row) -> const __nv_bfloat16* { return row < part.heads ? queries + row * HD : nullptr; };
    float* out = reinterpret_cast<float*>(stages);                                        // the warps' outputs, over the stages: [8][16][LD]
    float2 (*ml)[16] = reinterpret_cast<float2 (*)[16]>(stages + SmSmem<HD>::OUT);
    float* whole = reinterpret_cast<float*>(stages + SmSmem<HD>::OUT + SmSmem<HD>::ML);      // and the block's: [16][HD]
    static_assert(SmSmem<HD>::OUT + SmSmem<HD>::ML + 16 * HD * 4 <= SM_STAGES * SmSmem<HD>::STAGE, "the block's output lies behind the warps'");
    let_dependents_start();
    if (part.heads <= 8) {
        uint32_t qb[HD / 16][2];
        sm_queries_few<HD>(query_of, qb);
        SmFew<HD> x;
        sm_walk_few<HD>(a, part, warp, SA_THREADS / 32, warp, qb, x, sm_addr(stages));
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int row = 2 * (lane & 3) + h;
#pragma unroll
            for (int b = 0; b < HD / 16; b++) {
                out[(warp * 16 + row) * LD + b * 16 + (lane >> 2)] = x.o[b][h];
                out[(warp * 16 + row) * LD + b * 16 + (lane >> 2) + 8] = x.o[b][2 + h];
            }
            if (lane < 4) ml[warp][row] = make_float2(x.m[h], x.l[h]);
        }
    } else {
        uint32_t qf[HD / 16][4];
        sm_queries<HD>(query_of, 0, qf);
        SmRows<HD> x;
        sm_walk<HD, 1>(a, part, warp, SA_THREADS / 32, warp, 0, qf, x, sm_addr(stages));
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int row = (lane >> 2) + 8 * r;
#pragma unroll
            for (int b = 0; b < HD / 8; b++) *reinterpret_cast<float2*>(out + (warp * 16 + row) * LD + b * 8 + 2 * (lane & 3)) = make_float2(x.o[b][2 * r], x.o[b][2 * r + 1]);
            if ((lane & 3) == 0) ml[warp][row] = make_float2(x.m[r], x.l[r]);
        }
    }
    __syncthreads();
    sa_each_join<__nv_bfloat16, SA_THREADS / 32>(a, part, token, 16, LD, out, &ml[0][0], whole, row_m, row_l);
}

// Rows of the pool are counted in 32 bits here, and a row's largest score is that of its largest product.
bool attention_shared_mma_takes(const SaArgs& a, int dtype) {
    return dtype == 1 && (a.hd == 64 || a.hd == 128) && a.scale_log2 > 0.0f && (long long)a.pages * 2 * a.nkv * a.page_size < 0x7fffffffLL;
}

// Every member by itself, where all tables at their full width are few bytes (what the members really have is on the device).  Measured on families of 2 to 64 members, this way
// against the other (bytes of the whole tables in brackets).  Heads of 64: 64 members of 512 common and up to 64 own positions, 5 key-value heads (48 MB), 8.9 us against 14.8;
// 32 of 2,048, 5 heads (87 MB), 12.7 / 14.4; 8 of 2,048, 5 heads (44 MB), 6.6 / 9.8; 4 of 2,048, 32 heads (70 MB), 8.8 / 10.6; 16 of 512, 32 heads (78 MB), 10.3 / 11.3; 16 of 8,000, 3 heads
// (99 MB), 13.8 / 12.7; 64 of 128, 32 heads (109 MB), 20.4 / 15.6; 8 of 2,048, 32 heads (139 MB), 12.7 / 11.4; 64 of 512, 32 heads (310 MB), 34 / 17.  Heads of 128 (2 of them, 8 queries
// each): 16 of 8,000 (132 MB) 14.8 / 19.5, 64 of 2,048 (139 MB) 13.6 / 21.8, 32 of 8,000 (265 MB) 23.5 / 23.3, 64 of 8,000 (530 MB) 40 / 35.
// attention_decode, which reads every member's table too but in runs of 256 keys that meet through memory, has 4 key-value heads of four queries each, in tables of 4,096, so (this way / it):
// heads of 64, 4 members of 500 common positions 5.1 / 4.1 us, of 2,000 5.9 / 4.6, 8 of 2,000 6.6 / 5.3, 16 of 500 5.5 / 4.8, of 2,000 7.2 / 10.2; heads of 128, 4 of 500 5.8 / 5.0, of 2,000 7.5 / 5.9,
// 8 of 2,000 7.8 / 11.7, 16 of 500 6.3 / 11.0, of 2,000 10.0 / 23.0.  ops.attention chooses between the two by whole steps (attention_shared_pays).
bool attention_each_mma_takes(const SaArgs& a) {
    return (long long)a.n * a.max_blocks * a.page_size * a.nkv * a.hd * 4 <= (a.hd == 64 ? 96ll << 20 : 240ll << 20);
}
// A block for every 256 keys of a table, but no more blocks than run at once, and clusters of at most eight (four where a block fills a multiprocessor).
int launch_attention_each_mma(const SaArgs& a, int multiprocessors, cudaStream_t stream) {
    const int units = a.nkv * ((a.gq + 15) / 16) * a.n, room = multiprocessors * (a.hd == 64 ? 2 : 1), most = a.hd == 64 ? 8 : 4;
    int ranks = 1;
    while (ranks < most && ranks * 256 < (long long)a.max_blocks * a.page_size && 2 * ranks * units <= room) ranks *= 2;
    const dim3 grid(ranks, a.nkv * ((a.gq + 15) / 16), a.n);
#define GO(HD)                                                                                                                                  \
    do {                                                                                                                                        \
        const int e = sa_allow_smem(attention_each_mma_kernel<HD>, SM_STAGES * SmSmem<HD>::STAGE);                                              \
        if (e != VK_OK) return e;                                                                                                               \
        return launch_dependent_cluster(attention_each_mma_kernel<HD>, grid, dim3(SA_THREADS), ranks, SM_STAGES * SmSmem<HD>::STAGE, stream, a); \
    } while (0)
    if (a.hd == 64) GO(64);
    GO(128);
#undef GO
}

int launch_attention_shared_mma(SaArgs a, int multiprocessors, int* error, cudaStream_t stream) {
    a.prefix_rows = SM_PREFIX_ROWS;
    a.own_rows = 16;
    a.row_unit = 16.0f;
    const int blocks = multiprocessors * (a.hd == 64 ? 2 : 1);
    a.blocks = blocks;
    a.own_per_block = SA_THREADS / 32;
    a.min_prefix = 8;
    a.min_own = 4;
    a.prefix_cost = 16;
    a.own_cost = 8;
    a.tensor_rows = a.hd == 128 ? SM_TENSOR_ROWS : 0x7fffffff;
    a.tensor_unit = 1.0f;
#define GO(HD)                                                                                                                                          \
    do {                                                                                                                                        \
        auto kern = attention_shared_mma_kernel<HD>;                                                                                    \
        const int e = sa_allow_smem(kern, SmSmem<HD>::BYTES);                                                                                   \
        if (e != VK_OK) return e;                                                                                                               \
        return launch_dependent(kern, dim3(blocks), dim3(SA_THREADS), SmSmem<HD>::BYTES, stream, a, wait_ctl(error, WAIT_FAMILY_ATTENTION_SHARED)); \
    } while (0)
    if (a.hd == 64) GO(64);
    GO(128);
#undef GO
}

}  // namespace vk
