// Rows of an arena move: arena[l][dst_i] = arena[l][src_i] for every layer l and move i, in one launch.
//
// What a beam search does to the cache between two steps: a page pool's layers get a copy of the page that two beams would go on writing into, the slots of a
// recurrent model the state of the beam that was chosen.  No row is both read and written, which the caller sees to, so the
// blocks need no order.  Reads and writes of the moved bytes are all there is: a block moves 16 KB, four 16-byte pieces a thread asked for before
// the first is stored.  The moves are arguments of the launch (up to 128 at a time): nothing is copied to the device for them.  Seven states of 1 MB in
// twelve layers (176 MB read and written): 22.5 us, 7.8 TB/s (the second-level cache holds part of them); three pages of 12 KB in thirty layers: 1.2 us, and the host's call 7.
#include "common.cuh"

namespace vk {

constexpr int CR_THREADS = 256, CR_MOVES = 128, CR_PIECES = 4;

struct CrArgs {
    char* base;
    long long layer_stride, row_stride, row_bytes;
    int32_t src[CR_MOVES], dst[CR_MOVES];
};

template <typename V>
__global__ void __launch_bounds__(CR_THREADS) copy_rows_kernel(const __grid_constant__ CrArgs a) {
    dependency_wait();
    char* layer = a.base + (size_t)blockIdx.z * a.layer_stride;
    const char* src = layer + (size_t)a.src[blockIdx.y] * a.row_stride;
    char* dst = layer + (size_t)a.dst[blockIdx.y] * a.row_stride;
    const long long whole = a.row_bytes / (long long)sizeof(V), first = (long long)blockIdx.x * CR_THREADS * CR_PIECES + threadIdx.x;
    V v[CR_PIECES];
#pragma unroll
    for (int j = 0; j < CR_PIECES; j++)
        if (first + j * CR_THREADS < whole) v[j] = reinterpret_cast<const V*>(src)[first + j * CR_THREADS];
#pragma unroll
    for (int j = 0; j < CR_PIECES; j++)
        if (first + j * CR_THREADS < whole) reinterpret_cast<V*>(dst)[first + j * CR_THREADS] = v[j];
    // what is left of a row behind its last whole piece
    const long long rest = whole * (long long)sizeof(V) + threadIdx.x;
    if (blockIdx.x == 0 && rest < a.row_bytes) dst[rest] = src[rest];
}

}  // namespace vk

using namespace vk;

// src, dst: `moves` row numbers on the host, each below `rows`; no row may be written twice, or read and written.
VK_API int vk_copy_rows(void* base, int layers, int rows, long long layer_stride, long long row_stride, long long row_bytes, const int32_t* src,
                        const int32_t* dst, int moves, cudaStream_t stream) {
    if (layers <= 0 || moves <= 0 || row_bytes <= 0) return VK_OK;
    if (rows <= 0 || layers > 65535 || row_stride < row_bytes || !src || !dst) return VK_BAD_SHAPE;
    for (int i = 0; i < moves; i++)
        if (src[i] < 0 || src[i] >= rows || dst[i] < 0 || dst[i] >= rows) return VK_BAD_SHAPE;
    const bool wide = ((uintptr_t)base | (unsigned long long)layer_stride | (unsigned long long)row_stride) % 16 == 0;
    const bool words = ((uintptr_t)base | (unsigned long long)layer_stride | (unsigned long long)row_stride) % 4 == 0;
    const long long piece = wide ? 16 : words ? 4 : 1, blocks = (row_bytes + piece * CR_THREADS * CR_PIECES - 1) / (piece * CR_THREADS * CR_PIECES);
    if (blocks > 0x7fffffffLL) return VK_TOO_LARGE;
    for (int done = 0; done < moves; done += CR_MOVES) {
        CrArgs a;
        a.base = (char*)base;
        a.layer_stride = layer_stride; a.row_stride = row_stride; a.row_bytes = row_bytes;
        const int n = moves - done < CR_MOVES ? moves - done : CR_MOVES;
        for (int i = 0; i < n; i++) { a.src[i] = src[done + i]; a.dst[i] = dst[done + i]; }
        const dim3 grid((unsigned)blocks, n, layers);
        const int status = wide    ? launch_dependent(copy_rows_kernel<uint4>, grid, dim3(CR_THREADS), 0, stream, a)
                           : words ? launch_dependent(copy_rows_kernel<uint32_t>, grid, dim3(CR_THREADS), 0, stream, a)
                                   : launch_dependent(copy_rows_kernel<unsigned char>, grid, dim3(CR_THREADS), 0, stream, a);
        if (status != VK_OK) return status;
    }
    return VK_OK;
}
