// Blocks copied inside pools of equal blocks: buffer[dst] = buffer[src] for a list of (src, dst) pairs and up to
// COPY_MAX_BUFFERS buffers that share the list - a request's last page when it is forked, its state slots in every
// stateful layer, the pages that a compaction moves.
//
// Bound by memory: every source is read and every destination written once (a source with several destinations comes
// from L2 after its first read).  A thread block owns PART bytes of one pair, all of a thread's loads go out before
// its first store, and the buffers' addresses travel with the launch, so that a fork of all layers is one launch.
// 600 pages of 458,752 bytes: 84.6 us a call (6.5 TB/s, the rate of a plain copy; the kernel ends after 80, its last writes still in
// L2); one state of 1 MB in each of 24 layers for eight forks: 38 us (226 MB, 6.0 TB/s; the kernel 36); one page: 3.6 us, a chain of
// list, load and store.
// Pairs outside the pool are skipped and reported.
#include "common.cuh"

namespace fsie {

constexpr int COPY_MAX_BUFFERS = 64;
constexpr int COPY_THREADS = 256;
constexpr int COPY_UNROLL = 4;
enum { ERR_BLOCK_RANGE = 4 };

struct CopyBuffers { unsigned char* base[COPY_MAX_BUFFERS]; };

// V: 16 bytes where every block starts on them, else 4, 2 or 1
template <typename V>
__global__ void __launch_bounds__(COPY_THREADS)
copy_blocks_kernel(const __grid_constant__ CopyBuffers buffers, long long block_bytes, int blocks,
                   const int* __restrict__ moves, int parts, int* __restrict__ error) {
    grid_dependency_wait();
    grid_dependents_go();
    const int move = blockIdx.x / parts, part = blockIdx.x - move * parts;
    const int src = moves[2 * move], dst = moves[2 * move + 1];
    if ((unsigned)src >= (unsigned)blocks || (unsigned)dst >= (unsigned)blocks) {
        if (threadIdx.x == 0) atomicExch(error, ERR_BLOCK_RANGE);
        return;
    }
    if (src == dst) return;
    unsigned char* base = buffers.base[blockIdx.y];
    const V* from = reinterpret_cast<const V*>(base + src * block_bytes);
    V* to = reinterpret_cast<V*>(base + dst * block_bytes);
    const long long count = block_bytes / (long long)sizeof(V);
    const long long first = (long long)part * (COPY_THREADS * COPY_UNROLL) + threadIdx.x;
    V held[COPY_UNROLL];
#pragma unroll
    for (int i = 0; i < COPY_UNROLL; ++i)
        if (first + i * COPY_THREADS < count) held[i] = from[first + i * COPY_THREADS];
#pragma unroll
    for (int i = 0; i < COPY_UNROLL; ++i)
        if (first + i * COPY_THREADS < count) to[first + i * COPY_THREADS] = held[i];
}

template <typename V>
static int launch_copy(const CopyBuffers& buffers, int count, long long block_bytes, int blocks, const int* moves, int pairs,
                       int* error, cudaStream_t stream) {
    const long long per = (long long)COPY_THREADS * COPY_UNROLL * sizeof(V);
    const long long parts = (block_bytes + per - 1) / per;
    if (parts * pairs > 0x7fffffffLL) return ERR_UNSUPPORTED;
    return launch_dependent(copy_blocks_kernel<V>, dim3((unsigned)(parts * pairs), count), dim3(COPY_THREADS), 0, stream,
                            buffers, block_bytes, blocks, moves, (int)parts, error);
}

}  // namespace fsie

using namespace fsie;

extern "C" {

int fsie_copy_max_buffers() { return COPY_MAX_BUFFERS; }

// bases: `count` addresses in host memory; moves [pairs, 2] on the device
int fsie_copy_blocks(const long long* bases, int count, long long block_bytes, int blocks, const int* moves, int pairs,
                     int* error, cudaStream_t stream) {
    if (count < 0 || count > COPY_MAX_BUFFERS || block_bytes < 0 || blocks < 0 || pairs < 0 || !error) return ERR_BAD_ARGUMENT;
    if (count == 0 || pairs == 0 || block_bytes == 0) return 0;
    if (!bases || !moves) return ERR_BAD_ARGUMENT;
    CopyBuffers buffers = {};
    unsigned long long all = (unsigned long long)block_bytes;       // low bits: the alignment that all blocks share
    for (int i = 0; i < count; ++i) {
        buffers.base[i] = reinterpret_cast<unsigned char*>(bases[i]);
        all |= (unsigned long long)bases[i];
    }
    if (all % 16 == 0) return launch_copy<uint4>(buffers, count, block_bytes, blocks, moves, pairs, error, stream);
    if (all % 4 == 0) return launch_copy<uint32_t>(buffers, count, block_bytes, blocks, moves, pairs, error, stream);
    if (all % 2 == 0) return launch_copy<uint16_t>(buffers, count, block_bytes, blocks, moves, pairs, error, stream);
    return launch_copy<uint8_t>(buffers, count, block_bytes, blocks, moves, pairs, error, stream);
}

}  // extern "C"
