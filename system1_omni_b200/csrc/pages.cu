// Copies of pages between places of a paged cache, over all the pools (one per layer and kind) that
// share its page numbers: what a fork, a copy on write and a compaction ask for.
#include <algorithm>
#include <exception>
#include <vector>

#include "common.cuh"
#include "cs1_ops.h"
#include "s1_executor.h"

namespace s1 {
namespace {

// The lists travel as kernel parameters (4 KB at most for a launch), so that nothing on the device has
// to hold them and a launch recorded into a graph keeps its own.
constexpr int MAX_POOLS = 64, MAX_PAIRS = 400;
struct PageCopies {
    uint4* pool[MAX_POOLS];
    int2 pair[MAX_PAIRS];  // from, to
};

constexpr int THREADS = 256, UNROLL = 4, PIECE = THREADS * UNROLL;  // 16-byte packs a block copies

// Bytes alone: every block moves 16 KB of one page of one pool, each thread's loads all before its stores.
// Measured at 337 pages of 64 KB in 32 pools: 215 us for 1.41 GB, 6.58 TB/s, the card's rate for a copy.
__global__ void __launch_bounds__(THREADS) pages_copy_kernel(const __grid_constant__ PageCopies c, size_t packs, int pieces) {
    grid_dep_trigger();
    grid_dep_sync();
    const int piece = blockIdx.x % pieces, pair = blockIdx.x / pieces;
    uint4* pool = c.pool[blockIdx.y];
    const uint4* src = pool + (size_t)c.pair[pair].x * packs;
    uint4* dst = pool + (size_t)c.pair[pair].y * packs;
    const size_t first = (size_t)piece * PIECE + threadIdx.x;
    uint4 x[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; u++)
        if (first + u * THREADS < packs) x[u] = src[first + u * THREADS];
#pragma unroll
    for (int u = 0; u < UNROLL; u++)
        if (first + u * THREADS < packs) dst[first + u * THREADS] = x[u];
}

// Every page number in range, no destination twice and none that is a source too: then the copies
// may run in any order. O(n); `seen` stays zero between calls.
int check_pairs(int n_pages, const int* src, const int* dst, int n) {
    static thread_local std::vector<unsigned char> seen;
    for (int i = 0; i < n; i++)
        if (src[i] < 0 || src[i] >= n_pages || dst[i] < 0 || dst[i] >= n_pages) return cudaErrorInvalidValue;
    try {
        if (seen.size() < (size_t)n_pages) seen.resize((size_t)n_pages);
    } catch (const std::exception&) {
        return cudaErrorMemoryAllocation;
    }
    bool ok = true;
    int marked = 0;
    for (; marked < n && ok; marked++) {
        ok = !seen[dst[marked]];
        seen[dst[marked]] = 1;
    }
    for (int i = 0; i < n && ok; i++) ok = !seen[src[i]];
    for (int i = 0; i < marked; i++) seen[dst[i]] = 0;
    return ok ? cudaSuccess : cudaErrorInvalidValue;
}

}  // namespace
}  // namespace s1

using namespace s1;

extern "C" int s1_pages_copy(void* const* pools, int n_pools, int n_pages, size_t page_bytes, const int* src, const int* dst,
                             int n, void* stream) {
    if (n_pools < 0 || n_pages < 0 || n < 0 || page_bytes == 0 || page_bytes % 16 != 0 || page_bytes > ((size_t)1 << 34))
        return cudaErrorInvalidValue;
    if (n == 0 || n_pools == 0) return cudaSuccess;
    if (!pools || !src || !dst) return cudaErrorInvalidValue;
    for (int p = 0; p < n_pools; p++)
        if (!pools[p] || !aligned16(pools[p])) return cudaErrorInvalidValue;
    const int rc = check_pairs(n_pages, src, dst, n);
    if (rc != 0) return rc;
    const size_t packs = page_bytes / 16;
    const int pieces = (int)((packs + PIECE - 1) / PIECE);
    const int at_once = std::max(1, std::min(MAX_PAIRS, 0x7fffffff / pieces));
    PageCopies c;
    for (int p0 = 0; p0 < n_pools; p0 += MAX_POOLS) {
        const int np = std::min(MAX_POOLS, n_pools - p0);
        for (int p = 0; p < np; p++) c.pool[p] = static_cast<uint4*>(pools[p0 + p]);
        for (int i0 = 0; i0 < n; i0 += at_once) {
            const int m = std::min(at_once, n - i0);
            for (int i = 0; i < m; i++) c.pair[i] = make_int2(src[i0 + i], dst[i0 + i]);
            const cudaError_t e =
                launch_dep(pages_copy_kernel, dim3((unsigned)m * pieces, np), THREADS, 0, as_stream(stream), c, packs, pieces);
            if (e != cudaSuccess) return e;
        }
    }
    return cudaGetLastError();
}
