// Pages copied inside a pool: page src -> page dst in every cache entry of a group (what a request forked from another needs of the
// page that both would go on writing).
//
// The pairs travel with the launch, as kernel parameters: no copy to the device precedes it.  A block copies one slice of one page
// of one entry; every thread asks for its four vectors before it stores the first, so a block has 16 KB in flight and the kernel runs
// at the rate of device memory: 96 pages of 32 KB in 16 entries (100 MB read and written) take 17.1 us, 5.9 TB/s; three pages of 20 KB
// 1.7 us, a launch's latency.
//
// This kernel does not let the one behind it start early (no pdl_trigger): attention kernels fetch keys of earlier steps ahead of
// their wait for the kernel before them, which must not reach past a copy of such keys.
#include "common.cuh"

#include <algorithm>
#include <cstdlib>

namespace {

constexpr int kMaxPairs = 256;                 // pairs a launch carries (2 KB of parameters)
constexpr int kCopyThreads = 256, kCopyPer = 4;

struct CopyPairs { int2 pair[kMaxPairs]; };

// V: the widest type that divides a page's bytes and the pool's address.
template <typename V>
__global__ void __launch_bounds__(kCopyThreads)
copy_pages_kernel(uint8_t* pool, size_t entry_bytes, size_t page_bytes, const CopyPairs p) {
    pdl_wait();
    const int2 at = p.pair[blockIdx.y];
    uint8_t* entry = pool + blockIdx.z * entry_bytes;
    const V* src = reinterpret_cast<const V*>(entry + (size_t)at.x * page_bytes);
    V* dst = reinterpret_cast<V*>(entry + (size_t)at.y * page_bytes);
    const size_t n = page_bytes / sizeof(V), first = (size_t)blockIdx.x * (kCopyThreads * kCopyPer) + threadIdx.x;
    V v[kCopyPer];
#pragma unroll
    for (int i = 0; i < kCopyPer; ++i)
        if (first + i * kCopyThreads < n) v[i] = src[first + i * kCopyThreads];
#pragma unroll
    for (int i = 0; i < kCopyPer; ++i)
        if (first + i * kCopyThreads < n) dst[first + i * kCopyThreads] = v[i];
}

}  // namespace

// pool: entries of `pages` pages of `page_bytes` bytes each, contiguous.  pairs (host memory): n_pairs x {source page, destination
// page}; no destination may be a source or a destination of another pair (they are copied at the same time).
LLM_API int llm_copy_pages(void* pool, int entries, long long pages, long long page_bytes, const int* pairs, int n_pairs, cudaStream_t stream) {
    if (n_pairs == 0 || entries == 0 || page_bytes == 0) return 0;
    if (entries < 0 || entries > 65535) LLM_FAIL(-1, "copy_pages: %d entries (at most 65535)", entries);
    for (int i = 0; i < 2 * n_pairs; ++i)
        if (pairs[i] < 0 || pairs[i] >= pages) LLM_FAIL(-1, "copy_pages: page %d is not one of the pool's %lld pages", pairs[i], pages);
    // no destination twice, none that is a source: pages by what they are, side by side once sorted (2 page: source, + 1: destination)
    long long few[512];
    long long* seen = 2 * n_pairs <= 512 ? few : static_cast<long long*>(malloc(2 * (size_t)n_pairs * sizeof(long long)));
    if (!seen) LLM_FAIL(-2, "copy_pages: no memory for %d pairs", n_pairs);
    for (int i = 0; i < 2 * n_pairs; ++i) seen[i] = 2ll * pairs[i] + (i & 1);
    std::sort(seen, seen + 2 * n_pairs);
    int clash = -1, twice = 0;
    for (int i = 1; i < 2 * n_pairs && clash < 0; ++i)
        if (seen[i] / 2 == seen[i - 1] / 2 && (seen[i] & 1)) { clash = (int)(seen[i] / 2); twice = (int)(seen[i - 1] & 1); }
    if (seen != few) free(seen);
    if (clash >= 0)
        LLM_FAIL(-1, twice ? "copy_pages: page %d is the destination of two copies" : "copy_pages: page %d is the source of one copy and the destination of another", clash);
    const unsigned long long low = (unsigned long long)(uintptr_t)pool | (unsigned long long)page_bytes;
    const int width = low % 16 == 0 ? 16 : low % 4 == 0 ? 4 : 1;
    const long long slices = (page_bytes / width + kCopyThreads * kCopyPer - 1) / (kCopyThreads * kCopyPer);
    if (slices > 0x7fffffffll) LLM_FAIL(-1, "copy_pages: pages of %lld bytes are too large", page_bytes);
    for (int from = 0; from < n_pairs; from += kMaxPairs) {
        CopyPairs p;
        const int n = n_pairs - from < kMaxPairs ? n_pairs - from : kMaxPairs;
        for (int i = 0; i < n; ++i) p.pair[i] = make_int2(pairs[2 * (from + i)], pairs[2 * (from + i) + 1]);
        const dim3 grid((unsigned)slices, n, entries);
        const size_t entry_bytes = (size_t)pages * (size_t)page_bytes;
        if (width == 16) llm_launch(copy_pages_kernel<uint4>, grid, kCopyThreads, 0, stream, (uint8_t*)pool, entry_bytes, (size_t)page_bytes, p);
        else if (width == 4) llm_launch(copy_pages_kernel<uint32_t>, grid, kCopyThreads, 0, stream, (uint8_t*)pool, entry_bytes, (size_t)page_bytes, p);
        else llm_launch(copy_pages_kernel<uint8_t>, grid, kCopyThreads, 0, stream, (uint8_t*)pool, entry_bytes, (size_t)page_bytes, p);
        LLM_CHECK_LAUNCH("copy_pages");
    }
    return 0;
}

LLM_TRACE_EXPORT(copy_pages)
