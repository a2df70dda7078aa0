// Copying whole pages of a paged store: what copy-on-write and compaction of
// shared pages do (no counterpart in the reference, whose sequences share
// nothing, draftkv/paged.py:76-176).
//
// dst page <- src page, byte for byte. Bound: memory, each byte read and
// written once. A thread moves one vector: 160 pages of 2 MB 112 us (6.0 TB/s;
// a contiguous copy of as many bytes 126), 24 of them 15, 6 of 720 KB 3.3.
// Four vectors per thread, a bound before each: 136, 25.7 and 17.4.
#include "dkv_common.h"
#include "pages.h"

namespace dkv {

// Grid x: pair * pieces + piece. V is the widest type that the pages' size and
// address allow. A pair with an id outside the store is skipped.
template <class V>
__global__ void __launch_bounds__(COPY_THREADS) paged_copy_kernel(char* __restrict__ store, int64_t n_pages, int64_t page_bytes,
                                                                  const int32_t* __restrict__ src,
                                                                  const int32_t* __restrict__ dst, int64_t first, int pieces) {
    const int64_t pair = first + blockIdx.x / pieces;
    const int64_t a = src[pair], b = dst[pair];
    if (a < 0 || a >= n_pages || b < 0 || b >= n_pages || a == b) return;
    const int64_t at = ((int64_t)(blockIdx.x % pieces) * COPY_THREADS + threadIdx.x) * sizeof(V);
    if (at >= page_bytes) return;
    *reinterpret_cast<V*>(store + b * page_bytes + at) = *reinterpret_cast<const V*>(store + a * page_bytes + at);
}

template <class V>
static int copy_pages(char* store, int64_t n_pages, int64_t page_bytes, const int32_t* src, const int32_t* dst,
                      int64_t n_pairs, hipStream_t st) {
    const int64_t span = (int64_t)COPY_THREADS * sizeof(V);
    const int64_t pieces = (page_bytes + span - 1) / span;
    DKV_REQUIRE(pieces <= COPY_BLOCKS, "dkv_paged_copy: pages too large");
    const int64_t most = COPY_BLOCKS / pieces;   // pairs per launch
    for (int64_t i = 0; i < n_pairs; i += most) {
        const int64_t n = n_pairs - i < most ? n_pairs - i : most;
        hipLaunchKernelGGL(paged_copy_kernel<V>, dim3((unsigned)(n * pieces)), dim3(COPY_THREADS), 0, st, store, n_pages, page_bytes,
                           src, dst, i, (int)pieces);
        if (const int e = check_launch("dkv_paged_copy")) return e;
    }
    return DKV_OK;
}

}  // namespace dkv

extern "C" int dkv_paged_copy(void* store, int64_t n_pages, int64_t page_bytes, const int32_t* src, const int32_t* dst,
                              int64_t n_pairs, dkv_stream_t stream) {
    DKV_REQUIRE(n_pages >= 0 && page_bytes >= 0 && n_pairs >= 0, "dkv_paged_copy: negative size");
    if (n_pairs == 0 || n_pages == 0 || page_bytes == 0) return DKV_OK;
    DKV_REQUIRE(store && src && dst, "dkv_paged_copy: NULL argument");
    hipStream_t st = dkv::as_stream(stream);
    char* p = static_cast<char*>(store);
    const int64_t at = reinterpret_cast<intptr_t>(store) | page_bytes;
    if (at % 16 == 0) return dkv::copy_pages<uint4>(p, n_pages, page_bytes, src, dst, n_pairs, st);
    if (at % 4 == 0) return dkv::copy_pages<uint32_t>(p, n_pages, page_bytes, src, dst, n_pairs, st);
    if (at % 2 == 0) return dkv::copy_pages<uint16_t>(p, n_pages, page_bytes, src, dst, n_pairs, st);
    return dkv::copy_pages<uint8_t>(p, n_pages, page_bytes, src, dst, n_pairs, st);
}
