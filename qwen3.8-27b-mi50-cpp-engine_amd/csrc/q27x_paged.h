// q27x_paged.h -- the paged cache as its kernels see it (k_paged.hip, k_paged_attn.hip, k_evict.hip).
#pragma once
#include <atomic>

#include "q27x_dev.h"
#include "q27x_int.h"

namespace q27x {

struct PagedArgs {
    void* k; void* v;               // pages [n_pages][page][nkv*hd]: int8 codes, or bf16 (G = 0)
    float* ks; float* vs;           // their scales [n_pages][page][nkv*hd/G]
    int G, nkv, hd;
    int n_pages, shift, stride;     // 1 << shift positions a page, pages `stride` positions apart
    const int32_t* table; int table_stride;
    const int32_t* lens; const int32_t* row_start;
    int n_seq;
};
// Lets kernel K have `bytes` of dynamic LDS on the current device: once per device.
template <auto K>
inline hipError_t allow_lds(int bytes) {
    static std::atomic<uint64_t> known{0};
    int dev = 0;
    if (hipError_t e = hipGetDevice(&dev)) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (known.load(std::memory_order_relaxed) & bit) return hipSuccess;
    if (hipError_t e = hipFuncSetAttribute((const void*)K, hipFuncAttributeMaxDynamicSharedMemorySize, bytes)) return e;
    known.fetch_or(bit, std::memory_order_relaxed);
    return hipSuccess;
}
// the caller's handle, checked (negative: its status)
int paged_args(const q27x_paged_kv_t* kv, const char* who, PagedArgs* out);

// Positions a sequence's table can name.
__device__ __forceinline__ long long paged_cap(const PagedArgs& a) { return (long long)a.table_stride << a.shift; }
// The pool position of key `key` of sequence b, or -1: outside the table, or on a page that the pool has not.
__device__ __forceinline__ int paged_slot(const PagedArgs& a, int b, int key) {
    if (key < 0 || (key >> a.shift) >= a.table_stride) return -1;
    const int p = a.table[(size_t)b * a.table_stride + (key >> a.shift)];
    if ((unsigned)p >= (unsigned)a.n_pages) return -1;
    return p * a.stride + (key & ((1 << a.shift) - 1));
}
// Rows of sequence b: the first and how many (negative counts read as none).
__device__ __forceinline__ void paged_rows(const PagedArgs& a, int b, int& first, int& n) {
    first = a.row_start ? a.row_start[b] : b;
    n = a.row_start ? a.row_start[b + 1] - first : 1;
    if (n < 0 || first < 0) n = 0;
}

}  // namespace q27x
