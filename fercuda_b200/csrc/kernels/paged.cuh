// The layout of a paged key-value cache, shared by its kernels: pages
// [pages][kv_heads][page_size][head_dim] of 16-bit elements, so that the rows
// of one key head in one page are one contiguous run.
#pragma once

#include "fercuda/b200/native.h"
#include "sm100_util.cuh"

#include <cstdint>
#include <initializer_list>

namespace fer::dev {

// Fetches a line into L2. Only a hint: it may come before a programmatic
// launch wait, as the value is read behind it.
__device__ __forceinline__ void prefetch_l2(const void* at) { asm volatile("prefetch.global.L2 [%0];" ::"l"(at)); }

struct Paged {
    void* k;
    void* v;
    const int32_t* table;
    const int32_t* lengths;
    int max_pages, pages, kv_heads, head_dim;
    int shift;   // log2 of the page size

    __host__ __device__ __forceinline__ int page_size() const { return 1 << shift; }
    __host__ __device__ __forceinline__ int max_slots() const { return max_pages << shift; }
    // A sequence's length, clamped to what its row of the table can hold.
    __device__ __forceinline__ int length(int b, bool* bad) const {
        const int n = lengths[b], most = max_slots();
        *bad = n < 0 || n > most;
        return n < 0 ? 0 : n > most ? most : n;
    }
    __device__ __forceinline__ bool is_page(int id) const {
        return static_cast<unsigned>(id) < static_cast<unsigned>(pages);
    }
    // Page id of slot s of sequence b, -1 where the table holds none.
    __device__ __forceinline__ int page(int b, int s) const {
        const int id = table[static_cast<size_t>(b) * max_pages + (s >> shift)];
        return is_page(id) ? id : -1;
    }
    // First element of the row of slot s, given its page.
    __device__ __forceinline__ size_t row(int id, int h, int s) const {
        return ((((static_cast<size_t>(id) * kv_heads + h) << shift) + (s & ((1 << shift) - 1)))) * head_dim;
    }
};

}  // namespace fer::dev

namespace fer::host {

// Devices for which a launcher keeps what it asked the runtime once.
constexpr int kMaxDevices = 64;

// Whether all of these arrays of 32-bit numbers start at a multiple of 4 bytes (null does).
inline bool words_aligned(std::initializer_list<const void*> arrays) {
    uintptr_t at = 0;
    for (const void* a : arrays) at |= reinterpret_cast<uintptr_t>(a);
    return at % 4 == 0;
}

// Checks the view's sizes and pointers.
inline cudaError_t paged_params(const fer_paged_view_t* c, fer::dev::Paged* p) {
    if (!c || !c->k || !c->v || !c->page_table || !c->lengths) return cudaErrorInvalidValue;
    if (c->batch <= 0 || c->max_pages <= 0 || c->pages <= 0 || c->kv_heads <= 0) return cudaErrorInvalidValue;
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16) return cudaErrorInvalidValue;
    if (!words_aligned({c->page_table, c->lengths})) return cudaErrorInvalidValue;
    if (c->dtype != 1 && c->dtype != 2) return cudaErrorNotSupported;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return cudaErrorNotSupported;
    int shift = 3;
    while (shift < 8 && (1 << shift) != c->page_size) ++shift;
    if ((1 << shift) != c->page_size) return cudaErrorNotSupported;
    // slots of a sequence, (sequence, head) pairs and pages are counted in 31 bits
    if ((static_cast<long long>(c->max_pages) << shift) > 0x7fffffffll - 65536 ||
        static_cast<long long>(c->batch) * c->kv_heads > 0x7fffffffll)
        return cudaErrorNotSupported;
    p->k = c->k;
    p->v = c->v;
    p->table = c->page_table;
    p->lengths = c->lengths;
    p->max_pages = c->max_pages;
    p->pages = c->pages;
    p->kv_heads = c->kv_heads;
    p->head_dim = c->head_dim;
    p->shift = shift;
    return cudaSuccess;
}

}  // namespace fer::host
