// Layout and argument checks of the 8-bit key-value cache (include/qw_kv8.h), shared by its kernels (k_kv8*.cu).
#pragma once
#include "../../include/qw_kv8.h"
#include "qw_kern.h"

#define KV8_PAGE 256
#define KV8_MAX_ROWS 1024  // rows of a call: a piece of a prompt
#define KV8_MAX_BLOCKS 0x7fffffffu  // of a list: the kernels count its entries in 32 bits, in steps of up to 512
#define KV8_TINY 7.8886090522101181e-31f  // 2^-100

// What a kernel needs of a cache: one layer of it.
struct Kv8Dev {
    uint8_t *codes;
    float *scales;
    uint8_t *bounds;
    const int32_t *ptab;
    unsigned *status;
    uint32_t pages, layers, kvh, hd, block, slots, max_pages, layer;
};

// Number of the first row of (page, layer, K or V, head); a row is hd codes and one scale.  Fits 31 bits by kv8_check_cache.
__host__ __device__ inline uint32_t kv8_row0(const Kv8Dev &c, uint32_t page, uint32_t kv, uint32_t head) {
    return (((page * c.layers + c.layer) * 2 + kv) * c.kvh + head) * KV8_PAGE;
}
__host__ __device__ inline size_t kv8_bound_bytes(uint32_t hd) { return 2 * hd + 16; }
// The record of a block's bounds.
__host__ __device__ inline size_t kv8_bound_at(const Kv8Dev &c, uint32_t page, uint32_t head, uint32_t block_in_page) {
    return ((((size_t)page * c.layers + c.layer) * c.kvh + head) * (KV8_PAGE / c.block) + block_in_page) * kv8_bound_bytes(c.hd);
}
// Whether the table has an entry for page number n of the slot, and whether an entry names a page of the pool.
__host__ __device__ inline bool kv8_entry_ok(const Kv8Dev &c, int64_t slot, int64_t n) { return slot >= 0 && slot < c.slots && n >= 0 && n < c.max_pages; }
__host__ __device__ inline bool kv8_page_ok(const Kv8Dev &c, int64_t page) { return page >= 0 && page < c.pages; }

#ifdef __CUDACC__
// The page id of a slot's page number n, or -1 for anything outside the cache.
__device__ __forceinline__ int kv8_page(const Kv8Dev &c, int slot, int n) {
    if (!kv8_entry_ok(c, slot, n)) return -1;
    const int p = __ldcg(c.ptab + (size_t)slot * c.max_pages + n);
    return kv8_page_ok(c, p) ? p : -1;
}
#endif

// Host side (k_kv8.cu).  The checks return nullptr or what is wrong; they touch no device.
const char *kv8_check_cache(const qw_kv8_cache *c);
const char *kv8_check_layer(const qw_kv8_cache *c, uint32_t nb, uint32_t layer, uint32_t dtype);
Kv8Dev kv8_dev(const qw_kv8_cache *c, uint32_t layer);
// whether these pointers (nullptr ones pass) start at a boundary of their type: n2 of 2 bytes, then n4 of 4
bool kv8_aligned(int n2, int n4, const void *const *ptrs);
// whether two different (row, head) of results would share bytes: a row's hd values are contiguous, strides in elements
bool kv8_overlap(uint32_t nb, uint32_t heads, uint32_t hd, int64_t row, int64_t head);
// whether k and v share bytes; where their strides differ, whether the memory between the first and the last of each does
bool kv8_share(const qw_kv8_rows *a, uint32_t heads, uint32_t hd);
int kv8_fail(int code, const char *where, const char *msg, char *err, size_t errlen);
// nullptr, or why work on these pointers (nullptr ones are passed over) cannot be enqueued on the current device
const char *kv8_check_device(const void *const *ptrs, int n);
int kv8_sm_count();
// Batches: the cache of binds 0-3 and 15 with its buffers' sizes checked, and a strided [nb][heads][hd] tensor of 2-byte values in a bind
bool kv8_from_binds(const QwLaunch &L, qw_kv8_cache *c, qw_kv8_sizes *s);
bool kv8_rows_fit(const QwLaunch &L, int bind, uint32_t nb, uint32_t heads, uint32_t hd, int64_t row, int64_t head);
