// The 8-bit key-value cache: rows in (kv8_put) and out (kv8_get), and the bounds of its blocks.  include/qw_kv8.h has the formulas.
#include "common.cuh"
#include "kv8.h"
#include "kv8.cuh"

#include <cmath>
#include <cstdio>

using namespace qw;

namespace {
struct RowArgs {
    void *k, *v;
    const int32_t *slots, *pos;
    int64_t k_row, k_head, v_row, v_head;
    uint32_t nb;
};

// ------------------------------------------------------------------------------------------------ rows in
// One row of one head into row number `row` of the cache, by a warp; a lane holds hd / 32 consecutive values.
template <int HD, int FMT>
__device__ __forceinline__ void quantise_row(const Kv8Dev &c, size_t row, const float (&x)[HD / 32]) {
    constexpr int E = HD / 32;
    const uint32_t lane = threadIdx.x & 31;
    uint32_t m = 0;  // largest magnitude as bits: a NaN is above the infinities, those above all numbers
#pragma unroll
    for (int i = 0; i < E; i++) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    const float am = __uint_as_float(m), F = kv8_largest<FMT>();
    const bool nan = m >= 0x7f800000u, zero = !nan && am < KV8_TINY;
    const float inv = nan || zero ? 0.f : __fdiv_rn(F, am);
    uint32_t w[(E + 3) / 4] = {};
#pragma unroll
    for (int i = 0; i < E; i += 2) {
        const float y0 = nan ? 0.f : fminf(fmaxf(__fmul_rn(x[i], inv), -F), F), y1 = nan ? 0.f : fminf(fmaxf(__fmul_rn(x[i + 1], inv), -F), F);
        w[i / 4] |= kv8_encode2<FMT>(y0, y1) << (i % 4 * 8);
    }
    uint8_t *dst = c.codes + row * HD + lane * E;
    if (E == 8) *(uint2 *)dst = make_uint2(w[0], w[E == 8 ? 1 : 0]);
    else if (E == 4) *(uint32_t *)dst = w[0];
    else *(uint16_t *)dst = (uint16_t)w[0];
    if (lane == 0) c.scales[row] = nan ? __uint_as_float(0x7fffffffu) : zero ? 0.f : __fdiv_rn(am, F);
}

// A cache without bounds: a warp per (row, head, K or V).  Bound: the latency of slot, page, a look at all later rows for the same position, and values; per call in a
// captured graph 16 rows (hd 256, 2 kv heads) 1.9 us, 419 (hd 128, 8 kv heads) 4.7, 1024 (hd 256, 2 kv heads; 3.1 MB) 4.2.  grid nb x 256
template <int HD, int FMT, class T>
__global__ void __launch_bounds__(256) kv8_put_k(Kv8Dev c, RowArgs a) {
    constexpr int E = HD / 32;
    pdl_sync();
    const uint32_t r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slot = a.slots[r], pos = a.pos[r];
    if (slot < 0 || pos < 0) return;
    const int page = kv8_page(c, slot, pos / KV8_PAGE);
    if (page < 0) {
        if (tid == 0) set_status(c.status, ST_BAD_ARG | 0x21);
        return;
    }
    bool later = false;  // a later row for the same position
    for (uint32_t i = r + 1 + tid; i < a.nb; i += 256) later |= a.slots[i] == slot && a.pos[i] == pos;
    if (__syncthreads_or(later)) return;
    for (uint32_t t = warp; t < 2 * c.kvh; t += 8) {
        const uint32_t kv = t >= c.kvh, h = t - kv * c.kvh;
        float x[E];
        kv8_load<E>((const T *)(kv ? a.v : a.k) + (int64_t)r * (kv ? a.v_row : a.k_row) + (int64_t)h * (kv ? a.v_head : a.k_head) + lane * E, x);
        quantise_row<HD, FMT>(c, (size_t)kv8_row0(c, page, kv, h) + pos % KV8_PAGE, x);
    }
}

// A cache with bounds: of the rows for one block (16 to 256 tokens) the one with the newest position, its leader, stores all of them and then goes over the
// block's keys for the bounds.  The call's slots and positions are put into shared memory first; a row is asked after if neither of its neighbours in the call is of the same
// block and newer (most rows of a prompt are not), and leads if no other row is.  Keys (with the bounds) and values are different blocks of threads.
// Bound: the latency of one after the other: rows' numbers, their values, the block's keys from L2.  From a captured graph, per call: 16 rows (hd 256, 2 kv heads) 5.4 us, 419
// (hd 128, 8 kv heads) 7.1, 1024 (hd 256, 2 kv heads) 8.9; with the search in global memory and keys and values in the same block 5.3, 14.5 and 14.3; with that list of
// rows for calls of a row per block of threads too, 6.2 for the 16.  Work is shared out by blocks of the cache: 1024 rows with blocks of 256 and one kv head (hd 256) are five
// leaders for keys and for values each, and take 18.3 us; with blocks of 16 and eight kv heads (hd 128) 13.3.
// grid (blocks of threads that share the leaders, 2 kvh) x 512
template <int HD, int FMT, class T>
__global__ void __launch_bounds__(512, 2) kv8_put_blocks_k(Kv8Dev c, RowArgs a) {
    constexpr int E = HD / 32;
    constexpr uint32_t WC = HD / 4, NG = 512 / WC;  // columns of four channels, groups of tokens
    static_assert(KV8_MAX_ROWS == 1024, "two rows per thread");
    __shared__ float lo_s[NG][HD], hi_s[NG][HD];
    __shared__ int slot_s[KV8_MAX_ROWS], pos_s[KV8_MAX_ROWS];
    __shared__ uint16_t asked[KV8_MAX_ROWS];
    __shared__ int from[KV8_PAGE];  // of a token of the block: the last row for it, or -1
    __shared__ uint32_t wm[32];
    pdl_sync();
    const uint32_t kv = blockIdx.y >= c.kvh, h = blockIdx.y - kv * c.kvh, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wc = tid % WC, tg = tid / WC;
    const int bl = 31 - __clz(c.block);  // (a power of two)
    int sl[2], ps[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const uint32_t i = e * 512 + tid;
        sl[e] = i < a.nb ? a.slots[i] : -1;
        ps[e] = i < a.nb ? a.pos[i] : -1;
        slot_s[i] = sl[e], pos_s[i] = ps[e];
    }
    __syncthreads();
    auto newer = [&](uint32_t i, uint32_t r) {  // row i is of row r's block and newer (row r is in use)
        const int p = pos_s[i], q = pos_s[r];
        return slot_s[i] == slot_s[r] && p >= 0 && p >> bl == q >> bl && (p > q || (p == q && i > r));
    };
    uint32_t all = a.nb;
    const bool each = gridDim.x == a.nb;  // a row for every block of threads: no list of the rows to ask after
    if (!each) {
        uint32_t ask[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const uint32_t i = e * 512 + tid;
            ask[e] = __ballot_sync(0xffffffffu, sl[e] >= 0 && ps[e] >= 0 && !(i && newer(i - 1, i)) && !(i + 1 < a.nb && newer(i + 1, i)));
            if (lane == 0) wm[e * 16 + warp] = __popc(ask[e]);
        }
        __syncthreads();
        const uint32_t in_warps = wm[lane];
        all = __reduce_add_sync(0xffffffffu, in_warps);
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const uint32_t at = __reduce_add_sync(0xffffffffu, lane < e * 16 + warp ? in_warps : 0u);
            if (ask[e] >> lane & 1) asked[at + __popc(ask[e] & ((1u << lane) - 1))] = (uint16_t)(e * 512 + tid);
        }
    }
    for (uint32_t z = blockIdx.x; z < all; z += gridDim.x) {
        if (tid < c.block) from[tid] = -1;
        __syncthreads();
        const uint32_t r = each ? z : asked[z];
        const int slot = slot_s[r], pos = pos_s[r], blk = pos >> bl;
        if (slot < 0 || pos < 0) continue;
        const int page = kv8_page(c, slot, pos / KV8_PAGE);
        bool other = false;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const uint32_t i = e * 512 + tid;
            if (sl[e] != slot || ps[e] < 0 || ps[e] >> bl != blk) continue;
            other |= ps[e] > pos || (ps[e] == pos && i > r);
            atomicMax(&from[ps[e] & (c.block - 1)], (int)i);
        }
        if (__syncthreads_or(other)) continue;
        if (page < 0) {
            if (tid == 0 && blockIdx.y == 0) set_status(c.status, ST_BAD_ARG | 0x21);
            continue;
        }
        const uint32_t n = pos % c.block + 1;  // tokens of the block up to the newest
        const size_t row0 = (size_t)kv8_row0(c, page, kv, h) + blk * c.block % KV8_PAGE;
        const T *src = kv ? (const T *)a.v + (int64_t)h * a.v_head + lane * E : (const T *)a.k + (int64_t)h * a.k_head + lane * E;
        const int64_t stride = kv ? a.v_row : a.k_row;
        for (uint32_t p0 = warp; p0 < n; p0 += 64) {  // four rows at a time, all loads before the first store
            float x[4][E];
            int i[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                i[j] = p0 + 16 * j < n ? from[p0 + 16 * j] : -1;
                if (i[j] >= 0) kv8_load<E>(src + (int64_t)i[j] * stride, x[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i[j] >= 0) quantise_row<HD, FMT>(c, row0 + p0 + 16 * j, x[j]);
        }
        __syncthreads();
        if (kv) continue;
        // ---- bounds
        float lo[4], hi[4];
        bool nan = false;
#pragma unroll
        for (int j = 0; j < 4; j++) lo[j] = INFINITY, hi[j] = -INFINITY;
#pragma unroll 4
        for (uint32_t t = tg; t < n; t += NG) {
            const uint32_t w = __ldcg((const uint32_t *)(c.codes + (row0 + t) * HD) + wc);
            const float s = __ldcg(c.scales + row0 + t);
            float x[4];
            kv8_decode4<FMT>(w, x);
            const bool bad = s != s;
            nan |= bad;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float v = __fmul_rn(x[j], s);
                if (!bad) lo[j] = fminf(lo[j], v), hi[j] = fmaxf(hi[j], v);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) lo_s[tg][4 * wc + j] = lo[j], hi_s[tg][4 * wc + j] = hi[j];
        nan = __syncthreads_or(nan);
        float l = 0.f, u = 0.f;
        if (tid < HD) {
            l = lo_s[0][tid], u = hi_s[0][tid];
#pragma unroll
            for (uint32_t g = 1; g < NG; g++) l = fminf(l, lo_s[g][tid]), u = fmaxf(u, hi_s[g][tid]);
            if (l > u) l = u = 0.f;  // every row is NaN
        }
        const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fabsf(l), fabsf(u))));
        if (lane == 0) wm[warp] = m;
        __syncthreads();
        uint32_t b = 0;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) b = max(b, wm[i]);
        const float bm = __uint_as_float(b);
        const bool zero = bm < KV8_TINY;
        const float inv = zero ? 0.f : __fdiv_rn(127.f, bm);
        uint8_t *rec = c.bounds + kv8_bound_at(c, page, h, blk * c.block % KV8_PAGE / c.block);
        if (tid < HD) {
            rec[tid] = (uint8_t)(int8_t)fmaxf(-127.f, floorf(__fmul_rn(l, inv)));
            rec[HD + tid] = (uint8_t)(int8_t)fminf(127.f, ceilf(__fmul_rn(u, inv)));
        }
        if (tid < 4) ((float *)(rec + 2 * HD))[tid] = tid ? 0.f : nan ? INFINITY : zero ? 0.f : __fdiv_rn(bm, 127.f);
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------ rows out
// A warp per (row, head, K or V), as kv8_put_k.  grid nb x 256
template <int HD, int FMT, class T>
__global__ void __launch_bounds__(256) kv8_get_k(Kv8Dev c, RowArgs a) {
    constexpr int E = HD / 32;
    pdl_sync();
    const uint32_t r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slot = a.slots[r], pos = a.pos[r];
    if (slot < 0 || pos < 0) return;
    const int page = kv8_page(c, slot, pos / KV8_PAGE);
    if (page < 0 && tid == 0) set_status(c.status, ST_BAD_ARG | 0x22);
    for (uint32_t t = warp; t < 2 * c.kvh; t += 8) {
        const uint32_t kv = t >= c.kvh, h = t - kv * c.kvh;
        T *dst = (T *)(kv ? a.v : a.k) + (int64_t)r * (kv ? a.v_row : a.k_row) + (int64_t)h * (kv ? a.v_head : a.k_head) + lane * E;
        float x[8];
        if (page < 0) {
#pragma unroll
            for (int i = 0; i < E; i++) x[i] = __uint_as_float(0x7fffffffu);
        } else {
            const size_t row = (size_t)kv8_row0(c, page, kv, h) + pos % KV8_PAGE;
            const uint8_t *src = c.codes + row * HD + lane * E;
            uint32_t w[2] = {0, 0};
            if (E == 8) {
                const uint2 u = __ldcg((const uint2 *)src);
                w[0] = u.x, w[1] = u.y;
            } else if (E == 4) w[0] = __ldcg((const uint32_t *)src);
            else w[0] = __ldcg((const uint16_t *)src);
            const float s = __ldcg(c.scales + row);
#pragma unroll
            for (int i = 0; i < (E + 3) / 4; i++) {
                float q[4];
                kv8_decode4<FMT>(w[i], q);
#pragma unroll
                for (int j = 0; j < 4; j++) x[4 * i + j] = __fmul_rn(q[j], s);
            }
        }
        kv8_store<E>(dst, x);
    }
}


typedef void (*row_kernel)(Kv8Dev, RowArgs);
#define KV8_BY_DIM(NAME, FMT, T) (hd == 64 ? NAME<64, FMT, T> : hd == 128 ? NAME<128, FMT, T> : NAME<256, FMT, T>)
#define KV8_BY_ALL(NAME)                                                                            \
    (format == QW_KV8_E4M3 ? (dtype == QW_KV8_FP16 ? KV8_BY_DIM(NAME, QW_KV8_E4M3, __half) : KV8_BY_DIM(NAME, QW_KV8_E4M3, __nv_bfloat16)) \
                           : (dtype == QW_KV8_FP16 ? KV8_BY_DIM(NAME, QW_KV8_INT8, __half) : KV8_BY_DIM(NAME, QW_KV8_INT8, __nv_bfloat16)))
row_kernel put_kernel(uint32_t hd, uint32_t format, uint32_t dtype) { return KV8_BY_ALL(kv8_put_k); }
row_kernel get_kernel(uint32_t hd, uint32_t format, uint32_t dtype) { return KV8_BY_ALL(kv8_get_k); }
row_kernel put_blocks_kernel(uint32_t hd, uint32_t format, uint32_t dtype) { return KV8_BY_ALL(kv8_put_blocks_k); }

const char *check_rows(const qw_kv8_cache *c, const qw_kv8_rows *a) {
    if (!a) return "no arguments";
    if (const char *m = kv8_check_layer(c, a->nb, a->layer, a->dtype)) return m;
    if (!a->k || !a->v || !a->slots || !a->pos) return "null pointer argument";
    const void *ptrs[] = {a->k, a->v, a->slots, a->pos};
    if (!kv8_aligned(2, 2, ptrs)) return "a tensor does not start at a boundary of its type";
    return nullptr;
}
RowArgs row_args(const qw_kv8_rows *a) { return {a->k, a->v, a->slots, a->pos, a->k_row, a->k_head, a->v_row, a->v_head, a->nb}; }

cudaError_t enqueue_put(const qw_kv8_cache *c, const qw_kv8_rows *a, cudaStream_t st) {
    const Kv8Dev d = kv8_dev(c, a->layer);
    if (c->bounds) {  // about as many blocks of threads as are resident at once, or fewer
        const uint32_t most = c->kvh < 256 ? 256 / c->kvh : 1;
        return qw_launch(put_blocks_kernel(c->hd, c->format, a->dtype), dim3(a->nb < most ? a->nb : most, 2 * c->kvh), 512, 0, st, d, row_args(a));
    }
    return qw_launch(put_kernel(c->hd, c->format, a->dtype), a->nb, 256, 0, st, d, row_args(a));
}
cudaError_t enqueue_get(const qw_kv8_cache *c, const qw_kv8_rows *a, cudaStream_t st) {
    return qw_launch(get_kernel(c->hd, c->format, a->dtype), a->nb, 256, 0, st, kv8_dev(c, a->layer), row_args(a));
}

const char *check_out(const qw_kv8_cache *c, const qw_kv8_rows *a) {
    if (kv8_overlap(a->nb, c->kvh, c->hd, a->k_row, a->k_head) || kv8_overlap(a->nb, c->kvh, c->hd, a->v_row, a->v_head)) return "results that lie on one another";
    return nullptr;
}
typedef cudaError_t (*enqueue_rows)(const qw_kv8_cache *, const qw_kv8_rows *, cudaStream_t);
int rows_call(const char *where, enqueue_rows f, const qw_kv8_cache *c, const qw_kv8_rows *a, void *stream, char *err, size_t errlen) {
    const char *m = kv8_check_cache(c);
    if (!m) m = check_rows(c, a);
    if (!m && f == enqueue_get) m = check_out(c, a);
    if (m) return kv8_fail(-1, where, m, err, errlen);
    const void *ptrs[] = {c->codes, c->scales, c->bounds, c->page_table, c->status, a->k, a->v, a->slots, a->pos};
    if ((m = kv8_check_device(ptrs, 9))) return kv8_fail(-3, where, m, err, errlen);
    if (f == enqueue_get && kv8_share(a, c->kvh, c->hd)) return kv8_fail(-1, where, "k and v lie on one another", err, errlen);
    qw_pdl_current_family(where);
    const cudaError_t e = f(c, a, (cudaStream_t)stream);
    if (e != cudaSuccess) return cudaGetLastError(), kv8_fail(-3, where, cudaGetErrorString(e), err, errlen);
    if (err && errlen) err[0] = 0;
    return 0;
}

cudaError_t rows_batch(const QwLaunch &L, enqueue_rows f) {
    qw_kv8_cache c;
    qw_kv8_sizes s;
    QW_CHECK_ARG(kv8_from_binds(L, &c, &s) && L.has_bytes(8, 32));
    struct { int64_t s[4]; } st = L.bytes<decltype(st)>(8);
    const qw_kv8_rows a = {L.buf<void>(4), L.buf<void>(5), L.buf<int32_t>(6), L.buf<int32_t>(7), st.s[0], st.s[1], st.s[2], st.s[3], s.nb, s.layer, s.dtype, 0};
    QW_CHECK_ARG(!check_rows(&c, &a) && (f != enqueue_get || (!check_out(&c, &a) && !kv8_share(&a, s.kvh, s.hd))) && L.avail(6) >= (size_t)s.nb * 4 && L.avail(7) >= (size_t)s.nb * 4);
    QW_CHECK_ARG(kv8_rows_fit(L, 4, s.nb, s.kvh, s.hd, a.k_row, a.k_head) && kv8_rows_fit(L, 5, s.nb, s.kvh, s.hd, a.v_row, a.v_head));
    return f(&c, &a, L.stream);
}
cudaError_t launch_kv8_put(const QwLaunch &L) { return rows_batch(L, enqueue_put); }
cudaError_t launch_kv8_get(const QwLaunch &L) { return rows_batch(L, enqueue_get); }
}  // namespace
QW_FAMILY(kv8_put, launch_kv8_put, 512)
QW_FAMILY(kv8_get, launch_kv8_get, 256)

extern "C" int qw_kv8_put(const qw_kv8_cache *c, const qw_kv8_rows *a, void *stream, char *err, size_t errlen) {
    return rows_call("kv8_put", enqueue_put, c, a, stream, err, errlen);
}
extern "C" int qw_kv8_get(const qw_kv8_cache *c, const qw_kv8_rows *a, void *stream, char *err, size_t errlen) {
    return rows_call("kv8_get", enqueue_get, c, a, stream, err, errlen);
}

// ------------------------------------------------------------------------------------------------ host checks
static const char *check_sizes(const qw_kv8_cache *c) {
    if (!c) return "no cache";
    if (c->hd != 64 && c->hd != 128 && c->hd != 256) return "the head dimension is 64, 128 or 256";
    if (c->format != QW_KV8_E4M3 && c->format != QW_KV8_INT8) return "unknown format";
    if (c->block < 16 || c->block > KV8_PAGE || (c->block & (c->block - 1))) return "a block has 16, 32, 64, 128 or 256 tokens";
    if (c->pages < 1 || c->layers < 1 || c->kvh < 1 || c->slots < 1 || c->max_pages < 1) return "a cache has at least one page, layer, kv head, slot and page per slot";
    if (c->kvh > 32767) return "too many kv heads";
    if ((double)c->pages * c->layers * 2 * c->kvh * KV8_PAGE > 2147483647.0) return "more than 2^31 - 1 rows";
    if (c->max_pages > 0x7fffffffu / KV8_PAGE || c->slots > 0x7fffffffu) return "a slot has at most 2^31 - 1 tokens";
    return nullptr;
}
const char *kv8_check_cache(const qw_kv8_cache *c) {
    if (const char *m = check_sizes(c)) return m;
    if (!c->codes || !c->scales || !c->page_table) return "null pointer in the cache";
    if (((uintptr_t)c->codes | (uintptr_t)c->scales | (uintptr_t)c->bounds) & 15) return "codes, scales and bounds start at 16-byte boundaries";
    if (((uintptr_t)c->page_table | (uintptr_t)c->status) & 3) return "page table and status start at 4-byte boundaries";
    return nullptr;
}
const char *kv8_check_layer(const qw_kv8_cache *c, uint32_t nb, uint32_t layer, uint32_t dtype) {
    if (nb < 1 || nb > KV8_MAX_ROWS) return "a call has 1 to 1024 rows";
    if (layer >= c->layers) return "no such layer";
    if (dtype != QW_KV8_FP16 && dtype != QW_KV8_BF16) return "unknown type of rows";
    return nullptr;
}
Kv8Dev kv8_dev(const qw_kv8_cache *c, uint32_t layer) {
    return {c->codes, c->scales, c->bounds, c->page_table, c->status, c->pages, c->layers, c->kvh, c->hd, c->block, c->slots, c->max_pages, layer};
}
bool kv8_aligned(int n2, int n4, const void *const *ptrs) {
    for (int i = 0; i < n2 + n4; i++)
        if ((uintptr_t)ptrs[i] & (i < n2 ? 1 : 3)) return false;
    return true;
}
static int64_t floor_div(int64_t x, int64_t y) { return x / y - (x % y && (x < 0)); }  // y > 0
// Whether |d + i s1 + j s2| < hd for some |i| < n1 and |j| < n2; with `self` for others than i = j = 0.
static bool meet(int64_t d, uint32_t n1, int64_t s1, uint32_t n2, int64_t s2, int64_t hd, bool self) {
    const int64_t most = (int64_t)1 << 44;  // (no memory is that large: nothing below overflows)
    auto size = [&](uint32_t n, int64_t s) { return n <= 1 ? 0 : s < -most || s > most ? most : s < 0 ? -s : s; };  // i and j take both signs
    s1 = size(n1, s1), s2 = size(n2, s2);
    if (s1 < s2) {
        const int64_t s = s1;
        const uint32_t n = n1;
        s1 = s2, s2 = s, n1 = n2, n2 = n;
    }
    if (self && n2 > 1 && s2 == 0) return true;
    int64_t from = -(int64_t)(n1 - 1), to = n1 - 1;  // of i, as far as the shorter stride can bridge the rest: a few where rows are apart
    const int64_t reach = (n2 - 1) * s2 + hd - 1;
    if (s1 > 0) {
        const int64_t lo = floor_div(-reach - d, s1), hi = floor_div(reach - d, s1);
        from = lo > from ? lo : from, to = hi < to ? hi : to;
    }
    for (int64_t i = from; i <= to; i++) {
        const int64_t x = d + i * s1, j0 = s2 > 0 ? floor_div(-x, s2) : 0, last = n2 - 1;
        for (int64_t j = j0; j <= j0 + 1; j++) {
            const int64_t k = j < -last ? -last : j > last ? last : j, y = x + k * s2;
            if (y < hd && y > -hd && !(self && i == 0 && k == 0)) return true;
        }
    }
    return false;
}
bool kv8_overlap(uint32_t nb, uint32_t heads, uint32_t hd, int64_t row, int64_t head) { return meet(0, nb, row, heads, head, hd, true); }
bool kv8_share(const qw_kv8_rows *a, uint32_t heads, uint32_t hd) {
    const double d = ((double)(intptr_t)a->k - (double)(intptr_t)a->v) / 2;
    if (d > 1e17 || d < -1e17) return false;  // (addresses have 57 bits at most)
    if ((a->nb <= 1 || a->k_row == a->v_row) && (heads <= 1 || a->k_head == a->v_head))
        return meet(((intptr_t)a->k - (intptr_t)a->v) / 2, a->nb, a->k_row, heads, a->k_head, hd, false);
    auto ends = [&](double row, double head, double &lo, double &hi) {
        row *= a->nb - 1, head *= heads - 1;
        lo = fmin(row, 0) + fmin(head, 0), hi = fmax(row, 0) + fmax(head, 0) + hd;
    };
    double klo, khi, vlo, vhi;
    ends((double)a->k_row, (double)a->k_head, klo, khi);
    ends((double)a->v_row, (double)a->v_head, vlo, vhi);
    return d + klo < vhi && vlo < d + khi;
}
int kv8_fail(int code, const char *where, const char *msg, char *err, size_t errlen) {
    if (err && errlen) snprintf(err, errlen, "qw_%s: %s", where, msg);
    return code;
}
static const char *check_device(const void *const *ptrs, int n) {  // (a launch on another device's stream is refused by CUDA itself)
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) return cudaGetLastError(), "no CUDA device";
    for (int i = 0; i < n; i++) {
        if (!ptrs[i]) continue;
        cudaPointerAttributes at;
        if (cudaPointerGetAttributes(&at, ptrs[i]) != cudaSuccess) return cudaGetLastError(), "cannot look up a buffer";
        if (at.type == cudaMemoryTypeUnregistered) return "a buffer is not device memory";
        if (at.type == cudaMemoryTypeDevice && at.device != dev) return "a buffer is another device's";
    }
    return nullptr;
}
const char *kv8_check_device(const void *const *ptrs, int n) {
    // the look-ups change nothing, but in the default mode they would end a capture that this thread has open
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return cudaGetLastError(), "no CUDA device";
    const char *m = check_device(ptrs, n);
    cudaThreadExchangeStreamCaptureMode(&mode);
    return m;
}
int kv8_sm_count() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) return 1;
    return n;
}
static bool bytes_of(const qw_kv8_cache *c, size_t out[3]) {
    if (check_sizes(c)) return false;
    const size_t rows = (size_t)c->pages * c->layers * 2 * c->kvh * KV8_PAGE;
    out[0] = rows * c->hd;
    out[1] = rows * 4;
    out[2] = rows / 2 / c->block * kv8_bound_bytes(c->hd);
    return true;
}
extern "C" int qw_kv8_bytes(const qw_kv8_cache *c, size_t out[3]) { return c && out && bytes_of(c, out) ? 0 : -1; }
extern "C" int64_t qw_kv8_row_index(const qw_kv8_cache *c, int64_t slot, int64_t pos, int64_t page, uint32_t layer, uint32_t kv, uint32_t head) {
    if (check_sizes(c) || layer >= c->layers || kv > 1 || head >= c->kvh || pos < 0) return -1;
    const Kv8Dev d = kv8_dev(c, layer);
    if (!kv8_entry_ok(d, slot, pos / KV8_PAGE) || !kv8_page_ok(d, page)) return -1;
    return (int64_t)kv8_row0(d, (uint32_t)page, kv, head) + pos % KV8_PAGE;
}
bool kv8_from_binds(const QwLaunch &L, qw_kv8_cache *c, qw_kv8_sizes *s) {
    if (!L.has_bytes(15, sizeof *s)) return false;
    *s = L.bytes<qw_kv8_sizes>(15);
    *c = {L.buf<uint8_t>(0), L.buf<float>(1), L.buf<uint8_t>(2), L.buf<int32_t>(3), L.status, s->pages, s->layers, s->kvh, s->hd, s->format, s->block, s->slots, s->max_pages};
    size_t n[3];
    return !kv8_check_cache(c) && bytes_of(c, n) && L.avail(0) >= n[0] && L.avail(1) >= n[1] && (!c->bounds || L.avail(2) >= n[2]) &&
           L.avail(3) >= (size_t)s->slots * s->max_pages * 4;
}
bool kv8_rows_fit(const QwLaunch &L, int bind, uint32_t nb, uint32_t heads, uint32_t hd, int64_t row, int64_t head) {
    if (row < 0 || head < 0) return false;
    const double last = (double)(nb - 1) * (double)row + (double)(heads - 1) * (double)head + hd;
    return last * 2 <= (double)L.avail(bind);
}
