// The blocks of a row's context that are worth attending to: a score for every block from the bounds of its keys (kv8_score_k), then the best ones
// (kv8_best_k).  include/qw_kv8.h has the formulas.
#include "kv8.cuh"

using namespace qw;

namespace {
struct PickArgs {
    const void *q;
    const int32_t *lens, *slots;
    int32_t *out;
    uint32_t *keys;  // [nb][kvh][stride]
    int64_t q_row, q_head;
    uint32_t nb, qh, G, max_len, count, first, last, stride;
};
constexpr uint32_t RECORDS = 128;  // of a block of threads

__device__ __forceinline__ uint32_t row_blocks(const Kv8Dev &c, const PickArgs &a, int slot, int len) {
    return slot < 0 || len <= 0 ? 0 : (min((uint32_t)len, a.max_len) + c.block - 1) / c.block;
}
// Larger numbers have larger keys; no number has key 0 or 0xffffffff.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 becomes +0: the two are equal
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// Scores as keys: the products of 16 records and 8 heads at a time on the tensor cores (mma m16n8k32 on int8: sums of whole numbers, exact).  A record is
// [lower | upper bounds], a head's row [negative parts of q8 | positive parts].  Which byte is which k is free as long as both sides agree, so a lane takes 16
// bytes of a record with one load, all of them before the first product.  Bound: the latency of page id and record, then the bytes of the records.
// (dp4a with a sum across the warp for every head: 27 us for 100,000 records one after the other, 15 with eight in flight.)
// grid (ceil(most blocks / 128), kvh, nb) x 256
template <int HD, class T>
__global__ void __launch_bounds__(256) kv8_score_k(Kv8Dev c, PickArgs a) {
    constexpr int CC = 2 * HD / 64, STRIDE = 2 * HD + 64;  // a head's bytes: 64 more, so that neighbouring heads are in other banks
    __shared__ __align__(16) int8_t q8[16 * STRIDE];
    __shared__ float sqs[16];
    pdl_sync();
    const uint32_t h = blockIdx.y, r = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int len = a.lens[r], slot = a.slots[r];
    const uint32_t n = row_blocks(c, a, slot, len), per = KV8_PAGE / c.block, b0 = blockIdx.x * RECORDS + warp * 16;
    if (blockIdx.x * RECORDS >= n) return;
    int page[2];
#pragma unroll
    for (int e = 0; e < 2; e++) page[e] = b0 + g + 8 * e < n ? kv8_page(c, slot, (int)((b0 + g + 8 * e) / per)) : -1;
    for (uint32_t k = warp; k < 16; k += 8) {  // (heads beyond the last are zeros)
        float x[HD / 32];
#pragma unroll
        for (int i = 0; i < HD / 32; i++) x[i] = 0.f;
        if (k < a.G) kv8_load<HD / 32>((const T *)a.q + (int64_t)r * a.q_row + (int64_t)(h * a.G + k) * a.q_head + lane * (HD / 32), x);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
        m = __reduce_max_sync(0xffffffffu, m);
        const float am = __uint_as_float(m);
        const bool none = m >= 0x7f800000u || am < KV8_TINY;
        const float inv = none ? 0.f : __fdiv_rn(127.f, am);
#pragma unroll
        for (int i = 0; i < HD / 32; i++) {
            const int v = none ? 0 : __float2int_rn(__fmul_rn(x[i], inv));
            q8[k * STRIDE + lane * (HD / 32) + i] = (int8_t)min(v, 0);
            q8[k * STRIDE + HD + lane * (HD / 32) + i] = (int8_t)max(v, 0);
        }
        if (lane == 0) sqs[k] = none ? 0.f : __fdiv_rn(am, 127.f);
    }
    uint4 w[2][CC];
    float sb[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const uint8_t *rec = c.bounds + kv8_bound_at(c, page[e] < 0 ? 0 : page[e], h, (b0 + g + 8 * e) % per);
        sb[e] = page[e] < 0 ? 0.f : __ldcg((const float *)(rec + 2 * HD));
#pragma unroll
        for (int cc = 0; cc < CC; cc++) w[e][cc] = page[e] < 0 ? make_uint4(0, 0, 0, 0) : __ldcg((const uint4 *)(rec + 64 * cc + 16 * t));
    }
    __syncthreads();
    float best[2] = {-INFINITY, -INFINITY};
    for (uint32_t k0 = 0; k0 < a.G; k0 += 8) {
        int d[4] = {0, 0, 0, 0};
#pragma unroll
        for (int cc = 0; cc < CC; cc++) {
            const uint4 q = *(const uint4 *)(q8 + (k0 + g) * STRIDE + 64 * cc + 16 * t);
            mma_s8(d, w[0][cc].x, w[1][cc].x, w[0][cc].y, w[1][cc].y, q.x, q.y);
            mma_s8(d, w[0][cc].z, w[1][cc].z, w[0][cc].w, w[1][cc].w, q.z, q.w);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {  // record g + 8 (j / 2), head 2 t + j % 2
            const uint32_t k = k0 + 2 * t + (j & 1);
            if (k < a.G) best[j >> 1] = fmaxf(best[j >> 1], d[j] ? __fmul_rn(__fmul_rn(sqs[k], sb[j >> 1]), (float)d[j]) : 0.f);
        }
    }
#pragma unroll
    for (int e = 0; e < 2; e++) {
        best[e] = fmaxf(best[e], __shfl_xor_sync(0xffffffffu, best[e], 1));
        best[e] = fmaxf(best[e], __shfl_xor_sync(0xffffffffu, best[e], 2));
        const uint32_t b = b0 + g + 8 * e;
        if (t || b >= n) continue;
        uint32_t key = key_of(sb[e] == INFINITY ? INFINITY : best[e]);
        if (page[e] < 0) {
            key = 0;
            set_status(c.status, ST_BAD_ARG | 0x25);
        } else if (b < a.first || b + a.last >= n) key = 0xffffffffu;
        a.keys[((size_t)r * c.kvh + h) * a.stride + b] = key;
    }
}

// Block-wide exclusive prefix sum (512 threads); two barriers
__device__ __forceinline__ uint32_t scan_512(uint32_t v, uint32_t *ws, uint32_t &total) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= (uint32_t)o) s += u;
    }
    if (lane == 31) ws[warp] = s;
    __syncthreads();
    uint32_t e = s - v, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < 16; w++) {
        const uint32_t x = ws[w];
        if (w < warp) e += x;
        all += x;
    }
    total = all;
    __syncthreads();
    return e;
}

// The `count` largest keys in ascending order of their blocks; of the keys that equal the smallest of them the lowest blocks are taken.  Histograms of 2048
// equal parts of the range in play, which shrinks to the part that holds the threshold, until the threshold is found or the whole part is taken; usually two.
// Blocks that are always taken (key 0xffffffff) and such without a page (0) are not in it.  Up to 4096 keys stay in shared memory.  In the end a thread owns
// a run of consecutive blocks, so prefix sums give the places.  Bound: its barriers.  (Radix passes over the keys' bits, 1024 threads: 8 us for 750 blocks;
// two bits at a time with counters: 12.)  grid (kvh, nb) x 512
constexpr uint32_t BEST_KEYS = 4096;
__global__ void __launch_bounds__(512) kv8_best_k(Kv8Dev c, PickArgs a) {
    __shared__ __align__(16) uint32_t hist[2048];  // (gone over in fours)
    __shared__ uint32_t ws[16], red[16][4], found[3], kept[BEST_KEYS];
    pdl_sync();
    const uint32_t h = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int len = a.lens[r], slot = a.slots[r];
    if (slot < 0) return;
    const bool bad = len > 0 && (uint32_t)len > a.max_len;
    if (tid == 0 && bad) set_status(c.status, ST_BAD_ARG | 0x26);
    const uint32_t n = bad ? 0 : row_blocks(c, a, slot, len);
    const uint32_t *keys = a.keys + ((size_t)r * c.kvh + h) * a.stride;
    int32_t *out = a.out + ((size_t)r * c.kvh + h) * a.count;
    uint32_t lo = 0xffffffffu, hi = 0, fixed = 0, in = 0;  // smallest, largest of the keys in play; always taken ones, ones in play
    for (uint32_t i = tid; i < n; i += 512) {
        const uint32_t k = __ldcg(keys + i);
        if (i < BEST_KEYS) kept[i] = k;
        if (k == 0xffffffffu) fixed++;
        else if (k) lo = min(lo, k), hi = max(hi, k), in++;
    }
    if (n <= BEST_KEYS) keys = kept;
    lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi), fixed = __reduce_add_sync(0xffffffffu, fixed), in = __reduce_add_sync(0xffffffffu, in);
    if (lane == 0) red[warp][0] = lo, red[warp][1] = hi, red[warp][2] = fixed, red[warp][3] = in;
    for (uint32_t b = tid; b < 2048; b += 512) hist[b] = 0;
    __syncthreads();
    lo = 0xffffffffu, hi = fixed = in = 0;
#pragma unroll
    for (int w = 0; w < 16; w++) lo = min(lo, red[w][0]), hi = max(hi, red[w][1]), fixed += red[w][2], in += red[w][3];
    uint32_t T = 0, rem = 0;  // keys above T are taken, and `rem` of those equal to it
    const uint32_t want = a.count - min(a.count, fixed);
    if (want == 0) T = 0xfffffffeu;
    else if (in > want) {
        rem = want;
        for (;;) {
            const uint32_t bits = 32 - __clz(hi - lo), sh = bits > 11 ? bits - 11 : 0;
            for (uint32_t i = tid; i < n; i += 512) {
                const uint32_t k = keys[i];
                if (k >= lo && k <= hi) atomicAdd(&hist[(k - lo) >> sh], 1u);
            }
            __syncthreads();
            const uint32_t b = 2044 - 4 * tid;  // this thread's four parts
            const uint4 v = *(const uint4 *)&hist[b];
            *(uint4 *)&hist[b] = make_uint4(0, 0, 0, 0);
            uint32_t tot;
            const uint32_t e = scan_512(v.x + v.y + v.z + v.w, ws, tot);  // keys in all parts above these
            const uint32_t cnt[4] = {v.w, v.z, v.y, v.x};
            uint32_t at = e;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (at < rem && at + cnt[i] >= rem) found[0] = b + 3 - i, found[1] = rem - at, found[2] = cnt[i];
                at += cnt[i];
            }
            __syncthreads();
            lo += found[0] << sh;
            rem = found[1];
            if (sh == 0) {
                T = lo;
                break;
            }
            if (found[2] == rem) {  // all of them
                T = lo - 1;
                rem = 0;
                break;
            }
            hi = min(hi, lo + ((1u << sh) - 1));
        }
    }
    const uint32_t run = (n + 511) / 512, i0 = min(n, tid * run), i1 = min(n, i0 + run);
    uint32_t above = 0, equal = 0, tot_above, tot_equal = 0;
    for (uint32_t i = i0; i < i1; i++) {
        const uint32_t k = keys[i];
        above += k > T;
        equal += rem && k == T;
    }
    const uint32_t ea = scan_512(above, ws, tot_above), ee = rem ? scan_512(equal, ws, tot_equal) : 0;
    uint32_t at = ea + min(ee, rem), eq = ee;
    for (uint32_t i = i0; i < i1; i++) {
        const uint32_t k = keys[i];
        if (k > T || (rem && k == T && eq++ < rem)) out[at++] = (int32_t)i;
    }
    for (uint32_t i = tot_above + min(tot_equal, rem) + tid; i < a.count; i += 512) out[i] = -1;
}

typedef void (*pick_kernel)(Kv8Dev, PickArgs);
pick_kernel score_of(uint32_t hd, uint32_t dtype) {
    if (dtype == QW_KV8_FP16) return hd == 64 ? kv8_score_k<64, __half> : hd == 128 ? kv8_score_k<128, __half> : kv8_score_k<256, __half>;
    return hd == 64 ? kv8_score_k<64, __nv_bfloat16> : hd == 128 ? kv8_score_k<128, __nv_bfloat16> : kv8_score_k<256, __nv_bfloat16>;
}
uint32_t most_blocks(const qw_kv8_cache *c, uint32_t max_len) { return (uint32_t)(((uint64_t)max_len + c->block - 1) / c->block); }
size_t work_of(const qw_kv8_cache *c, uint32_t nb, uint32_t max_len) { return (size_t)nb * c->kvh * most_blocks(c, max_len) * 4; }
int check_pick(const qw_kv8_cache *c, const qw_kv8_pick_args *a, const char **m) {
    if (!a) return *m = "no arguments", -1;
    if (!c->bounds) return *m = "the cache has no bounds", -1;
    if ((*m = kv8_check_layer(c, a->nb, a->layer, a->dtype))) return -1;
    if (a->qh < c->kvh || a->qh % c->kvh || a->qh / c->kvh > 16) return *m = "1 to 16 query heads share a kv head", -1;
    if (a->max_len < 1 || (uint64_t)a->max_len > (uint64_t)c->max_pages * KV8_PAGE) return *m = "max_len is 1 to 256 max_pages", -1;
    if (a->nblocks < 1 || (uint64_t)a->first + a->last > a->nblocks) return *m = "at least one block is chosen, and first + last of them at most", -1;
    if (a->nblocks > KV8_MAX_BLOCKS) return *m = "a list holds at most 2^31 - 1 blocks", -1;
    if (!a->q || !a->lens || !a->slots || !a->blocks || !a->work) return *m = "null pointer argument", -1;
    const void *ptrs[] = {a->q, a->lens, a->slots, a->blocks};
    if (!kv8_aligned(1, 3, ptrs)) return *m = "a tensor does not start at a boundary of its type", -1;
    if ((uintptr_t)a->work & 15) return *m = "the workspace starts at a 16-byte boundary", -1;
    if (a->work_bytes < work_of(c, a->nb, a->max_len)) return *m = "the workspace is too small", -2;
    return 0;
}
cudaError_t enqueue_pick(const qw_kv8_cache *c, const qw_kv8_pick_args *a, cudaStream_t st) {
    const uint32_t most = most_blocks(c, a->max_len);
    const PickArgs k = {a->q, a->lens, a->slots, a->blocks, (uint32_t *)a->work, a->q_row, a->q_head, a->nb, a->qh, a->qh / c->kvh, a->max_len, a->nblocks, a->first, a->last, most};
    const Kv8Dev d = kv8_dev(c, a->layer);
    const cudaError_t e = qw_launch(score_of(c->hd, a->dtype), dim3((most + RECORDS - 1) / RECORDS, c->kvh, a->nb), 256, 0, st, d, k);
    if (e != cudaSuccess) return e;
    return qw_launch(kv8_best_k, dim3(c->kvh, a->nb), 512, 0, st, d, k);
}

cudaError_t launch_kv8_pick(const QwLaunch &L) {
    qw_kv8_cache c;
    qw_kv8_sizes s;
    QW_CHECK_ARG(kv8_from_binds(L, &c, &s) && L.has_bytes(11, 16));
    struct { int64_t s[2]; } st = L.bytes<decltype(st)>(11);
    const qw_kv8_pick_args a = {L.buf<void>(4), L.buf<int32_t>(7), L.buf<int32_t>(8), L.buf<int32_t>(9), L.buf<void>(10), L.avail(10), st.s[0], st.s[1],
                                s.nb, s.layer, s.dtype, s.qh, s.max_len, s.nblocks, s.first, s.last};
    const char *m;
    QW_CHECK_ARG(check_pick(&c, &a, &m) == 0 && L.avail(7) >= (size_t)s.nb * 4 && L.avail(8) >= (size_t)s.nb * 4 && L.avail(9) >= (size_t)s.nb * s.kvh * s.nblocks * 4);
    QW_CHECK_ARG(kv8_rows_fit(L, 4, s.nb, s.qh, s.hd, a.q_row, a.q_head));
    return enqueue_pick(&c, &a, L.stream);
}
}  // namespace
QW_FAMILY(kv8_pick, launch_kv8_pick, 512)

extern "C" size_t qw_kv8_pick_work(const qw_kv8_cache *c, uint32_t nb, uint32_t max_len) {
    size_t n[3];
    if (qw_kv8_bytes(c, n) || nb < 1 || nb > KV8_MAX_ROWS || max_len < 1 || (uint64_t)max_len > (uint64_t)c->max_pages * KV8_PAGE) return 0;
    return work_of(c, nb, max_len);
}
extern "C" int qw_kv8_pick(const qw_kv8_cache *c, const qw_kv8_pick_args *a, void *stream, char *err, size_t errlen) {
    const char *m = kv8_check_cache(c);
    if (m) return kv8_fail(-1, "kv8_pick", m, err, errlen);
    if (const int rc = check_pick(c, a, &m)) return kv8_fail(rc, "kv8_pick", m, err, errlen);
    const void *ptrs[] = {c->codes, c->scales, c->bounds, c->page_table, c->status, a->q, a->lens, a->slots, a->blocks, a->work};
    if ((m = kv8_check_device(ptrs, 10))) return kv8_fail(-3, "kv8_pick", m, err, errlen);
    qw_pdl_current_family("kv8_pick");
    const cudaError_t e = enqueue_pick(c, a, (cudaStream_t)stream);
    if (e != cudaSuccess) return cudaGetLastError(), kv8_fail(-3, "kv8_pick", cudaGetErrorString(e), err, errlen);
    if (err && errlen) err[0] = 0;
    return 0;
}
