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
constexpr uint32_t RECORDS = 64;  // of a block of threads

__device__ __forceinline__ uint32_t row_blocks(const Kv8Dev &c, const PickArgs &a, int slot, int len) {
    return slot < 0 || len <= 0 ? 0 : (min((uint32_t)len, a.max_len) + c.block - 1) / c.block;
}
// Larger numbers have larger keys; no number has key 0 or 0xffffffff.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 becomes +0: the two are equal
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// Scores as keys.  A warp has eight consecutive records and asks for all of them before it scores the first; a record is one load of the warp: half of its lanes
// the lower bounds, which the negative parts of q8 meet, the others the upper ones and the positive parts.  Four products at a time (dp4a), sums of whole
// numbers across the warp.  Bound: the latency of page id and record, then the bytes of the records (one record after the other took 27 us for 100,000).
// grid (ceil(most blocks / 64), kvh, nb) x 256
template <int HD, class T>
__global__ void __launch_bounds__(256) kv8_score_k(Kv8Dev c, PickArgs a) {
    constexpr int E = HD / 16, W = E / 4, PER = RECORDS / 8;  // bytes and words of a record per lane, records of a warp
    __shared__ __align__(16) int8_t q8[16][2][HD];            // negative parts, positive parts
    __shared__ float sqs[16];
    pdl_sync();
    const uint32_t h = blockIdx.y, r = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int len = a.lens[r], slot = a.slots[r];
    const uint32_t n = row_blocks(c, a, slot, len), per = KV8_PAGE / c.block, b0 = blockIdx.x * RECORDS + warp * PER;
    if (blockIdx.x * RECORDS >= n) return;
    // records of the warp, lanes 0 to 7 ask for their pages
    const uint32_t mine = b0 + (lane & (PER - 1));
    const int page = mine < n ? kv8_page(c, slot, (int)(mine / per)) : -1;
    for (uint32_t g = warp; g < a.G; g += 8) {
        float x[HD / 32];
        kv8_load<HD / 32>((const T *)a.q + (int64_t)r * a.q_row + (int64_t)(h * a.G + g) * a.q_head + lane * (HD / 32), x);
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
            q8[g][0][lane * (HD / 32) + i] = (int8_t)min(v, 0);
            q8[g][1][lane * (HD / 32) + i] = (int8_t)max(v, 0);
        }
        if (lane == 0) sqs[g] = none ? 0.f : __fdiv_rn(am, 127.f);
    }
    uint32_t w[PER][W];
    float sb[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int pg = __shfl_sync(0xffffffffu, page, i);
        sb[i] = 0.f;
#pragma unroll
        for (int j = 0; j < W; j++) w[i][j] = 0;
        if (pg < 0) continue;
        const uint8_t *rec = c.bounds + kv8_bound_at(c, pg, h, (b0 + i) % per);
        sb[i] = __ldcg((const float *)(rec + 2 * HD));
        if (W == 4) {
            const uint4 v = __ldcg((const uint4 *)rec + lane);
            w[i][0] = v.x, w[i][W > 1 ? 1 : 0] = v.y, w[i][W > 2 ? 2 : 0] = v.z, w[i][W > 3 ? 3 : 0] = v.w;
        } else if (W == 2) {
            const uint2 v = __ldcg((const uint2 *)rec + lane);
            w[i][0] = v.x, w[i][W > 1 ? 1 : 0] = v.y;
        } else w[i][0] = __ldcg((const uint32_t *)rec + lane);
    }
    __syncthreads();
    float best[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) best[i] = -INFINITY;
    for (uint32_t g = 0; g < a.G; g++) {
        int q[W];
#pragma unroll
        for (int j = 0; j < W; j++) q[j] = *(const int *)(&q8[g][0][0] + lane * E + 4 * j);
        const float sq = sqs[g];
#pragma unroll
        for (int i = 0; i < PER; i++) {
            int s = 0;
#pragma unroll
            for (int j = 0; j < W; j++) s = __dp4a((int)w[i][j], q[j], s);
            s = __reduce_add_sync(0xffffffffu, s);
            best[i] = fmaxf(best[i], s ? __fmul_rn(__fmul_rn(sq, sb[i]), (float)s) : 0.f);
        }
    }
    uint32_t key = 0;
#pragma unroll
    for (int i = 0; i < PER; i++)
        if (lane == (uint32_t)i) key = key_of(sb[i] == INFINITY ? INFINITY : best[i]);
    if (lane < PER && mine < n) {
        if (page < 0) {
            key = 0;
            set_status(c.status, ST_BAD_ARG | 0x25);
        } else if (mine < a.first || mine + a.last >= n) key = 0xffffffffu;
        a.keys[((size_t)r * c.kvh + h) * a.stride + mine] = key;
    }
}

// Block-wide exclusive prefix sum (1024 threads)
__device__ __forceinline__ uint32_t scan_1024(uint32_t v, uint32_t *ws, uint32_t &total) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= (uint32_t)o) s += t;
    }
    if (lane == 31) ws[warp] = s;
    __syncthreads();
    if (warp == 0) {
        uint32_t x = ws[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= (uint32_t)o) x += t;
        }
        ws[lane] = x;
    }
    __syncthreads();
    const uint32_t e = (warp ? ws[warp - 1] : 0) + s - v;
    total = ws[31];
    __syncthreads();
    return e;
}

// The `count` largest keys in ascending order of their blocks; of the keys that equal the smallest of them the lowest blocks are taken.  A thread owns a run of
// consecutive blocks, so prefix sums give the places.  grid (kvh, nb) x 1024
//   up to 4096 blocks: four keys per thread in registers; the threshold is found two bits at a time, one barrier each (three passes of histograms with
//   their barriers took 8 us for 750 blocks)
//   more: radix selection (11 + 11 + 10 bits) over the keys in memory
__global__ void __launch_bounds__(1024) kv8_best_k(Kv8Dev c, PickArgs a) {
    __shared__ uint32_t hist[2048], ws[32], sh_bin, sh_rem;
    pdl_sync();
    const uint32_t h = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
    const int len = a.lens[r], slot = a.slots[r];
    if (slot < 0) return;
    const bool bad = len > 0 && (uint32_t)len > a.max_len;
    if (tid == 0 && bad) set_status(c.status, ST_BAD_ARG | 0x26);
    const uint32_t n = bad ? 0 : row_blocks(c, a, slot, len);
    const uint32_t *keys = a.keys + ((size_t)r * c.kvh + h) * a.stride;
    int32_t *out = a.out + ((size_t)r * c.kvh + h) * a.count;
    uint32_t T = 0, rem = 0;  // keys above T are taken, and `rem` of those equal to it (T = 0: all that have a page)
    if (n <= 4096) {
        uint32_t k[4], at, taken = 0;
        if (4 * tid < n) {
            const uint4 v = __ldcg((const uint4 *)keys + tid);  // (a row's keys have room for a multiple of four)
            k[0] = v.x, k[1] = 4 * tid + 1 < n ? v.y : 0, k[2] = 4 * tid + 2 < n ? v.z : 0, k[3] = 4 * tid + 3 < n ? v.w : 0;
        } else k[0] = k[1] = k[2] = k[3] = 0;
        if (n > a.count) {
            uint32_t(*cnt)[4] = (uint32_t(*)[4])hist;
            if (tid < 64) hist[tid] = 0;
            __syncthreads();
            rem = a.count;  // of the keys that share T's bits so far
            for (int it = 0; it < 16; it++) {
                const int sh = 30 - 2 * it;
                // keys that share the bits above, by their next two bits: counts of 3, 2 and 1, at most 128 per warp each
                uint32_t s = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t x = k[i] >> sh, d = x & 3;
                    if (it == 0 || x >> 2 == T) s += d == 3 ? 1u : d == 2 ? 1u << 10 : d == 1 ? 1u << 20 : 0;
                }
                s = __reduce_add_sync(0xffffffffu, s);
                if ((tid & 31) == 0 && s) {
                    if (s & 1023) atomicAdd(&cnt[it][3], s & 1023);
                    if (s >> 10 & 1023) atomicAdd(&cnt[it][2], s >> 10 & 1023);
                    if (s >> 20) atomicAdd(&cnt[it][1], s >> 20);
                }
                __syncthreads();
                const uint32_t c3 = cnt[it][3], c2 = cnt[it][2], c1 = cnt[it][1];
                uint32_t d = 3;
                if (rem > c3) {
                    rem -= c3, d = 2;
                    if (rem > c2) {
                        rem -= c2, d = 1;
                        if (rem > c1) rem -= c1, d = 0;
                    }
                }
                T = T << 2 | d;
            }
            if (T == 0) rem = 0;  // (fewer blocks with a page than wanted)
        }
        uint32_t v = 0;  // taken ones above T | equal to T << 16
#pragma unroll
        for (int i = 0; i < 4; i++) v += k[i] > T ? 1u : T && k[i] == T ? 1u << 16 : 0;
        const uint32_t e = scan_1024(v, ws, at);
        uint32_t eq = e >> 16;
        taken = (at & 0xffff) + min(at >> 16, rem);
        uint32_t place = (e & 0xffff) + min(eq, rem);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (k[i] > T || (T && k[i] == T && eq++ < rem)) out[place++] = (int32_t)(4 * tid + i);
        for (uint32_t i = taken + tid; i < a.count; i += 1024) out[i] = -1;
        return;
    }
    if (n > a.count) {
        rem = a.count;
        const int shifts[3] = {21, 10, 0}, widths[3] = {11, 11, 10};
        for (int ps = 0; ps < 3; ps++) {
            const int sh = shifts[ps], nbins = 1 << widths[ps];
            for (uint32_t b = tid; b < 2048; b += 1024) hist[b] = 0;
            __syncthreads();
            for (uint32_t i = tid; i < n; i += 1024) {
                const uint32_t key = __ldcg(keys + i);
                if (ps == 0 || (key >> (sh + widths[ps])) == T) atomicAdd(&hist[(key >> sh) & (nbins - 1)], 1u);
            }
            __syncthreads();
            const uint32_t b1 = 2047 - 2 * tid, b0 = b1 - 1;
            const uint32_t h1 = b1 < (uint32_t)nbins ? hist[b1] : 0, h0 = b0 < (uint32_t)nbins ? hist[b0] : 0;
            uint32_t tot;
            const uint32_t e = scan_1024(h1 + h0, ws, tot);  // keys in all bins above b1
            if (e < rem && e + h1 >= rem) sh_bin = b1, sh_rem = rem - e;
            else if (e + h1 < rem && e + h1 + h0 >= rem) sh_bin = b0, sh_rem = rem - e - h1;
            __syncthreads();
            T = (T << widths[ps]) | sh_bin;
            rem = sh_rem;
            __syncthreads();
        }
        if (T == 0) rem = 0;
    }
    const uint32_t run = (n + 1023) / 1024, i0 = min(n, tid * run), i1 = min(n, i0 + run);
    uint32_t above = 0, equal = 0, tot_above, tot_equal;
    for (uint32_t i = i0; i < i1; i++) {
        const uint32_t key = __ldcg(keys + i);
        above += key > T;
        equal += T && key == T;
    }
    const uint32_t ea = scan_1024(above, ws, tot_above), ee = scan_1024(equal, ws, tot_equal);
    uint32_t at = ea + min(ee, rem), eq = ee;
    for (uint32_t i = i0; i < i1; i++) {
        const uint32_t key = __ldcg(keys + i);
        if (key > T || (T && key == T && eq++ < rem)) out[at++] = (int32_t)i;
    }
    for (uint32_t i = tot_above + min(tot_equal, rem) + tid; i < a.count; i += 1024) out[i] = -1;
}

typedef void (*pick_kernel)(Kv8Dev, PickArgs);
pick_kernel score_of(uint32_t hd, uint32_t dtype) {
    if (dtype == QW_KV8_FP16) return hd == 64 ? kv8_score_k<64, __half> : hd == 128 ? kv8_score_k<128, __half> : kv8_score_k<256, __half>;
    return hd == 64 ? kv8_score_k<64, __nv_bfloat16> : hd == 128 ? kv8_score_k<128, __nv_bfloat16> : kv8_score_k<256, __nv_bfloat16>;
}
uint32_t most_blocks(const qw_kv8_cache *c, uint32_t max_len) { return (uint32_t)(((uint64_t)max_len + c->block - 1) / c->block); }
uint32_t key_stride(const qw_kv8_cache *c, uint32_t max_len) { return (most_blocks(c, max_len) + 3) / 4 * 4; }
size_t work_of(const qw_kv8_cache *c, uint32_t nb, uint32_t max_len) { return (size_t)nb * c->kvh * key_stride(c, max_len) * 4; }
int check_pick(const qw_kv8_cache *c, const qw_kv8_pick_args *a, const char **m) {
    if (!a) return *m = "no arguments", -1;
    if (!c->bounds) return *m = "the cache has no bounds", -1;
    if ((*m = kv8_check_layer(c, a->nb, a->layer, a->dtype))) return -1;
    if (a->qh < c->kvh || a->qh % c->kvh || a->qh / c->kvh > 16) return *m = "1 to 16 query heads share a kv head", -1;
    if (a->max_len < 1 || (uint64_t)a->max_len > (uint64_t)c->max_pages * KV8_PAGE) return *m = "max_len is 1 to 256 max_pages", -1;
    if (a->nblocks < 1 || (uint64_t)a->first + a->last > a->nblocks) return *m = "at least one block is chosen, and first + last of them at most", -1;
    if (!a->q || !a->lens || !a->slots || !a->blocks || !a->work) return *m = "null pointer argument", -1;
    if ((uintptr_t)a->work & 15) return *m = "the workspace starts at a 16-byte boundary", -1;
    if (a->work_bytes < work_of(c, a->nb, a->max_len)) return *m = "the workspace is too small", -2;
    return 0;
}
cudaError_t enqueue_pick(const qw_kv8_cache *c, const qw_kv8_pick_args *a, cudaStream_t st) {
    const uint32_t most = most_blocks(c, a->max_len);
    const PickArgs k = {a->q, a->lens, a->slots, a->blocks, (uint32_t *)a->work, a->q_row, a->q_head, a->nb, a->qh, a->qh / c->kvh, a->max_len, a->nblocks, a->first, a->last, key_stride(c, a->max_len)};
    const Kv8Dev d = kv8_dev(c, a->layer);
    const cudaError_t e = qw_launch(score_of(c->hd, a->dtype), dim3((most + RECORDS - 1) / RECORDS, c->kvh, a->nb), 256, 0, st, d, k);
    if (e != cudaSuccess) return e;
    return qw_launch(kv8_best_k, dim3(c->kvh, a->nb), 1024, 0, st, d, k);
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
QW_FAMILY(kv8_pick, launch_kv8_pick, 1024)

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
