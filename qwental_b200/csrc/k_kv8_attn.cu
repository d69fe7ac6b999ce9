// Attention of one new token per row over the 8-bit key-value cache: split over chunks of 256 tokens, joined by kv8_merge_k.
//
//   s_t = scale q . k_t          k_t = code * ks_t: the dot product of q and the codes, times ks_t
//   y   = sum_t 2^(s'_t - m) vs_t code_t / sum_t 2^(s'_t - m),   s' = s log2(e)
// A value's scale goes into the exponent, w_t = 2^(s'_t + log2 vs_t - M) with a running maximum M of its own, so that the weights of the codes are at
// most 1 whatever the scales are.  A chunk leaves sum w_t code_t, M, m and l = sum 2^(s'_t - m) in fp32; the join is
//   y = 2^(M* - m*) sum_c 2^(M_c - M*) acc_c / sum_c 2^(m_c - m*) l_c      with M*, m* the maxima over the chunks, in the order of the chunks.
#include "kv8.cuh"

using namespace qw;

namespace {
constexpr uint32_t CHUNK = 256;

struct AttnArgs {
    const void *q, *gate;
    void *y;
    const int32_t *lens, *slots, *blocks;
    float *part;  // [nb][max_chunks][qh][hd + 4]: sum w code, then M, m, l, unused
    int64_t q_row, q_head, g_row, g_head, y_row, y_head;
    float scale2;  // softmax scale * log2(e)
    uint32_t nb, qh, G, max_len, nblocks, max_chunks;
};

// Tokens, or entries' tokens, that a row goes over (0: none or not in use), and whether its length is one the call allows.
__device__ __forceinline__ uint32_t row_tokens(const Kv8Dev &c, const AttnArgs &a, uint32_t r) {
    const int len = a.lens[r];
    if (a.slots[r] < 0 || len <= 0) return 0;
    const uint32_t n = min((uint32_t)len, a.max_len);
    return a.blocks ? min(a.nblocks, (n + c.block - 1) / c.block) * c.block : n;
}

// ------------------------------------------------------------------------------------------------ core
// A thread per token for the scores, a thread per channel for the values.  grid (max_chunks, kvh, nb) x 256
template <int HD, int FMT, class T>
__global__ void __launch_bounds__(256) kv8_attn_k(Kv8Dev c, AttnArgs a) {
    __shared__ float qs[16][HD], ss[16][CHUNK], ls[16][3];
    __shared__ uint32_t rowv[CHUNK];
    pdl_sync();
    const uint32_t ch = blockIdx.x, h = blockIdx.y, r = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t n = row_tokens(c, a, r);
    if (ch * CHUNK >= n) return;
    const int slot = a.slots[r];
    const uint32_t len = min((uint32_t)a.lens[r], a.max_len);
    for (uint32_t i = tid; i < a.G * HD; i += 256)
        qs[i / HD][i % HD] = kv8_float(((const T *)a.q)[(int64_t)r * a.q_row + (int64_t)(h * a.G + i / HD) * a.q_head + i % HD]);
    __syncthreads();
    int64_t t = ch * CHUNK + tid;
    if (a.blocks) {
        const uint32_t e = (uint32_t)t / c.block;
        const int b = e < a.nblocks ? a.blocks[((size_t)r * c.kvh + h) * a.nblocks + e] : -1;
        t = b < 0 ? (int64_t)len : (int64_t)b * c.block + tid % c.block;
        if (b >= 0 && (uint32_t)b >= (len + c.block - 1) / c.block) t = -1;
    }
    const bool in = t < (int64_t)len;
    const int page = in && t >= 0 ? kv8_page(c, slot, (int)(t / KV8_PAGE)) : -1;
    const bool bad = in && page < 0;
    if (bad) set_status(c.status, ST_BAD_ARG | 0x23);
    rowv[tid] = in && !bad ? kv8_row0(c, page, 0, h) + (uint32_t)(t % KV8_PAGE) : 0xffffffffu;
    const uint32_t vrows = c.kvh * KV8_PAGE;
    float vl = 0.f, sc[16];
    for (uint32_t g = 0; g < 16; g++) sc[g] = 0.f;
    if (in && !bad) {
        const uint32_t row = rowv[tid];
        for (uint32_t w = 0; w < HD / 4; w++) {
            float x[4];
            kv8_decode4<FMT>(__ldcg((const uint32_t *)(c.codes + (size_t)row * HD) + w), x);
            for (uint32_t g = 0; g < 16; g++)
                if (g < a.G)
                    for (int j = 0; j < 4; j++) sc[g] = fmaf(x[j], qs[g][4 * w + j], sc[g]);
        }
        const float ks = __ldcg(c.scales + row) * a.scale2;
        vl = log2f(__ldcg(c.scales + row + vrows));
        for (uint32_t g = 0; g < 16; g++) sc[g] *= ks;
    }
    // per head: maxima, the sum, and the weights
    __shared__ float red[8][16][2];
    for (uint32_t g = 0; g < a.G; g++) {
        const float s = bad ? __uint_as_float(0x7fffffffu) : in ? sc[g] : -INFINITY, sv = in ? s + vl : -INFINITY;
        const float m0 = warp_max(s), m1 = warp_max(sv);
        if (lane == 0) red[warp][g][0] = m0, red[warp][g][1] = m1;
    }
    __syncthreads();
    for (uint32_t g = 0; g < a.G; g++) {
        float m = red[0][g][0], M = red[0][g][1];
        for (int w = 1; w < 8; w++) m = fmaxf(m, red[w][g][0]), M = fmaxf(M, red[w][g][1]);
        const float s = bad ? __uint_as_float(0x7fffffffu) : in ? sc[g] : -INFINITY, sv = in ? s + vl : -INFINITY;
        ss[g][tid] = sv == -INFINITY ? 0.f : exp2f(sv - M);
        const float p = s == -INFINITY ? 0.f : exp2f(s - m), l = warp_sum(p);
        __syncthreads();
        if (lane == 0) red[warp][g][0] = l;
        __syncthreads();
        if (tid == 0) {
            float lt = 0.f;
            for (int w = 0; w < 8; w++) lt += red[w][g][0];
            ls[g][0] = M, ls[g][1] = m, ls[g][2] = lt;
        }
    }
    __syncthreads();
    const uint32_t nt = min(CHUNK, n - ch * CHUNK);
    if (tid < HD) {
        float acc[16];
        for (uint32_t g = 0; g < 16; g++) acc[g] = 0.f;
        for (uint32_t i = 0; i < nt; i++) {
            if (rowv[i] == 0xffffffffu) continue;
            float x[4];
            kv8_decode4<FMT>(c.codes[((size_t)rowv[i] + vrows) * HD + tid], x);
            for (uint32_t g = 0; g < 16; g++)
                if (g < a.G) acc[g] = fmaf(ss[g][i], x[0], acc[g]);
        }
        for (uint32_t g = 0; g < a.G; g++) {
            float *p = a.part + (((size_t)r * a.max_chunks + ch) * a.qh + h * a.G + g) * (HD + 4);
            p[tid] = acc[g];
            if (tid < 3) p[HD + tid] = ls[g][tid];
        }
    }
}

// ------------------------------------------------------------------------------------------------ join
// A block per (head, row): hd / 4 threads take four channels each of every 1024 / hd-th chunk.  grid (qh, nb) x 256
template <int HD, class T>
__global__ void __launch_bounds__(256) kv8_merge_k(Kv8Dev c, AttnArgs a) {
    constexpr uint32_t TC = HD / 4, NG = 256 / TC;
    __shared__ float4 accs[NG][TC];
    __shared__ float wm[8][3], lsum[NG];
    pdl_sync();
    const uint32_t qh = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wc = tid % TC, cg = tid / TC;
    if (a.slots[r] < 0) return;
    const uint32_t n = row_tokens(c, a, r), nch = (n + CHUNK - 1) / CHUNK;
    const float *base = a.part + ((size_t)r * a.max_chunks * a.qh + qh) * (HD + 4);
    const size_t cs = (size_t)a.qh * (HD + 4);
    float m = -INFINITY, M = -INFINITY, nan = 0.f;
    for (uint32_t k = tid; k < nch; k += 256) {
        const float Mk = __ldcg(base + k * cs + HD), mk = __ldcg(base + k * cs + HD + 1), lk = __ldcg(base + k * cs + HD + 2);
        m = fmaxf(m, mk);
        M = fmaxf(M, Mk);
        if (lk != lk) nan = 1.f;
    }
    m = warp_max(m), M = warp_max(M), nan = warp_max(nan);
    if (lane == 0) wm[warp][0] = m, wm[warp][1] = M, wm[warp][2] = nan;
    __syncthreads();
    for (int w = 0; w < 8; w++) m = fmaxf(m, wm[w][0]), M = fmaxf(M, wm[w][1]), nan = fmaxf(nan, wm[w][2]);
    float l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t k = cg; k < nch; k += NG) {
        const float *p = base + k * cs;
        const float Mk = __ldcg(p + HD), mk = __ldcg(p + HD + 1), lk = __ldcg(p + HD + 2);
        const float4 v = __ldcg((const float4 *)p + wc);
        const float w = Mk == -INFINITY ? 0.f : exp2f(Mk - M);
        if (mk != -INFINITY) l = fmaf(lk, exp2f(mk - m), l);
        acc.x = fmaf(v.x, w, acc.x), acc.y = fmaf(v.y, w, acc.y), acc.z = fmaf(v.z, w, acc.z), acc.w = fmaf(v.w, w, acc.w);
    }
    accs[cg][wc] = acc;
    if (wc == 0) lsum[cg] = l;
    __syncthreads();
    if (tid >= TC) return;
    l = lsum[0];
#pragma unroll
    for (uint32_t g = 1; g < NG; g++) {
        const float4 v = accs[g][tid];
        acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
        l += lsum[g];
    }
    const bool bad = a.lens[r] > 0 && (uint32_t)a.lens[r] > a.max_len;
    if (bad && tid == 0) set_status(c.status, ST_BAD_ARG | 0x24);
    const float f = nan > 0.f || bad ? __uint_as_float(0x7fffffffu) : M == -INFINITY ? 0.f : exp2f(M - m) / l;
    float y[4] = {acc.x * f, acc.y * f, acc.z * f, acc.w * f};
    if (a.gate) {
        float g[4];
        kv8_load<4>((const T *)a.gate + (int64_t)r * a.g_row + (int64_t)qh * a.g_head + 4 * tid, g);
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] *= 1.f / (1.f + expf(-g[j]));
    }
    kv8_store<4>((T *)a.y + (int64_t)r * a.y_row + (int64_t)qh * a.y_head + 4 * tid, y);
}

#define BY_DIM(NAME, ...) (hd == 64 ? NAME<64, __VA_ARGS__> : hd == 128 ? NAME<128, __VA_ARGS__> : NAME<256, __VA_ARGS__>)
typedef void (*attn_kernel)(Kv8Dev, AttnArgs);
attn_kernel core_of(uint32_t hd, uint32_t format, uint32_t dtype) {
    if (format == QW_KV8_E4M3) return dtype == QW_KV8_FP16 ? BY_DIM(kv8_attn_k, QW_KV8_E4M3, __half) : BY_DIM(kv8_attn_k, QW_KV8_E4M3, __nv_bfloat16);
    return dtype == QW_KV8_FP16 ? BY_DIM(kv8_attn_k, QW_KV8_INT8, __half) : BY_DIM(kv8_attn_k, QW_KV8_INT8, __nv_bfloat16);
}
attn_kernel merge_of(uint32_t hd, uint32_t dtype) { return dtype == QW_KV8_FP16 ? BY_DIM(kv8_merge_k, __half) : BY_DIM(kv8_merge_k, __nv_bfloat16); }

uint32_t chunks_of(const qw_kv8_cache *c, uint32_t max_len, uint32_t nblocks) {
    const uint64_t blocks = ((uint64_t)max_len + c->block - 1) / c->block;
    const uint64_t n = nblocks ? (nblocks < blocks ? nblocks : blocks) * c->block : max_len;
    return (uint32_t)((n + CHUNK - 1) / CHUNK);
}
const char *check_shape(const qw_kv8_cache *c, uint32_t nb, uint32_t qh, uint32_t max_len) {
    if (nb < 1 || nb > KV8_MAX_ROWS) return "a call has 1 to 1024 rows";
    if (qh < c->kvh || qh % c->kvh || qh / c->kvh > 16) return "1 to 16 query heads share a kv head";
    if (qh > 65535) return "too many query heads";
    if (max_len < 1 || (uint64_t)max_len > (uint64_t)c->max_pages * KV8_PAGE) return "max_len is 1 to 256 max_pages";
    return nullptr;
}
size_t work_of(const qw_kv8_cache *c, uint32_t nb, uint32_t qh, uint32_t max_len, uint32_t nblocks) {
    return (size_t)nb * chunks_of(c, max_len, nblocks) * qh * (c->hd + 4) * 4;
}
// 0, or -1 / -2 with a message
int check_attn(const qw_kv8_cache *c, const qw_kv8_attn_args *a, const char **m) {
    if (!a) return *m = "no arguments", -1;
    if ((*m = kv8_check_layer(c, a->nb, a->layer, a->dtype)) || (*m = check_shape(c, a->nb, a->qh, a->max_len))) return -1;
    if (!a->q || !a->y || !a->lens || !a->slots || !a->work) return *m = "null pointer argument", -1;
    if (a->blocks && a->nblocks < 1) return *m = "chosen blocks of no number", -1;
    if ((uintptr_t)a->work & 15) return *m = "the workspace starts at a 16-byte boundary", -1;
    if (!(a->scale > 0.f) || a->scale > 1e30f) return *m = "the softmax scale is a positive number", -1;
    if (a->work_bytes < work_of(c, a->nb, a->qh, a->max_len, a->blocks ? a->nblocks : 0)) return *m = "the workspace is too small", -2;
    return 0;
}
cudaError_t enqueue_attn(const qw_kv8_cache *c, const qw_kv8_attn_args *a, cudaStream_t st) {
    const uint32_t mc = chunks_of(c, a->max_len, a->blocks ? a->nblocks : 0);
    const AttnArgs k = {a->q, a->gate, a->y, a->lens, a->slots, a->blocks, (float *)a->work, a->q_row, a->q_head, a->gate_row, a->gate_head, a->y_row, a->y_head,
                        (float)(a->scale * 1.4426950408889634), a->nb, a->qh, a->qh / c->kvh, a->max_len, a->nblocks, mc};
    const Kv8Dev d = kv8_dev(c, a->layer);
    const cudaError_t e = qw_launch(core_of(c->hd, c->format, a->dtype), dim3(mc, c->kvh, a->nb), 256, 0, st, d, k);
    if (e != cudaSuccess) return e;
    return qw_launch(merge_of(c->hd, a->dtype), dim3(a->qh, a->nb), 256, 0, st, d, k);
}

cudaError_t launch_kv8_attn(const QwLaunch &L) {
    qw_kv8_cache c;
    qw_kv8_sizes s;
    QW_CHECK_ARG(kv8_from_binds(L, &c, &s) && L.has_bytes(11, 48));
    struct { int64_t s[6]; } st = L.bytes<decltype(st)>(11);
    const qw_kv8_attn_args a = {L.buf<void>(4), L.buf<void>(5), L.buf<void>(6), L.buf<int32_t>(7), L.buf<int32_t>(8), L.buf<int32_t>(9), L.buf<void>(10), L.avail(10),
                                st.s[0], st.s[1], st.s[2], st.s[3], st.s[4], st.s[5], s.scale, s.nb, s.layer, s.dtype, s.qh, s.max_len, s.nblocks, 0};
    const char *m;
    QW_CHECK_ARG(check_attn(&c, &a, &m) == 0 && L.avail(7) >= (size_t)s.nb * 4 && L.avail(8) >= (size_t)s.nb * 4);
    QW_CHECK_ARG(kv8_rows_fit(L, 4, s.nb, s.qh, s.hd, a.q_row, a.q_head) && kv8_rows_fit(L, 6, s.nb, s.qh, s.hd, a.y_row, a.y_head) &&
                 (!a.gate || kv8_rows_fit(L, 5, s.nb, s.qh, s.hd, a.gate_row, a.gate_head)) && (!a.blocks || L.avail(9) >= (size_t)s.nb * s.kvh * s.nblocks * 4));
    return enqueue_attn(&c, &a, L.stream);
}
}  // namespace
QW_FAMILY(kv8_attn, launch_kv8_attn, 256)

extern "C" size_t qw_kv8_attn_work(const qw_kv8_cache *c, uint32_t nb, uint32_t qh, uint32_t max_len, uint32_t nblocks) {
    size_t n[3];
    if (qw_kv8_bytes(c, n) || check_shape(c, nb, qh, max_len)) return 0;
    return work_of(c, nb, qh, max_len, nblocks);
}
extern "C" int qw_kv8_attn(const qw_kv8_cache *c, const qw_kv8_attn_args *a, void *stream, char *err, size_t errlen) {
    const char *m = kv8_check_cache(c);
    if (m) return kv8_fail(-1, "kv8_attn", m, err, errlen);
    if (const int rc = check_attn(c, a, &m)) return kv8_fail(rc, "kv8_attn", m, err, errlen);
    const void *ptrs[] = {c->codes, c->scales, c->page_table, c->status, a->q, a->gate, a->y, a->lens, a->slots, a->blocks, a->work};
    if ((m = kv8_check_device(ptrs, 11))) return kv8_fail(-3, "kv8_attn", m, err, errlen);
    qw_pdl_current_family("kv8_attn");
    const cudaError_t e = enqueue_attn(c, a, (cudaStream_t)stream);
    if (e != cudaSuccess) return cudaGetLastError(), kv8_fail(-3, "kv8_attn", cudaGetErrorString(e), err, errlen);
    if (err && errlen) err[0] = 0;
    return 0;
}
