// Attention of one new token per row over the 8-bit key-value cache: split over chunks of 256 tokens, joined by kv8_merge_k.
//
//   s_t = scale q . k_t          k_t = code * ks_t: the dot product of q and the codes, times ks_t
//   y   = sum_t 2^(s'_t - m) vs_t code_t / sum_t 2^(s'_t - m),   s' = s log2(e)
// A value's scale goes into the exponent, w_t = 2^(s'_t + log2 vs_t - M) with a running maximum M of its own, so that the weights of the codes are at
// most 1 whatever the scales are.  A chunk leaves sum w_t code_t, M, m and l = sum 2^(s'_t - m) in fp32; the join is
//   y = 2^(M* - m*) sum_c 2^(M_c - M*) acc_c / sum_c 2^(m_c - m*) l_c      with M*, m* the maxima over the chunks, in the order of the chunks.
#include "kv8.cuh"
#include "tmap.cuh"

using namespace qw;

namespace {
constexpr uint32_t CHUNK = 256;

struct AttnArgs {
    const void *q, *gate;
    void *y;
    const int32_t *lens, *slots, *blocks;
    float *part;  // [nb][max_chunks][qh][hd] sums of w code, then [nb][qh][max_chunks] of M, m, l, unused
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

__device__ __forceinline__ float4 *stats_of(const AttnArgs &a, uint32_t hd, uint32_t r, uint32_t qh) {
    return (float4 *)(a.part + (size_t)a.nb * a.max_chunks * a.qh * hd) + ((size_t)r * a.qh + qh) * a.max_chunks;
}

// Four channels of a head's result: times f, times sigmoid(gate), rounded once.
template <class T>
__device__ __forceinline__ void finish(const AttnArgs &a, uint32_t r, uint32_t qh, uint32_t ch, float4 v, float f) {
    float y[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
    if (a.gate) {
        float g[4];
        kv8_load<4>((const T *)a.gate + (int64_t)r * a.g_row + (int64_t)qh * a.g_head + ch, g);
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] *= 1.f / (1.f + expf(-g[j]));
    }
    kv8_store<4>((T *)a.y + (int64_t)r * a.y_row + (int64_t)qh * a.y_head + ch, y);
}

// ------------------------------------------------------------------------------------------------ core
// Persistent blocks of 8 warps; the (row, kv head, chunk) tasks of the launch are numbered in this order and a block takes a run of consecutive ones, so
// that the queries change rarely.  A task goes by tiles of TOK tokens, whose codes come by 2-D tiled copies (swizzled) into a ring of three slots, K and V
// in turn, with the scales of both beside K:
//   scores   S[16 tokens][8 heads] = codes[16][HD] . q^T     mma m16n8k16, a warp per 16 tokens.  Which channel is which k of the product is free as long as
//            both sides agree, so a lane takes 16 codes with one shared-memory load and they feed four products as they lie.
//   maxima   of the block's warps through shared memory, then the weights w as fp16 high part and remainder (22 bits)
//   values   O^T[32 channels][8 heads] += codes^T[32][16 tokens] . w^T: a warp has 32 channels and (for HD < 256) its share of the tokens; four bytes of
//            four tokens give the operands of two 16-channel products after byte permutations.  No sum crosses warps for HD = 256.
// Codes become fp16 numbers exactly (kv8.cuh), queries are scaled by a power of two of their own first, so the products are exact and the sums fp32.
// Two barriers per tile; the loads of the next tile leave right behind the first one.
template <int HD, int NT>
struct Core {
    static constexpr int TOK = HD == 256 ? 128 : HD == 128 && NT == 2 ? 128 : 256;
    static constexpr int BOX = HD < 128 ? HD : 128, HALVES = HD / BOX;  // bytes of a row in a copy, copies side by side
    static constexpr int MT = TOK / 128;             // 16-token tiles of a warp
    static constexpr int DG = HD / 32, TG = 8 / DG;  // groups of 32 channels, shares of the tokens
    static constexpr int KS = TOK / 16 / TG;         // 16-token steps of a warp's share
    static constexpr int SLOT = TOK * HD;
    // shared memory behind the slots
    static constexpr int SCALES = 3 * SLOT, P = SCALES + 3 * 2 * TOK * 4, WMAX = P + TOK / 16 * NT * 512, LSUM = WMAX + 8 * NT * 8 * 8, INFO = LSUM + 8 * NT * 8 * 4,
                         BARS = INFO + 64, FIRST = BARS + 32, BYTES = FIRST + (KV8_MAX_ROWS + 1) * 4 + 1024;
};

template <int HD, int FMT, class T, int NT>
__global__ void __launch_bounds__(256, 2) kv8_attn_k(const __grid_constant__ CUtensorMap tm, Kv8Dev c, AttnArgs a, uint32_t box_rows, unsigned *status) {
    typedef Core<HD, NT> X;
    constexpr int TOK = X::TOK, MT = X::MT;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    const uint32_t base = smem_u32(smem);
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    uint32_t *first = (uint32_t *)(smem + X::FIRST), *info = (uint32_t *)(smem + X::INFO);
    float *wmax = (float *)(smem + X::WMAX), *lsum = (float *)(smem + X::LSUM);
    uint64_t *full = (uint64_t *)(smem + X::BARS);
    if (tid == 0) {
        for (int i = 0; i < 3; i++) mbar_init(&full[i], 1);
        mbar_init_fence();
    }
    pdl_sync();
    // ---- chunks of every row, running sum: row r owns numbers first[r] .. first[r + 1] - 1
    {
        uint32_t n[4], s = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t r = tid * 4 + i;
            n[i] = r < a.nb ? (row_tokens(c, a, r) + CHUNK - 1) / CHUNK : 0;
            s += n[i];
        }
        uint32_t sum = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= (uint32_t)o) sum += u;
        }
        if (lane == 31) info[warp] = sum;
        __syncthreads();
        uint32_t at = sum - s;
        for (uint32_t w = 0; w < warp; w++) at += info[w];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (tid * 4 + i <= a.nb) first[tid * 4 + i] = at;
            at += n[i];
        }
        if (tid == 255 && a.nb == KV8_MAX_ROWS) first[KV8_MAX_ROWS] = at;
        __syncthreads();
    }
    const uint32_t tasks = first[a.nb] * c.kvh;
    const uint32_t lo = (uint32_t)((uint64_t)blockIdx.x * tasks / gridDim.x), hi = (uint32_t)((uint64_t)(blockIdx.x + 1) * tasks / gridDim.x);
    for (uint32_t r = blockIdx.x; r < a.nb; r += gridDim.x)  // rows of length 0
        if (first[r] == first[r + 1] && a.slots[r] >= 0)
            for (uint32_t i = tid; i < a.qh * HD; i += 256) ((T *)a.y)[(int64_t)r * a.y_row + (int64_t)(i / HD) * a.y_head + i % HD] = kv8_round<T>(0.f);
    if (lo >= hi) return;

    struct Task {
        uint32_t r, h, ch, nch, tiles, n;  // n: tokens (of entries) from the chunk's start
        int slot, len;
    };
    auto task_of = [&](uint32_t i) {
        Task k;
        const uint32_t x = i / c.kvh;
        uint32_t l = 0, u = a.nb;  // the last row with first[row] <= x
        while (u - l > 1) {
            const uint32_t m = (l + u) >> 1;
            if (first[m] <= x) l = m;
            else u = m;
        }
        k.r = l;
        k.nch = first[l + 1] - first[l];
        const uint32_t rem = i - first[l] * c.kvh;
        k.h = rem / k.nch;
        k.ch = rem - k.h * k.nch;
        k.slot = a.slots[l];
        k.len = (int)min((uint32_t)a.lens[l], a.max_len);
        k.n = min(CHUNK, row_tokens(c, a, l) - k.ch * CHUNK);
        k.tiles = (k.n + TOK - 1) / TOK;
        return k;
    };

    // ---- loads: lane i of warp 0 looks up and fetches rows i * box_rows .. of a tile
    uint32_t fi = lo, ftile = 0;  // the next tile to look up
    Task ft = task_of(lo);
    uint32_t frow = 0, finfo = 0;  // of the tile looked up: number of the first row; valid tokens | 0x10000 (not in the cache)
    bool fmore = true;             // a tile has been looked up and not fetched
    auto look_up = [&]() {
        frow = finfo = 0;
        fmore = fi < hi;
        if (!fmore) return;
        const uint32_t o = ftile * TOK + lane * box_rows;
        if (lane * box_rows < (uint32_t)TOK && o < ft.n) {
            int64_t tok = ft.ch * CHUNK + o;
            bool bad = false;
            if (a.blocks) {
                const uint32_t e = (uint32_t)tok / c.block;
                const int b = e < a.nblocks ? __ldcg(a.blocks + ((size_t)ft.r * c.kvh + ft.h) * a.nblocks + e) : -1;
                bad = b >= 0 && (uint32_t)b >= ((uint32_t)ft.len + c.block - 1) / c.block;
                tok = b < 0 || bad ? ft.len : (int64_t)b * c.block + (uint32_t)tok % c.block;
            }
            if (tok < ft.len) {
                finfo = min(box_rows, (uint32_t)(ft.len - tok));
                const int page = kv8_page(c, ft.slot, (int)(tok / KV8_PAGE));
                if (page < 0) bad = true;
                else frow = kv8_row0(c, page, 0, ft.h) + (uint32_t)tok % KV8_PAGE;
            }
            if (bad) finfo = box_rows | 0x10000u;
        }
        if (++ftile == ft.tiles) {
            ftile = 0;
            if (++fi < hi) ft = task_of(fi);
        }
    };
    auto fetch = [&](uint32_t j) {  // tile number j of the block: K into slot 2 j mod 3, V into the next
        if (!fmore) return;
        const uint32_t ks = 2 * j % 3, vs = (2 * j + 1) % 3;
        if (lane < 16) info[lane] = finfo;
        if (finfo >> 16) set_status(c.status, ST_BAD_ARG | 0x23);
        const bool mine = finfo && !(finfo >> 16);
        const uint32_t n = __popc(__ballot_sync(0xffffffffu, mine)) * box_rows;
        fence_proxy_async();  // the block's reads of the slots (ordered by the barrier) before the copies' writes
        __syncwarp();
        if (lane == 0) {
            mbar_expect_tx(&full[ks], n * (HD + 8));
            mbar_expect_tx(&full[vs], n * HD);
        }
        __syncwarp();
        if (mine) {
            const uint32_t row = lane * box_rows, vrow = frow + c.kvh * KV8_PAGE;
            float *sc = (float *)(smem + X::SCALES) + ks * 2 * TOK + row;
            bulk_g2s(sc, c.scales + frow, box_rows * 4, &full[ks]);
            bulk_g2s(sc + TOK, c.scales + vrow, box_rows * 4, &full[ks]);
#pragma unroll
            for (int d = 0; d < X::HALVES; d++) tma_load_2d(base + ks * X::SLOT + d * TOK * 128 + row * X::BOX, &tm, d * 128, (int)frow, &full[ks]);
#pragma unroll
            for (int d = 0; d < X::HALVES; d++) tma_load_2d(base + vs * X::SLOT + d * TOK * 128 + row * X::BOX, &tm, d * 128, (int)vrow, &full[vs]);
        }
    };
    if (warp == 0) {
        look_up();
        fetch(0);
        look_up();
    }

    bool dead = false, stop = false;  // this thread has given up a wait; some thread of the block has
    uint32_t j = 0;                   // tiles done
    uint32_t qf[NT][HD / 8];
    float fac[NT][2];
    uint32_t have_r = 0xffffffffu, have_h = 0;
    const uint32_t dg = warp % X::DG, tg = warp / X::DG;
    for (uint32_t i = lo; i < hi; i++) {
        const Task k = task_of(i);
        if (k.r != have_r || k.h != have_h) {
            // queries as B operands: lane (g, t) has head g, 16 channels of every 64, divided by a power of two that leaves the largest in [1, 2)
            have_r = k.r, have_h = k.h;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const uint32_t head = nt * 8 + g;
                const T *qp = (const T *)a.q + (int64_t)k.r * a.q_row + (int64_t)(k.h * a.G + min(head, a.G - 1)) * a.q_head;
                uint32_t m = 0;
#pragma unroll
                for (int cc = 0; cc < HD / 64; cc++) {
                    const int d0 = HD == 64 ? 16 * t : 128 * (cc >> 1) + 16 * (2 * t + (cc & 1));
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        uint32_t w[4];
                        kv8_load_raw8(qp + d0 + 8 * e, w);
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            qf[nt][cc * 8 + e * 4 + x] = w[x];
                            const float2 f = kv8_float2<T>(w[x]);
                            m = max(m, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
                        }
                    }
                }
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const uint32_t ex = min(max(m >> 23, 1u), 253u);
                const float down = __uint_as_float((254u - ex) << 23), up = __uint_as_float(ex << 23);
#pragma unroll
                for (int x = 0; x < HD / 8; x++) {
                    const float2 f = kv8_float2<T>(qf[nt][x]);
                    const __half2 h2 = __floats2half2_rn(f.x * down, f.y * down);
                    qf[nt][x] = head < a.G ? *(const uint32_t *)&h2 : 0u;
                }
                const float f = up * (a.scale2 * kv8_unit<FMT>());
                fac[nt][0] = __shfl_sync(0xffffffffu, f, 8 * t);
                fac[nt][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
            }
        }
        float o[2][NT][4], m[NT][2], M[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int x = 0; x < 4; x++) o[0][nt][x] = o[1][nt][x] = 0.f;
            m[nt][0] = m[nt][1] = M[nt][0] = M[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
        }
        for (uint32_t tile = 0; tile < k.tiles; tile++, j++) {
            const uint32_t ks = 2 * j % 3, vs = (2 * j + 1) % 3;
            if (!dead && !mbar_wait(&full[ks], 2 * j / 3 & 1)) dead = true;
            // ---- scores
            float s[MT][NT][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                const uint32_t tok0 = (warp * MT + mt) * 16;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.f;
#pragma unroll
                for (int cc = 0; cc < HD / 64; cc++) {
                    const uint32_t ad = base + ks * X::SLOT + (HD == 64 ? (tok0 + g) * 64 + ((t ^ (g >> 1 & 3)) << 4) : (cc >> 1) * TOK * 128 + (tok0 + g) * 128 + (((2 * t + (cc & 1)) ^ g) << 4));
                    uint32_t v[4], u[4];
                    lds128(v, ad);
                    lds128(u, ad + 8 * X::BOX);
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        uint32_t af[4];
                        kv8_halves<FMT>(v[x], af[0], af[2]);
                        kv8_halves<FMT>(u[x], af[1], af[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) mma_f16(s[mt][nt], af, qf[nt][cc * 8 + 2 * x], qf[nt][cc * 8 + 2 * x + 1], s[mt][nt]);
                    }
                }
            }
            float lv[MT][2];
            float x0[NT][2], x1[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) x0[nt][0] = x0[nt][1] = x1[nt][0] = x1[nt][1] = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                const uint32_t tok0 = (warp * MT + mt) * 16, inf = info[tok0 / box_rows], off = tok0 % box_rows;
                const float *sc = (const float *)(smem + X::SCALES) + ks * 2 * TOK + tok0;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint32_t row = g + 8 * e;
                    const bool in = off + row < (inf & 0xffffu), bad = inf >> 16;
                    const float kscale = sc[row];
                    lv[mt][e] = log2f(sc[TOK + row]);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int d = 0; d < 2; d++) {
                            float &v = s[mt][nt][2 * e + d];
                            v = bad ? __uint_as_float(0x7fffffffu) : in ? v * (kscale * fac[nt][d]) : -INFINITY;
                            x0[nt][d] = fmaxf(x0[nt][d], v);
                            if (in && !bad) x1[nt][d] = fmaxf(x1[nt][d], v + lv[mt][e]);
                        }
                    if (!in || bad) lv[mt][e] = -INFINITY;
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int d = 0; d < 2; d++)
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) {
                        x0[nt][d] = fmaxf(x0[nt][d], __shfl_xor_sync(0xffffffffu, x0[nt][d], off));
                        x1[nt][d] = fmaxf(x1[nt][d], __shfl_xor_sync(0xffffffffu, x1[nt][d], off));
                    }
            if (g == 0) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) *(float4 *)(wmax + ((warp * NT + nt) * 4 + t) * 4) = make_float4(x0[nt][0], x1[nt][0], x0[nt][1], x1[nt][1]);
            }
            if ((stop = __syncthreads_or(dead))) break;
            if (warp == 0) {
                fetch(j + 1);
                look_up();
            }
            // ---- weights
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float nm[2] = {m[nt][0], m[nt][1]}, nM[2] = {M[nt][0], M[nt][1]};
#pragma unroll
                for (int w = 0; w < 8; w++) {
                    const float4 v = *(const float4 *)(wmax + ((w * NT + nt) * 4 + t) * 4);
                    nm[0] = fmaxf(nm[0], v.x), nM[0] = fmaxf(nM[0], v.y);
                    nm[1] = fmaxf(nm[1], v.z), nM[1] = fmaxf(nM[1], v.w);
                }
#pragma unroll
                for (int d = 0; d < 2; d++) {
                    l[nt][d] *= m[nt][d] == -INFINITY ? 0.f : exp2f(m[nt][d] - nm[d]);
                    const float f = M[nt][d] == -INFINITY ? 0.f : exp2f(M[nt][d] - nM[d]);
#pragma unroll
                    for (int x = 0; x < 2; x++) o[x][nt][d] *= f, o[x][nt][2 + d] *= f;
                    m[nt][d] = nm[d], M[nt][d] = nM[d];
                }
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    uint32_t w[4];  // [token g, g + 8][head 2t, 2t + 1]: high part | remainder << 16
#pragma unroll
                    for (int e = 0; e < 2; e++)
#pragma unroll
                        for (int d = 0; d < 2; d++) {
                            const float v = s[mt][nt][2 * e + d], sv = v + lv[mt][e];
                            l[nt][d] += v == -INFINITY ? 0.f : exp2f(v - nm[d]);
                            const float wt = sv == -INFINITY ? 0.f : exp2f(sv - nM[d]);
                            const __half h = __float2half_rn(wt), r = __float2half_rn(wt - __half2float(h));
                            w[2 * e + d] = (uint32_t)__half_as_ushort(h) | (uint32_t)__half_as_ushort(r) << 16;
                        }
                    // lanes of tokens g, g ^ 1 swap: the even one writes both tokens of head 2t, the odd one those of head 2t + 1
                    const bool odd = g & 1;
                    const uint32_t p0 = __shfl_xor_sync(0xffffffffu, odd ? w[0] : w[1], 4), p1 = __shfl_xor_sync(0xffffffffu, odd ? w[2] : w[3], 4);
                    const uint32_t a0 = odd ? p0 : w[0], b0 = odd ? w[1] : p0, a1 = odd ? p1 : w[2], b1 = odd ? w[3] : p1;
                    *(uint4 *)(smem + X::P + (((warp * MT + mt) * NT + nt) * 8 + 2 * t + odd) * 64 + (g >> 1) * 16) =
                        make_uint4(__byte_perm(a0, b0, 0x5410), __byte_perm(a1, b1, 0x5410), __byte_perm(a0, b0, 0x7632), __byte_perm(a1, b1, 0x7632));
                }
            }
            __syncthreads();
            if (!dead && !mbar_wait(&full[vs], (2 * j + 1) / 3 & 1)) dead = true;
            // ---- values
            const uint32_t tv = base + vs * X::SLOT + (HD == 64 ? 2 * t * 64 + (((dg * 2 + (g >> 2)) ^ t) << 4) : (dg >> 2) * TOK * 128 + 2 * t * 128 + ((((dg & 3) * 2 + (g >> 2)) ^ (2 * t)) << 4)) + (g & 3) * 4;
            const uint32_t tv1 = HD == 64 ? tv + 64 : (tv ^ 16) + 128;  // the next token: its row, and its swizzle
#pragma unroll 4
            for (int q = 0; q < X::KS; q++) {
                const uint32_t st = tg * X::KS + q, ro = st * 16 * X::BOX;
                const uint32_t wa = lds32(tv + ro), wb = lds32(tv1 + ro), wc = lds32(tv + ro + 8 * X::BOX), wd = lds32(tv1 + ro + 8 * X::BOX);
                uint32_t a0[4], a1[4];  // channels 4g, 4g + 1 and 4g + 2, 4g + 3
                kv8_halves<FMT>(__byte_perm(wa, wb, 0x5140), a0[0], a0[1]);
                kv8_halves<FMT>(__byte_perm(wc, wd, 0x5140), a0[2], a0[3]);
                kv8_halves<FMT>(__byte_perm(wa, wb, 0x7362), a1[0], a1[1]);
                kv8_halves<FMT>(__byte_perm(wc, wd, 0x7362), a1[2], a1[3]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    uint32_t p[4];
                    lds128(p, base + X::P + (st * NT + nt) * 512 + lane * 16);
                    mma_f16(o[0][nt], a0, p[0], p[1], o[0][nt]);
                    mma_f16(o[1][nt], a1, p[0], p[1], o[1][nt]);
                    mma_f16(o[0][nt], a0, p[2], p[3], o[0][nt]);
                    mma_f16(o[1][nt], a1, p[2], p[3], o[1][nt]);
                }
            }
        }
        if (stop) break;
        // ---- the chunk's totals
        float *ex = (float *)(smem + X::P);  // sums over the tokens of other warps, [tg - 1][dg][NT][8 heads][32 channels], where the weights were
        if (X::TG > 1 && (stop = __syncthreads_or(dead))) break;
        if (X::TG > 1 && tg > 0) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int d = 0; d < 2; d++)
                    *(float4 *)(ex + (((((tg - 1) * X::DG + dg) * NT + nt) * 8 + 2 * t + d) * 8 + g) * 4) = make_float4(o[0][nt][d], o[0][nt][2 + d], o[1][nt][d], o[1][nt][2 + d]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int d = 0; d < 2; d++) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) l[nt][d] += __shfl_xor_sync(0xffffffffu, l[nt][d], off);
                if (g == 0) lsum[warp * NT * 8 + nt * 8 + 2 * t + d] = l[nt][d];
            }
        if ((stop = __syncthreads_or(dead))) break;
        if (tg == 0) {
            const bool poison = a.lens[k.r] > 0 && (uint32_t)a.lens[k.r] > a.max_len;
            if (poison && tid == 0) set_status(c.status, ST_BAD_ARG | 0x24);
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int d = 0; d < 2; d++) {
                    const uint32_t head = nt * 8 + 2 * t + d;
                    if (head >= a.G) continue;
                    float4 v = make_float4(o[0][nt][d], o[0][nt][2 + d], o[1][nt][d], o[1][nt][2 + d]);
#pragma unroll
                    for (int x = 1; x < X::TG; x++) {
                        const float4 u = *(const float4 *)(ex + (((((x - 1) * X::DG + dg) * NT + nt) * 8 + 2 * t + d) * 8 + g) * 4);
                        v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
                    }
                    float lt = lsum[head];
#pragma unroll
                    for (int w = 1; w < 8; w++) lt += lsum[w * NT * 8 + head];
                    const uint32_t qh = k.h * a.G + head, ch0 = 32 * dg + 4 * g;
                    constexpr float unit = kv8_unit<FMT>();
                    if (k.nch > 1) {
                        *(float4 *)(a.part + (((size_t)k.r * a.max_chunks + k.ch) * a.qh + qh) * HD + ch0) = make_float4(v.x * unit, v.y * unit, v.z * unit, v.w * unit);
                        if (dg == 0 && g == 0) stats_of(a, HD, k.r, qh)[k.ch] = make_float4(M[nt][d], m[nt][d], lt, 0.f);
                    } else finish<T>(a, k.r, qh, ch0, v, poison || lt != lt ? __uint_as_float(0x7fffffffu) : M[nt][d] == -INFINITY ? 0.f : exp2f(M[nt][d] - m[nt][d]) * unit / lt);
                }
        }
        // (the next task's first barrier stands between these reads of shared memory and its writes)
    }
    if (stop) {  // no block ends with copies of its own in flight: those that may be are waited for, with a limit again
        if (tid == 0) {
            set_status(status, ST_MBAR_TIMEOUT | 0x23);
            for (uint32_t e = 2 * j; e < 2 * j + 4; e++) mbar_wait(&full[e % 3], e / 3 & 1);
        }
    }
}

// ------------------------------------------------------------------------------------------------ join
// A block per 64 channels of a (head, row): 16 threads take four channels each of every 16th chunk, the 16 sums are added in order.  Bound: the latency of
// two rounds of loads -- a first form with a block per head went through 188 chunks (48000 tokens) in 47 dependent rounds.  grid (qh hd / 64, nb) x 256
template <int HD, class T>
__global__ void __launch_bounds__(256) kv8_merge_k(Kv8Dev c, AttnArgs a) {
    __shared__ float4 accs[16][16];
    __shared__ float wm[8][2], wl[8];
    pdl_sync();
    const uint32_t qh = blockIdx.x / (HD / 64), ch = blockIdx.x % (HD / 64) * 64, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wc = tid % 16, cg = tid / 16;
    const uint32_t n = row_tokens(c, a, r), nch = (n + CHUNK - 1) / CHUNK;
    if (nch < 2) return;  // written by the core
    const float4 *st = stats_of(a, HD, r, qh);
    float m = -INFINITY, M = -INFINITY;
    for (uint32_t k = tid; k < nch; k += 256) {
        const float4 s = __ldcg(st + k);
        M = fmaxf(M, s.x);
        m = fmaxf(m, s.y);
    }
    m = warp_max(m), M = warp_max(M);
    if (lane == 0) wm[warp][0] = m, wm[warp][1] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) m = fmaxf(m, wm[w][0]), M = fmaxf(M, wm[w][1]);
    float l = 0.f;
    for (uint32_t k = tid; k < nch; k += 256) {
        const float4 s = __ldcg(st + k);
        l += s.y == -INFINITY ? s.z : s.z * exp2f(s.y - m);  // (0, or NaN, where a chunk has no maximum)
    }
    l = warp_sum(l);
    if (lane == 0) wl[warp] = l;
    const float4 *p = (const float4 *)(a.part + ((size_t)r * a.max_chunks * a.qh + qh) * HD + ch) + wc;
    const size_t cs = (size_t)a.qh * (HD / 4);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (uint32_t k = cg; k < nch; k += 16) {
        const float Mk = __ldcg(&st[k].x), w = Mk == -INFINITY ? 0.f : exp2f(Mk - M);
        const float4 v = __ldcg(p + k * cs);
        acc.x = fmaf(v.x, w, acc.x), acc.y = fmaf(v.y, w, acc.y), acc.z = fmaf(v.z, w, acc.z), acc.w = fmaf(v.w, w, acc.w);
    }
    accs[cg][wc] = acc;
    __syncthreads();
    if (tid >= 16) return;
    l = wl[0];
#pragma unroll
    for (int w = 1; w < 8; w++) l += wl[w];
#pragma unroll
    for (int g = 1; g < 16; g++) {
        const float4 v = accs[g][tid];
        acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
    }
    const bool bad = (uint32_t)a.lens[r] > a.max_len;
    finish<T>(a, r, qh, ch + 4 * tid, acc, l != l || bad ? __uint_as_float(0x7fffffffu) : M == -INFINITY ? 0.f : exp2f(M - m) / l);
}

// Which kernel: by the format, the type of rows, and whether 8 or 16 heads share a kv head.
typedef void (*core_kernel)(CUtensorMap, Kv8Dev, AttnArgs, uint32_t, unsigned *);
typedef void (*merge_kernel)(Kv8Dev, AttnArgs);
struct Launch {
    core_kernel core;
    merge_kernel merge;
    int smem;
};
template <int HD, int FMT, class T>
Launch launch_of(bool wide) {
    return wide ? Launch{kv8_attn_k<HD, FMT, T, 2>, kv8_merge_k<HD, T>, Core<HD, 2>::BYTES} : Launch{kv8_attn_k<HD, FMT, T, 1>, kv8_merge_k<HD, T>, Core<HD, 1>::BYTES};
}
template <int HD>
Launch launch_of(uint32_t format, uint32_t dtype, bool wide) {
    if (format == QW_KV8_E4M3) return dtype == QW_KV8_FP16 ? launch_of<HD, QW_KV8_E4M3, __half>(wide) : launch_of<HD, QW_KV8_E4M3, __nv_bfloat16>(wide);
    return dtype == QW_KV8_FP16 ? launch_of<HD, QW_KV8_INT8, __half>(wide) : launch_of<HD, QW_KV8_INT8, __nv_bfloat16>(wide);
}
Launch launch_of(uint32_t hd, uint32_t format, uint32_t dtype, bool wide) {
    return hd == 64 ? launch_of<64>(format, dtype, wide) : hd == 128 ? launch_of<128>(format, dtype, wide) : launch_of<256>(format, dtype, wide);
}

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
cudaError_t enqueue_attn(const qw_kv8_cache *c, const qw_kv8_attn_args *a, cudaStream_t st, unsigned *status) {
    const uint32_t mc = chunks_of(c, a->max_len, a->blocks ? a->nblocks : 0), box_rows = a->blocks && c->block < 32 ? c->block : 32;
    const AttnArgs k = {a->q, a->gate, a->y, a->lens, a->slots, a->blocks, (float *)a->work, a->q_row, a->q_head, a->gate_row, a->gate_head, a->y_row, a->y_head,
                        (float)(a->scale * 1.4426950408889634), a->nb, a->qh, a->qh / c->kvh, a->max_len, a->nblocks, mc};
    const Kv8Dev d = kv8_dev(c, a->layer);
    CUtensorMap tm;
    const uint64_t rows = (uint64_t)c->pages * c->layers * 2 * c->kvh * KV8_PAGE;
    if (!tmap_2d(&tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, c->codes, c->hd, rows, c->hd, c->hd < 128 ? c->hd : 128, box_rows,
                 c->hd < 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B))
        return cudaErrorInvalidValue;
    const Launch L = launch_of(c->hd, c->format, a->dtype, k.G > 8);
    cudaError_t e = cudaFuncSetAttribute(L.core, cudaFuncAttributeMaxDynamicSharedMemorySize, L.smem);
    if (e != cudaSuccess) return e;
    const uint64_t most = (uint64_t)a->nb * mc * c->kvh, fit = 2 * (uint64_t)kv8_sm_count();
    e = qw_launch(L.core, (uint32_t)(most < fit ? most : fit), 256, L.smem, st, tm, d, k, box_rows, status);
    if (e != cudaSuccess || mc < 2) return e;
    return qw_launch(L.merge, dim3(a->qh * (c->hd / 64), a->nb), 256, 0, st, d, k);
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
    return enqueue_attn(&c, &a, L.stream, L.status);
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
    const cudaError_t e = enqueue_attn(c, a, (cudaStream_t)stream, c->status);
    if (e != cudaSuccess) return cudaGetLastError(), kv8_fail(-3, "kv8_attn", cudaGetErrorString(e), err, errlen);
    if (err && errlen) err[0] = 0;
    return 0;
}
