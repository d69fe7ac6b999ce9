// Attention of one new token per row over the 8-bit key-value cache: split over chunks of its tokens, joined by kv8_merge_k.
//
//   s_t = scale q . k_t          k_t = code * ks_t: the dot product of q and the codes, times ks_t
//   y   = sum_t 2^(s'_t) vs_t code_t / sum_t 2^(s'_t),   s' = s log2(e)
// A value's scale goes into the exponent, w_t = 2^(s'_t + log2 vs_t - M) with M the running maximum of s' + log2 vs, less 15, so that the weights of the codes are at
// most 2^15 whatever the scales are (of a row of zeros, whose scale is 0, it is 0).  They become two fp16 numbers, high part and remainder: 22 bits of a weight down to
// 2^-16 of the largest one so far in the chunk, below that to 2^-40 of it.  The denominator has a maximum of its own: l = sum 2^(s'_t - S) with S that of s',
// since M may be far from S both ways, by as much as the scales of the values are from 1.  (log2 and 2^x are the fast ones: 2^-22 of log2 vs, 2^-22 of a weight.)  A chunk
// leaves acc = sum w_t code_t, M, S and l in fp32; the join is
//   y = 2^(M* - S*) sum_c 2^(M_c - M*) acc_c / sum_c 2^(S_c - S*) l_c      with M*, S* the maxima over the chunks, in the order of the chunks.
#include "kv8.cuh"
#include "tmap.cuh"

using namespace qw;

namespace {
// Tokens of a chunk, by the tokens of its row alone (a row's result does not depend on the others of a call): short rows in small pieces, for their latency;
// a chunk of 128 leaves 12 % of its own bytes as fp32 sums, in L2.  With 256 from 8193 tokens on, one row of 48000 took 24 us instead of 20 and 16 ragged rows
// of 1K to 48K had single warps that ended 9 us after the others; beyond 65536 a warp has chunks enough, and half the sums to join count for more: one row of 131000 takes 42 us
// instead of 53, of 500000 135 instead of 163, 8 rows of 70K to 130K 163 instead of 179 (one of 66000, just behind the step, 33 instead of 29.5).
// Twice as many for more than eight heads, whose sums are larger, gained 4 to 8 % where there were many rows of up to 2048 tokens and lost 20 to 30 % in most other calls.
__host__ __device__ inline uint32_t chunk_log(uint32_t n) { return n <= 512 ? 5 : n <= 2048 ? 6 : n <= 65536 ? 7 : 8; }
__host__ __device__ inline uint32_t chunk_of(uint32_t n) { return 1u << chunk_log(n); }
__host__ __device__ inline uint32_t chunks_in(uint32_t n) { return (n + chunk_of(n) - 1) >> chunk_log(n); }

struct AttnArgs {
    const void *q, *gate;
    void *y;
    const int32_t *lens, *slots, *blocks;
    float *part;  // [nb][max_chunks][qh][hd] sums of w code, then [nb][qh][max_chunks] of M, S, l and one unused
    int64_t q_row, q_head, g_row, g_head, y_row, y_head;
    float scale2;  // softmax scale * log2(e)
    uint32_t nb, qh, G, max_len, nblocks, max_chunks;
};

// Tokens, or entries' tokens, that a row goes over (0: none or not in use).
__device__ __forceinline__ uint32_t row_tokens(const Kv8Dev &c, const AttnArgs &a, int slot, int len) {
    if (slot < 0 || len <= 0) return 0;
    const uint32_t n = min((uint32_t)len, a.max_len);
    return a.blocks ? min(a.nblocks, (n + c.block - 1) / c.block) * c.block : n;
}
__device__ __forceinline__ uint32_t warp_scan(uint32_t v) {  // inclusive sums
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= (uint32_t)o) v += u;
    }
    return v;
}
__device__ __forceinline__ float exp2_fast(float x) {  // 2^x: 0 below 2^-126
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float4 *stats_of(const AttnArgs &a, uint32_t hd, uint32_t r, uint32_t qh) {
    return (float4 *)(a.part + (size_t)a.nb * a.max_chunks * a.qh * hd) + ((size_t)r * a.qh + qh) * a.max_chunks;
}

// What some tokens leave of two channels, joined with what others leave.  Where there is no maximum the sum is 0 or a NaN.
struct Sums {
    float M, S, l;
    float2 acc;
};
__device__ __forceinline__ void join(Sums &x, float M, float S, float l, float2 acc) {
    const float m = fmaxf(x.M, M), f = x.M == -INFINITY ? 1.f : exp2f(x.M - m), f2 = M == -INFINITY ? 1.f : exp2f(M - m);
    const float n = fmaxf(x.S, S), g = x.S == -INFINITY ? 1.f : exp2f(x.S - n), g2 = S == -INFINITY ? 1.f : exp2f(S - n);
    x.M = m, x.S = n;
    x.l = fmaf(x.l, g, l * g2);
    x.acc.x = fmaf(x.acc.x, f, acc.x * f2);
    x.acc.y = fmaf(x.acc.y, f, acc.y * f2);
}

// ------------------------------------------------------------------------------------------------ core
// Independent warps: the (row, kv head, chunk) tasks of the launch are numbered in this order, each with as many steps of 32 tokens as it has, and a warp
// takes those that start within its share of all steps.  It owns a task completely -- queries, running maximum and the sums of all channels in registers --
// and is fed through a ring of K and V tiles of its own, so warps wait for nothing but their copies and overlap one another.  One warp of the block
// feeds the others, lane w the ring of warp w (feeding themselves cost the warps 2000 to 4000 cycles in a step of 6000).
//   scores   S[16 tokens][8 heads] = codes[16][HD] . q^T     mma m16n8k16.  Which channel is which k of the product is free as long as both sides agree, so a
//            lane takes 16 codes with one shared-memory load and they feed four products as they lie.
//   values   O^T[16 channels][8 heads] += codes^T[16][16 tokens] . w^T     a lane takes 16 codes of four tokens; byte permutations pair the tokens; the weights
//            change lanes by shuffles and travel as fp16 high part and remainder, in two products, or, of up to four heads, in the columns of one.
// Codes become fp16 numbers exactly (kv8.cuh).  Queries go in as fp16 too, times the power of two that leaves a head's largest element in [2^15, 2^16): fp16 ones
// stay what they are, bf16 ones too down to 2^-32 of the largest; smaller ones are rounded to 2^-40 of it.  The products are exact, their sums fp32.
// Measured for 16 ragged rows of 1K to 48K tokens (210 MB, e4m3) against forms that were left: blocks of 8 warps that share a tile of 128 tokens, with two
// barriers per tile, 87 us (scaling, maxima and barriers of a tile 2800 cycles, one after the other); e4m3 operands as they are (mma m16n8k32) no faster, that
// product being converted to fp16 ones by the assembler at every use (19 cycles instead of 8).
// Bound: 46 us (4.6 TB/s, 0.7 of the copy rate): 5 us before a first tile, a tail of 7; ALU pipe 29 %, tensor pipe 21 %, issue slots 25 %.  Nine to sixteen heads at hd 256: latency of
// seven warps per SM at 255 registers, about 300 bytes of them spilled (10 rows of 1612 tokens, 128 heads on 8: 34 us; issue slots 17 %, DRAM 20 %).
constexpr uint32_t STEP = 32;
__device__ __forceinline__ uint32_t share_start(uint32_t total, uint32_t w, uint32_t W) {  // total w / W, in 32 bits
    const uint32_t per = total / W, rest = total - per * W;
    return w * per + w * rest / W;
}

template <int HD, int MODE, bool FEW>
struct Core {
    static constexpr int NT = MODE == 2 ? 2 : 1;                        // tiles of 8 columns
    static constexpr bool DUP = MODE == 0;                              // up to four heads: columns 4 to 7 repeat them
    static constexpr int BOX = HD < 128 ? HD : 128, HALVES = HD / BOX;  // bytes of a row in a copy, copies side by side
    static constexpr int TILE = STEP * HD;                              // K or V
    // warps that compute: what shared memory and registers (for warps in fours, the feeding one among them) allow, one block per SM
    static constexpr int WARPS = FEW ? 6 : HD == 256 ? (NT == 1 ? 11 : 7) : NT == 1 ? 15 : 11;
    static constexpr int KR = FEW ? 2 * 256 / HD : HD == 256 ? 1 : HD == 128 ? 2 : NT == 1 ? 3 : 4;  // K and V tiles of a warp: 12 to 16 KB, or 32
    static constexpr int VR = FEW ? KR : HD == 256 ? 1 : HD == 128 ? (NT == 1 ? 1 : 2) : NT == 1 ? 3 : 4;
    static constexpr int CH = HALVES * (HD < 128 ? 4 : 8);              // 16-channel tiles
    static constexpr int LANE = HD < 128 ? 8 : 16;                      // channels of a lane in a row of a copy
    static constexpr int THREADS = 32 * (WARPS + 1);
    // shared memory behind the tiles: scales of K and V, what a tile is, mbarriers (full and empty, K and V); then 12 bytes per row
    static constexpr int SCALES = WARPS * (KR + VR) * TILE, INFO = SCALES + WARPS * KR * 2 * STEP * 4, BARS = INFO + WARPS * KR * 32, HAS = BARS + WARPS * (KR + VR) * 16,
                         ROWS = HAS + 64, BYTES = ROWS + 1024 + 16;
    static_assert(WARPS + 1 <= 16 && BYTES + 12 * KV8_MAX_ROWS <= 227 * 1024, "words of HAS, and what a block may have");
};

// Of a warp that gave up: what its share of the tasks leaves is not numbers, nor are the rows they are part of, whatever the workspace held.  A function of its own, so that
// nothing is kept for it in the registers of the loop.
__device__ __noinline__ void void_share(const Kv8Dev &c, const AttnArgs &a, const uint32_t *first, uint32_t w, uint32_t W, uint32_t hd) {
    __syncwarp();  // (behind what it may have left already)
    const uint32_t lane = threadIdx.x & 31, total = first[a.nb] * c.kvh, lo = share_start(total, w, W), hi = share_start(total, w + 1, W);
    for (uint32_t r = 0; r < a.nb; r++) {
        const uint32_t steps = first[r + 1] - first[r];
        if (!steps) continue;
        const uint32_t n = row_tokens(c, a, a.slots[r], a.lens[r]), cs = chunk_of(n) / STEP, chunks = chunks_in(n);
        for (uint32_t i = lane; i < c.kvh * chunks; i += 32) {
            const uint32_t h = i / chunks, ch = i % chunks, at = first[r] * c.kvh + h * steps + ch * cs;
            if (at >= lo && at < hi)
                for (uint32_t g = 0; g < a.G; g++) stats_of(a, hd, r, h * a.G + g)[ch] = make_float4(-INFINITY, -INFINITY, __uint_as_float(0x7fffffffu), 0.f);
        }
    }
}

template <int HD, int FMT, class T, int MODE, bool FEW>
__global__ void __launch_bounds__(Core<HD, MODE, FEW>::THREADS, 1) kv8_attn_k(const __grid_constant__ CUtensorMap tm, const __grid_constant__ Kv8Dev c, const __grid_constant__ AttnArgs a, uint32_t box_rows,
                                                                                 unsigned *status) {
    typedef Core<HD, MODE, FEW> X;
    constexpr int KR = X::KR, VR = X::VR, NT = X::NT;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);  // swizzled copies need it
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    uint32_t *has = (uint32_t *)(smem + X::HAS), *first = (uint32_t *)(smem + X::ROWS), *lenv = first + a.nb + 1, *slotv = lenv + a.nb;
    // of warp w: its K tiles, then its V tiles; full and empty barriers of both
    auto tiles_of = [&](uint32_t w) { return smem_u32(smem) + w * (KR + VR) * X::TILE; };
    auto scales_of = [&](uint32_t w) { return (float *)(smem + X::SCALES) + w * KR * 2 * STEP; };
    auto info_of = [&](uint32_t w) { return (uint4 *)(smem + X::INFO) + w * KR * 2; };
    auto bars_of = [&](uint32_t w) { return (uint64_t *)(smem + X::BARS) + w * (KR + VR) * 2; };
    constexpr int KF = 0, VF = KR, KE = KR + VR, VE = 2 * KR + VR;
    for (uint32_t i = tid; i < X::WARPS * (KR + VR) * 2; i += X::THREADS) mbar_init((uint64_t *)(smem + X::BARS) + i, 1);
    mbar_init_fence();
    __syncthreads();
    pdl_sync();
    // ---- rows: steps of one kv head, running sum; length (top bit: longer than the call allows), slot
    auto put_row = [&](uint32_t r) {  // returns its steps
        if (r >= a.nb) return 0u;
        const int len = a.lens[r], slot = a.slots[r];
        lenv[r] = len <= 0 ? 0u : (uint32_t)len > a.max_len ? a.max_len | 0x80000000u : (uint32_t)len;
        slotv[r] = (uint32_t)slot;
        return (row_tokens(c, a, slot, len) + STEP - 1) / STEP;
    };
    if (a.nb <= 64) {  // every warp for itself, all the same values: no barrier (the block's one took 1500 cycles of the 5 us that a row of 100 tokens takes)
        const uint32_t n0 = put_row(2 * lane), n1 = put_row(2 * lane + 1);
        const uint32_t at = warp_scan(n0 + n1) - n0 - n1;
        if (2 * lane <= a.nb) first[2 * lane] = at;
        if (2 * lane + 1 <= a.nb) first[2 * lane + 1] = at + n0;
        if (lane == 31 && a.nb == 64) first[64] = at + n0 + n1;
        __syncwarp();
    } else {
        constexpr uint32_t PER = (KV8_MAX_ROWS + X::THREADS - 1) / X::THREADS;
        uint32_t n[PER], sum = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) sum += n[i] = put_row(tid * PER + i);
        uint32_t at = warp_scan(sum);
        if (lane == 31) has[warp] = at;
        __syncthreads();
        at -= sum;
        for (uint32_t w = 0; w < warp; w++) at += has[w];
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (tid * PER + i < a.nb) first[tid * PER + i] = at;
            at += n[i];
            if (tid * PER + i + 1 == a.nb) first[a.nb] = at;
        }
        __syncthreads();
    }

    // ---- a warp's share, and its first task
    struct Cursor {
        uint32_t r, h, ch, at;          // row, kv head, chunk; the task's first step
        uint32_t steps, cs, len, n;     // of the row: steps, steps of a chunk, length, tokens (of entries)
        int slot;
    } f;
    const uint32_t total = first[a.nb] * c.kvh;
    auto row_of = [&]() {
        f.steps = first[f.r + 1] - first[f.r];
        f.len = lenv[f.r] & 0x7fffffffu;
        f.slot = (int)slotv[f.r];
        f.n = row_tokens(c, a, f.slot, (int)f.len);
        f.cs = chunk_of(f.n) / STEP;
    };
    auto settle = [&]() {  // after f.ch or f.h may have run over
        if (f.ch * f.cs >= f.steps) f.ch = 0, f.h++;
        if (f.h >= c.kvh) {
            f.h = 0;
            do f.r++;
            while (f.r < a.nb && first[f.r + 1] == first[f.r]);
            if (f.r < a.nb) row_of();
        }
        f.at = f.r < a.nb ? first[f.r] * c.kvh + f.h * f.steps + f.ch * f.cs : total;
    };
    auto find = [&](uint32_t w) {  // warp w's; returns the end of its share
        // few tasks go to different SMs first; many to neighbours, who mostly read the same queries
        const uint32_t W = gridDim.x * X::WARPS, w0 = FEW ? w * gridDim.x + blockIdx.x : blockIdx.x * X::WARPS + w;
        const uint32_t lo = share_start(total, w0, W), hi = share_start(total, w0 + 1, W);
        f.at = total;
        if (lo < hi) {
            uint32_t l = 0, u = a.nb;  // the last row that starts at or before lo
            while (u - l > 1) {
                const uint32_t m = (l + u) >> 1;
                if (first[m] * c.kvh <= lo) l = m;
                else u = m;
            }
            f.r = l;
            row_of();
            const uint32_t rem = lo - first[f.r] * c.kvh;
            f.h = rem / f.steps;
            f.ch = (rem - f.h * f.steps + f.cs - 1) / f.cs;
            settle();
        }
        return hi;
    };

    // ---- the feeding warp: lane w has the task whose tiles warp w gets next
    if (warp == X::WARPS) {
        const uint32_t hi = lane < X::WARPS ? find(lane) : 0;
        bool more = lane < X::WARPS && f.at < hi;
        // a tile: 16 tokens each -- valid ones | 0x10000 (not in the cache), token and page of the first
        uint32_t in[2], tok[2], fstep = 0;
        int page[2];
        auto ask = [&]() {
            const uint32_t o = (f.ch * f.cs + fstep) * STEP;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                in[e] = 0;
                page[e] = -1;
                uint32_t x = o + 16 * e;
                if (x >= f.n) continue;
                if (a.blocks) {
                    if (e && box_rows != 16) {  // the same block
                        x = tok[0] + 16;
                        if (!in[0] || in[0] >> 16) continue;
                    } else {
                        const uint32_t en = x / c.block;
                        const int b = en < a.nblocks ? __ldcg(a.blocks + ((size_t)f.r * c.kvh + f.h) * a.nblocks + en) : -1;
                        if (b < 0) continue;
                        if ((uint32_t)b >= (f.len + c.block - 1) / c.block) {
                            in[e] = 16 | 0x10000u;
                            continue;
                        }
                        x = (uint32_t)b * c.block + x % c.block;
                    }
                }
                tok[e] = x;
                if (x >= f.len) continue;
                in[e] = min(16u, f.len - x);
                if ((e == 0 || box_rows == 16) && kv8_entry_ok(c, f.slot, x / KV8_PAGE)) page[e] = __ldcg(c.ptab + (size_t)f.slot * c.max_pages + x / KV8_PAGE);
            }
        };
        if (more) ask();
        uint64_t *bars = bars_of(lane < X::WARPS ? lane : 0);
        uint4 *info = info_of(lane < X::WARPS ? lane : 0);
        float *scales = scales_of(lane < X::WARPS ? lane : 0);
        const uint32_t Kt = tiles_of(lane < X::WARPS ? lane : 0), Vt = Kt + KR * X::TILE, vrows = c.kvh * KV8_PAGE;
        uint32_t fed = 0, vfed = 0;  // K and V tiles so far
        const uint64_t once = evict_first_policy();
        uint64_t t0 = 0;
        uint32_t idle = 0;
        bool ok = true;
        while (__any_sync(0xffffffffu, more || vfed < fed)) {
            bool did = false;
            const uint32_t sl = fed % KR, vl = vfed % VR;
            if (more && fed < vfed + KR /* V of the tile whose place it takes has gone */ && (fed < KR || mbar_test(&bars[KE + sl], fed / KR - 1 & 1))) {
                uint32_t row[2] = {0, 0};
#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (in[e] && !(in[e] >> 16) && (e == 0 || box_rows == 16)) {
                        if (kv8_page_ok(c, page[e])) row[e] = kv8_row0(c, (uint32_t)page[e], 0, f.h) + tok[e] % KV8_PAGE;
                        else in[e] |= 0x10000u;
                    }
                if (box_rows != 16 && in[0] >> 16 && in[1]) in[1] |= 0x10000u;
                if ((in[0] | in[1]) >> 16) set_status(c.status, ST_BAD_ARG | 0x23);
                const bool on0 = in[0] && !(in[0] >> 16), on1 = box_rows == 16 && in[1] && !(in[1] >> 16);
                const uint32_t steps = min(f.cs, f.steps - f.ch * f.cs), of = (fstep == 0 ? 1u : 0u) | (fstep + 1 == steps ? 2u : 0u), r = f.r, h = f.h, ch = f.ch;
                info[2 * sl] = make_uint4(in[0], in[1], row[0], row[1]);
                if (++fstep == steps) {
                    fstep = 0;
                    f.ch++;
                    settle();
                    more = f.at < hi;
                }
                info[2 * sl + 1] = make_uint4(r, h, ch, of | (more ? 0u : 4u));
                mbar_expect_tx(&bars[KF + sl], (on0 + on1) * box_rows * (HD + 8));
#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (e ? on1 : on0) {
                        float *sc = scales + sl * 2 * STEP + e * 16;
#pragma unroll
                        for (int d = 0; d < X::HALVES; d++) tma_load_2d_hint(Kt + sl * X::TILE + d * STEP * 128 + e * 16 * X::BOX, &tm, d * 128, (int)row[e], &bars[KF + sl], once);
                        bulk_g2s(sc, c.scales + row[e], box_rows * 4, &bars[KF + sl]);
                        bulk_g2s(sc + STEP, c.scales + row[e] + vrows, box_rows * 4, &bars[KF + sl]);
                    }
                fed++;
                if (more) ask();
                did = true;
            }
            if (vfed < fed && (vfed < VR || mbar_test(&bars[VE + vl], vfed / VR - 1 & 1))) {
                const uint4 v = info[2 * (vfed % KR)];
                const bool on0 = v.x && !(v.x >> 16), on1 = box_rows == 16 && v.y && !(v.y >> 16);
                mbar_expect_tx(&bars[VF + vl], (on0 + on1) * box_rows * HD);
#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (e ? on1 : on0) {
#pragma unroll
                        for (int d = 0; d < X::HALVES; d++) tma_load_2d_hint(Vt + vl * X::TILE + d * STEP * 128 + e * 16 * X::BOX, &tm, d * 128, (int)((e ? v.w : v.z) + vrows), &bars[VF + vl], once);
                    }
                vfed++;
                did = true;
            }
            if (__any_sync(0xffffffffu, did)) idle = 0;
            else if ((++idle & 255) == 0) {  // a wait of two seconds is given up
                if (idle == 256) t0 = global_ns();
                else if (__any_sync(0xffffffffu, global_ns() - t0 > 2000000000ull)) {
                    ok = false;
                    break;
                }
            }
        }
        if (!ok) {  // no block ends with copies of its own in flight: those that may be are waited for, with a limit again
            if (lane == 0) set_status(status, ST_MBAR_TIMEOUT | 0x23);
            for (uint32_t x = fed < KR ? 0 : fed - KR; x < fed; x++) mbar_wait(&bars[KF + x % KR], x / KR & 1);
            for (uint32_t x = vfed < VR ? 0 : vfed - VR; x < vfed; x++) mbar_wait(&bars[VF + x % VR], x / VR & 1);
        }
        return;
    }
    const uint32_t share_end = find(warp);
    if (f.at >= share_end) return;

    // ---- the computing side
    bool ok = true, more = true;
    uint32_t n = 0, have_r = 0xffffffffu, have_h = 0;
    uint32_t qf[NT][HD / 8];
    float fac[NT][2], o[X::CH][NT][4], M[NT][2], S[NT][2], l[NT][2];  // S and l are of this lane's tokens alone until the chunk ends
    const uint32_t Kb = tiles_of(warp), Vb = Kb + KR * X::TILE;
    uint64_t *bars = bars_of(warp);
    auto load_queries = [&](uint32_t r, uint32_t h) {
        // queries as B operands: lane (g, t) has head g, 16 channels of every 64, times a power of two that leaves the largest in [2^15, 2^16)
        have_r = r, have_h = h;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const uint32_t head = X::DUP ? g & 3 : nt * 8 + g;
            const T *qp = (const T *)a.q + (int64_t)r * a.q_row + (int64_t)(h * a.G + min(head, a.G - 1)) * a.q_head;
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
            const uint32_t ex = max(m >> 23, 16u);  // (so that the power and its inverse are normal numbers)
            const float down = __uint_as_float((254u + 15u - ex) << 23), up = __uint_as_float((ex - 15u) << 23);
#pragma unroll
            for (int x = 0; x < HD / 8; x++) {
                const float2 f = kv8_float2<T>(qf[nt][x]);
                const __half2 h2 = __floats2half2_rn(f.x * down, f.y * down);
                qf[nt][x] = head < a.G ? *(const uint32_t *)&h2 : 0u;
            }
            const float f = m >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : up * a.scale2;  // an infinity or a NaN: the head's results are NaN
            fac[nt][0] = __shfl_sync(0xffffffffu, f, 8 * t);
            fac[nt][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
        }
    };
    load_queries(f.r, f.h);  // the first task's, while its tile is on its way
    for (; more; n++) {
        const uint32_t sl = n % KR, vl = n % VR;
        if (!__all_sync(0xffffffffu, mbar_wait(&bars[KF + sl], n / KR & 1))) {  // (the warp gives up as a whole: its lanes need one another below)
            ok = false;
            break;
        }
        const uint4 in = info_of(warp)[2 * sl], task = info_of(warp)[2 * sl + 1];
        more = !(task.w & 4);
        if (task.w & 1) {
            if (task.x != have_r || task.y != have_h) load_queries(task.x, task.y);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int x = 0; x < X::CH; x++) o[x][nt][0] = o[x][nt][1] = o[x][nt][2] = o[x][nt][3] = 0.f;
                M[nt][0] = M[nt][1] = S[nt][0] = S[nt][1] = -INFINITY;
                l[nt][0] = l[nt][1] = 0.f;
            }
        }
        // ---- scores
        const uint32_t cnt[2] = {in.x >> 16 ? 0u : in.x, in.y >> 16 ? 0u : in.y};  // valid tokens of either 16
        float kf[2][NT][4], lv[2][2];
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float *sc = scales_of(warp) + sl * 2 * STEP + mt * 16 + g + 8 * e;
                const float kscale = sc[0], vscale = sc[STEP];
                lv[mt][e] = __log2f(vscale);  // -infinity for a row of zeros: no weight
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int d = 0; d < 2; d++) kf[mt][nt][2 * e + d] = kscale * fac[nt][d];
            }
        float s[2][NT][4];
        {
            constexpr int CHAINS = HD == 64 ? 1 : 2;  // a product waits for the one before it in its sum
            float sa[CHAINS][2][NT][4];
#pragma unroll
            for (int y = 0; y < CHAINS; y++)
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) sa[y][mt][nt][0] = sa[y][mt][nt][1] = sa[y][mt][nt][2] = sa[y][mt][nt][3] = 0.f;
#pragma unroll
            for (int cc = 0; cc < HD / 64; cc++) {
                uint32_t v[2][4], u[2][4];
#pragma unroll
                for (int mt = 0; mt < 2; mt++) {
                    const uint32_t ad = Kb + sl * X::TILE + (HD == 64 ? (mt * 16 + g) * 64 + ((t ^ (g >> 1 & 3)) << 4) : (cc >> 1) * STEP * 128 + (mt * 16 + g) * 128 + (((2 * t + (cc & 1)) ^ g) << 4));
                    lds128(v[mt], ad);
                    lds128(u[mt], ad + 8 * X::BOX);
                }
#pragma unroll
                for (int x = 0; x < 4; x++)
#pragma unroll
                    for (int mt = 0; mt < 2; mt++) {
                        uint32_t af[4];
                        kv8_operands<FMT>(v[mt][x], af[0], af[2]);
                        kv8_operands<FMT>(u[mt][x], af[1], af[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            float(&y)[4] = sa[x % CHAINS][mt][nt];
                            mma_f16(y, af, qf[nt][cc * 8 + 2 * x], qf[nt][cc * 8 + 2 * x + 1], y);
                        }
                    }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[KE + sl]);
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int x = 0; x < 4; x++) s[mt][nt][x] = (sa[0][mt][nt][x] + (CHAINS > 1 ? sa[CHAINS - 1][mt][nt][x] : 0.f)) * kf[mt][nt][x];
        }
        if (cnt[0] + cnt[1] < 32) {  // rows behind the last token, and tokens that are not in the cache
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (g + 8 * e >= cnt[mt]) {
                        lv[mt][e] = -INFINITY;
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) s[mt][nt][2 * e] = s[mt][nt][2 * e + 1] = (mt ? in.y : in.x) >> 16 ? __uint_as_float(0x7fffffffu) : -INFINITY;
                    }
        }
        float x1[NT][2];
        bool up = false;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int d = 0; d < 2; d++) {
                x1[nt][d] = fmaxf(fmaxf(s[0][nt][d] + lv[0][0], s[0][nt][2 + d] + lv[0][1]), fmaxf(s[1][nt][d] + lv[1][0], s[1][nt][2 + d] + lv[1][1])) - 15.f;
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) x1[nt][d] = fmaxf(x1[nt][d], __shfl_xor_sync(0xffffffffu, x1[nt][d], off));
                up |= x1[nt][d] > M[nt][d];
            }
        if (__any_sync(0xffffffffu, up)) {  // a larger maximum
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int d = 0; d < 2; d++) {
                    const float nm = fmaxf(M[nt][d], x1[nt][d]), f = M[nt][d] == -INFINITY ? 0.f : exp2_fast(M[nt][d] - nm);
                    M[nt][d] = nm;
#pragma unroll
                    for (int x = 0; x < X::CH; x++) o[x][nt][d] *= f, o[x][nt][2 + d] *= f;
                }
        }
        // ---- the denominator
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int d = 0; d < 2; d++) {
                const float nm = fmaxf(fmaxf(fmaxf(s[0][nt][d], s[0][nt][2 + d]), fmaxf(s[1][nt][d], s[1][nt][2 + d])), S[nt][d]);
                const float at = nm == -INFINITY ? 0.f : nm;  // (nothing so far: every score is -infinity, or a NaN)
                l[nt][d] = l[nt][d] * exp2_fast(S[nt][d] - at) + (exp2_fast(s[0][nt][d] - at) + exp2_fast(s[0][nt][2 + d] - at)) + (exp2_fast(s[1][nt][d] - at) + exp2_fast(s[1][nt][2 + d] - at));
                S[nt][d] = nm;
            }
        // ---- weights as B operands: [16 tokens][high parts of tokens 2t, 2t + 1, of 2t + 8, 2t + 9, then the remainders] of head g
        uint32_t p[2][NT][4];
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float wt[4];
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int d = 0; d < 2; d++) {
                        // (no weight so far: M is -infinity, and so is every score or its value's log2, or one is a NaN)
                        wt[2 * e + d] = exp2_fast(s[mt][nt][2 * e + d] - (M[nt][d] == -INFINITY ? 0.f : M[nt][d]) + lv[mt][e]);
                    }
                const __half2 h01 = __floats2half2_rn(wt[0], wt[1]), h23 = __floats2half2_rn(wt[2], wt[3]);
                const float2 f01 = __half22float2(h01), f23 = __half22float2(h23);
                const __half2 r01 = __floats2half2_rn(wt[0] - f01.x, wt[1] - f01.y), r23 = __floats2half2_rn(wt[2] - f23.x, wt[3] - f23.y);
                const int srcA = 8 * t + (g >> 1), srcB = srcA + 4;
                const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;
                auto to_b = [&](const __half2 &h) {
                    const uint32_t x = *(const uint32_t *)&h;
                    return __byte_perm(__shfl_sync(0xffffffffu, x, srcA), __shfl_sync(0xffffffffu, x, srcB), sel);
                };
                if (X::DUP) p[mt][nt][0] = to_b(t < 2 ? h01 : r01), p[mt][nt][1] = to_b(t < 2 ? h23 : r23);  // columns 4 to 7 are the same heads: their remainders
                else p[mt][nt][0] = to_b(h01), p[mt][nt][1] = to_b(h23), p[mt][nt][2] = to_b(r01), p[mt][nt][3] = to_b(r23);
            }
        if (!__all_sync(0xffffffffu, mbar_wait(&bars[VF + vl], n / VR & 1))) {
            ok = false;
            break;
        }
        // ---- values
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int hf = 0; hf < X::HALVES; hf++) {
                uint32_t w[4][4];  // tokens 2t, 2t + 1, 2t + 8, 2t + 9: 16 channels from 16 g (HD = 64: 8 from 8 g)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t row = mt * 16 + 2 * t + (e & 1) + (e >> 1) * 8;
                    if (HD == 64) lds64(w[e][0], w[e][1], Vb + vl * X::TILE + row * 64 + (((g >> 1) ^ t) << 4) + (g & 1) * 8);
                    else lds128(w[e], Vb + vl * X::TILE + hf * STEP * 128 + row * 128 + ((g ^ (2 * t + (e & 1))) << 4));
                }
                if (cnt[mt] < 16) {  // rows behind the last token may hold anything, and 0 times a code that is no number would reach every head
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (2 * t + (e & 1) + (e >> 1) * 8 >= cnt[mt]) w[e][0] = w[e][1] = w[e][2] = w[e][3] = 0;
                }
#pragma unroll
                for (int x = 0; x < X::LANE / 4; x++) {
                    uint32_t a0[4], a1[4];  // channels 4x, 4x + 1 and 4x + 2, 4x + 3 of the lane
                    kv8_operands<FMT>(__byte_perm(w[0][x], w[1][x], 0x5140), a0[0], a0[1]);
                    kv8_operands<FMT>(__byte_perm(w[2][x], w[3][x], 0x5140), a0[2], a0[3]);
                    kv8_operands<FMT>(__byte_perm(w[0][x], w[1][x], 0x7362), a1[0], a1[1]);
                    kv8_operands<FMT>(__byte_perm(w[2][x], w[3][x], 0x7362), a1[2], a1[3]);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float(&y0)[4] = o[hf * 8 + 2 * x][nt], (&y1)[4] = o[hf * 8 + 2 * x + 1][nt];
                        mma_f16(y0, a0, p[mt][nt][0], p[mt][nt][1], y0);
                        mma_f16(y1, a1, p[mt][nt][0], p[mt][nt][1], y1);
                        if (!X::DUP) {
                            mma_f16(y0, a0, p[mt][nt][2], p[mt][nt][3], y0);
                            mma_f16(y1, a1, p[mt][nt][2], p[mt][nt][3], y1);
                        }
                    }
                }
            }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[VE + vl]);
        if (task.w & 2) {  // ---- the chunk's totals
            const size_t at = (size_t)task.x * a.max_chunks + task.z;
            float *dst = a.part + (at * a.qh + task.y * a.G + 2 * t) * HD + X::LANE * g;
            float4 *st = stats_of(a, HD, task.x, task.y * a.G + 2 * t) + task.z;
            if (X::DUP) {
#pragma unroll
                for (int x = 0; x < X::CH; x++)
#pragma unroll
                    for (int z = 0; z < 4; z++) o[x][0][z] += __shfl_xor_sync(0xffffffffu, o[x][0][z], 2);
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int d = 0; d < 2; d++) {
                    float sm = S[nt][d];
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) sm = fmaxf(sm, __shfl_xor_sync(0xffffffffu, sm, off));
                    float lt = S[nt][d] == -INFINITY ? l[nt][d] : l[nt][d] * exp2_fast(S[nt][d] - sm);  // (0 or a NaN where there is no score)
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) lt += __shfl_xor_sync(0xffffffffu, lt, off);
                    if (nt * 8 + 2 * t + d >= a.G) continue;
                    if (g == 0) st[(nt * 8 + d) * a.max_chunks] = make_float4(M[nt][d], sm, lt, 0.f);
#pragma unroll
                    for (int hf = 0; hf < X::HALVES; hf++)
#pragma unroll
                        for (int x = 0; x < X::LANE / 4; x++) {
                            const float(&y0)[4] = o[hf * 8 + 2 * x][nt], (&y1)[4] = o[hf * 8 + 2 * x + 1][nt];
                            *(float4 *)(dst + (nt * 8 + d) * HD + hf * 128 + 4 * x) = make_float4(y0[d], y0[2 + d], y1[d], y1[2 + d]);
                        }
                }
        }
    }
    if (!ok) {
        if (lane == 0) set_status(status, ST_MBAR_TIMEOUT | 0x23);
        void_share(c, a, first, FEW ? warp * gridDim.x + blockIdx.x : blockIdx.x * X::WARPS + warp, gridDim.x * X::WARPS, HD);
    }
}

// ------------------------------------------------------------------------------------------------ join
// 64 channels of a (head, row): two channels per lane.  A warp takes 32 chunks at a time, a lane knows one chunk's weight (within the 32: relative to their
// maximum) and every load leaves before the weights are known; the 32 are added in order, then joined with what the warp has.  W warps take every Wth 32 and are
// joined in order, so a row's result depends on its own chunks alone, and up to 32 chunks W does not matter.  Rows of length 0 get their zeros here.
// Bound: the latency of a few loads one after the other.  W = 1 for calls of up to 32 chunks (2048 (head, row) pairs of up to 32 chunks: 16 us in blocks of 256 threads
// per 64 channels, 8 this way), W = 4 for longer ones.  grid (8 / W) (head, row, 64 channels) per block of 256 (W = 1) or 1 per block of 128
template <int HD, class T, int W>
__global__ void __launch_bounds__(W == 1 ? 256 : 32 * W) kv8_merge_k(Kv8Dev c, AttnArgs a) {
    __shared__ float2 part[W][32];
    __shared__ float stat[W][3];
    pdl_sync();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, x = W == 1 ? blockIdx.x * 8 + warp : blockIdx.x;
    const uint32_t ch = x % (HD / 64) * 64 + 2 * lane, y = x / (HD / 64), r = y / a.qh, qh = y % a.qh;
    if (r >= a.nb) return;
    const int len = a.lens[r], slot = a.slots[r];
    if (slot < 0) return;
    const uint32_t nch = chunks_in(row_tokens(c, a, slot, len));
    const float4 *st = stats_of(a, HD, r, qh);
    const float *p = a.part + ((size_t)r * a.max_chunks * a.qh + qh) * HD + ch;
    const uint32_t cs = a.qh * HD;
    float2 gate = make_float2(0.f, 0.f);
    if (a.gate && warp % W == 0) {
        const T *gp = (const T *)a.gate + (int64_t)r * a.g_row + (int64_t)qh * a.g_head + ch;
        gate = make_float2(kv8_float(gp[0]), kv8_float(gp[1]));
    }
    bool over = false;  // the core reads as many entries of a list as the row has blocks: further ones name none of them
    if (a.blocks && nch && warp % W == 0) {
        const int32_t *list = a.blocks + ((size_t)r * c.kvh + qh / a.G) * a.nblocks;
#pragma unroll 8
        for (uint32_t i = (min((uint32_t)len, a.max_len) + c.block - 1) / c.block + lane; i < a.nblocks; i += 32) over |= __ldcg(list + i) >= 0;
        over = __any_sync(0xffffffffu, over);
        if (over && lane == 0) set_status(c.status, ST_BAD_ARG | 0x23);
    }
    Sums x0 = {-INFINITY, -INFINITY, 0.f, make_float2(0.f, 0.f)};
    for (uint32_t k0 = W == 1 ? 0 : 32 * warp; k0 < nch; k0 += 32 * W) {
        const float4 s = k0 + lane < nch ? __ldcg(st + k0 + lane) : make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
        float2 v[32];
#pragma unroll
        for (uint32_t k = 0; k < 32; k++) v[k] = k0 + k < nch ? __ldcg((const float2 *)(p + (size_t)(k0 + k) * cs)) : make_float2(0.f, 0.f);
        const float M = warp_max(s.x), S = warp_max(s.y), w = s.x == -INFINITY ? 0.f : exp2f(s.x - M);
        const float l = warp_sum(s.y == -INFINITY ? s.z : s.z * exp2f(s.y - S));  // (0, or NaN, where a chunk has no maximum)
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (uint32_t k = 0; k < 32; k++) {
            const float wk = __shfl_sync(0xffffffffu, w, k);
            sum.x = __fadd_rn(sum.x, __fmul_rn(v[k].x, wk));
            sum.y = __fadd_rn(sum.y, __fmul_rn(v[k].y, wk));
        }
        join(x0, M, S, l, sum);
    }
    if (W > 1) {
        part[warp % W][lane] = x0.acc;
        if (lane == 0) stat[warp % W][0] = x0.M, stat[warp % W][1] = x0.S, stat[warp % W][2] = x0.l;
        __syncthreads();
        if (warp) return;
#pragma unroll
        for (int i = 1; i < W; i++) join(x0, stat[i][0], stat[i][1], stat[i][2], part[i][lane]);
    }
    const bool longer = len > 0 && (uint32_t)len > a.max_len, bad = longer || over;
    if (longer && lane == 0) set_status(c.status, ST_BAD_ARG | 0x24);
    // a sum of nothing: no token, or scores of minus infinity alone
    const bool none = x0.l == 0.f && (nch == 0 || (a.blocks && __ldcg(a.blocks + ((size_t)r * c.kvh + qh / a.G) * a.nblocks) < 0));
    const float f = bad || (x0.l == 0.f && !none) ? __uint_as_float(0x7fffffffu) : none ? 0.f : exp2f(x0.M - x0.S) / x0.l;
    float out[2] = {x0.acc.x * f, x0.acc.y * f};
    if (a.gate && !none) out[0] *= 1.f / (1.f + expf(-gate.x)), out[1] *= 1.f / (1.f + expf(-gate.y));  // (no token: zero, whatever the gate)
    kv8_store<2>((T *)a.y + (int64_t)r * a.y_row + (int64_t)qh * a.y_head + ch, out);
}

// Which kernel: by the format, the type of rows, and whether 8 or 16 heads share a kv head.
typedef void (*core_kernel)(CUtensorMap, Kv8Dev, AttnArgs, uint32_t, unsigned *);
typedef void (*merge_kernel)(Kv8Dev, AttnArgs);
struct Launch {
    core_kernel core;
    merge_kernel merge, merge_few;  // of more than 32 chunks, of up to 32
    int smem, threads;  // shared memory but for 12 bytes per row
};
template <int HD, int FMT, class T, int MODE, bool FEW>
Launch launch_of() {
    return {kv8_attn_k<HD, FMT, T, MODE, FEW>, kv8_merge_k<HD, T, 4>, kv8_merge_k<HD, T, 1>, Core<HD, MODE, FEW>::BYTES, Core<HD, MODE, FEW>::THREADS};
}
template <int HD, int FMT, class T>
Launch launch_of(uint32_t G, bool few) {
    if (few) return G > 8 ? launch_of<HD, FMT, T, 2, true>() : G > 4 ? launch_of<HD, FMT, T, 1, true>() : launch_of<HD, FMT, T, 0, true>();
    return G > 8 ? launch_of<HD, FMT, T, 2, false>() : G > 4 ? launch_of<HD, FMT, T, 1, false>() : launch_of<HD, FMT, T, 0, false>();
}
template <int HD>
Launch launch_of(uint32_t format, uint32_t dtype, uint32_t G, bool few) {
    if (format == QW_KV8_E4M3) return dtype == QW_KV8_FP16 ? launch_of<HD, QW_KV8_E4M3, __half>(G, few) : launch_of<HD, QW_KV8_E4M3, __nv_bfloat16>(G, few);
    return dtype == QW_KV8_FP16 ? launch_of<HD, QW_KV8_INT8, __half>(G, few) : launch_of<HD, QW_KV8_INT8, __nv_bfloat16>(G, few);
}
Launch launch_of(uint32_t hd, uint32_t format, uint32_t dtype, uint32_t G, bool few) {
    return hd == 64 ? launch_of<64>(format, dtype, G, few) : hd == 128 ? launch_of<128>(format, dtype, G, few) : launch_of<256>(format, dtype, G, few);
}

uint32_t chunks_of(const qw_kv8_cache *c, uint32_t max_len, uint32_t nblocks) {
    const uint64_t blocks = ((uint64_t)max_len + c->block - 1) / c->block;
    const uint64_t n = nblocks ? (nblocks < blocks ? nblocks : blocks) * c->block : max_len;
    // the most chunks of a row of up to n tokens: a longer row may have fewer, at the steps of chunk_of
    const uint32_t m = (uint32_t)(n < 0xffffff00u ? n : 0xffffff00u);
    uint32_t most = chunks_in(m);
    for (uint32_t e : {512u, 2048u, 65536u})
        if (e < m && chunks_in(e) > most) most = chunks_in(e);
    return most;
}
const char *check_shape(const qw_kv8_cache *c, uint32_t nb, uint32_t qh, uint32_t max_len) {
    if (nb < 1 || nb > KV8_MAX_ROWS) return "a call has 1 to 1024 rows";
    if (qh < c->kvh || qh % c->kvh || qh / c->kvh > 16) return "1 to 16 query heads share a kv head";
    if (qh > 65535) return "too many query heads";
    if ((double)nb * c->kvh * ((double)max_len / 32 + 1) > 2147483647.0) return "more tokens than one call takes";
    if (max_len < 1 || (uint64_t)max_len > (uint64_t)c->max_pages * KV8_PAGE) return "max_len is 1 to 256 max_pages";
    return nullptr;
}
// Without blocks: enough for lists of blocks as well, whose last block may reach beyond max_len.
size_t work_of(const qw_kv8_cache *c, uint32_t nb, uint32_t qh, uint32_t max_len, uint32_t nblocks) {
    if (!nblocks) nblocks = (uint32_t)(((uint64_t)max_len + c->block - 1) / c->block);
    return (size_t)nb * chunks_of(c, max_len, nblocks) * qh * (c->hd + 4) * 4;
}
// 0, or -1 / -2 with a message
int check_attn(const qw_kv8_cache *c, const qw_kv8_attn_args *a, const char **m) {
    if (!a) return *m = "no arguments", -1;
    if ((*m = kv8_check_layer(c, a->nb, a->layer, a->dtype)) || (*m = check_shape(c, a->nb, a->qh, a->max_len))) return -1;
    if (!a->q || !a->y || !a->lens || !a->slots || !a->work) return *m = "null pointer argument", -1;
    if (a->blocks && a->nblocks < 1) return *m = "chosen blocks of no number", -1;
    if (a->blocks && a->nblocks > KV8_MAX_BLOCKS) return *m = "a list holds at most 2^31 - 1 blocks", -1;
    const void *ptrs[] = {a->q, a->gate, a->y, a->lens, a->slots, a->blocks};
    if (!kv8_aligned(3, 3, ptrs)) return *m = "a tensor does not start at a boundary of its type", -1;
    if (kv8_overlap(a->nb, a->qh, c->hd, a->y_row, a->y_head)) return *m = "results that lie on one another", -1;
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
    const uint64_t most = (uint64_t)a->nb * mc * c->kvh, sms = (uint64_t)kv8_sm_count();
    const Launch L = launch_of(c->hd, c->format, a->dtype, k.G, most <= 6 * sms);
    const int smem = L.smem + (int)a->nb * 12;
    // (the most of any call: another thread's call, or a captured one, may be of more rows than this)
    cudaError_t e = cudaFuncSetAttribute(L.core, cudaFuncAttributeMaxDynamicSharedMemorySize, L.smem + 12 * KV8_MAX_ROWS);
    if (e != cudaSuccess) return e;
    e = qw_launch(L.core, (uint32_t)(most < sms ? most : sms), L.threads, smem, st, tm, d, k, box_rows, status);
    if (e != cudaSuccess) return e;
    const uint32_t units = a->nb * a->qh * (c->hd / 64);  // (at most 2^28)
    if (mc <= 32) return qw_launch(L.merge_few, (units + 7) / 8, 256, 0, st, d, k);
    return qw_launch(L.merge, units, 128, 0, st, d, k);
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
