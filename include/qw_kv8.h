/* qw_kv8.h -- an 8-bit paged key-value cache and the attention that reads it: the operators beside qsa_prep / qsa_attn / qsa_merge
 * for hosts that want half the bytes per token, other head layouts, or attention over chosen blocks of a long context.  No counterpart in the
 * reference's src/gpu.h.
 *
 * Pages hold 256 tokens, as the fp16 cache's do.  A row is one token's key or value of one kv head:
 *   a = max |x|;  scale = a / F;  code = nearest(x * (F / a))      F = 448 (e4m3) or 127 (int8), every operation rounded to fp32
 * and code * scale is what the row stands for.  A row whose a is below 2^-100 is stored as zeros with scale 0; one that holds an infinity or a NaN
 * gets scale NaN, so that whatever attends to it turns NaN.  A host that writes codes itself does not use the e4m3 codes 0x7f and 0xff, nor infinite or
 * negative scales, in rows that are looked at; rows behind a slot's last token may hold anything.
 *
 * All pointers are device pointers of the device that is current and that `stream` (a cudaStream_t) belongs to; buffers of another device are
 * refused.  Calls only enqueue work: they do not allocate, do not wait and may be captured into a CUDA graph.  Calls that share a workspace
 * or write the same rows have to be ordered by their stream, or by events; this holds for captured graphs too.
 * Return values: 0, or a negative code with a message in err (-1: bad argument, -2: the workspace is too small, -3: CUDA error); on an error
 * nothing was enqueued, unless the code is -3.
 *
 * Slots, positions and page ids are device data, so the kernels check them: a slot or page outside the cache is never read or written; the row's
 * results are NaN (put: the row is dropped; pick: -1), and the word at `status`, if there is one, becomes 0x200 | n.  Attention whose copies do not arrive
 * within two seconds gives up: the rows concerned are NaN, and the word becomes 0x100 | n.
 */
#ifndef QW_KV8_H
#define QW_KV8_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { QW_KV8_E4M3 = 0, QW_KV8_INT8 = 1 }; /* format of the codes */
enum { QW_KV8_FP16 = 0, QW_KV8_BF16 = 1 }; /* type of rows outside the cache */

typedef struct {
    uint8_t *codes;            /* [pages][layers][K, V][kvh][256][hd], 16-byte aligned */
    float *scales;             /* [pages][layers][K, V][kvh][256], 16-byte aligned */
    uint8_t *bounds;           /* NULL, or [pages][layers][kvh][256 / block][2 hd + 16], 16-byte aligned: lo int8[hd], hi int8[hd], fp32 scale, 12 unused */
    const int32_t *page_table; /* [slots][max_pages] page ids; entries past a slot's tokens are never looked at */
    uint32_t *status;          /* NULL, or a word the device can write */
    uint32_t pages, layers, kvh; /* at most 32767 kv heads, and 2^31 - 1 rows: pages * layers * 2 * kvh * 256 */
    uint32_t hd;               /* 64, 128 or 256 */
    uint32_t format, block;    /* block: tokens per block of bounds and of chosen blocks: 16, 32, 64, 128 or 256 */
    uint32_t slots, max_pages;
} qw_kv8_cache;

/* Bytes of the three buffers: out[0] codes, out[1] scales, out[2] bounds.  0 or -1 (bad sizes). */
int qw_kv8_bytes(const qw_kv8_cache *c, size_t out[3]);

/* Row r (of nb <= 1024) goes to / comes from position pos[r] of slot slots[r]; rows with a negative slot or position are skipped (get: the output row
 * stays as it was).  k and v: [nb][kvh][hd] with these strides in elements, of any alignment; a row's hd values are contiguous. */
typedef struct {
    void *k, *v;
    const int32_t *slots, *pos; /* [nb] */
    int64_t k_row, k_head, v_row, v_head;
    uint32_t nb, layer, dtype, reserved;
} qw_kv8_rows;

/* Quantises the rows into the cache.  Of two rows for the same position the later one stays (two slots that share a page are not
 * both written through in one call).  Where the cache has bounds, those of every block that
 * got a row are computed anew from the block's tokens up to the newest one written:
 *   lo = min, hi = max per channel of code * scale;  b = max |lo|, |hi|;  scale = b / 127;
 *   lo8 = max(-127, floor(lo * (127 / b))), hi8 = min(127, ceil(hi * (127 / b)));  scale +infinity if a row of the block has scale NaN
 * so a block's tokens are to be written in order (or together). */
int qw_kv8_put(const qw_kv8_cache *c, const qw_kv8_rows *a, void *stream, char *err, size_t errlen);
/* Reads rows back: code * scale, rounded to the rows' type.  No two results share memory; k and v of different strides do not lie between one another either. */
int qw_kv8_get(const qw_kv8_cache *c, const qw_kv8_rows *a, void *stream, char *err, size_t errlen);

/* Attention of one new token per row over its slot's first lens[r] tokens: y = sum_t softmax_t(scale * q . k_t) v_t for each of the qh query heads
 * (qh / kvh = 1 .. 16 of them share a kv head, as consecutive ones), times sigmoid(gate) where there is a gate.  A row of length 0 is zero, whatever its
 * gate and its list of blocks hold; a row with a negative slot stays as it was.  With `blocks` ([nb][kvh][nblocks]: up to 2^31 - 1 distinct block numbers in any
 * order, then only negative ones, as pick leaves them) the tokens are those of the named blocks; a number beyond the row's last block makes the kv head's results
 * NaN, wherever it stands in the list.  An infinity or a NaN in a query makes its head's result NaN; so does a score beyond fp32's range, unless it is a
 * negative one beside others within it.
 * y shares no memory with what the call reads, but it may be q itself, or the gate itself.
 * max_len: no row is longer (a longer one is answered with NaN).  What a row yields does not depend on the other rows of the call.
 * work: qw_kv8_attn_work(...) bytes, 16-byte aligned, nothing has to be in it. */
typedef struct {
    const void *q, *gate; /* [nb][qh][hd]; gate may be NULL */
    void *y;              /* [nb][qh][hd] */
    const int32_t *lens, *slots; /* [nb] */
    const int32_t *blocks;       /* NULL, or the chosen blocks */
    void *work;
    size_t work_bytes;
    int64_t q_row, q_head, gate_row, gate_head, y_row, y_head; /* strides in elements */
    float scale;                 /* usually hd^-1/2 */
    uint32_t nb, layer, dtype, qh, max_len, nblocks, reserved;   /* nb <= 1024 */
} qw_kv8_attn_args;
int qw_kv8_attn(const qw_kv8_cache *c, const qw_kv8_attn_args *a, void *stream, char *err, size_t errlen);
/* Workspace of attention over up to max_len tokens; with nblocks, over that many blocks only (one for nblocks = 0 serves every list of blocks too).  0 for
 * sizes the call would refuse. */
size_t qw_kv8_attn_work(const qw_kv8_cache *c, uint32_t nb, uint32_t qh, uint32_t max_len, uint32_t nblocks);

/* The blocks of a row's context that are worth attending to, per kv head:  q8 = nearest(q * (127 / max |q|)), sq = max |q| / 127 per query head;
 *   score(block) = max over the kv head's query heads of  (sq * scale) * sum_d (max(q8, 0) hi8 + min(q8, 0) lo8)
 * an upper bound of q . k within the block up to the rounding of q, with a sum of whole numbers (the same whatever its order) and two fp32 products.
 * The first `first` and the last `last` blocks are always among them, then those of the highest scores, of equal ones the lowest number;
 * blocks: [nb][kvh][nblocks] block numbers in ascending order, -1 behind the last.  Needs a cache with bounds. */
typedef struct {
    const void *q;                /* [nb][qh][hd] */
    const int32_t *lens, *slots;  /* [nb] */
    int32_t *blocks;
    void *work;                   /* qw_kv8_pick_work(...) bytes, 16-byte aligned */
    size_t work_bytes;
    int64_t q_row, q_head;
    uint32_t nb, layer, dtype, qh, max_len, nblocks, first, last; /* first + last <= nblocks */
} qw_kv8_pick_args;
int qw_kv8_pick(const qw_kv8_cache *c, const qw_kv8_pick_args *a, void *stream, char *err, size_t errlen);
size_t qw_kv8_pick_work(const qw_kv8_cache *c, uint32_t nb, uint32_t max_len);

/* The same operators in a batch (qw_gpu.h): families kv8_put, kv8_get, kv8_attn, kv8_pick.  Binds 0 = codes, 1 = scales, 2 = bounds (may be absent for
 * get and attn, and for put), 3 = page table, 15 = the sizes as one qw_kv8_sizes; the buffers' sizes are checked.
 *   put, get: 4 = k, 5 = v, 6 = slots, 7 = pos, 8 = the strides k_row, k_head, v_row, v_head (int64 each)
 *   attn:     4 = q, 5 = gate (may be absent), 6 = y, 7 = lens, 8 = slots, 9 = blocks (may be absent), 10 = workspace, 11 = the strides q_row, q_head,
 *             gate_row, gate_head, y_row, y_head
 *   pick:     4 = q, 7 = lens, 8 = slots, 9 = blocks, 10 = workspace, 11 = the strides q_row, q_head
 * The grid given to the dispatch is not used.  A slot or page outside the cache makes the batch fail. */
typedef struct {
    uint32_t pages, layers, kvh, hd, format, block, slots, max_pages;
    uint32_t nb, layer, dtype, qh, max_len, nblocks, first, last;
    float scale;
} qw_kv8_sizes;

/* Where row (page, layer, K or V, head, token) starts, in rows of hd codes or in scales, and whether the kernels would touch it: the index of the row,
 * or -1 for what lies outside the cache.  Host arithmetic only (for hosts that move pages, and for tests). */
int64_t qw_kv8_row_index(const qw_kv8_cache *c, int64_t slot, int64_t pos, int64_t page, uint32_t layer, uint32_t kv, uint32_t head);

#ifdef __cplusplus
}
#endif
#endif
