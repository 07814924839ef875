/*
 * efm_b200_kv4.h -- operators of a key/value cache held in 4 bits (same library as efm_b200.h, same rules: plain C types, integer
 * status, message in efm_b200_last_error(NULL), no exceptions, no CPU path).
 *
 * For callers whose cache has to stay inside a fixed footprint: rows are appended in 4 bits (3.6 times as many as in 16), attention
 * reads them as they are and can sum every cached row's attention weights, and a cache that ran full is brought back to a budget by
 * those sums.  The operators stand beside efm_b200_op_decode_attention / _prefill_attention and take caller-owned device buffers;
 * unlike those they run on the given stream and return at once: nothing is allocated, copied to the host or waited for, so that a
 * step of them can be captured into a CUDA graph and replayed -- lengths, page numbers and row counts are read on the device.
 *
 * Pages.  A page holds 64 rows of one sequence; its tile for one kv head holds, in this order,
 *     key codes 64 x D/2 bytes | key parameters 64 x D/64 x {scale, min} fp16 | value codes | value parameters (the same sizes).
 * A group is 64 neighbouring channels of a row and head; a channel stands for min + scale * code, computed in fp32.  Of x:
 *     NaN counts as 0, anything beyond +-65504 as +-65504;  scale = fp16((max - min) * (1/15)), min = fp16(min), maximum and minimum of the group;
 *     code = rint((x - min) / scale), ties to even, clamped to 0 .. 15;  scale 0: code 0.
 * The rounding of min and scale may take a value up to 80 beyond 65504; as fp16 (outputs of that type, and where attention has many rows,
 * v and without mass k) it is 65504.
 * Eight channels c0 .. c7 share a 32-bit word, as nibbles c0 c2 c4 c6 c1 c3 c5 c7 from the lowest bits up.  Words of a value row are in
 * the order of the channels; the words of a key row (G = D/64 groups) in the order [quarter of a group 0..3][group 0..G-1][word 0..1].
 * Pages of a sequence are any pool pages; page k of its page_table row holds cache rows [64 k, 64 k + 64).
 *
 * Every pointer is device memory of one GPU (pool's; the call runs there whatever the current device is), pool, q, k, v and their
 * outputs on 16-byte boundaries, the rest on those of their elements.  Buffers of one call must not overlap unless a field says so.
 * Work on the buffers has to be ordered with the call through its stream.
 */
#ifndef EFM_B200_KV4_H_
#define EFM_B200_KV4_H_

#include "efm_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { EFM_KV4_PAGE_ROWS = 64, EFM_KV4_GROUP = 64 };
/* rotation: channel i turns with channel i + rot_dims / 2, or with its neighbour */
enum { EFM_KV4_ROT_HALVES = 0, EFM_KV4_ROT_NEIGHBOURS = 1 };
/* bits of *status; the calls only ever set them */
enum {
    EFM_KV4_BAD_PAGE = 1,     /* a page number outside [0, n_pages): its rows are not written, and count as absent when read */
    EFM_KV4_FULL = 2,         /* append: a sequence has no more page_table columns; the row is dropped and not counted */
    EFM_KV4_BAD_COUNT = 4,    /* a length or row count beyond what the call was given (max_len, max_new, max_rows) or negative: cut to it; where
                               * cu_rows falls, append takes its running maximum, so that a row stays with the first sequence that names it */
    EFM_KV4_WAIT = 8          /* attention: a bounded wait for a copy or product inside a kernel gave up; out is void, mass_out has what it had
                               * or, row by row, the whole sum */
};

typedef struct efm_kv4_cache {
    int32_t struct_size;          /* = sizeof(efm_kv4_cache) */
    int32_t dtype;                /* of q, k, v and the outputs: EFM_BF16 or EFM_F16 */
    int32_t q_heads, kv_heads;    /* q_heads a multiple of kv_heads, <= 1024 */
    int32_t head_dim;             /* 64 or 128 */
    int32_t n_pages;              /* pages in pool, <= 2^24 */
    int32_t batch;                /* sequences of the call, >= 1, <= 65535 */
    int32_t max_pages;            /* columns of page_table, >= 1, < 2^24 */
    void* pool;                   /* [n_pages, kv_heads, efm_b200_kv4_tile_bytes] */
    const int32_t* page_table;    /* [batch, max_pages]; columns behind a sequence's rows are not read */
    int32_t* status;              /* one word, EFM_KV4_* bits are or-ed in; may be NULL */
} efm_kv4_cache;

/* bytes of a tile: 4608 (head_dim 64) or 9216 (128) */
EFM_API efm_status efm_b200_kv4_tile_bytes(int32_t head_dim, int64_t* bytes);

/* New rows of a batch: rows cu_rows[b] .. cu_rows[b + 1] - 1 of q, k and v belong to sequence b (rows behind cu_rows[batch] are left
 * alone, in every output).  Each head of q and k is normed, turned, and q rounded to q_out; k (from its fp32 value) and v go into
 * the cache rows from lens_in[b] on. */
typedef struct efm_kv4_append {
    int32_t struct_size;
    int32_t max_rows;             /* rows the buffers hold; 0: only lens_out is written */
    const int32_t* cu_rows;       /* [batch + 1], ascending from 0 */
    const int32_t* lens_in;       /* [batch] rows held before the call */
    int32_t* lens_out;            /* [batch] and after it; not the same buffer as lens_in */
    const void *q, *k, *v;        /* [max_rows] rows of heads x head_dim; q may be NULL (keys and values only) */
    int64_t q_stride, k_stride, v_stride;   /* elements from row to row, multiples of 8, at least heads x head_dim */
    int32_t norm;                 /* 1: x / sqrt(mean(x^2) + norm_eps) * weight over the head's channels; 0: none */
    float norm_eps;
    const void *q_norm, *k_norm;  /* [head_dim] weights, NULL: 1 */
    int32_t rot_dims;             /* leading channels that turn, a multiple of 16; 0: none */
    int32_t rot_kind;             /* EFM_KV4_ROT_* */
    int32_t axes;                 /* 1, or 3: pairs [0, sections[0]) turn by positions[0], the next sections[1] by positions[1], ... */
    int32_t sections[3];          /* sum = rot_dims / 2 when axes = 3 */
    const double* inv_freq;       /* [rot_dims / 2] radians a position; angles, sines and cosines are taken in 64 bits */
    const int32_t* positions;     /* [axes, max_rows] */
    const int32_t* token_index;   /* [max_rows] running numbers of the tokens, for eviction; NULL: the cache row */
    void* q_out;                  /* [max_rows, q_heads, head_dim] */
    void *k_held, *v_held;        /* [max_rows, kv_heads, head_dim] what the cache now holds, rounded once; NULL: not wanted */
    int32_t* index;               /* [n_pages, kv_heads, 64] token numbers of the cached rows, NULL: not kept */
    float* mass;                  /* [n_pages, kv_heads, 64] summed weights, set to 0 for the new rows; NULL: not kept */
} efm_kv4_append;

/* Attention of new rows over the cache, which holds them already: row i of a sequence's n new rows sees its cache rows
 * [0, lens[b] - n + i].  out = softmax(scale q k^T) v; a row that sees nothing gets zeros.  Outputs are rounded once.  Before that, for EFM_BF16,
 * weights are rounded to fp16, and where a sequence has many new rows v, and without mass k, too: out may differ in its last bits with and
 * without mass.  Everything else, and all of it for EFM_F16, has 22 bits or more. */
typedef struct efm_kv4_attention {
    int32_t struct_size;
    int32_t max_rows;
    int32_t max_new;              /* most new rows of one sequence */
    int32_t max_len;              /* most cache rows of one sequence (sizes the split of the work); 0: 64 x max_pages */
    const int32_t *cu_rows, *lens;
    const void* q;                /* [max_rows, q_heads, head_dim] */
    void* out;                    /* the same */
    float scale;                  /* > 0 */
    int32_t reserved;
    const float* mass_in;         /* [n_pages, kv_heads, 64]; both or neither */
    float* mass_out;              /* mass_in + the row's weights, summed over the new rows and the q heads of its kv head, for all rows held; may be mass_in */
    void* workspace;              /* for this call alone while it runs; contents do not matter */
    int64_t workspace_bytes;
} efm_kv4_attention;

/* Sequences that hold more than `limit` rows are brought down to `budget`, each kv head by itself.  Kept first are rows with a token
 * number below keep_first or above the head's newest number - keep_last, then those with the largest mass (NaN lowest); equal ones by
 * lower row.  Kept rows below `budget` stay where they are; those behind move into the free rows, both in ascending order.  index and
 * mass move with them. */
typedef struct efm_kv4_evict {
    int32_t struct_size;
    int32_t budget;               /* >= 1 */
    int32_t limit;                /* >= budget */
    int32_t keep_first, keep_last;
    int32_t reserved;
    const int32_t* lens_in;
    int32_t* lens_out;            /* not the same buffer as lens_in */
    const int32_t* index_in;
    int32_t* index_out;           /* rows below lens_out are written; may be index_in */
    const float* mass_in;
    float* mass_out;              /* may be mass_in */
    void* workspace;
    int64_t workspace_bytes;
} efm_kv4_evict;

/* Rows [first, first + rows) of every sequence as values, rounded once: [batch, rows, kv_heads, head_dim], the layout of the 16-bit
 * attention entry points.  Rows a sequence does not hold are left alone.  k_out or v_out may be NULL. */
typedef struct efm_kv4_read {
    int32_t struct_size;
    int32_t first, rows;
    int32_t reserved;
    const int32_t* lens;
    void *k_out, *v_out;
} efm_kv4_read;

/* workspace bytes the calls below need for these sizes (the pointers in the structs are not looked at) */
EFM_API efm_status efm_b200_kv4_attention_workspace(const efm_kv4_cache* cache, const efm_kv4_attention* a, int64_t* bytes);
EFM_API efm_status efm_b200_kv4_evict_workspace(const efm_kv4_cache* cache, const efm_kv4_evict* a, int64_t* bytes);

/* stream: cudaStream_t, NULL the default one */
EFM_API efm_status efm_b200_op_kv4_append(const efm_kv4_cache* cache, const efm_kv4_append* a, void* stream);
EFM_API efm_status efm_b200_op_kv4_attention(const efm_kv4_cache* cache, const efm_kv4_attention* a, void* stream);
EFM_API efm_status efm_b200_op_kv4_evict(const efm_kv4_cache* cache, const efm_kv4_evict* a, void* stream);
EFM_API efm_status efm_b200_op_kv4_read(const efm_kv4_cache* cache, const efm_kv4_read* a, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* EFM_B200_KV4_H_ */
