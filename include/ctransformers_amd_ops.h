/* Operators on device memory: a KV cache held in 4 bits, in pages that several sequences may share.  Not part of the reference ABI.
 * ctransformers_amd/ops.py calls these with torch tensors; a handle created with CT_AMD_KV=q4 runs its own attention on the same kernels.
 *
 * Conventions.  Every pointer but `stream` (a hipStream_t, NULL: the default stream) names memory of the CURRENT device.  A call only queues work on `stream`
 * and returns 0, or -1; ctamd_ops_error() says why, per thread: arguments are refused before anything is queued, a launch that the runtime refuses ends the call there.  Nothing is kept between calls and no call allocates, copies to the host or waits,
 * so all of them can be captured into a graph; two calls at once need two workspaces.
 *
 * Row types: 0 fp16, 1 bf16, 2 fp32.  Strides count elements.  A cache is
 *   pages   [n_pages] pages of ctamd_kv4_page_bytes() bytes, page_stride bytes apart, 16-byte aligned
 *   table   int32 [n_seq][table_stride]: the first table_width entries of a row name the sequence's pages in order; an entry outside [0, n_pages) names none:
 *           rows for it are not stored, and attention treats its tokens as absent
 *   lens    int32 [n_seq]: tokens of each sequence INCLUDING the rows of this call
 *   cu      int32 [n_seq + 1], ascending: sequence b's rows are the packed rows cu[b] .. cu[b + 1] - 1, its last positions; NULL: one sequence, all rows
 * max_rows: no sequence has more rows than this (rows beyond it are not processed).  head_dim: a multiple of 8 up to 256; page_tokens: 32, 64, 128 or 256.
 * No two sequences of one append may write the same page (ctamd_kv_reserve sees to that). */
#ifndef CTRANSFORMERS_AMD_OPS_H_
#define CTRANSFORMERS_AMD_OPS_H_
#ifdef __cplusplus
extern "C" {
#endif
const char* ctamd_ops_error(void);
/* 1 if "device memory" of this build is host memory (the CPU emulation of the test suite), else 0 */
int ctamd_ops_host_memory(void);
/* bytes of a page, 0 where the sizes are not supported */
long long ctamd_kv4_page_bytes(int n_head_kv, int head_dim, int page_tokens);

typedef struct {
    void* pages;
    const int* table;
    const int* lens;
    const int* cu;
    long long page_stride;
    int n_pages, table_stride, table_width, n_seq, total, n_head_kv, head_dim, page_tokens, max_rows;
} ctamd_kv4_cache;
typedef struct {
    void* p;
    long long row, head, dim;   /* strides of [total][heads][head_dim] */
    int type;
} ctamd_rows;
/* Quantizes K and V rows [total][n_head_kv][head_dim] into the pages.  A token whose K or V of a head holds a NaN makes every row that sees it NaN. */
int ctamd_kv4_append(const ctamd_kv4_cache* cache, const ctamd_rows* k, const ctamd_rows* v, void* stream);
/* The last rows of every sequence as numbers (0 where there is no page or no position).  No two elements of k and v are the same memory. */
int ctamd_kv4_read(const ctamd_kv4_cache* cache, const ctamd_rows* k, const ctamd_rows* v, void* stream);
/* Causal attention of rows [total][n_head][head_dim] over the cache: row i of a sequence with n rows sees positions 0 .. lens - n + i; a row that sees nothing
 * becomes 0.  n_head is a multiple of n_head_kv, dims of q are adjacent (q.dim == out.dim == 1), scale is finite; out may be q itself, but shares no
 * memory with anything else, and no two of its elements are the same memory.  Rows that belong to no sequence are left as they are.
 * ws: ctamd_kv4_attention_ws() floats (a function of the sizes and the current device, 0 if none are wanted), 16-byte aligned. */
long long ctamd_kv4_attention_ws(const ctamd_kv4_cache* cache, int n_head);
int ctamd_kv4_attention(const ctamd_kv4_cache* cache, int n_head, const ctamd_rows* q, const ctamd_rows* out, float scale, float* ws, long long ws_floats,
                        void* stream);

/* Page bookkeeping in device memory.  refs: int32 [n_pages], references to each page (0: free).  Outputs are separate memory: a call whose output overlaps an input
 * is refused. */
typedef struct {
    const int* table;   /* [n_seq][width], dense */
    const int* lens;    /* [n_seq] */
    const int* refs;    /* [n_pages] */
    int* table_out;
    int* lens_out;
    int* refs_out;
    int n_seq, width, n_pages, page_tokens;
} ctamd_kv_tables;
/* New sequence i of n_new shares the pages of parents[i], those of its first keep[i] tokens (keep NULL: all); a parent outside [0, n_seq) makes it empty (-1 frees a
 * sequence).  table_out [n_new][width], lens_out [n_new]. */
int ctamd_kv_fork(const ctamd_kv_tables* t, const int* parents, const int* keep, int n_new, void* stream);
/* Room for add[s] more tokens: lens_out = lens + add, the pages for them taken lowest free first in the order of the sequences, and a shared last page that will be
 * written is copied (pages [layers] x layer_stride bytes of n_pages pages of page_bytes, a multiple of 16).  *status: 0; or the pages that were missing, or -1 where a
 * sequence would outgrow the table, or 2^31 - 1 tokens — then nothing changes.  ws: ctamd_kv_reserve_ws() ints. */
long long ctamd_kv_reserve_ws(int n_seq, int n_pages);
int ctamd_kv_reserve(const ctamd_kv_tables* t, const int* add, void* pages, int layers, long long layer_stride, long long page_bytes, int* status, int* ws,
                     void* stream);
/* The pages in use move to the front (those beyond the mark into the holes below it, in order); *status = their number.  lens and lens_out are not used.
 * ws: ctamd_kv_compact_ws() ints. */
long long ctamd_kv_compact_ws(int n_pages);
int ctamd_kv_compact(const ctamd_kv_tables* t, void* pages, int layers, long long layer_stride, long long page_bytes, int* status, int* ws, void* stream);
#ifdef __cplusplus
}
#endif
#endif
