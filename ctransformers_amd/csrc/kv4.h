// Launches of the 4-bit paged KV cache (kernels_kv4.h, kernels_kvpages.h): what the C entry points (include/ctransformers_amd_ops.h) and the engine share.
// All of them are asynchronous on `stream` of the current device and return false, with a message, without having launched anything if an argument is refused.
#pragma once
#include "gpu.h"

constexpr int kKv4Block = 1152;   // bytes of a block (32 tokens of one head) per group of 32 dims
constexpr int kUnitCost = 16;     // see kv4_decode_kernel
enum { KV4_F16 = 0, KV4_BF16 = 1, KV4_F32 = 2 };

struct Kv4Cache {
    uint8_t* pages;          // [n_pages] pages, page_stride bytes apart, 16-byte aligned
    long long page_stride;
    const int* table;        // [n_seq][table_stride], table_width entries of which name pages; an entry outside [0, n_pages) is no page: its tokens are absent
    const int* lens;         // [n_seq]: tokens of each sequence, the new ones among them ...
    const int* cu;           // [n_seq + 1]: first packed row of each sequence; null: one sequence, all rows
    int len_add;             // ... plus this
    int n_pages, table_stride, table_width, n_seq, total, n_head_kv, head_dim, groups, bshift;   // bshift: log2(blocks per page)
};
struct Kv4Rows {             // packed rows [total][n_head][head_dim], strides in elements
    const void* p;
    long long row, head, dim;
    int type, vec;           // vec: dims adjacent, everything a multiple of 16 bytes
};
struct Kv4Append {
    Kv4Cache c;
    Kv4Rows k, v;
    int blocks;     // most blocks that the new rows of one sequence touch
    int max_rows;   // rows of a sequence from here on are left out
    int absolute;   // 1: a row's place in k and v is its position in the sequence, not its place among the packed rows (kv4_append_kernel)
};
struct Kv4Attn {
    Kv4Cache c;
    Kv4Rows q;
    void* out;
    long long o_row, o_head;
    float* ws;               // partial results, head_dim + 2 floats a row: [share][2][rows of a tile] or [row tile][split][rows of a tile]
    int out_type, n_head, rep, tiles, nsplit, min_blocks, want_parts, max_rows;   // rep: query heads of a KV head; tiles: row tiles of a (sequence, KV head); max_rows: as above
    float scale;
};

struct KvPages {
    const int* table;   // [n_seq][width], rows adjacent; entries past a sequence's pages are -1
    const int* lens;
    const int* refs;    // [n_pages]
    int* table_o;
    int* lens_o;
    int* refs_o;
    int n_seq, width, n_pages, page_tokens;
    const int* parents; const int* keep; int n_new;      // fork: [n_new]; keep: tokens that stay, null: all
    const int* add;                     // reserve: [n_seq]
    int* status;                        // reserve: pages missing; compact: pages in use
    int* ws;
    uint8_t* pages; long long layer_stride, page_bytes; int layers;
};

namespace ctamd {

// groups of 32 dims that a head takes (5 and 7 take the room of 6 and 8); 0: not supported
int kv4_groups(int head_dim);
long long kv4_page_bytes(int n_head_kv, int head_dim, int page_tokens);   // 0: not supported
// fills groups and bshift from the head's size and the page's; checks the rest
bool kv4_check(Kv4Cache& c, int page_tokens, const char*& err);
bool kv4_append(Kv4Append& a, int max_rows, hipStream_t stream, const char*& err);
bool kv4_read(Kv4Append& a, int max_rows, hipStream_t stream, const char*& err);
// floats of workspace that kv4_attention wants for these arguments; 0: none
long long kv4_attention_plan(Kv4Attn& a, int max_rows);
bool kv4_attention(Kv4Attn& a, int max_rows, long long ws_floats, hipStream_t stream, const char*& err);
long long kv_pages_ws_ints(const KvPages& a);
bool kv_fork(const KvPages& a, hipStream_t stream, const char*& err);
bool kv_reserve(const KvPages& a, hipStream_t stream, const char*& err);
bool kv_compact(const KvPages& a, hipStream_t stream, const char*& err);

}  // namespace ctamd
