// Host side of the 4-bit paged KV cache: argument checks, launch shapes, and the C entry points of include/ctransformers_amd_ops.h.
#include "kv4.h"
#include "kernels_kv4.h"
#include "kernels_kvpages.h"

#include <float.h>
#include <stdio.h>
#include <string.h>

#include "../../include/ctransformers_amd_ops.h"

namespace ctamd {

int kv4_groups(int head_dim) {
    if (head_dim < 8 || head_dim > 256 || head_dim % 8) return 0;
    const int g = (head_dim + 31) / 32;
    return g == 5 ? 6 : g == 7 ? 8 : g;
}

long long kv4_page_bytes(int n_head_kv, int head_dim, int page_tokens) {
    const int g = kv4_groups(head_dim);
    if (!g || n_head_kv < 1 || n_head_kv > 1024 || !(page_tokens == 32 || page_tokens == 64 || page_tokens == 128 || page_tokens == 256)) return 0;
    return (long long)n_head_kv * (page_tokens / 32) * g * kKv4Block;
}

// Queues a kernel; false if THIS launch failed.  (What hipGetLastError says may be left from another call of the thread, and stays there for its owner.)
template <class T> struct Plain { typedef T type; };
#ifdef CT_EMU
template <class... P> static bool queue(const char*&, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, hipStream_t stream, typename Plain<P>::type... p) {
    (void)stream;
    CT_LAUNCH_DYN(kernel, grid, block, smem, stream, p...);
    return true;
}
#else
template <class... P> static bool queue(const char*& err, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, hipStream_t stream, typename Plain<P>::type... p) {
    void* args[] = {&p...};
    const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, args, smem, stream);
    if (e != hipSuccess) err = hipGetErrorString(e);
    return e == hipSuccess;
}
#endif
// the dynamic LDS of a kernel beyond 64 KB has to be allowed, once per device
#define KV4_OPTIN(fn, bytes) \
    do { if ((bytes) > 64 * 1024) (void)CT_SMEM_OPTIN(fn, bytes); } while (0)

#define KV4_BY_GROUPS(G_, ...) \
    switch (G_) { \
        case 1: { constexpr int G = 1; __VA_ARGS__ } break; \
        case 2: { constexpr int G = 2; __VA_ARGS__ } break; \
        case 3: { constexpr int G = 3; __VA_ARGS__ } break; \
        case 4: { constexpr int G = 4; __VA_ARGS__ } break; \
        case 6: { constexpr int G = 6; __VA_ARGS__ } break; \
        default: { constexpr int G = 8; __VA_ARGS__ } break; \
    }

bool kv4_check(Kv4Cache& c, int page_tokens, const char*& err) {
    const long long bytes = kv4_page_bytes(c.n_head_kv, c.head_dim, page_tokens);
    err = nullptr;
    if (!bytes) err = "sizes not supported: head_dim is a multiple of 8 up to 256, page_tokens 32, 64, 128 or 256, n_head_kv 1 .. 1024";
    else if (c.n_seq < 0 || c.total < 0 || c.n_pages < 0 || c.table_width < 0 || c.table_stride < c.table_width) err = "negative size, or table rows that overlap";
    else if (c.n_seq > (1 << 20) || c.total > (1 << 24)) err = "at most 2^20 sequences and 2^24 rows a call";
    else if ((long long)c.table_width * page_tokens > (1 << 30)) err = "table rows of more than 2^30 tokens";
    else if (c.n_seq && c.total && ((!c.table && c.table_width) || !c.lens || !c.pages) && c.n_pages) err = "null cache pointer";
    else if (c.n_seq != 1 && !c.cu && c.total) err = "cu is needed for more than one sequence";
    else if (c.page_stride < bytes && c.n_pages > 1) err = "pages overlap: page_stride is less than a page";
    else if (c.page_stride % 16 || (uintptr_t)c.pages % 16) err = "pages are 16-byte aligned";
    c.groups = kv4_groups(c.head_dim);
    c.bshift = page_tokens == 32 ? 0 : page_tokens == 64 ? 1 : page_tokens == 128 ? 2 : 3;
    return !err;
}

static void rows_vec(Kv4Rows& r) {   // 16-byte loads of dims that lie side by side
    const long long per = r.type == KV4_F32 ? 4 : 8;
    r.vec = r.dim == 1 && r.row % per == 0 && r.head % per == 0 && (uintptr_t)r.p % 16 == 0;
}

static bool append_grid(Kv4Append& a, int max_rows, dim3& grid, const char*& err) {
    const Kv4Cache& c = a.c;
    if (max_rows > c.total) max_rows = c.total;
    a.max_rows = max_rows;
    a.blocks = (int)(((long long)max_rows + 62) / 32);
    const long long x = (long long)a.blocks * c.n_seq * c.n_head_kv;
    if (x > 0x7FFFFFFF) { err = "too many rows times sequences for one call"; return false; }
    grid = dim3((unsigned)x);
    rows_vec(a.k);
    rows_vec(a.v);
    return true;
}

// A pool of no pages: nothing is stored, but reading and attention look at the lengths and the table all the same.
static bool tables_there(const Kv4Cache& c, const char*& err) {
    if (c.lens && (c.table || !c.table_width)) return true;
    err = "null cache pointer";
    return false;
}

bool kv4_append(Kv4Append& a, int max_rows, hipStream_t stream, const char*& err) {
    dim3 grid;
    if (a.c.total == 0 || a.c.n_seq == 0 || a.c.n_pages == 0 || max_rows <= 0) return true;
    if (!append_grid(a, max_rows, grid, err)) return false;
    KV4_BY_GROUPS(a.c.groups, return queue(err, kv4_append_kernel<G>, grid, dim3(256), 0, stream, a);)
    return true;
}

bool kv4_read(Kv4Append& a, int max_rows, hipStream_t stream, const char*& err) {
    dim3 grid;
    if (a.c.total == 0 || a.c.n_seq == 0 || max_rows <= 0) return true;
    if (!tables_there(a.c, err) || !append_grid(a, max_rows, grid, err)) return false;
    KV4_BY_GROUPS(a.c.groups, return queue(err, kv4_read_kernel<G>, grid, dim3(256), 0, stream, a);)
    return true;
}

// Rows of a tile: kv4_decode_kernel takes 16, or 32 where two tiles of a head fit the registers (128 dims), kv4_prompt_kernel 128.  The first streams the codes at
// memory speed once per tile, the second unpacks them once for 128 rows but takes at least as long for fewer.  Where they cross
// depends on how much work there is in all; the rule looks at the rows of a KV head alone.  The first against the second, us, 16 sequences of 2650 .. 7950 tokens, 8 KV heads:
// 128 dims 40 rows 77 / 82, 64 rows 83 / 87, 96 rows 110 / 96, 128 rows 140 / 107; 64 dims 64 rows 55 / 62, 96 rows 74 / 68, 128 rows 89 / 74, 192 rows 125 / 118, 256 rows
// 158 / 128.  One sequence, 128 dims, 128 rows: of 8000 tokens 37 / 38, of 400 tokens 30 / 24.  4 KV heads, 128 dims: 16 sequences of 2000 .. 6000 tokens 40 rows 43 / 42,
// 96 rows 57 / 53, one of 4000 24 / 25, 28 / 28.  (The first also keeps K exact and p in two halves.)
static int tile_rows(const Kv4Attn& a, long long rows) {
    if (rows <= 16) return 16;
    if (a.c.groups <= 4 && rows <= (a.c.groups <= 2 ? 192 : 96)) return 32;
    return 128;
}
static int chip_cus() {   // of the current device; asked for once per device
    static int n_cu[16] = {};
    int d = 0, n = 0;
#ifndef CT_EMU
    if (hipGetDevice(&d) != hipSuccess || d < 0 || d > 15) d = 0;
#endif
    if (!n_cu[d]) n_cu[d] = hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, d) == hipSuccess && n > 0 ? n : 256;
    return n_cu[d];
}
// workgroups of a line of at most `units` x `blocks` blocks
static long long shares(const Kv4Attn& a, long long units, long long blocks) {
    const long long most = units * (blocks + kUnitCost) / (a.min_blocks + kUnitCost) + 1;   // (a share is no shorter than that)
    return most < a.want_parts ? most : a.want_parts;
}

long long kv4_attention_plan(Kv4Attn& a, int max_rows) {
    const Kv4Cache& c = a.c;
    a.rep = a.n_head / c.n_head_kv;
    if (max_rows > c.total) max_rows = c.total;
    a.max_rows = max_rows;
    const long long rows = (long long)max_rows * a.rep;
    const int tr = tile_rows(a, rows);
    a.tiles = (int)((rows + tr - 1) / tr);
    // The grid is for the longest sequences that the table has room for: how long they are is known on the device only.
    const long long blocks = (long long)c.table_width << c.bshift, units = (long long)c.n_seq * c.n_head_kv * a.tiles;
    const int cus = chip_cus();
    if (tr < 128) {   // shares of the line (kv4_decode_kernel): as many as are resident at once; one unit a workgroup where a unit is no longer than the least share
        const int g = c.groups * tr / 16;
        a.min_blocks = 8;
        a.want_parts = cus * (g <= 2 ? 4 : g <= 4 ? 3 : 2);
        a.nsplit = blocks <= a.min_blocks ? 1 : 2;
        return a.nsplit > 1 ? 2ll * shares(a, units, blocks) * tr * (c.head_dim + 2) : 0;
    }
    // Where there are too few tiles to fill the chip their keys are split, in parts that come out at about two a CU over the whole call (kv4_part).
    a.min_blocks = 16;
    a.want_parts = 2 * cus;
    long long split = units ? a.want_parts / units : 1;
    const long long most = (blocks + a.min_blocks - 1) / a.min_blocks;
    if (split > most) split = most;
    if (split > 256) split = 256;
    if (split < 1) split = 1;
    a.nsplit = (int)split;
    return split > 1 ? units * split * tr * (c.head_dim + 2) : 0;
}

template <int G, int NT> static bool launch_decode(const Kv4Attn& a, hipStream_t stream, const char*& err) {
    constexpr size_t smem = (size_t)(4 * 16 * (32 * G + 4) + 4 * 16 * NT * 2) * 4;
    auto kfn = kv4_decode_kernel<G, NT>;
    KV4_OPTIN(kfn, smem);
    const long long units = (long long)a.c.n_seq * a.c.n_head_kv * a.tiles, n = a.nsplit > 1 ? shares(a, units, (long long)a.c.table_width << a.c.bshift) : units;
    return queue(err, kfn, dim3((unsigned)n), dim3(256), smem, stream, a);
}

template <int W> static bool launch_join(const Kv4Attn& a, int tr, dim3 grid, hipStream_t stream, const char*& err) {
    const dim3 block(64 * W);
    if (tr < 128)
        return a.c.head_dim <= 128 ? queue(err, kv4_join_kernel<1, true, W>, grid, block, 0, stream, a, tr) : queue(err, kv4_join_kernel<2, true, W>, grid, block, 0, stream, a, tr);
    return a.c.head_dim <= 128 ? queue(err, kv4_join_kernel<1, false, W>, grid, block, 0, stream, a, tr) : queue(err, kv4_join_kernel<2, false, W>, grid, block, 0, stream, a, tr);
}

bool kv4_attention(Kv4Attn& a, int max_rows, long long ws_floats, hipStream_t stream, const char*& err) {
    const Kv4Cache& c = a.c;
    if (a.n_head < 1 || a.n_head > 65536 || a.n_head % c.n_head_kv) { err = "n_head is a multiple of n_head_kv"; return false; }
    if (!(a.scale >= -FLT_MAX && a.scale <= FLT_MAX)) { err = "scale is not a finite number"; return false; }
    if (c.total && a.q.dim != 1) { err = "the dims of a query row are adjacent"; return false; }
    if (c.total == 0 || c.n_seq == 0 || max_rows <= 0) return true;
    if (!tables_there(c, err)) return false;
    const long long want = kv4_attention_plan(a, max_rows);
    if (want > ws_floats || (want && !a.ws)) { err = "workspace too small"; return false; }
    const long long pairs = (long long)c.n_seq * c.n_head_kv, grid = ((pairs + 7) & ~7ll) * a.tiles * a.nsplit;
    rows_vec(a.q);
    if (pairs * a.tiles * (((long long)c.table_width << c.bshift) + kUnitCost) > 0x7FFFFFFF) { err = "a table with room for 2^31 blocks or more over all heads"; return false; }
    if (grid > 0x7FFFFFFF || (long long)c.total * a.n_head > 0x7FFFFFFF) { err = "too many rows times sequences for one call"; return false; }
    const int tr = tile_rows(a, (long long)(max_rows > c.total ? c.total : max_rows) * a.rep);
    bool ok = false;
    if (tr == 16) {
        KV4_BY_GROUPS(c.groups, (ok = launch_decode<G, 1>(a, stream, err));)
    } else if (tr == 32) {
        switch (c.groups) {
            case 1: ok = launch_decode<1, 2>(a, stream, err); break;
            case 2: ok = launch_decode<2, 2>(a, stream, err); break;
            case 3: ok = launch_decode<3, 2>(a, stream, err); break;
            default: ok = launch_decode<4, 2>(a, stream, err); break;
        }
    } else {
        KV4_BY_GROUPS(c.groups, {
            auto kfn = kv4_prompt_kernel<G>;
            constexpr size_t smem = Kv4Lds<G>::BYTES;
            KV4_OPTIN(kfn, smem);
            ok = queue(err, kfn, dim3((unsigned)grid), dim3(256), smem, stream, a);
        })
    }
    if (!ok || a.nsplit <= 1) return ok;
    const dim3 jg((unsigned)((long long)c.total * a.n_head));
    // few rows: eight waves for each, their parts are many; many rows: a wave each, all of them resident at once
    return (long long)c.total * a.n_head <= 2048 ? launch_join<8>(a, tr, jg, stream, err) : launch_join<1>(a, tr, jg, stream, err);
}

// ---- pages ------------------------------------------------------------------------------------------------------------------------------------------
static bool overlap(const void* a, long long na, const void* b, long long nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return na > 0 && nb > 0 && x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}
static bool pages_check(const KvPages& a, bool lens, const char*& err) {
    err = nullptr;
    const long long cells = (long long)a.n_seq * a.width, rows = a.parents ? a.n_new : a.n_seq;
    if (a.n_seq < 0 || a.width < 0 || a.n_pages < 0 || a.n_new < 0) err = "negative size";
    else if (a.n_seq > (1 << 20) || a.n_new > (1 << 20) || a.width > (1 << 20)) err = "at most 2^20 sequences and pages a sequence";
    else if (a.page_tokens < 1) err = "page_tokens is positive";
    else if ((a.n_pages && (!a.refs || !a.refs_o)) || (cells && !a.table) || (rows * a.width && !a.table_o) || (lens && ((a.n_seq && !a.lens) || (rows && !a.lens_o)))) err = "null pointer";
    if (err) return false;
    const void* in[3] = {a.table, lens ? a.lens : nullptr, a.refs};
    const long long in_n[3] = {4 * cells, lens ? 4ll * a.n_seq : 0, 4ll * a.n_pages};
    const void* out[3] = {a.table_o, lens ? a.lens_o : nullptr, a.refs_o};
    const long long out_n[3] = {4 * rows * a.width, lens ? 4 * rows : 0, 4ll * a.n_pages};
    for (int i = 0; i < 3; ++i)
        for (int o = 0; o < 3; ++o) {
            if (overlap(in[i], in_n[i], out[o], out_n[o])) { err = "an output overlaps an input"; return false; }
            if (i < o && overlap(out[i], out_n[i], out[o], out_n[o])) { err = "two outputs overlap"; return false; }
        }
    return true;
}
static bool move_check(const KvPages& a, const char*& err) {
    if (a.layers < 0 || a.page_bytes < 0 || a.page_bytes % 16 || a.layer_stride % 16 || (uintptr_t)a.pages % 16) err = "pages are multiples of 16 bytes, 16-byte aligned";
    else if (a.layers && a.n_pages && a.page_bytes && !a.pages) err = "null pages";
    else if (a.layers > 1 && a.layer_stride < a.page_bytes * a.n_pages) err = "layers overlap";
    else if (!a.status || !a.ws) err = "null status or workspace";
    else return true;
    return false;
}
static unsigned groups_for(long long items, long long per, long long most) {
    const long long n = (items + per - 1) / per;
    return (unsigned)(n < 1 ? 1 : n > most ? most : n);
}
// workgroups that move pages: enough to fill the chip, no more than `most` pages could use
static unsigned movers(const KvPages& a, long long most) { return groups_for(most * a.layers * ((a.page_bytes + 16383) / 16384), 1, 2048); }

long long kv_pages_ws_ints(const KvPages& a) { return 4 + 6ll * a.n_seq + 3ll * a.n_pages; }   // enough for either
bool kv_fork(const KvPages& a, hipStream_t stream, const char*& err) {
    if (!pages_check(a, true, err)) return false;
    if (a.n_new && !a.parents) { err = "null parents"; return false; }
    const long long cells = (long long)a.n_new * a.width;
    if (!queue(err, kv_fork_rows_kernel, dim3(groups_for(cells > a.n_pages ? cells : a.n_pages, 256, 2048)), dim3(256), 0, stream, a)) return false;
    const int each = a.keep || a.n_new > kForkEach, rows = a.n_seq + (each ? a.n_new : 0);
    return !rows || queue(err, kv_fork_counts_kernel, dim3((unsigned)rows), dim3(256), 0, stream, a, each);
}
bool kv_reserve(const KvPages& a, hipStream_t stream, const char*& err) {
    if (!pages_check(a, true, err) || !move_check(a, err)) return false;
    if (a.n_seq && !a.add) { err = "null add"; return false; }
    const long long cells = (long long)a.n_seq * a.width;
    if (!queue(err, kv_reserve_plan_kernel, dim3(1 + groups_for(cells > a.n_pages ? cells : a.n_pages, kPlanThreads, 256)), dim3(kPlanThreads), 0, stream, a)) return false;
    const unsigned apply = groups_for(a.n_seq, 4, 256);
    return queue(err, kv_reserve_apply_kernel, dim3(apply + movers(a, a.n_seq)), dim3(256), 0, stream, a, (int)apply);
}
bool kv_compact(const KvPages& a, hipStream_t stream, const char*& err) {
    if (!pages_check(a, false, err) || !move_check(a, err)) return false;
    const long long cells = (long long)a.n_seq * a.width;
    if (!queue(err, kv_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, a)) return false;
    const unsigned apply = groups_for(cells > a.n_pages ? cells : a.n_pages, 256, 256);
    return queue(err, kv_compact_apply_kernel, dim3(apply + movers(a, a.n_pages / 2)), dim3(256), 0, stream, a, (int)apply);
}

}  // namespace ctamd

// ---- C entry points -----------------------------------------------------------------------------------------------------------------------------------
static thread_local char g_ops_error[160] = "";
static int ops_result(bool ok, const char* what, const char* why) {
    if (ok) return 0;
    snprintf(g_ops_error, sizeof g_ops_error, "%s: %s", what, why ? why : "failed");
    return -1;
}
static bool cache_of(const ctamd_kv4_cache* p, Kv4Cache& c, const char*& err) {
    if (!p) { err = "null cache"; return false; }
    c = Kv4Cache();
    c.pages = (uint8_t*)p->pages; c.page_stride = p->page_stride; c.table = p->table; c.lens = p->lens; c.cu = p->cu;
    c.n_pages = p->n_pages; c.table_stride = p->table_stride; c.table_width = p->table_width; c.n_seq = p->n_seq; c.total = p->total;
    c.n_head_kv = p->n_head_kv; c.head_dim = p->head_dim;
    return ctamd::kv4_check(c, p->page_tokens, err);
}
static bool rows_of(const ctamd_rows* p, Kv4Rows& r, int total, const char*& err) {
    if (!p || (total > 0 && !p->p)) { err = "null rows"; return false; }
    if (p->type < 0 || p->type > 2) { err = "row type is 0 (fp16), 1 (bf16) or 2 (fp32)"; return false; }
    r.p = p->p; r.row = p->row; r.head = p->head; r.dim = p->dim; r.type = p->type; r.vec = 0;
    return true;
}
// Rows that are written: no two elements share memory, shown by each stride reaching past everything that the smaller ones span.
static bool rows_apart(const Kv4Rows& r, int total, int heads, int dim, const char*& err) {
    long long size[3] = {total, heads, dim}, step[3] = {r.row < 0 ? -r.row : r.row, r.head < 0 ? -r.head : r.head, r.dim < 0 ? -r.dim : r.dim}, span = 0;
    for (int i = 0; i < 3; ++i) {
        int k = -1;
        for (int j = 0; j < 3; ++j) if (size[j] > 1 && (k < 0 || step[j] < step[k])) k = j;
        if (k < 0) break;
        if (step[k] <= span) { err = "two elements of an output share memory"; return false; }
        span += (size[k] - 1) * step[k];
        size[k] = 1;
    }
    return true;
}
static KvPages tables_of(const ctamd_kv_tables* t) {
    KvPages a = KvPages();
    a.table = t->table; a.lens = t->lens; a.refs = t->refs; a.table_o = t->table_out; a.lens_o = t->lens_out; a.refs_o = t->refs_out;
    a.n_seq = t->n_seq; a.width = t->width; a.n_pages = t->n_pages; a.page_tokens = t->page_tokens;
    return a;
}

extern "C" {

const char* ctamd_ops_error(void) { return g_ops_error; }
int ctamd_ops_host_memory(void) {
#ifdef CT_EMU
    return 1;
#else
    return 0;
#endif
}
long long ctamd_kv4_page_bytes(int n_head_kv, int head_dim, int page_tokens) { return ctamd::kv4_page_bytes(n_head_kv, head_dim, page_tokens); }

int ctamd_kv4_append(const ctamd_kv4_cache* cache, const ctamd_rows* k, const ctamd_rows* v, void* stream) {
    const char* err = nullptr;
    Kv4Append a = Kv4Append();
    const bool ok = cache_of(cache, a.c, err) && rows_of(k, a.k, a.c.total, err) && rows_of(v, a.v, a.c.total, err) &&
                    ctamd::kv4_append(a, cache->max_rows, (hipStream_t)stream, err);
    return ops_result(ok, "kv4_append", err);
}
int ctamd_kv4_read(const ctamd_kv4_cache* cache, const ctamd_rows* k, const ctamd_rows* v, void* stream) {
    const char* err = nullptr;
    Kv4Append a = Kv4Append();
    bool ok = cache_of(cache, a.c, err) && rows_of(k, a.k, a.c.total, err) && rows_of(v, a.v, a.c.total, err);
    if (ok && (k->dim != 1 || v->dim != 1)) { err = "the dims of an output row are adjacent"; ok = false; }
    ok = ok && rows_apart(a.k, a.c.total, a.c.n_head_kv, a.c.head_dim, err) && rows_apart(a.v, a.c.total, a.c.n_head_kv, a.c.head_dim, err);
    ok = ok && ctamd::kv4_read(a, cache->max_rows, (hipStream_t)stream, err);
    return ops_result(ok, "kv4_read", err);
}
long long ctamd_kv4_attention_ws(const ctamd_kv4_cache* cache, int n_head) {
    const char* err = nullptr;
    Kv4Attn a = Kv4Attn();
    if (!cache_of(cache, a.c, err) || n_head < 1 || n_head % a.c.n_head_kv || cache->max_rows <= 0) return 0;
    a.n_head = n_head;
    return ctamd::kv4_attention_plan(a, cache->max_rows);
}
int ctamd_kv4_attention(const ctamd_kv4_cache* cache, int n_head, const ctamd_rows* q, const ctamd_rows* out, float scale, float* ws, long long ws_floats,
                        void* stream) {
    const char* err = nullptr;
    Kv4Attn a = Kv4Attn();
    Kv4Rows o = Kv4Rows();
    bool ok = cache_of(cache, a.c, err) && rows_of(q, a.q, a.c.total, err) && rows_of(out, o, a.c.total, err);
    if (ok && a.c.total && o.dim != 1) { err = "the dims of an output row are adjacent"; ok = false; }
    ok = ok && rows_apart(o, a.c.total, n_head, a.c.head_dim, err);
    a.out = (void*)o.p; a.o_row = o.row; a.o_head = o.head; a.out_type = o.type; a.n_head = n_head; a.scale = scale; a.ws = ws;
    ok = ok && ctamd::kv4_attention(a, cache->max_rows, ws_floats, (hipStream_t)stream, err);
    return ops_result(ok, "kv4_attention", err);
}

int ctamd_kv_fork(const ctamd_kv_tables* t, const int* parents, const int* keep, int n_new, void* stream) {
    const char* err = "null tables";
    if (!t) return ops_result(false, "kv_fork", err);
    KvPages a = tables_of(t);
    static const int none = 0;
    a.parents = parents ? parents : n_new ? nullptr : &none; a.keep = keep; a.n_new = n_new;
    const bool ok = ctamd::kv_fork(a, (hipStream_t)stream, err);   // (before err is read)
    return ops_result(ok, "kv_fork", err);
}
long long ctamd_kv_reserve_ws(int n_seq, int n_pages) { return 4 + 6ll * n_seq + 2ll * n_pages; }
int ctamd_kv_reserve(const ctamd_kv_tables* t, const int* add, void* pages, int layers, long long layer_stride, long long page_bytes, int* status, int* ws,
                     void* stream) {
    const char* err = "null tables";
    if (!t) return ops_result(false, "kv_reserve", err);
    KvPages a = tables_of(t);
    a.add = add; a.pages = (uint8_t*)pages; a.layers = layers; a.layer_stride = layer_stride; a.page_bytes = page_bytes; a.status = status; a.ws = ws;
    const bool ok = ctamd::kv_reserve(a, (hipStream_t)stream, err);   // (before err is read)
    return ops_result(ok, "kv_reserve", err);
}
long long ctamd_kv_compact_ws(int n_pages) { return 4 + 3ll * n_pages; }
int ctamd_kv_compact(const ctamd_kv_tables* t, void* pages, int layers, long long layer_stride, long long page_bytes, int* status, int* ws, void* stream) {
    const char* err = "null tables";
    if (!t) return ops_result(false, "kv_compact", err);
    KvPages a = tables_of(t);
    a.pages = (uint8_t*)pages; a.layers = layers; a.layer_stride = layer_stride; a.page_bytes = page_bytes; a.status = status; a.ws = ws;
    const bool ok = ctamd::kv_compact(a, (hipStream_t)stream, err);   // (before err is read)
    return ops_result(ok, "kv_compact", err);
}

}  // extern "C"
