// Pages of a KV cache that several sequences share: forking, making room (with a copy of a shared last page before it is written), compaction.  The bookkeeping
// lives in device memory — tables of page numbers, lengths, one count of references per page (0: free) — so that no operation waits for the host and all of them can be
// captured into a graph.  Everything is deterministic: free pages are taken lowest first, in the order of the sequences.
//
// reserve and compact are two launches each: workgroup 0 of the first plans (a scan over the sequences and the pages: latency, ~1 us per 4096 pages and per 1024 sequences,
// more where many of those share their last page: each counts those before it among its 1024) while the others copy the tables; the second applies the plan and moves the
// pages, which is a plain copy and bound by memory.  Moving 424 MB (half of a pool of 16 layers): 189 us, 4.5 TB/s read and written (a large copy: 4.66).  256 sequences of
// up to 8192 tokens: fork 3.1 + 2.9 us, room for 16 more tokens 11.3 + 4.6 us.
#pragma once
#include "kv4.h"

constexpr int kPlanThreads = 1024;

#ifdef CT_EMU
static inline void kvp_atomic_add(int* p, int v) { *p += v; }
#else
DEV void kvp_atomic_add(int* p, int v) { (void)atomicAdd(p, v); }
#endif
// words that threads of one workgroup count in: read and cleared where atomics are performed
#ifdef CT_EMU
static inline int kvp_atomic_get(int* p) { return *p; }
static inline void kvp_atomic_clear(int* p) { *p = 0; }
#else
DEV int kvp_atomic_get(int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
DEV void kvp_atomic_clear(int* p) { __hip_atomic_store(p, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
#endif

// exclusive sum over the workgroup's threads; `all` = the total
DEV int kvp_scan(int v, int& all, int* lds) {
    const int lane = lane_id(), w = wave_id();
    int x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl(x, lane >= d ? lane - d : lane);
        if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 63) lds[w] = x;
    __syncthreads();
    int before = 0, sum = 0;
    for (int k = 0; k < (int)(blockDim.x >> 6); ++k) { const int y = lds[k]; if (k < w) before += y; sum += y; }
    all = sum;
    return before + x - v;
}
DEV int kvp_len(const KvPages& a, int s) { const int n = a.lens[s]; return n < 0 ? 0 : n; }
// table entries of a sequence that name pages of its own
DEV int kvp_entries(const KvPages& a, int s) {
    const int n = kvp_len(a, s), e = n / a.page_tokens + (n % a.page_tokens != 0);
    return e < a.width ? e : a.width;
}

DEV int kvp_new_len(const KvPages& a, int i) {
    const int p = a.parents[i];
    if (p < 0 || p >= a.n_seq) return 0;
    const int n = kvp_len(a, p), k = a.keep ? a.keep[i] : n;
    return k < 0 ? 0 : k < n ? k : n;
}
DEV int kvp_new_entries(const KvPages& a, int i) {
    const int n = kvp_new_len(a, i), e = n / a.page_tokens + (n % a.page_tokens != 0);
    return e < a.width ? e : a.width;
}

// ---- fork: new sequence i is a copy of parents[i], sharing its pages, or of its first keep[i] tokens; a parent outside [0, n_seq) gives an empty one ----
__global__ void __launch_bounds__(256) kv_fork_rows_kernel(const KvPages a) {
    const long long step = (long long)gridDim.x * 256, n = (long long)a.n_new * a.width;
    for (long long k = (long long)blockIdx.x * 256 + threadIdx.x; k < n; k += step) {
        const int s = (int)(k / a.width), e = (int)(k % a.width), p = a.parents[s];
        const bool ok = p >= 0 && p < a.n_seq;
        a.table_o[k] = ok && e < kvp_new_entries(a, s) ? a.table[(long long)p * a.width + e] : -1;
    }
    for (long long k = (long long)blockIdx.x * 256 + threadIdx.x; k < a.n_new; k += step) a.lens_o[k] = kvp_new_len(a, (int)k);
    for (long long k = (long long)blockIdx.x * 256 + threadIdx.x; k < a.n_pages; k += step) a.refs_o[k] = a.refs[k];
}
// Every page of an old sequence: one reference more per child, one less for the sequence itself (integer atomics: any order gives the same counts).  With `keep` the
// children's pages differ, and with many children it takes long to count them for every parent: then (`each`) the old sequences' workgroups take theirs away, the new ones'
// add theirs.  Both launches of a fork of 4 pages a sequence, us, children counted / taken and added: 4096 sequences 19 / 19, 8192 33 / 20, 65536 980 / 64.
constexpr int kForkEach = 4096;
__global__ void __launch_bounds__(256) kv_fork_counts_kernel(const KvPages a, int each) {
    __shared__ int lds[4];
    const int s = (int)blockIdx.x;
    if (each) {
        const bool old = s < a.n_seq;
        const int i = s - a.n_seq, row = old ? s : a.parents[i], n = old ? kvp_entries(a, s) : kvp_new_entries(a, i);
        for (int e = (int)threadIdx.x; e < n; e += 256) {
            const int p = a.table[(long long)row * a.width + e];
            if (p >= 0 && p < a.n_pages) kvp_atomic_add(&a.refs_o[p], old ? -1 : 1);
        }
        return;
    }
    int mine = 0, children;
    for (int k = (int)threadIdx.x; k < a.n_new; k += 256) mine += a.parents[k] == s;
    (void)kvp_scan(mine, children, lds);
    if (children == 1) return;
    const int n = kvp_entries(a, s);
    for (int e = (int)threadIdx.x; e < n; e += 256) {
        const int p = a.table[(long long)s * a.width + e];
        if (p >= 0 && p < a.n_pages) kvp_atomic_add(&a.refs_o[p], children - 1);
    }
}

// ---- reserve: room for add[s] more tokens in every sequence -----------------------------------------------------------------------------------------
// ws: [0] ok, [1] copies, [2] pages taken, [4 ..] per sequence {first entry that changes, entries, index of its first page among those taken, copied tail or -1},
// then the pages taken, then the copies (source, destination), then per page how many of the rounds' sequences had it as their partly filled last page
struct KvpWs { int* head; int* seq; int* taken; int* copy; int* sharers; };
DEV KvpWs kvp_ws(const KvPages& a) {
    KvpWs w;
    w.head = a.ws; w.seq = a.ws + 4; w.taken = w.seq + 4 * (long long)a.n_seq; w.copy = w.taken + a.n_pages; w.sharers = w.copy + 2 * (long long)a.n_seq;
    return w;
}
__global__ void __launch_bounds__(kPlanThreads) kv_reserve_plan_kernel(const KvPages a) {
    __shared__ int lds[kPlanThreads / 64], tails[kPlanThreads], flags;
    const int tid = (int)threadIdx.x;
    if (blockIdx.x > 0) {   // the tables as they are; what changes is written over by the second launch
        const long long step = (long long)(gridDim.x - 1) * kPlanThreads, first = (long long)(blockIdx.x - 1) * kPlanThreads + tid;
        for (long long k = first; k < (long long)a.n_seq * a.width; k += step) a.table_o[k] = a.table[k];
        for (long long k = first; k < a.n_pages; k += step) a.refs_o[k] = a.refs[k];
        for (long long k = first; k < a.n_seq; k += step) a.lens_o[k] = a.lens[k];
        return;
    }
    const KvpWs w = kvp_ws(a);
    if (tid == 0) flags = 0;
    const bool rounds = a.n_seq > kPlanThreads;   // a sequence of the first round finds those before it in LDS, one of a later round needs the counts too
    if (rounds) {
        for (int p = tid; p < a.n_pages; p += kPlanThreads) kvp_atomic_clear(&w.sharers[p]);
#ifndef CT_EMU
        __threadfence();
#endif
    }
    __syncthreads();
    int taken = 0, copies = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += kPlanThreads) {
        const int s = s0 + tid;
        int need = 0, start = 0, tail = -1, len = 0, more = 0, first = 0;
        long long last = 0;                          // (a sequence may end near 2^31, and a page be one token)
        bool partly = false;
        if (s < a.n_seq) {
            len = kvp_len(a, s);
            more = a.add[s] > 0 ? a.add[s] : 0;
            const long long to = (long long)len + more;
            first = len / a.page_tokens;
            last = (to + a.page_tokens - 1) / a.page_tokens;
            if (more && (last > a.width || to > 0x7FFFFFFF)) flags = 1;   // (several threads may write it: the same value)
            partly = more && len % a.page_tokens != 0;
            if (partly && first < a.width) {
                const int p = a.table[(long long)s * a.width + first];
                if (p >= 0 && p < a.n_pages) tail = p;
            }
        }
        __syncthreads();
        tails[tid] = tail;
        __syncthreads();
        bool copied = false;
        if (tail >= 0 && a.refs[tail] > 1) {         // shared: those that come before take their references away first
            int left = a.refs[tail] - (s0 ? kvp_atomic_get(&w.sharers[tail]) : 0);
            for (int k = 0; k < tid; ++k) left -= tails[k] == tail;
            copied = left > 1;
        }
        if (more) {
            start = first + (partly && tail >= 0 && !copied);
            need = last - start < a.width ? (int)(last - start) : a.width;   // (more than that is refused below)
        }
        __syncthreads();                             // every thread has read the earlier rounds' counts
        if (rounds && tail >= 0) kvp_atomic_add(&w.sharers[tail], 1);
        int all, c_all;
        const int at = kvp_scan(need, all, lds), c_at = kvp_scan(copied ? 1 : 0, c_all, lds);
        if (s < a.n_seq) {
            int* q = w.seq + 4 * (long long)s;
            q[0] = start; q[1] = need; q[2] = taken + at; q[3] = copied ? tail : -1;
            if (copied) { w.copy[2 * (copies + c_at)] = tail; w.copy[2 * (copies + c_at) + 1] = taken + at; }   // (an index among the taken pages, for now)
        }
        if (all > 0x3FFFFFFF - taken) all = 0x3FFFFFFF - taken;   // (saturates: more pages than there can be)
        taken += all;
        copies += c_all;
        __syncthreads();
    }
    // the lowest `taken` free pages
    int found = 0;
    for (int p0 = 0; p0 < a.n_pages && found < taken; p0 += 4 * kPlanThreads) {
        int free4[4], n = 0, all;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int p = p0 + 4 * tid + j;
            free4[j] = p < a.n_pages && a.refs[p] == 0;
            n += free4[j];
        }
        int at = found + kvp_scan(n, all, lds);
#pragma unroll
        for (int j = 0; j < 4; ++j) if (free4[j]) { if (at < taken) w.taken[at] = p0 + 4 * tid + j; ++at; }
        found += all;
    }
    __syncthreads();
    const bool ok = !flags && found >= taken;
    if (tid == 0) { w.head[0] = ok; w.head[1] = ok ? copies : 0; w.head[2] = taken; a.status[0] = flags ? -1 : found >= taken ? 0 : taken - found; }
    if (ok) for (int k = tid; k < copies; k += kPlanThreads) w.copy[2 * k + 1] = w.taken[w.copy[2 * k + 1]];
}

// pages from w.copy[2 k] to w.copy[2 k + 1], all layers: a work item is 16 KB of one page of one layer
DEV void kvp_move(const KvPages& a, const int* copy, int count, int first, int step) {
    constexpr int kItem = 16384;
    const long long chunks = (a.page_bytes + kItem - 1) / kItem, items = chunks * count * a.layers;
    for (long long it = first; it < items; it += step) {
        const int k = (int)(it / (chunks * a.layers)), l = (int)(it / chunks % a.layers);
        const long long o = it % chunks * kItem, n = a.page_bytes - o < kItem ? a.page_bytes - o : kItem;
        const uint8_t* src = a.pages + l * a.layer_stride + copy[2 * k] * a.page_bytes + o;
        uint8_t* dst = a.pages + l * a.layer_stride + copy[2 * k + 1] * a.page_bytes + o;
        u32x4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) if ((long long)(threadIdx.x + 256 * j) * 16 < n) v[j] = ld16(src + (threadIdx.x + 256 * j) * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) if ((long long)(threadIdx.x + 256 * j) * 16 < n) *(u32x4*)(dst + (threadIdx.x + 256 * j) * 16) = v[j];
    }
}
__global__ void __launch_bounds__(256) kv_reserve_apply_kernel(const KvPages a, int apply) {
    const KvpWs w = kvp_ws(a);
    if (!w.head[0]) return;
    if ((int)blockIdx.x >= apply) { kvp_move(a, w.copy, w.head[1], (int)blockIdx.x - apply, (int)gridDim.x - apply); return; }
    for (int s = (int)blockIdx.x * 4 + wave_id(); s < a.n_seq; s += apply * 4) {   // a wave per sequence
        const int* q = w.seq + 4 * (long long)s;
        const int start = q[0], need = q[1], at = q[2], tail = q[3], lane = lane_id();
        for (int k = lane; k < need; k += 64) {
            const int p = w.taken[at + k];
            a.table_o[(long long)s * a.width + start + k] = p;
            a.refs_o[p] = 1;
        }
        if (lane == 0) {
            if (tail >= 0) kvp_atomic_add(&a.refs_o[tail], -1);
            a.lens_o[s] = kvp_len(a, s) + (a.add[s] > 0 ? a.add[s] : 0);
        }
    }
}

// ---- compact: the pages in use become the first ones ------------------------------------------------------------------------------------------------
// ws: [0] pages in use, [1] moves, [4 ..] per page its new number (in use) or the index of its move (a hole below the mark), then the moves (source, destination)
__global__ void __launch_bounds__(kPlanThreads) kv_compact_plan_kernel(const KvPages a) {
    __shared__ int lds[kPlanThreads / 64];
    const int tid = (int)threadIdx.x;
    int used = 0;
    for (int p = tid; p < a.n_pages; p += kPlanThreads) used += a.refs[p] > 0;
    int all;
    (void)kvp_scan(used, all, lds);
    const int mark = all;
    int* rank = a.ws + 4;
    int* copy = rank + a.n_pages;
    int holes = 0, moves = 0;
    for (int p0 = 0; p0 < a.n_pages; p0 += 4 * kPlanThreads) {   // below the mark the holes are counted, from it on the pages that move
        int hit[4], n = 0, nh = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int p = p0 + 4 * tid + j;
            const bool in = p < a.n_pages && a.refs[p] > 0;
            hit[j] = p >= a.n_pages ? 0 : p < mark ? (in ? 0 : 1) : (in ? 2 : 0);
            nh += hit[j] == 1;
            n += hit[j] == 2;
        }
        int ah, am, h_at = 0, m_at = 0;
        h_at = holes + kvp_scan(nh, ah, lds);
        m_at = moves + kvp_scan(n, am, lds);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int p = p0 + 4 * tid + j;
            if (hit[j] == 1) { copy[2 * h_at + 1] = p; rank[p] = h_at++; }
            else if (hit[j] == 2) { copy[2 * m_at] = p; rank[p] = m_at++; }
        }
        holes += ah;
        moves += am;
    }
    if (tid == 0) { a.ws[0] = mark; a.ws[1] = moves; a.status[0] = mark; }
}
__global__ void __launch_bounds__(256) kv_compact_apply_kernel(const KvPages a, int apply) {
    const int* rank = a.ws + 4;
    const int* copy = rank + a.n_pages;
    const int mark = a.ws[0], moves = a.ws[1];
    if ((int)blockIdx.x >= apply) { kvp_move(a, copy, moves, (int)blockIdx.x - apply, (int)gridDim.x - apply); return; }
    const long long step = (long long)apply * 256, first = (long long)blockIdx.x * 256 + threadIdx.x;
    for (long long k = first; k < (long long)a.n_seq * a.width; k += step) {
        const int p = a.table[k];
        // an entry that names a free page names none afterwards: another page's content may come to lie there
        a.table_o[k] = p < 0 || p >= a.n_pages ? p : a.refs[p] <= 0 ? -1 : p < mark ? p : copy[2 * rank[p] + 1];
    }
    for (long long p = first; p < a.n_pages; p += step) a.refs_o[p] = p >= mark ? 0 : a.refs[p] > 0 ? a.refs[p] : a.refs[copy[2 * rank[p]]];
}
