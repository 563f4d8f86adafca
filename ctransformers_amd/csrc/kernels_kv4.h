// A KV cache held in 4 bits, in pages: quantization of K / V rows into it, reading back, attention over it.
//
// Format.  A head's dims fall into groups of 32 (G of them; dims past head_dim are zeros).  A group of one token is quantized as the framework's Q4_0 weights
// are (reference ggml.c:quantize_row_q4_0_reference): d = (the value of largest magnitude, the first on ties) / -8, code = min(15, (int)(x / d + 8.5)),
// value = f16(d) * (code - 8): 4.5 bits a value.  x is clamped to +-65504 first, so f16(d) * 8 is always a finite half.
// A BLOCK is 32 tokens of one head, G * 1152 bytes: [K codes 512 G | V codes 512 G | K scales 64 G | V scales 64 G]; a page is [KV head][page_tokens / 32]
// blocks, so a block never ends inside a page's neighbour and one (page, head) is one contiguous run.  Inside a block everything lies in the order in which the
// matrix instructions want their operands, so that the attention kernels load registers straight from memory, with no exchange between lanes:
//   K dword (token t, dim c)   (4 t + (c & 31) / 8) * G + c / 32, element c & 7    lane (token, quad) of a 16x16x32 product reads its G dwords as one load
//   V dword (token t, dim c)   ((t & 15) / 4) * 32 G + c, element (t & 3) + 4 (t / 16)    eight tokens of one dim: the k slots of a lane.  The tokens are
//                              those whose scores that lane holds after K.Q (rows 4 quad .. 4 quad + 3 of both 16-token tiles)
//   element e of a dword is its nibble e / 2 + 4 (e & 1): (w >> 4 p) & 0x000F000F are elements 2 p and 2 p + 1 as two 16-bit integers
//   K scales [t / 16][(t & 15) / 4][group][t & 3], V scales [(t & 15) / 4][group][element of t]
//
// A token whose K or V of a head holds a NaN gets K scales NaN and V scales 0: rows that see it become NaN through their score, rows that do not see it never
// multiply it (0 * NaN would reach them through the V product otherwise).
#pragma once
#include "gpu.h"

#ifdef CT_EMU
#define KV4_HD static inline
#else
#define KV4_HD __host__ __device__ __forceinline__ static
#endif

constexpr int kKv4Block = 1152;   // bytes of a block per group
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
struct Kv4Append { Kv4Cache c; Kv4Rows k, v; int blocks; };   // blocks: most blocks that the new rows of one sequence touch
struct Kv4Attn {
    Kv4Cache c;
    Kv4Rows q;
    void* out;
    long long o_row, o_head;
    float* ws;               // partial results: [row tile][split][rows of a tile][head_dim + 2]
    int out_type, n_head, rep, tiles, nsplit, min_blocks;   // rep: query heads of a KV head; tiles: row tiles of a (sequence, KV head)
    float scale;
};

// ---- small pieces ---------------------------------------------------------------------------------------------------------------------------------
#ifdef CT_EMU
static inline uint32_t kv4_op2(uint32_t a, uint32_t b, bool mul) {
    uint32_t r = 0;
    for (int s = 0; s < 32; s += 16) {
        const float x = f16_bits_to_f32((uint16_t)(a >> s)), y = f16_bits_to_f32((uint16_t)(b >> s));
        r |= (uint32_t)f32_to_f16_bits(mul ? x * y : x + y) << s;
    }
    return r;
}
static inline uint32_t kv4_add2(uint32_t a, uint32_t b) { return kv4_op2(a, b, false); }
static inline uint32_t kv4_mul2(uint32_t a, uint32_t b) { return kv4_op2(a, b, true); }
static inline uint32_t kv4_cvt2(float a, float b) { return (uint32_t)f32_to_f16_bits(a) | ((uint32_t)f32_to_f16_bits(b) << 16); }
static inline float exp2_fast(float x) { return exp2f(x); }
static inline u32x4 u32x4_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return u32x4{{a, b, c, d}}; }
static inline f32x4 f32x4_splat(float x) { return f32x4{{x, x, x, x}}; }
static inline uint32_t bits_of(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
static inline float float_of(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
static inline void atomic_add_i32(int* p, int v) { *p += v; }
#else
typedef _Float16 kv4_h2 __attribute__((ext_vector_type(2)));
DEV uint32_t kv4_add2(uint32_t a, uint32_t b) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(kv4_h2, a) + __builtin_bit_cast(kv4_h2, b)); }
DEV uint32_t kv4_mul2(uint32_t a, uint32_t b) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(kv4_h2, a) * __builtin_bit_cast(kv4_h2, b)); }
DEV uint32_t kv4_cvt2(float a, float b) { return __builtin_bit_cast(uint32_t, kv4_h2{(_Float16)a, (_Float16)b}); }   // nearest even
DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }   // v_exp_f32: 1 ulp, results below 2^-126 are 0
DEV u32x4 u32x4_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return u32x4{a, b, c, d}; }
DEV f32x4 f32x4_splat(float x) { return f32x4{x, x, x, x}; }
DEV uint32_t bits_of(float f) { return __builtin_bit_cast(uint32_t, f); }
DEV float float_of(uint32_t u) { return __builtin_bit_cast(float, u); }
DEV void atomic_add_i32(int* p, int v) { (void)atomicAdd(p, v); }
#endif
DEV float kv4_load_any(const void* p, long long i, int type) {
    if (type == KV4_F32) return ((const float*)p)[i];
    const uint16_t b = ((const uint16_t*)p)[i];
    return type == KV4_F16 ? f16_bits_to_f32(b) : float_of((uint32_t)b << 16);
}
DEV uint16_t bf16_of(float f) {   // nearest even; a NaN stays one
    const uint32_t u = bits_of(f);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}
DEV void kv4_store_any(void* p, long long i, int type, float f) {
    if (type == KV4_F32) ((float*)p)[i] = f;
    else ((uint16_t*)p)[i] = type == KV4_F16 ? f32_to_f16_bits(f) : bf16_of(f);
}
// eight neighbouring dims
DEV void kv4_load8(float (&x)[8], const Kv4Rows& r, long long at) {
    if (r.vec && r.type != KV4_F32) {
        const u32x4 w = ld16((const uint16_t*)r.p + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (r.type == KV4_F16) { x[2 * j] = f16_bits_to_f32((uint16_t)(w[j] & 0xFFFFu)); x[2 * j + 1] = f16_bits_to_f32((uint16_t)(w[j] >> 16)); }
            else { x[2 * j] = float_of(w[j] << 16); x[2 * j + 1] = float_of(w[j] & 0xFFFF0000u); }
        }
    } else if (r.vec) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u32x4 w = ld16((const float*)r.p + at + 4 * h);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * h + j] = float_of(w[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = kv4_load_any(r.p, at + j * r.dim, r.type);
    }
}
template <int N> DEV void kv4_ldw(uint32_t (&d)[N], const uint8_t* p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) { const u32x4 w = ld16(p + 16 * i); d[4 * i] = w[0]; d[4 * i + 1] = w[1]; d[4 * i + 2] = w[2]; d[4 * i + 3] = w[3]; }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) { const u32x2 w = ld8(p + 8 * i); d[2 * i] = w[0]; d[2 * i + 1] = w[1]; }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] = ((const uint32_t*)p)[i];
    }
}
// the packed rows [lo, hi) of sequence b and its length; rows outside the packed tensor are not there
DEV void kv4_seq(const Kv4Cache& c, int b, int& lo, int& hi, int& len) {
    lo = c.cu ? c.cu[b] : 0;
    hi = c.cu ? c.cu[b + 1] : c.total;
    if (lo < 0) lo = 0;
    if (hi > c.total) hi = c.total;
    if (hi < lo) hi = lo;
    const long long n = (long long)c.lens[b] + c.len_add;
    len = n < 0 ? 0 : n > (1 << 30) ? 1 << 30 : (int)n;
}
// block `blk` of head h of sequence b, null where the table names no page
DEV uint8_t* kv4_block(const Kv4Cache& c, int b, int h, int blk) {
    const int pi = blk >> c.bshift;
    if (blk < 0 || pi >= c.table_width) return nullptr;
    const int pid = c.table[(long long)b * c.table_stride + pi];
    if ((unsigned)pid >= (unsigned)c.n_pages) return nullptr;
    const long long in_page = ((long long)h << c.bshift) + (blk & ((1 << c.bshift) - 1));
    return c.pages + (long long)pid * c.page_stride + in_page * c.groups * kKv4Block;
}

// ---- rows into the cache --------------------------------------------------------------------------------------------------------------------------
// One workgroup per (block, head) that new rows fall into: it alone writes that block, so a V dword that keeps older tokens is read, changed and written without
// atomics.  A thread quantizes one group of one token; K codes and scales go straight out, V codes cross the workgroup through LDS (eight tokens to a dword).
// Memory-bound for prompts: the rows are read once, 16 bytes a lane, and 4.5 bits a value written.
template <int G> __global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4Append a) {
    __shared__ uint32_t vcode[32][8 * G + 1];   // V codes as bytes [token][dim]; + 1: tokens in different banks
    __shared__ uint16_t sc[2][32][G];
    __shared__ int poison[32];
    const Kv4Cache& c = a.c;
    const int tid = (int)threadIdx.x, h = (int)blockIdx.y, b = (int)blockIdx.x / a.blocks;
    int lo, hi, len;
    kv4_seq(c, b, lo, hi, len);
    const int start = len - (hi - lo);                          // position of the first new row (rows before position 0 are dropped)
    const int blk = (start > 0 ? start : 0) / 32 + (int)blockIdx.x % a.blocks;
    if (blk * 32 >= len || hi == lo) return;
    uint8_t* dst = kv4_block(c, b, h, blk);
    if (!dst) return;
    const int t_lo = start > blk * 32 ? start - blk * 32 : 0, t_hi = len - blk * 32 < 32 ? len - blk * 32 : 32;   // the new tokens of this block
    for (int t = tid; t < 32; t += 256) poison[t] = 0;
    __syncthreads();
    for (int it = tid; it < 2 * 32 * G; it += 256) {
        const int half = it / (32 * G), t = (it / G) & 31, g = it % G;
        if (t < t_lo || t >= t_hi) continue;
        const Kv4Rows& r = half ? a.v : a.k;
        const long long at = (long long)(lo + blk * 32 + t - start) * r.row + (long long)h * r.head;
        float x[32], top = 0.0f, big = 0.0f;
        bool nan = false;
#pragma unroll
        for (int o = 0; o < 4; ++o) {
            const int d0 = 32 * g + 8 * o;
            float y[8];
            if (d0 < c.head_dim) kv4_load8(y, r, at + d0 * r.dim);
            else for (int j = 0; j < 8; ++j) y[j] = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v = y[j] > 65504.0f ? 65504.0f : y[j] < -65504.0f ? -65504.0f : y[j];
                nan = nan || v != v;
                x[8 * o + j] = v;
                if (fabsf(v) > big) { big = fabsf(v); top = v; }
            }
        }
        const float d = top / -8.0f;
        const uint16_t dh = f32_to_f16_bits(d);
        const float inv = (dh & 0x7FFFu) ? 1.0f / d : 0.0f;     // a scale that f16 has as 0: every value is 0
        uint32_t w[4] = {0, 0, 0, 0}, bytes[8];
#pragma unroll
        for (int o = 0; o < 4; ++o) {
            bytes[2 * o] = bytes[2 * o + 1] = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float f = x[8 * o + j] * inv + 8.5f;      // two roundings, as the reference's expression has
                const int q = nan ? 8 : (int)f > 15 ? 15 : (int)f;
                w[o] |= (uint32_t)q << (4 * (j / 2) + 16 * (j & 1));
                bytes[2 * o + j / 4] |= (uint32_t)q << (8 * (j & 3));
            }
        }
        if (nan) poison[t] = 1;
        sc[half][t][g] = dh;
        if (half) {
#pragma unroll
            for (int j = 0; j < 8; ++j) vcode[t][8 * g + j] = bytes[j];
        } else {
#pragma unroll
            for (int o = 0; o < 4; ++o) ((uint32_t*)dst)[(4 * t + o) * G + g] = w[o];
        }
    }
    __syncthreads();
    for (int it = tid; it < 2 * 32 * G; it += 256) {
        const int half = it / (32 * G), t = (it / G) & 31, g = it % G;
        if (t < t_lo || t >= t_hi) continue;
        uint16_t* s = (uint16_t*)(dst + (16 + half) * 64 * G);
        const int i = (t & 15) / 4;
        if (half) s[(i * G + g) * 8 + (t & 3) + 4 * (t / 16)] = poison[t] ? (uint16_t)0 : sc[1][t][g];
        else s[(((t / 16) * 4 + i) * G + g) * 4 + (t & 3)] = poison[t] ? (uint16_t)0x7E00 : sc[0][t][g];
    }
    uint32_t* vd = (uint32_t*)(dst + 512 * G);
    for (int it = tid; it < 4 * 32 * G; it += 256) {
        const int i = it / (32 * G), dim = it % (32 * G);
        uint32_t w = 0, m = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int t = 4 * i + (e & 3) + 16 * (e / 4), sh = 4 * (e / 2) + 16 * (e & 1);
            if (t < t_lo || t >= t_hi) continue;
            w |= ((vcode[t][dim / 4] >> (8 * (dim & 3))) & 15u) << sh;
            m |= 15u << sh;
        }
        if (m) vd[it] = m == 0xFFFFFFFFu ? w : (vd[it] & ~m) | w;
    }
}

// The last rows of every sequence out of the cache, as numbers: the mirror image of kv4_append_kernel, same workgroups.  Rows whose page is absent are zeros.
template <int G> __global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4Append a) {
    const Kv4Cache& c = a.c;
    const int tid = (int)threadIdx.x, h = (int)blockIdx.y, b = (int)blockIdx.x / a.blocks;
    int lo, hi, len;
    kv4_seq(c, b, lo, hi, len);
    const int start = len - (hi - lo);
    const int blk = (start >= 0 ? start / 32 : -((31 - start) / 32)) + (int)blockIdx.x % a.blocks;   // rows before position 0 are written too (as zeros)
    if (blk * 32 >= len || hi == lo) return;
    const uint8_t* src = kv4_block(c, b, h, blk);
    const int t_lo = start > blk * 32 ? start - blk * 32 : 0, t_hi = len - blk * 32 < 32 ? len - blk * 32 : 32;
    for (int it = tid; it < 32 * 4 * G; it += 256) {   // K: eight dims of one token
        const int t = it / (4 * G), i = (it / G) & 3, g = it % G, d0 = 32 * g + 8 * i;
        if (t < t_lo || t >= t_hi || d0 >= c.head_dim) continue;
        const long long at = (long long)(lo + blk * 32 + t - start) * a.k.row + (long long)h * a.k.head + d0;
        const uint32_t w = src ? ((const uint32_t*)src)[it] : 0x88888888u;
        const float d = src ? f16_bits_to_f32(((const uint16_t*)(src + 1024 * G))[(((t / 16) * 4 + (t & 15) / 4) * G + g) * 4 + (t & 3)]) : 0.0f;
        for (int e = 0; e < 8; ++e) kv4_store_any((void*)a.k.p, at + e, a.k.type, d * (float)((int)((w >> (4 * (e / 2) + 16 * (e & 1))) & 15u) - 8));
    }
    for (int it = tid; it < 32 * 4 * G; it += 256) {   // V: the same eight dims, one nibble of each of their dwords
        const int t = it / (4 * G), g = (it / 4) % G, d0 = 32 * g + 8 * (it & 3), i = (t & 15) / 4, e = (t & 3) + 4 * (t / 16);
        if (t < t_lo || t >= t_hi || d0 >= c.head_dim) continue;
        const long long at = (long long)(lo + blk * 32 + t - start) * a.v.row + (long long)h * a.v.head + d0;
        const float d = src ? f16_bits_to_f32(((const uint16_t*)(src + 1088 * G))[(i * G + g) * 8 + e]) : 0.0f;
        const uint32_t* vd = (const uint32_t*)(src ? src + 512 * G : nullptr) + (src ? i * 32 * G + d0 : 0);
        for (int j = 0; j < 8; ++j)
            kv4_store_any((void*)a.v.p, at + j, a.v.type, src ? d * (float)((int)((vd[j] >> (4 * (e / 2) + 16 * (e & 1))) & 15u) - 8) : 0.0f);
    }
}

// ---- attention ------------------------------------------------------------------------------------------------------------------------------------
// The query rows of a (sequence, KV head) are r = token * rep + head, tiles of them share a workgroup; row r sees the positions below
// len - rows + token + 1.  The blocks of a tile are divided over `nsplit` workgroups at most; how many of them have work follows from the sequence's own length.
struct Kv4Range { int nq, n_rows, first_tok, len, lo, nb, per, parts; };
DEV Kv4Range kv4_range(const Kv4Attn& a, int b, int tile, int tile_rows) {
    Kv4Range r;
    int lo, hi;
    kv4_seq(a.c, b, lo, hi, r.len);
    r.lo = lo;
    r.nq = hi - lo;
    const int row0 = tile * tile_rows, all = r.nq * a.rep;
    r.n_rows = all - row0 < tile_rows ? all - row0 : tile_rows;
    r.first_tok = row0 / a.rep;
    const int last_tok = (row0 + r.n_rows - 1) / a.rep;
    const int seen = r.n_rows > 0 ? r.len - r.nq + last_tok + 1 : 0;   // positions that the tile's last row sees
    r.nb = seen > 0 ? (seen + 31) / 32 : 0;
    if (r.nb > a.c.table_width << a.c.bshift) r.nb = a.c.table_width << a.c.bshift;   // what the table has no room for is absent
    r.per = (r.nb + a.nsplit - 1) / a.nsplit;
    if (r.per < a.min_blocks) r.per = a.min_blocks;
    r.parts = (r.nb + r.per - 1) / r.per;
    return r;
}

// Eight halves of the dword's codes minus 8, times the scales of their tokens (or one scale for all): f16 products, one rounding (2^-11 of a value whose step is
// 1/8 of the group's largest) — the matrix instruction takes halves.
DEV u32x4 kv4_values(uint32_t w, uint32_t s0, uint32_t s1, uint32_t s2, uint32_t s3) {
    const uint32_t M = 0x000F000Fu, K = 0x64006400u, B = 0xE408E408u;   // 1024 + code, exactly; -1032
    return u32x4_of(kv4_mul2(kv4_add2((w & M) | K, B), s0), kv4_mul2(kv4_add2(((w >> 4) & M) | K, B), s1),
                    kv4_mul2(kv4_add2(((w >> 8) & M) | K, B), s2), kv4_mul2(kv4_add2(((w >> 12) & M) | K, B), s3));
}

// Few rows (a token step, a handful of drafted tokens): a wave takes whole blocks.  16x16x32 matrix products, transposed so that a query row is a COLUMN of both:
//   S = K_codes (A: lane = token) x Q (B: lane = row): lane (row, quad) then holds the scores of tokens 4 quad .. 4 quad + 3 of both 16-token tiles
//   O = V^T (A: lane = dim) x P (B: lane = row): those eight probabilities ARE the lane's k slots — V is stored in that order
// K's codes enter as f16 SUBNORMALS, the 16-bit integers themselves (code * 2^-24: no conversion); -8 * sum(Q) is the product's C operand and the group's scale
// multiplies the 32-dim product in f32, so K is used exactly.  Maximum, sum and O stay per lane in f32; the maximum is raised (and O rescaled) only when a score
// passes it by more than 2^8, so most blocks exchange nothing between lanes (p <= 256 fits f16 as well as p <= 1 does).
// The block after the one being computed is in flight in registers (40 dwords a lane at 128 dims).
template <int G> struct Kv4Raw { uint32_t kc[2][G], ks[2][2 * G], vc[2 * G], vs[2 * G + 2 * (G & 1)]; };
template <int G> DEV void kv4_fetch(Kv4Raw<G>& r, const uint8_t* blk, int m, int i) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        kv4_ldw<G>(r.kc[t], blk + (((t * 16 + m) * 4 + i) * G) * 4);
        kv4_ldw<2 * G>(r.ks[t], blk + 1024 * G + ((t * 4 + i) * G) * 8);
    }
#pragma unroll
    for (int p = 0; p < G / 2; ++p) {   // 64 dims: four neighbouring ones a lane
        const u32x4 w = ld16(blk + 512 * G + (i * 32 * G + 64 * p + 4 * m) * 4), s = ld16(blk + 1088 * G + (i * G + 2 * p + (m >> 3)) * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) { r.vc[4 * p + j] = w[j]; r.vs[4 * p + j] = s[j]; }
    }
    if constexpr (G & 1) {              // 32 dims: two a lane
        const u32x2 w = ld8(blk + 512 * G + (i * 32 * G + 32 * (G - 1) + 2 * m) * 4);
        const u32x4 s = ld16(blk + 1088 * G + (i * G + G - 1) * 16);
        r.vc[2 * G - 2] = w[0]; r.vc[2 * G - 1] = w[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) r.vs[2 * (G - 1) + j] = s[j];
    }
}
// row `row` of the tile, `dim` of the head that register r of dim tile `j` holds for quad i
template <int G> DEV int kv4_dim(int j, int i, int r) {
    return j < 4 * (G / 2) ? 64 * (j / 4) + 16 * i + 4 * r + (j & 3) : 32 * (G - 1) + 8 * i + 2 * r + (j & 1);
}

template <int G, int NT> __global__ void __launch_bounds__(256) kv4_decode_kernel(const Kv4Attn a) {
    constexpr int W = 4, DP = 32 * G, PITCH = DP + 4;
    CT_DYN_SMEM(smem);
    float* part = (float*)smem;                       // [wave][row][PITCH] of one row tile
    float* stat = part + W * 16 * PITCH;              // [wave][16 NT][2]: maximum, sum
    const Kv4Cache& c = a.c;
    const int lane = lane_id(), w = wave_id(), m = lane & 15, i = lane >> 4;
    const int pairs = c.n_seq * c.n_head_kv, id = (int)blockIdx.x;
    const int pair = id % pairs, rest = id / pairs, split = rest % a.nsplit, tile = rest / a.nsplit;
    const int b = pair / c.n_head_kv, kvh = pair % c.n_head_kv;
    const Kv4Range rg = kv4_range(a, b, tile, 16 * NT);
    if (rg.n_rows <= 0 || (split >= rg.parts && split > 0)) return;
    const int row0 = tile * 16 * NT;

    u32x4 q[NT][G];
    float cq[NT][G], sc2[NT], mx[NT], sum[NT];
    int lim[NT];
    f32x4 O[NT][2 * G];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = row0 + 16 * n + m;
        const bool on = 16 * n + m < rg.n_rows;
        const int tok = on ? r / a.rep : 0;
        lim[n] = on ? rg.len - rg.nq + tok + 1 : 0;
        const long long at = (long long)(rg.lo + tok) * a.q.row + (long long)(kvh * a.rep + (on ? r % a.rep : 0)) * a.q.head;
        float x[G][8], big = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int d0 = 32 * g + 8 * i;
            if (on && d0 < c.head_dim) kv4_load8(x[g], a.q, at + d0);
            else for (int j = 0; j < 8; ++j) x[g][j] = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(x[g][j]));
        }
        // Rows that f16 may not hold (bf16, f32) are scaled by a power of two that brings the largest value into [1, 2); bf16 stays exact but for values below
        // 2^-17 of the row's largest.
        float up = 1.0f, down = 1.0f;
        if (a.q.type != KV4_F16) {
            big = fmaxf(big, lane_xor16(big));
            big = fmaxf(big, lane_xor32(big));
            const int e = (int)((bits_of(big) >> 23) & 255u);
            if (e > 0 && e < 254) { up = float_of((uint32_t)(254 - e) << 23); down = float_of((uint32_t)e << 23); }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float s = 0.0f;
            uint32_t h[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                h[j] = kv4_cvt2(x[g][2 * j] * up, x[g][2 * j + 1] * up);
                s += f16_bits_to_f32((uint16_t)(h[j] & 0xFFFFu));
                s += f16_bits_to_f32((uint16_t)(h[j] >> 16));
            }
            s += lane_xor16(s);
            s += lane_xor32(s);
            cq[n][g] = s * (-8.0f / 16777216.0f);
            q[n][g] = u32x4_of(h[0], h[1], h[2], h[3]);
        }
        sc2[n] = a.scale * 1.44269504088896f * 16777216.0f * down;
        mx[n] = -INFINITY;
        sum[n] = 0.0f;
#pragma unroll
        for (int j = 0; j < 2 * G; ++j) O[n][j] = f32x4_splat(0.0f);
    }
    const int free_lim = rg.len - rg.nq + rg.first_tok + 1;   // every row of the tile sees the positions below

    const int end = (split + 1) * rg.per < rg.nb ? (split + 1) * rg.per : rg.nb;
    auto compute = [&](const Kv4Raw<G>& r, int blk) {
        const int p0 = blk * 32;
        const bool edge = p0 + 32 > free_lim || p0 + 32 > rg.len;
        u32x4 P[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float s[2][4];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const uint32_t k = r.kc[t][g], M = 0x000F000Fu;
                    const f32x4 acc = mfma_f16_16x16x32(u32x4_of(k & M, (k >> 4) & M, (k >> 8) & M, (k >> 12) & M), q[n][g], f32x4_splat(cq[n][g]));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t d2 = r.ks[t][2 * g + e / 2];
                        const float d = f16_bits_to_f32((uint16_t)(e & 1 ? d2 >> 16 : d2 & 0xFFFFu));
                        s[t][e] = g == 0 ? d * acc[e] : fmaf(d, acc[e], s[t][e]);
                    }
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[t][e] *= sc2[n];
                    if (edge && p0 + 16 * t + 4 * i + e >= lim[n]) s[t][e] = -INFINITY;
                    top = fmaxf(top, s[t][e]);
                }
            if (__ballot(top > mx[n] + 8.0f)) {   // (also the first block: -inf + 8)
                top = fmaxf(top, lane_xor16(top));
                top = fmaxf(top, lane_xor32(top));
                const float now = fmaxf(mx[n], top);
                const float f = now == -INFINITY ? 1.0f : exp2_fast(mx[n] - now);
                mx[n] = now;
                sum[n] *= f;
#pragma unroll
                for (int j = 0; j < 2 * G; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) O[n][j][e] *= f;
            }
            const float base = mx[n] == -INFINITY ? 0.0f : mx[n];
            uint32_t pk[4];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const float x = exp2_fast(s[t][e] - base), y = exp2_fast(s[t][e + 1] - base);
                    sum[n] += x;
                    sum[n] += y;
                    pk[2 * t + e / 2] = kv4_cvt2(x, y);   // the probabilities as halves: 2^-12 of each, independent of one another
                }
            P[n] = u32x4_of(pk[0], pk[1], pk[2], pk[3]);
        }
        // tokens past the sequence's end: whatever the page holds there must not meet p = 0 as an infinity
        uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
        if (p0 + 32 > rg.len) {
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const int t0 = p0 + 16 * (p / 2) + 4 * i + 2 * (p & 1);
                keep[p] = (t0 < rg.len ? 0xFFFFu : 0u) | (t0 + 1 < rg.len ? 0xFFFF0000u : 0u);
            }
        }
#pragma unroll
        for (int j = 0; j < 2 * G; ++j) {
            const int s0 = j < 4 * (G / 2) ? 4 * (j / 4) : 2 * (G - 1);
            const u32x4 v = kv4_values(r.vc[j], r.vs[s0] & keep[0], r.vs[s0 + 1] & keep[1], r.vs[s0 + 2] & keep[2], r.vs[s0 + 3] & keep[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) O[n][j] = mfma_f16_16x16x32(v, P[n], O[n][j]);
        }
    };
    {
        Kv4Raw<G> r0, r1;
        int blk = split * rg.per + w;
        const uint8_t* p0 = blk < end ? kv4_block(c, b, kvh, uniform_int(blk)) : nullptr;
        if (p0) kv4_fetch<G>(r0, p0, m, i);
        while (blk < end) {
            const uint8_t* p1 = blk + W < end ? kv4_block(c, b, kvh, uniform_int(blk + W)) : nullptr;
            if (p1) kv4_fetch<G>(r1, p1, m, i);
            if (p0) compute(r0, blk);
            blk += W;
            if (blk >= end) break;
            p0 = blk + W < end ? kv4_block(c, b, kvh, uniform_int(blk + W)) : nullptr;
            if (p0) kv4_fetch<G>(r0, p0, m, i);
            if (p1) compute(r1, blk);
            blk += W;
        }
    }
    // the waves' results meet in LDS, in wave order
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        sum[n] += lane_xor16(sum[n]);
        sum[n] += lane_xor32(sum[n]);
        if (i == 0) { stat[(w * 16 * NT + 16 * n + m) * 2] = mx[n]; stat[(w * 16 * NT + 16 * n + m) * 2 + 1] = sum[n]; }
    }
    const bool whole = rg.parts <= 1;
    float* out = a.ws + ((long long)(tile * (long long)pairs + pair) * a.nsplit + split) * (16 * NT) * (c.head_dim + 2);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        if (n) __syncthreads();
#pragma unroll
        for (int j = 0; j < 2 * G; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[(w * 16 + m) * PITCH + kv4_dim<G>(j, i, e)] = O[n][j][e];
        __syncthreads();
        for (int it = (int)threadIdx.x; it < 16 * DP; it += 64 * W) {
            const int row = it / DP, dim = it % DP;
            if (16 * n + row >= rg.n_rows || dim >= c.head_dim) continue;
            float M = -INFINITY, L = 0.0f, v = 0.0f;
#pragma unroll
            for (int k = 0; k < W; ++k) M = fmaxf(M, stat[(k * 16 * NT + 16 * n + row) * 2]);
            const float base = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const float f = exp2_fast(stat[(k * 16 * NT + 16 * n + row) * 2] - base);
                L += f * stat[(k * 16 * NT + 16 * n + row) * 2 + 1];
                v += f * part[(k * 16 + row) * PITCH + dim];
            }
            if (whole) {
                const int r = row0 + 16 * n + row;
                kv4_store_any(a.out, (long long)(rg.lo + r / a.rep) * a.o_row + (long long)(kvh * a.rep + r % a.rep) * a.o_head + dim, a.out_type, L == 0.0f ? 0.0f : v / L);
            } else {
                float* o = out + (16 * n + row) * (c.head_dim + 2);
                o[2 + dim] = v;
                if (dim == 0) { o[0] = M; o[1] = L; }
            }
        }
    }
}

// The parts of a row joined: one wave per (row, head).
template <int NR> __global__ void __launch_bounds__(256) kv4_join_kernel(const Kv4Attn a, int tile_rows) {
    const Kv4Cache& c = a.c;
    const int lane = lane_id(), item = (int)blockIdx.x * 4 + wave_id();
    const int row = item / a.n_head, head = item % a.n_head;
    if (row >= c.total) return;
    int b = 0;
    if (c.cu) {   // the last sequence that begins at or before the row
        int lo = 0, hi = c.n_seq;
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (c.cu[mid] <= row) lo = mid; else hi = mid; }
        b = lo;
        if (row < c.cu[b] || row >= c.cu[b + 1]) return;   // behind the last sequence
    }
    const int kvh = head / a.rep, r = (row - (c.cu ? c.cu[b] : 0)) * a.rep + head % a.rep, tile = r / tile_rows;
    if (tile >= a.tiles) return;
    const Kv4Range rg = kv4_range(a, b, tile, tile_rows);
    if (rg.parts <= 1) return;
    const long long pairs = (long long)c.n_seq * c.n_head_kv, step = (long long)tile_rows * (c.head_dim + 2);
    const float* in = a.ws + ((long long)(tile * pairs + (long long)b * c.n_head_kv + kvh) * a.nsplit) * step + (long long)(r % tile_rows) * (c.head_dim + 2);
    float M = -INFINITY;
    for (int s = lane; s < rg.parts; s += 64) M = fmaxf(M, in[s * step]);
    M = wave_max(M);
    const float base = M == -INFINITY ? 0.0f : M;
    float L = 0.0f, o[NR];
    for (int j = 0; j < NR; ++j) o[j] = 0.0f;
    for (int s0 = 0; s0 < rg.parts; s0 += 64) {
        const int s = s0 + lane;
        const float f = s < rg.parts ? exp2_fast(in[s * step] - base) : 0.0f;
        L += s < rg.parts ? f * in[s * step + 1] : 0.0f;
        const int n = rg.parts - s0 < 64 ? rg.parts - s0 : 64;
        for (int k = 0; k < n; ++k) {
            const float fk = __shfl(f, k);
#pragma unroll
            for (int j = 0; j < NR; ++j) if (lane + 64 * j < c.head_dim) o[j] += fk * in[(s0 + k) * step + 2 + lane + 64 * j];
        }
    }
    L = wave_sum(L);
    const long long at = (long long)row * a.o_row + (long long)head * a.o_head;
#pragma unroll
    for (int j = 0; j < NR; ++j) if (lane + 64 * j < c.head_dim) kv4_store_any(a.out, at + lane + 64 * j, a.out_type, L == 0.0f ? 0.0f : o[j] / L);
}

// Many rows (a prompt, a chunk of one): a workgroup of four waves takes 128 rows, a wave 32 of them; the blocks pass through LDS as halves, two at a time, so that a
// block is unpacked once for 128 rows.  32x32x16 products, transposed as above: lane (row, half) of S^T = K Q^T holds sixteen scores of ITS row, which are the k slots
// of O^T = V^T P^T if the lane of K's operand that gives row 16 t + 8 u + 4 h + e of the product reads token 16 u + 4 (2 t + h) + e (V's order again).
// LDS: K as 16-byte chunks [8 dims][token], a chunk column 32 bytes longer than its tokens (the four quads that write a token's chunks fall into different banks),
// V as 16-byte chunks [4 eights of tokens][dim]: both are read and written without bank conflicts.  Two buffers: while one pair of blocks is computed the next is
// fetched into registers, unpacked and written into the other, one barrier a pair.
// The row tiles of one (sequence, KV head) go to one XCD, whose L2 then holds that head's codes for all of them; tiles that see most come first.
template <int G> struct Kv4Lds { static constexpr int KC = 32 * 16 + 32, KB = 4 * G * KC, VB = 4 * 32 * G * 16, BLK = KB + VB, BYTES = 4 * BLK; };

#ifdef CT_EMU
static inline void lds_st16(unsigned char* p, u32x4 v) { memcpy(p, &v, 16); }
static inline u32x4 lds_ld16(const unsigned char* p) { u32x4 v; memcpy(&v, p, 16); return v; }
#else
DEV void lds_st16(unsigned char* p, u32x4 v) { *(u32x4*)p = v; }
DEV u32x4 lds_ld16(const unsigned char* p) { return *(const u32x4*)p; }
#endif

template <int G> __global__ void __launch_bounds__(256, G <= 4 ? 2 : 1) kv4_prompt_kernel(const Kv4Attn a) {
    typedef Kv4Lds<G> L;
    CT_DYN_SMEM(smem);
    const Kv4Cache& c = a.c;
    const int tid = (int)threadIdx.x, lane = lane_id(), w = wave_id(), n = lane & 31, h = lane >> 5;
    // workgroup -> (pair, split, tile): ids that are equal modulo 8 share an XCD
    const int pairs = c.n_seq * c.n_head_kv, per_pair = a.tiles * a.nsplit, id = (int)blockIdx.x;
    const int pair = (id & 7) + 8 * ((id >> 3) / per_pair), slot = (id >> 3) % per_pair;
    if (pair >= pairs) return;
    const int split = slot % a.nsplit, tile = a.tiles - 1 - slot / a.nsplit;
    const int b = pair / c.n_head_kv, kvh = pair % c.n_head_kv;
    const Kv4Range rg = kv4_range(a, b, tile, 128);
    if (rg.n_rows <= 0 || (split >= rg.parts && split > 0)) return;

    const int local = 32 * w + n, r = tile * 128 + local;
    const bool on = local < rg.n_rows;
    const int tok = on ? r / a.rep : 0, head = kvh * a.rep + (on ? r % a.rep : 0);
    const int lim = on ? rg.len - rg.nq + tok + 1 : 0;
    u32x4 q[2 * G];
    float sc2;
    {
        const long long at = (long long)(rg.lo + tok) * a.q.row + (long long)head * a.q.head;
        float big = 0.0f, up = 1.0f, down = 1.0f;
        if (a.q.type != KV4_F16) {   // as in kv4_decode_kernel: a power of two for the row
#pragma unroll
            for (int k = 0; k < 2 * G; ++k) {
                float x[8];
                if (on && 16 * k + 8 * h < c.head_dim) {
                    kv4_load8(x, a.q, at + 16 * k + 8 * h);
#pragma unroll
                    for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(x[j]));
                }
            }
            big = fmaxf(big, lane_xor32(big));
            const int e = (int)((bits_of(big) >> 23) & 255u);
            if (e > 0 && e < 254) { up = float_of((uint32_t)(254 - e) << 23); down = float_of((uint32_t)e << 23); }
        }
#pragma unroll
        for (int k = 0; k < 2 * G; ++k) {
            float x[8];
            if (on && 16 * k + 8 * h < c.head_dim) kv4_load8(x, a.q, at + 16 * k + 8 * h);
            else for (int j = 0; j < 8; ++j) x[j] = 0.0f;
            q[k] = u32x4_of(kv4_cvt2(x[0] * up, x[1] * up), kv4_cvt2(x[2] * up, x[3] * up), kv4_cvt2(x[4] * up, x[5] * up), kv4_cvt2(x[6] * up, x[7] * up));
        }
        sc2 = a.scale * 1.44269504088896f * down;
    }
    float mx = -INFINITY, sum = 0.0f;
    f32x16 O[G];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < 16; ++e) O[g][e] = 0.0f;
    const int begin = split * rg.per, end = begin + rg.per < rg.nb ? begin + rg.per : rg.nb;
    const int last_row = 32 * w + 31 < rg.n_rows ? 32 * w + 31 : rg.n_rows - 1;            // what the wave's rows see: all below `wfree`, none from `wend` on
    const int wend = 32 * w < rg.n_rows ? rg.len - rg.nq + (tile * 128 + last_row) / a.rep + 1 : 0;
    const int wfree = 32 * w < rg.n_rows ? rg.len - rg.nq + (tile * 128 + 32 * w) / a.rep + 1 : 0;

    // staging: a thread unpacks, of one block of the pair, K's G dwords of (token st, quad si) and V's dims sd, sd + 32, .. of the tokens' eight si
    const int sb = tid >> 7, st = (tid >> 2) & 31, si = tid & 3, sd = tid & 31, ve = (tid >> 5) & 3;
    uint32_t kc[G], ks[G], vc[G], vs[G][4];
    bool got = false;
    auto fetch = [&](int blk) {
        const int bb = blk + sb;
        const uint8_t* p = bb < end ? kv4_block(c, b, kvh, bb) : nullptr;
        got = p != nullptr;
        if (!got) return;
        kv4_ldw<G>(kc, p + ((st * 4 + si) * G) * 4);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            ks[g] = ((const uint16_t*)(p + 1024 * G))[(((st >> 4) * 4 + ((st & 15) >> 2)) * G + g) * 4 + (st & 3)];
            vc[g] = ((const uint32_t*)(p + 512 * G))[ve * 32 * G + 32 * g + sd];
            const u32x4 s = ld16(p + 1088 * G + (ve * G + g) * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) vs[g][j] = s[j];
        }
    };
    auto stage = [&](int blk, int buf) {
        unsigned char* kb = smem + (buf * 2 + sb) * L::BLK;
        unsigned char* vb = kb + L::KB;
        const int p0 = (blk + sb) * 32;
        uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
        if (p0 + 32 > rg.len) {
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const int t0 = p0 + 16 * (p / 2) + 4 * ve + 2 * (p & 1);
                keep[p] = (t0 < rg.len ? 0xFFFFu : 0u) | (t0 + 1 < rg.len ? 0xFFFF0000u : 0u);
            }
        }
        // an absent block: K is NaN only where it is masked anyway (see `gone`), V is 0
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const uint32_t s = got ? ks[g] | (ks[g] << 16) : 0u;
            lds_st16(kb + (4 * g + si) * L::KC + st * 16, got ? kv4_values(kc[g], s, s, s, s) : u32x4_of(0, 0, 0, 0));
            lds_st16(vb + (ve * 32 * G + 32 * g + sd) * 16,
                     got ? kv4_values(vc[g], vs[g][0] & keep[0], vs[g][1] & keep[1], vs[g][2] & keep[2], vs[g][3] & keep[3]) : u32x4_of(0, 0, 0, 0));
        }
    };
    const int tk = 16 * ((n >> 3) & 1) + 8 * (n >> 4) + 4 * ((n >> 2) & 1) + (n & 3);   // the token that this lane's row of K's operand is
    auto compute = [&](int blk, int buf) {
        const int p0 = blk * 32;
        if (p0 >= wend) return;
        f32x16 S[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const unsigned char* kb = smem + (buf * 2 + k) * L::BLK;
#pragma unroll
            for (int g = 0; g < 2 * G; ++g) {
                const u32x4 kf = lds_ld16(kb + (2 * g + h) * L::KC + tk * 16);
                S[k] = g == 0 ? mfma_f16_32x32x16(kf, q[g]) : mfma_f16_32x32x16_acc(kf, q[g], S[k]);
            }
        }
        const bool gone0 = !kv4_block(c, b, kvh, uniform_int(blk)), gone1 = blk + 1 >= end || !kv4_block(c, b, kvh, uniform_int(blk + 1));
        const bool edge = p0 + 64 > wfree || gone0 || gone1;
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                S[k][e] *= sc2;
                if (edge) {
                    const int p = p0 + 32 * k + 16 * ((e >> 2) & 1) + 8 * (e >> 3) + 4 * h + (e & 3);
                    if (p >= lim || (k ? gone1 : gone0)) S[k][e] = -INFINITY;
                }
                top = fmaxf(top, S[k][e]);
            }
        if (__ballot(top > mx + 8.0f)) {
            top = fmaxf(top, lane_xor32(top));
            const float now = fmaxf(mx, top);
            const float f = now == -INFINITY ? 1.0f : exp2_fast(mx - now);
            mx = now;
            sum *= f;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int e = 0; e < 16; ++e) O[g][e] *= f;
        }
        const float base = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const unsigned char* vb = smem + (buf * 2 + k) * L::BLK + L::KB;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                uint32_t pk[4];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float x = exp2_fast(S[k][8 * t + e] - base), y = exp2_fast(S[k][8 * t + e + 1] - base);
                    sum += x;
                    sum += y;
                    pk[e / 2] = kv4_cvt2(x, y);
                }
                const u32x4 P = u32x4_of(pk[0], pk[1], pk[2], pk[3]);
#pragma unroll
                for (int g = 0; g < G; ++g) O[g] = mfma_f16_32x32x16_acc(lds_ld16(vb + ((2 * t + h) * 32 * G + 32 * g + n) * 16), P, O[g]);
            }
        }
    };
    if (begin < end) {
        fetch(begin);
        stage(begin, 0);
        int buf = 0;
        for (int blk = begin; blk < end; blk += 2, buf ^= 1) {
            __syncthreads();
            const bool more = blk + 2 < end;
            if (more) fetch(blk + 2);
            compute(blk, buf);
            if (more) stage(blk + 2, buf ^ 1);
        }
    }
    sum += lane_xor32(sum);
    if (!on) return;
    if (rg.parts <= 1) {
        const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
        const long long at = (long long)(rg.lo + tok) * a.o_row + (long long)head * a.o_head;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int d = 32 * g + 2 * e + 4 * h;
                if (d >= c.head_dim) continue;
#pragma unroll
                for (int j = 0; j < 4; ++j) kv4_store_any(a.out, at + d + j, a.out_type, O[g][e + j] * f);
            }
    } else {
        float* o = a.ws + (((long long)tile * pairs + pair) * a.nsplit + split) * 128 * (c.head_dim + 2) + (long long)local * (c.head_dim + 2);
        if (h == 0) { o[0] = mx; o[1] = sum; }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int d = 32 * g + 8 * (e >> 2) + 4 * h + (e & 3);
                if (d < c.head_dim) o[2 + d] = O[g][e];
            }
    }
}
