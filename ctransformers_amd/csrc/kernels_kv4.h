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
#include "kv4.h"

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
static inline uint32_t kv4_fma2(uint32_t a, uint32_t b, uint32_t c) {   // (used where the result is exact)
    uint32_t r = 0;
    for (int s = 0; s < 32; s += 16) r |= (uint32_t)f32_to_f16_bits(fmaf(f16_bits_to_f32((uint16_t)(a >> s)), f16_bits_to_f32((uint16_t)(b >> s)), f16_bits_to_f32((uint16_t)(c >> s)))) << s;
    return r;
}
static inline float kv4_sum2(uint32_t a, float c) { return c + (f16_bits_to_f32((uint16_t)(a & 0xFFFFu)) + f16_bits_to_f32((uint16_t)(a >> 16))); }
static inline uint32_t kv4_and_or(uint32_t a, uint32_t b, uint32_t c) { return (a & b) | c; }
static inline float exp2_fast(float x) { return exp2f(x); }
static inline u32x4 u32x4_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return u32x4{{a, b, c, d}}; }
static inline f32x4 f32x4_splat(float x) { return f32x4{{x, x, x, x}}; }
static inline uint32_t bits_of(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
static inline float float_of(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
#else
typedef _Float16 kv4_h2 __attribute__((ext_vector_type(2)));
DEV uint32_t kv4_add2(uint32_t a, uint32_t b) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(kv4_h2, a) + __builtin_bit_cast(kv4_h2, b)); }
DEV uint32_t kv4_mul2(uint32_t a, uint32_t b) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(kv4_h2, a) * __builtin_bit_cast(kv4_h2, b)); }
DEV uint32_t kv4_cvt2(float a, float b) { return __builtin_bit_cast(uint32_t, kv4_h2{(_Float16)a, (_Float16)b}); }   // nearest even
DEV uint32_t kv4_fma2(uint32_t a, uint32_t b, uint32_t c) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(kv4_h2, a), __builtin_bit_cast(kv4_h2, b), __builtin_bit_cast(kv4_h2, c)));
}
DEV float kv4_sum2(uint32_t a, float c) { return __builtin_amdgcn_fdot2(__builtin_bit_cast(kv4_h2, a), kv4_h2{(_Float16)1.0f, (_Float16)1.0f}, c, false); }
DEV uint32_t kv4_and_or(uint32_t a, uint32_t b, uint32_t c) {   // one instruction; the compiler makes two
    uint32_t r;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "s"(b), "v"(c));   // (one scalar operand an instruction)
    return r;
}
DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }   // v_exp_f32: 1 ulp, results below 2^-126 are 0
DEV u32x4 u32x4_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return u32x4{a, b, c, d}; }
DEV f32x4 f32x4_splat(float x) { return f32x4{x, x, x, x}; }
DEV uint32_t bits_of(float f) { return __builtin_bit_cast(uint32_t, f); }
DEV float float_of(uint32_t u) { return __builtin_bit_cast(float, u); }
#endif
// an index that the compiler has to take as new: what follows from it is computed where it is used and not kept in registers around an outer loop
#ifdef CT_EMU
static inline int kv4_anew(int v) { return v; }
#else
DEV int kv4_anew(int v) { asm volatile("" : "+v"(v)); return v; }
#endif
// An entry of table, lens or cu: constant while a kernel runs, so that a load with a uniform index goes through the scalar cache — as a vector load it would wait
// behind every K and V load in flight.
#ifdef CT_EMU
static inline int kv4_entry(const int* p, long long i) { return p[i]; }
#else
DEV int kv4_entry(const int* p, long long i) { return ((const __attribute__((address_space(4))) int*)p)[i]; }
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
// eight neighbouring dims of a 16-bit type as they are
DEV u32x4 kv4_load8_raw(const Kv4Rows& r, long long at) {
    if (r.vec) return ld16((const uint16_t*)r.p + at);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = (uint32_t)((const uint16_t*)r.p)[at + 2 * j * r.dim] | ((uint32_t)((const uint16_t*)r.p)[at + (2 * j + 1) * r.dim] << 16);
    return u32x4_of(w[0], w[1], w[2], w[3]);
}
DEV void kv4_load8(float (&x)[8], const Kv4Rows& r, long long at) {
    if (r.type != KV4_F32) {
        const u32x4 w = kv4_load8_raw(r, at);
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
        for (int j = 0; j < 8; ++j) x[j] = ((const float*)r.p)[at + j * r.dim];
    }
}
// A query row's pieces as halves: N pieces of eight dims, piece k at at + 8 * (k * step + lane's), dims from head_dim on are zeros.  Rows that f16 may not hold (bf16,
// f32) are scaled by a power of two that brings the row's largest value into [1, 2) — all lanes that hold pieces of a row agree on it through `across` — so that bf16
// stays exact but for values below 2^-17 of the largest.  float32 is rounded to f16's 11 bits, 2^-11 of a value: the products that stream the codes at memory speed, and
// those that keep up with a prompt, take halves; a second half of q would be another product for each of K's.  Returns the inverse of the scale.
// A negative `scale` goes into the query's sign: scores can then be compared before they are scaled.
template <int N, class Across> DEV float kv4_query(u32x4 (&q)[N], const Kv4Rows& r, long long at, int d0, int step, int head_dim, bool on, float scale, Across across) {
    const uint32_t flip = scale < 0.0f ? 0x80008000u : 0u;
    if (r.type == KV4_F16) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const bool in = on && d0 + step * k < head_dim;
            q[k] = kv4_load8_raw(r, in ? at + d0 + step * k : at);
            q[k] = in ? u32x4_of(q[k][0] ^ flip, q[k][1] ^ flip, q[k][2] ^ flip, q[k][3] ^ flip) : u32x4_of(0, 0, 0, 0);
        }
        return 1.0f;
    }
    float x[N][8], big = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const bool in = on && d0 + step * k < head_dim;
        kv4_load8(x[k], r, in ? at + d0 + step * k : at);
#pragma unroll
        for (int j = 0; j < 8; ++j) { x[k][j] = in ? x[k][j] : 0.0f; big = fmaxf(big, fabsf(x[k][j])); }
    }
    big = across(big);
    float up = 1.0f, down = 1.0f, low = 1.0f;
    if (big < 0x1p-64f && big > 0.0f) {   // subnormals' exponents say nothing: 2^64 more, exactly
        big *= 0x1p64f;
        low = 0x1p-64f;
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[k][j] *= 0x1p64f;
    }
    int e = (int)((bits_of(big) >> 23) & 255u);
    e = e == 254 ? 253 : e;               // (the largest rows come to [2, 4): 2^-127 is no normal number)
    if (e > 0 && e < 254) { up = float_of((uint32_t)(254 - e) << 23); down = float_of((uint32_t)e << 23) * low; }
#pragma unroll
    for (int k = 0; k < N; ++k)
        q[k] = u32x4_of(kv4_cvt2(x[k][0] * up, x[k][1] * up) ^ flip, kv4_cvt2(x[k][2] * up, x[k][3] * up) ^ flip, kv4_cvt2(x[k][4] * up, x[k][5] * up) ^ flip,
                        kv4_cvt2(x[k][6] * up, x[k][7] * up) ^ flip);
    return down;
}
// The factor of a score in front of exp2: positive, also for a scale of 0 (whose scores are then as good as equal), so that -inf stays what it is; and at most 2^86,
// where unequal scores (2^-72 apart at least) have become further apart than exp2 can tell, and none overflows (float16 queries of 65504 with such keys: 2^40).
DEV float kv4_factor(float scale, float down, float unit) { return fminf(fmaxf((fabsf(scale) * down) * (1.44269504088896f * unit), 1e-30f), 0x1p86f); }
// exp2's arguments are fma(score, factor, -maximum): one shift by the rounded maximum for all of a row's weights, which their quotients do not see.  From here on that
// rounding could carry the largest weight out of the halves' range (and out of exp2's, further up): such rows round the products first, so that the maximum is one of them.
constexpr float kFar = 0x1p22f;
// Weights are halves for the matrix instructions.  They are relative to a number that lies kRaise below the row's running maximum and is moved only when a score passes that
// maximum by more than kLag: at most 2^15, and what is lost at the small end lies 2^-(24 + kRaise) below the maximum instead of 2^-24 (a long flat tail counts).
constexpr float kRaise = 11.0f, kLag = 15.0f - kRaise;   // (a prompt of 2048 tokens, us: 71.2 with 7, 71.4 with 9, 72.1 with 11; with 14 maxima move often, 5 % more; token steps the same)
// eight neighbouring dims out; vec: as for loads
DEV void kv4_store8(void* p, long long at, int type, int vec, const float (&x)[8]) {
    if (vec && type != KV4_F32) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            w[j] = type == KV4_F16 ? kv4_cvt2(x[2 * j], x[2 * j + 1]) : (uint32_t)bf16_of(x[2 * j]) | ((uint32_t)bf16_of(x[2 * j + 1]) << 16);
        *(u32x4*)((uint16_t*)p + at) = u32x4_of(w[0], w[1], w[2], w[3]);
    } else if (vec) {
        *(u32x4*)((float*)p + at) = u32x4_of(bits_of(x[0]), bits_of(x[1]), bits_of(x[2]), bits_of(x[3]));
        *(u32x4*)((float*)p + at + 4) = u32x4_of(bits_of(x[4]), bits_of(x[5]), bits_of(x[6]), bits_of(x[7]));
    } else {
        for (int j = 0; j < 8; ++j) kv4_store_any(p, at + j, type, x[j]);
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
    lo = c.cu ? kv4_entry(c.cu, b) : 0;
    hi = c.cu ? kv4_entry(c.cu, b + 1) : c.total;
    if (lo < 0) lo = 0;
    if (hi > c.total) hi = c.total;
    if (hi < lo) hi = lo;
    const long long n = (long long)kv4_entry(c.lens, b) + c.len_add;
    len = n < 0 ? 0 : n > (1 << 30) ? 1 << 30 : (int)n;
}
// block `blk` of head h of sequence b, null where the table names no page
DEV uint8_t* kv4_block(const Kv4Cache& c, int b, int h, int blk) {
    const int pi = blk >> c.bshift;
    if (blk < 0 || pi >= c.table_width) return nullptr;
    const int pid = kv4_entry(c.table, (long long)b * c.table_stride + pi);
    if ((unsigned)pid >= (unsigned)c.n_pages) return nullptr;
    const long long in_page = ((long long)h << c.bshift) + (blk & ((1 << c.bshift) - 1));
    return c.pages + (long long)pid * c.page_stride + in_page * c.groups * kKv4Block;
}

// the same in two steps, for loops that look a table entry up well before they need the block: the entry, and the block's address in that page
DEV int kv4_page_of(const Kv4Cache& c, int b, int blk) { return kv4_entry(c.table, (long long)b * c.table_stride + (blk >> c.bshift)); }   // blk < table_width << bshift
DEV const uint8_t* kv4_in_page(const Kv4Cache& c, int pid, int h, int blk) {
    if ((unsigned)pid >= (unsigned)c.n_pages) return nullptr;
    return c.pages + (long long)pid * c.page_stride + (((long long)h << c.bshift) + (blk & ((1 << c.bshift) - 1))) * c.groups * kKv4Block;
}

// ---- rows into the cache --------------------------------------------------------------------------------------------------------------------------
// One workgroup per (block, head) that new rows fall into: it alone writes that block, so a V dword that keeps older tokens is read, changed and written without
// atomics.  A lane takes eight dims (16 bytes of a half row, so that a wave reads whole lines), four lanes a group; they agree on the largest value by two quad
// exchanges.  K codes and scales go straight out, V codes cross the workgroup through LDS (eight tokens to a dword).  All loads of a lane are issued before the
// first value is used.  16 prompts of up to 1500 tokens, 64 heads of 112 in float32 (702 MB in, 113 MB out): 217 us, 3.8 TB/s; one token of 64 sequences, 8 heads:
// 6.4 us, latency (cursor -> table -> rows -> codes -> store).
template <int G> __global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4Append a) {
    __shared__ uint32_t vcode[32][8 * G + 1];   // V codes as bytes [token][dim]; + 1: tokens in different banks
    __shared__ uint16_t sc[2][32][G];
    __shared__ int poison[32];
    const Kv4Cache& c = a.c;
    const int tid = (int)threadIdx.x, h = (int)blockIdx.x % c.n_head_kv, place = (int)blockIdx.x / c.n_head_kv, b = place / a.blocks;   // (heads lie side by side in a row)
    int lo, hi, len;
    kv4_seq(c, b, lo, hi, len);
    const int start = len - (hi - lo);                          // position of the first new row (rows before position 0 are dropped)
    const int blk = (start > 0 ? start : 0) / 32 + place % a.blocks;
    const int stop = hi - lo > a.max_rows ? start + a.max_rows : len;   // behind the last row that is taken
    if (blk * 32 >= stop || hi == lo) return;
    uint8_t* dst = kv4_block(c, b, h, blk);
    if (!dst) return;
    const int t_lo = start > blk * 32 ? start - blk * 32 : 0, t_hi = stop - blk * 32 < 32 ? stop - blk * 32 : 32;   // the new tokens of this block
    if (tid < 32) poison[tid] = 0;
    uint32_t* vd = (uint32_t*)(dst + 512 * G);
    uint32_t old[(G + 1) / 2];   // the V dwords that keep older (or the neighbours of newer) tokens: fetched with the rows, not behind them
    if (t_hi - t_lo < 32) {
#pragma unroll
        for (int k = 0; k < (G + 1) / 2; ++k) old[k] = tid + 256 * k < 4 * 32 * G ? vd[tid + 256 * k] : 0u;
    }
    // piece `it` of 256 G: half (K, V), token, group, eight dims
    float x[G][8];
#pragma unroll
    for (int k = 0; k < G; ++k) {
        const int it = tid + 256 * k, half = it / (128 * G), t = (it / (4 * G)) & 31, d0 = 8 * (it % (4 * G));
#pragma unroll
        for (int j = 0; j < 8; ++j) x[k][j] = 0.0f;
        if (t < t_lo || t >= t_hi || d0 >= c.head_dim) continue;
        const long long at = a.absolute ? blk * 32 + t : (long long)(lo + blk * 32 + t - start);
        if (half) kv4_load8(x[k], a.v, at * a.v.row + (long long)h * a.v.head + d0 * a.v.dim);
        else kv4_load8(x[k], a.k, at * a.k.row + (long long)h * a.k.head + d0 * a.k.dim);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < G; ++k) {
        const int it = tid + 256 * k, half = it / (128 * G), t = (it / (4 * G)) & 31, g = (it / 4) % G, o = it & 3;
        const bool on = t >= t_lo && t < t_hi;
        if (!__ballot(on)) continue;   // (a token step: one wave has work)
        float top = 0.0f;
        int nan = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float v = x[k][j] > 65504.0f ? 65504.0f : x[k][j] < -65504.0f ? -65504.0f : x[k][j];
            nan |= v != v;
            x[k][j] = v;
            if (fabsf(v) > fabsf(top)) top = v;
        }
        // the quad's largest, the first of equals (the four lanes hold the group's dims in order)
        const float t1 = lane_xor1(top);
        top = (o & 1) ? (fabsf(t1) >= fabsf(top) ? t1 : top) : (fabsf(t1) > fabsf(top) ? t1 : top);
        const float t2 = lane_xor2(top);
        top = (o & 2) ? (fabsf(t2) >= fabsf(top) ? t2 : top) : (fabsf(t2) > fabsf(top) ? t2 : top);
        nan |= lane_xor1(nan);
        nan |= lane_xor2(nan);
        const float d = top / -8.0f;
        const uint16_t dh = f32_to_f16_bits(d);
        const float inv = (dh & 0x7FFFu) ? 1.0f / d : 0.0f;     // a scale that f16 has as 0: every value is 0
        uint32_t w = 0, lo4 = 0, hi4 = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float f = x[k][j] * inv + 8.5f;               // two roundings, as the reference's expression has
            const int q = nan ? 8 : (int)f > 15 ? 15 : (int)f;
            w |= (uint32_t)q << (4 * (j / 2) + 16 * (j & 1));
            if (j < 4) lo4 |= (uint32_t)q << (8 * j);
            else hi4 |= (uint32_t)q << (8 * (j - 4));
        }
        if (!on) continue;
        if (o == 0) {
            if (nan) poison[t] = 1;
            sc[half][t][g] = dh;
        }
        if (half) {
            vcode[t][8 * g + 2 * o] = lo4;
            vcode[t][8 * g + 2 * o + 1] = hi4;
        } else {
            ((uint32_t*)dst)[(4 * t + o) * G + g] = w;
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
#pragma unroll
    for (int k = 0; k < (G + 1) / 2; ++k) {
        const int it = tid + 256 * k, i = it / (32 * G), dim = it % (32 * G);
        if (it >= 4 * 32 * G) break;
        uint32_t w = 0, m = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int t = 4 * i + (e & 3) + 16 * (e / 4), sh = 4 * (e / 2) + 16 * (e & 1);
            if (t < t_lo || t >= t_hi) continue;
            w |= ((vcode[t][dim / 4] >> (8 * (dim & 3))) & 15u) << sh;
            m |= 15u << sh;
        }
        if (m) vd[it] = m == 0xFFFFFFFFu ? w : (old[k] & ~m) | w;
    }
}

// The last rows of every sequence out of the cache, as numbers: the mirror image of kv4_append_kernel, same workgroups.  Rows whose page is absent are zeros.
// The same prompts (113 MB in, 351 MB of halves out): 119 us, 3.9 TB/s.
template <int G> __global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4Append a) {
    const Kv4Cache& c = a.c;
    const int tid = (int)threadIdx.x, h = (int)blockIdx.x % c.n_head_kv, place = (int)blockIdx.x / c.n_head_kv, b = place / a.blocks;   // (heads lie side by side in a row)
    int lo, hi, len;
    kv4_seq(c, b, lo, hi, len);
    const int start = len - (hi - lo);
    const int blk = (start >= 0 ? start / 32 : -((31 - start) / 32)) + place % a.blocks;   // rows before position 0 are written too (as zeros)
    const int stop = hi - lo > a.max_rows ? start + a.max_rows : len;
    if (blk * 32 >= stop || hi == lo) return;
    const uint8_t* src = kv4_block(c, b, h, blk);
    const int t_lo = start > blk * 32 ? start - blk * 32 : 0, t_hi = stop - blk * 32 < 32 ? stop - blk * 32 : 32;
#pragma unroll
    for (int k = 0; k < G; ++k) {   // pieces as in kv4_append_kernel
        const int it = tid + 256 * k, half = it / (128 * G), t = (it / (4 * G)) & 31, g = (it / 4) % G, o = it & 3, d0 = 32 * g + 8 * o;
        if (t < t_lo || t >= t_hi || d0 >= c.head_dim) continue;
        const int i = (t & 15) / 4, e = (t & 3) + 4 * (t / 16);
        float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (src && half) {          // one nibble of each of the eight dims' dwords
            const float d = f16_bits_to_f32(((const uint16_t*)(src + 1088 * G))[(i * G + g) * 8 + e]);
            const uint8_t* vd = src + 512 * G + (i * 32 * G + d0) * 4;
            const u32x4 w0 = ld16(vd), w1 = ld16(vd + 16);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = d * (float)((int)(((j < 4 ? w0[j & 3] : w1[j & 3]) >> (4 * (e / 2) + 16 * (e & 1))) & 15u) - 8);
        } else if (src) {
            const float d = f16_bits_to_f32(((const uint16_t*)(src + 1024 * G))[(((t / 16) * 4 + i) * G + g) * 4 + (t & 3)]);
            const uint32_t w = ((const uint32_t*)src)[(4 * t + o) * G + g];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = d * (float)((int)((w >> (4 * (j / 2) + 16 * (j & 1))) & 15u) - 8);
        }
        const long long at = (long long)(lo + blk * 32 + t - start);
        if (half) kv4_store8((void*)a.v.p, at * a.v.row + (long long)h * a.v.head + d0, a.v.type, a.v.vec, x);
        else kv4_store8((void*)a.k.p, at * a.k.row + (long long)h * a.k.head + d0, a.k.type, a.k.vec, x);
    }
}

// ---- attention ------------------------------------------------------------------------------------------------------------------------------------
// The query rows of a (sequence, KV head) are r = token * rep + head, tiles of them share a workgroup; row r sees the positions below
// len - rows + token + 1.  The blocks that a tile sees are divided into parts of `per` blocks, one workgroup each, `nsplit` of them at most (the grid); a part is
// as long as it has to be for all of the call's parts to be about `want_parts`, whatever the sequences' lengths are: they are only known on the device.
DEV int kv4_rows(const Kv4Attn& a, int nq) { return nq < a.max_rows ? nq : a.max_rows; }   // rows of a sequence that are taken
struct Kv4Range { int nq, n_rows, first_tok, len, lo, nb, per, parts; };
DEV int kv4_part(const Kv4Attn& a) {   // every lane of the wave calls it
    if (a.nsplit <= 1) return 1;
    long long sum = 0;
    for (int b = lane_id(); b < a.c.n_seq; b += 64) {
        const long long n = (long long)a.c.lens[b] + a.c.len_add;
        sum += n < 0 ? 0 : (n + 31) / 32;
    }
    sum = wave_sum(sum) * a.c.n_head_kv * a.tiles;
    const long long per = (sum + a.want_parts - 1) / a.want_parts;
    return uniform_int((int)(per < a.min_blocks ? a.min_blocks : per > (1 << 25) ? 1 << 25 : per));
}
DEV Kv4Range kv4_range(const Kv4Attn& a, int b, int tile, int tile_rows, int part) {
    Kv4Range r;
    int lo, hi;
    kv4_seq(a.c, b, lo, hi, r.len);
    r.lo = lo;
    r.nq = hi - lo;
    const int row0 = tile * tile_rows, all = kv4_rows(a, r.nq) * a.rep;
    r.n_rows = all - row0 < tile_rows ? all - row0 : tile_rows;
    r.first_tok = row0 / a.rep;
    const int last_tok = (row0 + r.n_rows - 1) / a.rep;
    const int seen = r.n_rows > 0 ? r.len - r.nq + last_tok + 1 : 0;   // positions that the tile's last row sees
    r.nb = seen > 0 ? (seen + 31) / 32 : 0;
    if (r.nb > a.c.table_width << a.c.bshift) r.nb = a.c.table_width << a.c.bshift;   // what the table has no room for is absent
    r.per = (r.nb + a.nsplit - 1) / a.nsplit;
    if (r.per < part) r.per = part;
    r.parts = (r.nb + r.per - 1) / r.per;
    return r;
}

// kv4_decode_kernel: the work of all units — a unit is a (sequence, KV head, row tile) — stands in one line, which is cut into equal shares, one per workgroup, as
// many as are resident at once.  So every workgroup has the same work whatever the sequences' lengths are.  A unit's work is its blocks and, before them, kUnitCost
// blocks' worth for beginning and ending it: the queries, the first loads, the waves' results joined, one latency after the other.  (64 sequences of 0 .. 8192 tokens,
// 8 KV heads: 98 us at 4 blocks, 75 at 10, 70.5 at 14, 71 at 20, 72 at 28, 75 at 40.)
// Only the first and the last unit of a share can be a part of one; a part that does not begin its unit goes to the share's first place in the workspace, one that
// begins it to the second, whole units go straight out.  The line follows from lens and cu, which only the device knows: every wave sums it up for itself.
struct Kv4Line { int before, all, per; };                     // (the host refuses tables with room for 2^31 blocks)
DEV int kv4_unit_blocks(const Kv4Attn& a, int nq, int len) {   // blocks of each of a sequence's units (one, all masked, where there is nothing to see), 0: no rows
    if (nq <= 0) return 0;
    const int cap = a.c.table_width << a.c.bshift, nb = (len + 31) / 32;
    return nb < 1 ? 1 : nb > cap ? (cap < 1 ? 1 : cap) : nb;
}
DEV int kv4_tiles(const Kv4Attn& a, int nq, int tile_rows) {
    return (kv4_rows(a, nq) * a.rep + tile_rows - 1) / tile_rows;   // (at most a.tiles; 2^31 rows times heads at most: the host's check)
}
DEV int kv4_seq_work(const Kv4Attn& a, int tile_rows, int b) {
    if (b >= a.c.n_seq) return 0;
    int lo, hi, len;
    kv4_seq(a.c, b, lo, hi, len);
    const int nb = kv4_unit_blocks(a, hi - lo, len);
    return nb ? (nb + kUnitCost) * kv4_tiles(a, hi - lo, tile_rows) * a.c.n_head_kv : 0;
}
// all the work of the line, and what lies before sequence `stop`
DEV Kv4Line kv4_line(const Kv4Attn& a, int tile_rows, int stop) {
    int all = 0, before = 0;
    for (int b = lane_id(); b < ((a.c.n_seq + 63) & ~63); b += 64) {
        const int n = kv4_seq_work(a, tile_rows, b);
        all += n;
        before += b < stop ? n : 0;
    }
    Kv4Line r;
    r.all = uniform_int(wave_sum_fast(all));
    r.before = stop > 0 ? uniform_int(wave_sum_fast(before)) : 0;
    const int per = (int)(((long long)r.all + a.want_parts - 1) / a.want_parts);
    r.per = per < a.min_blocks + kUnitCost ? a.min_blocks + kUnitCost : per;
    return r;
}
// the sequence that place x of the line belongs to, and where that sequence begins
DEV int kv4_find(const Kv4Attn& a, int tile_rows, int x, int& begin) {
    int at = 0;
    for (int b0 = 0; b0 < a.c.n_seq; b0 += 64) {
        const int lane = lane_id(), n = kv4_seq_work(a, tile_rows, b0 + lane);
        int sum = n;                                           // inclusive
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl(sum, lane >= d ? lane - d : lane);
            if (lane >= d) sum += y;
        }
        const unsigned long long in = __ballot(n > 0 && x < at + sum);
        if (in) {
            const int l = __ffsll(in) - 1;
            begin = uniform_int(at + __shfl(sum - n, l));
            return b0 + l;
        }
        at += __shfl(sum, 63);
    }
    begin = uniform_int(at);
    return a.c.n_seq;
}

// Eight halves of the dword's codes minus 8, times the scales of their tokens (or one scale for all): f16 products, one rounding (2^-11 of a value whose step is
// 1/8 of the group's largest) — the matrix instruction takes halves.
DEV u32x4 kv4_values(uint32_t w, uint32_t s0, uint32_t s1, uint32_t s2, uint32_t s3) {
    // halves 1024 + code (low nibbles of the bytes) and 1024 + 16 code (high nibbles: no shift); - 1032 and / 16 - 72 give code - 8, all of it exact
    const uint32_t lo = 0x000F000Fu, hi = 0x00F000F0u, K = 0x64006400u, u = w >> 8;
    const uint32_t v0 = kv4_add2(kv4_and_or(w, lo, K), 0xE408E408u), v1 = kv4_fma2(kv4_and_or(w, hi, K), 0x2C002C00u, 0xD480D480u);
    const uint32_t v2 = kv4_add2(kv4_and_or(u, lo, K), 0xE408E408u), v3 = kv4_fma2(kv4_and_or(u, hi, K), 0x2C002C00u, 0xD480D480u);
    return u32x4_of(kv4_mul2(v0, s0), kv4_mul2(v1, s1), kv4_mul2(v2, s2), kv4_mul2(v3, s3));
}

// Few rows (a token step, a handful of drafted tokens): a wave takes whole blocks.  16x16x32 matrix products, transposed so that a query row is a COLUMN of both:
//   S = K_codes (A: lane = token) x Q (B: lane = row): lane (row, quad) then holds the scores of tokens 4 quad .. 4 quad + 3 of both 16-token tiles
//   O = V^T (A: lane = dim) x P (B: lane = row): those eight probabilities ARE the lane's k slots — V is stored in that order
// K's codes enter as f16 SUBNORMALS, the 16-bit integers themselves (code * 2^-24: no conversion); -8 * sum(Q) is the product's C operand and the group's scale
// multiplies the 32-dim product in f32, so K is used exactly.  Maximum, sum and O stay per lane in f32; the maximum is raised (and O rescaled) only when a score
// passes it by more than 2^kLag, so most blocks exchange nothing between lanes.  P enters as two halves, the rounded one and what it left (the matrix cores have the time:
// +2 % at most): off by 2^-22 of p, or 2^-36 of the row's largest where p is smaller than that allows.  V's product with its scale is one half, 2^-11.
// One sequence of 130 000 tokens, 8 KV heads of 128 with 8 query heads each (150 MB): 35 us, 4.3 TB/s; 64 sequences of 0 .. 8192 tokens (303 MB): 71 us, 4.3 TB/s.  A large
// copy moves 4.66 TB/s, reading alone reaches 6.4 .. 6.6: memory is not all of it.  Counters of the second: vector units 56 % busy, matrix cores 14 %, 2.1 waves a SIMD,
// which wait for data 30 % and for their turn to issue 36 % of their time.  One sequence of 140 tokens: 7.5 us, latency.
// The next block's K is fetched into the registers of this one's as soon as its scores are there, its V after the V product: 40 dwords a lane at 128 dims for a
// block in flight, which leaves room for three waves a SIMD (146 registers).
template <int G> DEV void kv4_fetch_k(uint32_t (&kc)[2][G], uint32_t (&ks)[2][2 * G], const uint8_t* blk, int m, int i) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        kv4_ldw<G>(kc[t], blk + (((t * 16 + m) * 4 + i) * G) * 4);
        kv4_ldw<2 * G>(ks[t], blk + 1024 * G + ((t * 4 + i) * G) * 8);
    }
}
template <int G> DEV void kv4_fetch_v(uint32_t (&vc)[2 * G], uint32_t (&vs)[2 * G + 2 * (G & 1)], const uint8_t* blk, int m, int i) {
#pragma unroll
    for (int p = 0; p < G / 2; ++p) {   // 64 dims: four neighbouring ones a lane
        const u32x4 w = ld16(blk + 512 * G + (i * 32 * G + 64 * p + 4 * m) * 4), s = ld16(blk + 1088 * G + (i * G + 2 * p + (m >> 3)) * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) { vc[4 * p + j] = w[j]; vs[4 * p + j] = s[j]; }
    }
    if constexpr (G & 1) {              // 32 dims: two a lane
        const u32x2 w = ld8(blk + 512 * G + (i * 32 * G + 32 * (G - 1) + 2 * m) * 4);
        const u32x4 s = ld16(blk + 1088 * G + (i * G + G - 1) * 16);
        vc[2 * G - 2] = w[0]; vc[2 * G - 1] = w[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) vs[2 * (G - 1) + j] = s[j];
    }
}
// row `row` of the tile, `dim` of the head that register r of dim tile `j` holds for quad i
template <int G> DEV int kv4_dim(int j, int i, int r) {
    return j < 4 * (G / 2) ? 64 * (j / 4) + 16 * i + 4 * r + (j & 3) : 32 * (G - 1) + 8 * i + 2 * r + (j & 1);
}

template <int G, int NT> __global__ void __launch_bounds__(256, G * NT <= 2 ? 4 : G * NT <= 4 ? 3 : 2) kv4_decode_kernel(const Kv4Attn a) {
    constexpr int W = 4, DP = 32 * G, PITCH = DP + 4, ROWS = 16 * NT;
    // -8 sum(q) is the K product's C operand, four registers of one value; two tiles of 128 dims have no room for them (20 registers were spilled) and add it afterwards.
    // us for 12, 24, 48 rows a KV head behind 4000 tokens, 16 sequences: 42 / 38, 46 / 42, 48 / 45 added afterwards; with one tile 66 / 68 (64 sequences).
    constexpr bool LATE = G == 4 && NT == 2;
    CT_DYN_SMEM(smem);
    float* part = (float*)smem;                       // [wave][row][PITCH] of one row tile
    float* stat = part + W * 16 * PITCH;              // [wave][ROWS][2]: maximum, sum
    const Kv4Cache& c = a.c;
    const int w = uniform_int(wave_id());
    // this workgroup's share [x, x_end) of the line; without a split a workgroup is one unit
    int x = 0, x_end = 1, seq_begin = 0;
    int b, in_seq;                                    // the unit's sequence, its index there
    if (a.nsplit > 1) {
        const Kv4Line line = kv4_line(a, ROWS, 0);
        if ((long long)blockIdx.x * line.per >= line.all) return;
        x = (int)blockIdx.x * line.per;
        x_end = line.all - x < line.per ? line.all : x + line.per;
        b = kv4_find(a, ROWS, x, seq_begin);
        in_seq = 0;
    } else {
        const int per_seq = c.n_head_kv * a.tiles;
        b = uniform_int((int)blockIdx.x / per_seq);
        in_seq = (int)blockIdx.x - b * per_seq;
    }
  while (x < x_end && b < c.n_seq) {   // (the second holds by itself unless lens or cu change meanwhile)
    const int lane = kv4_anew(lane_id()), m = lane & 15, i = lane >> 4;
    int lo, hi, len;
    kv4_seq(c, b, lo, hi, len);
    const int nq = hi - lo, nb = kv4_unit_blocks(a, nq, len), tiles = kv4_tiles(a, nq, ROWS);
    int begin = 0, end = nb;
    if (a.nsplit > 1) {
        const int unit = nb + kUnitCost;
        if (nb == 0 || x - seq_begin >= unit * tiles * c.n_head_kv) {   // on to the next sequence
            seq_begin += nb == 0 ? 0 : unit * tiles * c.n_head_kv;
            ++b;
            continue;
        }
        in_seq = uniform_int((x - seq_begin) / unit);
        const int at = x - seq_begin - in_seq * unit;
        begin = at < kUnitCost ? 0 : at - kUnitCost;
        end = x_end - x < unit - at ? at + x_end - x - kUnitCost : nb;
        x += unit - at < x_end - x ? unit - at : x_end - x;
        if (end <= begin) continue;                                     // the share ends before the unit's first block
    } else {
        x = x_end;
        if (in_seq >= tiles * c.n_head_kv) return;
    }
    const int kvh = uniform_int(in_seq / tiles), tile = in_seq - kvh * tiles, row0 = tile * ROWS, all = kv4_rows(a, nq) * a.rep, n_rows = all - row0 < ROWS ? all - row0 : ROWS;
    const bool whole = begin == 0 && end == nb;

    u32x4 q[NT][G];
    f32x4 cq[LATE ? 1 : NT][LATE ? 1 : G];
    float cl[LATE ? NT : 1][LATE ? G : 1];
    float sc2[NT], mx[NT], sum[NT];
    int lim[NT];
    f32x4 O[NT][2 * G];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = row0 + 16 * n + m;
        const bool on = 16 * n + m < n_rows;
        const int tok = on ? r / a.rep : 0;
        lim[n] = on ? len - nq + tok + 1 : 0;
        const long long at = (long long)(lo + tok) * a.q.row + (long long)(kvh * a.rep + (on ? r - tok * a.rep : 0)) * a.q.head;
        const float down = kv4_query<G>(q[n], a.q, at, 8 * i, 32, c.head_dim, on, a.scale, [](float v) { v = fmaxf(v, lane_xor16(v)); return fmaxf(v, lane_xor32(v)); });
#pragma unroll
        for (int g = 0; g < G; ++g) {   // -8 sum(Q) of the group in every row of the product: A all -8 (f16 bits 0x8008: -8 * 2^-24, as the codes are)
            const f32x4 c8 = mfma_f16_16x16x32(u32x4_of(0x80088008u, 0x80088008u, 0x80088008u, 0x80088008u), q[n][g], f32x4_splat(0.0f));
            if constexpr (LATE) cl[n][g] = c8[0];
            else cq[n][g] = c8;
        }
        sc2[n] = kv4_factor(a.scale, down, 16777216.0f);
        mx[n] = -INFINITY;
        sum[n] = 0.0f;
#pragma unroll
        for (int j = 0; j < 2 * G; ++j) O[n][j] = f32x4_splat(0.0f);
    }
    const int free_lim = len - nq + row0 / a.rep + 1;   // every row of the tile sees the positions below

    uint32_t kc[2][G], ks[2][2 * G], vc[2 * G], vs[2 * G + 2 * (G & 1)];
    int blk = begin + w;
    if (c.n_pages <= 0 || c.table_width <= 0) end = begin;   // (nothing to see: the unit's one block is not looked up)
    // Loads are never conditional (a wait for V would have to count K's as not issued, and wait for them too): where there is no block, the pool's first is read
    // and everything in it masked.
    bool here = false;
    int pid = -1;
    if (blk < end) {
        const uint8_t* p = kv4_in_page(c, kv4_page_of(c, b, blk), kvh, blk);
        here = p != nullptr;
        if (blk + W < end) pid = kv4_page_of(c, b, blk + W);
        p = here ? p : c.pages;
        kv4_fetch_k<G>(kc, ks, p, m, i);
        kv4_fetch_v<G>(vc, vs, p, m, i);
    }
    for (; blk < end; blk += W) {
        const int pid2 = blk + 2 * W < end ? kv4_page_of(c, b, blk + 2 * W) : -1;
        const uint8_t* nxt = kv4_in_page(c, pid, kvh, blk + W);
        const bool next_here = nxt != nullptr;
        nxt = next_here ? nxt : c.pages;
        const int p0 = blk * 32, there = here ? len : 0;   // tokens from `there` on are not there
        float s[NT][2][4];
        {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const uint32_t k = kc[t][g], M = 0x000F000Fu;
                    const u32x4 kf = u32x4_of(k & M, (k >> 4) & M, (k >> 8) & M, (k >> 12) & M);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        f32x4 acc;
                        if constexpr (LATE) acc = mfma_f16_16x16x32(kf, q[n][g], f32x4_splat(0.0f));
                        else acc = mfma_f16_16x16x32(kf, q[n][g], cq[n][g]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t d2 = ks[t][2 * g + e / 2];
                            const float d = f16_bits_to_f32((uint16_t)(e & 1 ? d2 >> 16 : d2 & 0xFFFFu));
                            const float x = LATE ? acc[e] + cl[LATE ? n : 0][LATE ? g : 0] : acc[e];
                            s[n][t][e] = g == 0 ? d * x : fmaf(d, x, s[n][t][e]);
                        }
                    }
                }
        }
        kv4_fetch_k<G>(kc, ks, nxt, m, i);
        {
            u32x4 P[NT], PL[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (p0 + 32 > free_lim || p0 + 32 > there) {
                    const int left = here ? lim[n] - p0 - 4 * i : -1;   // tokens of this lane's from here on that the row does not see
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[n][t][e] = 16 * t + e >= left ? -INFINITY : s[n][t][e];
                }
                float top = s[n][0][0];
#pragma unroll
                for (int e = 1; e < 8; ++e) top = fmaxf(top, s[n][e / 4][e & 3]);
                top *= sc2[n];
                if (__ballot(top > mx[n] + (kRaise + kLag))) {   // (also the first block: -inf + 15)
                    top = fmaxf(top, lane_xor16(top));
                    top = fmaxf(top, lane_xor32(top));
                    const float now = fmaxf(mx[n], top - kRaise);
                    const float f = now == -INFINITY ? 1.0f : exp2_fast(mx[n] - now);
                    mx[n] = now;
                    sum[n] *= f;
#pragma unroll
                    for (int j = 0; j < 2 * G; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) O[n][j][e] *= f;
                }
                float base = mx[n] == -INFINITY ? 0.0f : -mx[n], factor = sc2[n];
                if (__ballot(fabsf(base) > kFar)) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[n][e / 4][e & 3] = s[n][e / 4][e & 3] * factor + base;
                    factor = 1.0f;
                    base = 0.0f;
                }
                uint32_t pk[4], lo[4];
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const float x = exp2_fast(fmaf(s[n][p / 2][2 * (p & 1)], factor, base)), y = exp2_fast(fmaf(s[n][p / 2][2 * (p & 1) + 1], factor, base));
                    pk[p] = kv4_cvt2(x, y);
                    sum[n] += x;
                    sum[n] += y;
                    lo[p] = kv4_cvt2(x - f16_bits_to_f32((uint16_t)(pk[p] & 0xFFFFu)), y - f16_bits_to_f32((uint16_t)(pk[p] >> 16)));
                }
                P[n] = u32x4_of(pk[0], pk[1], pk[2], pk[3]);
                PL[n] = u32x4_of(lo[0], lo[1], lo[2], lo[3]);
            }
            if (p0 + 32 > there) {   // whatever the page holds past the sequence's end must not meet p = 0 as an infinity
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const int t0 = p0 + 16 * (p / 2) + 4 * i + 2 * (p & 1);
                    const uint32_t keep = (t0 < there ? 0xFFFFu : 0u) | (t0 + 1 < there ? 0xFFFF0000u : 0u);
#pragma unroll
                    for (int j = 0; j < 2 * G + 2 * (G & 1); j += 4) vs[j + p] &= keep;
                }
            }
#pragma unroll
            for (int j = 0; j < 2 * G; ++j) {
                const int s0 = j < 4 * (G / 2) ? 4 * (j / 4) : 2 * (G - 1);
                const u32x4 v = kv4_values(vc[j], vs[s0], vs[s0 + 1], vs[s0 + 2], vs[s0 + 3]);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    O[n][j] = mfma_f16_16x16x32(v, P[n], O[n][j]);
                    O[n][j] = mfma_f16_16x16x32(v, PL[n], O[n][j]);
                }
            }
        }
        kv4_fetch_v<G>(vc, vs, nxt, m, i);
        here = next_here;
        pid = pid2;
    }
    // the waves' results meet in LDS, in wave order
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        sum[n] += lane_xor16(sum[n]);
        sum[n] += lane_xor32(sum[n]);
        if (i == 0) { stat[(w * 16 * NT + 16 * n + m) * 2] = mx[n]; stat[(w * 16 * NT + 16 * n + m) * 2 + 1] = sum[n]; }
    }
    float* out = a.ws + ((long long)blockIdx.x * 2 + (begin == 0)) * ROWS * (c.head_dim + 2);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        if (n) __syncthreads();
#pragma unroll
        for (int j = 0; j < 2 * G; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[(w * 16 + m) * PITCH + kv4_dim<G>(j, i, e)] = O[n][j][e];
        __syncthreads();
        for (int it = 64 * w + lane; it < 16 * DP; it += 64 * W) {
            const int row = it / DP, dim = it % DP;
            if (16 * n + row >= n_rows || dim >= c.head_dim) continue;
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
                kv4_store_any(a.out, (long long)(lo + r / a.rep) * a.o_row + (long long)(kvh * a.rep + r % a.rep) * a.o_head + dim, a.out_type, L == 0.0f ? 0.0f : v / L);
            } else {
                float* o = out + (16 * n + row) * (c.head_dim + 2);
                o[2 + dim] = v;
                if (dim == 0) { o[0] = M; o[1] = L; }
            }
        }
    }
    if (a.nsplit > 1) __syncthreads();   // LDS is the next unit's
  }
}

// The parts of a row joined: a workgroup of W waves per (row, head); a wave takes every W-th part, four at a time, two dims a lane, with a maximum of its own.
// LINE: parts are shares' ends (kv4_decode_kernel), else the splits of kv4_prompt_kernel.  6.5 us for 64 rows of 95 parts as for 4096 rows of one or two: latency.
// (A join by the last workgroup to arrive would save this launch, but its counters would have to survive between calls: two graphs could meet in them.)
template <int NR, bool LINE, int W> __global__ void __launch_bounds__(64 * W) kv4_join_kernel(const Kv4Attn a, int tile_rows) {
    __shared__ float acc[W][128 * NR], stat[W][2];
    const Kv4Cache& c = a.c;
    const int lane = lane_id(), w = uniform_int(wave_id()), row = (int)blockIdx.x / a.n_head, head = (int)blockIdx.x % a.n_head;
    int b = 0;
    if (c.cu) {   // the last sequence that begins at or before the row (their number, less one)
        int n = 0;
        for (int k = 0; k < c.n_seq; k += 64) n += __popcll(__ballot(k + lane < c.n_seq && c.cu[k + lane] <= row));
        b = uniform_int(n) - 1;
        if (b < 0 || row >= c.cu[b + 1]) return;   // behind the last sequence
    }
    int lo, hi, len;
    kv4_seq(c, b, lo, hi, len);
    if (row < lo || row - lo >= a.max_rows) return;   // (cu does not ascend; rows that are not taken)
    const int kvh = head / a.rep, r = (row - lo) * a.rep + head % a.rep, tile = r / tile_rows, dim = c.head_dim;
    const long long step = (long long)tile_rows * (dim + 2);
    int parts;
    const float *in, *in0;   // part 0 and the others' origin
    if constexpr (LINE) {
        const Kv4Line line = kv4_line(a, tile_rows, b);
        const int nb = kv4_unit_blocks(a, hi - lo, len), tiles = kv4_tiles(a, hi - lo, tile_rows);
        if (tile >= tiles) return;
        const int x = line.before + (kvh * tiles + tile) * (nb + kUnitCost) + kUnitCost, s0 = x / line.per;   // the unit's first block
        parts = (x + nb - 1) / line.per - s0 + 1;
        in0 = a.ws + (2ll * s0 + 1) * step;
        in = a.ws + 2ll * s0 * step;
    } else {
        if (tile >= a.tiles) return;
        const Kv4Range rg = kv4_range(a, b, tile, tile_rows, kv4_part(a));
        parts = rg.parts;
        in0 = in = a.ws + ((long long)(tile * ((long long)c.n_seq * c.n_head_kv) + (long long)b * c.n_head_kv + kvh) * a.nsplit) * step;
    }
    if (parts <= 1) return;
    const long long at_row = (long long)(r % tile_rows) * (dim + 2);
    float M = -INFINITY, L = 0.0f, o[2 * NR];
#pragma unroll
    for (int j = 0; j < 2 * NR; ++j) o[j] = 0.0f;
    for (int s0 = w; s0 < parts; s0 += 4 * W) {
        float pm[4], pl[4], now = M;
        u32x2 v[4][NR];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int s = s0 + W * k;
            const float* p = (s == 0 || s >= parts ? in0 : in + (LINE ? 2 : 1) * s * step) + at_row;
            pm[k] = p[0];
            pl[k] = p[1];
#pragma unroll
            for (int j = 0; j < NR; ++j) v[k][j] = ld8(p + 2 + (2 * lane + 128 * j < dim ? 2 * lane + 128 * j : 0));
            if (s >= parts) pm[k] = -INFINITY;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) now = fmaxf(now, pm[k]);
        const float base = now == -INFINITY ? 0.0f : now, f = exp2_fast(M - base);
        M = now;
        L *= f;
#pragma unroll
        for (int j = 0; j < 2 * NR; ++j) o[j] *= f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (s0 + W * k >= parts) continue;
            const float g = exp2_fast(pm[k] - base);
            L += g * pl[k];
#pragma unroll
            for (int j = 0; j < NR; ++j) { o[2 * j] += g * float_of(v[k][j][0]); o[2 * j + 1] += g * float_of(v[k][j][1]); }
        }
    }
#pragma unroll
    for (int j = 0; j < NR; ++j) { acc[w][128 * j + 2 * lane] = o[2 * j]; acc[w][128 * j + 2 * lane + 1] = o[2 * j + 1]; }
    if (lane == 0) { stat[w][0] = M; stat[w][1] = L; }
    __syncthreads();
    for (int d = (int)threadIdx.x; d < dim; d += 64 * W) {
        float top = -INFINITY, sum = 0.0f, v = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) top = fmaxf(top, stat[k][0]);
        const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const float f = exp2_fast(stat[k][0] - base);
            sum += f * stat[k][1];
            v += f * acc[k][d];
        }
        kv4_store_any(a.out, (long long)row * a.o_row + (long long)head * a.o_head + d, a.out_type, sum == 0.0f ? 0.0f : v / sum);
    }
}

// Many rows (a prompt, a chunk of one): a workgroup of four waves takes 128 rows, a wave 32 of them; the blocks pass through LDS as halves, two at a time, so that a
// block is unpacked once for 128 rows.  32x32x16 products, transposed as above: lane (row, half) of S^T = K Q^T holds sixteen scores of ITS row, which are the k slots
// of O^T = V^T P^T if the lane of K's operand that gives row 16 t + 8 u + 4 h + e of the product reads token 16 u + 4 (2 t + h) + e (V's order again).
// LDS: K as 16-byte chunks [8 dims][token], a chunk column 32 bytes longer than its tokens (the four quads that write a token's chunks fall into different banks),
// V as 16-byte chunks [4 eights of tokens][dim]: both are read and written without bank conflicts.  Two buffers: while one pair of blocks is computed the next is
// fetched into registers, unpacked and written into the other, one barrier a pair.
// The row tiles of one (sequence, KV head) go to one XCD, whose L2 then holds that head's codes for all of them; tiles that see most come first.
// Rounded on the way: K's and V's values and p to halves (2^-11 each at most, p below 2^-25 of the row's largest by up to 2^-36 of that; the 32 x 32 products want halves).  A float16 result is off by 3.8e-4 of its norm, its own
// rounding alone by 2.1e-4; K exact, as in the kernel above, would take 128 more fused multiply-adds and 32 more LDS reads a step.
// 2048 tokens, 32 heads of 128 (34 GFLOP): 72 - 81 us, 424 - 477 TFLOP/s; 4 chunks of up to 512 behind up to 8000 tokens, 64 / 8 heads (252 GFLOP): 333 - 391 us, 645 - 758
// TFLOP/s (a large f16 product: 1142).  Neither pipe is full: counters of the chunks have the vector units 42 % busy and the matrix cores 31 %, with 1.6 waves a SIMD of the two
// that fit, which wait 33 % of their time (the prompt: 26 %, 18 %, 1.2 waves, 35 %).  What is lost is overlap — 270 vector instructions a step and wave beside 1024 cycles of
// matrix products — and the ends of launches, where the longest tiles run alone.  Measured and not taken: one block a step and three waves a SIMD (96 / 421 us), unpacking
// between the K.Q products (82 / 371), wave priorities around them (no change), all pairs' long tiles first (chunks 635).
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
    __shared__ int here[4];   // [buffer][block]: the block is there
    const Kv4Cache& c = a.c;
    const int lane = lane_id(), w = uniform_int(wave_id()), tid = 64 * w + lane, n = lane & 31, h = lane >> 5;
    // workgroup -> (pair, split, tile): ids that are equal modulo 8 share an XCD
    const int pairs = c.n_seq * c.n_head_kv, per_pair = a.tiles * a.nsplit, id = (int)blockIdx.x;
    const int j = id >> 3, np = (pairs - (id & 7) + 7) >> 3;   // pairs of this XCD
    if (np <= 0 || j >= np * per_pair) return;
    int pair, slot;
    if ((int)gridDim.x <= a.want_parts) {   // all resident, two a CU: the tiles that see most first, then those that see least upwards, so that a CU has one of each
        pair = (id & 7) + 8 * (j % np);
        slot = j / np;
        if (slot >= (per_pair + 1) / 2) slot = per_pair - 1 - (slot - (per_pair + 1) / 2);
    } else {                                // one pair after the other, its long tiles first
        pair = (id & 7) + 8 * (j / per_pair);
        slot = j % per_pair;
    }
    const int split = slot % a.nsplit, tile = a.tiles - 1 - slot / a.nsplit;
    const int b = uniform_int(pair / c.n_head_kv), kvh = pair - b * c.n_head_kv;
    const Kv4Range rg = kv4_range(a, b, tile, 128, kv4_part(a));
    if (rg.n_rows <= 0 || (split >= rg.parts && split > 0)) return;

    const int local = 32 * w + n, r = tile * 128 + local;
    const bool on = local < rg.n_rows;
    const int tok = on ? r / a.rep : 0, head = kvh * a.rep + (on ? r % a.rep : 0);
    const int lim = on ? rg.len - rg.nq + tok + 1 : 0;
    u32x4 q[2 * G];
    const float down = kv4_query<2 * G>(q, a.q, (long long)(rg.lo + tok) * a.q.row + (long long)head * a.q.head, 8 * h, 16, c.head_dim, on, a.scale,
                                        [](float v) { return fmaxf(v, lane_xor32(v)); });
    const float sc2 = kv4_factor(a.scale, down, 1.0f);
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
    const int sb = w >> 1, st = (tid >> 2) & 31, si = tid & 3, sd = tid & 31, ve = (tid >> 5) & 3;   // (sb: the same for a whole wave)
    uint32_t kc[G], ks[G], vc[G], vs[G][4];
    bool got = false;
    int pid = -1;
    auto look_up = [&](int blk) { pid = blk + sb < end ? kv4_page_of(c, b, blk + sb) : -1; };
    auto fetch = [&](int blk) {   // where there is no block the pool's first is read, and masked
        const uint8_t* p = kv4_in_page(c, pid, kvh, blk + sb);
        got = p != nullptr;
        p = got ? p : c.pages;
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
        const int there = got ? rg.len : 0;
        if (p0 + 32 > there) {   // V past the sequence's end (K's scores are masked there)
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const int t0 = p0 + 16 * (p / 2) + 4 * ve + 2 * (p & 1);
                const uint32_t keep = (t0 < there ? 0xFFFFu : 0u) | (t0 + 1 < there ? 0xFFFF0000u : 0u);
#pragma unroll
                for (int g = 0; g < G; ++g) vs[g][p] &= keep;
            }
        }
        if ((tid & 127) == 0) here[buf * 2 + sb] = got;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const uint32_t s = ks[g] | (ks[g] << 16);
            lds_st16(kb + (4 * g + si) * L::KC + st * 16, kv4_values(kc[g], s, s, s, s));
            lds_st16(vb + (ve * 32 * G + 32 * g + sd) * 16, kv4_values(vc[g], vs[g][0], vs[g][1], vs[g][2], vs[g][3]));
        }
    };
    const int tk = 16 * ((n >> 3) & 1) + 8 * (n >> 4) + 4 * ((n >> 2) & 1) + (n & 3);   // the token that this lane's row of K's operand is
    auto compute = [&](int blk, int buf) {
        const int p0 = blk * 32;
        if (p0 >= wend) return;
        f32x16 S[2];
#pragma unroll
        for (int g = 0; g < 2 * G; ++g)   // two independent sums
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const u32x4 kf = lds_ld16(smem + (buf * 2 + k) * L::BLK + (2 * g + h) * L::KC + tk * 16);
                S[k] = g == 0 ? mfma_f16_32x32x16(kf, q[g]) : mfma_f16_32x32x16_acc(kf, q[g], S[k]);
            }
        const int here0 = uniform_int(here[buf * 2]), here1 = uniform_int(here[buf * 2 + 1]);
        if (p0 + 64 > wfree || !here0 || !here1) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int left = (k ? here1 : here0) ? lim - p0 - 32 * k - 4 * h : -1;   // tokens of this lane's from here on that the row does not see
#pragma unroll
                for (int e = 0; e < 16; ++e) S[k][e] = 16 * ((e >> 2) & 1) + 8 * (e >> 3) + (e & 3) >= left ? -INFINITY : S[k][e];
            }
        }
        float top = S[0][0];
#pragma unroll
        for (int e = 1; e < 32; ++e) top = fmaxf(top, S[e / 16][e & 15]);
        top *= sc2;
        if (__ballot(top > mx + (kRaise + kLag))) {
            top = fmaxf(top, lane_xor32(top));
            const float now = fmaxf(mx, top - kRaise);
            const float f = now == -INFINITY ? 1.0f : exp2_fast(mx - now);
            mx = now;
            sum *= f;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int e = 0; e < 16; ++e) O[g][e] *= f;
        }
        float base = mx == -INFINITY ? 0.0f : -mx, factor = sc2;
        if (__ballot(fabsf(base) > kFar)) {
#pragma unroll
            for (int e = 0; e < 32; ++e) S[e / 16][e & 15] = S[e / 16][e & 15] * factor + base;
            factor = 1.0f;
            base = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const unsigned char* vb = smem + (buf * 2 + k) * L::BLK + L::KB;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                uint32_t pk[4];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float x = exp2_fast(fmaf(S[k][8 * t + e], factor, base)), y = exp2_fast(fmaf(S[k][8 * t + e + 1], factor, base));
                    pk[e / 2] = kv4_cvt2(x, y);
                    sum = kv4_sum2(pk[e / 2], sum);
                }
                const u32x4 P = u32x4_of(pk[0], pk[1], pk[2], pk[3]);
#pragma unroll
                for (int g = 0; g < G; ++g) O[g] = mfma_f16_32x32x16_acc(lds_ld16(vb + ((2 * t + h) * 32 * G + 32 * g + n) * 16), P, O[g]);
            }
        }
    };
    if (begin < end && c.n_pages > 0) {
        look_up(begin);
        fetch(begin);
        look_up(begin + 2);
        stage(begin, 0);
        int buf = 0;
        for (int blk = begin; blk < end; blk += 2, buf ^= 1) {
            __syncthreads();
            const bool more = blk + 2 < end;
            if (more) { fetch(blk + 2); look_up(blk + 4); }
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
