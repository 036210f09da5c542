// The paged key / value cache: rows of unlike length share one pool of pages, and a table names the page of every stretch of positions of a row.
//   write      new keys / values (rotated by position, with the queries) into the pages, quantised to 8 bits where the cache holds e4m3
//   read       cached keys / values back as contiguous bf16
//   attention  one new token for each row over the row's pages
// Every index that comes from device memory (row offsets, lengths, page numbers) is checked here before it becomes an address: a position without
// a page is not written and what would have been read from it is NaN, so that a bad table shows in the result and in that row alone.
#include "common.h"
#include "kernels.h"
#include "paged_split.h"

namespace merv {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994530942f;

MERV_DEVICE void unpack8f(const u32x4 r, float* f) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[2 * j] = bflo(r[j]);
        f[2 * j + 1] = bfhi(r[j]);
    }
}

// the row a token belongs to: how many of offsets[1 .. rows] are <= t, 64 at a time (independent loads, one round trip for up to 64 rows, where a
// binary search would make six dependent ones). rows: behind the last row. Called by whole waves with a uniform t.
MERV_DEVICE int row_of_token(const int* offsets, int rows, long t) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int base = 1; base <= rows; base += 64) {
        const int i = base + lane;
        n += __popcll(__ballot(i <= rows && offsets[i <= rows ? i : rows] <= t));
    }
    return n;
}

// the same for any lane's t, from a row at or before it: mostly that row or, a few steps on, the next one that has tokens
MERV_DEVICE int row_from(const int* offsets, int rows, int row, long t) {
    if (row >= rows || offsets[row + 1] > t) return row;
    int lo = row + 1, hi = rows;  // the first row in [lo, hi) whose end is behind t, or rows
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

struct TokenPlace {
    long pos;   // the token's position in its row
    long page;  // its page's number, -1: it has none
    bool idle;  // belongs to no row, or to one that sits this call out
};

MERV_DEVICE TokenPlace place_of_token(const PagedCacheArgs& c, const int* offsets, const int* start, long t, int row) {
    TokenPlace p{0, -1, true};
    if (row >= c.rows) return p;
    const long first = offsets ? offsets[row] : t;
    const int s = start ? start[row] : 0;
    if (s < 0 || t < first) return p;
    p.idle = false;
    p.pos = s + (t - first);
    const long col = p.pos >> c.page_log2;
    if (col < c.table_width) {
        const int id = c.table[(long)row * c.table_stride + col];
        if (id >= 0 && id < c.n_pages) p.page = id;
    }
    return p;
}

// largest power-of-two exponent rule for one row of one head: the smallest 2^e under which no finite element is over 448 (common.h,
// mx_shared_exponent), kept at -126 or more so that the byte is 1 .. 247 and 2^-e a normal number
MERV_DEVICE int row_exponent(float amax) {
    const int e = mx_shared_exponent(amax);
    return e < -126 ? -126 : e;
}

MERV_DEVICE float finite_abs(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;  // NaN and infinities take no part in the scale
}

// e4m3 has no infinity: what is not finite becomes its NaN. x * 2^-e is exact, so the conversion's rounding to nearest even is the only one.
MERV_DEVICE float e4m3_input(float x, float inv) {
    const float y = x * inv;
    return fabsf(x) < INFINITY ? y : __builtin_nanf("");
}

MERV_DEVICE uint32_t e4m3_pack4(const float* x, float inv) {
    int p = 0;
    p = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_input(x[0], inv), e4m3_input(x[1], inv), p, false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_input(x[2], inv), e4m3_input(x[3], inv), p, true);
    return (uint32_t)p;
}

MERV_DEVICE void e4m3_unpack8(const u32x2 r, float* f) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        f[4 * w + 0] = __builtin_amdgcn_cvt_f32_fp8((int)r[w], 0);
        f[4 * w + 1] = __builtin_amdgcn_cvt_f32_fp8((int)r[w], 1);
        f[4 * w + 2] = __builtin_amdgcn_cvt_f32_fp8((int)r[w], 2);
        f[4 * w + 3] = __builtin_amdgcn_cvt_f32_fp8((int)r[w], 3);
    }
}

// ---- write ----
// All vectors of the call (a token's keys, values and queries, token after token) are one line, of which a block takes 256 / (hd / 16): it is full whatever the
// numbers of heads are. A lane holds elements d .. d + 7 of a vector and their partners d + hd/2 .. (the rotation mixes just these), so hd / 16 lanes
// hold a vector, and queries and keys may be rotated in place. The vectors are requested before their places are looked up: the two chains of loads overlap.
// rot(x) = x cos + rotate_half(x) sin: with bf16 operands and bf16 tables both products are exact in fp32, so the sum's rounding to fp32 and its
// rounding to bf16 are the only two.
// Bound by HBM: 16 prompts of up to 2049 tokens (32 / 8 heads, e4m3, 446 MB moved) 91.8 us, 4.86 TB/s; a prompt of 1049 (28 / 4, bf16) 6.2 us; one token
// 3.4 us, a chain of three round trips. Stores are non-temporal: 97.7 and 7.4 us without (what reads the queries next does not get slower); two
// vectors a group of lanes: 92.0 and 7.1 us, and 4.4 for one token.
template <int HD, bool E4M3>
__global__ __launch_bounds__(256) void paged_write_kernel(PagedWriteArgs p) {
    constexpr int LPV = HD / 16, VPB = 256 / LPV;  // lanes for a vector, vectors a block holds at a time
    const int Hkv = p.c.kv_heads, nvec = 2 * Hkv + p.H;
    const long v0 = (long)blockIdx.x * VPB, t0 = v0 / nvec;
    const int sub = threadIdx.x % LPV, d0 = sub * 8;
    const unsigned y = (unsigned)(v0 - t0 * nvec) + threadIdx.x / LPV;
    const long t = t0 + y / (unsigned)nvec;
    const int i = y % (unsigned)nvec;
    const bool is_k = i < Hkv, is_q = i >= 2 * Hkv;
    const int h = is_q ? i - 2 * Hkv : is_k ? i : i - Hkv;
    u32x4 olo = {0, 0, 0, 0}, ohi = olo;
    if (t < p.T) {
        const bf16_t* src = is_q ? p.q + t * p.q_st + (long)h * p.q_sh : is_k ? p.k + t * p.k_st + (long)h * p.k_sh : p.v + t * p.v_st + (long)h * p.v_sh;
        olo = *(const u32x4*)(src + d0);
        ohi = *(const u32x4*)(src + d0 + HD / 2);
    }
    const int row0 = p.offsets ? row_of_token(p.offsets, p.c.rows, t0) : 0;
    if (t >= p.T) return;
    const TokenPlace at = place_of_token(p.c, p.offsets, p.start, t, p.offsets ? row_from(p.offsets, p.c.rows, row0, t) : (int)t);
    if (at.idle) return;
    const long slot = at.pos & ((1 << p.c.page_log2) - 1);
    if (p.cos && (is_k || is_q)) {
        float lo[8], hi[8], cl[8], ch[8], sl[8], sh[8];
        unpack8f(olo, lo);
        unpack8f(ohi, hi);
        const bool in_tables = at.pos < p.rope_len, ok = in_tables && at.page >= 0;
        const long row = in_tables ? at.pos : 0;
        unpack8f(*(const u32x4*)(p.cos + row * p.rope_st + d0), cl);
        unpack8f(*(const u32x4*)(p.cos + row * p.rope_st + d0 + HD / 2), ch);
        unpack8f(*(const u32x4*)(p.sin + row * p.rope_st + d0), sl);
        unpack8f(*(const u32x4*)(p.sin + row * p.rope_st + d0 + HD / 2), sh);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float a = lo[j], b = hi[j];
            lo[j] = ok ? a * cl[j] - b * sl[j] : __builtin_nanf("");
            hi[j] = ok ? b * ch[j] + a * sh[j] : __builtin_nanf("");
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            olo[j] = pack2bf(lo[2 * j], lo[2 * j + 1]);
            ohi[j] = pack2bf(hi[2 * j], hi[2 * j + 1]);
        }
    }
    if (is_q || (is_k && p.k_out)) {
        bf16_t* dst = is_q ? p.q_out + t * p.qo_st + (long)h * p.qo_sh : p.k_out + t * p.ko_st + (long)h * p.ko_sh;
        __builtin_nontemporal_store(olo, (u32x4*)(dst + d0));
        __builtin_nontemporal_store(ohi, (u32x4*)(dst + d0 + HD / 2));
    }
    if (is_q) return;
    if constexpr (E4M3) {
        float lo[8], hi[8];
        unpack8f(olo, lo);  // the cache's numbers are bf16 ones, whichever way it holds them
        unpack8f(ohi, hi);
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fmaxf(finite_abs(lo[j]), finite_abs(hi[j])));
#pragma unroll
        for (int o = LPV / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
        const int ex = row_exponent(amax);
        const float inv = __uint_as_float((uint32_t)(127 - ex) << 23);
        if (at.page < 0) return;
        uint8_t* dst = (uint8_t*)(is_k ? p.c.k : p.c.v) + at.page * p.c.s_page + (long)h * p.c.s_head + slot * p.c.s_tok;
        __builtin_nontemporal_store(u32x2{e4m3_pack4(lo, inv), e4m3_pack4(lo + 4, inv)}, (u32x2*)(dst + d0));
        __builtin_nontemporal_store(u32x2{e4m3_pack4(hi, inv), e4m3_pack4(hi + 4, inv)}, (u32x2*)(dst + d0 + HD / 2));
        if (sub == 0) (is_k ? p.c.k_scale : p.c.v_scale)[at.page * p.c.ss_page + (long)h * p.c.ss_head + slot] = (uint8_t)(ex + 127);
    } else {
        if (at.page < 0) return;
        bf16_t* dst = (bf16_t*)(is_k ? p.c.k : p.c.v) + at.page * p.c.s_page + (long)h * p.c.s_head + slot * p.c.s_tok;
        __builtin_nontemporal_store(olo, (u32x4*)(dst + d0));
        __builtin_nontemporal_store(ohi, (u32x4*)(dst + d0 + HD / 2));
    }
}

// ---- read ----
// The same line of vectors, READ_EACH for each group of lanes: all places first, then all loads, then all stores. A lane moves 16 bytes of the cache.
// Bound by memory: 32 rows of up to 4000 positions (2 kv heads, bf16, 154 MB moved) 27.0 us, 5.7 TB/s with two, 29.0 with one, 28.5 with four; 41.4 without
// non-temporal stores (repeated calls: these pages, 77 MB, stay in the 256 MB Infinity Cache). e4m3 of the same rows 23.9 us, 4.9 TB/s. Pages beyond that cache:
// 32 x 4000, 8 kv heads, bf16 142 us, 4.3 TB/s; 32 x 8000, e4m3 222 us, 4.3. 1049 positions (8 kv heads, e4m3): 3.9 us with one, 4.8 with two.
template <int HD, bool E4M3, int READ_EACH>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedReadArgs p) {
    constexpr int LPV = E4M3 ? HD / 16 : HD / 8, VPB = 256 / LPV, EPL = HD / LPV;
    const int Hkv = p.c.kv_heads, nvec = 2 * Hkv;
    const long v0 = (long)blockIdx.x * (VPB * READ_EACH), t0 = v0 / nvec;
    const int r0 = (int)(v0 - t0 * nvec), d0 = (threadIdx.x % LPV) * EPL;
    int row = row_of_token(p.offsets, p.c.rows, t0);
    bf16_t* dst[READ_EACH];
    u32x4 x[READ_EACH];
    int ex[READ_EACH];
#pragma unroll
    for (int e = 0; e < READ_EACH; ++e) {
        const unsigned y = r0 + e * VPB + threadIdx.x / LPV;
        const long t = t0 + y / (unsigned)nvec;
        const int i = y % (unsigned)nvec;
        dst[e] = nullptr;
        if (t >= p.T) continue;
        row = row_from(p.offsets, p.c.rows, row, t);
        const TokenPlace at = place_of_token(p.c, p.offsets, p.start, t, row);
        if (at.idle) continue;
        const bool is_k = i < Hkv;
        const int h = is_k ? i : i - Hkv;
        const long slot = at.pos & ((1 << p.c.page_log2) - 1);
        dst[e] = (is_k ? p.k_out + t * p.ko_st + (long)h * p.ko_sh : p.v_out + t * p.vo_st + (long)h * p.vo_sh) + d0;
        const uint32_t nan = E4M3 ? 0x7f7f7f7fu : 0x7fc07fc0u;  // a position without a page
        x[e] = u32x4{nan, nan, nan, nan};
        ex[e] = 0;
        if (at.page < 0) continue;
        const long off = at.page * p.c.s_page + (long)h * p.c.s_head + slot * p.c.s_tok + d0;
        x[e] = *(const u32x4*)((const char*)(is_k ? p.c.k : p.c.v) + off * (E4M3 ? 1 : 2));
        if constexpr (E4M3) ex[e] = (int)(is_k ? p.c.k_scale : p.c.v_scale)[at.page * p.c.ss_page + (long)h * p.c.ss_head + slot] - 127;
    }
#pragma unroll
    for (int e = 0; e < READ_EACH; ++e) {
        if (!dst[e]) continue;
        if constexpr (E4M3) {
            float f[16];
            e4m3_unpack8(u32x2{x[e][0], x[e][1]}, f);
            e4m3_unpack8(u32x2{x[e][2], x[e][3]}, f + 8);
            u32x4 o[2];
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j >> 2][j & 3] = pack2bf(ldexpf(f[2 * j], ex[e]), ldexpf(f[2 * j + 1], ex[e]));
            __builtin_nontemporal_store(o[0], (u32x4*)dst[e]);
            __builtin_nontemporal_store(o[1], (u32x4*)(dst[e] + 8));
        } else {
            __builtin_nontemporal_store(x[e], (u32x4*)dst[e]);
        }
    }
}

// ---- attention of one new token ----
// out = softmax(scale q K^T) V for a block of up to 16 query heads that share a kv head, in one pass over the pages. A wave takes 32 positions at a time:
//   S^T = K Q^T  (v_mfma_f32_16x16x32_bf16, A = 16 keys x 32 dims, B = the heads' queries): a lane gets, for head lane % 16, the scores of positions
//                4 (lane / 16) + i of each half tile -- which is, half after half, the layout of the B operand of
//   O^T += V^T P^T (A = 16 dims x 32 positions): the order of the summed positions is free, so P goes from one product into the other in registers.
// V's operand wants 8 positions of one dim in a lane; a lane loads 8 positions x HD/16 neighbouring dims in whole lines and transposes them in registers
// (v_perm_b32), row r of product dt being dim r * HD/16 + dt. K's operand wants a key in a lane: loaded so, a wave's 64 16-byte pieces lie in 16 lines of memory
// (62 GB/s a CU); loaded in whole lines and turned in the wave's own corner of LDS, 80 (16 bits; one row of 4096 positions, unsplit, 38.6 and 30.2 us).
// Scores, maximum, sum and output are fp32, and so are the weights: the 24 bits of a p are three bf16 numbers of 8 each (split_weight), whose products with
// bf16 values are exact in fp32. Two of them (2^-17 off) turned 0.3 - 0.6 % of the outputs to the other side of their rounding; the
// third costs 0.6 of 22 us where a call is bound by instructions (33 rows of up to 3001, 8 bits), elsewhere nothing.
// The running maximum moves only when a weight would exceed 2^RAISE: the rescaling of the 32 output registers is then rare. A row's weights may so add up to
// 2^RAISE times its positions; they and their sum are used 2^-shift times that, `shift` chosen from the longest possible row, so that a sum
// of weighted values never exceeds the largest value: the result is finite where the formula's is. (At the other end fp32's smallest numbers begin: weights, with e4m3
// times their value's power of two, under 2^(shift - 102) lose bits, and are NaN with an infinite value; the shift is 20 for 16384 positions.)
// e4m3 codes become bf16 exactly; a key's power of two multiplies its score, a value's its weight.
constexpr int RAISE = 6;

template <int HD, bool E4M3>
struct PagedTile {  // 32 positions of one head in a wave's registers
    static constexpr int DV = HD / 16;                   // dims of a value in a lane
    static constexpr int CPR = HD * (E4M3 ? 1 : 2) / 16; // 16-byte chunks of a key
    static constexpr int VW = E4M3 ? DV / 4 : DV / 2;    // words of a value's lane share
    u32x4 k[CPR / 2];
    uint32_t v[8][VW];
    uint32_t ks[2], vs[2];
};

template <int N>
MERV_DEVICE void load_words(uint32_t (&dst)[N], const char* src) {
    if constexpr (N == 4) {
        const u32x4 x = *(const u32x4*)src;
        dst[0] = x[0], dst[1] = x[1], dst[2] = x[2], dst[3] = x[3];
    } else if constexpr (N == 2) {
        const u32x2 x = *(const u32x2*)src;
        dst[0] = x[0], dst[1] = x[1];
    } else {
        dst[0] = *(const uint32_t*)src;
    }
}

MERV_DEVICE uint32_t e4m3_pair(uint32_t w, int hi) {  // two neighbouring codes as bf16
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
    const bf16x2_t r = hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
    return __builtin_bit_cast(uint32_t, r);
}

MERV_DEVICE float max_over_rows(float x) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float y = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
MERV_DEVICE float sum_over_rows(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float y = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

struct PagedAt {  // where a tile's halves lie
    int hkv, slot0, slot1, id0, id1;
};

template <int HD, bool E4M3>
MERV_DEVICE void load_tile(PagedTile<HD, E4M3>& t, const PagedCacheArgs& c, const PagedAt& at) {
    typedef PagedTile<HD, E4M3> Tile;
    constexpr int ELT = E4M3 ? 1 : 2;
    const int lane = threadIdx.x & 63, r = lane & 15, tg = lane >> 4;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
        const long id = tt ? at.id1 : at.id0;
        const int slot = tt ? at.slot1 : at.slot0;
        const long off = (id * c.s_page + (long)at.hkv * c.s_head + slot * c.s_tok) * ELT;
        const char* kp = (const char*)c.k + off;
        const char* vp = (const char*)c.v + off;
        const unsigned krow = (unsigned)(lane / Tile::CPR) * (unsigned)(c.s_tok * ELT) + lane % Tile::CPR * 16;
#pragma unroll
        for (int i = 0; i < Tile::CPR / 4; ++i) t.k[tt * (Tile::CPR / 4) + i] = *(const u32x4*)(kp + i * (64 / Tile::CPR) * c.s_tok * ELT + krow);
        const unsigned vrow = (unsigned)tg * 4u * (unsigned)(c.s_tok * ELT) + r * Tile::DV * ELT;
#pragma unroll
        for (int i = 0; i < 4; ++i) load_words(t.v[tt * 4 + i], vp + i * c.s_tok * ELT + vrow);
        if constexpr (E4M3) {
            const long sat = id * c.ss_page + (long)at.hkv * c.ss_head + slot;
            t.ks[tt] = *(const uint32_t*)(c.k_scale + sat + tg * 4);
            t.vs[tt] = *(const uint32_t*)(c.v_scale + sat + tg * 4);
        }
    }
}

template <int HD>
struct PagedState {  // of a wave: lane l has head l % 16
    float m, l;
    f32x4 o[HD / 16];
};

// p >= 0 as the sum of three bf16 numbers (the upper halves of x), exactly: p cut off behind 8 bits, the rest cut off, the rest of that, which has 8 bits left.
// POSITIVE, where values may be infinite: all three parts of a p >= 2^-102 are over zero, so that none turns an infinity round or makes it NaN. For that the number
// before p is cut off instead of p: what is left is over zero and, where p itself had 8 bits only, a power of two.
template <bool POSITIVE>
MERV_DEVICE void split_weight(float p, uint32_t (&x)[3]) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const uint32_t bits = __float_as_uint(p);
        x[n] = (POSITIVE ? __builtin_elementwise_sub_sat(bits, 1u) : bits) & 0xffff0000u;
        p -= __uint_as_float(x[n]);
    }
    x[2] = __float_as_uint(p);
}

template <int HD, bool E4M3>
MERV_DEVICE void use_tile(PagedState<HD>& st, PagedTile<HD, E4M3>& t, const bf16x8 (&q)[HD / 32], float scale2, int shift, int tok, int lo, int len,
                          char* room) {
    typedef PagedTile<HD, E4M3> Tile;
    constexpr int CPR = Tile::CPR, RPL = 16 / CPR;  // keys in 256 bytes of LDS
    const int lane = threadIdx.x & 63, tg = lane >> 4;
    // keys pass through the wave's own part of LDS: loaded in whole lines, 64 / CPR at a time, wanted a key in a lane. Chunk c of key j lies at c ^ (j / RPL): the
    // 16 lanes of one access, here and below, touch all banks once.
#pragma unroll
    for (int i = 0; i < CPR / 2; ++i) {
        const int j = i * (64 / CPR) + lane / CPR;
        *(u32x4*)(room + j * (CPR * 16) + ((lane % CPR) ^ (j / RPL % CPR)) * 16) = t.k[i];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    f32x4 s[2];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
        s[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
        u32x4 codes = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
            const int key = tt * 16 + (lane & 15);
            auto chunk = [&](int c) { return *(const u32x4*)(room + key * (CPR * 16) + (c ^ (key / RPL % CPR)) * 16); };
            bf16x8 a;
            if constexpr (E4M3) {
                if ((j & 1) == 0) codes = chunk((j >> 1) * 4 + tg);
                const uint32_t w0 = codes[(j & 1) * 2], w1 = codes[(j & 1) * 2 + 1];
                a = __builtin_bit_cast(bf16x8, u32x4{e4m3_pair(w0, 0), e4m3_pair(w0, 1), e4m3_pair(w1, 0), e4m3_pair(w1, 1)});
            } else {
                a = __builtin_bit_cast(bf16x8, chunk(j * 4 + tg));
            }
            s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q[j], s[tt], 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[tt][i] *= scale2;
            if constexpr (E4M3) s[tt][i] = ldexpf(s[tt][i], (int)((t.ks[tt] >> (8 * i)) & 0xff) - 127);
        }
    }
    if (tok + 32 > len || tok < lo) {  // the row's first or last tile: what is not seen may hold anything
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = tok + tt * 16 + tg * 4 + i;
                const bool seen = j >= lo && j < len;
                s[tt][i] = seen ? s[tt][i] : -INFINITY;
#pragma unroll
                for (int w = 0; w < Tile::VW; ++w) t.v[tt * 4 + i][w] = seen ? t.v[tt * 4 + i][w] : 0u;
                if constexpr (E4M3) t.vs[tt] = seen ? t.vs[tt] : t.vs[tt] & ~(0xffu << (8 * i));
            }
    }
    float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    top = max_over_rows(top);
    if (__any(top > st.m + (float)RAISE)) {
        const float m = fmaxf(st.m, top);
        const float a = __builtin_amdgcn_exp2f(st.m - (m == -INFINITY ? 0.f : m));
        st.m = m;
        st.l *= a;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) st.o[d] *= a;
    }
    const float base = st.m == -INFINITY ? 0.f : st.m;
    const float down = __uint_as_float((uint32_t)(127 - shift) << 23);
    u32x4 part[3];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[i] = __builtin_amdgcn_exp2f(s[tt][i] - base);
            st.l += p[i];
            if constexpr (E4M3) p[i] = ldexpf(p[i], (int)((t.vs[tt] >> (8 * i)) & 0xff) - 127 - shift);
            else p[i] *= down;
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            uint32_t x[3], y[3];
            split_weight<!E4M3>(p[2 * w], x);
            split_weight<!E4M3>(p[2 * w + 1], y);
#pragma unroll
            for (int n = 0; n < 3; ++n) part[n][tt * 2 + w] = __builtin_amdgcn_perm(y[n], x[n], 0x07060302u);
        }
    }
#pragma unroll
    for (int w = 0; w < Tile::DV / 2; ++w) {  // dims 2w and 2w + 1 of the lane's
        uint32_t x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (E4M3) x[i] = e4m3_pair(t.v[i][w >> 1], w & 1);
            else x[i] = t.v[i][w];
        }
        u32x4 even, odd;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            even[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x05040100u);
            odd[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x07060302u);
        }
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            const bf16x8 pn = __builtin_bit_cast(bf16x8, part[n]);
            st.o[2 * w] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, even), pn, st.o[2 * w], 0, 0, 0);
            st.o[2 * w + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, odd), pn, st.o[2 * w + 1], 0, 0, 0);
        }
    }
}

// over the lanes up to and with the own one
MERV_DEVICE int wave_scan_add(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return x;
}
MERV_DEVICE int wave_scan_max(int x) {  // of numbers that are not negative
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
    return x;
}

MERV_DEVICE PagedSpan span_of_len(const PagedAttnArgs& p, int len) { return paged_span(len, p.window, p.c.table_width << p.c.page_log2); }
// of a row that is the same for the whole wave: through the scalar cache, which leaves the order of the vector loads (and the waits for them) alone
MERV_DEVICE PagedSpan span_of(const PagedAttnArgs& p, int row) {
    return span_of_len(p, *(const __attribute__((address_space(4))) int*)(uintptr_t)(p.lens + row));
}

// The workspace: a PagedOpen of each worker, then two partial sums of each (of a head: HD numbers, maximum, sum, 2 of padding).
struct PagedOpen {  // of the pair that begins in a worker and ends in a later one
    int row, pair, slot, last;  // last: the worker that it ends in, -1: there is no such pair
};
// (the first sums of all workers, then the second ones: those of one pair, most of them first ones, lie together)
template <int HD>
MERV_DEVICE float* paged_sum(const PagedAttnArgs& p, int slot, int head) {
    const int block = min(p.H / p.c.kv_heads, PAGED_HEAD_BLOCK);
    return (float*)((PagedOpen*)p.ws + p.workers) + ((size_t)((slot & 1) * p.workers + (slot >> 1)) * block + head) * (HD + 4);
}

template <int HD, int NW>
struct PagedLds {
    float o[NW][PAGED_HEAD_BLOCK][HD + 4];  // (padded: heads lie in other banks)
    float m[NW][PAGED_HEAD_BLOCK], l[NW][PAGED_HEAD_BLOCK];
};

struct PagedSegment {  // units u .. u + n - 1 of one pair. slot < 0: all of the pair, the result is written.
    int base, lo, len, units, row, pair, u, n, slot;
};

// What a wave (of NW) holds of a segment: its tiles are 32 positions at first + 32 NW i, the pages of 32 of them at a time lie in `ids`, one half tile in each lane.
struct PagedWalk {
    int first, tiles, ids;
};

template <int NW>
MERV_DEVICE int half_tile(const PagedSegment& g, int first, int t0) {  // the lane's one of 32 tiles from t0 on
    const int lane = threadIdx.x & 63;
    return min(first + (t0 + (lane >> 1)) * (32 * NW) + (lane & 1) * 16, g.len - 1);  // behind the row's end: the row's last position
}
template <int NW>
MERV_DEVICE int load_ids(const PagedAttnArgs& p, const PagedSegment& g, int first, int t0) {
    return (p.c.table + (long)g.row * p.c.table_stride)[half_tile<NW>(g, first, t0) >> p.c.page_log2];
}

// `pages`, where given: the row's pages, one in each lane
template <int NW, bool GIVEN>
MERV_DEVICE PagedWalk begin_walk(const PagedAttnArgs& p, const PagedSegment& g, int pages) {
    PagedWalk w;
    w.first = g.base + g.u * PAGED_UNIT + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 32;
    const int left = g.len - w.first;
    w.tiles = left <= 0 || p.c.n_pages <= 0 ? 0 : (min(left, g.n * PAGED_UNIT) + 32 * NW - 1) / (32 * NW);
    if (GIVEN && p.c.table_width <= 64) w.ids = __shfl(pages, half_tile<NW>(g, w.first, 0) >> p.c.page_log2, 64);
    else w.ids = load_ids<NW>(p, g, w.first, 0);
    return w;
}

// page numbers that are none become page 0, and mark the segment
MERV_DEVICE int checked_ids(const PagedAttnArgs& p, int ids, int& bad) {
    const bool ok = ids >= 0 && ids < p.c.n_pages;
    bad |= ok ? 0 : 1;
    return ok ? ids : 0;
}

template <int NW>
MERV_DEVICE PagedAt tile_at(const PagedAttnArgs& p, const PagedSegment& g, const PagedWalk& w, int i) {
    const int tok = w.first + i * (32 * NW), mask = (1 << p.c.page_log2) - 1;
    const int half1 = tok + 16 < g.len ? tok + 16 : tok;  // behind the row's end: the first half again
    return PagedAt{g.pair / p.head_blocks, tok & mask, half1 & mask, __builtin_amdgcn_readlane(w.ids, 2 * (i & 31)),
                   __builtin_amdgcn_readlane(w.ids, 2 * (i & 31) + 1)};
}

// the queries of a segment's heads, as the second operand of S^T: lane l has head l % 16, the dims in the order in which its keys hold them
template <int HD, bool E4M3>
MERV_DEVICE void load_queries(bf16x8 (&q)[HD / 32], const PagedAttnArgs& p, const PagedSegment& g) {
    const int lane = threadIdx.x & 63, group = p.H / p.c.kv_heads, hkv = g.pair / p.head_blocks, hb = g.pair - hkv * p.head_blocks;
    const int h0 = hkv * group + hb * PAGED_HEAD_BLOCK, heads = min(PAGED_HEAD_BLOCK, group - hb * PAGED_HEAD_BLOCK);
    const bf16_t* qp = p.q + (long)g.row * p.q_st + (long)(h0 + min(lane & 15, heads - 1)) * p.q_sh;
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) {
        const int d = E4M3 ? (j >> 1) * 64 + (lane >> 4) * 16 + (j & 1) * 8 : j * 32 + (lane >> 4) * 8;
        q[j] = __builtin_bit_cast(bf16x8, *(const u32x4*)(qp + d));
    }
}

// the waves' sums of a segment, together: the result, or a partial sum
template <int HD, int NW>
MERV_DEVICE void end_segment(const PagedAttnArgs& p, PagedLds<HD, NW>& lds, const PagedSegment& g, PagedState<HD>& st, int bad) {
    constexpr int DV = HD / 16;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int group = p.H / p.c.kv_heads, hkv = g.pair / p.head_blocks, hb = g.pair - hkv * p.head_blocks;
    const int h0 = hkv * group + hb * PAGED_HEAD_BLOCK, heads = min(PAGED_HEAD_BLOCK, group - hb * PAGED_HEAD_BLOCK);
    st.l = ldexpf(sum_over_rows(st.l), -p.shift);  // as the weights
    if (__any(bad)) st.l = __builtin_nanf("");
    const int h = lane & 15;
    if (h < heads) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float* dst = &lds.o[wave][h][((lane >> 4) * 4 + i) * DV];
#pragma unroll
            for (int d = 0; d < DV; d += 4) *(f32x4*)(dst + d) = f32x4{st.o[d][i], st.o[d + 1][i], st.o[d + 2][i], st.o[d + 3][i]};
        }
        if (lane < 16) {
            lds.m[wave][h] = st.m;
            lds.l[wave][h] = st.l;
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < heads * (HD / 4); e += 64 * NW) {
        const int hh = e / (HD / 4), d = e % (HD / 4) * 4;
        float M = lds.m[0][hh];
#pragma unroll
        for (int w = 1; w < NW; ++w) M = fmaxf(M, lds.m[w][hh]);
        const float base = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(lds.m[w][hh] - base);
            L += f * lds.l[w][hh];
            O += f * *(const f32x4*)&lds.o[w][hh][d];
        }
        if (g.slot < 0) {
            const u32x2 o = {pack2bf(O[0] / L, O[1] / L), pack2bf(O[2] / L, O[3] / L)};
            *(u32x2*)(p.out + (long)g.row * p.o_st + (long)(h0 + hh) * p.o_sh + d) = o;
            if (p.lse && d == 0) p.lse[(long)g.row * p.H + h0 + hh] = (M + __builtin_amdgcn_logf(ldexpf(L, p.shift))) * LN2;
        } else {
            float* ws = paged_sum<HD>(p, g.slot, hh);
            *(f32x4*)(ws + d) = O;
            if (d == 0) *(f32x2*)(ws + HD) = f32x2{M, L};
        }
    }
    __syncthreads();
}

template <int HD>
MERV_DEVICE void write_unseen(const PagedAttnArgs& p, int row, int h, int d) {  // a row without positions, or with more than its table has
    const float x = p.lens[row] > 0 ? __builtin_nanf("") : 0.f;
    p.out[(long)row * p.o_st + (long)h * p.o_sh + d] = f2bf(x);
    if (p.lse && d == 0) p.lse[(long)row * p.H + h] = p.lens[row] > 0 ? x : -INFINITY;
}

// what a worker leaves beside its sums: word of the pair that goes on behind it, and the results of every p.workers-th row that has no units
template <int HD>
MERV_DEVICE void end_worker(const PagedAttnArgs& p, PagedOpen open, const PagedShare& share) {
    if (open.last >= 0) open.last = paged_owner(share, open.last);  // (until here: the pair's last unit)
    if (threadIdx.x == 0) ((PagedOpen*)p.ws)[blockIdx.x] = open;
    for (int r = blockIdx.x; r < p.c.rows; r += p.workers)
        if (span_of(p, r).units == 0)
            for (int e = threadIdx.x; e < p.H * HD; e += 256) write_unseen<HD>(p, r, e / HD, e % HD);
}

// DIRECT: a workgroup for each pair of each row, which writes the result. Else the line of units is shared out, or, where the lengths are so, the pairs are
// left whole as well (paged_split.h).
//
// One tile is always on its way: while a tile is used the next one is loaded, which behind a segment's last is the first of the workgroup's next segment
// (whose pages were looked up a segment ahead). Behind the very last it is that one again, from the cache: a load that were left out there would make
// the compiler wait, at each use, for the newer loads too. Lengths come through the scalar cache for the same reason.
//
// Bound by HBM where the call is large, by its chain of round trips (length, pages, keys and values, sums) where it is small. Measured, 128 dims:
//   96 rows of 2458 .. 8192 positions, 32 / 8 heads, 16 bits: 352 us, 5.87 TB/s of keys and values (a copy of 1 GiB on this card: 5.05)
//   1 row of 131072, 32 / 8 heads, 8 bits: 58.6 us, 4.6 TB/s, 6 of them the join;  33 rows of up to 3001, 28 / 4, 8 bits: 22.4 us, 2.7 TB/s
//   1 row of 77, 16 / 2 heads: 4.5 us;  1 row of 1049, 32 / 32, 16 bits: 11.5 us in a table of 1088 positions (one launch), 12.0 in one of 1280 (shared out)
// 512 workers: with 1024 the large call takes 363 us and 33 x 3001 takes a fifth more (twice the segments); with 256 half the loads are on their way.
// Two workgroups a CU: 8 waves x 2 tiles of 16 KB (16 bits) outstanding cover the latency; registers, not LDS, set the limit (three for 8 bits: 33
// registers spill, 33 x 3001 takes 25.9 us, 131072 75.5).
template <int HD, bool E4M3, bool DIRECT, int NW>
__global__ __launch_bounds__(64 * NW, 2) void paged_attention_kernel(PagedAttnArgs p) {
    static_assert(DIRECT || NW == 4, "a unit is one tile for each of four waves");
    __shared__ __attribute__((aligned(16))) PagedLds<HD, NW> lds;
    const int pairs = p.c.kv_heads * p.head_blocks;
    PagedSegment g;
    int x = 0, end = 0, w = 0;  // units of the line: behind this segment, behind this worker; the worker
    PagedShare share{0, 0, 0};
    PagedOpen open{0, 0, 0, -1};
    int pages = 0;
    bool whole = DIRECT;  // one pair of one row
    if constexpr (!DIRECT) {
        const int rows = p.c.rows, per = (rows + 63) / 64, lane = threadIdx.x & 63, r0 = min(rows, lane * per), r1 = min(rows, r0 + per);
        int mine = 0, most = 0, len = 0;
        for (int r = r0; r < r1; ++r) {
            len = p.lens[r];
            const int n = span_of_len(p, len).units;
            mine += n;
            most = max(most, n);
        }
        const int sum = wave_scan_add(mine), total = __builtin_amdgcn_readlane(sum, 63) * pairs;
        most = __builtin_amdgcn_readlane(wave_scan_max(most), 63);
        whole = paged_whole(total, most, rows * pairs, gridDim.x);
        w = blockIdx.x;
        share = paged_share(total, p.workers);
        if (whole) {
            if (threadIdx.x == 0 && w < p.workers) ((PagedOpen*)p.ws)[w] = open;
            if (w >= rows * pairs) return;
        } else if (w >= share.workers) {
            if (w < p.workers) end_worker<HD>(p, open, share);
            return;
        } else {
            x = paged_start(share, w);
            end = paged_start(share, w + 1);
            // the lane whose rows hold the first unit
            const int at = __ffsll(__ballot(x >= (sum - mine) * pairs && x < sum * pairs)) - 1;
            int before = __builtin_amdgcn_readlane(sum - mine, at);
            g.row = at * per;
            PagedSpan sp = per == 1 ? span_of_len(p, __builtin_amdgcn_readlane(len, at)) : span_of(p, g.row);
            while (x >= (before + sp.units) * pairs) {  // (per > 1)
                before += sp.units;
                sp = span_of(p, ++g.row);
            }
            g.base = sp.base, g.lo = sp.lo, g.len = sp.len, g.units = sp.units;
            const int in_row = x - before * pairs;
            g.pair = in_row / sp.units;
            g.u = in_row - g.pair * sp.units;
            g.n = min(g.units - g.u, end - x);
            g.slot = g.n == g.units ? -1 : paged_slot(w, true);
            if (g.u == 0 && g.n < g.units) open = PagedOpen{g.row, g.pair, g.slot, x + g.units - 1};
            x += g.n;
        }
    }
    if (whole) {
        g.row = blockIdx.x / pairs;
        g.pair = blockIdx.x - g.row * pairs;
        if constexpr (DIRECT) {  // a row's first 64 pages are requested together with its length
            const int col = min((int)(threadIdx.x & 63), p.c.table_width - 1);
            if (col >= 0) pages = (p.c.table + (long)g.row * p.c.table_stride)[col];
        }
        const PagedSpan sp = span_of(p, g.row);
        if (sp.units == 0) {
            const int group = p.H / p.c.kv_heads, hkv = g.pair / p.head_blocks, hb = g.pair - hkv * p.head_blocks;
            const int heads = min(PAGED_HEAD_BLOCK, group - hb * PAGED_HEAD_BLOCK);
            for (int e = threadIdx.x; e < heads * HD; e += 64 * NW) write_unseen<HD>(p, g.row, hkv * group + hb * PAGED_HEAD_BLOCK + e / HD, e % HD);
            return;
        }
        g.base = sp.base, g.lo = sp.lo, g.len = sp.len, g.units = sp.units;
        g.u = 0, g.n = sp.units, g.slot = -1;
    }
    const float scale2 = p.scale * LOG2E;
    PagedTile<HD, E4M3> a, b;
    bf16x8 q[HD / 32];
    char* room = (char*)&lds.o[__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)][0][0];
    int bad = 0;
    PagedWalk walk = begin_walk<NW, DIRECT>(p, g, pages);
    load_queries<HD, E4M3>(q, p, g);
    walk.ids = checked_ids(p, walk.ids, bad);
    if (walk.tiles > 0) load_tile(a, p.c, tile_at<NW>(p, g, walk, 0));
    for (;;) {
        PagedSegment g2 = g;
        PagedWalk walk2 = walk;
        int bad2 = 0;
        bool more = false;
        if constexpr (!DIRECT) {
            more = x < end;
            if (more) {
                g2.u = 0;
                if (++g2.pair == pairs) {
                    g2.pair = 0;
                    PagedSpan sp;
                    do sp = span_of(p, ++g2.row);
                    while (sp.units == 0);
                    g2.base = sp.base, g2.lo = sp.lo, g2.len = sp.len, g2.units = sp.units;
                }
                g2.n = min(g2.units, end - x);
                g2.slot = g2.n == g2.units ? -1 : paged_slot(w, false);
                if (g2.n < g2.units) open = PagedOpen{g2.row, g2.pair, g2.slot, x + g2.units - 1};
                x += g2.n;
                walk2 = begin_walk<NW, false>(p, g2, 0);
            }
        }
        PagedState<HD> st;
        st.m = -INFINITY;
        st.l = 0.f;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) st.o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
        // where the tile behind i lies
        auto behind = [&](int i) {
            if (i + 1 < walk.tiles) {
                if (((i + 1) & 31) == 0) walk.ids = checked_ids(p, load_ids<NW>(p, g, walk.first, i + 1), bad);
                return tile_at<NW>(p, g, walk, i + 1);
            }
            if (more && walk2.tiles > 0) {
                walk2.ids = checked_ids(p, walk2.ids, bad2);
                return tile_at<NW>(p, g2, walk2, 0);
            }
            return tile_at<NW>(p, g, walk, i);
        };
        bool in_b = false;  // the next segment's first tile
        for (int i = 0; i < walk.tiles;) {
            load_tile(b, p.c, behind(i));
            __builtin_amdgcn_sched_barrier(0);  // all of the next tile is requested before the first wait for this one
            use_tile(st, a, q, scale2, p.shift, walk.first + i * (32 * NW), g.lo, g.len, room);
            if (++i == walk.tiles) {
                in_b = true;
                break;
            }
            load_tile(a, p.c, behind(i));
            __builtin_amdgcn_sched_barrier(0);
            use_tile(st, b, q, scale2, p.shift, walk.first + i * (32 * NW), g.lo, g.len, room);
            ++i;
        }
        if (more) {
            load_queries<HD, E4M3>(q, p, g2);
            if (walk.tiles == 0 && walk2.tiles > 0) {  // else it is on its way
                walk2.ids = checked_ids(p, walk2.ids, bad2);
                load_tile(a, p.c, tile_at<NW>(p, g2, walk2, 0));
            }
        }
        end_segment(p, lds, g, st, bad);
        if (!more) break;
        if (in_b) a = b;
        g = g2;
        walk = walk2;
        walk.ids = checked_ids(p, walk.ids, bad2);
        bad = bad2;
    }
    if constexpr (!DIRECT)
        if (!whole) end_worker<HD>(p, open, share);
}

// Joins the partial sums of the pair that begins in a worker and ends in a later one, if there is one; the worker left word of it (PagedOpen), so nothing
// about the lengths is worked out again. A workgroup for a worker and a head. Up to JOIN_MANY sums: the first of four heads' workgroups takes all four, a
// wave each. More: each takes its own, wave w the workers w, w + 4 .. behind the first, and the four meet in LDS.
constexpr int JOIN_MANY = 16;

template <int HD>
struct PagedSum {
    float m, l, o[HD / 64];
};

// EACH sums are requested at a time (behind the last one, that one again: a load that is left out would keep the others from going out together)
template <int HD, int EACH>
MERV_DEVICE PagedSum<HD> join_sums(const PagedAttnArgs& p, const PagedOpen& open, int w0, int hh, int from, int step) {
    constexpr int DPL = HD / 64;
    const int lane = threadIdx.x & 63;
    PagedSum<HD> s{-INFINITY, 0.f, {}};
    for (int w = w0 + from; w <= open.last; w += step * EACH) {
        f32x2 ml[EACH];
        float o[EACH][DPL];
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int v = min(w + step * e, open.last);
            const float* x = paged_sum<HD>(p, v == w0 ? open.slot : 2 * v, hh);
            ml[e] = *(const f32x2*)(x + HD);
            if constexpr (DPL == 2) {
                const f32x2 y = *(const f32x2*)(x + lane * 2);
                o[e][0] = y[0], o[e][1] = y[1];
            } else {
                o[e][0] = x[lane];
            }
        }
        float top = s.m;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            asm volatile("" : "+v"(ml[e]));  // (here, so that no load sinks to its use)
#pragma unroll
            for (int d = 0; d < DPL; ++d) asm volatile("" : "+v"(o[e][d]));
            top = fmaxf(top, ml[e][0]);
        }
        const float base = top == -INFINITY ? 0.f : top, a = __builtin_amdgcn_exp2f(s.m - base);
        s.m = top;
        s.l *= a;
#pragma unroll
        for (int d = 0; d < DPL; ++d) s.o[d] *= a;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const bool on = w + step * e <= open.last;
            const float f = __builtin_amdgcn_exp2f(ml[e][0] - base);
            s.l += on ? f * ml[e][1] : 0.f;
#pragma unroll
            for (int d = 0; d < DPL; ++d) s.o[d] += on ? f * o[e][d] : 0.f;
        }
    }
    return s;
}

template <int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs p) {
    constexpr int DPL = HD / 64;
    __shared__ float sm[4], sl[4], so[4][HD];
    // (one long row's pairs begin in every 64th worker or so: in a row of workgroups that is one XCD)
    const int w0 = xcd_remap(blockIdx.x, p.workers), lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const PagedOpen open = ((const PagedOpen*)p.ws)[w0];
    const bool few = open.last - w0 < JOIN_MANY;
    if (open.last < 0 || (few && (blockIdx.y & 3))) return;
    const int group = p.H / p.c.kv_heads, hkv = open.pair / p.head_blocks, hb = open.pair - hkv * p.head_blocks;
    const int hh = few ? blockIdx.y + wave : blockIdx.y, h = hkv * group + hb * PAGED_HEAD_BLOCK + hh;
    if (hb * PAGED_HEAD_BLOCK + hh >= group || hh >= PAGED_HEAD_BLOCK) return;  // (not few: the whole workgroup)
    PagedSum<HD> s;
    if (few) {
        s = join_sums<HD, 4>(p, open, w0, hh, 0, 1);
    } else {
        s = join_sums<HD, JOIN_MANY>(p, open, w0, hh, wave, 4);
        if (lane == 0) {
            sm[wave] = s.m;
            sl[wave] = s.l;
        }
#pragma unroll
        for (int d = 0; d < DPL; ++d) so[wave][lane * DPL + d] = s.o[d];
        __syncthreads();
        if (wave) return;
        const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), base = top == -INFINITY ? 0.f : top;
        s = PagedSum<HD>{top, 0.f, {}};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(sm[w] - base);
            s.l += f * sl[w];
#pragma unroll
            for (int d = 0; d < DPL; ++d) s.o[d] += f * so[w][lane * DPL + d];
        }
    }
    bf16_t* out = p.out + (long)open.row * p.o_st + (long)h * p.o_sh + lane * DPL;
    if constexpr (DPL == 2) *(uint32_t*)out = pack2bf(s.o[0] / s.l, s.o[1] / s.l);
    else *out = f2bf(s.o[0] / s.l);
    if (p.lse && lane == 0) p.lse[(long)open.row * p.H + h] = (s.m + __builtin_amdgcn_logf(ldexpf(s.l, p.shift))) * LN2;
}

}  // namespace

template <int HD, bool E4M3>
static void launch_paged_write_as(const PagedWriteArgs& a, hipStream_t s) {
    const long vectors = (long)a.T * (2 * a.c.kv_heads + a.H), each = 256 / (HD / 16);
    hipLaunchKernelGGL((paged_write_kernel<HD, E4M3>), dim3((unsigned)((vectors + each - 1) / each)), dim3(256), 0, s, a);
}

hipError_t launch_paged_write(const PagedWriteArgs& a, hipStream_t s) {
    if (a.T <= 0) return hipSuccess;
    if (a.c.hd == 128) a.c.e4m3 ? launch_paged_write_as<128, true>(a, s) : launch_paged_write_as<128, false>(a, s);
    else if (a.c.hd == 64) a.c.e4m3 ? launch_paged_write_as<64, true>(a, s) : launch_paged_write_as<64, false>(a, s);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

template <int HD, bool E4M3, int EACH>
static void launch_paged_read_each(const PagedReadArgs& a, long vectors, hipStream_t s) {
    const long each = 256 / (E4M3 ? HD / 16 : HD / 8) * EACH;
    hipLaunchKernelGGL((paged_read_kernel<HD, E4M3, EACH>), dim3((unsigned)((vectors + each - 1) / each)), dim3(256), 0, s, a);
}
template <int HD, bool E4M3>
static void launch_paged_read_as(const PagedReadArgs& a, hipStream_t s) {
    const long vectors = (long)a.T * 2 * a.c.kv_heads;
    // two vectors for a group of lanes where that leaves the card two workgroups a CU
    if (vectors >= 512L * 2 * 256 / (E4M3 ? HD / 16 : HD / 8)) launch_paged_read_each<HD, E4M3, 2>(a, vectors, s);
    else launch_paged_read_each<HD, E4M3, 1>(a, vectors, s);
}

hipError_t launch_paged_read(const PagedReadArgs& a, hipStream_t s) {
    if (a.T <= 0) return hipSuccess;
    if (a.c.hd == 128) a.c.e4m3 ? launch_paged_read_as<128, true>(a, s) : launch_paged_read_as<128, false>(a, s);
    else if (a.c.hd == 64) a.c.e4m3 ? launch_paged_read_as<64, true>(a, s) : launch_paged_read_as<64, false>(a, s);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

size_t paged_attention_workspace_bytes(int rows, int H, int kv_heads, int hd, long capacity) {
    const PagedPlan pl = paged_plan(rows, H, kv_heads, capacity);
    const int group = H / kv_heads;
    return pl.direct ? 0 : pl.workers * (sizeof(PagedOpen) + (size_t)2 * (group < PAGED_HEAD_BLOCK ? group : PAGED_HEAD_BLOCK) * (hd + 4) * sizeof(float));
}

template <int HD, bool E4M3>
static hipError_t launch_paged_attention_as(const PagedAttnArgs& a, const PagedPlan& pl, hipStream_t s) {
    if (pl.direct) {
        if (pl.waves == 8) hipLaunchKernelGGL((paged_attention_kernel<HD, E4M3, true, 8>), dim3((unsigned)pl.grid), dim3(512), 0, s, a);
        else hipLaunchKernelGGL((paged_attention_kernel<HD, E4M3, true, 4>), dim3((unsigned)pl.grid), dim3(256), 0, s, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((paged_attention_kernel<HD, E4M3, false, 4>), dim3((unsigned)pl.grid), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int group = a.H / a.c.kv_heads;
    hipLaunchKernelGGL((paged_join_kernel<HD>), dim3((unsigned)a.workers, (unsigned)(group < PAGED_HEAD_BLOCK ? group : PAGED_HEAD_BLOCK)), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_paged_attention(const PagedAttnArgs& args, hipStream_t s) {
    if (args.c.rows <= 0) return hipSuccess;
    PagedAttnArgs a = args;
    const PagedPlan pl = paged_plan(a.c.rows, a.H, a.c.kv_heads, (long)a.c.table_width << a.c.page_log2);
    a.head_blocks = pl.head_blocks;
    a.workers = pl.workers;
    const long capacity = (long)a.c.table_width << a.c.page_log2, most = a.window > 0 && a.window < capacity ? a.window : capacity;
    for (a.shift = RAISE; (1L << (a.shift - RAISE)) < most;) ++a.shift;  // (most <= 2^30)
    if (a.c.hd == 128) return a.c.e4m3 ? launch_paged_attention_as<128, true>(a, pl, s) : launch_paged_attention_as<128, false>(a, pl, s);
    if (a.c.hd == 64) return a.c.e4m3 ? launch_paged_attention_as<64, true>(a, pl, s) : launch_paged_attention_as<64, false>(a, pl, s);
    return hipErrorInvalidValue;
}

}  // namespace merv
