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

// the row a new token belongs to: how many of offsets[1 .. rows] are <= t, 64 at a time (independent loads, one round trip for up to 64 rows, where a
// binary search would make six dependent ones). rows: behind the last row. Called by whole waves with a uniform t.
MERV_DEVICE int row_of_token(const int* offsets, int rows, int t) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int base = 1; base <= rows; base += 64) {
        const int i = base + lane;
        n += __popcll(__ballot(i <= rows && offsets[i <= rows ? i : rows] <= t));
    }
    return n;
}

struct TokenPlace {
    long pos;   // the token's position in its row
    long page;  // its page's number, -1: it has none
    bool idle;  // belongs to no row, or to one that sits this call out
};

MERV_DEVICE TokenPlace place_of_token(const PagedCacheArgs& c, const int* offsets, const int* start, int t) {
    TokenPlace p{0, -1, true};
    const int row = offsets ? row_of_token(offsets, c.rows, t) : t;
    if (row >= c.rows) return p;
    const int first = offsets ? offsets[row] : t, s = start ? start[row] : 0;
    if (s < 0 || t < first) return p;
    p.idle = false;
    p.pos = (long)s + (t - first);
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
// One block per new token. A lane holds elements d .. d + 7 of one head's vector and their partners d + hd/2 .. (the rotation mixes just these), so
// hd / 16 lanes hold a vector and the queries may be rotated in place. rot(x) = x cos + rotate_half(x) sin: with bf16 operands and bf16 tables both
// products are exact in fp32, so the sum's rounding to fp32 and its rounding to bf16 are the only two.
template <int HD, bool E4M3>
__global__ __launch_bounds__(256) void paged_write_kernel(PagedWriteArgs p) {
    constexpr int LPV = HD / 16, VPB = 256 / LPV;  // lanes for a vector, vectors a block holds at a time
    const int t = blockIdx.x;
    const TokenPlace at = place_of_token(p.c, p.offsets, p.start, t);
    if (at.idle) return;
    const int sub = threadIdx.x % LPV, d0 = sub * 8;
    const bool rotate = p.cos != nullptr;
    const bool in_tables = at.pos < p.rope_len;
    const int Hkv = p.c.kv_heads, nvec = 2 * Hkv + (p.q ? p.H : 0);
    const long slot = at.pos & ((1 << p.c.page_log2) - 1);
    for (int i = threadIdx.x / LPV; i < nvec; i += VPB) {
        const bool is_k = i < Hkv, is_q = i >= 2 * Hkv;
        const int h = is_q ? i - 2 * Hkv : is_k ? i : i - Hkv;
        const bf16_t* src = is_q ? p.q + (long)t * p.q_st + (long)h * p.q_sh
                                 : is_k ? p.k + (long)t * p.k_st + (long)h * p.k_sh : p.v + (long)t * p.v_st + (long)h * p.v_sh;
        float lo[8], hi[8];
        unpack8f(*(const u32x4*)(src + d0), lo);
        unpack8f(*(const u32x4*)(src + d0 + HD / 2), hi);
        u32x4 olo, ohi;
        if (rotate && (is_k || is_q)) {
            float cl[8], ch[8], sl[8], sh[8];
            const bool ok = in_tables && at.page >= 0;
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
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            olo[j] = pack2bf(lo[2 * j], lo[2 * j + 1]);
            ohi[j] = pack2bf(hi[2 * j], hi[2 * j + 1]);
        }
        if (is_q || (is_k && p.k_out)) {
            bf16_t* dst = is_q ? p.q_out + (long)t * p.qo_st + (long)h * p.qo_sh : p.k_out + (long)t * p.ko_st + (long)h * p.ko_sh;
            *(u32x4*)(dst + d0) = olo;
            *(u32x4*)(dst + d0 + HD / 2) = ohi;
        }
        if (is_q) continue;
        if constexpr (E4M3) {
            unpack8f(olo, lo);  // the cache's numbers are bf16 ones, whichever way it holds them
            unpack8f(ohi, hi);
            float amax = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fmaxf(finite_abs(lo[j]), finite_abs(hi[j])));
#pragma unroll
            for (int o = LPV / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
            const int e = row_exponent(amax);
            const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
            if (at.page < 0) continue;
            uint8_t* dst = (uint8_t*)(is_k ? p.c.k : p.c.v) + at.page * p.c.s_page + (long)h * p.c.s_head + slot * p.c.s_tok;
            *(u32x2*)(dst + d0) = u32x2{e4m3_pack4(lo, inv), e4m3_pack4(lo + 4, inv)};
            *(u32x2*)(dst + d0 + HD / 2) = u32x2{e4m3_pack4(hi, inv), e4m3_pack4(hi + 4, inv)};
            if (sub == 0) (is_k ? p.c.k_scale : p.c.v_scale)[at.page * p.c.ss_page + (long)h * p.c.ss_head + slot] = (uint8_t)(e + 127);
        } else {
            if (at.page < 0) continue;
            bf16_t* dst = (bf16_t*)(is_k ? p.c.k : p.c.v) + at.page * p.c.s_page + (long)h * p.c.s_head + slot * p.c.s_tok;
            *(u32x4*)(dst + d0) = olo;
            *(u32x4*)(dst + d0 + HD / 2) = ohi;
        }
    }
}

// ---- read ----
template <int HD, bool E4M3>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedReadArgs p) {
    constexpr int LPV = HD / 8, VPB = 256 / LPV;
    const int t = blockIdx.x;
    const TokenPlace at = place_of_token(p.c, p.offsets, p.start, t);
    if (at.idle) return;
    const int d0 = (threadIdx.x % LPV) * 8, Hkv = p.c.kv_heads;
    const long slot = at.pos & ((1 << p.c.page_log2) - 1);
    for (int i = threadIdx.x / LPV; i < 2 * Hkv; i += VPB) {
        const bool is_k = i < Hkv;
        const int h = is_k ? i : i - Hkv;
        u32x4 o = {0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};  // NaN: a position without a page
        if (at.page >= 0) {
            const long off = at.page * p.c.s_page + (long)h * p.c.s_head + slot * p.c.s_tok + d0;
            if constexpr (E4M3) {
                float f[8];
                e4m3_unpack8(*(const u32x2*)((const uint8_t*)(is_k ? p.c.k : p.c.v) + off), f);
                const int e = (int)(is_k ? p.c.k_scale : p.c.v_scale)[at.page * p.c.ss_page + (long)h * p.c.ss_head + slot] - 127;
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = pack2bf(ldexpf(f[2 * j], e), ldexpf(f[2 * j + 1], e));
            } else {
                o = *(const u32x4*)((const bf16_t*)(is_k ? p.c.k : p.c.v) + off);
            }
        }
        bf16_t* dst = is_k ? p.k_out + (long)t * p.ko_st + (long)h * p.ko_sh : p.v_out + (long)t * p.vo_st + (long)h * p.vo_sh;
        *(u32x4*)(dst + d0) = o;
    }
}

// ---- attention of one new token ----
// out = softmax(scale q K^T) V for a block of up to 16 query heads that share a kv head, in one pass over the pages. A wave takes 32 positions at a time:
//   S^T = K Q^T  (v_mfma_f32_16x16x32_bf16, A = 16 keys x 32 dims, B = the heads' queries): a lane gets, for head lane % 16, the scores of positions
//                4 (lane / 16) + i of each half tile -- which is, half after half, the layout of the B operand of
//   O^T += V^T P^T (A = 16 dims x 32 positions): the order of the summed positions is free, so P goes from one product into the other in registers.
// V's operand wants 8 positions of one dim in a lane; a lane loads 8 positions x HD/16 neighbouring dims in whole lines and transposes them in registers
// (v_perm_b32), row r of product dt being dim r * HD/16 + dt. Nothing passes through LDS until the four waves of a workgroup meet.
// Scores, maximum, sum and output are fp32. A weight p is used as the sum of two bf16 numbers, p cut off and the rest rounded (2^-15 relative: one bf16
// alone would add as much error as the output's own rounding); where values may be infinite the rest is kept above zero (by 2^-20 p), so that it
// neither turns an infinity round nor makes it NaN. The running maximum moves only when a score exceeds it by 2^6: the rescaling of the 32 output
// registers is then rare, and nothing overflows that would not without it.
// e4m3 codes become bf16 exactly; a key's power of two multiplies its score, a value's its weight.
constexpr float RAISE = 6.f;

template <int HD, bool E4M3>
struct PagedTile {  // 32 positions of one head in a wave's registers
    static constexpr int DV = HD / 16;                  // dims of a value in a lane
    static constexpr int KL = E4M3 ? HD / 64 : HD / 32; // 16-byte loads of a key's lane share
    static constexpr int VW = E4M3 ? DV / 4 : DV / 2;   // words of a value's lane share
    u32x4 k[2][KL];
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

// tile at position tok (a multiple of 16): its halves lie in pages id0 and id1. `half1` is where the second half is read from: tok + 16, or tok again
// where that is behind the row's last position
template <int HD, bool E4M3>
MERV_DEVICE void load_tile(PagedTile<HD, E4M3>& t, const PagedCacheArgs& c, int hkv, long tok, long half1, int id0, int id1) {
    typedef PagedTile<HD, E4M3> Tile;
    constexpr int ELT = E4M3 ? 1 : 2;
    const int lane = threadIdx.x & 63, r = lane & 15, tg = lane >> 4;
    const int mask = (1 << c.page_log2) - 1;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
        const long id = tt ? id1 : id0;
        const int slot = (int)((tt ? half1 : tok) & mask);
        const long at = (id * c.s_page + (long)hkv * c.s_head + slot * c.s_tok) * ELT;
        const char* kp = (const char*)c.k + at;
        const char* vp = (const char*)c.v + at;
        const unsigned krow = (unsigned)r * (unsigned)(c.s_tok * ELT) + tg * 16;
#pragma unroll
        for (int j = 0; j < Tile::KL; ++j) t.k[tt][j] = *(const u32x4*)(kp + (krow + j * 64));
        const unsigned vrow = (unsigned)tg * 4u * (unsigned)(c.s_tok * ELT) + r * Tile::DV * ELT;
#pragma unroll
        for (int i = 0; i < 4; ++i) load_words(t.v[tt * 4 + i], vp + i * c.s_tok * ELT + vrow);
        if constexpr (E4M3) {
            const long sat = id * c.ss_page + (long)hkv * c.ss_head + slot;
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

template <int HD, bool E4M3>
MERV_DEVICE void use_tile(PagedState<HD>& st, PagedTile<HD, E4M3>& t, const bf16x8 (&q)[HD / 32], float scale2, long tok, long lo, long len) {
    typedef PagedTile<HD, E4M3> Tile;
    const int lane = threadIdx.x & 63, tg = lane >> 4;
    f32x4 s[2];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
        s[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
            bf16x8 a;
            if constexpr (E4M3) {
                const uint32_t w0 = t.k[tt][j >> 1][(j & 1) * 2], w1 = t.k[tt][j >> 1][(j & 1) * 2 + 1];
                a = __builtin_bit_cast(bf16x8, u32x4{e4m3_pair(w0, 0), e4m3_pair(w0, 1), e4m3_pair(w1, 0), e4m3_pair(w1, 1)});
            } else {
                a = __builtin_bit_cast(bf16x8, t.k[tt][j]);
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
                const long j = tok + tt * 16 + tg * 4 + i;
                const bool seen = j >= lo && j < len;
                s[tt][i] = seen ? s[tt][i] : -INFINITY;
#pragma unroll
                for (int w = 0; w < Tile::VW; ++w) t.v[tt * 4 + i][w] = seen ? t.v[tt * 4 + i][w] : 0u;
                if constexpr (E4M3) t.vs[tt] = seen ? t.vs[tt] : t.vs[tt] & ~(0xffu << (8 * i));
            }
    }
    float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    top = max_over_rows(top);
    if (__any(top > st.m + RAISE)) {
        const float m = fmaxf(st.m, top);
        const float a = __builtin_amdgcn_exp2f(st.m - (m == -INFINITY ? 0.f : m));
        st.m = m;
        st.l *= a;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) st.o[d] *= a;
    }
    const float base = st.m == -INFINITY ? 0.f : st.m;
    uint32_t hi[4], lo_[4];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[i] = __builtin_amdgcn_exp2f(s[tt][i] - base);
            st.l += p[i];
            if constexpr (E4M3) p[i] = ldexpf(p[i], (int)((t.vs[tt] >> (8 * i)) & 0xff) - 127);
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const float p0 = p[2 * w], p1 = p[2 * w + 1];
            const uint32_t h0 = __float_as_uint(p0) & 0xffff0000u, h1 = __float_as_uint(p1) & 0xffff0000u;
            float l0 = p0 - __uint_as_float(h0), l1 = p1 - __uint_as_float(h1);
            if constexpr (!E4M3) l0 = fmaxf(l0, p0 * 0x1p-20f), l1 = fmaxf(l1, p1 * 0x1p-20f);
            hi[tt * 2 + w] = __builtin_amdgcn_perm(h1, h0, 0x07060302u);
            lo_[tt * 2 + w] = pack2bf(l0, l1);
        }
    }
    const bf16x8 ph = __builtin_bit_cast(bf16x8, u32x4{hi[0], hi[1], hi[2], hi[3]});
    const bf16x8 pl = __builtin_bit_cast(bf16x8, u32x4{lo_[0], lo_[1], lo_[2], lo_[3]});
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
        st.o[2 * w] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, even), ph, st.o[2 * w], 0, 0, 0);
        st.o[2 * w + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, odd), ph, st.o[2 * w + 1], 0, 0, 0);
        st.o[2 * w] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, even), pl, st.o[2 * w], 0, 0, 0);
        st.o[2 * w + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, odd), pl, st.o[2 * w + 1], 0, 0, 0);
    }
}

// The units of `rows` rows, summed: thread t has those of rows t * per ... Returns the total; `before`: those of the rows before the thread's own.
// Called by all 256 threads; scratch: 4 ints.
MERV_DEVICE int scan_units(int mine, int& before, int* scratch) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    if (lane == 63) scratch[wave] = x;
    __syncthreads();
    int total = 0, under = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < wave) under += scratch[w];
        total += scratch[w];
    }
    before = under + x - mine;
    return total;
}

MERV_DEVICE PagedSpan span_of(const PagedAttnArgs& p, int row) {
    return paged_span(p.lens[row], p.window, (long)p.c.table_width << p.c.page_log2);
}

template <int HD>
struct PagedLds {
    float o[4][PAGED_HEAD_BLOCK][HD];
    float m[4][PAGED_HEAD_BLOCK], l[4][PAGED_HEAD_BLOCK];
    int scan[4], row, before;
};

// units u .. u + n - 1 of one pair, by the whole workgroup. slot < 0: all of the pair, the result is written.
template <int HD, bool E4M3>
MERV_DEVICE void paged_segment(const PagedAttnArgs& p, PagedLds<HD>& lds, int row, int pair, const PagedSpan sp, int u, int n, int slot) {
    constexpr int DV = HD / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = p.H / p.c.kv_heads, blocks = p.head_blocks;
    const int hkv = pair / blocks, hb = pair - hkv * blocks;
    const int h0 = hkv * group + hb * PAGED_HEAD_BLOCK;
    const int heads = min(PAGED_HEAD_BLOCK, group - hb * PAGED_HEAD_BLOCK);
    // the first dims of a lane's keys: bf16 16 bytes of every 64; e4m3 16 codes of every 64
    bf16x8 q[HD / 32];
    {
        const bf16_t* qp = p.q + (long)row * p.q_st + (long)(h0 + min(lane & 15, heads - 1)) * p.q_sh;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
            const int d = E4M3 ? (j >> 1) * 64 + (lane >> 4) * 16 + (j & 1) * 8 : j * 32 + (lane >> 4) * 8;
            q[j] = __builtin_bit_cast(bf16x8, *(const u32x4*)(qp + d));
        }
    }
    PagedState<HD> st;
    st.m = -INFINITY;
    st.l = 0.f;
#pragma unroll
    for (int d = 0; d < DV; ++d) st.o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float scale2 = p.scale * LOG2E;
    const int* table = p.c.table + (long)row * p.c.table_stride;
    const long first = sp.base + (long)u * PAGED_UNIT + wave * 32;  // this wave's tiles: first + 128 i
    const long left = sp.len - first;
    const int tiles = left <= 0 ? 0 : min(n, (int)((left + PAGED_UNIT - 1) / PAGED_UNIT));
    bool bad = false;
    for (int t0 = 0; t0 < tiles; t0 += 32) {
        // the pages of the next 32 tiles' halves, one in each lane; a half behind the row's end takes the page of the row's last position
        long half = first + (long)(t0 + (lane >> 1)) * PAGED_UNIT + (lane & 1) * 16;
        half = half < sp.len ? half : sp.len - 1;
        int ids = table[half >> p.c.page_log2];
        if (ids < 0 || ids >= p.c.n_pages) {
            bad = true;
            ids = 0;
        }
        const int end = min(32, tiles - t0);
        const long tok0 = first + (long)t0 * PAGED_UNIT;
        PagedTile<HD, E4M3> a, b;
        auto load = [&](PagedTile<HD, E4M3>& t, int i) {
            const long tok = tok0 + (long)i * PAGED_UNIT;
            load_tile(t, p.c, hkv, tok, tok + 16 < sp.len ? tok + 16 : tok, __builtin_amdgcn_readlane(ids, 2 * i), __builtin_amdgcn_readlane(ids, 2 * i + 1));
        };
        auto use = [&](PagedTile<HD, E4M3>& t, int i) { use_tile(st, t, q, scale2, tok0 + (long)i * PAGED_UNIT, sp.lo, sp.len); };
        if (p.c.n_pages > 0) {
            load(a, 0);
            for (int i = 0; i < end; i += 2) {
                if (i + 1 < end) load(b, i + 1);
                use(a, i);
                if (i + 1 < end) {
                    if (i + 2 < end) load(a, i + 2);
                    use(b, i + 1);
                }
            }
        }
    }
    st.l = sum_over_rows(st.l);
    if (__any(bad)) st.l = __builtin_nanf("");
    const int h = lane & 15;
    if (h < heads) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < DV; ++d) lds.o[wave][h][((lane >> 4) * 4 + i) * DV + d] = st.o[d][i];
        if (lane < 16) {
            lds.m[wave][h] = st.m;
            lds.l[wave][h] = st.l;
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < heads * HD; e += 256) {
        const int hh = e / HD, d = e % HD;
        const float M = fmaxf(fmaxf(lds.m[0][hh], lds.m[1][hh]), fmaxf(lds.m[2][hh], lds.m[3][hh])), base = M == -INFINITY ? 0.f : M;
        float L = 0.f, O = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(lds.m[w][hh] - base);
            L += f * lds.l[w][hh];
            O += f * lds.o[w][hh][d];
        }
        if (slot < 0) {
            p.out[(long)row * p.o_st + (long)(h0 + hh) * p.o_sh + d] = f2bf(O / L);
            if (p.lse && d == 0) p.lse[(long)row * p.H + h0 + hh] = (M + __builtin_amdgcn_logf(L)) * LN2;
        } else {
            float* ws = (float*)p.ws + ((size_t)slot * PAGED_HEAD_BLOCK + hh) * (HD + 4);
            ws[d] = O;
            if (d == 0) {
                ws[HD] = M;
                ws[HD + 1] = L;
            }
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

// DIRECT: a workgroup for each pair of each row, which writes the result. Else the line of units is shared out (paged_split.h).
template <int HD, bool E4M3, bool DIRECT>
__global__ __launch_bounds__(256, 2) void paged_attention_kernel(PagedAttnArgs p) {
    __shared__ PagedLds<HD> lds;
    const int pairs = p.c.kv_heads * p.head_blocks;
    if constexpr (DIRECT) {
        const int row = blockIdx.x / pairs, pair = blockIdx.x % pairs;
        const PagedSpan sp = span_of(p, row);
        if (sp.units > 0) {
            paged_segment<HD, E4M3>(p, lds, row, pair, sp, 0, sp.units, -1);
        } else {
            const int group = p.H / p.c.kv_heads, hkv = pair / p.head_blocks, hb = pair % p.head_blocks;
            const int heads = min(PAGED_HEAD_BLOCK, group - hb * PAGED_HEAD_BLOCK);
            for (int e = threadIdx.x; e < heads * HD; e += 256) write_unseen<HD>(p, row, hkv * group + hb * PAGED_HEAD_BLOCK + e / HD, e % HD);
        }
    } else {
        const int rows = p.c.rows, per = (rows + 255) / 256, r0 = min(rows, (int)threadIdx.x * per), r1 = min(rows, r0 + per);
        int mine = 0, before = 0;
        for (int r = r0; r < r1; ++r) mine += span_of(p, r).units;
        const long total = (long)scan_units(mine, before, lds.scan) * pairs;
        const int workers = paged_workers(total, gridDim.x), w = blockIdx.x;
        if (w >= workers) return;
        const long begin = paged_start(w, total, workers), end = paged_start(w + 1, total, workers);
        if (begin >= (long)before * pairs && begin < (long)(before + mine) * pairs) {  // this thread's rows hold the first unit
            int r = r0;
            for (; r < r1; ++r) {
                const int n = span_of(p, r).units;
                if (begin < (long)(before + n) * pairs) break;
                before += n;
            }
            lds.row = r;
            lds.before = before;
        }
        __syncthreads();
        int row = __builtin_amdgcn_readfirstlane(lds.row);
        PagedSpan sp = span_of(p, row);
        const long in_row = begin - (long)__builtin_amdgcn_readfirstlane(lds.before) * pairs;
        int pair = (int)(in_row / sp.units), u = (int)(in_row % sp.units);
        for (long x = begin; x < end;) {
            const int n = (int)min((long)(sp.units - u), end - x);
            paged_segment<HD, E4M3>(p, lds, row, pair, sp, u, n, n == sp.units ? -1 : x == begin ? 2 * w : 2 * w + 1);
            x += n;
            u = 0;
            if (++pair == pairs && x < end) {
                pair = 0;
                do sp = span_of(p, ++row);
                while (sp.units == 0);
            }
        }
    }
}

// one workgroup for a row and a query head: the partial sums of its pair, 256 / HD of them at a time
template <int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs p) {
    constexpr int PARTS = 256 / HD;
    __shared__ int scan[4], found;
    __shared__ float sm[PARTS][2], so[PARTS][HD];
    const int row = blockIdx.x / p.H, h = blockIdx.x % p.H, pairs = p.c.kv_heads * p.head_blocks;
    const int rows = p.c.rows, per = (rows + 255) / 256, r0 = min(rows, (int)threadIdx.x * per), r1 = min(rows, r0 + per);
    int mine = 0, before = 0;
    for (int r = r0; r < r1; ++r) mine += span_of(p, r).units;
    const long total = (long)scan_units(mine, before, scan) * pairs;
    if (row >= r0 && row < r1) {
        for (int r = r0; r < row; ++r) before += span_of(p, r).units;
        found = before;
    }
    __syncthreads();
    const int part = threadIdx.x / HD, d = threadIdx.x % HD;
    const int units = span_of(p, row).units;
    if (units == 0) {
        if (part == 0) write_unseen<HD>(p, row, h, d);
        return;
    }
    const int group = p.H / p.c.kv_heads, hkv = h / group, hb = (h % group) / PAGED_HEAD_BLOCK, hh = (h % group) % PAGED_HEAD_BLOCK;
    const long first = (long)found * pairs + (long)(hkv * p.head_blocks + hb) * units;
    const int workers = paged_workers(total, p.workers);
    const int w0 = paged_owner(first, total, workers), w1 = paged_owner(first + units - 1, total, workers);
    if (w0 == w1) return;  // written by its worker
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int w = w0 + part; w <= w1; w += PARTS) {
        const float* ws = (const float*)p.ws + ((size_t)paged_slot(w, first, total, workers) * PAGED_HEAD_BLOCK + hh) * (HD + 4);
        const float m = ws[HD], l = ws[HD + 1], o = ws[d];
        const float top = fmaxf(M, m), base = top == -INFINITY ? 0.f : top;
        const float a = __builtin_amdgcn_exp2f(M - base), b = __builtin_amdgcn_exp2f(m - base);
        L = L * a + l * b;
        O = O * a + o * b;
        M = top;
    }
    so[part][d] = O;
    if (d == 0) {
        sm[part][0] = M;
        sm[part][1] = L;
    }
    __syncthreads();
    if (part) return;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) top = fmaxf(top, sm[i][0]);
    const float base = top == -INFINITY ? 0.f : top;
    L = O = 0.f;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        const float f = __builtin_amdgcn_exp2f(sm[i][0] - base);
        L += f * sm[i][1];
        O += f * so[i][d];
    }
    p.out[(long)row * p.o_st + (long)h * p.o_sh + d] = f2bf(O / L);
    if (p.lse && d == 0) p.lse[(long)row * p.H + h] = (top + __builtin_amdgcn_logf(L)) * LN2;
}

}  // namespace

hipError_t launch_paged_write(const PagedWriteArgs& a, hipStream_t s) {
    if (a.T <= 0) return hipSuccess;
    const dim3 grid((unsigned)a.T), block(256);
    if (a.c.hd == 128) {
        if (a.c.e4m3) hipLaunchKernelGGL((paged_write_kernel<128, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((paged_write_kernel<128, false>), grid, block, 0, s, a);
    } else if (a.c.hd == 64) {
        if (a.c.e4m3) hipLaunchKernelGGL((paged_write_kernel<64, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((paged_write_kernel<64, false>), grid, block, 0, s, a);
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_paged_read(const PagedReadArgs& a, hipStream_t s) {
    if (a.T <= 0) return hipSuccess;
    const dim3 grid((unsigned)a.T), block(256);
    if (a.c.hd == 128) {
        if (a.c.e4m3) hipLaunchKernelGGL((paged_read_kernel<128, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((paged_read_kernel<128, false>), grid, block, 0, s, a);
    } else if (a.c.hd == 64) {
        if (a.c.e4m3) hipLaunchKernelGGL((paged_read_kernel<64, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((paged_read_kernel<64, false>), grid, block, 0, s, a);
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

// What a call launches, from sizes alone (the rows' lengths are on the device): up to DIRECT_UNITS units a row, one workgroup for each pair takes the
// whole row and there is no join.
constexpr long DIRECT_UNITS = 4;

struct PagedPlan {
    int head_blocks, workers;
    bool direct;
};
static PagedPlan paged_plan(int rows, int H, int kv_heads, long capacity) {
    PagedPlan pl;
    pl.head_blocks = (H / kv_heads + PAGED_HEAD_BLOCK - 1) / PAGED_HEAD_BLOCK;
    const long units = (capacity + PAGED_UNIT - 1) / PAGED_UNIT;
    const long most = units * rows * kv_heads * pl.head_blocks;
    pl.direct = units <= DIRECT_UNITS;
    pl.workers = (int)(most < PAGED_MAX_WORKERS ? most : PAGED_MAX_WORKERS);
    return pl;
}

size_t paged_attention_workspace_bytes(int rows, int H, int kv_heads, int hd, long capacity) {
    const PagedPlan pl = paged_plan(rows, H, kv_heads, capacity);
    return pl.direct ? 0 : (size_t)2 * pl.workers * PAGED_HEAD_BLOCK * (hd + 4) * sizeof(float);
}

template <int HD, bool E4M3>
static hipError_t launch_paged_attention_as(const PagedAttnArgs& a, bool direct, hipStream_t s) {
    if (direct) {
        hipLaunchKernelGGL((paged_attention_kernel<HD, E4M3, true>), dim3((unsigned)(a.c.rows * a.c.kv_heads * a.head_blocks)), dim3(256), 0, s, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((paged_attention_kernel<HD, E4M3, false>), dim3((unsigned)a.workers), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((paged_join_kernel<HD>), dim3((unsigned)(a.c.rows * a.H)), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_paged_attention(const PagedAttnArgs& args, hipStream_t s) {
    if (args.c.rows <= 0) return hipSuccess;
    PagedAttnArgs a = args;
    const PagedPlan pl = paged_plan(a.c.rows, a.H, a.c.kv_heads, (long)a.c.table_width << a.c.page_log2);
    a.head_blocks = pl.head_blocks;
    a.workers = pl.workers;
    if (a.c.hd == 128) return a.c.e4m3 ? launch_paged_attention_as<128, true>(a, pl.direct, s) : launch_paged_attention_as<128, false>(a, pl.direct, s);
    if (a.c.hd == 64) return a.c.e4m3 ? launch_paged_attention_as<64, true>(a, pl.direct, s) : launch_paged_attention_as<64, false>(a, pl.direct, s);
    return hipErrorInvalidValue;
}

}  // namespace merv
