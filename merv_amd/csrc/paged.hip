// The paged key / value cache: rows of unlike length share one pool of pages, and a table names the page of every stretch of positions of a row.
//   write      new keys / values (rotated by position, with the queries) into the pages, quantised to 8 bits where the cache holds e4m3
//   read       cached keys / values back as contiguous bf16
//   attention  one new token for each row over the row's pages
// Every index that comes from device memory (row offsets, lengths, page numbers) is checked here before it becomes an address: a position without
// a page is not written and what would have been read from it is NaN, so that a bad table shows in the result and in that row alone.
#include "common.h"
#include "kernels.h"

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
// One block for a row and a query head: 16 groups of 16 lanes take the positions in turn, each with a running maximum and sum of its own (softmax in
// one pass over the cache), and meet in LDS.
template <int HD, bool E4M3>
__global__ __launch_bounds__(256) void paged_attention_kernel(PagedAttnArgs p) {
    constexpr int DPL = HD / 16;  // elements of a vector in a lane
    __shared__ float sm_m[16], sm_l[16];
    __shared__ float sm_o[16][HD];
    const int b = blockIdx.y, h = blockIdx.x, hkv = h / (p.H / p.c.kv_heads);
    const int g = threadIdx.x >> 4, sub = threadIdx.x & 15;
    long n = p.lens[b];
    const long most = (long)p.c.table_width << p.c.page_log2;
    bool bad = n > most;
    n = n < 0 ? 0 : n > most ? most : n;
    const long j0 = p.window > 0 && n > p.window ? n - p.window : 0;
    float q[DPL], o[DPL], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < DPL; ++d) {
        q[d] = bf2f(p.q[(long)b * p.q_st + (long)h * p.q_sh + sub * DPL + d]);
        o[d] = 0.f;
    }
    for (long j = j0 + g; j < n; j += 16) {
        int id = p.c.table[(long)b * p.c.table_stride + (j >> p.c.page_log2)];
        if (id < 0 || id >= p.c.n_pages) {
            bad = true;
            continue;
        }
        const long slot = j & ((1 << p.c.page_log2) - 1);
        const long off = id * p.c.s_page + (long)hkv * p.c.s_head + slot * p.c.s_tok + sub * DPL;
        float k[DPL], v[DPL], ks = 1.f, vs = 1.f;
        if constexpr (E4M3) {
            const long so = id * p.c.ss_page + (long)hkv * p.c.ss_head + slot;
            ks = ldexpf(1.f, (int)p.c.k_scale[so] - 127);
            vs = ldexpf(1.f, (int)p.c.v_scale[so] - 127);
#pragma unroll
            for (int d = 0; d < DPL; ++d) {
                k[d] = __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t*)p.c.k)[off + d], 0);
                v[d] = __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t*)p.c.v)[off + d], 0);
            }
        } else {
#pragma unroll
            for (int d = 0; d < DPL; ++d) {
                k[d] = bf2f(((const bf16_t*)p.c.k)[off + d]);
                v[d] = bf2f(((const bf16_t*)p.c.v)[off + d]);
            }
        }
        float s = 0.f;
#pragma unroll
        for (int d = 0; d < DPL; ++d) s = fmaf(q[d], k[d], s);
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) s += __shfl_xor(s, x, 64);
        s *= p.scale * LOG2E * ks;
        const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
        const float a = __builtin_amdgcn_exp2f(m - base), e = __builtin_amdgcn_exp2f(s - base);
        m = top;
        l = l * a + e;
#pragma unroll
        for (int d = 0; d < DPL; ++d) o[d] = o[d] * a + e * vs * v[d];
    }
    if (bad) l = __builtin_nanf("");
    if (sub == 0) {
        sm_m[g] = m;
        sm_l[g] = l;
    }
#pragma unroll
    for (int d = 0; d < DPL; ++d) sm_o[g][sub * DPL + d] = o[d];
    __syncthreads();
    if (threadIdx.x >= HD) return;
    float M = -INFINITY;
    for (int i = 0; i < 16; ++i) M = fmaxf(M, sm_m[i]);
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f, O = 0.f;
    for (int i = 0; i < 16; ++i) {
        const float w = __builtin_amdgcn_exp2f(sm_m[i] - base);
        L += w * sm_l[i];
        O += w * sm_o[i][threadIdx.x];
    }
    p.out[(long)b * p.o_st + (long)h * p.o_sh + threadIdx.x] = f2bf(n == 0 && !bad ? 0.f : O / L);
    if (p.lse && threadIdx.x == 0) p.lse[(long)b * p.H + h] = n == 0 && !bad ? -INFINITY : (M + __builtin_amdgcn_logf(L)) * LN2;
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

size_t paged_attention_workspace_bytes(int, int, int, int, long) { return 0; }

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t s) {
    if (a.c.rows <= 0) return hipSuccess;
    const dim3 grid((unsigned)a.H, (unsigned)a.c.rows), block(256);
    if (a.c.hd == 128) {
        if (a.c.e4m3) hipLaunchKernelGGL((paged_attention_kernel<128, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((paged_attention_kernel<128, false>), grid, block, 0, s, a);
    } else if (a.c.hd == 64) {
        if (a.c.e4m3) hipLaunchKernelGGL((paged_attention_kernel<64, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((paged_attention_kernel<64, false>), grid, block, 0, s, a);
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace merv
