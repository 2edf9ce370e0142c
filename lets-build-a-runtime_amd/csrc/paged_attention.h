// paged_attention.h — what the kernels of attention over the paged cache share.
//
// Row i of sequence b attends to positions 0 .. start[b] + i; the rows of the query heads that share a K/V
// head go together, row r of a K/V head being token r / G of its query head r % G.
//
// Products run on the fp16 matrix cores with 32-bit accumulators.  A stored K or V value is an fp16 number
// exactly (int8, e4m3, float16) or the sum of two to 22 bits (float32, scaled into range by its row's power
// of two); q and the weights are split into two fp16 numbers each, h = fp16(x), l = fp16(x − h), so that a
// product of an exact value takes two MFMAs and one of two split ones three (the product of the low halves, below
// 2^-22 of the whole, is left out).  Rows of q are brought to [2^14, 2^15) by a power of two first, and weights are
// taken times the V row's scale over a running power of two, so that nothing overflows and the low halves
// keep their bits.  The error against 64 bits is that of a 32-bit product (2e-7 .. 5e-7 of the outputs' norm).
#pragma once

#include <math.h>

#include "paged_common.h"

// Launchers: rows of at most 32 a K/V head (paged_attention.hip), and more (paged_tiles.hip).
step_fn paged_tiles_launcher(int type, int hd);
// Ranges of the keys of paged_tiles (Step::i[10]), and its workspace.
int paged_tiles_splits(const Step& s);
size_t paged_tiles_workspace(const Step& s);
// Row tiles of a K/V head.
int paged_row_tiles(const Step& s);

namespace {

constexpr float LOG2E = 1.44269504088896340736f;

struct PagedAttn {
    PagedCache c;
    const float* q;           // [B][H][S][hd]
    float* out;
    float* parts;             // partial results of split segments
    int B, H, G, S;           // G: query heads of a K/V head
    int G_m, G_s;             // divisor by G (lbr_fdiv)
    int rows;                 // G · S: rows of a K/V head
    float scale;              // of the scores, times log2 e
    bool vec;                 // rows of q and out on 16-byte boundaries
};

// A sequence's rows and keys: count of rows 0 .. S, keys 0 .. the table's end, at most 2^30 (0 where start is negative).
struct Span {
    int start, count, keys;
};
__device__ __forceinline__ Span span_of(const PagedAttn& a, int b) {
    Span s;
    s.start = a.c.start[b];
    s.count = min(max(a.c.count[b], 0), a.S);
    const long long all = (long long)s.start + s.count, cap = (long long)a.c.wide << a.c.shift;
    s.keys = s.start < 0 || s.count == 0 ? 0 : (int)min(all, cap);
    return s;
}

// The last key of a row, −1 for a row that has none; a row that reaches past the table ends with the table.
__device__ __forceinline__ int last_key(const Span& s, int token) {
    return token < s.count ? (int)min((long long)s.start + token, (long long)s.keys - 1) : -1;
}

// A row's result from its sum: zeros behind the sequence's rows, NaN where the table does not reach.
__device__ __forceinline__ float row_value(const PagedAttn& a, const Span& s, int token, float v) {
    if (token >= s.count) return 0.f;
    return s.start < 0 || (long long)s.start + token >= ((long long)a.c.wide << a.c.shift) ? __uint_as_float(0x7fc00000u) : v;
}

// ---------------------------------------------------------------- fp16 operands

__device__ __forceinline__ halfx2 to_half2(float x, float y) {
    return __builtin_convertvector((floatx2{x, y}), halfx2);
}

// h + l of eight floats.
__device__ __forceinline__ void split8(const float (&x)[8], halfx8& h, halfx8& l) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const halfx2 hi = to_half2(x[2 * k], x[2 * k + 1]);
        const halfx2 lo = to_half2(x[2 * k] - (float)hi[0], x[2 * k + 1] - (float)hi[1]);
        h[2 * k] = hi[0];
        h[2 * k + 1] = hi[1];
        l[2 * k] = lo[0];
        l[2 * k + 1] = lo[1];
    }
}

// Eight stored one-byte values (two words) as fp16.
template <int TYPE>
__device__ __forceinline__ halfx8 widen8(unsigned w0, unsigned w1) {
    union {
        halfx2 h[4];
        halfx8 v;
    } r;
    const unsigned w[2] = {w0, w1};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if constexpr (TYPE == LBR_CACHE_I8) {
            // byte + 128 under the exponent of 1024: 1024 + 128 + x, exactly
            const unsigned u = w[k] ^ 0x80808080u;
            const halfx2 bias = {(_Float16)-1152.f, (_Float16)-1152.f};
            r.h[2 * k] = __builtin_bit_cast(halfx2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + bias;
            r.h[2 * k + 1] = __builtin_bit_cast(halfx2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + bias;
        } else {
            r.h[2 * k] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[k], 1.0f, false);
            r.h[2 * k + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[k], 1.0f, true);
        }
    }
    return r.v;
}

// max / sum over the four lanes that hold the same row (lane ^ 16, lane ^ 32).
__device__ __forceinline__ float quad_max(float v) {
    const unsigned u = __float_as_uint(v);
    auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const unsigned w = __float_as_uint(v);
    auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quad_sum(float v) {
    const unsigned u = __float_as_uint(v);
    auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const unsigned w = __float_as_uint(v);
    auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// Adds a partial result (a row's maximum, sum and weighted mean over some keys) to a running maximum, sum and
// weighted sum.
__device__ __forceinline__ void merge_part(float& m, float& l, floatx4& o, float pm, float pl, floatx4 mean) {
    const float mx = fmaxf(m, pm), base = mx == -INFINITY ? 0.f : mx;
    const float f = __builtin_amdgcn_exp2f(m - base), g = __builtin_amdgcn_exp2f(pm - base) * pl;
    o = o * f + mean * g;
    l = l * f + g;
    m = mx;
}

// Biased exponent of the power of two that brings a magnitude's bits into [2^14, 2^15), at most 2^127.
__device__ __forceinline__ int up_exponent(unsigned bits) { return min(268 - max((int)(bits >> 23), 1), 254); }

PagedAttn attn_args(const Step& s) {
    PagedAttn a;
    a.c = paged_cache(s);
    a.q = (const float*)s.in[4];
    a.out = (float*)s.out;
    a.parts = (float*)s.ws;
    a.B = (int)s.i[1];
    a.H = (int)s.i[8];
    a.S = (int)s.i[7];
    a.G = a.H / a.c.heads;
    lbr_fast_divisor((unsigned)a.G, &a.G_m, &a.G_s);
    a.rows = a.G * a.S;
    a.scale = s.f[0] * LOG2E;
    a.vec = s.i[9] != 0;
    return a;
}

}  // namespace
