// paged.hip — the paged key/value cache: writing a chunk's rows with their scales, and reading
// positions back (layout and types: paged_common.h).
//
// Both move rows at memory speed.  A wavefront takes eight positions that share a V group of one head, in
// the fp32 tensors eight rows in a row: LPR lanes a row hold four columns each, so that an access of the
// wavefront is 1 KiB in a row there (lanes of eight columns, two accesses of every other 16 bytes, took 36 µs for
// 127 MB read back, against 26.6), and a row's largest magnitude is a reduction over LPR lanes.  V changes its order,
// [8][hdp] to [hdp][8], through 8·hdp elements of LDS that only its wavefront touches; a group that the chunk covers
// only in part is written element by element, its other positions left alone.
//
// 4096 positions of 8 heads of 128, int8, 42 MB either way: written in 13 µs (what bounds it beside memory: the row's
// scale is a chain from the loads to the first store), read in 9 (4.8 TB/s).
#include "paged_common.h"

#include <math.h>

namespace {

// ---------------------------------------------------------------- stored values

// x / s, rounded so that one more rounding to fewer bits (at least two fewer) gives what rounding the exact
// quotient once would: toward zero, with the last bit set where anything was cut off.  s > 0; where
// both are tiny they are scaled up, so that the remainder is exact.
__device__ __forceinline__ float quotient_odd(float x, float s) {
#pragma clang fp contract(off)
    if (s < 0x1p-60f) {
        x *= 0x1p64f;
        s *= 0x1p64f;
    }
    const float q = x / s;
    const float r = fmaf(-q, s, x);   // exact: x − q·s has no more bits than s
    unsigned u = __float_as_uint(q);
    // a quotient this small rounds to zero in either type; no remainder: exact
    if (r == 0.f || fabsf(q) < 0x1p-20f) return q;
    if ((r < 0.f) != (q < 0.f)) u -= 1;   // rounded away from zero
    return __uint_as_float(u | 1u);
}

// Scale of a row from the bits of its largest magnitude (as integers, NaN > infinity > finite).
template <int TYPE>
__device__ __forceinline__ float row_scale(unsigned amax) {
    if (amax >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    if (TYPE == LBR_CACHE_F32 || TYPE == LBR_CACHE_F16) {
        const int e = (int)(amax >> 23) - 14;
        return __uint_as_float((unsigned)max(e, 1) << 23);
    }
    const float top = __uint_as_float(amax);
    return fmaxf(TYPE == LBR_CACHE_I8 ? top / 127.0f : top / 448.0f, 0x1p-126f);
}

// A value's stored bytes as the cache and the LDS stage hold them; both are read back in other widths.
typedef unsigned __attribute__((may_alias)) word;
typedef unsigned short __attribute__((may_alias)) word2;
typedef uint2 __attribute__((may_alias)) word8;
typedef uint4 __attribute__((may_alias)) word16;

// Four neighbouring values of a row as stored: one word to four.
template <int TYPE>
struct Quad {
    static constexpr int ES = cache_elem(TYPE);
    unsigned w[ES];

    __device__ __forceinline__ void load(const char* p) {
        if constexpr (ES == 1) {
            w[0] = *(const word*)p;
        } else if constexpr (ES == 2) {
            const uint2 v = *(const word8*)p;
            w[0] = v.x;
            w[1] = v.y;
        } else {
            const uint4 v = *(const word16*)p;
            w[0] = v.x;
            w[1] = v.y;
            w[2] = v.z;
            w[3] = v.w;
        }
    }
    __device__ __forceinline__ void store(char* p) const {
        if constexpr (ES == 1) *(word*)p = w[0];
        else if constexpr (ES == 2) *(word8*)p = make_uint2(w[0], w[1]);
        else *(word16*)p = make_uint4(w[0], w[1], w[2], w[3]);
    }
    // Value q alone, to or from its place.
    __device__ __forceinline__ void store_one(char* p, int q) const {
        if constexpr (ES == 4) *(word*)p = w[q];
        if constexpr (ES == 2) *(word2*)p = (unsigned short)(w[q / 2] >> (16 * (q & 1)));
        if constexpr (ES == 1) *(unsigned char*)p = (unsigned char)(w[0] >> (8 * q));
    }
    __device__ __forceinline__ void load_one(const char* p, int q) {   // q = 0, 1, 2, 3 in turn
        if constexpr (ES == 4) w[q] = *(const word*)p;
        if constexpr (ES == 2) w[q / 2] = (q & 1 ? w[q / 2] : 0u) | (unsigned)*(const word2*)p << (16 * (q & 1));
        if constexpr (ES == 1) w[0] = (q ? w[0] : 0u) | (unsigned)*(const unsigned char*)p << (8 * q);
    }

    // From values and their row's scale (NaN: zeros).
    __device__ __forceinline__ void encode(const float (&x)[4], float s) {
        const bool bad = s != s;
        if constexpr (ES > 1) {
            // s is a power of two, 2^-126 .. 2^113; a product with 1/s would lose -0 in its conversion to
            // halves (one instruction that adds +0)
            const int up = 127 - (int)(__float_as_uint(s) >> 23);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float y = bad ? 0.f : __builtin_amdgcn_ldexpf(x[k], up);
                if constexpr (ES == 4) {
                    w[k] = __float_as_uint(y);
                } else {
                    const unsigned h = __builtin_bit_cast(unsigned short, (_Float16)y);
                    w[k / 2] = (k & 1 ? w[k / 2] : 0u) | h << (16 * (k & 1));
                }
            }
        } else {
            // The quotient lies between x·lo and x·hi; where both round to the same stored values, those are
            // its roundings.  The others, a few in a million and exact ties, are divided.
            const float inv = bad ? 0.f : 1.f / s, lo = inv * (1.f - 0x1p-21f), hi = inv * (1.f + 0x1p-21f);
            if constexpr (TYPE == LBR_CACHE_I8) {
                unsigned u[4], far = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {   // 1.5·2^23 + n holds n in its low bits, rounded once
                    u[k] = __float_as_uint(fmaf(bad ? 0.f : x[k], hi, 0x1.8p23f));
                    far |= u[k] ^ __float_as_uint(fmaf(bad ? 0.f : x[k], lo, 0x1.8p23f));
                }
                if (far) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) u[k] = (unsigned)(int)rintf(quotient_odd(x[k], s));
                }
                w[0] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[3], u[2], 0x0c0c0400u),
                                             __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), 0x05040100u);
            } else {
                auto pack = [](float y0, float y1, float y2, float y3) {
                    const int half = __builtin_amdgcn_cvt_pk_fp8_f32(y0, y1, 0, false);
                    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y2, y3, half, true);
                };
                float y[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] = bad ? 0.f : x[k];
                w[0] = pack(y[0] * hi, y[1] * hi, y[2] * hi, y[3] * hi);
                if (w[0] != pack(y[0] * lo, y[1] * lo, y[2] * lo, y[3] * lo))
                    w[0] = pack(quotient_odd(x[0], s), quotient_odd(x[1], s), quotient_odd(x[2], s), quotient_odd(x[3], s));
            }
        }
    }
    // To values, times their row's scale.
    __device__ __forceinline__ float4 decode(float s) const {
        float y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (ES == 4) y[k] = __uint_as_float(w[k]);
            if constexpr (ES == 2)
                y[k] = (float)__builtin_bit_cast(_Float16, (unsigned short)(w[k / 2] >> (16 * (k & 1))));
            if constexpr (TYPE == LBR_CACHE_I8) y[k] = (float)((int)(w[0] << (24 - 8 * k)) >> 24);
        }
        if constexpr (TYPE == LBR_CACHE_E4M3) {
            const floatx2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[0], false);
            const floatx2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[0], true);
            y[0] = a[0];
            y[1] = a[1];
            y[2] = b[0];
            y[3] = b[1];
        }
        return make_float4(y[0] * s, y[1] * s, y[2] * s, y[3] * s);
    }
};

// Four columns of a row of the fp32 tensors, zeros where there are none.
__device__ __forceinline__ void load4(const float* p, int col, int hd, bool vec, float (&x)[4]) {
    if (vec && col < hd) {   // hd is a multiple of four
        const float4 v = *(const float4*)(p + col);
        x[0] = v.x;
        x[1] = v.y;
        x[2] = v.z;
        x[3] = v.w;
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) x[q] = col + q < hd ? p[col + q] : 0.f;
    }
}
__device__ __forceinline__ void store4(float* p, int col, int hd, bool vec, float4 v) {
    if (vec && col < hd) {
        *(float4*)(p + col) = v;
    } else {
        const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (col + q < hd) p[col + q] = x[q];
    }
}

// ---------------------------------------------------------------- the write

// Unit of a wavefront: (b, h, g), V group start[b]/8 + g of the sequence.  LPR: lanes of a row (head_dim / 4, to 8, 16,
// 32 or 64); pass j takes positions j·64/LPR .. of the group.
template <int TYPE, int LPR>
__global__ __launch_bounds__(256) void cache_write(PagedCache c, const float* __restrict__ k,
                                                   const float* __restrict__ v, int S, int groups, unsigned units,
                                                   bool vec) {
    constexpr int ES = cache_elem(TYPE), RP = 64 / LPR, NP = 8 / RP;
    __shared__ __attribute__((aligned(16))) char stage[4][4 * LPR * 8 * ES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned unit = blockIdx.x * 4u + wave;
    if (unit >= units) return;   // whole wavefronts; no barrier below
    const int g = unit % groups, bh = unit / groups;
    const int h = bh % c.heads, b = bh / c.heads;
    const int start = c.start[b], count = min(max(c.count[b], 0), S);
    const long long group = (start >> 3) + g;           // of eight positions
    const long long row0 = group * 8 - start;           // of the chunk, may lie before it
    if (row0 + 8 <= 0 || row0 >= count) return;
    const int col = lane % LPR * 4;
    float xk[NP][4], xv[NP][4];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const long long row = row0 + j * RP + lane / LPR;
#pragma unroll
        for (int q = 0; q < 4; ++q) xk[j][q] = xv[j][q] = 0.f;
        if (row >= 0 && row < count) {
            const long long at = ((long long)bh * S + row) * c.hd;
            load4(k + at, col, c.hd, vec, xk[j]);
            load4(v + at, col, c.hd, vec, xv[j]);
        }
    }
    char* const head = cache_head(c, b, h, group * 8);   // a group never crosses a page
    if (!head) return;
    const int page_mask = (1 << c.shift) - 1, slot0 = (int)(group * 8) & page_mask;
    const bool full = row0 >= 0 && row0 + 8 <= count;    // else element by element
    char* const vg = head + c.part + (long long)slot0 * c.hdp * ES;   // [hdp][8]
    char* const st = stage[wave];
    char* const to = full ? st : vg;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int r = j * RP + lane / LPR;
        const long long row = row0 + r;
        unsigned mk = 0, mv = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            mk = max(mk, __float_as_uint(xk[j][q]) & 0x7fffffffu);
            mv = max(mv, __float_as_uint(xv[j][q]) & 0x7fffffffu);
        }
        const float sk = row_scale<TYPE>(row_max_bits<LPR>(mk)), sv = row_scale<TYPE>(row_max_bits<LPR>(mv));
        if (row < 0 || row >= count || col >= c.hdp) continue;
        if (col == 0) {
            float* const sc = (float*)(head + 2 * c.part);
            sc[slot0 + r] = sk;
            sc[page_mask + 1 + slot0 + r] = sv;
        }
        Quad<TYPE> pk, pv;
        pk.encode(xk[j], sk);
        pv.encode(xv[j], sv);
        pk.store(head + ((long long)(slot0 + r) * c.hdp + col) * ES);
#pragma unroll
        for (int q = 0; q < 4; ++q) pv.store_one(to + ((col + q) * 8 + r) * ES, q);
    }
    if (full) {
        __builtin_amdgcn_wave_barrier();
        const int bytes = c.hdp * 8 * ES;
        for (int o = lane * 16; o < bytes; o += 1024) *(word16*)(vg + o) = *(const word16*)(st + o);
    }
}

// ---------------------------------------------------------------- the read

// Unit of a wavefront: (b, h, g) as in the write, for rows 0 .. T − 1 from position start[b].
template <int TYPE, int LPR>
__global__ __launch_bounds__(256) void cache_read(PagedCache c, float* __restrict__ out, int B, int T, int groups,
                                                  unsigned units, bool vec) {
    constexpr int ES = cache_elem(TYPE), RP = 64 / LPR, NP = 8 / RP;
    __shared__ __attribute__((aligned(16))) char stage[4][4 * LPR * 8 * ES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned unit = blockIdx.x * 4u + wave;
    if (unit >= units) return;
    const int g = unit % groups, bh = unit / groups;
    const int h = bh % c.heads, b = bh / c.heads;
    const int start = c.start[b], count = min(max(c.count[b], 0), T);
    const long long group = (start >> 3) + g;
    const long long row0 = group * 8 - start;
    if (row0 + 8 <= 0 || row0 >= T) return;
    const bool some = row0 < count;                     // of the rows have a position
    const char* const head = some ? cache_head(c, b, h, group * 8) : nullptr;
    const int page_mask = (1 << c.shift) - 1, slot0 = (int)(group * 8) & page_mask;
    const int col = lane % LPR * 4;
    const float nan = __uint_as_float(0x7fc00000u);
    char* const st = stage[wave];
    Quad<TYPE> pk[NP];
    float sk[NP], sv[NP];
    if (head) {
        const char* const vg = head + c.part + (long long)slot0 * c.hdp * ES;
        const float* const sc = (const float*)(head + 2 * c.part);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int r = j * RP + lane / LPR;
            pk[j].load(head + ((long long)(slot0 + r) * c.hdp + (col < c.hdp ? col : 0)) * ES);
            sk[j] = sc[slot0 + r];
            sv[j] = sc[page_mask + 1 + slot0 + r];
        }
        const int bytes = c.hdp * 8 * ES;
        for (int o = lane * 16; o < bytes; o += 1024) *(word16*)(st + o) = *(const word16*)(vg + o);
        __builtin_amdgcn_wave_barrier();
    }
    const long long half = (long long)B * c.heads * T * c.hd;   // K, then V
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int r = j * RP + lane / LPR;
        const long long row = row0 + r;
        if (row < 0 || row >= T || col >= c.hd) continue;
        float4 yk = make_float4(0.f, 0.f, 0.f, 0.f), yv = yk;
        if (row < count) {
            yk = yv = make_float4(nan, nan, nan, nan);
            if (head) {
                Quad<TYPE> pv;
#pragma unroll
                for (int q = 0; q < 4; ++q) pv.load_one(st + ((col + q) * 8 + r) * ES, q);
                yk = pk[j].decode(sk[j]);
                yv = pv.decode(sv[j]);
            }
        }
        float* const to = out + ((long long)bh * T + row) * c.hd;
        store4(to, col, c.hd, vec, yk);
        store4(to + half, col, c.hd, vec, yv);
    }
}

// ---------------------------------------------------------------- launchers

template <int TYPE, int LPR>
void launch_write(const Step& s, hipStream_t st) {
    const int S = (int)s.i[7], groups = (int)((s.i[7] + 14) / 8);
    const long long units = s.i[1] * s.i[2] * groups;
    if (S <= 0 || units <= 0) return;
    hipLaunchKernelGGL((cache_write<TYPE, LPR>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, paged_cache(s),
                       (const float*)s.in[4], (const float*)s.in[5], S, groups, (unsigned)units, s.i[9] != 0);
}

template <int TYPE, int LPR>
void launch_read(const Step& s, hipStream_t st) {
    const int T = (int)s.i[7], groups = (int)((s.i[7] + 14) / 8);
    const long long units = s.i[1] * s.i[2] * groups;
    if (T <= 0 || units <= 0) return;
    hipLaunchKernelGGL((cache_read<TYPE, LPR>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, paged_cache(s),
                       (float*)s.out, (int)s.i[1], T, groups, (unsigned)units, s.i[9] != 0);
}

// Lanes of a row: the fewest that hold it.  2184 positions of 14 sequences, 21 heads of 24, e4m3: 43 µs written and
// 32 read with 8 lanes, 60 and 37 with 16; head_dim 32, float16: 42 and 41, 53 and 43.
template <int TYPE>
step_fn write_for(int hd) {
    return hd <= 32 ? launch_write<TYPE, 8> : hd <= 64 ? launch_write<TYPE, 16> : hd <= 128 ? launch_write<TYPE, 32> : launch_write<TYPE, 64>;
}
template <int TYPE>
step_fn read_for(int hd) {
    return hd <= 32 ? launch_read<TYPE, 8> : hd <= 64 ? launch_read<TYPE, 16> : hd <= 128 ? launch_read<TYPE, 32> : launch_read<TYPE, 64>;
}

// Whether a launch holds a wavefront for each eight rows of a head: its threads are counted in 32 bits.
bool units_fit(const Step& s, const char* what) {
    const long long groups = (s.i[7] + 14) / 8, most = (1LL << 26) - 4;
    if (s.i[1] <= most / s.i[2] && (s.i[1] == 0 || groups <= most / (s.i[1] * s.i[2]))) return true;
    lbr_set_error("%s: %lld sequences of %lld rows are more than one launch takes", what, s.i[1], s.i[7]);
    return false;
}

}  // namespace

int decode_paged_common(const OpNode* n, Step* s, int cache, int first, long long B) {
    const int* x = n->extra;
    if (n->n_inputs != first + 3 || !n->output) {
        lbr_set_error("expected %d inputs and an output", first + 3);
        return LBR_ERR_INVALID;
    }
    for (int k = 0; k < n->n_inputs; ++k)
        if (!n->inputs[k]) {
            lbr_set_error("input %d is null", k);
            return LBR_ERR_INVALID;
        }
    const int page = x[0], heads = x[1], hd = x[2], type = x[3];
    if (page < 16 || page > 32768 || (page & (page - 1)) || hd < 1 || hd > 256 || heads < 1 || type < 0 || type > 3) {
        lbr_set_error("cache of page_size %d, %d heads of %d, type %d", page, heads, hd, type);
        return LBR_ERR_INVALID;
    }
    const long long head_bytes = (long long)page * (2LL * ((hd + 15) / 16 * 16) * cache_elem(type) + 8);
    if (heads > ((1LL << 31) - 1) / head_bytes || x[4] < 1 || x[5] < 1 || (long long)x[5] * page > (1LL << 30)) {
        lbr_set_error("cache of %d pages of %d heads, tables of %d pages of %d positions", x[4], heads, x[5], page);
        return LBR_ERR_INVALID;
    }
    if (B < 0 || B > LBR_MAX_ELEMENTS / x[5]) {
        lbr_set_error("%lld sequences", B);
        return LBR_ERR_INVALID;
    }
    if (!lbr_aligned(n->inputs[cache], 16)) {
        lbr_set_error("the cache does not start on a 16-byte boundary");
        return LBR_ERR_INVALID;
    }
    for (int k = first; k < first + 3; ++k)
        if (!lbr_aligned(n->inputs[k], 4)) {
            lbr_set_error("input %d does not start on a 4-byte boundary", k);
            return LBR_ERR_INVALID;
        }
    s->in[0] = n->inputs[cache];
    for (int k = 0; k < 3; ++k) s->in[1 + k] = n->inputs[first + k];
    s->out = n->output;
    s->i[0] = type;
    s->i[1] = B;
    s->i[2] = heads;
    s->i[3] = hd;
    s->i[4] = __builtin_ctz((unsigned)page);
    s->i[5] = x[4];
    s->i[6] = x[5];
    return LBR_OK;
}

int decode_cache_write(const OpNode* n, Step* s) {
    if (int rc = decode_paged_common(n, s, 0, 3, n->extra[7])) return rc;
    if (n->inputs[0] != n->output || n->elem_size != 1) {
        lbr_set_error("cache_write: the output is the cache itself, in bytes");
        return LBR_ERR_INVALID;
    }
    if (n->n_dims != 2 || n->out_shape[0] != s->i[5] || n->out_shape[1] != paged_cache(*s).page_bytes) {
        lbr_set_error("cache_write: the output is not a cache of %lld pages of %lld bytes", s->i[5],
                      paged_cache(*s).page_bytes);
        return LBR_ERR_INVALID;
    }
    s->i[7] = n->extra[6];
    if (s->i[7] < 0 || !units_fit(*s, "cache_write")) {
        if (s->i[7] < 0) lbr_set_error("cache_write: %lld rows", s->i[7]);
        return LBR_ERR_INVALID;
    }
    for (int k = 1; k < 3; ++k)
        if (!lbr_aligned(n->inputs[k], 4)) {
            lbr_set_error("cache_write: input %d does not start on a 4-byte boundary", k);
            return LBR_ERR_INVALID;
        }
    s->in[4] = n->inputs[1];
    s->in[5] = n->inputs[2];
    s->i[9] = s->i[3] % 4 == 0 && lbr_aligned(s->in[4], 16) && lbr_aligned(s->in[5], 16);
    const int hd = (int)s->i[3];
    s->run = s->i[0] == LBR_CACHE_F32   ? write_for<LBR_CACHE_F32>(hd)
             : s->i[0] == LBR_CACHE_F16 ? write_for<LBR_CACHE_F16>(hd)
             : s->i[0] == LBR_CACHE_I8  ? write_for<LBR_CACHE_I8>(hd)
                                        : write_for<LBR_CACHE_E4M3>(hd);
    s->name = "cache_write";
    return LBR_OK;
}

int decode_cache_read(const OpNode* n, Step* s) {
    const int* d = n->out_shape;
    if (n->n_dims != 5 || n->elem_size != 4 || d[0] != 2 || d[2] != n->extra[1] || d[4] != n->extra[2]) {
        lbr_set_error("cache_read: the output is not float [2, B, heads, T, head_dim]");
        return LBR_ERR_INVALID;
    }
    if (int rc = decode_paged_common(n, s, 0, 1, d[1])) return rc;
    s->i[7] = d[3];
    if (!units_fit(*s, "cache_read")) return LBR_ERR_INVALID;
    if (!lbr_aligned(s->out, 4)) {
        lbr_set_error("cache_read: the output does not start on a 4-byte boundary");
        return LBR_ERR_INVALID;
    }
    const int hd = (int)s->i[3];
    s->i[9] = hd % 4 == 0 && lbr_aligned(s->out, 16);
    s->run = s->i[0] == LBR_CACHE_F32   ? read_for<LBR_CACHE_F32>(hd)
             : s->i[0] == LBR_CACHE_F16 ? read_for<LBR_CACHE_F16>(hd)
             : s->i[0] == LBR_CACHE_I8  ? read_for<LBR_CACHE_I8>(hd)
                                        : read_for<LBR_CACHE_E4M3>(hd);
    s->name = "cache_read";
    return LBR_OK;
}

long long lbr_paged_input_bytes(const OpNode* n, int k) {
    // products of extents, −1 where one is negative or they pass 2^42
    auto mul = [](std::initializer_list<long long> f) {
        long long r = 1;
        for (long long v : f) {
            if (v < 0 || (v > 0 && r > (LBR_MAX_ELEMENTS * 4) / v)) return -1LL;
            r *= v;
        }
        return r;
    };
    const int* x = n->extra;
    const int* d = n->out_shape;
    if (n->op == OP_VERIFY_DRAFT) {
        if (n->n_dims != 2 || d[1] < 1) return -1;
        const long long B = d[0], D = d[1] - 1;
        switch (k) {
            case 0: return mul({B, D + 1, x[0], 4});
            case 1: return mul({B, D, x[0], 4});
            case 2: return mul({B, D, 8});
            case 3: return mul({B, D + 1, 4});
            default: return k == 4 ? mul({B, 4}) : -1;
        }
    }
    const int first = n->op == OP_CACHE_WRITE ? 3 : n->op == OP_PAGED_ATTENTION ? 2 : 1;
    const int cache = n->op == OP_PAGED_ATTENTION ? 1 : 0;
    const long long B = n->op == OP_CACHE_WRITE ? x[7] : n->op == OP_CACHE_READ ? d[1] : d[0];
    if (k == cache) {
        if (x[3] < 0 || x[3] > 3 || x[2] < 0) return -1;
        const long long row = 2LL * ((x[2] + 15LL) / 16 * 16) * cache_elem(x[3]) + 8;
        return mul({x[4], x[1], x[0], row});
    }
    if (k == first) return mul({B, x[5], 4});
    if (k == first + 1 || k == first + 2) return mul({B, 4});
    if (n->op == OP_CACHE_WRITE && (k == 1 || k == 2)) return mul({B, x[1], x[6], x[2], 4});
    if (n->op == OP_PAGED_ATTENTION && k == 0) return mul({node_total(n), 4});
    return -1;
}
