// paged_tiles.hip — attention over the paged cache: chunks of more than 32 rows a K/V head.
#include "paged_attention.h"

#include <algorithm>
#include <type_traits>

namespace {

// ---------------------------------------------------------------- many rows: tiles of rows and keys
//
// A workgroup takes 128 rows of a K/V head, 32 a wavefront, and goes over the keys in tiles of KT, double
// buffered in LDS; S^T = K·Q^T and O^T = V^T·P^T as for few rows, on 32×32×16 MFMAs.  V lies in LDS as in the cache,
// [group of 8 keys][column].  float16 goes straight into LDS; one-byte values are widened, and floats split, once on
// their way there for all four wavefronts.  While a tile is computed the next one's loads are in
// flight.  A wavefront's 64 MFMAs a tile (head_dim 128, exact types) take 2048 cycles and the softmax of its 32 values
// a lane about 1400 of the other unit's: two wavefronts a SIMD overlap the two.
//
// The matrix cores bound it, at the clock that they leave under load (about 1.8 GHz).  2048 tokens behind 2048, 32 heads
// of 128, float16: 250 µs, 412 TFLOP/s of the formula's two products, each run twice for the halves of q and
// of the weights: 824 on the matrix cores, 75 % of what a large fp16 product of matrices reaches here.  1024
// behind 1024, 32 heads over 8, int8: 94 µs, of which the merge takes 10.
//
// A small grid is multiplied by ranges of the keys, which paged_tiles_merge joins.

constexpr int ROWS_WG = 128;
constexpr int KS_UP = 40;           // K scales are held this many powers of two lower, q's higher
constexpr int VUP_MOST = 127 + 100;   // weights times at most 2^100: their sums stay finite

// Floats of a workgroup's partial result: rows of outputs, each row's maximum and sum.
template <int HD>
constexpr int tile_floats() { return ROWS_WG * (HD + 2); }

// The row tile's keys: those its last row reaches.
__device__ __forceinline__ int tile_keys(const PagedAttn& a, const Span& sp, int tile) {
    const int first = (int)lbr_fdiv((unsigned)(tile * ROWS_WG), a.G_m, a.G_s);
    const int last = (int)lbr_fdiv((unsigned)min(tile * ROWS_WG + ROWS_WG, a.rows) - 1u, a.G_m, a.G_s);
    return sp.keys == 0 || first >= sp.count ? 0 : last_key(sp, min(last, sp.count - 1)) + 1;
}

// (K/V head of a sequence, row tile, range of its keys) of a workgroup: the tiles with the most keys first; with a
// multiple of eight heads all tiles of a head on one XCD, whose L2 then holds its keys for them.  `fold`: all
// workgroups are there at once, two a CU; the second half then goes from the fewest keys up, beside the first's most.
__device__ __forceinline__ void tile_of(int id, int tiles, int heads, int splits, bool fold, int& bh, int& tile, int& split) {
    const int lanes = heads % 8 == 0 ? 8 : 1, own = heads / lanes, all = own * tiles * splits;
    int at = id / lanes;
    if (fold && at >= (all + 1) / 2) at = all - 1 - (at - (all + 1) / 2);
    bh = at % own * lanes + id % lanes;
    split = at / own % splits;
    tile = tiles - 1 - at / own / splits;
}

// K rows lie in LDS as chunks of eight columns, chunk ch of key k at place ch ^ swizzle(k): 16 keys' reads of a
// chunk then lie in 16 different places of the 256 bytes that all banks make.
template <int CH>
__device__ __forceinline__ int swizzle(int key) { return CH == 8 ? key >> 1 & 7 : key & 15; }

// max over each row of 16 lanes.
__device__ __forceinline__ float max16(float v) {
    v = fmaxf(v, lbr_dpp<0x128>(v));   // rotated by 8, 4, 2, 1
    v = fmaxf(v, lbr_dpp<0x124>(v));
    v = fmaxf(v, lbr_dpp<0x122>(v));
    return fmaxf(v, lbr_dpp<0x121>(v));
}

template <int TYPE, int HD>
__global__ __launch_bounds__(256, HD > 128 ? 1 : 2) void paged_tiles(PagedAttn a, int tiles, int splits, bool fold) {
    constexpr int ES = cache_elem(TYPE);
    constexpr int PL = TYPE == LBR_CACHE_F32 ? 2 : 1;
    constexpr int KT = PL == 2 ? 32 : 64;       // keys a tile
    constexpr int BK = KT / 4;                  // of a wavefront's loads
    constexpr int NB = KT / 32;                 // blocks of 32 keys
    constexpr int NK = HD / 16, ND = HD / 32;
    constexpr int CH = HD / 8;                  // chunks of eight columns
    constexpr int PLANE = KT * HD;              // halves of a plane of K or V
    constexpr bool DMA = TYPE == LBR_CACHE_F16; // straight into LDS
    constexpr int KU = HD * ES / 16, VU = HD * ES / 2;   // 16-byte units of a K row, of a V group
    constexpr int NL = BK * KU / 64;            // 16-byte loads a thread, of K and of V
    static_assert(NL >= 1 && NL * 64 == BK * KU && BK * KU == BK / 8 * VU, "a wavefront's keys split evenly over its lanes");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    // [2 buffers][K planes, V planes, ks, vs], then the tiles' largest V scales
    constexpr int BUF = 2 * PL * PLANE * 2 + 2 * KT * 4;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, hf = lane >> 5;
    const PagedCache& c = a.c;
    const int mask = (1 << c.shift) - 1;
    int bh, tile, split;
    tile_of(blockIdx.x, tiles, a.B * c.heads, splits, fold, bh, tile, split);
    const int b = bh / c.heads, h = bh % c.heads;
    const Span sp = span_of(a, b);
    const int keys = tile_keys(a, sp, tile);
    const int all = (keys + KT - 1) / KT;                       // tiles of keys
    const int t0 = (int)((long long)all * split / splits), t1 = (int)((long long)all * (split + 1) / splits);

    // this lane's row
    const int row = tile * ROWS_WG + wave * 32 + n;
    const int rc = min(row, a.rows - 1);
    const int token = (int)lbr_fdiv((unsigned)rc, a.G_m, a.G_s), g = rc - token * a.G;
    const long long qat = ((long long)(b * a.H + h * a.G + g) * a.S + token) * c.hd;
    const bool mine = row < a.rows && token < sp.count;
    const int last = mine ? last_key(sp, token) : -1;          // its last key
    int wave_last = last;
    for (int o = 16; o; o >>= 1) wave_last = max(wave_last, __shfl_xor(wave_last, o, 64));
    wave_last = __builtin_amdgcn_readfirstlane(wave_last);   // the halves hold the same rows

    halfx8 qh[NK], ql[NK];
    float qs;
    {
        unsigned top = 0;
        float v[NK][8];
#pragma unroll
        for (int j = 0; j < NK; ++j) {
            const int col = j * 16 + hf * 8;
#pragma unroll
            for (int k = 0; k < 8; ++k) v[j][k] = 0.f;
            if (mine) {
                if (a.vec && col + 8 <= c.hd) {
                    const float4 u0 = *(const float4*)(a.q + qat + col), u1 = *(const float4*)(a.q + qat + col + 4);
                    v[j][0] = u0.x; v[j][1] = u0.y; v[j][2] = u0.z; v[j][3] = u0.w;
                    v[j][4] = u1.x; v[j][5] = u1.y; v[j][6] = u1.z; v[j][7] = u1.w;
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (col + k < c.hd) v[j][k] = a.q[qat + col + k];
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[j][k] *= a.scale;
                top = max(top, __float_as_uint(v[j][k]) & 0x7fffffffu);
            }
        }
        auto sw = __builtin_amdgcn_permlane32_swap(top, top, false, false);
        top = max((unsigned)sw[0], (unsigned)sw[1]);
        const int up = up_exponent(top);
        const float by = __uint_as_float((unsigned)up << 23);
        // KS_UP: the scales of K rows are held 2^40 lower, so that a sum of products times one stays finite
        qs = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __builtin_amdgcn_ldexpf(1.f, 127 - up + KS_UP);
#pragma unroll
        for (int j = 0; j < NK; ++j) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[j][k] *= by;
            split8(v[j], qh[j], ql[j]);
        }
    }

    // Loads of a tile.  A wavefront takes BK keys, which share a block of 16 positions and so a page: K rows and V
    // groups in 16-byte units, past the page's range (which reads as zero) for columns that the rows do not have,
    // groups behind the end and pages that are none.
    typedef const __attribute__((address_space(4))) int* Table;
    const Table table = (Table)(c.table + (long long)b * c.wide);
    const int own = wave * BK;                            // the wavefront's first key in a tile
    auto page_of = [&](int t) { return table[min(t * KT + own, keys - 1) >> c.shift]; };
    constexpr unsigned NONE = 0x7ffffff0u;
    unsigned koff[NL], voff[NL];
    int kdst[NL];                                         // halves, in the K plane
#pragma unroll
    for (int u = 0; u < NL; ++u) {
        const int unit = u * 64 + lane;
        if constexpr (DMA) {   // LDS is filled in order: lane l's unit is the one that belongs there
            const int r = unit / CH, ch = unit % CH ^ swizzle<CH>(own + r);
            koff[u] = ch * 8 < c.hdp ? (unsigned)(r * c.hdp + ch * 8) * ES : NONE;
        } else {
            const int r = unit / KU, col = unit % KU * (16 / ES);
            koff[u] = col < c.hdp ? (unsigned)(r * c.hdp + col) * ES : NONE;
            kdst[u] = (own + r) * HD + ((col / 8) ^ swizzle<CH>(own + r)) * 8 + col % 8;
        }
        const int gr = unit / VU, at = unit % VU * 16;
        voff[u] = at < c.hdp * 8 * ES ? (unsigned)(c.part + gr * 8 * c.hdp * ES + at) : NONE;
    }
    uint4 kr[NL], vr[NL];
    float scale_r = 0.f;
    bool bad_r = false;
    float* const tops = (float*)(lds + 2 * BUF);          // [2][4]: the largest V scale of each wavefront's keys
    auto load = [&](int t, int page, int buf) {
        const int key0 = t * KT + own;
        const bool bad = page < 0 || page >= c.pages;
        const char* const hd = c.base + (bad ? 0 : page) * c.page_bytes + (long long)h * c.head_bytes;
        const int slot = min(key0, keys - 1) & mask & ~(BK - 1);
        const bool none = bad || key0 >= keys;
        const __amdgpu_buffer_rsrc_t rs =
            __builtin_amdgcn_make_buffer_rsrc((void*)hd, (short)0, none ? 0 : c.head_bytes, 0x00020000);
        const unsigned soff = (unsigned)(slot * c.hdp * ES);
        if constexpr (DMA) {
            _Float16* const kp = (_Float16*)(lds + buf * BUF) + own * HD;
            _Float16* const vp = (_Float16*)(lds + buf * BUF) + PLANE + own * HD;
#pragma unroll
            for (int u = 0; u < NL; ++u) {
                lbr_dma16(rs, (float*)(kp + u * 512), koff[u], soff);
                const bool there = key0 + (u * 64 + lane) / VU * 8 < keys;
                lbr_dma16(rs, (float*)(vp + u * 512), there ? voff[u] : NONE, soff);
            }
        } else {
#pragma unroll
            for (int u = 0; u < NL; ++u) {
                kr[u] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rs, koff[u], soff, 0));
                const bool there = key0 + (u * 64 + lane) / VU * 8 < keys;
                vr[u] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rs, there ? voff[u] : NONE, soff, 0));
            }
        }
        // scales: lanes 0 .. BK−1 of K rows, BK .. 2·BK−1 of V rows; zero behind the end.  Whatever used the value
        // here would wait for all of the tile's loads.
        const int k = key0 + (lane & (BK - 1));
        const unsigned at = (unsigned)(2 * c.part) + 4u * ((lane & BK ? mask + 1 : 0) + (k & mask));
        scale_r = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, k < keys ? at : NONE, 0, 0));
        bad_r = bad;
    };
    auto store = [&](int t, int buf) {
        _Float16* const kp = (_Float16*)(lds + buf * BUF);
        _Float16* const vp = kp + PL * PLANE;
        const int key0 = t * KT + own;
        if constexpr (!DMA) {
            // the end lies inside a group: what is behind it may be anything
            if (key0 < keys && key0 + BK > keys && (keys & 7)) {
#pragma unroll
                for (int u = 0; u < NL; ++u) {
                    const int keep = keys - (key0 + (u * 64 + lane) / VU * 8);
                    if (ES == 4) {
                        const int k0 = lane % 2 * 4;   // four of a column's eight keys
                        if (k0 >= keep) vr[u].x = 0;
                        if (k0 + 1 >= keep) vr[u].y = 0;
                        if (k0 + 2 >= keep) vr[u].z = 0;
                        if (k0 + 3 >= keep) vr[u].w = 0;
                    } else {
                        const unsigned lo = keep >= 4 ? ~0u : keep <= 0 ? 0u : (1u << (8 * keep)) - 1u;
                        const unsigned hi = keep >= 8 ? ~0u : keep <= 4 ? 0u : (1u << (8 * (keep - 4))) - 1u;
                        vr[u].x &= lo;
                        vr[u].y &= hi;
                        vr[u].z &= lo;
                        vr[u].w &= hi;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < NL; ++u) {
                _Float16* const vd = vp + own * HD + (u * 64 + lane) * (16 / ES);
                if constexpr (TYPE == LBR_CACHE_F32) {
                    const float fk[4] = {__uint_as_float(kr[u].x), __uint_as_float(kr[u].y), __uint_as_float(kr[u].z), __uint_as_float(kr[u].w)};
                    const float fv[4] = {__uint_as_float(vr[u].x), __uint_as_float(vr[u].y), __uint_as_float(vr[u].z), __uint_as_float(vr[u].w)};
                    halfx4 hk, lk, hv, lv;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        hk[e] = (_Float16)fk[e];
                        lk[e] = (_Float16)(fk[e] - (float)hk[e]);
                        hv[e] = (_Float16)fv[e];
                        lv[e] = (_Float16)(fv[e] - (float)hv[e]);
                    }
                    *(halfx4*)(kp + kdst[u]) = hk;
                    *(halfx4*)(kp + PLANE + kdst[u]) = lk;
                    *(halfx4*)vd = hv;
                    *(halfx4*)(vd + PLANE) = lv;
                } else if constexpr (ES == 1) {
                    *(halfx8*)(kp + kdst[u]) = widen8<TYPE>(kr[u].x, kr[u].y);
                    *(halfx8*)(kp + (kdst[u] ^ 8)) = widen8<TYPE>(kr[u].z, kr[u].w);   // the next chunk
                    *(halfx8*)vd = widen8<TYPE>(vr[u].x, vr[u].y);
                    *(halfx8*)(vd + 8) = widen8<TYPE>(vr[u].z, vr[u].w);
                }
            }
        }
        float* const sc = (float*)(lds + buf * BUF + 2 * PL * PLANE * 2);
        if (bad_r && key0 + (lane & (BK - 1)) < keys) scale_r = __uint_as_float(0x7fc00000u);
        if (lane < BK) sc[own + lane] = __builtin_amdgcn_ldexpf(scale_r, -KS_UP);
        else if (lane < 2 * BK) sc[KT + own + lane - BK] = scale_r;
        const float top = max16(lane & BK ? fmaxf(scale_r, 0.f) : 0.f);   // lanes 0 .. 2·BK − 1 are one or two rows
        if (lane == BK) tops[buf * 4 + wave] = top;
    };

    floatx16 o[ND];
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[j][i] = 0.f;
    float m = -INFINITY, l = 0.f;
    int vup = VUP_MOST;   // biased exponent of the power of two that weights are taken by (see the sums below)

    // block row m of the MFMA is key (m / 16)·16 + (m / 4 % 2)·8 + (m / 8 % 2)·4 + m % 4 of its 32
    const int kk = (n >> 4) * 16 + (n >> 2 & 1) * 8 + (n >> 3 & 1) * 4 + (n & 3);
    // EDGE: some row of the workgroup ends in the tile
    auto compute = [&](int t, int buf, auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
        const int k0 = t * KT;
        const _Float16* const kp = (const _Float16*)(lds + buf * BUF);
        const _Float16* const vp = kp + PL * PLANE;
        const float* const ks = (const float*)(lds + buf * BUF + 2 * PL * PLANE * 2);
        const float* const vs = ks + KT;
        floatx16 s[NB];
#pragma unroll
        for (int q = 0; q < NB; ++q) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[q][i] = 0.f;
#pragma unroll
            for (int j = 0; j < NK; ++j) {
                const int at = (q * 32 + kk) * HD + ((2 * j + hf) ^ swizzle<CH>(kk)) * 8;   // the swizzle has period 16
                const halfx8 kh = *(const halfx8*)(kp + at);
                s[q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, ql[j], s[q], 0, 0, 0);
                if constexpr (PL == 2) {
                    const halfx8 kl = *(const halfx8*)(kp + PLANE + at);
                    s[q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, qh[j], s[q], 0, 0, 0);
                }
                s[q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qh[j], s[q], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);   // or reads hoisted over the phases spill
        // scores (over qs), the row's maximum; accumulator i of block q is key 32·q + (i / 8)·16 + 8·hf + i % 8
        float top = -INFINITY;
#pragma unroll
        for (int q = 0; q < NB; ++q)
#pragma unroll
            for (int i8 = 0; i8 < 16; i8 += 4) {
                const int key = 32 * q + (i8 >> 3) * 16 + 8 * hf + (i8 & 7);
                const floatx4 sc = *(const floatx4*)(ks + key);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = s[q][i8 + e] * sc[e];
                    if (EDGE && k0 + key + e > last) v = -INFINITY;
                    s[q][i8 + e] = v;
                    top = fmaxf(top, v);
                }
            }
        {
            const unsigned u = __float_as_uint(top);
            auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
            top = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * qs;
        }
        __builtin_amdgcn_sched_barrier(0);
        // Weights are taken times 2^(vup − 127), which brings the largest V scale so far to [2^14, 2^15): their
        // products with the scales then fit fp16, and the sums carry the same factor.
        const floatx4 vt = *(const floatx4*)(tops + buf * 4);
        const float vtop = fmaxf(fmaxf(vt[0], vt[1]), fmaxf(vt[2], vt[3]));
        const int vnew = __builtin_amdgcn_readfirstlane(min(vup, min(up_exponent(__float_as_uint(vtop)), VUP_MOST)));
        const float mx = fmaxf(m, top);
        const float base = mx == -INFINITY ? 0.f : mx;
        const float f = __builtin_amdgcn_exp2f(m - base + (float)(vnew - vup));
        const float sub = base - (float)(vnew - 127);
        m = mx;
        vup = vnew;
        float sum = 0.f;
        halfx8 ph[2 * NB], pl[2 * NB];
#pragma unroll
        for (int q = 0; q < 2 * NB; ++q) {
            float p[8];
#pragma unroll
            for (int i4 = 0; i4 < 8; i4 += 4) {
                const floatx4 sc = *(const floatx4*)(vs + 16 * q + 8 * hf + i4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = s[q >> 1][(q & 1) * 8 + i4 + e];
                    const float w = __builtin_amdgcn_exp2f(fmaf(v, qs, -sub));
                    sum += w;
                    p[i4 + e] = w * sc[e];
                    if (EDGE && v == -INFINITY) p[i4 + e] = 0.f;   // no weight, whatever the V row holds
                }
            }
            split8(p, ph[q], pl[q]);
        }
        l = l * f + sum;
        if (__any(f != 1.f)) {
            asm volatile("");   // a branch: done ahead of it, the products would need registers of their own
#pragma unroll
            for (int j = 0; j < ND; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[j][i] *= f;
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
            for (int q = 0; q < 2 * NB; ++q) {
                const int at = ((2 * q + hf) * HD + 32 * j + n) * 8;
                const halfx8 vh = *(const halfx8*)(vp + at);
                o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, pl[q], o[j], 0, 0, 0);
                if constexpr (PL == 2) {
                    const halfx8 vl = *(const halfx8*)(vp + PLANE + at);
                    o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, ph[q], o[j], 0, 0, 0);
                }
                o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, ph[q], o[j], 0, 0, 0);
            }
    };

    int page = 0;
    if (t0 < t1) {
        load(t0, page_of(t0), 0);
        if (t0 + 1 < t1) page = page_of(t0 + 1);
        store(t0, 0);
    }
    if (DMA) __builtin_amdgcn_s_waitcnt(lbr_waitcnt_vm(0));
    __syncthreads();
    auto step = [&](int t, auto edge) {
        const int buf = (t - t0) & 1;
        if (DMA && decltype(edge)::value && t * KT + KT > keys && (keys & 7)) {
            // the end lies inside a group of V: what is behind it may be anything
            _Float16* const vp = (_Float16*)(lds + buf * BUF) + PLANE + (keys - t * KT) / 8 * 8 * HD;
            for (int at = tid; at < HD * 8; at += 256)
                if (at % 8 >= (keys & 7)) vp[at] = (_Float16)0.f;
            __syncthreads();
        }
        if (t + 1 < t1) load(t + 1, page, buf ^ 1);
        if (t + 2 < t1) page = page_of(t + 2);
        if (t * KT <= wave_last) compute(t, buf, edge);
        if (t + 1 < t1) store(t + 1, buf ^ 1);
        if (DMA) __builtin_amdgcn_s_waitcnt(lbr_waitcnt_vm(0));
        __syncthreads();
    };
    // tiles that all rows of the workgroup reach to their end, then the others
    const int te = min(t1, max(t0, (min(sp.start, keys - 1) + 1) / KT));
    for (int t = t0; t < te; ++t) step(t, std::false_type());
    for (int t = te; t < t1; ++t) step(t, std::true_type());

    {
        const unsigned u = __float_as_uint(l);
        auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const bool whole = splits == 1;
    float* const part = a.parts + ((long long)(bh * tiles + tile) * splits + split) * tile_floats<HD>();
    if (!whole && hf == 0) {
        part[ROWS_WG * HD + wave * 32 + n] = m;
        part[ROWS_WG * HD + ROWS_WG + wave * 32 + n] = __builtin_amdgcn_ldexpf(l, 127 - vup);
    }
    if (row >= a.rows) return;
    float* const to = whole ? a.out + qat : part + (wave * 32 + n) * HD;
    const int cols = whole ? c.hd : HD;
    const bool vec = !whole || a.vec;
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int col = 32 * j + 2 * i + 4 * hf;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = whole ? row_value(a, sp, token, o[j][i + e] * inv) : o[j][i + e] * inv;
            if (vec && col + 4 <= cols) {
                *(float4*)(to + col) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (col + e < cols) to[col + e] = v[e];
            }
        }
}

// Joins the ranges of the keys: one workgroup eight rows of a workgroup of paged_tiles.  AHEAD: ranges whose loads
// are in flight at once.
template <int HD, int AHEAD>
__global__ __launch_bounds__(256) void paged_tiles_merge(PagedAttn a, int tiles, int splits) {
    constexpr int LANES = HD / 4, EACH = 256 / LANES;
    const PagedCache& c = a.c;
    const int bh = blockIdx.x / tiles, tile = blockIdx.x % tiles;
    const int b = bh / c.heads, h = bh % c.heads;
    const int r = blockIdx.y * EACH + threadIdx.x / LANES, row = tile * ROWS_WG + r, col = threadIdx.x % LANES * 4;
    if (row >= a.rows) return;
    float m = -INFINITY, l = 0.f;
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < splits; k0 += AHEAD) {
        float pm[AHEAD], ps[AHEAD];
        floatx4 v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const float* const part = a.parts + ((long long)blockIdx.x * splits + min(k0 + k, splits - 1)) * tile_floats<HD>();
            pm[k] = part[ROWS_WG * HD + r];
            ps[k] = part[ROWS_WG * HD + ROWS_WG + r];
            v[k] = *(const floatx4*)(part + r * HD + col);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (k0 + k < splits) merge_part(m, l, o, pm[k], ps[k], v[k]);
    }
    const float inv = 1.f / l;
    const Span sp = span_of(a, b);
    const int token = (int)lbr_fdiv((unsigned)row, a.G_m, a.G_s), g = row - token * a.G;
    float* const to = a.out + ((long long)(b * a.H + h * a.G + g) * a.S + token) * c.hd;
    if (a.vec && col + 4 <= c.hd) {
        float4 v;
        v.x = row_value(a, sp, token, o[0] * inv);
        v.y = row_value(a, sp, token, o[1] * inv);
        v.z = row_value(a, sp, token, o[2] * inv);
        v.w = row_value(a, sp, token, o[3] * inv);
        *(float4*)(to + col) = v;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (col + e < c.hd) to[col + e] = row_value(a, sp, token, o[e] * inv);
}

template <int TYPE, int HD>
constexpr size_t tiles_lds() {
    constexpr int pl = TYPE == LBR_CACHE_F32 ? 2 : 1, kt = pl == 2 ? 32 : 64;
    return 2 * (2 * pl * kt * HD * 2 + 2 * kt * 4) + 32;
}

template <int TYPE, int HD>
void launch_tiles(const Step& s, hipStream_t st) {
    const PagedAttn a = attn_args(s);
    const int tiles = paged_row_tiles(s), splits = (int)s.i[10];
    const unsigned wgs = (unsigned)(tiles * s.i[1] * s.i[2]);
    if (!wgs) return;
    const unsigned lds = (unsigned)tiles_lds<TYPE, HD>();
    const bool fold = wgs * (unsigned)splits <= 2u * (unsigned)lbr_device_cus();
    hipLaunchKernelGGL((paged_tiles<TYPE, HD>), dim3(wgs * (unsigned)splits), dim3(256), lds, st, a, tiles, splits, fold);
    const dim3 joins(wgs, ROWS_WG * (HD / 4) / 256);
    if (splits == 2)
        hipLaunchKernelGGL((paged_tiles_merge<HD, 2>), joins, dim3(256), 0, st, a, tiles, splits);
    else if (splits > 2)
        hipLaunchKernelGGL((paged_tiles_merge<HD, 8>), joins, dim3(256), 0, st, a, tiles, splits);
}

template <int TYPE>
step_fn tiles_for(int hd) {
    return hd <= 64 ? launch_tiles<TYPE, 64> : hd <= 128 ? launch_tiles<TYPE, 128> : launch_tiles<TYPE, 256>;
}

template <int TYPE, int HD>
hipError_t raise_lds() {
    return hipFuncSetAttribute((const void*)paged_tiles<TYPE, HD>, hipFuncAttributeMaxDynamicSharedMemorySize,
                               (int)tiles_lds<TYPE, HD>());
}
template <int TYPE>
hipError_t raise_lds_of() {
    hipError_t e = raise_lds<TYPE, 64>();
    if (e == hipSuccess) e = raise_lds<TYPE, 128>();
    if (e == hipSuccess) e = raise_lds<TYPE, 256>();
    return e;
}

}  // namespace

int paged_row_tiles(const Step& s) { return (int)((s.i[8] / s.i[2] * s.i[7] + ROWS_WG - 1) / ROWS_WG); }

// Ranges of the keys for a small grid: up to two workgroups a CU where each keeps two tiles of keys at the table's full
// length, up to one a CU where each keeps one.  64 tokens behind 1000, 8 heads of 128, float16: 49.9 µs in one range, 23.3
// with four tiles a range, 19.0 with two, 15.1 with one (136 workgroups); 512 tokens, 12 heads of 64: 23.0, 18.4, 16.3 and
// 19.8 (384); 3 × 77 behind 2000, 5 heads of 80, int8: 102, 28.2, 26.6, 30.2 (510), and 24.9 by this rule (255).
int paged_tiles_splits(const Step& s) {
    const long long cus = lbr_device_cus() > 0 ? lbr_device_cus() : 256;
    const long long wgs = paged_row_tiles(s) * s.i[1] * s.i[2], tile = s.i[0] == LBR_CACHE_F32 ? 32 : 64;
    if (wgs <= 0) return 1;
    const long long tiles = (s.i[6] << s.i[4]) / tile;
    const long long two = std::min(2 * cus / wgs, tiles / 2), one = std::min(cus / wgs, tiles);
    return (int)std::max(1LL, std::max(two, one));
}

size_t paged_tiles_workspace(const Step& s) {
    const int wide = s.i[3] <= 64 ? 64 : s.i[3] <= 128 ? 128 : 256;
    if (s.i[10] <= 1) return 0;
    return (size_t)(paged_row_tiles(s) * s.i[1] * s.i[2] * s.i[10] * ROWS_WG * (wide + 2)) * sizeof(float);
}

step_fn paged_tiles_launcher(int type, int hd) {
    return type == LBR_CACHE_F32   ? tiles_for<LBR_CACHE_F32>(hd)
           : type == LBR_CACHE_F16 ? tiles_for<LBR_CACHE_F16>(hd)
           : type == LBR_CACHE_I8  ? tiles_for<LBR_CACHE_I8>(hd)
                                   : tiles_for<LBR_CACHE_E4M3>(hd);
}

hipError_t paged_prepare_device() {
    hipError_t e = raise_lds_of<LBR_CACHE_F32>();
    if (e == hipSuccess) e = raise_lds_of<LBR_CACHE_F16>();
    if (e == hipSuccess) e = raise_lds_of<LBR_CACHE_I8>();
    if (e == hipSuccess) e = raise_lds_of<LBR_CACHE_E4M3>();
    return e;
}
