// paged_tiles.hip — attention over the paged cache: chunks of more than 64 rows a K/V head.
#include "paged_attention.h"

namespace {

// ---------------------------------------------------------------- many rows: tiles of rows and keys
//
// A workgroup takes 128 rows of a K/V head, 32 a wavefront, and goes over the keys in tiles of KT, double
// buffered in LDS; S^T = K·Q^T and O^T = V^T·P^T as above, on 32×32×16 MFMAs.  K lies in LDS by chunks of eight columns,
// [chunk][key], keys swizzled by the chunk, so that the reads (32 keys of a chunk) and the writes (16 chunks of a
// key) both touch every bank once; V lies as in the cache, [group of 8 keys][column].  One-byte values are widened once on
// their way into LDS, for all four wavefronts.  While a tile is computed the next one's loads are in
// flight.  A wavefront's 64 MFMAs a tile (head_dim 128, exact types) take 2048 cycles and the softmax of its 32 values
// a lane about 1400 of the other unit's: two wavefronts a SIMD overlap the two.
//
// A small grid is multiplied by ranges of the keys (blockIdx.y), which paged_tiles_merge joins.

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
    return sp.keys == 0 || first >= sp.count ? 0 : min(sp.start + min(last, sp.count - 1) + 1, sp.keys);
}

// (K/V head of a sequence, row tile) of a workgroup: the tiles with the most keys first, and with eight or a
// multiple of eight heads all tiles of a head on one XCD, whose L2 then holds its keys for them.
__device__ __forceinline__ void tile_of(int id, int tiles, int heads, int& bh, int& tile) {
    if (heads % 8 == 0) {
        const int at = id >> 3;
        bh = at / tiles * 8 + (id & 7);
        tile = tiles - 1 - at % tiles;
    } else {
        bh = id / tiles;
        tile = tiles - 1 - id % tiles;
    }
}

template <int TYPE, int HD>
__global__ __launch_bounds__(256, HD > 128 ? 1 : 2) void paged_tiles(PagedAttn a, int tiles) {
    constexpr int ES = cache_elem(TYPE);
    constexpr int PL = TYPE == LBR_CACHE_F32 ? 2 : 1;
    constexpr int KT = PL == 2 ? 32 : 64;       // keys a tile
    constexpr int NB = KT / 32;                 // blocks of 32 keys
    constexpr int NK = HD / 16, ND = HD / 32;
    constexpr int PLANE = KT * HD;              // halves of a plane of K or V
    constexpr int NL = KT * HD * ES / 16 / 256; // 16-byte loads a thread, of K and of V
    static_assert(NL >= 1 && NL * 256 * 16 == KT * HD * ES, "a tile splits evenly over the threads");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    // [2 buffers][K planes, V planes, ks, vs], then the tiles' largest V scales
    constexpr int BUF = 2 * PL * PLANE * 2 + 2 * KT * 4;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, hf = lane >> 5;
    const PagedCache& c = a.c;
    const int mask = (1 << c.shift) - 1;
    int bh, tile;
    tile_of(blockIdx.x, tiles, a.B * c.heads, bh, tile);
    const int b = bh / c.heads, h = bh % c.heads;
    const Span sp = span_of(a, b);
    const int keys = tile_keys(a, sp, tile);
    const int all = (keys + KT - 1) / KT;                       // tiles of keys
    const int splits = gridDim.y, split = blockIdx.y;
    const int t0 = (int)((long long)all * split / splits), t1 = (int)((long long)all * (split + 1) / splits);

    // this lane's row
    const int row = tile * ROWS_WG + wave * 32 + n;
    const int rc = min(row, a.rows - 1);
    const int token = (int)lbr_fdiv((unsigned)rc, a.G_m, a.G_s), g = rc - token * a.G;
    const long long qat = ((long long)(b * a.H + h * a.G + g) * a.S + token) * c.hd;
    const bool mine = row < a.rows && token < sp.count;
    const int last = mine ? sp.start + token : -1;             // its last key
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

    // a thread's 16-byte loads of a tile: K row and columns, V group and columns; each lies in one block of 16
    // positions, the same for the whole wavefront, and so in one page
    uint4 kr[NL], vr[NL];
    float ksr = 0.f, vsr = 0.f;
    constexpr int KU = HD * ES / 16, VU = HD * ES / 2;   // 16-byte units of a K row, of a V group
    int base_key = 0;
    auto head_of = [&](int key, bool& bad) {   // key wave-uniform, below the end
        const int page = c.table[(long long)b * c.wide + (key >> c.shift)];
        bad = page < 0 || page >= c.pages;
        return c.base + (bad ? 0 : page) * c.page_bytes + (long long)h * c.head_bytes;
    };
    auto load = [&](int t) {
        base_key = t * KT;
#pragma unroll
        for (int u = 0; u < NL; ++u) {
            const int unit = u * 256 + tid;
            {
                const int r = unit / KU, col = unit % KU * (16 / ES);
                const int blk = __builtin_amdgcn_readfirstlane(r >> 4);
                const int key0 = min(base_key + blk * 16, (keys - 1) & ~15);
                bool bad;
                const char* const hd = head_of(key0, bad);
                kr[u] = *(const uint4*)(hd + ((long long)(key0 & mask) + (r & 15)) * c.hdp * ES + (col < c.hdp ? col : 0) * ES);
            }
            {
                const int gr = unit / VU, at = unit % VU * 16;   // byte of the group's [column][8]
                const int blk = __builtin_amdgcn_readfirstlane(gr >> 1);
                const int key0 = min(base_key + blk * 16, (keys - 1) & ~15);
                bool bad;
                const char* const hd = head_of(key0, bad);
                const char* const p = hd + c.part + ((long long)(key0 & mask) + (gr & 1) * 8) * c.hdp * ES;
                uint4 v = *(const uint4*)(p + (at < c.hdp * 8 * ES ? at : 0));
                // positions behind the end, and pages that are none, hold anything
                const int keep = bad ? 0 : keys - (base_key + gr * 8);
                if (bad || base_key + KT > keys) {
                    if (ES == 4) {
                        const int k0 = at / 4 % 8;
                        if (k0 >= keep) v.x = 0;
                        if (k0 + 1 >= keep) v.y = 0;
                        if (k0 + 2 >= keep) v.z = 0;
                        if (k0 + 3 >= keep) v.w = 0;
                    } else if (ES == 2) {
                        if (keep < 1) v.x = 0; else if (keep < 2) v.x &= 0xffffu;
                        if (keep < 3) v.y = 0; else if (keep < 4) v.y &= 0xffffu;
                        if (keep < 5) v.z = 0; else if (keep < 6) v.z &= 0xffffu;
                        if (keep < 7) v.w = 0; else if (keep < 8) v.w &= 0xffffu;
                    } else {
                        const unsigned lo = keep >= 4 ? ~0u : keep <= 0 ? 0u : (1u << (8 * keep)) - 1u;
                        const unsigned hi = keep >= 8 ? ~0u : keep <= 4 ? 0u : (1u << (8 * (keep - 4))) - 1u;
                        v.x &= lo;
                        v.y &= hi;
                        v.z &= lo;
                        v.w &= hi;
                    }
                }
                vr[u] = v;
            }
        }
        if (tid < KT) {   // the scales
            const int key = base_key + tid, k1 = min(key, keys - 1);
            const int page = c.table[(long long)b * c.wide + (k1 >> c.shift)];
            const bool bad = page < 0 || page >= c.pages;
            const float* const sc = (const float*)(c.base + (bad ? 0 : page) * c.page_bytes + (long long)h * c.head_bytes + 2 * c.part);
            ksr = bad ? __uint_as_float(0x7fc00000u) : sc[k1 & mask];
            vsr = key >= keys ? 0.f : bad ? __uint_as_float(0x7fc00000u) : sc[mask + 1 + (k1 & mask)];
        }
    };
    float* const tops = (float*)(lds + 2 * BUF);
    auto store = [&](int buf) {
        _Float16* const kp = (_Float16*)(lds + buf * BUF);
        _Float16* const vp = kp + PL * PLANE;
        float* const ks = (float*)(lds + buf * BUF + 2 * PL * PLANE * 2);
#pragma unroll
        for (int u = 0; u < NL; ++u) {
            const int unit = u * 256 + tid;
            const int r = unit / KU;
            auto slot = [&](int ch) { return (ch * KT + (r ^ (ch & 15))) * 8; };
            if constexpr (TYPE == LBR_CACHE_F32) {
                const int ch = unit % KU / 2, part = unit % 2 * 4;   // four of the eight columns
                const int vat = unit * 4;                            // [group][column][8], four of the eight keys
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
                *(halfx4*)(kp + slot(ch) + part) = hk;
                *(halfx4*)(kp + PLANE + slot(ch) + part) = lk;
                *(halfx4*)(vp + vat) = hv;
                *(halfx4*)(vp + PLANE + vat) = lv;
            } else if constexpr (TYPE == LBR_CACHE_F16) {
                *(halfx8*)(kp + slot(unit % KU)) = __builtin_bit_cast(halfx8, kr[u]);
                *(halfx8*)(vp + unit * 8) = __builtin_bit_cast(halfx8, vr[u]);
            } else {
                const int ch = unit % KU * 2;
                *(halfx8*)(kp + slot(ch)) = widen8<TYPE>(kr[u].x, kr[u].y);
                *(halfx8*)(kp + slot(ch + 1)) = widen8<TYPE>(kr[u].z, kr[u].w);
                *(halfx8*)(vp + unit * 16) = widen8<TYPE>(vr[u].x, vr[u].y);
                *(halfx8*)(vp + unit * 16 + 8) = widen8<TYPE>(vr[u].z, vr[u].w);
            }
        }
        if (tid < KT) {
            ks[tid] = __builtin_amdgcn_ldexpf(ksr, -KS_UP);
            ks[KT + tid] = vsr;
            float top = fmaxf(vsr, 0.f);
            for (int o = KT / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, KT));
            if (tid == 0) tops[buf] = top;
        }
    };

    floatx16 o[ND];
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[j][i] = 0.f;
    float m = -INFINITY, l = 0.f;
    int vup = VUP_MOST;   // biased exponent of the power of two that weights are taken by (see the sums below)

    if (t0 < t1) {
        load(t0);
        store(0);
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1;
        if (t + 1 < t1) load(t + 1);
        const int k0 = t * KT;
        if (k0 <= wave_last) {
            const _Float16* const kp = (const _Float16*)(lds + buf * BUF);
            const _Float16* const vp = kp + PL * PLANE;
            const float* const ks = (const float*)(lds + buf * BUF + 2 * PL * PLANE * 2);
            const float* const vs = ks + KT;
            floatx16 s[NB];
            // block row m of the MFMA is key (m / 16)·16 + (m / 4 % 2)·8 + (m / 8 % 2)·4 + m % 4
            const int kk = (n >> 4) * 16 + (n >> 2 & 1) * 8 + (n >> 3 & 1) * 4 + (n & 3);
#pragma unroll
            for (int q = 0; q < NB; ++q) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[q][i] = 0.f;
#pragma unroll
                for (int j = 0; j < NK; ++j) {
                    const int ch = 2 * j + hf;
                    const int at = (ch * KT + ((q * 32 + kk) ^ (ch & 15))) * 8;
                    const halfx8 kh = *(const halfx8*)(kp + at);
                    s[q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, ql[j], s[q], 0, 0, 0);
                    if constexpr (PL == 2) {
                        const halfx8 kl = *(const halfx8*)(kp + PLANE + at);
                        s[q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, qh[j], s[q], 0, 0, 0);
                    }
                    s[q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qh[j], s[q], 0, 0, 0);
                }
            }
            // scores (over qs), the row's maximum; accumulator i of block q is key 32·q + (i / 8)·16 + 8·hf + i % 8
            float top = -INFINITY;
            const bool edge = k0 + KT - 1 > sp.start || k0 + KT > keys;   // some row ends in this tile
#pragma unroll
            for (int q = 0; q < NB; ++q)
#pragma unroll
                for (int i8 = 0; i8 < 16; i8 += 4) {
                    const int key = 32 * q + (i8 >> 3) * 16 + 8 * hf + (i8 & 7);
                    const floatx4 sc = *(const floatx4*)(ks + key);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v = s[q][i8 + e] * sc[e];
                        if (edge && k0 + key + e > last) v = -INFINITY;
                        s[q][i8 + e] = v;
                        top = fmaxf(top, v);
                    }
                }
            {
                const unsigned u = __float_as_uint(top);
                auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
                top = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * qs;
            }
            // Weights are taken times 2^(vup − 127), which brings the largest V scale so far to [2^14, 2^15): their
            // products with the scales then fit fp16, and the sums carry the same factor.
            const int vnew = __builtin_amdgcn_readfirstlane(min(vup, min(up_exponent(__float_as_uint(tops[buf])), VUP_MOST)));
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
                        if (edge && v == -INFINITY) p[i4 + e] = 0.f;   // no weight, whatever the V row holds
                    }
                }
                split8(p, ph[q], pl[q]);
            }
            l = l * f + sum;
            if (__any(f != 1.f)) {
#pragma unroll
                for (int j = 0; j < ND; ++j)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[j][i] *= f;
            }
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
        }
        if (t + 1 < t1) store(buf ^ 1);
        __syncthreads();
    }

    {
        const unsigned u = __float_as_uint(l);
        auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const bool whole = splits == 1;
    float* const part = a.parts + ((long long)split * gridDim.x + blockIdx.x) * tile_floats<HD>();
    if (!whole && hf == 0) {
        part[ROWS_WG * HD + wave * 32 + n] = m;
        part[ROWS_WG * HD + ROWS_WG + wave * 32 + n] = __builtin_amdgcn_ldexpf(l, 127 - vup);
    }
    if (whole && row >= a.rows) return;
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

// Joins the ranges of the keys: one workgroup eight rows of a workgroup of paged_tiles.
template <int HD>
__global__ __launch_bounds__(256) void paged_tiles_merge(PagedAttn a, int tiles, int splits) {
    constexpr int LANES = HD / 4, EACH = 256 / LANES;
    const PagedCache& c = a.c;
    int bh, tile;
    tile_of(blockIdx.x, tiles, a.B * c.heads, bh, tile);
    const int b = bh / c.heads, h = bh % c.heads;
    const int r = blockIdx.y * EACH + threadIdx.x / LANES, row = tile * ROWS_WG + r, col = threadIdx.x % LANES * 4;
    if (row >= a.rows) return;
    float m = -INFINITY, l = 0.f;
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < splits; ++k) {
        const float* const part = a.parts + ((long long)k * gridDim.x + blockIdx.x) * tile_floats<HD>();
        const float pm = part[ROWS_WG * HD + r], pl = part[ROWS_WG * HD + ROWS_WG + r];
        const floatx4 v = *(const floatx4*)(part + r * HD + col);
        const float mx = fmaxf(m, pm), base = mx == -INFINITY ? 0.f : mx;
        const float f = __builtin_amdgcn_exp2f(m - base), g = __builtin_amdgcn_exp2f(pm - base) * pl;
        o = o * f + v * g;
        l = l * f + g;
        m = mx;
    }
    const float inv = 1.f / l;
    const Span sp = span_of(a, b);
    const int token = (int)lbr_fdiv((unsigned)row, a.G_m, a.G_s), g = row - token * a.G;
    float* const to = a.out + ((long long)(b * a.H + h * a.G + g) * a.S + token) * c.hd;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (col + e < c.hd) to[col + e] = row_value(a, sp, token, o[e] * inv);
}

template <int TYPE, int HD>
constexpr size_t tiles_lds() {
    constexpr int pl = TYPE == LBR_CACHE_F32 ? 2 : 1, kt = pl == 2 ? 32 : 64;
    return 2 * (2 * pl * kt * HD * 2 + 2 * kt * 4) + 16;
}

template <int TYPE, int HD>
void launch_tiles(const Step& s, hipStream_t st) {
    const PagedAttn a = attn_args(s);
    const int tiles = paged_row_tiles(s), splits = (int)s.i[10];
    const unsigned wgs = (unsigned)(tiles * s.i[1] * s.i[2]);
    if (!wgs) return;
    const unsigned lds = (unsigned)tiles_lds<TYPE, HD>();
    hipLaunchKernelGGL((paged_tiles<TYPE, HD>), dim3(wgs, (unsigned)splits), dim3(256), lds, st, a, tiles);
    if (splits > 1)
        hipLaunchKernelGGL((paged_tiles_merge<HD>), dim3(wgs, ROWS_WG * (HD / 4) / 256), dim3(256), 0, st, a, tiles, splits);
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

// Enough for two workgroups a CU, none shorter than four tiles of keys at the table's full length.
int paged_tiles_splits(const Step& s) {
    const long long cus = lbr_device_cus() > 0 ? lbr_device_cus() : 256;
    const long long wgs = paged_row_tiles(s) * s.i[1] * s.i[2], keys = s.i[6] << s.i[4];
    const long long want = wgs > 0 ? 2 * cus / wgs : 1, most = keys / (4 * (s.i[0] == LBR_CACHE_F32 ? 32 : 64));
    return (int)(want < most ? (want > 1 ? want : 1) : (most > 1 ? most : 1));
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
