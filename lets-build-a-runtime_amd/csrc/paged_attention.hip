// paged_attention.hip — attention over the paged cache: few rows a K/V head, and the choice between the kernels.
#include "paged_attention.h"

namespace {

// ---------------------------------------------------------------- few rows: split over the keys
//
// At most 32 rows a K/V head (single tokens, drafted tokens): the cache is read once and bounds the time.  A
// step is 32 keys of one wavefront, 128 of a workgroup; the steps of all (sequence, K/V head) segments lie in
// one line, which the workgroups cut into equal ranges, so that a batch of one long and many short
// sequences fills the chip as an even one does.  A segment inside one range is finished there; one that ranges cut
// leaves a partial result a range, which paged_merge joins.
//
// Operands go from memory to registers in the layout the MFMA takes, without LDS.  S^T = K·Q^T: lane (m, kg) =
// (lane % 16, lane / 16) loads columns of K row m, in the order that makes a load 16 contiguous bytes, and q's columns
// are taken in the same order.  The accumulators of two 16-key blocks then hold, in lane (n, kg), row n's scores
// for four keys of each; with the blocks' rows dealt out as key(t, m) = 8·(m / 4) + 4·t + m % 4 these are the eight keys
// 8·kg .. 8·kg + 7, just what O^T = V^T·P^T takes as its operand from that lane, and V lies in groups of eight positions
// for the same reason.  Weights never leave their lane.
//
// A token for each of 32 sequences of up to 4096, 32/8 heads of 128, float16: 60 µs for 274 MB, merge included; for 4 of
// 40 900, int8: 71 µs for 346 MB.  16 sequences of five drafted tokens over up to 2048 positions, e4m3, are 37 MB and
// take 26 µs: two steps a workgroup, bound by the chain from the search to the join of its wavefronts, and by the merge.

constexpr int STEP = 32, WAVES = 4, STEP_WG = STEP * WAVES;

// Steps of a workgroup (128 keys) that a sequence takes, at least one: its rows are written in any case.
__device__ __forceinline__ int steps_of(const Span& s) { return max(1, (s.keys + STEP_WG - 1) / STEP_WG); }

// The line, 64 sequences at a time: lane b holds sequence first + b and the inclusive sum of steps up to it, both
// of one K/V head.  Every wavefront builds it for itself, without a barrier.
struct Line {
    Span sp;
    int first, steps, run;
    int before;   // steps of the sequences before `first`
};

__device__ __forceinline__ void line_load(const PagedAttn& a, Line& ln) {
    const int lane = threadIdx.x & 63, b = ln.first + lane;
    ln.sp = span_of(a, min(b, a.B - 1));
    ln.steps = b < a.B ? steps_of(ln.sp) : 0;
    ln.run = ln.steps;
    for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(ln.run, o, 64);
        if (lane >= o) ln.run += t;
    }
}
// From the first sequence on, and all steps of a head.
__device__ __forceinline__ int line_begin(const PagedAttn& a, Line& ln) {
    int all = 0;
    for (int first = (a.B - 1) / 64 * 64; first >= 0; first -= 64) {
        ln.first = first;
        line_load(a, ln);
        all += __builtin_amdgcn_readlane(ln.run, 63);
    }
    ln.before = 0;
    return all;
}
__device__ __forceinline__ void line_next(const PagedAttn& a, Line& ln) {
    ln.before += __builtin_amdgcn_readlane(ln.run, 63);
    ln.first += 64;
    line_load(a, ln);
}

// A sequence of the line: itself, its span and steps, and the steps before it.
struct Place {
    int b, steps;
    Span sp;
    int before;
};
__device__ __forceinline__ Place line_place(const Line& ln, int lane) {
    Place p;
    p.b = ln.first + lane;
    p.steps = __builtin_amdgcn_readlane(ln.steps, lane);
    p.sp.start = __builtin_amdgcn_readlane(ln.sp.start, lane);
    p.sp.count = __builtin_amdgcn_readlane(ln.sp.count, lane);
    p.sp.keys = __builtin_amdgcn_readlane(ln.sp.keys, lane);
    p.before = ln.before + __builtin_amdgcn_readlane(ln.run, lane) - p.steps;
    return p;
}
// The sequence that step x of all heads' falls to; x lies in the line.
__device__ __forceinline__ Place line_seek(const PagedAttn& a, Line& ln, int x) {
    const int heads = a.c.heads;
    while (x >= (ln.before + __builtin_amdgcn_readlane(ln.run, 63)) * heads) line_next(a, ln);
    return line_place(ln, __builtin_ctzll(__ballot(x < (ln.before + ln.run) * heads)));
}

// Range w of W ≤ T over T steps starts at w·T/W; the range that step x falls to.
__device__ __forceinline__ int range_start(int w, int W, int T) { return (int)((unsigned long long)w * T / W); }
__device__ __forceinline__ int range_of(int x, int W, int T) { return (int)(((unsigned long long)x * W + W - 1) / T); }

// Floats of a partial result: rows of outputs, then each row's maximum and sum.
template <int HD, int NR>
constexpr int part_floats() { return 16 * NR * (HD + 2); }

// A wavefront's registers, about: tiles in flight, accumulators, the rest.  Two workgroups a CU where 256 registers
// are enough, with two tiles or else one; otherwise one, with two tiles where they fit.  (32 sequences, float16: two
// workgroups of one tile 63 µs, one of two 80.)
template <int TYPE, int HD, int NR>
constexpr int split_registers(int tiles) {
    return tiles * (HD * cache_elem(TYPE) / 4 + 16) + NR * HD / 4 + 64 + 20 * NR;
}
template <int TYPE, int HD, int NR>
constexpr int split_occupancy() { return split_registers<TYPE, HD, NR>(1) <= 256 ? 2 : 1; }
template <int TYPE, int HD, int NR>
constexpr int split_tiles() { return split_registers<TYPE, HD, NR>(2) <= (split_occupancy<TYPE, HD, NR>() == 2 ? 256 : 440) ? 2 : 1; }

// EXACT: rows have HD columns; else loads of columns that they do not have take the first ones (q is zero there).
template <int TYPE, int HD, int NR, bool EXACT>
__global__ __launch_bounds__(256, (split_occupancy<TYPE, HD, NR>())) void paged_split(PagedAttn a) {
    constexpr int ES = cache_elem(TYPE);
    constexpr int NK = HD / 32;          // MFMA steps over the columns
    constexpr int ND = HD / 16;          // 16-column blocks of the output
    constexpr int PL = TYPE == LBR_CACHE_F32 ? 2 : 1;
    constexpr int ROWS = 16 * NR;
    constexpr bool TWO = split_tiles<TYPE, HD, NR>() == 2;
    constexpr int LPR = HD / 4;          // threads of a row where all load or store it
    constexpr int PAD = HD + 4;          // floats of a row in `hand`: 16 rows' float4s then hit every bank once
    // q until the last step, [16 rows][MFMA step][h, l][lane][8]; then each wavefront's sums, `hand`[wave][row][PAD]
    __shared__ __attribute__((aligned(16))) char shared[WAVES * ROWS * PAD * 4];
    static_assert(2 * NR * NK * 1024 <= sizeof(shared), "q fits where the sums go");
    _Float16* const q_lds = (_Float16*)shared;
    float* const hand = (float*)shared;
    __shared__ float q_scale[ROWS], row_m[ROWS], row_l[ROWS];
    __shared__ float wave_m[WAVES][ROWS], wave_l[WAVES][ROWS];
    __shared__ int wave_up[WAVES];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, kg = lane >> 4;
    const PagedCache& c = a.c;
    const int page = 1 << c.shift, mask = page - 1;

    Line line;
    const int T = line_begin(a, line) * c.heads, W = min((int)gridDim.x, T), w = blockIdx.x;
    if (w >= W) return;
    int x = range_start(w, W, T);
    const int first = x, end = range_start(w + 1, W, T);
    Place pl = line_seek(a, line, x);
    int h = (x - pl.before * c.heads) / pl.steps;
    int at = x - pl.before * c.heads - h * pl.steps;

    const int hdp = EXACT ? HD : c.hdp;
    // bytes into a K row and into a V group of a lane's loads
    auto koff = [&](int j) {
        const int col = ES == 1 ? (j / 2) * 64 + kg * 16 + (j % 2) * 8 : j * 32 + kg * 8;
        return (EXACT || col < hdp ? col : 0) * ES;
    };
    auto voff = [&](int j) {
        const int col = ES == 1 ? (j / 2) * 32 + 2 * n + (j & 1) : j * 16 + n;
        return (EXACT || col < hdp ? col : 0) * 8 * ES;
    };

    // a wavefront's 32 keys of a step, as loaded
    struct Tile {
        uint4 k[2][NK * ES / 2], v[ND * ES / 2];
        float ks[8], vs[8];
    };
    struct Pages {
        int lo, hi;   // of its first and its last 16 keys
    };

    while (x < end) {   // segments
        const Span sp = pl.sp;
        const int b = pl.b, steps = pl.steps;
        const int stop = min(steps, at + (end - x));   // steps at .. stop − 1 of this segment
        // the wavefront's own: those that begin before the end
        const int mine = min(stop, (sp.keys - wave * STEP + STEP_WG - 1) / STEP_WG);
        const int lastg = (sp.keys - 1) & ~7;
        // Read through the scalar cache: in the order of vector loads a wait for them would be one for the tile
        // behind them.
        typedef const __attribute__((address_space(4))) int* Table;
        const Table tab = (Table)(c.table + (long long)b * c.wide);
        auto pages = [&](int st) {
            const int k0 = st * STEP_WG + wave * STEP;
            return Pages{tab[min(k0, lastg) >> c.shift], tab[min(k0 + 16, lastg) >> c.shift]};
        };
        auto is_page = [&](int p) { return p >= 0 && p < c.pages; };
        auto load = [&](Tile& t, int st, Pages p) {
            // the groups of eight keys that a lane loads K rows (n / 4) and V columns (kg) of, clamped to the last
            const int k0 = st * STEP_WG + wave * STEP;
            const int gk = min(k0 + 8 * (n >> 2), lastg), gv = min(k0 + 8 * kg, lastg);
            const char* const lo = c.base + (is_page(p.lo) ? p.lo : 0) * c.page_bytes + (long long)h * c.head_bytes;
            const char* const hi = c.base + (is_page(p.hi) ? p.hi : 0) * c.page_bytes + (long long)h * c.head_bytes;
            const char* const hk = n >= 8 ? hi : lo;
            const char* const hv = kg >= 2 ? hi : lo;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const char* const row = hk + ((gk & mask) + 4 * u + (n & 3)) * hdp * ES;
#pragma unroll
                for (int j = 0; j < NK; ++j) {
                    if (ES == 1) {
                        if (j % 2 == 0) t.k[u][j / 2] = *(const uint4*)(row + koff(j));
                    } else {
#pragma unroll
                        for (int e = 0; e < ES / 2; ++e) t.k[u][j * (ES / 2) + e] = *(const uint4*)(row + koff(j) + 16 * e);
                    }
                }
            }
            const float* const sc = (const float*)(hv + 2 * c.part) + (gv & mask);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float4 u = *(const float4*)(sc + 4 * e), v = *(const float4*)(sc + page + 4 * e);
                t.ks[4 * e] = u.x; t.ks[4 * e + 1] = u.y; t.ks[4 * e + 2] = u.z; t.ks[4 * e + 3] = u.w;
                t.vs[4 * e] = v.x; t.vs[4 * e + 1] = v.y; t.vs[4 * e + 2] = v.z; t.vs[4 * e + 3] = v.w;
            }
            const char* const vb = hv + c.part + (gv & mask) * hdp * ES;
#pragma unroll
            for (int j = 0; j < ND; ++j) {
                if (ES == 1) {
                    if (j % 2 == 0) t.v[j / 2] = *(const uint4*)(vb + voff(j));
                } else {
#pragma unroll
                    for (int e = 0; e < ES / 2; ++e) t.v[j * (ES / 2) + e] = *(const uint4*)(vb + voff(j) + 16 * e);
                }
            }
        };
        // rows of q into LDS: two halves, scaled, in the order of the MFMAs' operands
        int hd = c.hd;
        asm volatile("" : "+s"(hd));   // or what depends on it alone is worked out ahead of the loop, and spilled
        const int col = tid % LPR * 4;
        constexpr int EACH = ROWS * LPR / 256;   // rows a thread
        float v[EACH][4];
        {
#pragma unroll
            for (int i = 0; i < EACH; ++i) {   // all loads go out together, ahead of the first tile's
                const int r = i * (256 / LPR) + tid / LPR;
                const int token = (int)lbr_fdiv((unsigned)min(r, a.rows - 1), a.G_m, a.G_s), g = min(r, a.rows - 1) - token * a.G;
                const float* const qr = a.q + ((long long)(b * a.H + h * a.G + g) * a.S + token) * hd;
#pragma unroll
                for (int k = 0; k < 4; ++k) v[i][k] = 0.f;
                if (r < a.rows && token < sp.count) {
                    if (a.vec && col < hd) {
                        const float4 u = *(const float4*)(qr + col);
                        v[i][0] = u.x;
                        v[i][1] = u.y;
                        v[i][2] = u.z;
                        v[i][3] = u.w;
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (col + k < hd) v[i][k] = qr[col + k];
                    }
                }
            }
        }
        Tile ta, tb;
        Pages here = {0, 0}, next = {0, 0};   // of the step being computed, and of the next
        if (at < mine) {
            here = pages(at);
            if (at + 1 < mine) next = pages(at + 1);
            load(ta, at, here);
        }

        {
            const int j = ES == 1 ? col / 64 * 2 + col % 16 / 8 : col / 32, g4 = ES == 1 ? col % 64 / 16 : col % 32 / 8;
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int r = i * (256 / LPR) + tid / LPR;
                unsigned top = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[i][k] *= a.scale;
                    top = max(top, __float_as_uint(v[i][k]) & 0x7fffffffu);
                }
                top = row_max_bits<LPR>(top);
                const int up = up_exponent(top);
                const float by = __uint_as_float((unsigned)up << 23);
                halfx4 hi, lo;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    hi[k] = (_Float16)(v[i][k] * by);
                    lo[k] = (_Float16)(v[i][k] * by - (float)hi[k]);
                }
                _Float16* const to = q_lds + ((r / 16 * NK + j) * 2 * 64 + g4 * 16 + r % 16) * 8 + col % 8;
                *(halfx4*)to = hi;
                *(halfx4*)(to + 512) = lo;
                if (col == 0)
                    q_scale[r] = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float((unsigned)(254 - up) << 23);
            }
        }
        __syncthreads();
        float qs[NR];
        int last[NR];   // last key of row 16·t + n
#pragma unroll
        for (int t = 0; t < NR; ++t) {
            const int r = 16 * t + n, token = (int)lbr_fdiv((unsigned)min(r, a.rows - 1), a.G_m, a.G_s);
            qs[t] = q_scale[r];
            last[t] = r < a.rows ? last_key(sp, token) : -1;
        }

        floatx4 o[NR][ND];
        float m[NR], l[NR];
        int vup = 254;   // biased exponent of the power of two that V rows' scales are taken by
#pragma unroll
        for (int t = 0; t < NR; ++t) {
            m[t] = -INFINITY;
            l[t] = 0.f;
#pragma unroll
            for (int j = 0; j < ND; ++j) o[t][j] = floatx4{0.f, 0.f, 0.f, 0.f};
        }

        auto compute = [&](Tile& t, int st, Pages at_page) {
            const int k0 = st * STEP_WG + wave * STEP;
            // keys behind the end, and pages that are none, hold anything
            const bool badv = !is_page(kg >= 2 ? at_page.hi : at_page.lo);
            const int keep = sp.keys - (k0 + 8 * kg);   // of the lane's eight keys
            const bool tail = k0 + STEP > sp.keys;
            if (tail || !is_page(at_page.lo) || !is_page(at_page.hi)) {
                const int keepv = badv ? 0 : keep;
                unsigned to[4];   // words of eight values, as far as the type has them
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int bits = ES == 1 ? 8 * min(max(keepv - 4 * (e & 1), 0), 4) : 16 * min(max(keepv - 2 * e, 0), 2);
                    to[e] = bits == 32 ? ~0u : (1u << bits) - 1u;
                }
#pragma unroll
                for (int j = 0; j < ND * ES / 2; ++j) {
                    if (ES == 4) {
                        const int e = j % 2 * 4;
                        t.v[j].x = e < keepv ? t.v[j].x : 0u;
                        t.v[j].y = e + 1 < keepv ? t.v[j].y : 0u;
                        t.v[j].z = e + 2 < keepv ? t.v[j].z : 0u;
                        t.v[j].w = e + 3 < keepv ? t.v[j].w : 0u;
                    } else {
                        t.v[j].x &= to[0];
                        t.v[j].y &= to[1];
                        t.v[j].z &= to[2];
                        t.v[j].w &= to[3];
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (badv) t.ks[e] = t.vs[e] = __uint_as_float(0x7fc00000u);
                    if (e >= keep) t.vs[e] = 0.f;
                }
            }

            // scores, two blocks of 16 keys
            floatx4 s[NR][2];
#pragma unroll
            for (int r = 0; r < NR; ++r) s[r][0] = s[r][1] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < NK; ++j) {
                halfx8 kh[2], kl[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if constexpr (TYPE == LBR_CACHE_F32) {
                        const uint4 y = t.k[u][2 * j], z = t.k[u][2 * j + 1];
                        const float f[8] = {__uint_as_float(y.x), __uint_as_float(y.y), __uint_as_float(y.z), __uint_as_float(y.w),
                                            __uint_as_float(z.x), __uint_as_float(z.y), __uint_as_float(z.z), __uint_as_float(z.w)};
                        split8(f, kh[u], kl[u]);
                    } else if constexpr (TYPE == LBR_CACHE_F16) {
                        kh[u] = __builtin_bit_cast(halfx8, t.k[u][j]);
                    } else {
                        const uint4 y = t.k[u][j / 2];
                        kh[u] = j % 2 ? widen8<TYPE>(y.z, y.w) : widen8<TYPE>(y.x, y.y);
                    }
                }
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const halfx8 hi = *(const halfx8*)(q_lds + ((r * NK + j) * 2 * 64 + lane) * 8);
                    const halfx8 lo = *(const halfx8*)(q_lds + ((r * NK + j) * 2 * 64 + 64 + lane) * 8);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        s[r][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[u], lo, s[r][u], 0, 0, 0);
                        if constexpr (PL == 2) s[r][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl[u], hi, s[r][u], 0, 0, 0);
                        s[r][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[u], hi, s[r][u], 0, 0, 0);
                    }
                }
            }

            __builtin_amdgcn_sched_barrier(0);   // or values widened ahead of their phase spill
            // the V rows' scales over a running power of two
            float vtop = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) vtop = fmaxf(vtop, t.vs[e]);
            vtop = quad_max(vtop);
            const int vnew = __builtin_amdgcn_readfirstlane(min(vup, up_exponent(__float_as_uint(vtop))));
            const float vby = __uint_as_float((unsigned)vnew << 23);
            float vs[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) vs[e] = t.vs[e] * vby;

            const bool edge = tail || k0 + STEP - 1 > sp.start;   // some row ends among these keys
            halfx8 ph[NR], pl[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float sc[8], top = -INFINITY;
#pragma unroll
                for (int e = 0; e < 8; ++e) sc[e] = s[r][e >> 2][e & 3] * (t.ks[e] * qs[r]);
                if (edge) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (k0 + 8 * kg + e > last[r]) sc[e] = -INFINITY;   // a row's last key lies before the end
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, sc[e]);
                const float mx = fmaxf(m[r], quad_max(top));
                const float base = mx == -INFINITY ? 0.f : mx;
                const float alpha = __builtin_amdgcn_exp2f(m[r] - base);
                m[r] = mx;
                float p[8], sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    p[e] = __builtin_amdgcn_exp2f(sc[e] - base);
                    sum += p[e];
                    p[e] *= vs[e];
                }
                if (edge) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (sc[e] == -INFINITY) p[e] = 0.f;   // no weight, whatever the V row holds
                }
                l[r] = l[r] * alpha + sum;
                split8(p, ph[r], pl[r]);
                const float f = __builtin_amdgcn_ldexpf(alpha, vnew - vup);
#pragma unroll
                for (int j = 0; j < ND; ++j) o[r][j] *= f;
            }
            vup = vnew;
            __builtin_amdgcn_sched_barrier(0);

#pragma unroll
            for (int j = 0; j < ND; ++j) {
                halfx8 vh, vl;
                if constexpr (TYPE == LBR_CACHE_F32) {
                    const uint4 y = t.v[2 * j], z = t.v[2 * j + 1];
                    const float f[8] = {__uint_as_float(y.x), __uint_as_float(y.y), __uint_as_float(y.z), __uint_as_float(y.w),
                                        __uint_as_float(z.x), __uint_as_float(z.y), __uint_as_float(z.z), __uint_as_float(z.w)};
                    split8(f, vh, vl);
                } else if constexpr (TYPE == LBR_CACHE_F16) {
                    vh = __builtin_bit_cast(halfx8, t.v[j]);
                } else {
                    const uint4 y = t.v[j / 2];
                    vh = j % 2 ? widen8<TYPE>(y.z, y.w) : widen8<TYPE>(y.x, y.y);
                }
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    o[r][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl[r], o[r][j], 0, 0, 0);
                    if constexpr (PL == 2) o[r][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph[r], o[r][j], 0, 0, 0);
                    o[r][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph[r], o[r][j], 0, 0, 0);
                }
            }
        };

        // while a step is computed the next one's loads are in flight (where registers hold both), and the page ids
        // of the one after
        auto step = [&](Tile& t, Tile& other, int st) {
            const Pages at_page = here;
            here = next;
            if (TWO && st + 1 < mine) load(other, st + 1, here);
            if (st + 2 < mine) next = pages(st + 2);
            compute(t, st, at_page);
            if (!TWO && st + 1 < mine) load(t, st + 1, here);
        };
        if constexpr (TWO) {
            for (int st = at; st < mine; st += 2) {
                step(ta, tb, st);
                if (st + 1 < mine) step(tb, ta, st + 1);
            }
        } else {
            for (int st = at; st < mine; ++st) step(ta, ta, st);
        }

        // join the wavefronts: each brings its sums to the rows' maximum and the smallest power of two and hands them
        // over, and all threads add up
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            l[r] = quad_sum(l[r]);
            if (kg == 0) {
                wave_m[wave][16 * r + n] = m[r];
                wave_l[wave][16 * r + n] = l[r];
            }
        }
        if (lane == 0) wave_up[wave] = vup;
        __syncthreads();
        const int up = min(min(wave_up[0], wave_up[1]), min(wave_up[2], wave_up[3]));
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            float mx = m[r];
#pragma unroll
            for (int k = 0; k < WAVES; ++k) mx = fmaxf(mx, wave_m[k][16 * r + n]);
            const float f = __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(m[r] - (mx == -INFINITY ? 0.f : mx)), up - vup);
            float* const to = hand + ((wave * ROWS) + 16 * r + n) * PAD;
            // a lane's accumulators are columns 4·kg .. of a block, or every other one of 8·kg .. of two
#pragma unroll
            for (int j = 0; j < ND; j += ES == 1 ? 2 : 1) {
                const floatx4 x = o[r][j] * f;
                if constexpr (ES == 1) {
                    const floatx4 y = o[r][j + 1] * f;
                    *(floatx4*)(to + j * 16 + 8 * kg) = floatx4{x[0], y[0], x[1], y[1]};
                    *(floatx4*)(to + j * 16 + 8 * kg + 4) = floatx4{x[2], y[2], x[3], y[3]};
                } else {
                    *(floatx4*)(to + j * 16 + 4 * kg) = x;
                }
            }
        }
        if (tid < ROWS) {
            float mx = wave_m[0][tid], sum = 0.f;
#pragma unroll
            for (int k = 1; k < WAVES; ++k) mx = fmaxf(mx, wave_m[k][tid]);
            const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
            for (int k = 0; k < WAVES; ++k) sum += wave_l[k][tid] * __builtin_amdgcn_exp2f(wave_m[k][tid] - base);
            row_m[tid] = mx;
            row_l[tid] = sum;
        }
        __syncthreads();

        const int seg = pl.before * c.heads + h * steps;   // its first step in the line
        const bool whole = seg >= first && seg + steps <= end;
        float* const part = a.parts + (2LL * w + (seg >= first)) * part_floats<HD, NR>();
        for (int r = tid / LPR; r < a.rows; r += 256 / LPR) {
            const float sum = row_l[r];
            const float inv = sum == 0.f ? 0.f : 1.f / sum;   // no keys in this range
            floatx4 t = *(const floatx4*)(hand + r * PAD + col);
#pragma unroll
            for (int k = 1; k < WAVES; ++k) t += *(const floatx4*)(hand + (k * ROWS + r) * PAD + col);
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = __builtin_amdgcn_ldexpf(t[k] * inv, 127 - up);
            if (!whole) {
                *(float4*)(part + r * HD + col) = make_float4(v[0], v[1], v[2], v[3]);
                if (col == 0) {
                    part[ROWS * HD + r] = row_m[r];
                    part[ROWS * HD + ROWS + r] = sum;
                }
                continue;
            }
            const int token = (int)lbr_fdiv((unsigned)r, a.G_m, a.G_s), g = r - token * a.G;
            float* const to = a.out + ((long long)(b * a.H + h * a.G + g) * a.S + token) * hd;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = row_value(a, sp, token, v[k]);
            if (a.vec && col < hd) {
                *(float4*)(to + col) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (col + k < hd) to[col + k] = v[k];
            }
        }
        if (stop - at + x < end) __syncthreads();   // the next segment's q goes where the sums are
        // the next segment
        x += stop - at;
        at = 0;
        if (++h == c.heads && x < end) {
            h = 0;
            const int lane1 = b + 1 - line.first;
            if (lane1 == 64) line_next(a, line);
            pl = line_place(line, lane1 & 63);
        }
    }
}

// Joins the partial results of a segment that ranges cut, gridDim.y workgroups its rows: HD / 4 threads across a
// row, and the results dealt out over the rest, which add up in LDS.
template <int HD, int NR>
__global__ __launch_bounds__(256) void paged_merge(PagedAttn a, int ranges) {
    constexpr int ROWS = 16 * NR, LANES = HD / 4, SLICES = 256 / LANES;
    __shared__ float slice_m[SLICES], slice_l[SLICES];
    __shared__ floatx4 slice_o[SLICES][LANES];
    const int tid = threadIdx.x;
    const PagedCache& c = a.c;
    const int b = blockIdx.x / c.heads, h = blockIdx.x % c.heads;
    Line line;
    const int T = line_begin(a, line) * c.heads, W = min(ranges, T);
    while (b >= line.first + 64) line_next(a, line);
    const Place pl = line_place(line, b - line.first);
    const int seg = pl.before * c.heads + h * pl.steps;
    const int w0 = range_of(seg, W, T), w1 = range_of(seg + pl.steps - 1, W, T);
    if (w0 == w1) return;   // finished by its range
    const int lane = tid % LANES, slice = tid / LANES;
    for (int row = blockIdx.y; row < a.rows; row += gridDim.y) {
        float m = -INFINITY, l = 0.f;
        floatx4 o = {0.f, 0.f, 0.f, 0.f};
        constexpr int AHEAD = 4;   // loads in flight
        for (int w = w0 + slice; w <= w1; w += AHEAD * SLICES) {
            float pm[AHEAD], ps[AHEAD];
            floatx4 v[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int at = min(w + k * SLICES, w1);
                const float* const part = a.parts + (2LL * at + (at == w0)) * part_floats<HD, NR>();
                pm[k] = part[ROWS * HD + row];
                ps[k] = w + k * SLICES <= w1 ? part[ROWS * HD + ROWS + row] : 0.f;
                v[k] = *(const floatx4*)(part + row * HD + 4 * lane);
            }
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
                if (w + k * SLICES <= w1) merge_part(m, l, o, pm[k], ps[k], v[k]);
        }
        __syncthreads();   // of the row before
        if (lane == 0) {
            slice_m[slice] = m;
            slice_l[slice] = l;
        }
        slice_o[slice][lane] = o;
        __syncthreads();
        if (slice) continue;
        for (int k = 1; k < SLICES; ++k) {   // sums, not weighted means
            const float mx = fmaxf(m, slice_m[k]), base = mx == -INFINITY ? 0.f : mx;
            const float f = __builtin_amdgcn_exp2f(m - base), g = __builtin_amdgcn_exp2f(slice_m[k] - base);
            o = o * f + slice_o[k][lane] * g;
            l = l * f + slice_l[k] * g;
            m = mx;
        }
        const float inv = 1.f / l;
        const int token = (int)lbr_fdiv((unsigned)row, a.G_m, a.G_s), g = row - token * a.G;
        float* const to = a.out + ((long long)(b * a.H + h * a.G + g) * a.S + token) * c.hd;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (4 * lane + e < c.hd) to[4 * lane + e] = row_value(a, pl.sp, token, o[e] * inv);
    }
}

// ---------------------------------------------------------------- launch

// Ranges of the split kernel: the workgroups that the chip holds at once (Step::i[11] a CU), or as many as there can
// be steps.
long long split_ranges(const Step& s) {
    const long long wgs = s.i[11] * (lbr_device_cus() > 0 ? lbr_device_cus() : 256);
    const long long steps = (((s.i[6] << s.i[4]) + STEP_WG - 1) / STEP_WG) * s.i[1] * s.i[2];
    return steps < wgs ? steps : wgs;
}
// Whether a segment can be longer than a step, and so cut.
bool split_cuts(const Step& s) { return (s.i[6] << s.i[4]) > STEP_WG; }

template <int TYPE, int HD, int NR>
void launch_split(const Step& s, hipStream_t st) {
    const PagedAttn a = attn_args(s);
    const long long W = split_ranges(s);
    if (W <= 0 || a.rows <= 0) return;
    if (a.c.hdp == HD) hipLaunchKernelGGL((paged_split<TYPE, HD, NR, true>), dim3((unsigned)W), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_split<TYPE, HD, NR, false>), dim3((unsigned)W), dim3(256), 0, st, a);
    if (split_cuts(s)) {
        // at most the workgroups that the chip holds at once: a row takes one about as long as finding out that a
        // segment was not cut
        const long long segments = (long long)a.B * a.c.heads, each = 2048 / segments;
        const unsigned rows = (unsigned)(each < 1 ? 1 : each < a.rows ? each : a.rows);
        hipLaunchKernelGGL((paged_merge<HD, NR>), dim3((unsigned)segments, rows), dim3(256), 0, st, a, (int)W);
    }
}

template <int TYPE, int HD, int NR>
void choose(Step* s) {
    s->i[11] = split_occupancy<TYPE, HD, NR>();
    s->ws_bytes = split_cuts(*s) ? (size_t)(split_ranges(*s) * 2 * part_floats<HD, NR>()) * sizeof(float) : 0;
    s->run = launch_split<TYPE, HD, NR>;
}
template <int TYPE, int HD>
void choose_rows(Step* s, int nr) {
    nr == 1 ? choose<TYPE, HD, 1>(s) : choose<TYPE, HD, 2>(s);
}
template <int TYPE>
void choose_split(Step* s, int hd, int nr) {
    hd <= 64 ? choose_rows<TYPE, 64>(s, nr) : hd <= 128 ? choose_rows<TYPE, 128>(s, nr) : choose<TYPE, 256, 1>(s);
}

}  // namespace

int decode_paged_attention(const OpNode* n, Step* s) {
    const int* d = n->out_shape;
    if (n->n_dims != 4 || n->elem_size != 4 || d[3] != n->extra[2]) {
        lbr_set_error("paged_attention: the output is not float [B, H, S, head_dim]");
        return LBR_ERR_INVALID;
    }
    if (int rc = decode_paged_common(n, s, 1, 2, d[0])) return rc;
    s->in[4] = n->inputs[0];
    s->i[7] = d[2];
    s->i[8] = d[1];
    s->f[0] = node_extra_float(n, 6);
    if (d[1] < 1 || d[1] % s->i[2]) {
        lbr_set_error("paged_attention: %d query heads over %lld K/V heads", d[1], s->i[2]);
        return LBR_ERR_INVALID;
    }
    if (!(s->f[0] > 0.f) || s->f[0] > 3.4e38f) {
        lbr_set_error("paged_attention: the score scale is not a positive number");
        return LBR_ERR_INVALID;
    }
    if (!lbr_aligned(s->in[4], 4) || !lbr_aligned(s->out, 4)) {
        lbr_set_error("paged_attention: Q or the output does not start on a 4-byte boundary");
        return LBR_ERR_INVALID;
    }
    if (node_total(n) / d[3] >= (1LL << 31)) {
        lbr_set_error("paged_attention: %lld rows are more than one launch takes", node_total(n) / d[3]);
        return LBR_ERR_INVALID;
    }
    // a launch's threads are counted in 32 bits, 256 a workgroup
    if (s->i[1] * s->i[2] >= 1LL << 24) {
        lbr_set_error("paged_attention: %lld sequences of %lld heads are more than one launch takes", s->i[1], s->i[2]);
        return LBR_ERR_INVALID;
    }
    const int hd = (int)s->i[3];
    const long long rows = s->i[8] / s->i[2] * s->i[7];
    s->i[9] = hd % 4 == 0 && lbr_aligned(s->in[4], 16) && lbr_aligned(s->out, 16);
    // At most 32 rows a K/V head are split over the keys, in one or two blocks of 16; more go in tiles.  16 sequences
    // of 2048 keys, 32/8 heads of 128, 20 rows: 41 µs split and 52 in tiles (int8), 43 and 48 (float16), 76 and 78
    // (float32); 40 rows (in four blocks): 68 and 56, 99 and 52, 134 and 86.
    if (rows <= (hd <= 128 ? 32 : 16)) {   // two blocks of 256 columns do not fit the registers
        const long long steps = ((s->i[6] << s->i[4]) + STEP_WG - 1) / STEP_WG;
        if (s->i[1] * s->i[2] > 0 && steps > ((1LL << 31) - 1) / s->i[2] / s->i[1]) {
            lbr_set_error("paged_attention: tables of %lld sequences reach more steps than one launch takes", s->i[1]);
            return LBR_ERR_INVALID;
        }
        const int nr = rows <= 16 ? 1 : 2;
        if (s->i[0] == LBR_CACHE_F32) choose_split<LBR_CACHE_F32>(s, hd, nr);
        else if (s->i[0] == LBR_CACHE_F16) choose_split<LBR_CACHE_F16>(s, hd, nr);
        else if (s->i[0] == LBR_CACHE_I8) choose_split<LBR_CACHE_I8>(s, hd, nr);
        else choose_split<LBR_CACHE_E4M3>(s, hd, nr);
        s->name = "paged_split";
        return LBR_OK;
    }
    // grid: row tiles of all K/V heads
    if (paged_row_tiles(*s) >= (1LL << 24) / (s->i[2] * (s->i[1] > 0 ? s->i[1] : 1))) {
        lbr_set_error("paged_attention: %lld rows are more than one launch takes", node_total(n) / d[3]);
        return LBR_ERR_INVALID;
    }
    s->i[10] = paged_tiles_splits(*s);
    s->ws_bytes = paged_tiles_workspace(*s);
    s->run = paged_tiles_launcher((int)s->i[0], hd);
    s->name = "paged_tiles";
    return LBR_OK;
}
