// paged_attention.hip — attention over the paged cache: few rows a K/V head, and the choice between the kernels.
#include "paged_attention.h"

namespace {

// ---------------------------------------------------------------- few rows: split over the keys
//
// At most 64 rows a K/V head (single tokens, drafted tokens): the cache is read once and bounds the time.  A
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

constexpr int STEP = 32, WAVES = 4, STEP_WG = STEP * WAVES;

// Steps of a workgroup (128 keys) that sequence b takes, at least one: its rows are written in any case.
__device__ __forceinline__ int steps_of(const PagedAttn& a, int b) {
    return max(1, (span_of(a, b).keys + STEP_WG - 1) / STEP_WG);
}

// Where the ranges lie: sums of steps before each of 256 blocks of sequences (LDS), and the whole.
struct Line {
    long long before[257];
};

__device__ __forceinline__ void line_build(const PagedAttn& a, Line& ln) {
    __shared__ long long wave_sum[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (a.B + 255) / 256;
    long long mine = 0;
    for (int b = tid * per; b < min((tid + 1) * per, a.B); ++b) mine += steps_of(a, b);
    long long run = mine;
    for (int o = 1; o < 64; o <<= 1) {
        const long long t = __shfl_up(run, o, 64);
        if (lane >= o) run += t;
    }
    if (lane == 63) wave_sum[wave] = run;
    __syncthreads();
    for (int w = 0; w < wave; ++w) run += wave_sum[w];
    ln.before[tid + 1] = run;
    if (tid == 0) ln.before[0] = 0;
    __syncthreads();
}

// Sequence that step x (of one head's worth of steps a sequence, all heads: x / heads) falls to, and the steps before it.
__device__ __forceinline__ void line_find(const PagedAttn& a, const Line& ln, long long x, int& b, long long& before) {
    __shared__ int found_b;
    __shared__ long long found_before;
    const int tid = threadIdx.x, per = (a.B + 255) / 256;
    const long long heads = a.c.heads;
    if (x >= ln.before[tid] * heads && x < ln.before[tid + 1] * heads) {
        long long at = ln.before[tid];
        int k = tid * per;
        for (;; ++k) {
            const int n = steps_of(a, k);
            if (x < (at + n) * heads) break;
            at += n;
        }
        found_b = k;
        found_before = at;
    }
    __syncthreads();
    b = found_b;
    before = found_before;
}

// Range w of W ≤ T over T steps starts at w·T/W; the range that step x falls to.
__device__ __forceinline__ long long range_start(long long w, long long W, long long T) { return w * T / W; }
__device__ __forceinline__ long long range_of(long long x, long long W, long long T) { return ((x + 1) * W - 1) / T; }

// Floats of a partial result: rows of outputs, then each row's maximum and sum.
template <int HD, int NR>
constexpr int part_floats() { return 16 * NR * (HD + 2); }

template <int TYPE, int HD, int NR>
__global__ __launch_bounds__(256, 2) void paged_split(PagedAttn a) {
    constexpr int ES = cache_elem(TYPE);
    constexpr int NK = HD / 32;          // MFMA steps over the columns
    constexpr int ND = HD / 16;          // 16-column blocks of the output
    constexpr int PL = TYPE == LBR_CACHE_F32 ? 2 : 1;
    constexpr int ROWS = 16 * NR;
    __shared__ Line line;
    __shared__ float wave_m[WAVES][ROWS], wave_l[WAVES][ROWS];
    __shared__ int wave_up[WAVES];
    __shared__ __attribute__((aligned(16))) float hand[2][ROWS * HD];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, kg = lane >> 4;
    const PagedCache& c = a.c;
    const int page = 1 << c.shift, mask = page - 1;

    line_build(a, line);
    const long long T = line.before[256] * c.heads, W = min((long long)gridDim.x, T), w = blockIdx.x;
    if (w >= W) return;
    long long x = range_start(w, W, T);
    const long long first = x, end = range_start(w + 1, W, T);
    int b;
    long long before;
    line_find(a, line, x, b, before);
    int steps = steps_of(a, b);
    int h = (int)((x - before * c.heads) / steps);
    int at = (int)(x - before * c.heads - (long long)h * steps);

    // columns of a lane's loads, clamped to the row (q is zero behind it)
    int koff[NK], voff[ND];
#pragma unroll
    for (int j = 0; j < NK; ++j) {
        const int col = ES == 1 ? (j / 2) * 64 + kg * 16 + (j % 2) * 8 : j * 32 + kg * 8;
        koff[j] = (col < c.hdp ? col : 0) * ES;
    }
#pragma unroll
    for (int j = 0; j < ND; ++j) {
        const int col = ES == 1 ? (j / 2) * 32 + 2 * n + (j & 1) : j * 16 + n;
        voff[j] = (col < c.hdp ? col : 0) * 8 * ES;
    }

    while (x < end) {   // segments
        const Span sp = span_of(a, b);
        const int stop = (int)min((long long)steps, at + (end - x));   // steps at .. stop − 1 of this segment

        // rows of q: two halves, scaled; row 16·t + n
        halfx8 qh[NR][NK], ql[NR][NK];
        float qs[NR];
        int last[NR];   // last key of the row
#pragma unroll
        for (int t = 0; t < NR; ++t) {
            const int r = 16 * t + n;
            const int token = (int)lbr_fdiv((unsigned)min(r, a.rows - 1), a.G_m, a.G_s), g = min(r, a.rows - 1) - token * a.G;
            const float* const qr = a.q + ((long long)(b * a.H + h * a.G + g) * a.S + token) * c.hd;
            last[t] = r < a.rows && token < sp.count ? sp.start + token : -1;
            float v[NK][8];
            unsigned top = 0;
#pragma unroll
            for (int j = 0; j < NK; ++j) {
                const int col = ES == 1 ? (j / 2) * 64 + kg * 16 + (j % 2) * 8 : j * 32 + kg * 8;
#pragma unroll
                for (int k = 0; k < 8; ++k) v[j][k] = 0.f;
                if (last[t] >= 0) {
                    if (a.vec && col + 8 <= c.hd) {
                        const float4 u0 = *(const float4*)(qr + col), u1 = *(const float4*)(qr + col + 4);
                        v[j][0] = u0.x; v[j][1] = u0.y; v[j][2] = u0.z; v[j][3] = u0.w;
                        v[j][4] = u1.x; v[j][5] = u1.y; v[j][6] = u1.z; v[j][7] = u1.w;
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (col + k < c.hd) v[j][k] = qr[col + k];
                    }
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    v[j][k] *= a.scale;
                    top = max(top, __float_as_uint(v[j][k]) & 0x7fffffffu);
                }
            }
            top = quad_max_bits(top);
            const int up = up_exponent(top);
            const float by = __uint_as_float((unsigned)up << 23);
            qs[t] = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float((unsigned)(254 - up) << 23);
#pragma unroll
            for (int j = 0; j < NK; ++j) {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[j][k] *= by;
                split8(v[j], qh[t][j], ql[t][j]);
            }
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

        for (int st = at; st < stop; ++st) {
            const int k0 = st * STEP_WG + wave * STEP;
            if (k0 >= sp.keys) break;   // wave-uniform
            // the groups of eight keys that this lane loads K rows (n / 4) and V columns (kg) of, clamped to the last
            const int lastg = (sp.keys - 1) & ~7;
            const int gk = min(k0 + 8 * (n >> 2), lastg), gv = min(k0 + 8 * kg, lastg);
            const int* const tab = c.table + (long long)b * c.wide;
            const int pk = tab[gk >> c.shift], pv = tab[gv >> c.shift];
            const bool badv = pv < 0 || pv >= c.pages;
            const char* const hk = c.base + (pk < 0 || pk >= c.pages ? 0 : pk) * c.page_bytes + (long long)h * c.head_bytes;
            const char* const hv = c.base + (badv ? 0 : pv) * c.page_bytes + (long long)h * c.head_bytes;

            uint4 kr[2][NK * ES / 2], vr[ND * ES / 2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const char* const row = hk + (long long)((gk & mask) + 4 * t + (n & 3)) * c.hdp * ES;
#pragma unroll
                for (int j = 0; j < NK; ++j) {
                    if (ES == 1) {
                        if (j % 2 == 0) kr[t][j / 2] = *(const uint4*)(row + koff[j]);
                    } else {
#pragma unroll
                        for (int e = 0; e < ES / 2; ++e) kr[t][j * (ES / 2) + e] = *(const uint4*)(row + koff[j] + 16 * e);
                    }
                }
            }
            const char* const vb = hv + c.part + (long long)(gv & mask) * c.hdp * ES;
#pragma unroll
            for (int j = 0; j < ND; ++j) {
                if (ES == 1) {
                    if (j % 2 == 0) vr[j / 2] = *(const uint4*)(vb + voff[j]);
                } else {
#pragma unroll
                    for (int e = 0; e < ES / 2; ++e) vr[j * (ES / 2) + e] = *(const uint4*)(vb + voff[j] + 16 * e);
                }
            }
            float ks[8], vs[8];
            {
                const float* const sc = (const float*)(hv + 2 * c.part) + (gv & mask);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float4 u = *(const float4*)(sc + 4 * e), v = *(const float4*)(sc + page + 4 * e);
                    ks[4 * e] = u.x; ks[4 * e + 1] = u.y; ks[4 * e + 2] = u.z; ks[4 * e + 3] = u.w;
                    vs[4 * e] = v.x; vs[4 * e + 1] = v.y; vs[4 * e + 2] = v.z; vs[4 * e + 3] = v.w;
                }
            }
            // keys behind the end, and pages that are none
            const bool tail = k0 + STEP > sp.keys;
            const int keep = sp.keys - (k0 + 8 * kg);   // of the lane's eight keys
            const int keepv = badv ? 0 : keep;
            const bool cut = tail || __any(badv);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (badv) ks[e] = vs[e] = __uint_as_float(0x7fc00000u);
                if (tail && e >= keep) vs[e] = 0.f;
            }

            // scores, two blocks of 16 keys
            floatx4 s[NR][2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int r = 0; r < NR; ++r) s[r][t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < NK; ++j) {
                    halfx8 kh, kl;
                    if constexpr (TYPE == LBR_CACHE_F32) {
                        const uint4 u = kr[t][2 * j], v = kr[t][2 * j + 1];
                        const float f[8] = {__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w),
                                            __uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
                        split8(f, kh, kl);
                    } else if constexpr (TYPE == LBR_CACHE_F16) {
                        kh = __builtin_bit_cast(halfx8, kr[t][j]);
                    } else {
                        const uint4 u = kr[t][j / 2];
                        kh = j % 2 ? widen8<TYPE>(u.z, u.w) : widen8<TYPE>(u.x, u.y);
                    }
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        s[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, ql[r][j], s[r][t], 0, 0, 0);
                        if constexpr (PL == 2) s[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl, qh[r][j], s[r][t], 0, 0, 0);
                        s[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qh[r][j], s[r][t], 0, 0, 0);
                    }
                }
            }

            // the V rows' scales over a running power of two
            float vtop = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) vtop = fmaxf(vtop, vs[e]);
            vtop = quad_max(vtop);
            const int vnew = __builtin_amdgcn_readfirstlane(min(vup, up_exponent(__float_as_uint(vtop))));
            const float vby = __uint_as_float((unsigned)vnew << 23);
#pragma unroll
            for (int e = 0; e < 8; ++e) vs[e] *= vby;

            halfx8 ph[NR], pl[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float sc[8], top = -INFINITY;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    sc[e] = s[r][e >> 2][e & 3] * (ks[e] * qs[r]);
                    if (k0 + 8 * kg + e > last[r] || (tail && e >= keep)) sc[e] = -INFINITY;
                    top = fmaxf(top, sc[e]);
                }
                const float mx = fmaxf(m[r], quad_max(top));
                const float base = mx == -INFINITY ? 0.f : mx;
                const float alpha = __builtin_amdgcn_exp2f(m[r] - base);
                m[r] = mx;
                float p[8], sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    p[e] = __builtin_amdgcn_exp2f(sc[e] - base);
                    sum += p[e];
                    p[e] = sc[e] == -INFINITY ? 0.f : p[e] * vs[e];   // no weight, whatever the V row holds
                }
                l[r] = l[r] * alpha + sum;
                split8(p, ph[r], pl[r]);
                const float f = __builtin_amdgcn_ldexpf(alpha, vnew - vup);
                if (__any(f != 1.f)) {
                    asm volatile("");   // a branch: done ahead of it, the products would need registers of their own
#pragma unroll
                    for (int j = 0; j < ND; ++j) o[r][j] *= f;
                }
            }
            vup = vnew;

#pragma unroll
            for (int j = 0; j < ND; ++j) {
                halfx8 vh, vl;
                if constexpr (TYPE == LBR_CACHE_F32) {
                    const uint4 u = vr[2 * j], v = vr[2 * j + 1];
                    const float f[8] = {__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w),
                                        __uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
                    split8(f, vh, vl);
                } else if constexpr (TYPE == LBR_CACHE_F16) {
                    vh = __builtin_bit_cast(halfx8, vr[j]);
                } else {
                    const uint4 u = vr[j / 2];
                    vh = j % 2 ? widen8<TYPE>(u.z, u.w) : widen8<TYPE>(u.x, u.y);
                }
                if (cut) {   // what lies behind the end may be anything
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (e >= keepv) vh[e] = (_Float16)0.f;
                        if (PL == 2 && e >= keepv) vl[e] = (_Float16)0.f;
                    }
                }
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    o[r][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl[r], o[r][j], 0, 0, 0);
                    if constexpr (PL == 2) o[r][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph[r], o[r][j], 0, 0, 0);
                    o[r][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph[r], o[r][j], 0, 0, 0);
                }
            }
        }

        // join the wavefronts: 2 and 3 hand theirs to 0 and 1, then 1 to 0
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
        int up = wave_up[0];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) up = min(up, wave_up[k]);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            float mx = wave_m[0][16 * r + n], sum = 0.f;
#pragma unroll
            for (int k = 1; k < WAVES; ++k) mx = fmaxf(mx, wave_m[k][16 * r + n]);
            const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
            for (int k = 0; k < WAVES; ++k) sum += wave_l[k][16 * r + n] * __builtin_amdgcn_exp2f(wave_m[k][16 * r + n] - base);
            const float f = __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(m[r] - base), up - vup);
#pragma unroll
            for (int j = 0; j < ND; ++j) o[r][j] *= f;
            m[r] = mx;
            l[r] = sum;
        }
#pragma unroll
        for (int half = WAVES / 2; half; half >>= 1) {
            if (wave >= half && wave < 2 * half) {
                floatx4* const to = (floatx4*)hand[wave - half];
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int j = 0; j < ND; ++j) to[(r * ND + j) * 64 + lane] = o[r][j];
            }
            __syncthreads();
            if (wave < half) {
                const floatx4* const from = (const floatx4*)hand[wave];
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int j = 0; j < ND; ++j) o[r][j] += from[(r * ND + j) * 64 + lane];
            }
            __syncthreads();
        }

        if (wave == 0) {
            const long long seg = (before * c.heads) + (long long)h * steps;   // its first step in the line
            const bool whole = seg >= first && seg + steps <= end;
            float* const part = a.parts + (2 * w + (seg >= first)) * part_floats<HD, NR>();
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const int row = 16 * r + n;
                const int token = (int)lbr_fdiv((unsigned)min(row, a.rows - 1), a.G_m, a.G_s), g = min(row, a.rows - 1) - token * a.G;
                const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];   // no keys in this range
                float* const to = whole ? a.out + ((long long)(b * a.H + h * a.G + g) * a.S + token) * c.hd : part + row * HD;
                if (!whole && kg == 0) {
                    part[ROWS * HD + row] = m[r];
                    part[ROWS * HD + ROWS + row] = l[r];
                }
                if (whole && row >= a.rows) continue;
                const bool vec = !whole || a.vec;
                const int cols = whole ? c.hd : HD;
#pragma unroll
                for (int j = 0; j < ND; j += ES == 1 ? 2 : 1) {
                    // four (eight) neighbouring columns
                    constexpr int NC = ES == 1 ? 8 : 4;
                    const int col = ES == 1 ? (j / 2) * 32 + 8 * kg : j * 16 + 4 * kg;
                    float v[NC];
#pragma unroll
                    for (int k = 0; k < NC; ++k) {
                        const float e = ES == 1 ? o[r][j + (k & 1)][k >> 1] : o[r][j][k];
                        v[k] = __builtin_amdgcn_ldexpf(e * inv, 127 - up);
                        if (whole) v[k] = row_value(a, sp, token, v[k]);
                    }
#pragma unroll
                    for (int k = 0; k < NC; k += 4) {
                        if (vec && col + k + 4 <= cols) {
                            *(float4*)(to + col + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (col + k + e < cols) to[col + k + e] = v[k + e];
                        }
                    }
                }
            }
        }
        // the next segment
        x += stop - at;
        at = 0;
        if (++h == c.heads && x < end) {
            h = 0;
            before += steps;
            steps = steps_of(a, ++b);
        }
    }
}

// Joins the partial results of a segment that ranges cut: one workgroup a (sequence, K/V head, 16 rows).
template <int HD, int NR>
__global__ __launch_bounds__(256) void paged_merge(PagedAttn a, long long ranges) {
    constexpr int ROWS = 16 * NR;
    __shared__ Line line;
    const int tid = threadIdx.x;
    const PagedCache& c = a.c;
    const int b = blockIdx.x / c.heads, h = blockIdx.x % c.heads;
    line_build(a, line);
    // steps before sequence b: those before its block of sequences, and of the block's before it
    const int per = (a.B + 255) / 256;
    long long before = line.before[b / per];
    for (int k = b / per * per; k < b; ++k) before += steps_of(a, k);
    const int steps = steps_of(a, b);
    const long long T = line.before[256] * c.heads, W = min(ranges, T), seg = before * c.heads + (long long)h * steps;
    const long long w0 = range_of(seg, W, T), w1 = range_of(seg + steps - 1, W, T);
    if (w0 == w1) return;   // finished by its range
    const Span sp = span_of(a, b);
    constexpr int LANES = HD / 4;    // threads a row
    for (int row = blockIdx.y * 16 + tid / LANES; row < min(a.rows, (int)blockIdx.y * 16 + 16); row += 256 / LANES) {
        const int col = tid % LANES * 4;
        float m = -INFINITY, l = 0.f;
        floatx4 o = {0.f, 0.f, 0.f, 0.f};
        for (long long w = w0; w <= w1; ++w) {
            const float* const part = a.parts + (2 * w + (w == w0)) * part_floats<HD, NR>();
            const float pm = part[ROWS * HD + row], pl = part[ROWS * HD + ROWS + row];
            const floatx4 v = *(const floatx4*)(part + row * HD + col);
            const float mx = fmaxf(m, pm), base = mx == -INFINITY ? 0.f : mx;
            const float f = __builtin_amdgcn_exp2f(m - base), g = __builtin_amdgcn_exp2f(pm - base) * pl;
            o = o * f + v * g;
            l = l * f + g;
            m = mx;
        }
        const float inv = 1.f / l;
        const int token = (int)lbr_fdiv((unsigned)row, a.G_m, a.G_s), g = row - token * a.G;
        float* const to = a.out + ((long long)(b * a.H + h * a.G + g) * a.S + token) * c.hd;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < c.hd) to[col + e] = row_value(a, sp, token, o[e] * inv);
    }
}

// ---------------------------------------------------------------- launch

// Ranges of the split kernel: two workgroups a CU, as many as there can be steps.
long long split_ranges(const Step& s) {
    const int cus = lbr_device_cus() > 0 ? lbr_device_cus() : 256;
    const long long steps = (((s.i[6] << s.i[4]) + STEP_WG - 1) / STEP_WG) * s.i[1] * s.i[2];
    return steps < 2LL * cus ? steps : 2LL * cus;
}
// Whether a segment can be longer than a step, and so cut.
bool split_cuts(const Step& s) { return (s.i[6] << s.i[4]) > STEP_WG; }

template <int TYPE, int HD, int NR>
void launch_split(const Step& s, hipStream_t st) {
    const PagedAttn a = attn_args(s);
    const long long W = split_ranges(s);
    if (W <= 0 || a.rows <= 0) return;
    hipLaunchKernelGGL((paged_split<TYPE, HD, NR>), dim3((unsigned)W), dim3(256), 0, st, a);
    if (split_cuts(s))
        hipLaunchKernelGGL((paged_merge<HD, NR>), dim3((unsigned)(a.B * a.c.heads), (unsigned)((a.rows + 15) / 16)),
                           dim3(256), 0, st, a, W);
}

template <int TYPE, int HD>
step_fn split_rows(int nr) {
    return nr == 1 ? launch_split<TYPE, HD, 1> : nr == 2 ? launch_split<TYPE, HD, 2> : launch_split<TYPE, HD, 4>;
}
template <int TYPE>
step_fn split_for(int hd, int nr) {
    return hd <= 64 ? split_rows<TYPE, 64>(nr) : hd <= 128 ? split_rows<TYPE, 128>(nr) : split_rows<TYPE, 256>(nr);
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
    const int hd = (int)s->i[3];
    const long long rows = s->i[8] / s->i[2] * s->i[7];
    s->i[9] = hd % 4 == 0 && lbr_aligned(s->in[4], 16) && lbr_aligned(s->out, 16);
    if (rows <= 64) {
        const int nr = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
        const int wide = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
        s->ws_bytes = split_cuts(*s) ? (size_t)(split_ranges(*s) * 2 * 16 * nr * (wide + 2)) * sizeof(float) : 0;
        s->run = s->i[0] == LBR_CACHE_F32   ? split_for<LBR_CACHE_F32>(hd, nr)
                 : s->i[0] == LBR_CACHE_F16 ? split_for<LBR_CACHE_F16>(hd, nr)
                 : s->i[0] == LBR_CACHE_I8  ? split_for<LBR_CACHE_I8>(hd, nr)
                                            : split_for<LBR_CACHE_E4M3>(hd, nr);
        s->name = "paged_split";
        return LBR_OK;
    }
    // grid: row tiles of all K/V heads
    if (paged_row_tiles(*s) > ((1LL << 31) - 1) / (s->i[2] * (s->i[1] > 0 ? s->i[1] : 1))) {
        lbr_set_error("paged_attention: %lld rows are more than one launch takes", node_total(n) / d[3]);
        return LBR_ERR_INVALID;
    }
    s->i[10] = paged_tiles_splits(*s);
    s->ws_bytes = paged_tiles_workspace(*s);
    s->run = paged_tiles_launcher((int)s->i[0], hd);
    s->name = "paged_tiles";
    return LBR_OK;
}
