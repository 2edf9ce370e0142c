// verify.hip — drafted tokens against the target's probabilities, from given random numbers.
//
// Token i (i < count) stands while u_i · draft_i[t_i] < target_i[t_i] and all before it stood; each
// product is of two floats and exact in 64 bits.  Behind the n that stand comes one drawn from
// r = max(target_n − draft_n, 0), or from target_n where all stand or r is zero everywhere: the first index
// whose running sum passes u_D · Σ r, sums in 64 bits.
//
// What bounds it: the two rows of V floats that r takes, of a sequence whose position n is known only
// from its first D probabilities; for one sequence the chain of dependent loads.  So a first kernel lets every
// wavefront find n for itself (its loads of tokens, numbers and probabilities, one vote) and sum 1024 entries of
// r; a second, one wavefront a sequence, finds the part in which the running sum passes and goes through that
// part's entries alone again, 16 in a row a lane.
//
// 64 sequences of five drafts, 151 936 entries: 19 µs (78 MB); one of four, 50 257: 9, two chains of loads and launches.
#include "lbr_device.h"

namespace {

constexpr int EACH = 16, PART = 64 * EACH;   // entries of a lane and of a wavefront
constexpr int WAVES = 4;                     // of a workgroup of the sums

struct VerifyArgs {
    const float* target;
    const float* draft;
    const long long* tokens;
    const float* uniforms;
    const int* count;
    long long* out;
    double* sums;              // [B][parts][2]: of r, of the target's own row
    int* standing;             // [B]: n
    int D, V, parts;
};

// Tokens of sequence b that stand; every lane of the wavefront gets the number.
__device__ __forceinline__ int standing(const VerifyArgs& a, int b, int count) {
    const int lane = threadIdx.x & 63;
    for (int i0 = 0; i0 < a.D; i0 += 64) {
        const int i = i0 + lane;
        bool falls = i >= count;
        if (i < a.D) {   // loaded beside the count, whether it is used or not
            const long long t = a.tokens[(long long)b * a.D + i];
            const double u = a.uniforms[(long long)b * (a.D + 1) + i];
            if (t >= 0 && t < a.V) {
                const float q = a.draft[((long long)b * a.D + i) * a.V + t];
                const float p = a.target[((long long)b * (a.D + 1) + i) * a.V + t];
                falls = falls || !(u * (double)q < (double)p);
            } else {
                falls = true;
            }
        }
        const unsigned long long votes = __ballot(falls);
        if (votes) return min(i0 + __builtin_ctzll(votes), count);
    }
    return count;
}

// The part of a probability that counts: none of a NaN or a negative one.
__device__ __forceinline__ double above(double x) { return x > 0.0 ? x : 0.0; }

__device__ __forceinline__ double wave_sum64(double v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ double wave_scan64(double v) {   // inclusive
    const int lane = threadIdx.x & 63;
    for (int o = 1; o < 64; o <<= 1) {
        const double t = __shfl_up(v, o, 64);
        if (lane >= o) v += t;
    }
    return v;
}

// Rows start wherever V puts them: four floats on a 4-byte boundary.
struct __attribute__((packed, aligned(4))) Four {
    float v[4];
};
// Entries v .. v + 3 of a row of V, zeros behind it.
__device__ __forceinline__ Four four(const float* row, int v, int V) {
    Four f;
    if (v + 4 <= V) return *(const Four*)(row + v);
#pragma unroll
    for (int k = 0; k < 4; ++k) f.v[k] = v + k < V ? row[v + k] : 0.f;
    return f;
}

__global__ __launch_bounds__(64 * WAVES) void verify_sums(VerifyArgs a) {
    const int b = blockIdx.y, lane = threadIdx.x & 63;
    const int part = blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (part >= a.parts) return;
    const int count = min(max(a.count[b], 0), a.D);
    const int n = __builtin_amdgcn_readfirstlane(standing(a, b, count));
    const float* const p = a.target + ((long long)b * (a.D + 1) + n) * a.V;
    const float* const q = n < count ? a.draft + ((long long)b * a.D + n) * a.V : nullptr;
    Four x[EACH / 4], y[EACH / 4];
    const int v0 = part * PART + 4 * lane;
#pragma unroll
    for (int k = 0; k < EACH / 4; ++k) {
        x[k] = four(p, v0 + 256 * k, a.V);
        y[k] = q ? four(q, v0 + 256 * k, a.V) : Four{{0.f, 0.f, 0.f, 0.f}};
    }
    double sr = 0.0, sp = 0.0;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const float e = x[k / 4].v[k % 4];
        sr += above((double)e - (double)y[k / 4].v[k % 4]);
        sp += above(e);
    }
    sr = wave_sum64(sr);
    sp = wave_sum64(sp);
    if (lane < 2) a.sums[((long long)b * a.parts + part) * 2 + lane] = lane ? sp : sr;
    if (part == 0 && lane == 0) a.standing[b] = n;
}

// One wavefront a sequence.
__global__ __launch_bounds__(64) void verify_draw(VerifyArgs a) {
    const int b = blockIdx.x, lane = threadIdx.x;
    const int n = __builtin_amdgcn_readfirstlane(a.standing[b]);
    const int count = min(max(a.count[b], 0), a.D);
    const double u = a.uniforms[(long long)b * (a.D + 1) + a.D];
    const double* const sums = a.sums + (long long)b * a.parts * 2;
    long long* const out = a.out + (long long)b * (a.D + 1);
    double whole = 0.0, own = 0.0;
    for (int i = lane; i < a.parts; i += 64) {
        whole += sums[2 * i];
        own += sums[2 * i + 1];
    }
    for (int i = lane; i <= a.D; i += 64)
        if (i != n) out[i] = i < n ? a.tokens[(long long)b * a.D + i] : -1;
    whole = wave_sum64(whole);
    own = wave_sum64(own);
    const int which = whole > 0.0 ? 0 : 1;
    if (which) whole = own;
    if (!(whole > 0.0)) {   // nothing to draw from
        if (lane == 0) out[n] = -1;
        return;
    }
    // the first part whose running sum passes the mark, or the last with an entry
    const double mark = u * whole;
    double before = 0.0, full_before = 0.0;   // sums before the part, and before the last one with an entry
    int part = -1, full = 0;
    for (int i0 = 0; i0 < a.parts && part < 0; i0 += 64) {
        const double mine = i0 + lane < a.parts ? sums[2 * (i0 + lane) + which] : 0.0;
        const double run = wave_scan64(mine);
        const unsigned long long some = __ballot(mine > 0.0), passes = __ballot(mine > 0.0 && before + run > mark);
        if (passes) {
            part = i0 + __builtin_ctzll(passes);
            before += __shfl(run - mine, __builtin_ctzll(passes), 64);
        } else {
            if (some) {
                full = i0 + 63 - __builtin_clzll(some);
                full_before = before + __shfl(run - mine, 63 - __builtin_clzll(some), 64);
            }
            before += __shfl(run, 63, 64);
        }
    }
    if (part < 0) {
        part = full;
        before = full_before;
    }

    const float* const p = a.target + ((long long)b * (a.D + 1) + n) * a.V;
    const float* const q = !which && n < count ? a.draft + ((long long)b * a.D + n) * a.V : nullptr;
    const int v0 = part * PART + lane * EACH;
    double e[EACH], mine = 0.0;
    Four x[EACH / 4], y[EACH / 4];
#pragma unroll
    for (int k = 0; k < EACH / 4; ++k) {
        x[k] = four(p, v0 + 4 * k, a.V);
        y[k] = q ? four(q, v0 + 4 * k, a.V) : Four{{0.f, 0.f, 0.f, 0.f}};
    }
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        e[k] = above((double)x[k / 4].v[k % 4] - (double)y[k / 4].v[k % 4]);
        mine += e[k];
    }
    double at = before + (wave_scan64(mine) - mine);
    int pick = -1, last = -1;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        at += e[k];
        if (e[k] > 0.0) {
            last = v0 + k;
            if (at > mark && pick < 0) pick = v0 + k;
        }
    }
    const unsigned long long picks = __ballot(pick >= 0), lasts = __ballot(last >= 0);
    if (picks) last = __shfl(pick, __builtin_ctzll(picks), 64);
    else if (lasts) last = __shfl(last, 63 - __builtin_clzll(lasts), 64);
    if (lane == 0) out[n] = last;
}

// in[0..4] = target, draft, tokens, uniforms, count; i[0] = B, i[1] = D, i[2] = V, i[3] = parts
void launch_verify(const Step& s, hipStream_t st) {
    if (s.i[0] <= 0) return;
    VerifyArgs a;
    a.target = (const float*)s.in[0];
    a.draft = (const float*)s.in[1];
    a.tokens = (const long long*)s.in[2];
    a.uniforms = (const float*)s.in[3];
    a.count = (const int*)s.in[4];
    a.out = (long long*)s.out;
    a.D = (int)s.i[1];
    a.V = (int)s.i[2];
    a.parts = (int)s.i[3];
    a.sums = (double*)s.ws;
    a.standing = (int*)(a.sums + s.i[0] * a.parts * 2);
    hipLaunchKernelGGL(verify_sums, dim3((unsigned)((a.parts + WAVES - 1) / WAVES), (unsigned)s.i[0]), dim3(64 * WAVES), 0, st, a);
    hipLaunchKernelGGL(verify_draw, dim3((unsigned)s.i[0]), dim3(64), 0, st, a);
}

}  // namespace

int decode_verify_draft(const OpNode* n, Step* s) {
    if (n->n_inputs != 5 || !n->output || n->elem_size != 8 || n->n_dims != 2 || n->out_shape[1] < 1) {
        lbr_set_error("verify_draft: expected 5 inputs and an int64 output [B, D + 1]");
        return LBR_ERR_INVALID;
    }
    for (int k = 0; k < 5; ++k)
        if (!n->inputs[k] || !lbr_aligned(n->inputs[k], k == 2 ? 8 : 4)) {
            lbr_set_error("verify_draft: input %d is null or not aligned to its elements", k);
            return LBR_ERR_INVALID;
        }
    if (!lbr_aligned(n->output, 8)) {
        lbr_set_error("verify_draft: the output does not start on an 8-byte boundary");
        return LBR_ERR_INVALID;
    }
    const long long B = n->out_shape[0], D = n->out_shape[1] - 1, V = n->extra[0];
    if (V < 1 || V > (1 << 30) || B > 65535 || lbr_paged_input_bytes(n, 0) < 0) {
        lbr_set_error("verify_draft: %lld sequences of %lld tokens over a vocabulary of %lld", B, D, V);
        return LBR_ERR_INVALID;
    }
    for (int k = 0; k < 5; ++k) s->in[k] = n->inputs[k];
    s->out = n->output;
    s->i[0] = B;
    s->i[1] = D;
    s->i[2] = V;
    s->i[3] = (V + PART - 1) / PART;
    s->ws_bytes = (size_t)(B * s->i[3] * 2) * sizeof(double) + (size_t)B * sizeof(int);
    s->run = launch_verify;
    s->name = "verify_draft";
    return LBR_OK;
}
