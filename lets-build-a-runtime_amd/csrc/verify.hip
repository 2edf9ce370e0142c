// verify.hip — drafted tokens against the target's probabilities, from given random numbers.
//
// Token i (i < count) stands while u_i · draft_i[t_i] < target_i[t_i] and all before it stood; each
// product is of two floats and exact in 64 bits.  Behind the n that stand comes one drawn from
// r = max(target_n − draft_n, 0), or from target_n where all stand or r is zero everywhere: the first index
// whose running sum passes u_D · Σ r, sums in 64 bits.
//
// What bounds it: the two rows of V floats that r takes, of a sequence whose position n is known only
// from its first D probabilities.  So a first kernel lets every workgroup find n for itself (D loads, one
// vote) and sum one part of r; a second, one workgroup a sequence, finds the part in which the running
// sum passes and goes through that part alone again.
#include "lbr_device.h"

namespace {

constexpr int THREADS = 256, EACH = 16, PART = THREADS * EACH;   // entries of a part's pass

struct VerifyArgs {
    const float* target;
    const float* draft;
    const long long* tokens;
    const float* uniforms;
    const int* count;
    long long* out;
    double* sums;              // [B][parts][2]: of r, of the target's own row
    int D, V, parts;
};

// Tokens of sequence b that stand; every lane of the wavefront gets the number.
__device__ __forceinline__ int standing(const VerifyArgs& a, int b) {
    const int lane = threadIdx.x & 63;
    const int count = min(max(a.count[b], 0), a.D);
    for (int i0 = 0; i0 < count; i0 += 64) {
        const int i = i0 + lane;
        bool falls = false;
        if (i < count) {
            const long long t = a.tokens[(long long)b * a.D + i];
            falls = true;
            if (t >= 0 && t < a.V) {
                const double u = a.uniforms[(long long)b * (a.D + 1) + i];
                falls = !(u * (double)a.draft[((long long)b * a.D + i) * a.V + t] <
                          (double)a.target[((long long)b * (a.D + 1) + i) * a.V + t]);
            }
        }
        const unsigned long long votes = __ballot(falls);
        if (votes) return i0 + __builtin_ctzll(votes);
    }
    return count;
}

struct Rows {
    const float* p;
    const float* q;   // null: all stood
};

__device__ __forceinline__ Rows rows_of(const VerifyArgs& a, int b, int n) {
    const bool all = n >= min(max(a.count[b], 0), a.D);
    return {a.target + ((long long)b * (a.D + 1) + n) * a.V, all ? nullptr : a.draft + ((long long)b * a.D + n) * a.V};
}

// The part of a probability that counts: none of a NaN or a negative one.
__device__ __forceinline__ double above(double x) { return x > 0.0 ? x : 0.0; }

__device__ __forceinline__ double wave_sum64(double v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__global__ __launch_bounds__(THREADS) void verify_sums(VerifyArgs a) {
    __shared__ double red[2][THREADS / 64];
    const int b = blockIdx.y, tid = threadIdx.x;
    const Rows r = rows_of(a, b, standing(a, b));
    const int v0 = blockIdx.x * PART + tid;
    float p[EACH], q[EACH];
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const int v = v0 + k * THREADS;
        p[k] = v < a.V ? r.p[v] : 0.f;
        q[k] = r.q && v < a.V ? r.q[v] : 0.f;
    }
    double sr = 0.0, sp = 0.0;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        sr += above((double)p[k] - (double)q[k]);
        sp += above(p[k]);
    }
    sr = wave_sum64(sr);
    sp = wave_sum64(sp);
    if ((tid & 63) == 0) {
        red[0][tid >> 6] = sr;
        red[1][tid >> 6] = sp;
    }
    __syncthreads();
    if (tid < 2) {
        double t = 0.0;
        for (int w = 0; w < THREADS / 64; ++w) t += red[tid][w];
        a.sums[((long long)b * a.parts + blockIdx.x) * 2 + tid] = t;
    }
}

// One workgroup a sequence.  Parts are searched by thread 0's wavefront, then the part itself: thread t takes
// its entries t·EACH .. in order, and the sums before it come from a scan.
__global__ __launch_bounds__(THREADS) void verify_draw(VerifyArgs a) {
    __shared__ double wsum[THREADS / 64];
    __shared__ int pick, last;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = standing(a, b);
    const Rows r = rows_of(a, b, n);
    const double* const sums = a.sums + (long long)b * a.parts * 2;
    for (int i = tid; i <= a.D; i += THREADS)
        if (i != n) a.out[(long long)b * (a.D + 1) + i] = i < n ? a.tokens[(long long)b * a.D + i] : -1;

    // every wavefront for itself: the whole, and the first part whose running sum passes the mark
    double whole = 0.0;
    for (int i = lane; i < a.parts; i += 64) whole += sums[2 * i];
    whole = wave_sum64(whole);
    const int which = whole > 0.0 ? 0 : 1;
    if (which) {
        whole = 0.0;
        for (int i = lane; i < a.parts; i += 64) whole += sums[2 * i + 1];
        whole = wave_sum64(whole);
    }
    if (!(whole > 0.0)) {   // nothing to draw from
        if (tid == 0) a.out[(long long)b * (a.D + 1) + n] = -1;
        return;
    }
    const double mark = (double)a.uniforms[(long long)b * (a.D + 1) + a.D] * whole;
    double before = 0.0;    // of the parts before `part`
    int part = -1, full = 0;
    double full_before = 0.0;
    for (int i0 = 0; i0 < a.parts && part < 0; i0 += 64) {
        const double mine = i0 + lane < a.parts ? sums[2 * (i0 + lane) + which] : 0.0;
        double run = mine;   // inclusive scan
        for (int o = 1; o < 64; o <<= 1) {
            const double t = __shfl_up(run, o, 64);
            if (lane >= o) run += t;
        }
        const unsigned long long passes = __ballot(mine > 0.0 && before + run > mark);
        const unsigned long long some = __ballot(mine > 0.0);
        if (passes) {
            const int at = __builtin_ctzll(passes);
            part = i0 + at;
            before += __shfl(run - mine, at, 64);
        } else {
            if (some) {
                const int at = 63 - __builtin_clzll(some);
                full = i0 + at;
                full_before = before + __shfl(run - mine, at, 64);
            }
            before += __shfl(run, 63, 64);
        }
    }
    if (part < 0) {   // the mark is not below the whole: the last entry above zero
        part = full;
        before = full_before;
    }

    double e[EACH], mine = 0.0;
    const int v0 = part * PART + tid * EACH;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const int v = v0 + k;
        const double p = v < a.V ? (double)r.p[v] : 0.0;
        e[k] = above(which || !r.q || v >= a.V ? p : p - (double)r.q[v]);
        mine += e[k];
    }
    double run = mine;
    for (int o = 1; o < 64; o <<= 1) {
        const double t = __shfl_up(run, o, 64);
        if (lane >= o) run += t;
    }
    if (lane == 63) wsum[wave] = run;
    if (tid == 0) {
        pick = 0x7fffffff;
        last = -1;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) before += wsum[w];
    double at = before + (run - mine);
    int mine_pick = 0x7fffffff, mine_last = -1;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        at += e[k];
        if (e[k] > 0.0) {
            mine_last = v0 + k;
            if (at > mark && mine_pick == 0x7fffffff) mine_pick = v0 + k;
        }
    }
    if (mine_pick != 0x7fffffff) atomicMin(&pick, mine_pick);
    if (mine_last >= 0) atomicMax(&last, mine_last);
    __syncthreads();
    if (tid == 0) a.out[(long long)b * (a.D + 1) + n] = pick != 0x7fffffff ? pick : last;
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
    a.sums = (double*)s.ws;
    a.D = (int)s.i[1];
    a.V = (int)s.i[2];
    a.parts = (int)s.i[3];
    hipLaunchKernelGGL(verify_sums, dim3((unsigned)a.parts, (unsigned)s.i[0]), dim3(THREADS), 0, st, a);
    hipLaunchKernelGGL(verify_draw, dim3((unsigned)s.i[0]), dim3(THREADS), 0, st, a);
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
    s->ws_bytes = (size_t)(B * s->i[3] * 2) * sizeof(double);
    s->run = launch_verify;
    s->name = "verify_draft";
    return LBR_OK;
}
