// paged_attention.hip — attention of a chunk of new tokens over the paged cache.
#include "paged_common.h"

#include <math.h>

namespace {

constexpr int MAX_HD = 256;

// One workgroup a row of Q: scores of 256 keys at a time, the running maximum and sum of the softmax
// over them, and the weighted sum of the V rows, thread d holding column d.
template <int TYPE>
__global__ __launch_bounds__(256) void paged_rows(PagedCache c, const float* __restrict__ q, float* __restrict__ out,
                                                  int H, int S, float scale) {
    __shared__ float qs[MAX_HD], ps[256], red[4];
    const int row = blockIdx.x % S, bh = blockIdx.x / S;
    const int h = bh % H, b = bh / H, kvh = h / (H / c.heads);
    const int tid = threadIdx.x;
    const long long at = (long long)blockIdx.x * c.hd;
    const int start = c.start[b], count = min(max(c.count[b], 0), S);
    if (row >= count) {
        if (tid < c.hd) out[at + tid] = 0.f;
        return;
    }
    const long long keys = (long long)start + row + 1;
    if (start < 0 || keys > ((long long)c.wide << c.shift)) {
        if (tid < c.hd) out[at + tid] = __uint_as_float(0x7fc00000u);
        return;
    }
    if (tid < c.hd) qs[tid] = q[at + tid] * scale;
    constexpr int ES = cache_elem(TYPE);
    const int page = 1 << c.shift;
    auto value = [&](const char* p) {
        if constexpr (TYPE == LBR_CACHE_F32) return *(const float*)p;
        if constexpr (TYPE == LBR_CACHE_F16) return (float)*(const _Float16*)p;
        if constexpr (TYPE == LBR_CACHE_I8) return (float)*(const signed char*)p;
        if constexpr (TYPE == LBR_CACHE_E4M3)
            return __builtin_amdgcn_cvt_f32_fp8((int)*(const unsigned char*)p, 0);
    };
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (long long k0 = 0; k0 < keys; k0 += 256) {
        const long long key = k0 + tid;
        __syncthreads();
        float sc = -INFINITY;
        if (key < keys) {
            const char* head = cache_head(c, b, kvh, key);
            const int slot = (int)key & (page - 1);
            if (head) {
                float dot = 0.f;
                for (int d = 0; d < c.hd; ++d) dot += qs[d] * value(head + ((long long)slot * c.hdp + d) * ES);
                sc = dot * ((const float*)(head + 2 * c.part))[slot];
            } else {
                sc = __uint_as_float(0x7fc00000u);
            }
        }
        const bool nan = __syncthreads_or(sc != sc);
        const float mx = fmaxf(m, block_max(sc, red));
        const float p = nan ? __uint_as_float(0x7fc00000u) : expf(sc - mx);
        ps[tid] = p;
        const float sum = block_sum(p, red);
        const float alpha = expf(m - mx);
        l = l * alpha + sum;
        o *= alpha;
        m = mx;
        if (tid < c.hd)
            for (int j = 0; j < 256 && k0 + j < keys; ++j) {
                const char* head = cache_head(c, b, kvh, k0 + j);
                const int slot = (int)(k0 + j) & (page - 1);
                if (!head) continue;
                const float v = value(head + c.part + ((long long)(slot >> 3) * c.hdp + tid) * 8 * ES + (slot & 7) * ES);
                o += ps[j] * (v * ((const float*)(head + 2 * c.part))[page + slot]);
            }
    }
    if (tid < c.hd) out[at + tid] = o / l;
}

template <int TYPE>
void launch_rows(const Step& s, hipStream_t st) {
    const long long rows = s.i[1] * s.i[8] * s.i[7];
    if (rows <= 0) return;
    hipLaunchKernelGGL((paged_rows<TYPE>), dim3((unsigned)rows), dim3(256), 0, st, paged_cache(s),
                       (const float*)s.in[4], (float*)s.out, (int)s.i[8], (int)s.i[7], s.f[0]);
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
    s->run = s->i[0] == LBR_CACHE_F32   ? launch_rows<LBR_CACHE_F32>
             : s->i[0] == LBR_CACHE_F16 ? launch_rows<LBR_CACHE_F16>
             : s->i[0] == LBR_CACHE_I8  ? launch_rows<LBR_CACHE_I8>
                                        : launch_rows<LBR_CACHE_E4M3>;
    s->name = "paged_attention_rows";
    return LBR_OK;
}
